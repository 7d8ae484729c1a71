"""Operators of expert-parallel layers, on either side of an alltoallv.

    weights, ids = route(logits, k)           # which experts, how much
    p = plan(ids, num_experts)                # token copies, by expert
    rows = pack(x, p)                         # the alltoallv's send buffer
    ...                                       # the experts
    out = combine(rows, p, weights)           # back to tokens

`pack_fp8` packs in 8 bits with a scale for each block of 128 instead, and
`fp8_matmul` multiplies such rows by their experts' weights; `ExpertExchange`
runs the whole way over a process group. All operators are hand-written HIP
kernels (csrc/hip/experts.hip, csrc/hip/fp8.hip, called by csrc/torch) that
run asynchronously on the current stream of their tensors' device, allocate
with torch's allocator and may be captured into a graph (a backward pass only
while no autograd graph of the same leaves from outside the capture is alive,
as torch has it). Tensors have to be on a GPU; wrong arguments raise
ValueError before anything is launched, and so do inputs with a forward-mode
gradient, which no operator has.

8-bit values are torch.float8_e4m3fn. Their scales are powers of two
(torch.float8_e8m0fnu): the least that brings a block's largest value to 448
or less, 2^-127 at least, 2^0 for a block of zeros and NaN for one that holds
inf or NaN.
"""
from typing import NamedTuple, Optional

import torch
import torch.distributed as dist

import gloo_amd as ga
from gloo_amd import _operators as _ops

_C = ga._C
_ops.set_launchers(_C.expert_launchers())

FP8 = torch.float8_e4m3fn
FP8_SCALE = torch.float8_e8m0fnu
FP8_BLOCK = 128
_FP8_EXPERTS = 65533  # of the 8-bit products
_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


class ExpertPlan(NamedTuple):
    """Token copies sorted by expert, in order of tokens within one.

    position [tokens, k] int32: a copy's row. A copy for no expert stands
        behind all others, and its row r is told as ~r, a negative number.
    counts [experts] int32: copies of each expert.
    offsets [experts + 1] int32: where each expert's rows begin; the last
        one is the number of copies that have an expert.
    """
    position: torch.Tensor
    counts: torch.Tensor
    offsets: torch.Tensor


def _tensor(t, name, dim, dtypes, like=None):
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name}: a tensor is needed")
    if t.dim() != dim:
        raise ValueError(f"{name}: {dim} dimensions are needed, got "
                         f"{tuple(t.shape)}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name}: one of {[str(d) for d in dtypes]} is "
                         f"needed, got {t.dtype}")
    if like is not None and t.device != like.device:
        raise ValueError(f"{name}: is on {t.device}, and others are on "
                         f"{like.device}")


def _gpu(t, name):
    """The last check before a launch: the others hold on any device."""
    if not t.is_cuda:
        raise ValueError(
            f"{name}: tensors on a GPU are needed, got {t.device}")


def _stream(t):
    """The current stream's handle alone: a Stream object takes 2 us."""
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def _differentiated(*tensors):
    return torch.is_grad_enabled() and any(
        t is not None and t.requires_grad for t in tensors)


def _once():
    """Backward passes run in grad mode only where they are to be
    differentiated themselves."""
    if torch.is_grad_enabled():
        raise RuntimeError("the expert operators' gradients cannot be "
                           "differentiated again (create_graph=True)")


def _blocks(n):
    return (n + FP8_BLOCK - 1) // FP8_BLOCK


# ------------------------------------------------------------------- router


def route(logits, k, *, score="softmax", bias=None, groups=1, topk_groups=1,
          group_score="max", renormalize=True, scale=1.0):
    """The k experts of each token and their weights.

    logits [tokens, experts] in float32, float16 or bfloat16. Scores are
    their softmax or sigmoid. The k experts with the largest score + bias
    (bias [experts] float32; without one, with the largest logits) are
    chosen, ties go to the lower number, and they are listed from the best
    on. With groups > 1 the experts are parted into groups of adjacent ones,
    and only those of the topk_groups best groups can be chosen; a group is
    as good as its best expert ("max") or as its two best ones' sum
    ("top2"). The bias takes part in the choice only: a chosen expert's
    weight is its score, divided by the sum of the chosen ones' where
    `renormalize` is set, times `scale`.

    An expert whose logit or bias is -inf or NaN is never chosen: where a
    token has fewer experts than k, the others are -1, with weight 0. A logit
    of +inf counts as the largest float32.

    Returns (weights [tokens, k] float32, experts [tokens, k] int32). The
    weights are differentiable with respect to the logits.
    """
    _tensor(logits, "logits", 2, _FLOATS)
    tokens, experts = logits.shape
    if not 1 <= experts <= _C.MAX_EXPERTS:
        raise ValueError(
            f"route: 1 to {_C.MAX_EXPERTS} experts, got {experts}")
    if tokens >= 2 ** 26 - 4:
        raise ValueError(f"route: fewer than 2^26 - 4 tokens, got {tokens}")
    if not 1 <= k <= min(experts, _C.MAX_TOPK):
        raise ValueError(
            f"route: k is 1 to {min(experts, _C.MAX_TOPK)} here, got {k}")
    if score not in ("softmax", "sigmoid"):
        raise ValueError(
            f"route: score is 'softmax' or 'sigmoid', got {score!r}")
    if group_score not in ("max", "top2"):
        raise ValueError(
            f"route: group_score is 'max' or 'top2', got {group_score!r}")
    if not 1 <= groups <= _C.MAX_EXPERT_GROUPS or experts % groups != 0:
        raise ValueError(
            f"route: {experts} experts in {groups} equal groups (at most "
            f"{_C.MAX_EXPERT_GROUPS})")
    if not 1 <= topk_groups <= groups:
        raise ValueError(
            f"route: topk_groups is 1 to {groups}, got {topk_groups}")
    if groups != 1 and k > topk_groups * (experts // groups):
        raise ValueError(
            f"route: {topk_groups} groups of {experts // groups} experts hold "
            f"fewer than k = {k}")
    if bias is not None:
        _tensor(bias, "bias", 1, (torch.float32,), logits)
        if bias.shape[0] != experts:
            raise ValueError(
                f"bias: {experts} values are needed, got {bias.shape[0]}")
        bias = bias.detach().contiguous()
    _gpu(logits, "route")
    return _ops.route(
        logits, bias, k, score == "sigmoid", groups, topk_groups,
        group_score == "top2", bool(renormalize), float(scale),
        _stream(logits))


# ------------------------------------------------- plan, pack and combine


def plan(experts, num_experts):
    """Sorts token copies by expert (stable). experts [tokens, k] int32, as
    `route` gives them; numbers outside [0, num_experts) are no expert."""
    _tensor(experts, "experts", 2, (torch.int32,))
    if not 1 <= num_experts <= _C.MAX_EXPERTS:
        raise ValueError(
            f"plan: 1 to {_C.MAX_EXPERTS} experts, got {num_experts}")
    if experts.numel() >= 2 ** 31:
        raise ValueError(f"plan: fewer than 2^31 token copies, got "
                         f"{experts.numel()}")
    _gpu(experts, "plan")
    return ExpertPlan(*_ops.plan(experts, num_experts, _stream(experts)))


def _check_plan(p, tokens, like):
    position = p.position
    _tensor(position, "plan.position", 2, (torch.int32,), like)
    if not position.is_contiguous():
        raise ValueError("plan.position has to be contiguous")
    if tokens is not None and position.shape[0] != tokens:
        raise ValueError(
            f"the plan is for {position.shape[0]} tokens, got {tokens}")
    if (position.shape[1] <= 0 or position.numel() >= 2 ** 31
            or position.shape[0] >= 2 ** 24):
        raise ValueError(f"plan.position: at least one copy of a token, and "
                         f"fewer than 2^24 tokens and 2^31 copies, got "
                         f"{tuple(position.shape)}")
    if like.shape[1] > 2 ** 23:
        raise ValueError(f"rows: at most 2^23 elements, got {like.shape[1]}")
    return position


def pack(x, plan):
    """Copies tokens to their rows: rows[plan.position[t, j]] = x[t].

    x [tokens, hidden] in float32, float16 or bfloat16; returns [tokens * k,
    hidden]. The rows of copies for no expert, behind plan.offsets[-1], are
    zeros. Differentiable."""
    _tensor(x, "x", 2, _FLOATS)
    position = _check_plan(plan, x.shape[0], x)
    _gpu(x, "pack")
    return _ops.pack(x, position, _stream(x))


def pack_fp8(x, plan):
    """`pack` in 8 bits: (rows [tokens * k, hidden] float8_e4m3fn, scales
    [tokens * k, ceil(hidden / 128)] float8_e8m0fnu), quantised as
    `quantize_fp8` does it, in the same pass over x. Rows of copies for no
    expert are zeros, with scales of 1. It has no gradient."""
    _tensor(x, "x", 2, _FLOATS)
    _no_gradient("pack_fp8", x)
    position = _check_plan(plan, x.shape[0], x)
    _gpu(x, "pack_fp8")
    return _ops.pack_fp8(x, position, _stream(x))


def combine(rows, plan, weights=None):
    """Adds each token's rows up: out[t] = sum over j of weights[t, j] *
    rows[plan.position[t, j]], in float32 and rounded once; copies for no
    expert count nothing, and neither rows nor weights of theirs are read.

    rows [tokens * k, hidden] in float32, float16 or bfloat16, weights
    [tokens, k] float32 (all 1 if None); returns [tokens, hidden].
    Differentiable with respect to rows and weights."""
    _tensor(rows, "rows", 2, _FLOATS)
    position = _check_plan(plan, None, rows)
    if rows.shape[0] != position.numel():
        raise ValueError(
            f"rows: the plan has {position.numel()}, got {rows.shape[0]}")
    if weights is not None:
        _tensor(weights, "weights", 2, (torch.float32,), rows)
        if weights.shape != position.shape:
            raise ValueError(
                f"weights: {tuple(position.shape)} is needed, got "
                f"{tuple(weights.shape)}")
        weights = weights.contiguous()  # a part of the gradient's way
    _gpu(rows, "combine")
    return _ops.combine(rows, position, weights, _stream(rows))


# ------------------------------------------------------------ 8-bit products


def _no_gradient(name, *tensors):
    if _differentiated(*tensors):
        raise ValueError(f"{name} has no gradient: detach() its inputs")


def quantize_fp8(x, tile=False):
    """8-bit values of x and their scales: x is about q * scale.

    x [rows, cols] in float32, float16 or bfloat16, of any strides. A scale
    is for 128 elements of a row: returns (q [rows, cols] float8_e4m3fn,
    scales [rows, ceil(cols / 128)] float8_e8m0fnu). With `tile` it is for
    128 x 128 elements, as weights have it, scales are [ceil(rows / 128),
    ceil(cols / 128)], and x may have a leading dimension for experts. For
    scales along the columns (a weight gradient's operands) quantise x.t().
    Rows of q begin on borders of 128 bytes. It has no gradient."""
    three = tile and isinstance(x, torch.Tensor) and x.dim() == 3
    _tensor(x, "x", 3 if three else 2, _FLOATS)
    _no_gradient("quantize_fp8", x)
    if x.shape[-1] > 65535 * FP8_BLOCK:
        raise ValueError(f"quantize_fp8: at most {65535 * FP8_BLOCK} "
                         f"columns, got {x.shape[-1]}")
    if x.shape[-2] * _blocks(x.shape[-1]) >= 2 ** 29 - 32:
        raise ValueError(f"quantize_fp8: fewer than 2^29 - 32 blocks, got "
                         f"{tuple(x.shape)}")
    _gpu(x, "quantize_fp8")
    return _ops.quantize_fp8(x, bool(tile), _stream(x))


def _fp8_operand(q, scale, name, dim, scale_shape, like=None):
    _tensor(q, name, dim, (FP8,), like)
    _tensor(scale, f"{name}_scale", dim, (FP8_SCALE,), q)
    if tuple(scale.shape) != scale_shape:
        raise ValueError(f"{name}_scale: {scale_shape} is needed, got "
                         f"{tuple(scale.shape)}")


def _offsets(offsets, experts, like):
    if offsets is None:
        return
    _tensor(offsets, "offsets", 1, (torch.int32,), like)
    if offsets.shape[0] != experts + 1 or not offsets.is_contiguous():
        raise ValueError(f"offsets: {experts + 1} adjacent numbers are "
                         f"needed, got {tuple(offsets.shape)}")


def fp8_matmul(a, a_scale, b, b_scale, offsets=None, dtype=torch.bfloat16):
    """Products of rows with weights in 8 bits: a b^T, or each expert's.

    a [rows, inner] float8_e4m3fn with a scale for each 128 of a row
    (a_scale [rows, ceil(inner / 128)] float8_e8m0fnu), b [n, inner] with one
    for each 128 x 128 (b_scale [ceil(n / 128), ceil(inner / 128)]): returns
    [rows, n] in `dtype` (float32, float16 or bfloat16), added up in float32
    and rounded once. For bfloat16 the matrix unit adds groups of eight
    products in fewer bits first: a product's bits below 2^-13 of its group's
    largest are lost, which halves the time of the exact sums that float32
    and float16 get. With `offsets` (int32 [experts + 1], a plan's) b and
    b_scale have a leading dimension for experts, and rows offsets[e] to
    offsets[e + 1] are multiplied by b[e]; rows before the first expert's (some
    of a plan's experts will do) and behind the last one's are zeros. The data
    gradient is the same product with the weights' transposed copy, and
    `fp8_weight_grad` is the other one: operands that want a gradient are
    refused."""
    if not isinstance(a, torch.Tensor) or a.dim() != 2:
        raise ValueError("a: a tensor of 2 dimensions is needed")
    if (not isinstance(b, torch.Tensor)
            or b.dim() != (2 if offsets is None else 3)):
        raise ValueError("b: [n, inner], or [experts, n, inner] with offsets")
    if dtype not in _FLOATS:
        raise ValueError(f"fp8_matmul: cannot return {dtype}")
    rows, inner = a.shape
    n = b.shape[-2]
    experts = 1 if offsets is None else b.shape[0]
    if b.shape[-1] != inner:
        raise ValueError(
            f"b: an inner dimension of {inner} is needed, got {b.shape[-1]}")
    if n <= 0 or not 0 < experts <= _FP8_EXPERTS:
        raise ValueError(f"b: 1 to {_FP8_EXPERTS} experts, got "
                         f"{tuple(b.shape)}")
    _fp8_operand(a, a_scale, "a", 2, (rows, _blocks(inner)))
    _fp8_operand(b, b_scale, "b", b.dim(),
                 tuple(b.shape[:-2]) + (_blocks(n), _blocks(inner)), a)
    _offsets(offsets, experts, a)
    _no_gradient("fp8_matmul", a, a_scale, b, b_scale)
    _gpu(a, "fp8_matmul")
    return _ops.fp8_matmul(a, a_scale, b, b_scale, offsets, dtype,
                           _stream(a))


def fp8_weight_grad(dy, dy_scale, x, x_scale, offsets=None,
                    dtype=torch.float32):
    """The weights' gradient dy x^T in 8 bits, or each expert's.

    dy [m, rows] and x [n, rows] float8_e4m3fn with a scale for each 128 of
    the rows (dy_scale [m, ceil(rows / 128)], x_scale [n, ...]), which is
    what quantize_fp8 makes of the transposed matrices: returns [m, n] in
    `dtype`, added up and rounded as `fp8_matmul` does it. With `offsets` (int32
    [experts + 1]) rows offsets[e] to offsets[e + 1] are expert e's, and the
    result is [experts, m, n], zeros for an expert without rows. Experts may
    begin anywhere: two of them can share a block and its scale. It has no
    gradient."""
    if (not isinstance(dy, torch.Tensor) or dy.dim() != 2 or not
            isinstance(x, torch.Tensor) or x.dim() != 2):
        raise ValueError("dy, x: tensors of 2 dimensions are needed")
    if dtype not in _FLOATS:
        raise ValueError(f"fp8_weight_grad: cannot return {dtype}")
    (m, rows), n = dy.shape, x.shape[0]
    if x.shape[1] != rows:
        raise ValueError(f"x: {rows} rows are needed, got {x.shape[1]}")
    if m <= 0 or n <= 0:
        raise ValueError(f"dy, x: got {tuple(dy.shape)}, "
                         f"{tuple(x.shape)}")
    _fp8_operand(dy, dy_scale, "dy", 2, (m, _blocks(rows)))
    _fp8_operand(x, x_scale, "x", 2, (n, _blocks(rows)), dy)
    if offsets is not None and (
            not isinstance(offsets, torch.Tensor) or offsets.dim() != 1
            or not 2 <= offsets.shape[0] <= _FP8_EXPERTS + 1):
        raise ValueError(f"offsets: [experts + 1] is needed, for 1 to "
                         f"{_FP8_EXPERTS} experts")
    _offsets(offsets, 0 if offsets is None else offsets.shape[0] - 1, dy)
    _no_gradient("fp8_weight_grad", dy, dy_scale, x, x_scale)
    _gpu(dy, "fp8_weight_grad")
    return _ops.fp8_weight_grad(dy, dy_scale, x, x_scale, offsets, dtype,
                                _stream(dy))


# ------------------------------------------------------- over a process group


def _alltoall(pg, rows, send, recv):
    """Rows [sum(send), ...] to the ranks in turn; returns [sum(recv), ...]."""
    out = rows.new_empty((sum(recv),) + rows.shape[1:])
    if pg.size() == 1:
        return out.copy_(rows)
    # by memory: a negative view's would be the values' opposite
    pg.alltoall_base(out, rows.resolve_neg().contiguous(), recv, send,
                     dist.AllToAllOptions()).wait()
    return out


class _AllToAll(torch.autograd.Function):
    @staticmethod
    def forward(ctx, pg, rows, send, recv):
        ctx.way = pg, send, recv
        return _alltoall(pg, rows.detach(), send, recv)

    @staticmethod
    def backward(ctx, grad):
        _once()
        pg, send, recv = ctx.way
        return None, _alltoall(pg, grad, recv, send), None, None


class ExpertBatch(NamedTuple):
    """What a rank's experts are given, and the way back.

    rows [n, hidden]: the token copies for this rank's experts, from all
        ranks, by expert; scales [n, ceil(hidden / 128)] with 8-bit rows.
    offsets [experts of a rank + 1] int32: where each expert's rows begin.
    """
    rows: torch.Tensor
    scales: Optional[torch.Tensor]
    offsets: torch.Tensor
    sent: ExpertPlan
    received: ExpertPlan
    send: list
    recv: list


class ExpertExchange:
    """Token copies to the ranks that hold their experts, and back.

        exchange = ExpertExchange(num_experts, group)
        weights, ids = route(logits, k)
        batch = exchange.dispatch(x, ids)
        y = ...                       # of batch.rows, by batch.offsets
        out = exchange.combine(y, batch, weights)

    Rank r of `group` (a "glooamd" process group, the default one if None)
    holds experts r * E / size to (r + 1) * E / size - 1. Each rank packs its
    tokens by expert, the counts travel as a small alltoall of host tensors,
    the rows as one alltoall with split sizes, and what arrives from the ranks
    is packed by expert again. An alltoall with split sizes goes through host
    memory and the CPU transport in this backend: dispatch, combine and their
    backward passes wait for the GPU and copy their rows there and back (a
    group of one rank does not).
    All ranks call both methods, ranks without tokens too, with rows of one
    length and type. With 16- or 32-bit rows the whole way is differentiable,
    and all ranks run its backward pass; with `fp8` the rows and their scales
    travel in 8 bits.
    """

    def __init__(self, num_experts, group=None):
        self._pg = group
        if group is None:
            self._pg = dist.distributed_c10d._get_default_group()
        size = self._pg.size()
        if num_experts < 1 or num_experts % size:
            raise ValueError(f"ExpertExchange: {num_experts} experts over "
                             f"{size} ranks")
        if num_experts > _C.MAX_EXPERTS:
            raise ValueError(f"ExpertExchange: at most {_C.MAX_EXPERTS} "
                             f"experts, got {num_experts}")
        self.num_experts = num_experts
        self.local_experts = num_experts // size

    def _counts(self, counts):
        """Copies of each local expert that each rank sends: a host tensor
        [size, local experts], and this rank's own counts like it."""
        mine = counts.view(-1, self.local_experts)
        theirs = _alltoall(self._pg, mine, [1] * len(mine), [1] * len(mine))
        return mine, theirs

    def dispatch(self, x, experts, fp8=False):
        """x [tokens, hidden], experts [tokens, k] int32 (-1: none): an
        ExpertBatch with this rank's experts' rows."""
        _tensor(x, "x", 2, _FLOATS)
        _tensor(experts, "experts", 2, (torch.int32,), x)
        if x.shape[1] < 1:
            raise ValueError(f"x: rows of one element at least, got "
                             f"{tuple(x.shape)}")
        if experts.shape[0] != x.shape[0] or experts.shape[1] < 1:
            raise ValueError(f"experts: one row a token, got "
                             f"{tuple(experts.shape)} for {x.shape[0]}")
        _gpu(x, "dispatch")
        if fp8:
            _no_gradient("dispatch(fp8=True)", x)
        hidden = x.shape[1]
        sent = plan(experts, self.num_experts)
        mine, theirs = self._counts(sent.counts.cpu())
        send, recv = mine.sum(1).tolist(), theirs.sum(1).tolist()
        if fp8:
            rows = _joined(*pack_fp8(x, sent))[:sum(send)]
        else:
            rows = pack(x, sent)[:sum(send)]
        rows = _AllToAll.apply(self._pg, rows, send, recv)
        # from each rank its rows for the first expert, the second ...
        ids = torch.arange(self.local_experts, dtype=torch.int32)
        ids = ids.repeat(len(theirs)).repeat_interleave(theirs.reshape(-1))
        received = plan(ids.view(-1, 1).to(x.device), self.local_experts)
        scales = None
        if fp8:
            rows = pack(rows.view(torch.float32), received)
            rows, scales = _parted(rows.view(torch.uint8), hidden)
        else:
            rows = pack(rows, received)
        return ExpertBatch(rows, scales, received.offsets, sent, received,
                           send, recv)

    def combine(self, rows, batch, weights=None):
        """The experts' results for batch.rows (float32, float16 or
        bfloat16) back to the tokens: their sum by `weights` [tokens, k]."""
        _tensor(rows, "rows", 2, _FLOATS, batch.offsets)
        if rows.shape[0] != sum(batch.recv):
            raise ValueError(f"rows: the batch has {sum(batch.recv)}, got "
                             f"{rows.shape[0]}")
        rows = combine(rows, batch.received)  # one row each: a permutation
        rows = _AllToAll.apply(self._pg, rows, batch.recv, batch.send)
        none = batch.sent.position.numel() - rows.shape[0]
        if none:  # places of copies for no expert
            rows = torch.cat([rows, rows.new_zeros(none, rows.shape[1])])
        return combine(rows, batch.sent, weights)


def _joined(q, scales):
    """8-bit rows and their scales as rows of bytes, 16 at a time."""
    n, wide = q.shape[0], _blocks(q.shape[1]) * FP8_BLOCK
    rest = (scales.shape[1] + 15) // 16 * 16
    out = torch.zeros(n, wide + rest, dtype=torch.uint8, device=q.device)
    out[:, :q.shape[1]] = q.view(torch.uint8)
    out[:, wide:wide + scales.shape[1]] = scales.view(torch.uint8)
    return out


def _parted(rows, hidden):
    blocks = _blocks(hidden)
    wide = blocks * FP8_BLOCK
    scales = rows[:, wide:wide + blocks].contiguous()
    return rows[:, :hidden].view(FP8), scales.view(FP8_SCALE)
