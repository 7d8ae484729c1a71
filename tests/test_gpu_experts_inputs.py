"""Expert operators on inputs that are not plain tensors, and on values where
sums and exponentials lose what matters.

Tolerances count roundings, as in test_gpu_experts.py."""
import pytest

import gloo_amd as ga

torch = pytest.importorskip("torch")

import torch.autograd.forward_ad as fw  # noqa: E402

from gloo_amd import experts as ex  # noqa: E402

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("no GPU", allow_module_level=True)

F8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
U = 2.0 ** -24  # half a step of fp32


def nb(n):
    return -(-n // 128)


def same(got, want):
    for a, b in zip(got, want):
        assert torch.equal(a.float(), b.float())


# ------------------------------------------------------------ negative views


def negative(gen, *shape):
    """Views whose values are the negated ones of their memory, as the
    imaginary part of a conjugate is: of stride 2, and adjacent."""
    z = torch.randn(shape, generator=gen, dtype=torch.complex64).cuda()
    views = [z.conj().imag, torch._neg_view(z.real.contiguous())]
    assert all(v.is_neg() for v in views)
    return views


def small_plan(t, k, e, gen):
    ids = torch.stack([torch.randperm(e, generator=gen)[:k]
                       for _ in range(t)]).to(torch.int32)
    return ex.plan(ids.cuda(), e)


@pytest.mark.parametrize("width", [1, 7, 64, 256])
def test_negative_views(width):
    gen = torch.Generator().manual_seed(width)
    t, k, e = 12, 2, 8
    p = small_plan(t, k, e, gen)
    for v in negative(gen, t, width):
        r = v.resolve_neg()
        same(ex.quantize_fp8(v), ex.quantize_fp8(r))
        same(ex.quantize_fp8(v.t()), ex.quantize_fp8(r.t()))
        same(ex.quantize_fp8(v, tile=True), ex.quantize_fp8(r, tile=True))
        same(ex.quantize_fp8(v.view(3, 4, width), tile=True),
             ex.quantize_fp8(r.view(3, 4, width), tile=True))
        same(ex.pack_fp8(v, p), ex.pack_fp8(r, p))
        same([ex.pack(v, p)], [ex.pack(r, p)])
        same(ex.route(v, 1), ex.route(r, 1))
        same(ex.route(r, 1, bias=v[0]), ex.route(r, 1, bias=r[0]))
    for w in negative(gen, t, k):
        rows = torch.randn(t * k, width, generator=gen).cuda()
        same([ex.combine(rows, p, w)], [ex.combine(rows, p, w.resolve_neg())])
    for rows in negative(gen, t * k, width):
        same([ex.combine(rows, p)], [ex.combine(rows.resolve_neg(), p)])


@pytest.mark.parametrize("width", [1, 64])
def test_gradients_of_negative_views(width):
    """As inputs, and as what the gradient of the outputs is."""
    gen = torch.Generator().manual_seed(width)
    t, k, e = 12, 2, 8
    p = small_plan(t, k, e, gen)
    x = torch.randn(t, width, generator=gen).cuda().requires_grad_()
    rows = torch.randn(t * k, width, generator=gen).cuda().requires_grad_()
    w = torch.rand(t, k, generator=gen).cuda().requires_grad_()
    z = torch.randn(t, e, generator=gen).cuda().requires_grad_()
    calls = [(lambda a: ex.pack(a, p), (x,), (t * k, width)),
             (lambda a, b: ex.combine(a, p, b), (rows, w), (t, width)),
             (lambda a: ex.combine(a, p), (rows,), (t, width)),
             (lambda a: ex.route(a, k)[0], (z,), (t, k))]
    for call, leaves, shape in calls:
        for g in negative(gen, *shape):
            got = torch.autograd.grad(call(*leaves), leaves, g)
            want = torch.autograd.grad(call(*leaves), leaves, g.resolve_neg())
            same(got, want)
        g = torch.randn(shape, generator=gen).cuda()
        for i, leaf in enumerate(leaves):
            for v in negative(gen, *leaf.shape):
                v = v.detach().requires_grad_()
                r = v.detach().resolve_neg().requires_grad_()
                got, want = (torch.autograd.grad(
                    call(*leaves[:i], y, *leaves[i + 1:]), y, g)
                    for y in (v, r))
                same(got, want)


# ------------------------------------------------------- forward-mode inputs


def test_forward_mode_is_refused():
    """A dual tensor's tangent would be lost without a word."""
    gen = torch.Generator().manual_seed(1)
    t, k, e = 12, 2, 8
    p = small_plan(t, k, e, gen)
    x = torch.randn(t, 64, generator=gen).cuda()
    rows = torch.randn(t * k, 64, generator=gen).cuda()
    w = torch.rand(t, k, generator=gen).cuda()
    q, s = ex.quantize_fp8(x)
    b, bs = ex.quantize_fp8(x, tile=True)
    with fw.dual_level():
        for grad in (False, True):
            def dual(v):
                return fw.make_dual(v.clone().requires_grad_(grad),
                                    torch.ones_like(v))

            calls = [lambda: ex.route(dual(x), 2),
                     lambda: ex.pack(dual(x), p),
                     lambda: ex.pack_fp8(dual(x), p),
                     lambda: ex.combine(dual(rows), p),
                     lambda: ex.combine(dual(rows), p, w),
                     lambda: ex.combine(rows, p, dual(w)),
                     lambda: ex.quantize_fp8(dual(x)),
                     lambda: ex.quantize_fp8(dual(x), tile=True),
                     lambda: ex.fp8_matmul(dual(q), s, b, bs),
                     lambda: ex.fp8_matmul(q, s, dual(b), bs),
                     lambda: ex.fp8_weight_grad(dual(q), s, q, s),
                     lambda: ex.fp8_weight_grad(q, s, dual(q), s)]
            for call in calls:
                with pytest.raises(ValueError, match="gradient"):
                    call()
        ex.pack(dual(x).detach(), p)  # its value alone


# ----------------------------------------------------------- router's weights


@pytest.mark.parametrize("gap", [0, 100, 700, 709, 720, 744, 746, 1000, 3e4])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("groups", [1, 4])
def test_renormalised_weights_far_below_the_top(gap, dtype, groups):
    """A bias keeps the largest logit out: weights are a softmax over the
    chosen ones, however far below it they are, and sum up to the scale."""
    gen = torch.Generator().manual_seed(int(gap))
    t, e, k, scale = 9, 16, 3, 2.5
    x = torch.randn(t, e, generator=gen).to(dtype).float() - gap
    x[:, 0] = 2.0
    x = x.to(dtype)
    bias = torch.linspace(1, 4, e)
    bias[0] = -9.0
    xg = x.cuda().requires_grad_()
    w, ids = ex.route(xg, k, bias=bias.cuda(), groups=groups,
                      topk_groups=groups, scale=scale)
    assert (ids > 0).all()
    g = torch.randn(t, k, generator=gen)
    dx, = torch.autograd.grad(w, xg, g.cuda())
    y = x.double().requires_grad_()
    ref = scale * torch.softmax(y.gather(1, ids.cpu().long()), 1)
    want, = torch.autograd.grad(ref, y, g.double())
    err = (w.detach().double().cpu() - ref.detach()).abs()
    assert (err <= ref * (U + 2.0 ** -44)).all(), err.max()
    half = torch.finfo(dtype).eps / 2
    slack = g.abs().max().item() * scale * k * 2.0 ** -40
    most = (want.abs() + slack) * (half + U) + slack
    assert ((dx.double().cpu() - want).abs() <= most).all()


# ------------------------------------------------- sums of 16-bit results


def off_by_one_large(rows, inner, gen):
    """One value of 448 in each block of 128, small ones of one sign: what is
    cut below the largest of a few products is missed in the sum."""
    x = torch.full((rows, nb(inner) * 128), 0.0234375)
    at = torch.randint(0, 128, (rows, nb(inner), 1), generator=gen)
    x.view(rows, nb(inner), 128).scatter_(2, at, 448.0)
    return x[:, :inner].contiguous()


SHAPES = [(1, 64, 128), (7, 130, 200), (16, 100, 300), (31, 70, 512),
          (40, 130, 128), (300, 516, 256), (1024, 1300, 384),
          (2500, 2570, 656), (4200, 4100, 2176)]


def check16(got, a, b, out):
    ref, size = a.double() @ b.double().t(), a.abs().double() @ \
        b.abs().double().t()
    half = torch.finfo(out).eps / 2
    # an addition in fp32 is off by a step at most; and fp16's smallest
    most = half * ref.abs() + (1 + half) * 2 * U * a.shape[1] * size + \
        2.0 ** -25
    err = (got.double() - ref).abs()
    assert (err <= most).all(), ((err - most).max().item(),
                                 (err / size.clamp_min(1e-30)).max().item())


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("kind", ["large", "random"])
def test_float16_products_are_summed_in_32_bits(m, n, k, kind):
    gen = torch.Generator().manual_seed(m + k)
    if kind == "large":
        a, b = off_by_one_large(m, k, gen), torch.ones(n, k)
    else:
        a = (torch.randn(m, k, generator=gen) * 4).to(F8).float()
        b = (torch.randn(n, k, generator=gen) * 4).to(F8).float()
    a, b = a.cuda(), b.cuda()
    qa, qb = a.to(F8), b.to(F8)
    sa = torch.full((m, nb(k)), 2.0 ** -6).to(E8).cuda()
    one = torch.ones(nb(n), nb(k)).to(E8).cuda()
    a = a * 2.0 ** -6
    got = ex.fp8_matmul(qa, sa, qb, one, dtype=torch.float16)
    check16(got, a, b, torch.float16)
    off = torch.tensor([0, m // 3, m // 3, m], dtype=torch.int32).cuda()
    got = ex.fp8_matmul(qa, sa, qb[None].expand(3, n, k),
                        one[None].expand(3, nb(n), nb(k)), offsets=off,
                        dtype=torch.float16)
    check16(got, a, b, torch.float16)
    ones = torch.ones(n, nb(k)).to(E8).cuda()
    got = ex.fp8_weight_grad(qa, sa, qb, ones, dtype=torch.float16)
    check16(got, a, b, torch.float16)
    at = [0, k // 3, k // 3, k]
    off = torch.tensor(at, dtype=torch.int32).cuda()
    got = ex.fp8_weight_grad(qa, sa, qb, ones, offsets=off,
                             dtype=torch.float16)
    for e in range(3):
        check16(got[e], a[:, at[e]:at[e + 1]], b[:, at[e]:at[e + 1]],
                torch.float16)


@pytest.mark.parametrize("out", [torch.float32, torch.float16,
                                 torch.bfloat16])
def test_products_repeat_themselves(out):
    """The same inputs give the same bits, call by call."""
    gen = torch.Generator().manual_seed(3)
    for m, n, k in ((1, 512, 4096), (16, 512, 1024), (256, 1024, 2048),
                    (4095, 1024, 512), (4096, 4096, 640)):
        a, sa = ex.quantize_fp8(torch.randn(m, k, generator=gen).cuda())
        b, sb = ex.quantize_fp8(
            torch.randn(n, k, generator=gen).cuda(), tile=True)
        x, sx = ex.quantize_fp8(torch.randn(n, k, generator=gen).cuda())
        runs = [(ex.fp8_matmul(a, sa, b, sb, dtype=out),
                 ex.fp8_weight_grad(a, sa, x, sx, dtype=out))
                for _ in range(3)]
        for run in runs[1:]:
            same(run, runs[0])


@pytest.mark.parametrize("out", [torch.float32, torch.float16,
                                 torch.bfloat16])
@pytest.mark.parametrize("experts,n", [(1, 72), (3, 16), (16, 1030),
                                       (16, 4096), (70, 1024), (70, 20)])
@pytest.mark.parametrize("inner", [16, 208, 1024, 4224])
def test_few_rows_of_experts(experts, n, inner, out):
    """Whole numbers, whose sums are exact, on either side of where tiles take
    over, with rows before the first expert's and behind the last one's."""
    gen = torch.Generator().manual_seed(experts + n + inner)
    b = torch.randint(-3, 4, (experts, n, inner), generator=gen).float()
    qb = b.cuda().to(F8)
    sb = torch.ones(experts, nb(n), nb(inner)).to(E8).cuda()
    for rows in range(1, 10):
        a = torch.randint(-3, 4, (rows, inner), generator=gen).float()
        at = torch.randint(0, rows + 1, (experts + 1,), generator=gen)
        at = torch.sort(at).values
        sa = torch.ones(rows, nb(inner)).to(E8).cuda()
        got = ex.fp8_matmul(a.cuda().to(F8), sa, qb, sb,
                            offsets=at.int().cuda(), dtype=out).cpu()
        want = torch.zeros(rows, n)
        for e in range(experts):
            part = slice(int(at[e]), int(at[e + 1]))
            if part.start < part.stop:
                want[part] = a[part] @ b[e].t()
        assert torch.equal(got, want.to(out)), rows


# ---------------------------------------------------------------- what is kept


def test_sums_without_weights_keep_no_rows():
    """Their gradient does not need them: they may change, and are free."""
    gen = torch.Generator().manual_seed(4)
    p = small_plan(12, 2, 8, gen)
    leaf = torch.randn(24, 64, generator=gen).cuda().requires_grad_()
    g = torch.randn(12, 64, generator=gen).cuda()
    want, = torch.autograd.grad(ex.combine(leaf * 1, p), leaf, g)
    rows = leaf * 1
    out = ex.combine(rows, p)
    rows.zero_()
    got, = torch.autograd.grad(out, leaf, g)
    assert torch.equal(got, want)


# ------------------------------------------------- refusals by the launches


def test_launches_that_are_too_large_are_wrong_arguments():
    one = torch.ones(1, device="cuda")
    with pytest.raises(ValueError):
        ex.quantize_fp8(one.expand(2 ** 24, 1, 1), tile=True)
    e, n = 65533, 257 * 128
    q, s = one.to(F8), one.to(E8)
    off = torch.zeros(e + 1, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        ex.fp8_weight_grad(q.expand(1, 8), s.expand(1, 1), q.expand(n, 8),
                           s.expand(n, 1), offsets=off,
                           dtype=torch.bfloat16)


def test_wrong_offsets_leave_what_is_around_the_result():
    """Offsets are read on the device. Wrong ones write nothing before or
    behind the result, which lies in the middle of a larger buffer here."""
    gen = torch.Generator().manual_seed(2)
    c = ga._C
    kinds = [(ga.DType.f32, torch.float32), (ga.DType.bf16, torch.bfloat16),
             (ga.DType.f16, torch.float16)]
    for rows in (3, 20, 700):
        e, n, k, margin = 3, 72, 256, 4096
        a, sa = ex.quantize_fp8(torch.randn(rows, k, generator=gen).cuda())
        b, sb = ex.quantize_fp8(
            torch.randn(e, n, k, generator=gen).cuda(), tile=True)
        x, sx = ex.quantize_fp8(torch.randn(n, rows, generator=gen).cuda())
        for at in ([-5, 3, 2 ** 31 - 1, 2 ** 30], [rows, 4, 2, 0],
                   [-2 ** 31, -1, -1, 99], [0, rows, 0, rows],
                   [2 ** 31 - 1] * 4):
            off = torch.tensor(at, dtype=torch.int32).cuda()
            for gdt, tdt in kinds:
                for grad in (False, True):
                    size = e * n * n if grad else rows * n
                    room = torch.full((size + 2 * margin,), 7.0, dtype=tdt,
                                      device="cuda")
                    out = room[margin:margin + size]
                    if grad:
                        c.hip_fp8_weight_grad(
                            x.data_ptr(), x.stride(0), sx.data_ptr(),
                            x.data_ptr(), x.stride(0), sx.data_ptr(),
                            off.data_ptr(), n, n, rows, e, out.data_ptr(),
                            gdt, 0, 0)
                    else:
                        c.hip_fp8_matmul(
                            a.data_ptr(), a.stride(0), sa.data_ptr(),
                            b.data_ptr(), b.stride(1), b.stride(0),
                            sb.data_ptr(), off.data_ptr(), rows, n, k, e,
                            out.data_ptr(), gdt, 0, 0)
                    torch.cuda.synchronize()
                    assert (room[:margin] == 7).all()
                    assert (room[margin + size:] == 7).all()
