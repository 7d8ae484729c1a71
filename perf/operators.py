"""Cases that measure the expert-parallel operators of gloo_amd.experts.

An expert-parallel layer routes each token to k experts (route), sorts the
token copies by expert into the send buffer of an alltoallv (plan + pack, in
the tokens' type or in 8 bits with a scale for each block of 128), multiplies
the received rows by their expert's weights (fp8_matmul; fp8_weight_grad for
training) and adds the results back per token (combine).

A case is one pass through one of these. run() computes it in elementary
torch operations, or, where `own` is true, with the framework's operators.
"""
import torch

own = False

BLOCK = 128  # elements that share a scale
FP8 = torch.float8_e4m3fn  # the values: up to 448
E8M0 = torch.float8_e8m0fnu  # the scales: powers of two, 2^-127 and up
DTYPES = {"float32": torch.float32, "float16": torch.float16,
          "bfloat16": torch.bfloat16}


def listed():
    return [
        # Decoding: the router of a layer of 256 experts in 8 node groups
        # sees a handful of tokens; latency is all that counts.
        {"name": "route_decode", "op": "route", "tokens": 8, "experts": 256,
         "k": 8, "score": "sigmoid", "bias": True, "groups": 8,
         "topk_groups": 4, "group_score": "top2", "renormalize": True,
         "scale": 2.5, "dtype": "float32", "padded": 0, "backward": False},
        # Training: the same router over a rank's whole batch, with the
        # gradient of its logits; the last rows are padding.
        {"name": "route_train", "op": "route", "tokens": 16381,
         "experts": 256, "k": 8, "score": "sigmoid", "bias": True,
         "groups": 8, "topk_groups": 4, "group_score": "top2",
         "renormalize": True, "scale": 2.5, "dtype": "float32",
         "padded": 61, "backward": True},
        # Decoding: 32 tokens to 256 experts, 8-bit rows for the wire.
        {"name": "dispatch_decode", "op": "dispatch", "tokens": 32,
         "experts": 256, "k": 8, "hidden": 4096, "dtype": "bfloat16",
         "fp8": True, "padded": 0, "backward": False},
        # Training: a rank's batch in bf16, and the tokens' gradient.
        {"name": "dispatch_train", "op": "dispatch", "tokens": 16384,
         "experts": 64, "k": 4, "hidden": 4096, "dtype": "bfloat16",
         "fp8": False, "padded": 0, "backward": True},
        # Prefill of a ragged batch, 8-bit rows, the last rows padding.
        {"name": "dispatch_prefill", "op": "dispatch", "tokens": 8190,
         "experts": 256, "k": 8, "hidden": 5120, "dtype": "bfloat16",
         "fp8": True, "padded": 37, "backward": False},
        # The way back of the decoding step, and of the training step with
        # the gradients of rows and weights.
        {"name": "combine_decode", "op": "combine", "tokens": 32,
         "experts": 256, "k": 8, "hidden": 4096, "dtype": "bfloat16",
         "padded": 0, "backward": False},
        {"name": "combine_train", "op": "combine", "tokens": 16384,
         "experts": 64, "k": 4, "hidden": 4096, "dtype": "bfloat16",
         "padded": 0, "backward": True},
        # One token through the expert that all tokens share.
        {"name": "product_token", "op": "product", "rows": 1, "n": 8192,
         "inner": 4096, "experts": 0, "out": "bfloat16"},
        # The same expert over a prefill.
        {"name": "product_dense", "op": "product", "rows": 4095, "n": 8192,
         "inner": 4096, "experts": 0, "out": "bfloat16"},
        # Decoding: a few rows for each of a rank's 64 experts.
        {"name": "product_grouped_decode", "op": "product", "rows": 256,
         "n": 4096, "inner": 2048, "experts": 64, "out": "bfloat16"},
        # Prefill: ragged groups of a few hundred rows for each expert.
        {"name": "product_grouped", "op": "product", "rows": 16384,
         "n": 4096, "inner": 4096, "experts": 32, "out": "bfloat16"},
        # Training: every expert's weight gradient from its ragged rows.
        {"name": "weight_grad", "op": "weight_grad", "rows": 16384,
         "m": 4096, "n": 2048, "experts": 16, "out": "float32"},
    ]


def _log(rng, low, high):
    """A whole number from low to high, spread over its logarithm."""
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    op = rng.choice(["route", "dispatch", "combine", "product", "product",
                     "weight_grad"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    padded = rng.choice([0, 0, 5, 64])
    if op == "route":
        per, groups = rng.choice([(32, 8), (16, 4), (64, 1), (128, 1), (8, 1),
                                  (24, 6), (20, 8), (17, 3)])
        experts = per * groups
        kept = rng.randint(1, groups)
        tokens = _log(rng, 1, 16384)
        k = rng.randint(1, min(8, kept * per))
        return {"op": op, "tokens": tokens, "experts": experts, "k": k,
                "score": rng.choice(["softmax", "sigmoid"]),
                "bias": rng.random() < 0.5, "groups": groups,
                "topk_groups": kept,
                "group_score": rng.choice(["max", "top2"]),
                # one weight alone is always renormalised to the scale
                "renormalize": k > 1 and rng.random() < 0.7,
                "scale": rng.choice([1.0, 2.5]), "dtype": dtype,
                "padded": min(padded, tokens // 2),
                "backward": rng.random() < 0.5}
    if op in ("dispatch", "combine"):
        hidden = rng.choice([512, 1000, 1024, 2048, 2880, 4096, 5120, 8192])
        k = rng.randint(1, 8)
        tokens = _log(rng, 1, min(16384, 2 ** 28 // (hidden * k)))
        case = {"op": op, "tokens": tokens,
                "experts": rng.choice([8, 16, 60, 64, 128, 256]), "k": k,
                "hidden": hidden, "dtype": dtype,
                "padded": min(padded, tokens // 2),
                "backward": rng.random() < 0.5}
        if op == "dispatch":
            case["fp8"] = not case["backward"]
        return case
    if op == "product":
        return {"op": op, "rows": _log(rng, 1, 16384),
                "n": rng.choice([512, 1000, 1024, 1536, 2048, 2816, 4096]),
                "inner": 16 * rng.choice([32, 44, 64, 88, 125, 128, 256]),
                "experts": rng.choice([0, 8, 16, 32]),
                "out": rng.choice(["bfloat16", "float16", "float32"])}
    return {"op": op, "rows": _log(rng, 32, 16384),
            "m": rng.choice([256, 1000, 1024, 1408, 2048]),
            "n": rng.choice([512, 1024, 1536, 2048]),
            "experts": rng.choice([0, 4, 8, 16]),
            "out": rng.choice(["float32", "bfloat16"])}


# ---------------------------------------------------------------- inputs


def _chosen(gen, tokens, experts, k, padded):
    """k different experts a token, some experts more popular than others;
    -1 (no expert) for the `padded` last tokens."""
    liked = torch.randn(experts, generator=gen, device="cuda") * 0.7
    noise = torch.rand(tokens, experts, generator=gen, device="cuda")
    noise = -(-(noise.clamp(1e-9, 1 - 1e-7)).log()).log()
    ids = (liked + noise).topk(k, dim=1).indices.to(torch.int32)
    if padded:
        ids[max(0, tokens - padded):] = -1
    return ids


def _splits(gen, rows, experts):
    """Where each expert's rows begin, as the counts of an alltoallv give
    it: ragged, one expert without any."""
    share = torch.rand(experts, generator=gen, device="cuda").add(0.2)
    share[experts // 2] = 0
    at = (share.cumsum(0) / share.sum() * rows).round().to(torch.int32)
    at[-1] = rows
    return torch.cat([at.new_zeros(1), at])


def _activations(gen, rows, width, dtype):
    x = torch.randn(rows, width, generator=gen, device="cuda")
    x *= 0.5 + torch.rand(width, generator=gen, device="cuda") * 3
    return x.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, state = case["op"], {"case": case}
    if op == "route":
        dtype = DTYPES[case["dtype"]]
        x = torch.randn(case["tokens"], case["experts"], generator=gen,
                        device="cuda") * 1.5
        x += torch.randn(case["experts"], generator=gen, device="cuda") * 0.5
        if case["padded"]:
            x[max(0, case["tokens"] - case["padded"]):] = -torch.inf
        state["logits"] = x.to(dtype).requires_grad_(case["backward"])
        state["bias"] = (
            torch.randn(case["experts"], generator=gen, device="cuda") * 0.1
            if case["bias"] else None)
        state["grad"] = torch.randn(case["tokens"], case["k"], generator=gen,
                                    device="cuda")
    elif op in ("dispatch", "combine"):
        dtype = DTYPES[case["dtype"]]
        tokens, k, hidden = case["tokens"], case["k"], case["hidden"]
        ids = _chosen(gen, tokens, case["experts"], k, case["padded"])
        if op == "dispatch":
            state["ids"] = ids
            x = _activations(gen, tokens, hidden, dtype)
            state["x"] = x.requires_grad_(case["backward"])
            if case["backward"]:
                state["grad"] = _activations(gen, tokens * k, hidden, dtype)
        else:
            position, counts, offsets = _plan(ids, case["experts"])
            state.update(position=position, counts=counts, offsets=offsets)
            rows = _activations(gen, tokens * k, hidden, dtype)
            w = torch.rand(tokens, k, generator=gen, device="cuda") + 0.05
            w = w / w.sum(1, keepdim=True)
            state["rows"] = rows.requires_grad_(case["backward"])
            state["weights"] = w.requires_grad_(case["backward"])
            if case["backward"]:
                state["grad"] = _activations(gen, tokens, hidden, dtype)
    elif op == "product":
        experts, inner = case["experts"], case["inner"]
        x = _activations(gen, case["rows"], inner, torch.bfloat16)
        w = torch.randn(max(1, experts) * case["n"], inner, generator=gen,
                        device="cuda") / inner ** 0.5
        w = w.view(max(1, experts), case["n"], inner)
        q, s = _quantized_tiles(w)
        if experts:
            state["offsets"] = _splits(gen, case["rows"], experts)
            state["at"] = state["offsets"].tolist()
            state["a"] = _quantized(x)
        else:
            q, s = q[0], s[0]
            state["x"] = x
        state["b"] = (q, s)
    else:
        state["dy"] = _activations(gen, case["rows"], case["m"],
                                   torch.bfloat16) / 64
        state["x"] = _activations(gen, case["rows"], case["n"],
                                  torch.bfloat16)
        if case["experts"]:
            state["offsets"] = _splits(gen, case["rows"], case["experts"])
            state["at"] = state["offsets"].tolist()
        else:
            state["offsets"] = None
            state["at"] = [0, case["rows"]]
    return state


# ----------------------------------------------------------- plain forms


def _scales(most):
    """The least power of two, from 2^-127 on, that brings `most` to 448 or
    less; 2^0 for a block of zeros."""
    part, power = torch.frexp(most)  # part in [1/2, 1)
    e = (power - 9 + (part > 0.875).int()).clamp_min(-127)
    e = torch.where(most > 0, e, torch.zeros_like(e))
    return (e + 127).to(torch.uint8).view(E8M0)


def _quantized(x):
    """8-bit values of x and a scale for each 128 elements of a row."""
    rows, width = x.shape
    blocks = -(-width // BLOCK)
    x = torch.nn.functional.pad(x.float(), (0, blocks * BLOCK - width))
    x = x.view(rows, blocks, BLOCK)
    s = _scales(x.abs().amax(2))
    q = (x / s.float().unsqueeze(2)).to(FP8).view(rows, blocks * BLOCK)
    return q[:, :width], s


def _quantized_tiles(w):
    """8-bit values of w [E, N, K] and a scale for each tile of 128 x 128."""
    e, n, k = w.shape
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    x = torch.nn.functional.pad(
        w.float(), (0, kb * BLOCK - k, 0, nb * BLOCK - n))
    x = x.view(e, nb, BLOCK, kb, BLOCK)
    s = _scales(x.abs().amax((2, 4)))
    q = (x / s.float()[:, :, None, :, None]).to(FP8)
    q = q.view(e, nb * BLOCK, kb * BLOCK)[:, :n, :k].contiguous()
    return q, s


def _wide(s, n, dim):
    """Each scale for its 128 elements, along dim, which has n of them."""
    return s.float().repeat_interleave(BLOCK, dim).narrow(dim, 0, n)


def _plan(ids, experts):
    """Where each token copy goes when copies are sorted by expert, in
    order of tokens within one. A copy for no expert (-1) goes behind the
    last one, and its place is told as ~place."""
    flat = ids.reshape(-1).long()
    key = torch.where(flat < 0, experts, flat)
    order = key.argsort(stable=True)
    place = torch.empty_like(order)
    place[order] = torch.arange(len(order), device=ids.device)
    counts = torch.zeros(experts + 1, dtype=torch.long, device=ids.device)
    counts = counts.index_add(0, key, torch.ones_like(key))[:experts]
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    place = torch.where(flat < 0, ~place, place).view(ids.shape)
    return place.int(), counts.int(), offsets.int()


def _route(st):
    c, x = st["case"], st["logits"].detach().double()
    k, t = c["k"], x.shape[0]
    none = x == -torch.inf
    if c["score"] == "softmax":
        top = x.amax(1, keepdim=True)
        p = torch.where(none, 0, (x - top).exp())
        total = p.sum(1, keepdim=True)
        s = p / torch.where(total > 0, total, torch.ones_like(total))
    else:
        s = 1 / (1 + (-x).exp())
    b = st["bias"]
    value = s if b is None else s + b.double()
    choice = x if b is None else value
    value = value.masked_fill(none, -torch.inf)
    choice = choice.masked_fill(none, -torch.inf)
    if c["groups"] > 1:
        g = c["groups"]
        if c["group_score"] == "max":
            score = choice.view(t, g, -1).amax(2)
        else:
            best = value.view(t, g, -1).topk(2, dim=2).values
            rest = torch.where(best[..., 1] > -torch.inf, best[..., 1], 0.0)
            score = best[..., 0] + rest
        kept = score.sort(dim=1, descending=True, stable=True).indices
        out = torch.ones_like(score, dtype=torch.bool)
        out.scatter_(1, kept[:, :c["topk_groups"]], False)
        out = out.repeat_interleave(x.shape[1] // g, 1)
        choice = choice.masked_fill(out, -torch.inf)
    best, ids = choice.sort(dim=1, descending=True, stable=True)
    ids = ids[:, :k]
    gone = best[:, :k] == -torch.inf
    w = s.gather(1, ids).masked_fill(gone, 0)
    scale = torch.full_like(w[:, :1], c["scale"])
    if c["renormalize"]:
        total = w.sum(1, keepdim=True)
        scale = scale / torch.where(total > 0, total, torch.ones_like(total))
    weights = (w * scale).float()
    chosen = ids.masked_fill(gone, -1).int()
    if not c["backward"]:
        return {"weights": weights, "experts": chosen}
    # d weights / d scores, then d scores / d logits
    g = st["grad"].double().masked_fill(gone, 0)
    if c["renormalize"]:
        g = g - (g * w).sum(1, keepdim=True) * scale / c["scale"]
    g = g * scale
    if c["score"] == "softmax":
        dx = torch.zeros_like(s).scatter_add(1, ids, g)
        dx = s * (dx - (g * w).sum(1, keepdim=True))
    else:
        dx = torch.zeros_like(s).scatter_add(1, ids, g * w * (1 - w))
    return {"weights": weights, "experts": chosen,
            "dlogits": dx.to(st["logits"].dtype)}


def _dispatch(st):
    c, x = st["case"], st["x"].detach()
    position, counts, offsets = _plan(st["ids"], c["experts"])
    place = torch.where(position < 0, ~position, position).long().view(-1)
    gone = (position < 0).view(-1)
    token = torch.empty_like(place)
    token[place] = torch.arange(len(place), device=place.device) // c["k"]
    empty = torch.zeros_like(gone)
    empty[place] = gone
    got = {"position": position, "counts": counts, "offsets": offsets}
    if c["fp8"]:
        q, s = _quantized(x)
        # as bytes: a row for no expert holds zeros, with scales of 2^0
        q = q.view(torch.uint8)[token].masked_fill(empty[:, None], 0)
        s = s.view(torch.uint8)[token].masked_fill(empty[:, None], 127)
        got.update(rows=q.view(FP8), scales=s.view(E8M0))
        return got
    got["rows"] = x[token].masked_fill(empty[:, None], 0)
    if c["backward"]:
        g = st["grad"][place].float().masked_fill(gone[:, None], 0)
        got["dx"] = g.view(*position.shape, -1).sum(1).to(x.dtype)
    return got


def _combine(st):
    c, rows, w = st["case"], st["rows"].detach(), st["weights"].detach()
    position = st["position"].long()
    gone = position < 0
    place = torch.where(gone, ~position, position)
    y = rows[place.view(-1)].float().view(*place.shape, -1)
    w = w.masked_fill(gone, 0)
    out = (y * w.unsqueeze(2)).sum(1).to(rows.dtype)
    if not c["backward"]:
        return {"out": out}
    g = st["grad"].float().unsqueeze(1)
    drows = torch.empty_like(rows)
    drows[place.view(-1)] = (w.unsqueeze(2) * g).to(rows.dtype).flatten(0, 1)
    dw = (y * g).sum(2).masked_fill(gone, 0)
    return {"out": out, "drows": drows, "dweights": dw}


def _product(st):
    c, (bq, bs) = st["case"], st["b"]
    aq, a_s = st["a"] if c["experts"] else _quantized(st["x"])
    a = aq.float() * _wide(a_s, c["inner"], 1)
    b = bq.float() * _wide(_wide(bs, c["n"], -2), c["inner"], -1)
    dtype = DTYPES[c["out"]]
    if not c["experts"]:
        return {"out": (a @ b.t()).to(dtype)}
    out = torch.empty(c["rows"], c["n"], dtype=dtype, device=a.device)
    for e in range(c["experts"]):  # the ragged groups: one product each
        i, j = st["at"][e], st["at"][e + 1]
        out[i:j] = (a[i:j] @ b[e].t()).to(dtype)
    return {"out": out}


def _weight_grad(st):
    c = st["case"]
    yq, ys = _quantized(st["dy"].t())
    xq, xs = _quantized(st["x"].t())
    dy = yq.float() * _wide(ys, c["rows"], 1)
    x = xq.float() * _wide(xs, c["rows"], 1)
    got = []
    for i, j in zip(st["at"], st["at"][1:]):  # the ragged groups
        got.append((dy[:, i:j] @ x[:, i:j].t()).to(DTYPES[c["out"]]))
    return {"dw": torch.stack(got) if c["experts"] else got[0]}


def _own(st):
    from gloo_amd import experts as ex

    c = st["case"]
    if c["op"] == "route":
        weights, chosen = ex.route(
            st["logits"], c["k"], score=c["score"], bias=st["bias"],
            groups=c["groups"], topk_groups=c["topk_groups"],
            group_score=c["group_score"], renormalize=c["renormalize"],
            scale=c["scale"])
        got = {"weights": weights, "experts": chosen}
        if c["backward"]:
            got["dlogits"], = torch.autograd.grad(
                weights, st["logits"], st["grad"])
        return got
    if c["op"] == "dispatch":
        plan = ex.plan(st["ids"], c["experts"])
        got = {"position": plan.position, "counts": plan.counts,
               "offsets": plan.offsets}
        if c["fp8"]:
            got["rows"], got["scales"] = ex.pack_fp8(st["x"], plan)
            return got
        got["rows"] = ex.pack(st["x"], plan)
        if c["backward"]:
            got["dx"], = torch.autograd.grad(got["rows"], st["x"],
                                             st["grad"])
        return got
    if c["op"] == "combine":
        plan = ex.ExpertPlan(st["position"], st["counts"], st["offsets"])
        out = ex.combine(st["rows"], plan, st["weights"])
        if not c["backward"]:
            return {"out": out}
        drows, dw = torch.autograd.grad(
            out, (st["rows"], st["weights"]), st["grad"])
        return {"out": out, "drows": drows, "dweights": dw}
    if c["op"] == "product":
        a, a_scale = st["a"] if c["experts"] else ex.quantize_fp8(st["x"])
        return {"out": ex.fp8_matmul(a, a_scale, *st["b"],
                                     offsets=st.get("offsets"),
                                     dtype=DTYPES[c["out"]])}
    dy, dy_scale = ex.quantize_fp8(st["dy"].t())
    x, x_scale = ex.quantize_fp8(st["x"].t())
    return {"dw": ex.fp8_weight_grad(dy, dy_scale, x, x_scale,
                                     offsets=st["offsets"],
                                     dtype=DTYPES[c["out"]])}


_PLAIN = {"route": _route, "dispatch": _dispatch, "combine": _combine,
          "product": _product, "weight_grad": _weight_grad}


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["case"]["op"]](state)


# ------------------------------------------------------------------ work


def work(case):
    """Bytes and operations that a pass cannot do without."""
    op = case["op"]
    if op == "route":
        t, e, k = case["tokens"], case["experts"], case["k"]
        size = DTYPES[case["dtype"]].itemsize
        n = t * e * size + t * k * 8 + (e * 4 if case["bias"] else 0)
        if case["backward"]:
            n += t * k * 4 + t * e * size  # weights' gradient in, logits' out
        return {"bytes": n, "flops": t * e * (4 + 4 * case["backward"])}
    if op in ("dispatch", "combine"):
        t, k, h = case["tokens"], case["k"], case["hidden"]
        size = DTYPES[case["dtype"]].itemsize
        token, rows = t * h * size, t * k * h * size
        if op == "dispatch":
            n = token + t * k * 8 + case["experts"] * 8
            n += t * k * (h + -(-h // BLOCK)) if case["fp8"] else rows
            if case["backward"]:
                n += rows + token
            return {"bytes": n, "flops": t * h * (3 + k * case["backward"])}
        n = rows + token + t * k * 8
        if case["backward"]:
            n += token + rows + t * k * 4
        return {"bytes": n, "flops": t * k * h * (2 + 3 * case["backward"])}
    rows, out = case["rows"], DTYPES[case["out"]].itemsize
    if op == "product":
        n, inner, e = case["n"], case["inner"], case["experts"]
        most = min(rows, e) if e else 1  # weights that rows ask for
        a = rows * (inner + -(-inner // BLOCK)) if e else rows * inner * 2
        b = most * (n * inner + -(-n // BLOCK) * -(-inner // BLOCK))
        return {"bytes": a + b + rows * n * out,
                "flops": 2 * rows * n * inner}
    m, n = case["m"], case["n"]
    return {"bytes": rows * (m + n) * 2 + max(1, case["experts"]) * m * n
            * out, "flops": 2 * rows * m * n}


# ---------------------------------------------------- in 64 bits, apart


def _power(e):
    """2^e as the 64-bit number with these bits: exp2 may be off by one."""
    return (e.long() + 1023 << 52).view(torch.float64)


def _to_e4m3(v):
    """v rounded to the nearest of the 8-bit values (ties to even): three
    bits behind the leading one, steps of 2^-9 below 2^-6."""
    power = torch.frexp(v).exponent.sub(1).clamp_min(-6).sub(3)
    step = _power(power)
    return (v / step).round().mul(step)


def _blocks64(x):
    """(8-bit values, scales) of a matrix, both in 64 bits, from the
    definition: the smallest power of two that brings a block to 448."""
    parts = []
    for part in x.detach().double().split(BLOCK, dim=1):
        top = part.abs().max(dim=1, keepdim=True).values
        half, e = torch.frexp(top / 448)  # 2^(e-1) <= top / 448 < 2^e
        e = torch.where(half == 0.5, e - 1, e).clamp_min(-127)
        s = _power(torch.where(top > 0, e, torch.zeros_like(e)))
        parts.append((_to_e4m3(part / s), s))
    return torch.cat([p[0] for p in parts], 1), torch.cat(
        [p[1] for p in parts], 1)


def exact(case, seed):
    st, op = prepare(case, seed), case["op"]
    if op == "route":
        return _exact_route(case, st)
    if op == "dispatch":
        ids = st["ids"].long()
        flat = ids.reshape(-1)
        # a copy's place: copies of lower experts, and earlier ones of its own
        key = torch.where(flat < 0, case["experts"], flat)
        hits = torch.nn.functional.one_hot(key, case["experts"] + 1)
        before = hits.cumsum(0).gather(1, key[:, None])[:, 0] - 1
        counts = hits.sum(0)
        start = counts.cumsum(0) - counts
        place = start[key] + before
        rows = st["x"].detach().double()
        got = {"position": None, "counts": None, "offsets": None}
        real = flat >= 0
        token = torch.arange(len(flat), device=flat.device) // case["k"]
        if case["fp8"]:
            q, s = _blocks64(rows)
            got["rows"] = q.new_zeros(len(flat), q.shape[1])
            got["scales"] = s.new_ones(len(flat), s.shape[1])
            got["rows"][place[real]] = q[token[real]]
            got["scales"][place[real]] = s[token[real]]
            return got
        got["rows"] = rows.new_zeros(len(flat), rows.shape[1])
        got["rows"][place[real]] = rows[token[real]]
        if case["backward"]:
            got["dx"] = torch.zeros_like(rows).index_add(
                0, token[real], st["grad"].double()[place[real]])
        return got
    if op == "combine":
        rows, w = st["rows"].detach().double(), st["weights"].detach()
        out = rows.new_zeros(case["tokens"], case["hidden"])
        drows, dw = torch.zeros_like(rows), torch.zeros_like(w).double()
        g = st["grad"].double() if case["backward"] else None
        for j in range(case["k"]):
            at = st["position"][:, j].long()
            real = at >= 0
            here = rows[at[real]]
            out[real] += here * w[real, j, None].double()
            if g is not None:
                drows[at[real]] = g[real] * w[real, j, None].double()
                dw[real, j] = (here * g[real]).sum(1)
        return {"out": out} if g is None else {
            "out": out, "drows": drows, "dweights": dw}
    if op == "product":
        aq, a_s = st["a"] if case["experts"] else _blocks64(st["x"])
        bq, bs = st["b"]
        if not case["experts"]:
            bq, bs = bq[None], bs[None]
        at = st.get("at", [0, case["rows"]])
        out = torch.zeros(case["rows"], case["n"], dtype=torch.float64,
                          device="cuda")
        a = torch.cat([p.double() * a_s[:, i, None].float().double() for i, p in
                       enumerate(aq.split(BLOCK, 1))], 1)
        for e in range(len(bq)):
            if at[e] == at[e + 1]:
                continue
            s = bs[e].float().double()
            s = s.repeat_interleave(BLOCK, 0).repeat_interleave(BLOCK, 1)
            b = bq[e].double() * s[:case["n"], :case["inner"]]
            out[at[e]:at[e + 1]] = a[at[e]:at[e + 1]] @ b.t()
        return {"out": out}
    yq, ys = _blocks64(st["dy"].t())
    xq, xs = _blocks64(st["x"].t())
    n = case["rows"]
    dy = yq * ys.repeat_interleave(BLOCK, 1)[:, :n]
    x = xq * xs.repeat_interleave(BLOCK, 1)[:, :n]
    dw = [dy[:, i:j] @ x[:, i:j].t() for i, j in zip(st["at"], st["at"][1:])]
    return {"dw": torch.stack(dw) if case["experts"] else dw[0]}


def _exact_route(case, st):
    """By autograd of the definition in 64 bits, for the experts that the
    scores choose."""
    x = st["logits"].detach().double().requires_grad_()
    alive = x.detach() > -torch.inf
    safe = torch.where(alive, x, torch.zeros_like(x))
    if case["score"] == "softmax":
        far = torch.where(alive, x, torch.full_like(x, -1e300))
        s = torch.where(alive, torch.softmax(far, 1), torch.zeros_like(x))
    else:
        s = torch.where(alive, torch.sigmoid(safe), torch.zeros_like(x))
    with torch.no_grad():
        low = torch.full_like(x, -1e300)
        bias = 0 if st["bias"] is None else st["bias"].double()
        value = torch.where(alive, s + bias, low)
        rank = torch.where(alive, x, low) if st["bias"] is None else value
        groups, per = case["groups"], x.shape[1] // case["groups"]
        if groups > 1:
            if case["group_score"] == "max":
                of = rank.view(-1, groups, per).max(2).values
            else:
                two = value.view(-1, groups, per).sort(2).values[..., -2:]
                of = torch.where(two > -1e299, two, 0 * two).sum(2)
                of = torch.where(two[..., 1] > -1e299, of, two[..., 1])
            # a group is kept if fewer than topk_groups stand before it
            i = torch.arange(groups, device=x.device)
            first = (of[:, None, :] > of[:, :, None]) | (
                (of[:, None, :] == of[:, :, None]) & (i[None] < i[:, None]))
            kept = first.sum(2) < case["topk_groups"]
            kept = kept.repeat_interleave(per, 1)
            rank = torch.where(kept, rank, low)
        ids = rank.argsort(dim=1, descending=True, stable=True)[:, :case["k"]]
        real = rank.gather(1, ids) > -1e299
    w = torch.where(real, s.gather(1, ids), torch.zeros((), device="cuda",
                                                        dtype=s.dtype))
    if case["renormalize"]:
        total = w.sum(1, keepdim=True)
        w = w / torch.where(total > 0, total, torch.ones_like(total))
    w = w * case["scale"]
    got = {"weights": w.detach(), "experts": None}
    if case["backward"]:
        got["dlogits"], = torch.autograd.grad(w, x, st["grad"].double())
    return got
