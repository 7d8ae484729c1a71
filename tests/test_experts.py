"""What the expert-parallel operators refuse (no GPU needed: every argument
is checked before anything is launched, tensors' devices last)."""
import pytest

import gloo_amd as ga

torch = pytest.importorskip("torch")

from gloo_amd import experts as ex  # noqa: E402

F8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _plan(tokens=4, k=2, experts=8):
    z = torch.zeros
    return ex.ExpertPlan(z(tokens, k, dtype=torch.int32),
                         z(experts, dtype=torch.int32),
                         z(experts + 1, dtype=torch.int32))


@pytest.mark.parametrize("options", [
    {"k": 0}, {"k": 9}, {"k": 2, "score": "tanh"}, {"k": 2, "groups": 3},
    {"k": 2, "groups": 0}, {"k": 2, "groups": 4, "topk_groups": 5},
    {"k": 2, "groups": 4, "topk_groups": 0},
    {"k": 3, "groups": 4, "topk_groups": 1},
    {"k": 2, "group_score": "sum"},
    {"k": 2, "bias": torch.zeros(7)},
    {"k": 2, "bias": torch.zeros(8, dtype=torch.float64)},
    {"k": 2, "bias": torch.zeros(1, 8)},
])
def test_route_refuses(options):
    with pytest.raises(ValueError):
        ex.route(torch.zeros(4, 8), **options)


@pytest.mark.parametrize("logits", [
    torch.zeros(8), torch.zeros(4, 8, dtype=torch.float64),
    torch.zeros(4, 0), torch.zeros(4, 1025), [[0.0]],
])
def test_route_refuses_logits(logits):
    with pytest.raises(ValueError):
        ex.route(logits, 1)


def test_operators_refuse_the_cpu():
    p = _plan()
    q, s = torch.zeros(4, 128).to(F8), torch.ones(4, 1).to(E8)
    w, ws = torch.zeros(8, 128).to(F8), torch.ones(1, 1).to(E8)
    calls = [
        lambda: ex.route(torch.zeros(4, 8), 2),
        lambda: ex.plan(torch.zeros(4, 2, dtype=torch.int32), 8),
        lambda: ex.pack(torch.zeros(4, 16), p),
        lambda: ex.pack_fp8(torch.zeros(4, 16), p),
        lambda: ex.combine(torch.zeros(8, 16), p, torch.zeros(4, 2)),
        lambda: ex.quantize_fp8(torch.zeros(4, 16)),
        lambda: ex.quantize_fp8(torch.zeros(2, 4, 16), tile=True),
        lambda: ex.fp8_matmul(q, s, w, ws),
        lambda: ex.fp8_weight_grad(q, s, q, s),
    ]
    for call in calls:
        with pytest.raises(ValueError, match="on a GPU"):
            call()


@pytest.mark.parametrize("ids,experts", [
    (torch.zeros(4, 2), 8), (torch.zeros(4, 2, dtype=torch.int64), 8),
    (torch.zeros(8, dtype=torch.int32), 8),
    (torch.zeros(4, 2, dtype=torch.int32), 0),
    (torch.zeros(4, 2, dtype=torch.int32), 1025),
])
def test_plan_refuses(ids, experts):
    with pytest.raises(ValueError):
        ex.plan(ids, experts)


def test_rows_refuse():
    p = _plan()
    with pytest.raises(ValueError, match="4 tokens"):
        ex.pack(torch.zeros(5, 16), p)
    with pytest.raises(ValueError, match="needed"):
        ex.pack(torch.zeros(4, 16, dtype=torch.int32), p)
    with pytest.raises(ValueError, match="contiguous"):
        ex.pack(torch.zeros(2, 16), ex.ExpertPlan(
            p.position.t(), p.counts, p.offsets))
    with pytest.raises(ValueError, match="no gradient"):
        ex.pack_fp8(torch.zeros(4, 16, requires_grad=True), p)
    with pytest.raises(ValueError, match="the plan has 8"):
        ex.combine(torch.zeros(9, 16), p)
    with pytest.raises(ValueError, match="weights"):
        ex.combine(torch.zeros(8, 16), p, torch.zeros(4, 3))
    with pytest.raises(ValueError, match="weights"):
        ex.combine(torch.zeros(8, 16), p,
                   torch.zeros(4, 2, dtype=torch.bfloat16))


def test_what_is_too_large_is_refused():
    # one element's memory each
    one = torch.zeros(1)
    with pytest.raises(ValueError, match="tokens"):
        ex.route(one.expand(2 ** 26, 8), 2)
    with pytest.raises(ValueError, match="copies"):
        ex.plan(torch.zeros(1, dtype=torch.int32).expand(2 ** 30, 2), 8)
    with pytest.raises(ValueError, match="blocks"):
        ex.quantize_fp8(one.expand(2 ** 28, 256))
    with pytest.raises(ValueError, match="columns"):
        ex.quantize_fp8(one.expand(1, 2 ** 23))
    p = ex.ExpertPlan(torch.empty(2 ** 24, 1, dtype=torch.int32), None, None)
    for call in (lambda: ex.pack(one.expand(2 ** 24, 8), p),
                 lambda: ex.pack_fp8(one.expand(2 ** 24, 8), p),
                 lambda: ex.combine(one.expand(2 ** 24, 8), p)):
        with pytest.raises(ValueError, match="fewer than 2"):
            call()
    with pytest.raises(ValueError, match="elements"):
        ex.pack(one.expand(4, 2 ** 23 + 1), _plan())
    e = 65534
    q, s, off = one.to(F8), one.to(E8), torch.zeros(e + 1, dtype=torch.int32)
    with pytest.raises(ValueError, match="65533 experts"):
        ex.fp8_matmul(q.expand(4, 128), s.expand(4, 1), q.expand(e, 8, 128),
                      s.expand(e, 1, 1), offsets=off)
    with pytest.raises(ValueError, match="65533 experts"):
        ex.fp8_weight_grad(q.expand(4, 128), s.expand(4, 1),
                           q.expand(8, 128), s.expand(8, 1), offsets=off)


def _operands(rows=4, n=8, inner=200, experts=0):
    b = (experts, n, inner) if experts else (n, inner)
    bs = ((experts,) if experts else ()) + (-(-n // 128), -(-inner // 128))
    return [torch.zeros(rows, inner).to(F8),
            torch.ones(rows, -(-inner // 128)).to(E8),
            torch.zeros(b).to(F8), torch.ones(bs).to(E8)]


def test_products_refuse():
    a, s, b, t = _operands()
    wrong = [
        (a.float(), s, b, t), (a, s.float(), b, t), (a, s[:, :1], b, t),
        (a, s, b[:, :100], t), (a, s, b, t[:, :1]), (a[0], s, b, t),
        (a, s, b[None], t[None]), (a, s, b[:0], t),
    ]
    for args in wrong:
        with pytest.raises(ValueError):
            ex.fp8_matmul(*args)
    with pytest.raises(ValueError, match="cannot return"):
        ex.fp8_matmul(a, s, b, t, dtype=torch.int32)
    a, s, b, t = _operands(experts=3)
    at = torch.zeros(4, dtype=torch.int32)
    for off in (at[:3], at.long(), at[None], torch.zeros(
            8, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError):
            ex.fp8_matmul(a, s, b, t, offsets=off)
    dy, dys = a, s
    with pytest.raises(ValueError, match="rows are needed"):
        ex.fp8_weight_grad(dy, dys, dy[:, :100], dys)
    with pytest.raises(ValueError):
        ex.fp8_weight_grad(dy, dys[:, :1], dy, dys)
    with pytest.raises(ValueError):
        ex.fp8_weight_grad(dy, dys, dy, dys, offsets=at[:1])
    with pytest.raises(ValueError, match="no gradient"):
        ex.quantize_fp8(torch.zeros(4, 16, requires_grad=True))
    with pytest.raises(ValueError):
        ex.quantize_fp8(torch.zeros(2, 4, 16))


def test_launchers_check_for_themselves():
    """The raw entry points throw before they touch a device."""
    f, s = ga.DType.f32, 0
    with pytest.raises(ga.EnforceNotMet):  # k > experts
        ga._C.hip_expert_route(0, 8, f, 0, 4, 8, 9, "softmax", 1, 1, "max",
                               True, 1.0, 0, 0, 0, s)
    with pytest.raises(ga.EnforceNotMet):  # groups that are not equal
        ga._C.hip_expert_route(0, 8, f, 0, 4, 8, 2, "softmax", 3, 1, "max",
                               True, 1.0, 0, 0, 0, s)
    with pytest.raises(ga.EnforceNotMet):
        ga._C.hip_expert_route(0, 8, f, 0, 4, 8, 2, "other", 1, 1, "max",
                               True, 1.0, 0, 0, 0, s)
    with pytest.raises(ga.EnforceNotMet):  # no workspace
        ga._C.hip_expert_plan(0, 1 << 20, 64, 0, 0, 0, 0, 0, 0, s)
    with pytest.raises(ga.EnforceNotMet):  # 2^31 copies
        ga._C.hip_expert_pack(0, 1 << 30, 2, 16, f, 0, 16, 0, 0, s)
    with pytest.raises(ga.EnforceNotMet):  # rows of q on no border of 16
        ga._C.hip_expert_pack_fp8(0, 4, 2, 16, f, 0, 16, 0, 24, 0, 0, s)
    with pytest.raises(ga.EnforceNotMet):
        ga._C.hip_quantize_fp8(0, 16, 1, f, 4, 16, False, 0, 8, 0, 0, s)
    with pytest.raises(ga.EnforceNotMet):  # experts without offsets
        ga._C.hip_fp8_matmul(0, 128, 0, 0, 128, 0, 0, 0, 4, 8, 128, 2, 0, f,
                             0, s)
    with pytest.raises(ga.EnforceNotMet):
        ga._C.hip_fp8_weight_grad(0, 128, 0, 0, 128, 0, 0, 4, 0, 8, 1, 0, f,
                                  0, s)
    for out in (4, 8):  # results on no border of 16
        with pytest.raises(ga.EnforceNotMet, match="16 bytes"):
            ga._C.hip_fp8_matmul(0, 128, 0, 0, 128, 0, 0, 0, 4, 8, 128, 1,
                                 out, f, 0, s)
        with pytest.raises(ga.EnforceNotMet, match="16 bytes"):
            ga._C.hip_fp8_weight_grad(0, 128, 0, 0, 128, 0, 0, 4, 4, 8, 1,
                                      out, f, 0, s)


def test_exchange_of_rows_between_ranks():
    """The row exchange of ExpertExchange on host tensors, its gradient and
    the counts, over three ranks; one rank sends nothing."""
    from test_pg import spawn_pg

    table = [[2, 0, 3, 1, 0, 4], [0] * 6, [1, 1, 0, 0, 5, 0]]

    def fn(pg, rank, size):
        exchange = ex.ExpertExchange(6, pg)
        assert exchange.local_experts == 2
        mine, theirs = exchange._counts(
            torch.tensor(table[rank], dtype=torch.int32))
        assert mine.tolist() == [table[rank][i:i + 2] for i in (0, 2, 4)]
        assert theirs.tolist() == [
            table[r][2 * rank:2 * rank + 2] for r in range(size)]
        send, recv = mine.sum(1).tolist(), theirs.sum(1).tolist()
        rows = torch.arange(sum(send) * 3.0).view(-1, 3) + 1000 * rank
        rows.requires_grad_()
        out = ex._AllToAll.apply(pg, rows, send, recv)
        expect = []
        for r in range(size):
            n = [sum(table[r][2 * d:2 * d + 2]) for d in range(size)]
            all_rows = torch.arange(sum(n) * 3.0).view(-1, 3) + 1000 * r
            expect.append(all_rows.split(n)[rank])
        assert torch.equal(out.detach(), torch.cat(expect))
        grad, = torch.autograd.grad(out, rows, 2 * out.detach())
        assert torch.equal(grad, 2 * rows.detach())
        return True

    spawn_pg(3, fn)


def test_exchange_refuses():
    from test_pg import spawn_pg

    def fn(pg, rank, size):
        for experts in (0, 3, 1026):
            with pytest.raises(ValueError):
                ex.ExpertExchange(experts, pg)
        exchange = ex.ExpertExchange(4, pg)
        ids = torch.zeros(4, 2, dtype=torch.int32)
        with pytest.raises(ValueError, match="one row a token"):
            exchange.dispatch(torch.zeros(5, 8), ids)
        with pytest.raises(ValueError, match="one element"):
            exchange.dispatch(torch.zeros(4, 0), ids)
        with pytest.raises(ValueError, match="on a GPU"):
            exchange.dispatch(torch.zeros(4, 8), ids)
        return True

    spawn_pg(2, fn)
