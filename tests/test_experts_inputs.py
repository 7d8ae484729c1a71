"""Expert operators on inputs that are not plain tensors (no GPU needed)."""
import pytest

torch = pytest.importorskip("torch")

import torch.autograd.forward_ad as fw  # noqa: E402

from gloo_amd import experts as ex  # noqa: E402


def test_negative_rows_between_ranks():
    """ExpertExchange's rows and gradients with the negative bit set: what
    travels are the values."""
    from test_pg import spawn_pg

    def fn(pg, rank, size):
        gen = torch.Generator().manual_seed(rank)
        counts = [[1, 2], [3, 0]]
        send, recv = counts[rank], [counts[r][rank] for r in range(size)]
        z = torch.randn(sum(send), 4, generator=gen, dtype=torch.complex64)
        for v in (z.conj().imag, torch._neg_view(z.real.contiguous())):
            assert v.is_neg()
            want = ex._AllToAll.apply(pg, v.resolve_neg(), send, recv)
            assert torch.equal(ex._AllToAll.apply(pg, v, send, recv), want)
        rows = z.real.clone().requires_grad_()
        out = ex._AllToAll.apply(pg, rows, send, recv)
        g = torch._neg_view(torch.randn(out.shape, generator=gen))
        got, = torch.autograd.grad(out, rows, g, retain_graph=True)
        want, = torch.autograd.grad(out, rows, g.resolve_neg())
        assert torch.equal(got, want)
        return True

    spawn_pg(2, fn)


def test_forward_mode_is_refused():
    """Below the check of the device, on batches without tokens: an input's
    tangent would be lost."""
    ops = ex._ops
    ids = torch.zeros(0, 2, dtype=torch.int32)
    q = torch.zeros(0, 128).to(torch.float8_e4m3fn)
    s = torch.zeros(0, 1).to(torch.float8_e8m0fnu)
    b, bs = torch.zeros(4, 128).to(q.dtype), torch.ones(1, 1).to(s.dtype)
    with fw.dual_level():
        for grad in (False, True):
            def dual(v):
                return fw.make_dual(v.clone().requires_grad_(grad),
                                    torch.ones_like(v))

            x = torch.zeros(0, 8)
            calls = [
                lambda: ops.route(dual(x), None, 2, False, 1, 1, False, True,
                                  1.0, 0),
                lambda: ops.pack(dual(x), ids, 0),
                lambda: ops.combine(dual(x), ids, None, 0),
                lambda: ops.combine(x, ids, dual(torch.zeros(0, 2)), 0),
                lambda: ops.pack_fp8(dual(x), ids, 0),
                lambda: ops.quantize_fp8(dual(x), False, 0),
                lambda: ops.fp8_matmul(dual(q), s, b, bs, None,
                                       torch.float32, 0),
                lambda: ops.fp8_matmul(q, s, dual(b), bs, None,
                                       torch.float32, 0)]
            for call in calls:
                with pytest.raises(ValueError, match="forward-mode"):
                    call()
        ops.pack(dual(x).detach(), ids, 0)


def test_products_refuse_operands_with_a_gradient():
    """x.to(float8) is differentiable in torch, products of it are not."""
    x = torch.zeros(4, 128, requires_grad=True)
    q, s = x.to(torch.float8_e4m3fn), torch.ones(4, 1).to(
        torch.float8_e8m0fnu)
    w, ws = q.detach(), torch.ones(1, 1).to(s.dtype)
    assert q.requires_grad
    for call in (lambda: ex.fp8_matmul(q, s, w, ws),
                 lambda: ex.fp8_matmul(w, s, q, ws),
                 lambda: ex.fp8_weight_grad(q, s, w, s),
                 lambda: ex.fp8_weight_grad(w, s, q, s)):
        with pytest.raises(ValueError, match="no gradient"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="on a GPU"):
            call()


def test_what_a_launch_refuses_is_a_wrong_argument():
    """Launches check for themselves, before they touch a device."""
    for k, groups in ((9, 1), (2, 3)):
        with pytest.raises(ValueError):
            ex._ops.route(torch.zeros(0, 8), None, k, False, groups, 1, False,
                          True, 1.0, 0)
