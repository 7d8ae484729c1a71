"""Expert operators on inputs that are not plain tensors (no GPU needed)."""
import pytest

torch = pytest.importorskip("torch")

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
