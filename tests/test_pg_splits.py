"""alltoall_base with split sizes, ranks without any rows among them."""
import torch

from test_pg import spawn_pg


def _exchange(pg, rank, size, counts, shape):
    """Rank r sends counts[r][d] rows of value 10 r + d to rank d."""
    ins = [torch.full((counts[rank][d],) + shape, 10.0 * rank + d)
           for d in range(size)]
    inp = torch.cat(ins)
    outs = [counts[s][rank] for s in range(size)]
    out = torch.full((sum(outs),) + shape, -1.0)
    pg.alltoall_base(out, inp, outs, counts[rank]).wait()
    expect = torch.cat([torch.full((n,) + shape, 10.0 * s + rank)
                        for s, n in enumerate(outs)])
    assert torch.equal(out, expect)
    return True


def test_alltoall_splits():
    counts = [[1, 4, 0], [2, 0, 3], [5, 1, 1]]
    for shape in ((), (7,), (2, 3)):
        spawn_pg(3, lambda pg, r, n: _exchange(pg, r, n, counts, shape))


def test_alltoall_splits_without_rows():
    """One rank sends nothing, one receives nothing, none moves any."""
    for counts in ([[0, 0], [3, 2]], [[0, 3], [0, 2]], [[0, 0], [0, 0]]):
        for shape in ((), (5,)):
            spawn_pg(2, lambda pg, r, n: _exchange(pg, r, n, counts, shape))


def test_alltoall_splits_of_plainly_empty_tensors():
    """A rank without rows need not know their shape."""
    counts = [[0, 0], [3, 2]]

    def fn(pg, rank, size):
        outs = [counts[s][rank] for s in range(size)]
        inp = (torch.empty(0) if rank == 0 else
               torch.arange(25.0).view(5, 5))
        out = torch.full((sum(outs), 5), -1.0)
        pg.alltoall_base(out, inp, outs, counts[rank]).wait()
        at = slice(0, 3) if rank == 0 else slice(3, 5)
        assert torch.equal(out, torch.arange(25.0).view(5, 5)[at])
        # and the way back: the other rank's output is empty
        back = torch.empty(0) if rank == 0 else torch.full((5, 5), -1.0)
        pg.alltoall_base(back, out, counts[rank], outs).wait()
        if rank == 1:
            assert torch.equal(back, torch.arange(25.0).view(5, 5))
        return True

    spawn_pg(2, fn)
