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
