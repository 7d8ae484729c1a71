"""Ranks that are threads of one process on one GPU: they wait for flags on
the host, so that their streams may share hardware queues with each other's,
torch's and the null stream (tests/test_queue_model.py has the argument)."""
import threading

import pytest

import gloo_amd as ga

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("no GPU", allow_module_level=True)


def whole(rank, n, run=0):
    gen = torch.Generator("cpu").manual_seed(1000 * run + rank)
    return torch.randint(-50, 50, (n,), generator=gen).float()


def ranks(size, fn):
    """fn(ctx, rank) on `size` threads, each with a stream of its own for
    torch's work: with torch's pool there are more streams than queues."""
    store, errors = ga.HashStore(), []

    def worker(rank):
        try:
            ctx = ga.Context(rank, size)
            ctx.connect_full_mesh(store, ga.create_tcp_device())
            ctx.set_timeout(30000)
            torch.cuda.set_device(0)
            with torch.cuda.stream(torch.cuda.Stream()):
                fn(ctx, rank)
        except Exception:  # noqa: BLE001
            import traceback

            errors.append(traceback.format_exc())

    threads = [threading.Thread(target=worker, args=(r,), daemon=True)
               for r in range(size)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(100)
    assert not errors, errors[0]
    assert not any(t.is_alive() for t in threads)


def stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.parametrize("size", [2, 3, 4])
@pytest.mark.parametrize("engine", ["HipAllreduceRing", "HipAllreduceDirect",
                                    "HipAllreduceHalvingDoubling"])
def test_allreduce(engine, size):
    """Runs of two shapes, not in step: no barrier between them."""

    def fn(ctx, rank):
        algo = getattr(ga._C, engine)(ctx, 0)
        for run, n in enumerate((400_000, 400_000, 400_000, 300_001,
                                 400_000)):
            x = whole(rank, n, run).cuda()
            algo.run(x.data_ptr(), n, ga.DType.f32, ga.ReduceOp.sum,
                     stream=stream())
            want = sum(whole(r, n, run) for r in range(size))
            assert torch.equal(x.cpu(), want), (engine, run)

    ranks(size, fn)


@pytest.mark.parametrize("size", [2, 4])
def test_other_collectives(size):
    def fn(ctx, rank):
        n = 150_000
        gather = ga._C.HipAllgatherRing(ctx, 0)
        scatter = ga._C.HipReduceScatterRing(ctx, 0)
        swap = ga._C.HipAlltoall(ctx, 0)
        cast = ga._C.HipBroadcastOneToAll(ctx, 0, size - 1)
        for run in range(3):
            mine = whole(rank, n, run).cuda()
            every = [whole(r, n, run) for r in range(size)]
            out = torch.empty(size * n, device="cuda")
            gather.run(mine.data_ptr(), out.data_ptr(), n, 4,
                       stream=stream())
            assert torch.equal(out.cpu(), torch.cat(every))
            many = [whole(r + 10, size * n, run) for r in range(size)]
            mine = many[rank].cuda()
            out = torch.empty(n, device="cuda")
            scatter.run(mine.data_ptr(), out.data_ptr(), n, ga.DType.f32,
                        ga.ReduceOp.sum, stream=stream())
            part = slice(rank * n, (rank + 1) * n)
            assert torch.equal(out.cpu(), sum(many)[part])
            out = torch.empty(size * n, device="cuda")
            swap.run(mine.data_ptr(), out.data_ptr(), n, 4, stream=stream())
            assert torch.equal(out.cpu(),
                               torch.cat([m[part] for m in many]))
            x = whole(rank, n, run).cuda()
            cast.run(x.data_ptr(), n * 4, stream=stream())
            assert torch.equal(x.cpu(), every[-1])

    ranks(size, fn)


@pytest.mark.parametrize("orders", [("sr", "sr"), ("rs", "rs"), ("sr", "rs")])
def test_point_to_point(orders):
    """Messages of several chunks both ways, whatever is posted first."""

    def fn(ctx, rank):
        engine, peer = ga._C.HipP2P(ctx, 0), 1 - rank
        for run, n in enumerate((3_000_000, 100, 5_000_001)):
            src = whole(rank, n, run).cuda()
            dst = torch.zeros(n, device="cuda")
            for op in orders[rank]:
                if op == "s":
                    engine.post_send(peer, src.data_ptr(), n * 4, stream())
                else:
                    engine.post_recv(peer, dst.data_ptr(), n * 4, stream())
            for op in orders[rank]:
                if op == "s":
                    engine.flush_sends()
                else:
                    engine.flush_recvs()
            assert torch.equal(dst.cpu(), whole(peer, n, run))
            ga.barrier(ctx, tag=800 + run)

    ranks(2, fn)


def test_a_rank_that_does_not_come_is_given_up():
    """The wait on the host ends with the communicator's timeout."""
    from gloo_amd import IoError

    def fn(ctx, rank):
        algo = ga._C.HipAllreduceRing(ctx, 0)
        ga.barrier(ctx, tag=820)
        if rank == 0:
            ctx.set_timeout(500)
            x = torch.ones(400_000, device="cuda")
            with pytest.raises(IoError, match="timed out"):
                algo.run(x.data_ptr(), 400_000, ga.DType.f32,
                         ga.ReduceOp.sum, stream=stream())
        ga.barrier(ctx, tag=821)

    ranks(2, fn)


def test_sends_that_nobody_receives_are_given_up():
    """And what was still to go is dropped: the tensor may be freed."""
    from gloo_amd import IoError

    def fn(ctx, rank):
        engine = ga._C.HipP2P(ctx, 0)
        ga.barrier(ctx, tag=830)
        if rank == 0:
            ctx.set_timeout(500)
            x = torch.ones(6_000_000, device="cuda")
            engine.post_send(1, x.data_ptr(), x.numel() * 4, stream())
            with pytest.raises(IoError, match="timed out"):
                engine.flush_sends()
            engine.flush_sends()  # nothing is left
        ga.barrier(ctx, tag=831)

    ranks(2, fn)
