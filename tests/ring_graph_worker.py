"""One rank of a ring allreduce whose schedule is captured and replayed (see
test_gpu_ring_graph.py): a process for each rank, where the device waits."""
import sys

sys.path.insert(0, __file__.rsplit("/", 2)[0])

import torch  # noqa: E402

import gloo_amd as ga  # noqa: E402


def inputs(rank, n, run):
    gen = torch.Generator("cpu").manual_seed(1000 * run + rank)
    return torch.randint(-50, 50, (n,), generator=gen).float()


def main():
    rank, size, storedir = int(sys.argv[1]), int(sys.argv[2]), sys.argv[3]
    ctx = ga.Context(rank, size)
    ctx.connect_full_mesh(ga.FileStore(storedir), ga.create_tcp_device())
    ctx.set_timeout(60000)
    torch.cuda.set_device(0)
    algo = ga._C.HipAllreduceRing(ctx, 0, True, 0)
    buf = {n: torch.empty(n, device="cuda") for n in (1_000_000, 700_001)}
    # the second run of a shape is captured, a switch goes without a graph
    shapes = [1_000_000] * 6 + [700_001, 700_001, 700_001, 1_000_000,
                                1_000_000]
    for run, n in enumerate(shapes):
        x = buf[n]
        x.copy_(inputs(rank, n, run))
        algo.run(x.data_ptr(), n, ga.DType.f32, ga.ReduceOp.sum,
                 stream=torch.cuda.current_stream().cuda_stream)
        expect = sum(inputs(r, n, run) for r in range(size))
        assert torch.equal(x.cpu(), expect), run  # whole numbers
        print(f"rank {rank} run {run} ok", flush=True)
    print("ALL OK", flush=True)


if __name__ == "__main__":
    main()
