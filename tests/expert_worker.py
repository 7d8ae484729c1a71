"""One rank of an expert-parallel layer on cuda:0 (see test_gpu_experts.py):
ExpertExchange over init_process_group("glooamd") against the same layer
computed in this process alone."""
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402
import torch.distributed as dist  # noqa: E402

import gloo_amd.pg  # noqa: F401,E402  (registers the backend)
from gloo_amd import experts as ex  # noqa: E402


def tokens_of(rank, case):
    gen = torch.Generator().manual_seed(100 * case + rank)
    t = [[5, 9, 64], [0, 33, 7], [8, 0, 0]][case][rank]
    x = torch.randn(t, 200, generator=gen)
    ids = torch.stack([torch.randperm(12, generator=gen)[:4]
                       for _ in range(t)]) if t else torch.zeros(0, 4)
    ids = ids.to(torch.int32)
    if case != 1:
        ids[torch.rand(t, 4, generator=gen) < 0.2] = -1
    if case == 2:
        ids[ids > 3] = 2  # two ranks' experts get nothing
    w = torch.rand(t, 4, generator=gen)
    return x, ids, w


def main():
    rank, size, port = int(sys.argv[1]), int(sys.argv[2]), sys.argv[3]
    dist.init_process_group(
        "glooamd", init_method=f"tcp://127.0.0.1:{port}", rank=rank,
        world_size=size)
    exchange = ex.ExpertExchange(12)
    gen = torch.Generator().manual_seed(7)
    scale = torch.rand(12, generator=gen) + 0.5  # an expert multiplies by it
    local = scale.cuda()[rank * exchange.local_experts:]
    for case in range(3):
        x, ids, w = tokens_of(rank, case)
        xg, wg = x.cuda().requires_grad_(), w.cuda().requires_grad_()
        batch = exchange.dispatch(xg, ids.cuda())
        assert batch.rows.shape == (sum(batch.recv), 200)
        at = batch.offsets.tolist()
        assert at[-1] == batch.rows.shape[0]
        parts = [batch.rows[i:j] * local[e]
                 for e, (i, j) in enumerate(zip(at, at[1:]))]
        out = exchange.combine(torch.cat(parts), batch, wg)
        real = ids >= 0
        s = torch.where(real, scale[ids.clamp(min=0).long()],
                        torch.zeros(()))
        ref = x.double() * (s.double() * w).sum(1, keepdim=True)
        # four products of two factors, added up in fp32
        tol = 8 * 2.0 ** -24 * (x.double().abs() * (
            s.double() * w).sum(1, keepdim=True)) + 1e-30
        assert ((out.detach().double().cpu() - ref).abs() <= tol).all()
        g = torch.randn(x.shape, generator=gen)
        dx, dw = torch.autograd.grad(out, (xg, wg), g.cuda())
        refx = g.double() * (s.double() * w).sum(1, keepdim=True)
        assert ((dx.double().cpu() - refx).abs()
                <= 8 * 2.0 ** -24 * refx.abs() + 1e-30).all()
        dot = (g.double() * x).abs().sum(1, keepdim=True) * s
        refw = (g.double() * x).sum(1, keepdim=True) * s
        assert ((dw.double().cpu() - refw).abs()
                <= 204 * 2.0 ** -24 * dot + 1e-30).all()

        # the same rows in 8 bits: what arrives is what this rank's experts
        # would get of everybody's tokens quantised in one place
        with torch.no_grad():
            got = exchange.dispatch(x.cuda(), ids.cuda(), fp8=True)
            assert torch.equal(got.offsets, batch.offsets)
            q, sc = ex.quantize_fp8(batch.rows)
            assert torch.equal(got.rows.float(), q.float())
            assert torch.equal(got.scales.float(), sc.float())
            weights = torch.randn(exchange.local_experts, 64, 200,
                                  generator=gen).cuda()
            b, bs = ex.quantize_fp8(weights, tile=True)
            y = ex.fp8_matmul(got.rows, got.scales, b, bs,
                              offsets=got.offsets)
            z = ex.fp8_matmul(q, sc, b, bs, offsets=batch.offsets)
            assert torch.equal(y, z)
            back = exchange.combine(y, got, w.cuda())
            assert back.shape == (x.shape[0], 64)
            assert torch.isfinite(back).all()
        print(f"case {case} rank {rank} ok", flush=True)
    dist.barrier()
    dist.destroy_process_group()
    print("ALL OK", flush=True)


if __name__ == "__main__":
    main()
