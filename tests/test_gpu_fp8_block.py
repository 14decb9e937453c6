"""Routing, row quantiser, 8-bit experts and the combine there was, one after the other as a serving loop runs them."""
import pytest
import torch

from tests.test_gpu_fp8_rows import expert_layer, expert_rows, rows

pytestmark = pytest.mark.gpu


def run(backend, block, logits, x, k, out, **kw):
    """The block on the caller's own logits, in 8-bit arithmetic: out [T,H] bf16."""
    T, H = x.shape
    r = backend.route_logits_dev(logits, k, norm_topk=True, **kw)
    codes, scales = backend.quantize_rows_fp8_dev(x, r.row_token)
    y = torch.empty((T * k, H), dtype=torch.bfloat16, device=x.device)
    block.experts_fp8_dev(codes, scales, r.expert_rows, T * k, y)
    partial = torch.empty((T, H), device=x.device)
    st = torch.cuda.current_stream().cuda_stream
    block.combine_partial_dev(y, r.slot, r.w, partial, st)
    block.finish_dev(partial, None, out, st)
    return r, codes, scales


def test_calls_on_a_given_stream(gpu_backend):
    # results and the router's counts come from the given stream's memory, so that calls in turn on two streams share none in flight
    b, side = gpu_backend, [torch.cuda.Stream() for _ in range(2)]
    x, z = torch.randn((5000, 512), device="cuda"), torch.randn((5000, 64), device="cuda")
    codes, scales = b.quantize_fp8_b128_dev(torch.randn((256, 512), device="cuda"))
    w = b.CudaTensor.from_device(8, codes, scales, 1.0, 512, 256)
    want = [*b.route_logits_dev(z, 4), *b.quantize_rows_fp8_dev(x)]
    want.append(b.matmul_fp8_dev(w, want[5], want[6]))
    torch.cuda.synchronize()
    got = []
    for i in range(24):
        s = 0 if i % 3 == 2 else side[i % 3].cuda_stream
        r, (q, sx) = b.route_logits_dev(z, 4, stream=s), b.quantize_rows_fp8_dev(x, stream=s)
        got.append([*r, q, sx, b.matmul_fp8_dev(w, q, sx, stream=s)])
    torch.cuda.synchronize()
    assert torch.cuda.current_stream() == torch.cuda.default_stream()
    for r in got:
        assert all(torch.equal(a, v) for a, v in zip(r, want))
    w.free()


@pytest.mark.parametrize("T,E,k,H,I,pad", [(1, 8, 2, 256, 128, 0), (7, 8, 1, 128, 64, 2), (40, 16, 4, 512, 264, 3), (300, 8, 2, 640, 256, 50)])
def test_the_operators_in_a_row(gpu_backend, T, E, k, H, I, pad):
    from speedycolibri_b200.configs import FMT_FP8_B128
    from speedycolibri_b200.moe import Config, MoeBlock

    one, values = expert_layer(gpu_backend, E, H, I, T)
    block = MoeBlock(Config(H, E, k, I, fmt=FMT_FP8_B128), one.layer, T)
    x = rows(T, H, 40).to(torch.bfloat16)
    z = rows(T, E, 41)
    z[T - pad :] = float("-inf")
    out = torch.empty((T, H), dtype=torch.bfloat16, device="cuda")
    r, codes, scales = run(gpu_backend, block, z, x, k, out)
    block.check()
    n = int(r.expert_rows.sum())
    assert n == (T - pad) * k
    y, tol = expert_rows(codes[:n], scales[:n], r.expert_rows.tolist(), values)
    slot, w = r.slot.long(), r.w.double()
    want = (y[slot.clamp_min(0)] * w[:, :, None] * (slot >= 0)[:, :, None]).sum(1)
    size = (y[slot.clamp_min(0)].abs() * w[:, :, None] * (slot >= 0)[:, :, None]).sum(1)
    off = (tol[slot.clamp_min(0)] * w[:, :, None] * (slot >= 0)[:, :, None]).sum(1)
    # y's own error weighted, k sums in f32, one rounding to bf16
    assert ((out.double() - want).abs() <= off + (k + 1) * 2.0**-24 * size + 2.0**-8 * (want.abs() + off)).all()
    assert (out[T - pad :] == 0).all()

    # the same sequence captured and replayed on other inputs of the same shapes
    g = torch.cuda.CUDAGraph()
    captured = torch.empty_like(out)
    with torch.cuda.graph(g):
        run(gpu_backend, block, z, x, k, captured)
    x2, z2 = rows(T, H, 42).to(torch.bfloat16), rows(T, E, 43)
    run(gpu_backend, block, z2, x2, k, out)
    x.copy_(x2)
    z.copy_(z2)
    g.replay()
    block.check()
    assert torch.equal(captured, out)
    block.close()
    one.close()
