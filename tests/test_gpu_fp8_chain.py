"""Calls in a row that write over what the calls before them read: launches start early, so each must wait for all of its inputs and see
the new ones.  Small grids, so that several launches are resident at once."""
import pytest
import torch

from tests.test_gpu_fp8_rows import expert_layer, rows, weight

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [3, 20, 40, 300])
def test_quantise_and_product_over_the_same_buffers(gpu_backend, T):
    b, (w, _), n = gpu_backend, weight(gpu_backend, 600, 700, 1), 60
    xs = [rows(T, 700, 2 + i) * (1 + i) for i in range(4)]
    want = [b.matmul_fp8_dev(w, *b.quantize_rows_fp8_dev(x)) for x in xs]
    torch.cuda.synchronize()
    q, s = b.quantize_rows_fp8_dev(xs[0])
    ys = torch.empty((n, *want[0].shape), dtype=want[0].dtype, device="cuda")
    for i in range(n):
        b.quantize_rows_fp8_dev(xs[i % 4], out=(q, s))
        b.matmul_fp8_dev(w, q, s, out=ys[i])
    for i in range(n):
        assert torch.equal(ys[i], want[i % 4]), i


@pytest.mark.parametrize("T", [2, 30, 600])
def test_routing_quantiser_and_experts_over_the_same_buffers(gpu_backend, T):
    b, E, k, H, n = gpu_backend, 8, 2, 256, 40
    block, _ = expert_layer(b, E, H, 264, T * k)
    xs, zs = [rows(T, H, 5 + i) * (1 + i) for i in range(3)], [rows(T, E, 9 + i) for i in range(3)]
    bias = [rows(1, E, 15 + i)[0] * 0.1 for i in range(3)]

    def call(x, z, bias, r, q, y):
        r = b.route_logits_dev(z, k, norm_topk=True, select_bias=bias, out=r)
        q = b.quantize_rows_fp8_dev(x, r.row_token, out=q)
        block.experts_fp8_dev(*q, r.expert_rows, T * k, y)
        return r, q

    want, y = [], torch.empty((T * k, H), dtype=torch.bfloat16, device="cuda")
    for i in range(3):
        r, q = call(xs[i], zs[i], bias[i], None, None, y)
        torch.cuda.synchronize()
        want.append((y.clone(), r.w.clone()))
    ys, ws = torch.empty((n, T * k, H), dtype=torch.bfloat16, device="cuda"), torch.empty((n, T, k), device="cuda")
    for i in range(n):
        call(xs[i % 3], zs[i % 3], bias[i % 3], r._replace(w=ws[i]), q, ys[i])
    block.check()
    for i in range(n):
        assert torch.equal(ys[i], want[i % 3][0]) and torch.equal(ws[i], want[i % 3][1]), i
    block.close()
