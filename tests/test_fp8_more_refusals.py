"""Arguments of the 8-bit row and routing calls that were cut or written over one another, refused before anything is launched."""
import pytest

from tests.test_fp8_refusals_cpu import A, B, S, bind


def quantise(fake, rows, K, sr, sb):
    fake.fake_reset(0)
    ld = (K + 15) // 16 * 16
    return fake.coli_b200_quantize_rows_fp8(0, A, 2, K, None, rows, rows, K, B, ld, S, sr, sb, None), fake.fake_queued()


def test_columns(fake_cuda):
    fake, most = bind(fake_cuda), 65535 * 1024
    assert quantise(fake, 1, most, 0, 1) == (1, 1)
    for K in (most + 1, 2**31 - 1100, 2**31 - 300, 2**31 - 256, 2**31 - 1):  # (the grid's columns of these pass 32 bits)
        assert quantise(fake, 1, K, 0, 1) == (0, 0), K


def test_scales_in_one_place(fake_cuda):
    fake = bind(fake_cuda)
    for rows, K, sr, sb in ((5, 300, 1, 5), (5, 300, 3, 1), (5, 300, 7, 2), (5, 300, 2, 3), (1, 300, 0, 1), (5, 100, 1, 0), (1, 128, 0, 0), (5, 300, 3, 15), (5, 300, 9, 6)):
        places = {r * sr + b * sb for r in range(rows) for b in range((K + 127) // 128)}
        fits = len(places) == rows * ((K + 127) // 128)
        assert quantise(fake, rows, K, sr, sb) == ((1, 1) if fits else (0, 0)), (rows, K, sr, sb)
    for rows, K, sr, sb in ((5, 300, 0, 1), (5, 300, 1, 0), (5, 300, 0, 0), (5, 300, 1, 1), (5, 300, 1, 4), (2, 300, 1, 1), (5, 128, 0, 1)):
        assert quantise(fake, rows, K, sr, sb) == (0, 0), (rows, K, sr, sb)


@pytest.mark.gpu
def test_sizes_past_32_bits_in_python(gpu_backend):
    import torch

    from tests.test_gpu_fp8_rows import expert_layer, rows

    z = torch.zeros((4, 16), device="cuda")
    for kw in (dict(k=2**32 + 1), dict(k=2, n_group=2**32 + 1), dict(k=2, topk_group=2**32 + 1), dict(k=2, score=2**32), dict(k=2, n_group=-(2**32) + 1)):
        with pytest.raises(ValueError):
            gpu_backend.route_logits_dev(z, **kw)
    block, _ = expert_layer(gpu_backend, 2, 128, 64, 40)
    q, s = gpu_backend.quantize_rows_fp8_dev(rows(40, 128, 1))
    seg, y = torch.tensor([20, 20], dtype=torch.int32, device="cuda"), [torch.empty((40, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    block.experts_fp8_dev(q, s, seg, 40, y[0])
    block.experts_fp8_dev(q, s, seg, 2**32, y[1])  # more than there are rows: the rows there are
    assert torch.equal(*y)
    with pytest.raises(gpu_backend.CudaError):
        block.experts_fp8_dev(q, s, seg, -(2**32), y[0])
    with pytest.raises(gpu_backend.CudaError):
        gpu_backend.quantize_rows_fp8_dev(rows(4, 256, 1), out=(q[:4].new_empty((4, 256)), s.new_empty((4, 1)).expand(4, 2)))
    block.close()
