"""Products whose scales, multiplied with each other, leave f32's normal range, where scale x scale x sum does not."""
import numpy as np
import pytest
import torch

from tests.test_gpu_fp8_rows import E4M3, expert_rows

pytestmark = pytest.mark.gpu


def product(q, s, w, ws):
    """f64; scales applied one block after the other."""
    y = torch.zeros((q.shape[0], w.shape[0]), dtype=torch.float64, device="cuda")
    size = torch.zeros_like(y)
    for b in range(s.shape[1]):
        c = slice(128 * b, 128 * (b + 1))
        sc = s[:, b : b + 1].double() * ws[:, b].double().repeat_interleave(128)[: w.shape[0]]
        y += (q.view(E4M3)[:, c].double() @ w.view(E4M3)[:, c].double().t()) * sc
        size += (q.view(E4M3)[:, c].double().abs() @ w.view(E4M3)[:, c].double().abs().t()) * sc
    return y, size


def random_codes(R, K, seed, bits=0x7E):
    """Codes of magnitudes up to `bits`, of either sign."""
    g = torch.Generator("cuda").manual_seed(seed)
    q = torch.randint(0, bits + 1, (R, (K + 15) // 16 * 16), dtype=torch.uint8, device="cuda", generator=g)
    return (q | (torch.rand(q.shape, device="cuda", generator=g) < 0.5).to(torch.uint8) * 128)[:, :K]


# scale of the rows, of the weights: their product is below 2^-126 (at (2^-140, 1) one factor is itself), below 2^-149, above 2^128
@pytest.mark.parametrize("sx,sw", [(2.0**-120, 2.0**-12), (2.0**-120, 2.0**-20), (1e-38, 1e-6), (1e-38, 1e-8), (1e-8, 1e-38), (2.0**-75, 2.0**-75),
                                   (2.0**-140, 1.0), (1e36, 1e5), (1e5, 1e36), (1e20, 1e20), (1e34, 1e5), (1e5, 1e34)])
@pytest.mark.parametrize("T", [1, 8, 40, 65, 200, 1300])
def test_product_of_scales_outside_f32(gpu_backend, sx, sw, T):
    from speedycolibri_b200.configs import FMT_FP8_B128

    K, O = 1300, 200
    big = sx * sw > 1
    q, w = random_codes(T, K, 1, 0x07 if big else 0x7E), random_codes(O, K, 2, 0x07 if big else 0x7E).contiguous()  # (codes up to 2^-6: results in range)
    if T > 2:
        q[2] = 0  # a row of zeros gives zeros
    g = torch.Generator("cuda").manual_seed(3)
    vary = lambda *n: torch.exp2(torch.rand(n, device="cuda", generator=g).double())  # noqa: E731
    s, ws = (vary(T, (K + 127) // 128) * sx).float(), (vary((O + 127) // 128, (K + 127) // 128) * sw).float()
    s[:, 3], ws[:, 4] = 1.0 / sw if big else s[:, 3], ws[:, 4]  # (a block with ordinary scales among them)
    h = gpu_backend.CudaTensor.from_device(FMT_FP8_B128, w, ws, 1.0, K, O)
    y = gpu_backend.matmul_fp8_dev(h, q, s, out_dtype=torch.float32)
    gpu_backend.fp8_check()
    want, size = product(q, s, w, ws)
    # A sum whose magnitudes add up beyond f32 (1300 (7 2^-9)^2 4 1e41 = 9.8e40 with the largest scales) may leave it on the way,
    # whatever the order, so that only a product whose magnitudes fit has one value.
    fits = size < 3e38
    # K sums in any order, three roundings of a term; below 2^-126 half a step, 2^-150, a term and sum
    tol = (K + 4) * 2.0**-24 * size + (s.shape[1] * 2 + 2) * 2.0**-149
    assert ((y.double() - want).abs() <= tol)[fits].all() and (fits.float().mean() > 0.9 or sx * sw > 1e39)
    if T > 2:
        assert (y[2] == 0).all()
    h.free()


@pytest.mark.parametrize("odd", [1.0, 2.0**-120])
@pytest.mark.parametrize("T", [1, 8, 40, 200, 1300])
def test_scales_of_zero(gpu_backend, T, odd):
    """Rows and blocks of weights whose scale is 0 add nothing; the rows beside them keep their results, with tiny scales among them too."""
    from speedycolibri_b200.configs import FMT_FP8_B128

    K, O = 1300, 333
    q, w = random_codes(T, K, 4), random_codes(O, K, 5).contiguous()
    s, ws = torch.full((T, 11), 0.01, device="cuda"), torch.full((3, 11), 0.01, device="cuda")
    ws[0, 2], ws[1, :], ws[2, 10] = 0.0, 0.0, 0.0
    s[0, 3] = 0.0
    if T > 1:
        s[1, :], s[T - 1, 10] = 0.0, 0.0
        s[T // 2, 5] = odd
    h = gpu_backend.CudaTensor.from_device(FMT_FP8_B128, w, ws * (1.0 if odd == 1.0 else 2.0**-10), 1.0, K, O)
    y = gpu_backend.matmul_fp8_dev(h, q, s, out_dtype=torch.float32)
    gpu_backend.fp8_check()
    want, size = product(q, s, w, ws * (1.0 if odd == 1.0 else 2.0**-10))
    assert ((y.double() - want).abs() <= (K + 4) * 2.0**-24 * size + 24 * 2.0**-149).all()
    assert (y[:, 128:256] == 0).all()
    h.free()


@pytest.mark.parametrize("counts", [[1, 1], [9, 7], [40, 90], [200, 300]])
def test_experts_with_scales_outside_f32(gpu_backend, counts):
    """A block of zero codes adds nothing, whatever its scale, and what the weights' scales lose the rows' gain: the same results up
    to the order of the sums (the bounds are those of any call)."""
    from speedycolibri_b200.configs import FMT_FP8_B128
    from speedycolibri_b200.moe import Config, Expert, Layer, MoeBlock

    H, I, R, E = 512, 136, sum(counts), len(counts)

    def made(O, K, seed, scale):
        w = random_codes(O, K, seed).contiguous()
        return gpu_backend.CudaTensor.from_device(FMT_FP8_B128, w, torch.full(((O + 127) // 128, (K + 127) // 128), scale, device="cuda"), 1.0, K, O)

    seg = torch.tensor(counts, dtype=torch.int32, device="cuda")
    q, s = random_codes(R, H, 9), torch.full((R, H // 128), 2.0**-20, device="cuda")
    q[:, 128:256] = 0
    values = [[random_codes(o, k, base + e).view(E4M3).double() * 2.0**-8 for o, k, base in ((I, H, 20), (I, H, 30), (H, I, 40))] for e in range(E)]
    want, tol = expert_rows(q, s, counts, values)
    assert want.abs().max() > 0
    for scale, rows_scale in ((2.0**-8, 1.0), (2.0**100, 2.0**-108), (2.0**-120, 2.0**112)):
        experts = [Expert(made(I, H, 20 + e, scale), made(I, H, 30 + e, scale), made(H, I, 40 + e, 2.0**-8)) for e in range(E)]
        block = MoeBlock(Config(H, E, 1, I, fmt=FMT_FP8_B128), Layer(np.zeros((E, H), np.uint16), experts), R)
        sc = s * rows_scale
        sc[:, 1] = 2.0**100  # of zeros
        y, again = (torch.empty((R, H), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        for out in (y, again):
            block.experts_fp8_dev(q, sc, seg, R, out)
        block.check()
        assert ((y.double() - want).abs() <= tol).all() and torch.equal(y, again)
        block.close()
