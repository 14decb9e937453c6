"""The row quantiser code by code.

The definition has one rounding a step, so that f32 arithmetic that rounds correctly (the host's division) gives its scales and codes:
s = max(f32(a / 448), 2^-126), code = e4m3(f32(x / s)), to nearest even.  (A zero's and a NaN's sign carry nothing.)"""
import numpy as np
import pytest
import torch

from tests.test_gpu_fp8_rows import E4M3, rows

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def definition(x):
    """Rows of any type -> (codes as bytes, scales f32), on the host."""
    v = x.cpu().float().numpy()
    T, K = v.shape
    codes, scales = np.empty((T, K), np.uint8), np.empty((T, (K + 127) // 128), np.float32)
    for b, c in enumerate(range(0, K, 128)):
        part = v[:, c : c + 128]
        a = np.abs(part).max(1)
        s = np.where(a > 0, np.maximum(a / np.float32(448), np.float32(2.0**-126)), np.float32(1)).astype(np.float32)
        with np.errstate(invalid="ignore"):  # infinity by infinity
            quotient = part / s[:, None]
        q = torch.from_numpy(quotient).clamp(-448, 448).to(E4M3).view(torch.uint8).numpy()
        codes[:, c : c + 128], scales[:, b] = q, s
    return torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda()


def half_way_rows(K, dtype):
    """Blocks whose largest value makes the scale an odd number of few bits times a power of two, and whose other values are that scale
    times every value half-way between two codes: all exact in 8 bits."""
    mids = [m * 2.0**e for e in range(-5, 9) for m in (17, 19, 21, 23, 25, 27, 29, 31) if m * 2.0**e < 448] + [(2 * i + 1) * 2.0**-10 for i in range(8)]
    mids = np.array(mids + [-m for m in mids])
    out = []
    for r in range(64):
        s = (1, 3, 5, 7)[r % 4] * 2.0 ** ((r // 4) % 6 - 3)
        row = np.random.default_rng(r).choice(mids, K) * s
        row[::128] = 448 * s * (-1) ** r
        out.append(row)
    x = torch.from_numpy(np.array(out)).cuda()
    assert torch.equal(x.to(dtype).double(), x)
    return x.to(dtype)


def same(got, want):
    assert torch.equal(got[1], want[1])
    a, b = (c.view(E4M3).float() for c in (got[0], want[0]))
    assert ((a == b) | (a.isnan() & b.isnan())).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K", [1, 128, 300, 1000, 2048, 3000])
def test_codes_of_random_rows(gpu_backend, dtype, K):
    for seed, size in ((1, 1.0), (2, 1e-3), (3, 40.0)):
        x = (rows(200, K, seed) * size).to(dtype)
        same(gpu_backend.quantize_rows_fp8_dev(x), definition(x))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K", [136, 1000, 2048])
def test_codes_of_values_half_way(gpu_backend, dtype, K):
    x = half_way_rows(K, dtype)
    want = definition(x)
    same(gpu_backend.quantize_rows_fp8_dev(x), want)
    # off the 16-byte grid, value by value
    base = torch.zeros((64, K + 5), dtype=dtype, device="cuda")
    base[:, 3 : 3 + K] = x
    same(gpu_backend.quantize_rows_fp8_dev(base[:, 3 : 3 + K]), want)
    # gathered, whole pieces and value by value
    take = torch.randperm(64, device="cuda").to(torch.int32)
    for src in (x, base[:, 3 : 3 + K]):
        q, s = gpu_backend.quantize_rows_fp8_dev(src, take)
        same((q, s), (want[0][take.long()], want[1][take.long()]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("exponent", [-140, -133, -126, -125, -124, -120, -118, -117, -116, -110, -105, -101, -100, -99, -50, 60, 118])
def test_codes_at_the_ends_of_the_range(gpu_backend, dtype, exponent):
    x = (rows(100, 384, 7).double() * 2.0**exponent).to(dtype)
    same(gpu_backend.quantize_rows_fp8_dev(x), definition(x))
    x = (half_way_rows(256, torch.float32).double() * 2.0 ** min(exponent, 115)).to(dtype)
    same(gpu_backend.quantize_rows_fp8_dev(x), definition(x))
