"""The row quantiser bit for bit, and scales whose product leaves f32's normal range.

The quantiser's definition has one rounding a step, so that f32 arithmetic that rounds correctly (the host's division) gives its bits:
s = max(f32(a / 448), 2^-126), code = e4m3(f32(x / s)), to nearest even."""
import numpy as np
import pytest
import torch

from tests.test_gpu_fp8_rows import E4M3, expert_layer, rows

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
        q = torch.from_numpy(part / s[:, None]).clamp(-448, 448).to(E4M3).view(torch.uint8).numpy()
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
    assert torch.equal(got[0], want[0])


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
                                   (2.0**-140, 1.0), (1e36, 1e5), (1e5, 1e36), (1e20, 1e20)])
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
    want, size = product(q, s, w, ws.repeat_interleave(1, 0))
    big_enough = want.abs() < 3e38
    # K sums in any order, three roundings of a term; below 2^-126 half a step, 2^-150, a term and sum
    tol = (K + 4) * 2.0**-24 * size + (s.shape[1] * 2 + 2) * 2.0**-149
    assert ((y.double() - want).abs() <= tol)[big_enough].all() and big_enough.float().mean() > 0.99
    if T > 2:
        assert (y[2] == 0).all()
    h.free()


@pytest.mark.parametrize("counts", [[1, 1], [9, 7], [40, 90], [200, 300]])
def test_experts_with_scales_outside_f32(gpu_backend, counts):
    """A block of zero codes adds nothing, whatever its scale; small scales on both sides are kept."""
    from speedycolibri_b200.configs import FMT_FP8_B128
    from speedycolibri_b200.moe import Config, Expert, Layer, MoeBlock

    H, I, R = 512, 136, sum(counts)

    def made(O, K, seed, scale):
        w = random_codes(O, K, seed).contiguous()
        return gpu_backend.CudaTensor.from_device(FMT_FP8_B128, w, torch.full(((O + 127) // 128, (K + 127) // 128), scale, device="cuda"), 1.0, K, O)

    seg = torch.tensor(counts, dtype=torch.int32, device="cuda")
    q, s = random_codes(R, H, 9), torch.full((R, H // 128), 2.0**-20, device="cuda")
    q[:, 128:256] = 0
    out = []
    for scale, rows_scale in ((2.0**-8, 1.0), (2.0**100, 2.0**-108), (2.0**-120, 2.0**112)):
        # the same values in all: what the weights' scales lose the rows' gain
        experts = [Expert(made(I, H, 20 + e, scale), made(I, H, 30 + e, scale), made(H, I, 40 + e, 2.0**-8)) for e in range(len(counts))]
        block = MoeBlock(Config(H, len(counts), 1, I, fmt=FMT_FP8_B128), Layer(np.zeros((len(counts), H), np.uint16), experts), R)
        sc = s * rows_scale
        sc[:, 1] = 2.0**100  # of zeros
        y = torch.empty((R, H), dtype=torch.bfloat16, device="cuda")
        block.experts_fp8_dev(q, sc, seg, R, y)
        block.check()
        out.append(y)
        block.close()
    assert out[0].isfinite().all() and out[0].abs().max() > 0
    assert torch.equal(out[1], out[0]) and torch.equal(out[2], out[0])
