"""The codes of h inside the 8-bit expert call are those of the row quantiser's rule, whichever kernel makes them.

gate x = 64 (silu(64) is 64 in f32), up x = whole numbers summed of 4-bit digits, so that h is exact; down is the identity, so that y
shows h's codes times their scale (a code has 4 bits, the scale 4 more at most: exact in bf16)."""
import numpy as np
import pytest
import torch

from tests.test_gpu_fp8_exact import definition
from tests.test_gpu_fp8_rows import E4M3

pytestmark = pytest.mark.gpu

ODD = [1, 3, 5, 7, 9, 11, 13, 15]  # the scales, times a power of two


def codes_of(v):
    return torch.from_numpy(np.asarray(v, np.float32)).to(E4M3).view(torch.uint8)


@pytest.mark.parametrize("H", [256, 1024])       # (one CTA a tile, or several that share its k-tiles)
@pytest.mark.parametrize("each", [1, 5, 30, 100])  # rows of an expert
@pytest.mark.parametrize("power", [0, -100])
def test_half_way_values_of_h(gpu_backend, H, each, power):
    from speedycolibri_b200.configs import FMT_FP8_B128
    from speedycolibri_b200.moe import Config, Expert, Layer, MoeBlock

    I, E = 256, len(ODD)
    R = E * each
    x = np.zeros((R, H), np.float32)
    x[:, :5] = 1, 16, 256, 256, 64
    up_scale, down_scale = np.float32(2.0 ** (power - 16)), np.float32(1.0)
    rng, experts, h = np.random.default_rng(1), [], np.zeros((E, I))
    mids = np.array([m * 2**e for m in range(17, 32, 2) for e in range(4)])  # half-way between two codes
    for e, odd in enumerate(ODD):
        v = rng.choice(mids, I) * odd
        v[::128] = 448 * odd  # the largest of its block: the scale is `odd` times a power of two
        gate, up, down = np.zeros((I, H), np.float32), np.zeros((I, H), np.float32), np.zeros((H, I), np.float32)
        gate[:, 4] = 1
        up[:, 0], up[:, 1], up[:, 2], up[:, 3] = v % 16, v // 16 % 16, v // 256 % 16, v // 4096 * 16
        down[np.arange(I), np.arange(I)] = 1
        made = [gpu_backend.CudaTensor.from_device(FMT_FP8_B128, codes_of(m).cuda(), torch.full(((m.shape[0] + 127) // 128, (m.shape[1] + 127) // 128), float(s), device="cuda"),
                                                   1.0, m.shape[1], m.shape[0]) for m, s in ((gate, 1.0), (up, up_scale), (down, down_scale))]
        assert all((codes_of(m).view(E4M3).float().numpy() == m).all() for m in (gate, up, down))
        experts.append(Expert(*made))
        h[e] = 64.0 * v * float(up_scale)
    assert (h == h.astype(np.float32)).all()
    q, s = definition(torch.from_numpy(h.astype(np.float32)))
    want = (q.view(E4M3).double() * s.double().repeat_interleave(128, 1)).repeat_interleave(each, 0)
    assert torch.equal(want, want.to(torch.bfloat16).double())
    block = MoeBlock(Config(H, E, 1, I, fmt=FMT_FP8_B128), Layer(np.zeros((E, H), np.uint16), experts), R)
    codes = codes_of(x).cuda()
    y = torch.empty((R, H), dtype=torch.bfloat16, device="cuda")
    block.experts_fp8_dev(codes, torch.ones((R, (H + 127) // 128), device="cuda"), torch.full((E,), each, dtype=torch.int32, device="cuda"), R, y)
    block.check()
    assert torch.equal(y[:, :I].double(), want) and (y[:, I:] == 0).all()
    block.close()
