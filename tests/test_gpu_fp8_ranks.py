"""The 8-bit expert call on a rank's handle: its own experts in its own order, beside a shared expert."""
import numpy as np
import pytest
import torch

from tests.test_gpu_fp8_rows import rows, weight

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("each", [1, 20])
@pytest.mark.parametrize("owner", [None, [1, 0, 0, 1, 1, 0]])
def test_a_ranks_experts(gpu_backend, owner, each):
    from speedycolibri_b200.configs import FMT_FP8_B128
    from speedycolibri_b200.moe import Config, Expert, Layer, MoeBlock

    E, H, I = 6, 256, 136
    made = [Expert(*(weight(gpu_backend, o, k, 3 * e + i)[0] for i, (o, k) in enumerate([(I, H), (I, H), (H, I)]))) for e in range(E + 1)]
    router = np.zeros((E, H), np.uint16)
    for rank in range(2):
        mine = [e for e in range(E) if (owner[e] if owner else e * 2 // E) == rank]
        block = MoeBlock(Config(H, E, 1, I, fmt=FMT_FP8_B128), Layer(router, [made[e] if e in mine else None for e in range(E)], shared=made[E]), 64,
                         ep_rank=rank, ep_world=2, expert_owner=owner)
        alone = MoeBlock(Config(H, len(mine), 1, I, fmt=FMT_FP8_B128), Layer(router[: len(mine)], [made[e] for e in mine]), 64)
        assert block.local_experts() == len(mine)
        counts = [each + i for i in range(len(mine))]
        R = sum(counts)
        q, s = gpu_backend.quantize_rows_fp8_dev(rows(R, H, 40 + rank))
        seg = torch.tensor(counts, dtype=torch.int32, device="cuda")
        y, want = (torch.empty((R, H), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        block.experts_fp8_dev(q, s, seg, R, y)
        alone.experts_fp8_dev(q, s, seg, R, want)
        block.check()
        assert torch.equal(y, want)
        block.close()
        alone.close()
