"""A handle's workspace over expert calls of rising sizes (host side over a fake runtime)."""
import ctypes as C

import numpy as np

from speedycolibri_b200 import _lib
from tests.test_fp8_refusals_cpu import A, S, W, Y, bind, weight


def test_rising_sizes_grow_the_workspace_a_few_times(fake_cuda):
    fake, H, I, E = bind(fake_cuda), 32, 16, 4
    fake.coli_b200_moe_workspace_bytes.restype, fake.coli_b200_moe_workspace_bytes.argtypes = _lib.SIGNATURES["coli_b200_moe_workspace_bytes"]
    tables = [(C.c_void_p * E)(*[weight(fake, o, k) for _ in range(E)]) for o, k in ((I, H), (I, H), (H, I))]
    router = np.zeros((E, H), np.uint16)
    L = _lib.ColiMoeLayer(H=H, E=E, k=2, I=I, fmt=8, n_group=1, topk_group=1, ep_world=1, router_w=router.ctypes.data)
    L.gate, L.up, L.down = (C.cast(t, C.POINTER(C.c_void_p)) for t in tables)
    h = C.c_void_p()
    assert fake.coli_b200_moe_create(C.byref(h), C.byref(L), 64)
    for expected in (lambda rows: 8, lambda rows: rows):  # few rows an expert: h in f32 too
        start, sizes = fake.coli_b200_moe_workspace_bytes(h), set()
        for rows in range(1, 6001):
            fake.fake_reset(0)
            assert fake.coli_b200_moe_experts_fp8_dev(h, A, 32, S, 1, rows, W, rows, expected(rows), Y, None)
            sizes.add(fake.coli_b200_moe_workspace_bytes(h))
        need = 6000 * (16 + 4 + 64) + 16
        assert len(sizes) <= 16 and max(sizes) - start <= 4 * need, (len(sizes), max(sizes) - start)
