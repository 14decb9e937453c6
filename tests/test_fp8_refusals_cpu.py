"""What the 8-bit row calls and routing from logits refuse before anything is launched (host side over a fake runtime)."""
import ctypes as C

import numpy as np
import pytest

from speedycolibri_b200 import _lib

A, B, S, W, Y = (C.c_void_p(0x7000000 + i * 0x1000000) for i in range(5))  # stand-ins for device buffers: nothing reads them here
H, I, E = 32, 16, 4


def bind(fake):
    for name in ("coli_b200_quantize_rows_fp8", "coli_b200_matmul_fp8_dev", "coli_b200_moe_experts_fp8_dev", "coli_b200_route_logits",
                 "coli_b200_route_logits_workspace", "coli_cuda_last_error"):
        fn = getattr(fake, name)
        fn.restype, fn.argtypes = _lib.SIGNATURES[name]
    return fake


def weight(fake, O, K, fmt=8):
    h = C.c_void_p()
    q, s = np.zeros((O, K), np.uint8), np.ones(O * K, np.float32)
    fake.fake_reset(0)
    assert fake.coli_cuda_tensor_upload(C.byref(h), q.ctypes.data_as(C.c_void_p), s.ctypes.data_as(C.c_void_p), fmt, K, O, 0)
    return h


def at(p, d):
    return C.c_void_p(p.value + d)


def test_quantise(fake_cuda):
    fake = bind(fake_cuda)
    good = dict(device=0, x=A, ty=2, stride=40, take=None, T=5, rows=5, K=40, codes=B, ld=48, scales=S, sr=1, sb=5)

    def call(**kw):
        a = {**good, **kw}
        fake.fake_reset(0)
        ok = fake.coli_b200_quantize_rows_fp8(a["device"], a["x"], a["ty"], a["stride"], a["take"], a["T"], a["rows"], a["K"], a["codes"], a["ld"],
                                              a["scales"], a["sr"], a["sb"], None)
        return ok, fake.fake_queued()

    assert call() == (1, 1) and call(take=W, rows=9) == (1, 1) and call(x=at(A, 2), stride=41) == (1, 1) and call(rows=0) == (1, 1)
    for bad in (dict(ty=3), dict(ty=-1), dict(K=0), dict(T=-1), dict(rows=-1), dict(rows=6), dict(x=None), dict(codes=None), dict(scales=None),
                dict(take=W, rows=2**30 + 1), dict(x=at(A, 1)), dict(ty=0, x=at(A, 2)), dict(stride=-1), dict(ld=47), dict(ld=32), dict(ld=56), dict(codes=at(B, 8)),
                dict(scales=at(S, 2)), dict(sr=-1), dict(sb=-1), dict(take=at(W, 2)), dict(device=3)):
        assert call(**bad) == (0, 0), bad


def test_product(fake_cuda):
    fake = bind(fake_cuda)
    w, row_scaled = weight(fake, 24, 40), weight(fake, 24, 40, fmt=4)
    good = dict(w=w, codes=A, ld=48, scales=S, sr=1, sb=5, rows=5, y=Y, ty=2, ys=24)

    def call(**kw):
        a = {**good, **kw}
        fake.fake_reset(0)
        return fake.coli_b200_matmul_fp8_dev(a["w"], a["codes"], a["ld"], a["scales"], a["sr"], a["sb"], a["rows"], a["y"], a["ty"], a["ys"],
                                             None), fake.fake_queued()

    assert call() == (1, 1) and call(y=at(Y, 2), ys=33) == (1, 1) and call(rows=1, ys=0) == (1, 1)
    for bad in (dict(w=None), dict(w=row_scaled), dict(codes=None), dict(codes=at(A, 4)), dict(ld=40), dict(ld=50), dict(scales=None), dict(rows=-1), dict(rows=2**30 + 1),
                dict(y=None), dict(y=at(Y, 1)), dict(ty=0, y=at(Y, 2)), dict(ty=9), dict(ys=23), dict(sr=-1), dict(sb=-1), dict(ld=1 << 41)):
        assert call(**bad) == (0, 0), bad


@pytest.fixture(scope="module")
def handles(fake_cuda):
    fake = bind(fake_cuda)
    made = {}
    for fmt in (8, 4):
        tables = [(C.c_void_p * E)(*[weight(fake, o, k, fmt) for _ in range(E)]) for o, k in ((I, H), (I, H), (H, I))]
        router = np.zeros((E, H), np.uint16)
        L = _lib.ColiMoeLayer(H=H, E=E, k=2, I=I, fmt=fmt, n_group=1, topk_group=1, ep_world=1, router_w=router.ctypes.data)
        L.gate, L.up, L.down = (C.cast(t, C.POINTER(C.c_void_p)) for t in tables)
        h = C.c_void_p()
        assert fake.coli_b200_moe_create(C.byref(h), C.byref(L), 64)
        made[fmt] = h
    return made


def test_experts(fake_cuda, handles):
    fake = bind(fake_cuda)
    good = dict(m=handles[8], codes=A, ld=32, scales=S, sr=1, sb=9, counts=W, cap=9, expected=9, y=Y)

    def call(**kw):
        a = {**good, **kw}
        fake.fake_reset(0)
        return fake.coli_b200_moe_experts_fp8_dev(a["m"], a["codes"], a["ld"], a["scales"], a["sr"], a["sb"], a["counts"], a["cap"], a["expected"], a["y"],
                                                  None), fake.fake_queued()

    # gate/up and down, and between them the row quantiser where segments have two rows on average or fewer
    assert call() == (1, 2) and call(expected=2 * E) == (1, 3) and call(cap=0) == (1, 0) and call(expected=0) == (1, 3)
    assert call(cap=1000, expected=1000) == (1, 2)
    for bad in (dict(m=None), dict(m=handles[4]), dict(codes=None), dict(codes=at(A, 8)), dict(ld=24), dict(scales=None), dict(counts=None),
                dict(counts=at(W, 1)), dict(cap=-1), dict(cap=2**31 - 1), dict(expected=-1), dict(y=None), dict(y=at(Y, 8)), dict(sr=-2)):
        assert call(**bad) == (0, 0), bad


def test_routing(fake_cuda):
    fake = bind(fake_cuda)
    good = dict(device=0, z=A, ty=0, stride=64, sb=None, lb=None, T=2000, E=64, k=4, score=1, norm=1, scale=1.0, G=8, kept=4, idx=B, w=S, rows=W, slot=Y,
                token=at(Y, 4096), work=at(Y, 8192))

    def call(**kw):
        a = {**good, **kw}
        fake.fake_reset(0)
        return fake.coli_b200_route_logits(*[a[n] for n in ("device", "z", "ty", "stride", "sb", "lb", "T", "E", "k", "score", "norm", "scale", "G", "kept", "idx",
                                                            "w", "rows", "slot", "token", "work")], None), fake.fake_queued()

    assert call() == (1, 1) and call(T=512, work=None) == (1, 1) and call(T=0) == (1, 1) and call(T=1, stride=0) == (1, 1)
    assert fake.coli_b200_route_logits_workspace(512, 64) == 0 and fake.coli_b200_route_logits_workspace(513, 66) == 17 * 68
    for bad in (dict(T=-1), dict(E=0), dict(E=513, G=1, kept=1), dict(k=0), dict(k=33), dict(G=1, kept=1, E=3, k=4), dict(ty=5), dict(score=2), dict(G=0),
                dict(kept=0), dict(kept=9), dict(G=7), dict(G=64, kept=32), dict(G=16, kept=1, k=5), dict(z=None), dict(idx=None), dict(w=None),
                dict(rows=None), dict(slot=None), dict(token=None), dict(work=None), dict(stride=63), dict(stride=-1), dict(z=at(A, 2)),
                dict(sb=at(A, 1)), dict(lb=at(A, 2)), dict(idx=at(B, 2)), dict(device=5), dict(T=2**27, k=32, G=1, kept=1)):
        assert call(**bad) == (0, 0), bad
