"""Every form of the tensor-memory product that a call can take: which one a call takes (host side, on the CPU), and its results on the GPU."""
import ctypes as C
import subprocess

import pytest

from speedycolibri_b200 import _lib

STREAM = (0, 0, 0)
# (rows, K, O): rows and columns of a tile, CTAs that share one
PRODUCTS = {
    (65, 170, 9997): (128, 128, 1), (2477, 2177, 153): (128, 128, 2), (1252, 1518, 151): (128, 128, 4),
    (66, 155, 19195): (128, 256, 1), (65, 5663, 9575): (128, 256, 2), (67, 5067, 5381): (128, 256, 4), (4096, 1024, 4096): (128, 256, 1),
    (33, 158, 151): (64, 128, 1), (34, 1480, 4835): (64, 128, 2), (49, 975, 154): (64, 128, 4),
    (35, 154, 19642): (64, 256, 1), (33, 2483, 9817): (64, 256, 2), (35, 1798, 4769): (64, 256, 4),
    (9, 157, 19277): (32, 256, 1), (19, 2268, 9541): (32, 256, 2), (30, 1388, 4855): (32, 256, 4),
    (8, 1388, 4855): STREAM,
}
# (experts, H, I, rows, rows expected): of gate and up (the columns are 128 features of each), of down
EXPERTS = {
    (38, 136, 136, 4936, 4936): ((128, 256, 1), (128, 256, 1)), (32, 648, 640, 3200, 3200): ((128, 256, 1), (128, 128, 1)),
    (53, 296, 136, 3513, 3513): ((64, 256, 1), (128, 128, 1)), (42, 136, 128, 5515, 5515): ((64, 256, 1), (128, 256, 1)),
    (17, 1416, 144, 94, 94): ((32, 256, 2), (32, 256, 1)), (2, 928, 936, 10, 10): ((32, 256, 4), (32, 256, 4)), (35, 136, 1424, 195, 195): ((32, 256, 1), (32, 256, 2)),
    (14, 1440, 136, 428, 428): ((64, 256, 2), (64, 256, 1)), (3, 928, 1032, 66, 66): ((64, 256, 4), (64, 128, 4)), (11, 136, 1424, 529, 529): ((64, 256, 1), (64, 128, 2)),
    (33, 144, 2456, 667, 667): ((64, 256, 1), (64, 256, 2)), (13, 136, 1832, 385, 385): ((64, 256, 1), (64, 256, 4)), (2, 136, 136, 46, 46): ((64, 256, 1), (64, 128, 1)),
    # many more rows than expected: a cluster takes several tiles, one after the other
    (2, 1440, 1032, 3000, 50): ((64, 256, 4), (64, 128, 4)), (2, 1440, 1032, 3000, 12): ((32, 256, 4), (32, 256, 4)),
    (2, 1440, 1032, 300, 4): (STREAM, STREAM),
}
NEVER = {(True, 128, 256, 2), (True, 128, 256, 4)}  # 128-row tiles of gate and up are more than the SMs

SOURCE = r"""
#include "fp8.cuh"
extern "C" void plan_of(int rows, int K, int O, int nseg, int expected, int gated, int *out) {
  colib::Fp8MmParams p = {};
  p.rows = rows, p.K = K, p.O = O, p.nseg = nseg ? nseg : 1, p.rows_expected = expected, p.KT = (K + 127) / 128;
  static const int counts = 0;
  if (nseg) p.seg_count = &counts;
  static uint8_t codes;
  if (gated) p.h_codes = &codes;
  if (colib::fp8_stream_ok(p)) return;
  const colib::Fp8Plan plan = colib::fp8_plan(p);
  out[0] = plan.ar, out[1] = plan.bn, out[2] = plan.split;
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("fp8_plan")
    src, lib = str(d / "plan.cu"), str(d / "libplan.so")
    open(src, "w").write(SOURCE)
    subprocess.run(["nvcc", *_lib.NVCC_FLAGS, "-I", _lib._CSRC, "-o", lib, src], check=True, capture_output=True)
    fn = C.CDLL(lib).plan_of

    def call(rows, K, O, nseg=0, expected=0, gated=False):
        out = (C.c_int * 3)()
        fn(rows, K, O, nseg, min(rows, expected) if nseg else rows, gated, out)
        return tuple(out)

    return call


def test_products_take_their_form(plan):
    assert {c: plan(*c) for c in PRODUCTS} == PRODUCTS


def test_experts_take_their_form(plan):
    assert {c: (plan(c[3], c[1], c[2], c[0], c[4], True), plan(c[3], c[2], c[1], c[0], c[4])) for c in EXPERTS} == EXPERTS


def test_every_form_is_among_them(plan):
    """Over many shapes no form comes up that the cases above have not."""
    import random

    have = {(False, *f) for f in PRODUCTS.values()} | {(True, *g) for g, _ in EXPERTS.values()} | {(False, *d) for _, d in EXPERTS.values()}
    rng, seen = random.Random(1), set()
    size = lambda lo, hi: int(lo * (hi / lo) ** rng.random())  # noqa: E731
    for _ in range(60000):
        rows, E, H, I = size(1, 20000), size(1, 400), size(1, 16384), size(1, 8192)
        seen |= {(False, *plan(rows, H, I)), (True, *plan(rows, H, I, E, rows, True)), (False, *plan(rows, I, H, E, rows))}
    assert seen <= have and not seen & NEVER


def product_case(backend, T, K, O, dtype):
    import torch

    from tests.test_gpu_fp8_rows import E4M3, product_bound, rows, spread, weight

    w, wv = weight(backend, O, K, 5)
    q, s = backend.quantize_rows_fp8_dev(rows(T, K, 6))
    y = backend.matmul_fp8_dev(w, q, s, out_dtype=dtype)
    backend.fp8_check()
    want = (q.view(E4M3).double() * spread(s.double(), K)) @ wv.t()
    assert ((y.double() - want).abs() <= product_bound(q, s, wv, want, dtype)).all()
    assert torch.equal(y, backend.matmul_fp8_dev(w, q, s, out_dtype=dtype))
    w.free()


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("case", PRODUCTS)
def test_product(gpu_backend, case, ty):
    import torch

    product_case(gpu_backend, *case, getattr(torch, ty))


@pytest.mark.gpu
@pytest.mark.parametrize("skew", [False, True])
@pytest.mark.parametrize("case", EXPERTS)
def test_experts(gpu_backend, case, skew):
    import torch

    from tests.test_gpu_fp8_rows import expert_layer, expert_rows, rows

    E, H, I, R, expected = case
    counts = [R // E + (e < R % E) for e in range(E)]
    if skew:  # some experts without a row, their rows at the others (the form goes by the average alone)
        for e in range(0, E - 1, 2):
            counts[e], counts[e + 1] = counts[e] % 2, counts[e + 1] + counts[e] - counts[e] % 2
    block, values = expert_layer(gpu_backend, E, H, I, R)
    q, s = gpu_backend.quantize_rows_fp8_dev(rows(R, H, 30))
    seg = torch.tensor(counts, dtype=torch.int32, device="cuda")
    y = torch.empty((R, H), dtype=torch.bfloat16, device="cuda")
    block.experts_fp8_dev(q, s, seg, expected, y)
    block.check()
    want, tol = expert_rows(q, s, counts, values)
    assert ((y.double() - want).abs() <= tol).all()
    again = torch.empty_like(y)
    block.experts_fp8_dev(q, s, seg, expected, again)
    assert torch.equal(y, again)
    block.close()
