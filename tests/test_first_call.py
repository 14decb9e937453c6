"""The calls without a handle as a program's first ones, before the library is initialised."""
import os
import subprocess
import sys

import pytest

from tests.conftest import ROOT
from tests.test_fp8_refusals_cpu import A, B, S, W, Y, at, bind


def test_before_initialisation(tmp_path):
    from tests.fake_cuda import load

    fake = bind(load(tmp_path))  # a library of its own: the session's keeps its devices
    fake.coli_cuda_shutdown()
    assert fake.coli_cuda_device_count() == 0

    def quantise(device):
        fake.fake_reset(0)
        return fake.coli_b200_quantize_rows_fp8(device, A, 2, 40, None, 5, 5, 40, B, 48, S, 1, 5, None), fake.fake_queued()

    def route(device):
        fake.fake_reset(0)
        return fake.coli_b200_route_logits(device, A, 0, 64, None, None, 100, 64, 4, 1, 1, 1.0, 1, 1, B, S, W, Y, at(Y, 4096), None, None), fake.fake_queued()

    for call in (quantise, route):
        assert call(0) == (1, 1) and call(1) == (0, 0) and call(-1) == (0, 0) and call(40) == (0, 0)
    assert fake.coli_cuda_device_count() == 0  # the calls initialise nothing: any set of devices may follow


PROGRAM = """
import torch
from speedycolibri_b200 import backend
x = torch.randn((33, 300), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
z = x[:, :64]
first = [*(backend.quantize_rows_fp8_dev(x) if {quantise} else ()), *backend.route_logits_dev(z, 4), *backend.quantize_rows_fp8_dev(x)]
backend.init([0])
then = [*(backend.quantize_rows_fp8_dev(x) if {quantise} else ()), *backend.route_logits_dev(z, 4), *backend.quantize_rows_fp8_dev(x)]
assert all(torch.equal(a, b) for a, b in zip(first, then))
print("equal", len(first))
"""


@pytest.mark.gpu
@pytest.mark.parametrize("quantise", [True, False])
def test_before_initialisation_on_the_gpu(quantise):
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    r = subprocess.run([sys.executable, "-c", PROGRAM.format(quantise=quantise)], cwd=ROOT, env=dict(os.environ, PYTHONPATH=ROOT), capture_output=True,
                       text=True, timeout=240)
    assert r.returncode == 0 and "equal" in r.stdout, r.stderr[-2000:]


CAPTURED = """
import torch
from speedycolibri_b200 import backend
x, z = torch.randn((33, 300), device="cuda"), torch.randn((3000, 64), device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    first = [*backend.quantize_rows_fp8_dev(x), *backend.route_logits_dev(z, 4)]
g.replay()
then = [*backend.quantize_rows_fp8_dev(x), *backend.route_logits_dev(z, 4)]
assert all(torch.equal(a, b) for a, b in zip(first, then))
print("equal")
"""


@pytest.mark.gpu
def test_captured_first_calls():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    r = subprocess.run([sys.executable, "-c", CAPTURED], cwd=ROOT, env=dict(os.environ, PYTHONPATH=ROOT), capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and "equal" in r.stdout, r.stderr[-2000:]
