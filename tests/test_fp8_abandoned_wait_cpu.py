"""After a bounded wait has given up, a tile's addresses may never have been published: the warp that brings the scales must not use them.
The wait cannot be made to run out without a fault being risked, so this reads the role's source."""
import os
import re

from speedycolibri_b200 import _lib


def test_scales_are_loaded_only_while_every_wait_has_been_met():
    src = open(os.path.join(_lib._CSRC, "fp8.cu")).read()
    role = src[src.index("// ---------------- scales:") : src.index("// ---------------- scaled sums")]
    loads = [line for line in role.splitlines() if re.search(r"__ld\w+\(", line)]
    assert len(loads) == 2 and all("alive &&" in line.split("__ld")[0] for line in loads), loads
    assert "*sw" not in role.replace("float *sw", "") and "*sx" not in role.replace("float *sx", "")  # no other way to them
