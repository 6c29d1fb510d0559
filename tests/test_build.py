"""What the build refuses: compiled with the build's own flags, no GPU needed."""

import subprocess

import pytest

from ascendflow_amd import build

KERNEL = """
#include <hip/hip_runtime.h>
__global__ void sum(float* out, const float* in, int n) {
  float s = 0.f;
#pragma clang loop unroll(full)
  for (int i = 0; i < %s; ++i) s += in[i];
  *out = s;
}
"""


@pytest.mark.parametrize("count,taken", [("8", True), ("n", False)])
def test_a_loop_that_is_not_unrolled_as_marked_is_an_error(tmp_path, count, taken):
    source = tmp_path / "kernel.hip"
    source.write_text(KERNEL % count)
    run = subprocess.run([build.hipcc(), *build.HIP_FLAGS, "-c", str(source), "-o", str(tmp_path / "kernel.o")], capture_output=True, text=True)
    assert (run.returncode == 0) == taken, run.stderr
    assert taken or "loop not unrolled" in run.stderr
