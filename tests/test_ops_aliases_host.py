"""What the operators on rows refuse of buffers that lie upon each other, without a GPU: no call here names a device that exists, so
one that is not refused ends with PSKV_EHIP, and nothing is ever launched."""
import os
import subprocess

import pytest

from conftest import REPO


# --- the gradient of the position bias ---------------------------------------------------------------------------

@pytest.fixture(scope="module")
def entry(tmp_path_factory):
    folder = tmp_path_factory.mktemp("entry")
    exe, obj = str(folder / "entry_check"), str(folder / "entry_check.o")
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    subprocess.run([hipcc, "-x", "hip", "--offload-arch=gfx950", "--offload-host-only", "-O0", "-std=c++17", "-I" + os.path.join(REPO, "include"),
                    "-c", os.path.join(REPO, "tests", "entry_check.cc"), "-o", obj], check=True, capture_output=True)
    # (there is no code for a device to be found)
    subprocess.run(["g++", "-no-pie", obj, "-Wl,--unresolved-symbols=ignore-all", "-o", exe], check=True)
    return exe


@pytest.mark.parametrize("shape", [(0, 10, 10), (2, 0, 10), (2, 10, 0)])
def test_empty_gradient_with_working_memory(capi, entry, shape):
    """A gradient of nothing has no strides to be looked at."""
    done = subprocess.run([entry] + [str(x) for x in shape], capture_output=True, text=True)
    assert done.returncode == 0 and done.stdout.split() == [str(capi.EHIP)], done
