"""The assembly of the paged attention's kernels (device pass only, no GPU needed): what its sources take for granted."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "moda_amd", "csrc")


@pytest.fixture(scope="module")
def paged_assembly(tmp_path_factory):
    if shutil.which("hipcc") is None:
        pytest.skip("hipcc not found")
    dst = str(tmp_path_factory.mktemp("asm") / "paged.s")
    subprocess.run(["hipcc", "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
                    "--cuda-device-only", "-S", os.path.join(CSRC, "paged_kernel.hip"), "-o", dst], check=True, stdout=subprocess.PIPE, stderr=subprocess.PIPE)
    return dst


def calls(text):
    return re.findall(r"^\s*(s_swappc_b64|s_setpc_b64|s_call_b64)\b.*$", text, re.M)


def test_calls_are_seen():
    assert calls("\ts_getpc_b64 s[2:3]\n\ts_swappc_b64 s[30:31], s[4:5]\n\ts_setpc_b64 s[30:31]\n") and not calls("\ts_getpc_b64 s[2:3]\n\ts_branch .LBB0_1\n")


def test_kernels_call_no_function(paged_assembly):
    """They read their arguments again from the kernel's argument segment (paged_kernel.hip: reload), whose address is zero in a function that
    is called and not inlined: a second use of a member function is enough for the compiler to make it one."""
    text = open(paged_assembly).read()
    assert text.count(".amdhsa_kernel") >= 10
    assert not calls(text)
