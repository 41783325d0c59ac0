"""The scans of test_matrix_result_hazards_cpu.py and test_inline_asm_hazards_cpu.py over all kernels that have such instructions, with the
wait states that the compiler itself puts between a matrix instruction and a vector instruction that reads its result."""
import os
import re
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

import test_inline_asm_hazards_cpu as inline_asm
import test_matrix_result_hazards_cpu as results

CSRC = results.CSRC
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "--cuda-device-only", "-S"]
KERNELS = sorted(f for f in os.listdir(CSRC) if f.endswith("_kernel.hip") or f.endswith("_kernels.hip"))
NEED = {"v_mfma_f32_16x16x32_bf16": 8, "v_mfma_f32_16x16x32_f16": 8, "v_mfma_f32_32x32x16_bf16": 12, "v_mfma_f32_32x32x16_f16": 12,
        "v_mfma_f32_16x16x4_f32": 10}


def assemble(source, dst):
    subprocess.run(["hipcc", *FLAGS, source, "-o", dst], check=True, stdout=subprocess.PIPE, stderr=subprocess.PIPE)
    return dst


@pytest.fixture(scope="module")
def assembly(tmp_path_factory):
    if shutil.which("hipcc") is None:
        pytest.skip("hipcc not found")
    out = tmp_path_factory.mktemp("all")
    with ThreadPoolExecutor(8) as ex:
        return dict(zip(KERNELS, ex.map(lambda k: assemble(os.path.join(CSRC, k), str(out / (k + ".s"))), KERNELS)))


def test_the_compiler_waits_as_long(tmp_path):
    """A product whose result the next instruction reads, of each kind: what the compiler puts between is what the scan asks for."""
    if shutil.which("hipcc") is None:
        pytest.skip("hipcc not found")
    lines = ["#include <hip/hip_runtime.h>", "typedef float c4 __attribute__((ext_vector_type(4)));",
             "typedef float c16 __attribute__((ext_vector_type(16)));", "typedef __bf16 bf16 __attribute__((ext_vector_type(8)));",
             "typedef _Float16 f16 __attribute__((ext_vector_type(8)));", "typedef float f32;"]
    for op in NEED:
        shape, kind = re.fullmatch(r"v_mfma_f32_(\d+x\d+x\d+)_(\w+)", op).groups()
        c = "c16" if shape.startswith("32") else "c4"
        builtin = f"__builtin_amdgcn_mfma_f32_{shape}{'' if kind == 'f32' else '_'}{kind}"
        lines.append(f"__global__ void k_{shape}_{kind}(const {kind}* a, const {kind}* b, {c}* o) {{ const int i = threadIdx.x; "
                     f"o[i] = {builtin}(a[i], b[i], o[i + 64], 0, 0, 0) * 2.f; }}")
    source = tmp_path / "waits.hip"
    source.write_text("\n".join(lines) + "\n")
    text = open(assemble(str(source), str(tmp_path / "waits.s"))).read()
    for op, need in NEED.items():
        m = re.search(rf"^\t{op} .*\n((?:\ts_nop \d+\n)*)\tv_", text, re.M)
        assert m and sum(int(n) + 1 for n in re.findall(r"s_nop (\d+)", m.group(1))) == need, op


def test_matrix_results_are_read_late_enough(assembly):
    kinds, found = set(), 0
    for name, path in assembly.items():
        products = set(re.findall(r"^\t(v_s?mfma\w+)", open(path).read(), re.M))
        assert products <= set(NEED), f"{name}: no wait states known for {products - set(NEED)}"
        kinds |= products
        sites, bad = results.scan(path, NEED)
        found += sites
        assert not bad, f"{name}: {len(bad)} reads too early, e.g. {bad[:3]}"
    assert kinds == set(NEED) and found > 5000


def test_tile_loads_keep_their_wait_states(assembly):
    found = {}
    for name, path in assembly.items():
        found[name], bad = inline_asm.scan(path)
        assert not bad, f"{name}: {len(bad)} tile loads too close to a vector-ALU scalar write, e.g. {bad[:3]}"
    assert found["paged_kernel.hip"] > 20 and sum(found.values()) > 1000, found
