"""A matrix instruction's result may be read by anything but another matrix instruction only some wait states later (the
hardware does not wait), and the compiler's hazard pass has been seen to leave them out where the first reader comes behind a
branch: a skipped branch that led straight from the last product to the read of its fourth register, which then held an
earlier sum.  This test compiles the paged attention's kernels to assembly (device pass only, no GPU needed) and follows every way on
from every matrix instruction, through branches and around loops.
"""
import os
import re
import shutil
import subprocess
import tempfile

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "moda_amd", "csrc")
# wait states between the instruction and a vector instruction that reads its result: four passes of four cycles, and eight
NEED = {"v_mfma_f32_16x16x32_bf16": 7, "v_mfma_f32_16x16x32_f16": 7, "v_mfma_f32_16x16x4_f32": 10}


def registers(text):
    out = set()
    for kind, a, b in re.findall(r"\b([va])\[(\d+):(\d+)\]", text):
        out |= {(kind, i) for i in range(int(a), int(b) + 1)}
    for kind, a in re.findall(r"\b([va])(\d+)\b", text):
        out.add((kind, int(a)))
    return out


def parse(path):
    """[(text, label targets)] of each kernel: a list of instructions and where its labels are."""
    kernels, code, labels = [], None, None
    for raw in open(path):
        line = raw.split(";")[0].rstrip()
        if re.match(r"^_ZN\S+:", line):
            code, labels = [], {}
            kernels.append((code, labels))
            continue
        if code is None or not line.strip():
            continue
        m = re.match(r"^(\.L\w+):", line)
        if m:
            labels[m.group(1)] = len(code)
        elif line.startswith("\t") and not line.strip().startswith("."):
            code.append(line.strip())
    return [k for k in kernels if k[0]]


def reads(ins):
    """Registers an instruction reads: all operands behind its destination (stores and LDS writes: all)."""
    op, _, rest = ins.partition(" ")
    if re.match(r"(global_store|buffer_store|scratch_store|ds_write|ds_bpermute|flat_store|global_load|buffer_load)", op):
        return registers(rest)
    first, _, others = rest.partition(",")
    return registers(others) | (registers(first) if "swap" in op else set())


def scan(path, need=NEED):
    sites, bad = 0, []
    for code, labels in parse(path):
        for at, ins in enumerate(code):
            op = ins.split()[0]
            if op not in need:
                continue
            sites += 1
            result = registers(ins.split(",")[0])
            seen, ways = {}, [(at + 1, 0, frozenset(result))]
            while ways:
                pc, waited, live = ways.pop()
                while pc < len(code) and waited < need[op] and live:
                    if seen.get((pc, live), 99) <= waited:
                        break
                    seen[(pc, live)] = waited
                    cur = code[pc]
                    name = cur.split()[0]
                    if name.startswith("v_mfma"):
                        live = live - registers(cur.split(",")[0])  # a later product's result now
                    else:
                        if reads(cur) & live:
                            bad.append((ins, cur, waited))
                            break
                        if name.startswith("v_") and not name.startswith("v_cmp"):
                            live = live - registers(cur.partition(" ")[2].split(",")[0])
                    m = re.match(r"s_nop (\d+)", cur)
                    waited += int(m.group(1)) + 1 if m else 1
                    target = re.match(r"(s_c?branch\S*)\s+(\.L\w+)", cur)
                    if target and target.group(2) in labels:
                        ways.append((labels[target.group(2)], waited, live))
                        if target.group(1) == "s_branch":
                            break
                    if name in ("s_endpgm", "s_setpc_b64"):
                        break
                    pc += 1
    return sites, bad


def _scan_text(text):
    with tempfile.NamedTemporaryFile("w", suffix=".s", delete=False) as f:
        f.write(text)
    try:
        return scan(f.name)
    finally:
        os.unlink(f.name)


def test_scanner_follows_branches():
    head = "_ZN1kE:\n\tv_mfma_f32_16x16x4_f32 a[0:3], v1, v2, a[0:3]\n\ts_cbranch_execz .LBB0_1\n"
    long_way = "".join("\ts_nop 7\n" for _ in range(2))
    sites, bad = _scan_text(head + long_way + ".LBB0_1:\n\tv_accvgpr_read_b32 v5, a3\n\ts_endpgm\n")
    assert sites == 1 and len(bad) == 1 and bad[0][2] == 1
    sites, bad = _scan_text(head + "\ts_nop 7\n\ts_nop 1\n\tv_accvgpr_read_b32 v5, a3\n.LBB0_1:\n\ts_nop 7\n\ts_nop 1\n\tv_mul_f32 v1, v2, v3\n"
                            "\tv_accvgpr_read_b32 v5, a3\n\ts_endpgm\n")
    assert sites == 1 and not bad
    sites, bad = _scan_text(".text\n_ZN1kE:\n.LBB0_0:\n\tv_mul_f32 v9, v4, v4\n\tv_mfma_f32_16x16x32_bf16 v[4:7], v[0:3], v[0:3], 0\n\ts_branch .LBB0_0\n")
    assert sites == 1 and len(bad) == 1


def test_matrix_results_are_read_late_enough(tmp_path):
    if shutil.which("hipcc") is None:
        pytest.skip("hipcc not found")
    dst = str(tmp_path / "paged.s")
    subprocess.run(["hipcc", "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
                    "--cuda-device-only", "-S", os.path.join(CSRC, "paged_kernel.hip"), "-o", dst], check=True, stdout=subprocess.PIPE, stderr=subprocess.PIPE)
    sites, bad = scan(dst)
    assert not bad, f"{len(bad)} reads too early, e.g. {bad[:3]}"
    assert sites > 300
