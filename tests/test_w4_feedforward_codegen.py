"""The 4-wavefront kernel's gated and MXFP4 forms, compiled to assembly: what test_w4_codegen.py asks of its plain forms (nothing
of the compiler's in the accumulation registers, no spills, no parked scalar in front of a load in inline assembly or inside the
steady K loop), and that no vector instruction writes an operand of a matrix instruction in inline assembly right in front of it,
where the compiler, which does not look into assembly, keeps no distance."""
import os
import re
import subprocess

import pytest

from test_w4_codegen import CSRC, HIPCC, too_early

FORMS = {"gated_w4.hip": ("gemm_gated_w4_kernel", "v_mfma_f32_16x16x32", 4), "gemm_mx_w4.hip": ("gemm_mx_w4_kernel", "v_mfma_scale_f32_16x16x128", 6)}


@pytest.fixture(scope="module", params=sorted(FORMS))
def listing(request, tmp_path_factory):
    out = tmp_path_factory.mktemp("w4") / "w4.s"
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Wno-unused-command-line-argument",
                    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "-S", "--cuda-device-only",
                    "-o", str(out), os.path.join(CSRC, request.param)], check=True, capture_output=True, timeout=600)
    return request.param, out.read_text()


def looped(lines):
    """Pieces of the listing: all of it, and once more around every loop."""
    yield lines
    labels = {l.split(":")[0]: i for i, l in enumerate(lines) if re.match(r"^\.LBB\d+_\d+:", l)}
    for i, l in enumerate(lines):
        branch = re.match(r"^\s*s_c?branch\w*\s+(\.LBB\d+_\d+)", l)
        if branch and labels.get(branch[1], i) < i:
            yield lines[max(0, i - 16):i] + lines[labels[branch[1]] + 1:labels[branch[1]] + 17]


def test_compiler_never_touches_the_accumulators(listing):
    source, text = listing
    name, mfma, count = FORMS[source]
    kernels = re.findall(r"^(_ZN4beam\d+%s\w+):" % name, text, flags=re.M)
    assert len(kernels) == count, kernels
    for bad in ("v_accvgpr_write", "v_accvgpr_mov", "scratch_load", "scratch_store"):
        assert bad not in text, f"the compiler emitted {bad} in a 4-wavefront kernel"
    assert set(re.findall(r"\.vgpr_spill_count:\s*(\d+)", text)) == {"0"}
    assert set(re.findall(r"\.private_segment_fixed_size:\s*(\d+)", text)) == {"0"}
    # the steady K loop: the blocks with a whole K tile's MFMAs that are their own successor
    steady = [b for b in re.split(r"^(?=\.LBB\d+_\d+:)", text, flags=re.M)
              if b.count(mfma) >= 128 and re.search(r"s_cbranch_\w+ %s\b" % re.escape(b.split(":")[0]), b)]
    assert len(steady) == count, len(steady)
    for b in steady:
        assert "v_readlane" not in b and "v_writelane" not in b, "a scalar register is reloaded inside the steady K loop"
        # one wait for fills in a K tile, for all but the youngest eight: nothing of the compiler's drains the ring
        assert re.findall(r"vmcnt\((\d+)\)", b) == ["8"], re.findall(r"vmcnt\((\d+)\)", b)


def test_restored_scalars_reach_memory_instructions_late_enough(listing):
    for piece in looped(listing[1].splitlines()):
        bad, _ = too_early(piece)
        assert not bad, bad[:4]


def vectors(operand):
    regs = {int(r) for r in re.findall(r"\bv(\d+)\b", operand)}
    for first, last in re.findall(r"\bv\[(\d+):(\d+)\]", operand):
        regs |= set(range(int(first), int(last) + 1))
    return regs


def written_too_late(lines):
    """Matrix instructions of `lines` that read a vector register fewer than 2 wait states after a vector instruction wrote it."""
    at, written, bad = 0, {}, []
    for line in lines:
        line = line.split(";")[0].strip()
        if not line or line.startswith(".") or line.endswith(":"):
            continue
        op, _, args = line.replace("\t", " ").partition(" ")
        at += int(args, 0) + 1 if op == "s_nop" else 1
        if op.startswith("v_mfma"):
            late = [r for r in vectors(args) if at - written.get(r, -9) - 1 < 2]
            if late:
                bad.append(f"`{line}` reads v{late}")
        elif op.startswith("v_") and not op.startswith(("v_cmp", "v_readlane", "v_readfirstlane")):
            target = args if op.startswith(("v_permlane", "v_swap")) else args.partition(",")[0]
            written.update((r, at) for r in vectors(target))
    return bad


def test_operands_of_matrix_instructions_are_there(listing):
    for piece in looped(listing[1].splitlines()):
        bad = written_too_late(piece)
        assert not bad, bad[:4]


@pytest.mark.parametrize("lines,finds", [
    (["v_mov_b32_e32 v7, v1", "v_mfma_f32_16x16x32_f16 a[0:3], v[4:7], v[8:11], a[0:3]"], 1),
    (["v_mov_b32_e32 v7, v1", "s_nop 1", "v_mfma_f32_16x16x32_f16 a[0:3], v[4:7], v[8:11], a[0:3]"], 0),
    (["v_mov_b32_e32 v7, v1", "s_add_i32 s1, s2, s3", "v_mfma_f32_16x16x32_f16 a[0:3], v[8:11], v[4:7], a[0:3]"], 1),
    (["v_permlane32_swap_b32_e32 v1, v7", "s_nop 0", "v_mfma_f32_16x16x32_f16 a[0:3], v[4:7], v[8:11], a[0:3]"], 1),
    (["v_mov_b32_e32 v12, v7", "v_mfma_f32_16x16x32_f16 a[0:3], v[4:7], v[8:11], a[0:3]"], 0),
])
def test_the_scan_finds_what_it_looks_for(lines, finds):
    assert len(written_too_late(lines)) == finds
