"""The waits round inline asm in the compiled kernels that need them, on the CPU.

The compiler keeps wait states between an instruction that writes a vector register
and an MFMA, DPP or lane instruction that reads it (two), and between v_exp, v_rcp and
the like and what reads their result (one), but not where one of the two is inline
asm.  The sources whose asm results reach such readers are compiled to assembly with
the build's flags, and each reader's operands are looked for among the asm
instructions less than that far before it."""
import re
import shutil
import subprocess

import pytest

import build as B

TRANS = re.compile(r"v_(exp|log|rcp|rsq|sqrt|sin|cos)_")
LANES = ("v_permlane", "v_readlane", "v_readfirstlane", "v_writelane")
DPP = ("quad_perm:", "row_", "bank_mask:")


def _regs(text):
    out = set()
    for one, n, many, lo, hi in re.findall(r"\b(?:([va])(\d+)\b|([va])\[(\d+):(\d+)\])", text):
        out |= {one + n} if one else {f"{many}{i}" for i in range(int(lo), int(hi) + 1)}
    return out


def short_waits(lines):
    """(line number, reader, writer, wait states between them) of each that is short."""
    found, before, in_asm = [], [], False
    for number, line in enumerate(lines, 1):
        text = line.strip()
        if text.startswith(";;#ASM"):
            in_asm = text.startswith(";;#ASMSTART")
            continue
        text = text.split(";")[0].strip()
        if not text or text[0] == "." or text.endswith(":"):
            continue
        name, _, rest = text.partition(" ")
        if name == "s_nop":
            before.append((name, set(), int(rest, 0) + 1, False))
            continue
        vector, swap, ops = name.startswith("v_"), "swap" in name, rest.split(",")
        dst = _regs(",".join(ops[:1 + swap])) if vector else set()
        src = _regs(",".join(ops[0 if swap or "fmac" in name or "dot2c" in name else 1:]))
        reader = name.startswith("v_mfma") or name.startswith(LANES) or any(
            k in rest for k in DPP)
        kinds = []
        if reader:
            kinds.append((2, lambda w, asm: asm or (in_asm and w.startswith("v_"))))
        if in_asm and vector:
            kinds.append((1, lambda w, asm: TRANS.match(w)))
        for need, bad in kinds:
            states, left = 0, set(src)
            for writer, written, length, asm in reversed(before[-8:]):
                if states >= need:
                    break
                if left & written and bad(writer, asm):
                    found.append((number, text, writer, states))
                left -= written
                states += length
        before.append((name, dst, 1, in_asm and vector))
    return found


def test_the_scan_sees_each_kind():
    asm = lambda *body: ["\t;;#ASMSTART", *body, "\t;;#ASMEND"]
    cvt = "\tv_cvt_pk_bf16_f32 v5, v1, v2"
    mfma = "\tv_mfma_f32_16x16x32_bf16 v[8:11], v[12:15], v[4:7], v[8:11]"
    dpp = "\tv_mov_b32_dpp v9, v5 row_ror:8 row_mask:0xf bank_mask:0xf"
    assert len(short_waits([*asm(cvt), mfma])) == 1
    assert len(short_waits([*asm(cvt), "\ts_nop 0", mfma])) == 1
    assert len(short_waits([*asm(cvt), "\ts_waitcnt lgkmcnt(0)", dpp])) == 1
    assert len(short_waits(["\tv_exp_f32_e32 v1, v3", *asm(cvt)])) == 1
    assert not short_waits([*asm(cvt), "\ts_nop 1", mfma])
    assert not short_waits([cvt, mfma])  # not asm: the compiler's own waits
    assert not short_waits([*asm(cvt), "\tv_mov_b32_e32 v5, v0", mfma])
    assert not short_waits(["\tv_exp_f32_e32 v1, v3", "\ts_nop 0", *asm(cvt)])


@pytest.mark.parametrize("source", ["dip_kv4", "dip_kv4_attn", "dip_kv4_prompt", "dip_gemm"])
def test_asm_results_wait_for_their_readers(source, tmp_path):
    if shutil.which(B.HIPCC) is None:
        pytest.skip("hipcc not available")
    out = tmp_path / "kernels.s"
    subprocess.run([B.HIPCC, *B.COMMON, *B.EXTRA.get(source, []), "--cuda-device-only", "-S",
                    str(B.CSRC / f"{source}.hip"), "-o", str(out)],
                   check=True, capture_output=True, text=True, timeout=600)
    lines = out.read_text().splitlines()
    assert any("v_mfma" in l for l in lines) or source == "dip_kv4"
    assert not short_waits(lines)
