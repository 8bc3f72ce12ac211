"""Compile-time check of the attention's listing for gfx950 (needs hipcc, no
GPU): no instruction reads or writes an MFMA's result registers before the
MFMA is done with them. The hardware does not hold such an instruction back:
the compiler counts the issue slots in between and fills them with s_nop, and
has been seen to count one way into a block only where a branch follows the
MFMA (scores then differed from run to run)."""

from __future__ import annotations

import re
import shutil
from pathlib import Path

import pytest

from jeeves_amd import build
from tests.test_kernel_resources import FUNCTION_LABEL, compile_device

# Issue slots until a result may be read: passes of four cycles, and four more.
SLOTS = {"16x16": 8, "32x32": 12}
REGISTERS = re.compile(r"\b([va])(?:\[(\d+):(\d+)\]|(\d+)\b)")


def registers(operand: str) -> set[tuple[str, int]]:
    out = set()
    for kind, first, last, one in REGISTERS.findall(operand):
        out |= {(kind, i) for i in (range(int(first), int(last) + 1) if first else (int(one),))}
    return out


def operands(args: str) -> list[str]:
    return [p.strip() for p in re.split(r",(?![^\[]*\])", args)]


def functions(asm: str) -> dict[str, list[tuple[str, str]]]:
    """Per function its instructions as (operation, operands), labels as ("label", name)."""
    found: dict[str, list[tuple[str, str]]] = {}
    body = None
    for line in asm.splitlines():
        text = line.split(";")[0].strip()
        if m := FUNCTION_LABEL.match(text):
            if not m.group(1).startswith(".L"):
                body = found.setdefault(m.group(1), [])
        elif text.startswith(".section") or text.startswith(".end_amdhsa"):
            body = None
        if body is None or not text:
            continue
        if m := re.match(r"^(\.L\w+):", text):
            body.append(("label", m.group(1)))
        elif not text.startswith(".") and not text.endswith(":"):
            op, _, args = text.partition(" ") if " " in text else text.partition("\t")
            body.append((op, args.strip()))
    return found


def early_uses(asm: str) -> list[tuple[str, str, str]]:
    """(function, MFMA, instruction) where, on some path, the instruction meets
    the MFMA's result too soon. A later MFMA that adds to the same registers,
    or overwrites them, waits by itself and ends the search there; any other
    counts for the slots of its own passes."""
    bad = []
    for fn, body in functions(asm).items():
        at = {name: i for i, (op, name) in enumerate(body) if op == "label"}
        for i, (op, args) in enumerate(body):
            if not op.startswith("v_mfma"):
                continue
            result = registers(operands(args)[0])
            slots = next((n for shape, n in SLOTS.items() if shape in op), max(SLOTS.values()))
            reached: dict[int, int] = {}
            paths = [(i + 1, 0)]
            while paths:
                k, waited = paths.pop()
                if k >= len(body) or waited >= slots or reached.get(k, slots) <= waited:
                    continue
                reached[k] = waited
                o, a = body[k]
                if o == "label":
                    paths.append((k + 1, waited))
                elif o == "s_branch":
                    paths.append((at[a], waited + 1))
                elif o.startswith("s_cbranch"):
                    paths += [(at[a], waited + 1), (k + 1, waited + 1)]
                elif o == "s_nop":
                    paths.append((k + 1, waited + 1 + int(a, 0)))
                elif o.startswith("v_mfma"):
                    to, *sources = operands(a)
                    if (registers(sources[0]) | registers(sources[1])) & result:
                        bad.append((fn, f"{op} {args}", f"{o} {a}"))
                    elif registers(to) != result:
                        paths.append((k + 1, waited + (8 if "32x32" in o else 4)))
                elif re.match(r"(v|ds|global|buffer|flat)_", o) and registers(a) & result:
                    bad.append((fn, f"{op} {args}", f"{o} {a}"))
                elif o != "s_endpgm":
                    paths.append((k + 1, waited + 1))
    return bad


@pytest.mark.skipif(shutil.which("hipcc") is None and not Path("/opt/rocm/bin/hipcc").exists(), reason="needs hipcc")
def test_attention_waits_for_its_products(tmp_path):
    _, asm = compile_device(build.CSRC / "attention.hip", tmp_path)
    assert len(re.findall(r"^\s*v_mfma", asm, re.M)) > 500
    assert len(functions(asm)) > 10
    assert not early_uses(asm)


def test_scan_follows_the_branch_taken():
    listing = """kern:
\tv_mfma_f32_16x16x32_bf16 v[26:29], v[68:71], v[6:9], v[72:75]
\ts_cbranch_scc1 .LBB0_2
\tv_add_u32_e32 v67, s44, v43
\ts_nop 7
\tv_cndmask_b32_e32 v26, v53, v26, vcc
.LBB0_2:
\tv_max_f32_e32 v67, v29, v29
\ts_endpgm
"""
    assert [(fn, use) for fn, _, use in early_uses(listing)] == [("kern", "v_max_f32_e32 v67, v29, v29")]
    assert not early_uses(listing.replace("\ts_cbranch", "\ts_nop 7\n\ts_cbranch"))


def test_scan_counts_slots():
    listing = """kern:
\tv_mfma_f32_32x32x16_f16 v[0:15], v[16:19], v[20:23], v[0:15]
\ts_nop 9
\tv_exp_f32_e32 v30, v15
\ts_endpgm
"""
    assert len(early_uses(listing)) == 1
    assert not early_uses(listing.replace("s_nop 9", "s_nop 11"))
    # its own accumulation goes on at once, another product may not read it
    chained = listing.replace("s_nop 9", "v_mfma_f32_32x32x16_f16 v[0:15], v[24:27], v[20:23], v[0:15]\n\ts_nop 11")
    assert not early_uses(chained)
    assert early_uses(listing.replace("s_nop 9", "v_mfma_f32_32x32x16_f16 v[32:47], v[0:3], v[20:23], v[32:47]"))
