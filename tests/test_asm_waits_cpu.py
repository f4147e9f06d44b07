"""Inline assembly and the results of matrix products, in the assembly that hipcc makes of the kernels.

A product's result is in its registers only some wait states after the instruction was issued (12 for 32x32x16, 8 for
16x16x32), and its third operand is read for about as long. The compiler keeps its own instructions away from both for that
long but does not look into inline assembly. So, over all paths of each kernel: an inline vector instruction neither reads nor
writes a register of a product before that."""

import concurrent.futures as cf
import pathlib
import re
import shutil
import subprocess
import sys

import pytest

PKG = pathlib.Path(__file__).resolve().parent.parent / "iree-adreno-genai-tuner_amd"
sys.path.insert(0, str(PKG))
import build  # noqa: E402

SOURCES = ["paged_attn", "attn_bucket", "q4_rows", "q4_linear", "q4_gemv_mx", "gemm_f16"]  # those with products
CAP = 24  # distances from here on are not told apart


def regs(operand):
    m = re.fullmatch(r"[-|]*([va])(?:(\d+)|\[(\d+):(\d+)\])\|?", operand.strip())
    if not m:
        return ()
    lo, hi = (m[2], m[2]) if m[2] else (m[3], m[4])
    return [(m[1], r) for r in range(int(lo), int(hi) + 1)]


def functions(text):
    """{name: [(label,) or (op, operands, inline)]}"""
    out, cur, inline = {}, None, False
    for line in text.splitlines():
        if "#ASMSTART" in line or "#ASMEND" in line:
            inline = "#ASMSTART" in line
            continue
        t = line.split(";")[0].strip()
        if m := re.fullmatch(r"(_Z\w+):", t):
            cur = out.setdefault(m[1], [])
        elif t.startswith(".section"):
            cur = None
        elif cur is None or not t:
            continue
        elif t.startswith(".LBB"):
            cur.append((t[:-1],))
        elif not t.startswith("."):
            op, _, rest = t.partition(" ")
            cur.append((op, re.split(r",\s*(?![^\[]*\])", rest.strip()) if rest else [], inline))
    return out


def least_states(ins):
    """{(op, product, what): wait states} of the inline vector instructions that touch a product's registers: a forward pass to
    a fixed point over each register's least distance from a product that writes it ('result') or adds it ('addend')."""
    at = {i[0]: k for k, i in enumerate(ins) if len(i) == 1}
    seen, found = {}, {}

    def merged(k, state):
        """The state at k with this one taken in; None: nothing new."""
        old = seen.get(k)
        if old is None:
            seen[k] = dict(state)
            return seen[k]
        new = {r: v for r, v in state.items() if r not in old or old[r][0] > v[0]}
        old.update(new)
        return old if new else None

    work = [(0, {})]
    while work:
        k, state = work.pop()
        while k < len(ins):
            if len(ins[k]) == 1:
                state = merged(k, state)
                if state is None:
                    break
                state, k = dict(state), k + 1
                continue
            op, ops, inline = ins[k]
            if op.startswith("v_mfma"):
                state = {r: (n + 1, p) for r, (n, p) in state.items() if n + 1 < CAP}
                state.update({("addend", r): (0, op) for r in regs(ops[3])})
                state.update({("result", r): (0, op) for r in regs(ops[0])})
            else:
                vector = op.startswith("v_")
                writes = [r for o in (ops[:2] if "swap" in op else ops[:1]) for r in regs(o)] if vector and "cmp" not in op else \
                    [r for r in regs(ops[0])] if re.match(r"(ds_read|global_load|buffer_load)", op) and ops else []
                if inline and vector:
                    for what, rs in (("result", [r for o in ops for r in regs(o)]), ("addend", writes)):
                        for r in rs:
                            if (what, r) in state:
                                n, p = state[what, r]
                                key = (op, p, what)
                                found[key] = min(found.get(key, CAP), n)
                step = 1 + (int(ops[0], 0) if op == "s_nop" else 0)
                state = {r: (n + step, p) for r, (n, p) in state.items() if n + step < CAP}
                for r in writes:
                    state.pop(("result", r), None)
                    state.pop(("addend", r), None)
            k += 1
            if op.startswith("s_cbranch") or op == "s_branch":
                work.append((at[ops[0]], dict(state)))
            if op in ("s_branch", "s_endpgm", "s_setpc_b64"):
                break
    return found


def short(found):
    return {k: n for k, n in found.items() if n < (12 if "32x32" in k[1] else 8)}


def test_the_scan_finds_a_read_that_comes_too_soon():
    """On a listing of its own: a read at once, behind a branch, and behind enough wait states."""
    mfma = "v_mfma_f32_32x32x16_f16 v[2:17], v[20:23], v[24:27], v[2:17]\n"
    asm = "\t;;#ASMSTART\n\tv_max3_f32 v1, v2, v3, v4\n\t;;#ASMEND\n"
    scan = lambda body: short(least_states(functions("_Zk:\n" + body + "\ts_endpgm\n")["_Zk"]))  # noqa: E731
    assert scan(mfma + asm) and scan(mfma + "\ts_cbranch_vccnz .LBB0_1\n\ts_nop 15\n.LBB0_1:\n" + asm)
    assert scan(".LBB0_1:\n" + asm + mfma + "\ts_branch .LBB0_1\n")
    assert not scan(mfma + "\ts_nop 11\n" + asm) and not scan(mfma + "\ts_nop 7\n\ts_nop 3\n" + asm)
    assert not scan(mfma + "\tv_mov_b32_e32 v2, 0\n\tv_mov_b32_e32 v3, 0\n\tv_mov_b32_e32 v4, 0\n" + asm)
    assert scan("v_mfma_f32_32x32x16_f16 v[2:17], v[20:23], v[24:27], v[30:45]\n" + asm.replace("v1, v2, v3, v4", "v30, v50, v51, v52"))


@pytest.mark.skipif(not shutil.which(build.HIPCC), reason="needs hipcc")
def test_inline_assembly_waits_for_products(tmp_path):
    def compiled(name):
        out = tmp_path / f"{name}.s"
        subprocess.run([build.HIPCC, *build.COMMON, "--cuda-device-only", "-S", str(build.CSRC / f"{name}.hip"), "-o", str(out)],
                       check=True, capture_output=True)
        return functions(out.read_text())

    bad, kernels = [], 0
    with cf.ThreadPoolExecutor(max_workers=6) as ex:
        for name, fns in zip(SOURCES, ex.map(compiled, SOURCES)):
            for fn, ins in fns.items():
                if any(i[0].startswith("v_mfma") for i in ins):
                    kernels += 1
                    bad += [(name, fn, k, n) for k, n in short(least_states(ins)).items()]
    assert kernels > 6 and not bad
