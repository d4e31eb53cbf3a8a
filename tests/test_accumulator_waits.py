"""The products of csrc/mfma_tile.h stand in inline assembly, so the compiler
does not know how long their results take. This looks at the code that was
built: no other instruction touches an accumulator within the 11 wait states
that v_mfma_f32_16x16x32 needs, on any path, and no vector instruction writes
an operand or the accumulator of one within the 4 before it (2 are asked for)."""

import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SO = os.path.join(ROOT, "distributed_vgg_f_amd", "_hipops.so")
OBJDUMP = shutil.which("llvm-objdump") or "/opt/rocm/llvm/bin/llvm-objdump"
RESULT, OPERAND = 11, 4


def registers(text, bank):
    found = set()
    for m in re.finditer(r"\b%s\[(\d+):(\d+)\]" % bank, text):
        found |= set(range(int(m.group(1)), int(m.group(2)) + 1))
    return found | {int(m.group(1))
                    for m in re.finditer(r"\b%s(\d+)\b" % bank, text)}


def states(text):
    return int(text.split()[1], 0) + 1 if text.startswith("s_nop") else 1


def too_early(code):
    """code: (address, text, address of the branch's target or None)."""
    where = {a: i for i, (a, _, _) in enumerate(code)}
    bad = []
    for i, (_, text, _) in enumerate(code):
        if not text.startswith("v_mfma"):
            continue
        dst = registers(text.split(",")[0], "a")
        src = registers(",".join(text.split(",")[1:3]), "v")
        gap = 0
        for _, before, _ in reversed(code[max(0, i - OPERAND):i]):
            if gap >= OPERAND:
                break
            if before.startswith("v_") and not before.startswith("v_mfma"):
                to = before.split(",")[0]
                if registers(to, "v") & src or registers(to, "a") & dst:
                    bad.append((before, text))
            gap += states(before)
        paths, seen = [(i + 1, 0)], set()
        while paths:
            j, w = paths.pop()
            while j < len(code) and w < RESULT and (j, w) not in seen:
                seen.add((j, w))
                _, t, target = code[j]
                if not t.startswith("v_mfma") and registers(t, "a") & dst:
                    bad.append((text, t))
                    break
                w += states(t)
                if t.startswith("s_endpgm"):
                    break
                if t.startswith("s_branch"):
                    j = where[target]
                    continue
                if t.startswith("s_cbranch"):
                    paths.append((where[target], w))
                j += 1
    return bad


def test_the_scan_sees_planted_mistakes():
    mfma = "v_mfma_f32_16x16x32_bf16 a[0:3], v[0:3], v[4:7], a[0:3]"
    read = "v_accvgpr_read_b32 v9, a2"
    far = [(8 * i, t, None) for i, t in enumerate([mfma, "s_nop 10", read])]
    near = [(8 * i, t, None) for i, t in enumerate([mfma, "s_nop 9", read])]
    assert not too_early(far)
    assert too_early(near) == [(mfma, read)]
    jump = [(0, mfma, None), (8, "s_cbranch_scc0 1", 24),
            (16, "s_nop 15", None), (24, read, None)]
    assert too_early(jump) == [(mfma, read)]
    write = "v_mov_b32_e32 v5, v9"
    assert too_early([(0, write, None), (8, mfma, None)]) == [(write, mfma)]
    assert not too_early([(0, write, None), (8, "s_nop 3", None),
                          (16, mfma, None)])
    zero = "v_accvgpr_write_b32 a1, 0"
    assert too_early([(0, zero, None), (8, mfma, None)]) == [(zero, mfma)]


@pytest.mark.skipif(not (os.path.exists(SO) and os.path.exists(OBJDUMP)),
                    reason="needs the built extension and llvm-objdump")
def test_built_products_wait(tmp_path):
    shutil.copy(SO, tmp_path / "x.so")
    subprocess.run([OBJDUMP, "--offloading", "x.so"], cwd=tmp_path,
                   check=True, capture_output=True)
    kernels = {}
    for part in tmp_path.glob("x.so.*gfx950"):
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", part],
                              check=True, capture_output=True,
                              text=True).stdout
        code = start = None
        for line in text.splitlines():
            head = re.match(r"^([0-9a-f]+) <(\S+)>:", line)
            if head:
                start = int(head.group(1), 16)
                code = kernels.setdefault(head.group(2), []) \
                    if "product_kernel" in head.group(2) else None
            elif code is not None and "//" in line:
                t, note = line.strip().split("//")
                at = int(note.strip().split(":")[0].split()[0], 16)
                hit = re.search(r"<\S+\+0x([0-9a-f]+)>", note)
                code.append((at, t.strip(),
                             start + int(hit.group(1), 16) if hit else None))
    assert len(kernels) >= 6
    for name, code in kernels.items():
        assert sum(t.startswith("v_mfma") for _, t, _ in code) >= 16, name
        assert too_early(code) == [], name
