"""Direct-to-LDS loads whose waits are counted in the source, checked in the code that the compiler made of it (no GPU).

The 4-bit tile kernels keep the rows of several stages in flight and release a stage's rows to the other waves by one
barrier. A wave may pass the barrier of stage s only when its own loads of that stage have landed: of the loads to LDS at
most those of the NST - 2 stages after it, the latest that it issued, may be outstanding."""

from __future__ import annotations

import re
import shutil
import subprocess
from pathlib import Path

import pytest

TILE = re.compile(r"fp4_tile_kernelILb([01])ELi(\d+)ELi(\d+)ELi(\d+)ELi(\d+)ELb([01])E")
LINE = re.compile(r"\s+([a-z]\w+)\s*(.*?)\s*// ([0-9A-F]+):(.*)")


@pytest.fixture(scope="module")
def listing(pkg, tmp_path_factory):
    return _listing(pkg, tmp_path_factory.mktemp("code"))


def _listing(pkg, folder) -> dict[str, list[tuple[int, str, str, int | None]]]:
    """The kernels of the built library: (address, instruction, operands, branch target) in order."""
    objdump = shutil.which("llvm-objdump") or "/opt/rocm/lib/llvm/bin/llvm-objdump"
    if not Path(objdump).exists():
        pytest.skip("needs llvm-objdump")
    shutil.copy(pkg.LIB_PATH, folder / "lib.so")
    subprocess.run([objdump, "--offloading", "lib.so"], cwd=folder, check=True, capture_output=True)
    kernels = {}
    for obj in sorted(folder.glob("*gfx950")):
        text = subprocess.run([objdump, "-d", "--no-show-raw-insn", obj.name], cwd=folder, check=True, capture_output=True,
                              text=True).stdout
        for part in re.split(r"\n(?=[0-9a-f]+ <)", text)[1:]:
            start, name = re.match(r"([0-9a-f]+) <(\w+)>:", part).groups()
            code = []
            for m in filter(None, map(LINE.match, part.splitlines())):
                to = re.search(r"<\w+?\+0x([0-9a-f]+)>", m[4])
                code.append((int(m[3], 16), m[1], m[2], int(start, 16) + int(to[1], 16) if to else None))
            kernels[name] = code
    return kernels


def _most_at_a_barrier(code) -> int:
    """The most loads to LDS that may be outstanding at a barrier, over every way through the code. Loads return in order,
    so what is outstanding are the latest ones: a string of "L" (to LDS) and "R" (to registers), newest last."""
    at = {address: i for i, (address, *_) in enumerate(code)}
    most, seen, todo = 0, set(), [(0, "")]
    while todo:
        i, flying = todo.pop()
        while i < len(code):
            _, op, args, target = code[i]
            if op == "s_endpgm":
                break
            if op.startswith(("buffer_load", "global_load")):
                flying = (flying + ("L" if re.search(r"\blds\b", args) or "_lds_" in op else "R"))[-64:]
            elif op.startswith(("buffer_store", "global_store")):
                flying = (flying + "R")[-64:]
            elif op == "s_waitcnt" and (m := re.search(r"vmcnt\((\d+)\)", args)):
                flying = flying[len(flying) - min(len(flying), int(m[1])):]
            elif op == "s_barrier":
                most = max(most, flying.count("L"))
            if op == "s_branch" or op.startswith("s_cbranch"):
                if (target, flying) not in seen:
                    seen.add((target, flying))
                    todo.append((at[target], flying))
                if op == "s_branch":
                    break
            i += 1
    return most


def test_the_walk_counts_loads():
    code = [(0, "buffer_load_dwordx4", "v1, s[0:3], 0 offen lds", None), (1, "buffer_load_dword", "v2, off", None),
            (2, "s_waitcnt", "vmcnt(2) lgkmcnt(0)", None), (3, "s_barrier", "", None), (4, "s_cbranch_scc1", "", 0),
            (5, "s_waitcnt", "vmcnt(1)", None), (6, "s_barrier", "", None), (7, "s_endpgm", "", None)]
    assert _most_at_a_barrier(code) == 1
    assert _most_at_a_barrier(code[5:]) == 0
    code[2] = (2, "s_waitcnt", "vmcnt(4)", None)
    assert _most_at_a_barrier(code) == 2


def test_a_stages_rows_have_landed_at_its_barrier(listing):
    tiles = 0
    for name, code in listing.items():
        if not (m := TILE.search(name)):
            continue
        rows8, bm, _, _, slots, _ = map(int, m.groups())
        loads = bm // (4 * (8 if rows8 else 4)) + (rows8 and -(-bm // 256))  # a wave's of a stage: rows, and their scales
        assert sum(op.startswith("buffer_load") and " lds" in args for _, op, args, _ in code) >= loads * 4
        assert _most_at_a_barrier(code) <= (slots - 2) * loads, name
        tiles += 1
    assert tiles == 12


def _loads_right_after_m0(code) -> list[int]:
    """Loads to LDS with no instruction between them and the scalar one that wrote M0, where their address is: they need
    one wait state there."""
    return [b[0] for a, b in zip(code, code[1:])
            if re.match(r"s_\w+", a[1]) and re.match(r"m0\b", a[2]) and b[1].startswith(("buffer_load", "global_load"))
            and (re.search(r"\blds\b", b[2]) or "_lds_" in b[1])]


def test_the_address_of_a_load_to_lds_is_there_before_it(listing):
    early = [(0, "s_add_u32", "m0, s1, 0x400", None), (4, "buffer_load_dword", "v1, s[0:3], 0 offen lds", None)]
    assert _loads_right_after_m0(early) == [4]
    assert not _loads_right_after_m0([early[0], (2, "s_nop", "0", None), early[1]])
    found = {name: _loads_right_after_m0(code) for name, code in listing.items()}
    assert not {name: len(at) for name, at in found.items() if at}
