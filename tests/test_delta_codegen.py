"""The wait for loads that write LDS, in the built gfx950 code of the delta rule's chains (CPU; no GPU needed).

Those loads are inline assembly, which the compiler does not wait for.  A wavefront's memory operations complete in order, so
it has them in LDS once it has waited for a load that it issued later: the scales', whose values it stores to LDS before the
barrier behind which others read the tiles.  A store that a wavefront skips for want of live lanes leaves its part of the
tiles without that wait, so no branch on the lanes may lead past it.  (Branches on what all wavefronts share, whether there is
a next chunk, lead past the loads and the stores alike.)"""

import os
import re
import shutil
import subprocess

import pytest

from test_codegen import BUILD, LLVM, TARGET, _tools

TO_LDS = re.compile(r"^buffer_load_dwordx4 .*\blds\b")
LOAD = re.compile(r"^global_load_dword ([va]\d+),")
WRITE = re.compile(r"^ds_write(?:2|2st64)?_b32 v\d+, ([va]\d+)(?:, ([va]\d+))?")
BRANCH = re.compile(r"^s_(c?)branch\S* (\d+)")


def _unwaited(lines):
    """Of a kernel's instructions (address, text): the addresses of barriers that a path through a branch on the lanes reaches
    with loads into LDS behind which it has stored no later load's value."""
    at = {a: i for i, (a, _) in enumerate(lines)}
    nothing = (False, frozenset(), False)  # loads into LDS on their way, registers of loads after them, whether lanes were skipped
    seen, work, bad = set(), [(0, nothing)], set()
    while work:
        i, state = work.pop()
        while (i, state) not in seen:
            seen.add((i, state))
            a, text = lines[i]
            pending, later, skipped = state
            if TO_LDS.match(text):
                state = (True, frozenset(), False)
            elif pending and LOAD.match(text):
                state = (True, later | {LOAD.match(text).group(1)}, skipped)
            elif pending and WRITE.match(text) and later & set(WRITE.match(text).groups()):
                state = nothing
            elif text.startswith("s_barrier") and pending and skipped:
                bad.add(a)
            if text.startswith("s_endpgm"):
                break
            m = BRANCH.match(text)
            if m:
                off = int(m.group(2))
                to = at[a + 4 + 4 * (off - 65536 if off >= 32768 else off)]
                if m.group(1):
                    work.append((to, (*state[:2], state[2] or "exec" in text.split()[0])))
                else:
                    i = to
                    continue
            i += 1
    return bad


def _kernels(obj, tmp):
    fb, co = os.path.join(tmp, "fb"), os.path.join(tmp, "co")
    subprocess.run(["objcopy", f"--dump-section=.hip_fatbin={fb}", obj, os.path.join(tmp, "o")], check=True)
    subprocess.run([os.path.join(LLVM, "clang-offload-bundler"), "--type=o", f"--targets={TARGET}", f"--input={fb}",
                    f"--output={co}", "--unbundle"], check=True, capture_output=True)
    text = subprocess.run([os.path.join(LLVM, "llvm-objdump"), "-d", "--no-show-raw-insn", co], check=True, capture_output=True,
                          text=True).stdout
    name, lines = None, []
    for line in text.splitlines():
        m = re.match(r"^[0-9a-f]+ <(\S+)>:", line)
        if m:
            if name:
                yield name, lines
            name, lines = m.group(1), []
        elif "//" in line:
            ins, where = line.split("//")
            lines.append((int(where.split(":")[0], 16), " ".join(ins.split())))
    if name:
        yield name, lines


@pytest.mark.parametrize("unit", ["delta_bf16", "delta_bf16_wide"])
def test_every_wavefront_waits_for_its_loads_into_lds(unit, tmp_path):
    obj = os.path.join(BUILD, unit + ".o")
    if not os.path.exists(obj) or not _tools() or shutil.which("objcopy") is None:
        pytest.skip("no build objects or no tools to read them")
    direct = {name: _unwaited(lines) for name, lines in _kernels(obj, str(tmp_path)) if any(TO_LDS.match(t) for _, t in lines)}
    assert direct, "no kernel loads into LDS"
    bad = {name: sorted(map(hex, b)) for name, b in direct.items() if b}
    assert not bad, f"barriers that loads into LDS reach without a wait of their wavefront's: {bad}"


def test_the_walk_finds_a_store_that_can_be_skipped():
    text = ["buffer_load_dwordx4 v1, s[0:3], s4 offen lds", "global_load_dword v2, v3, s[0:1]", "s_cbranch_execz 1",
            "ds_write_b32 v4, v2", "s_barrier", "s_endpgm"]
    lines = [(4 * i, t) for i, t in enumerate(text)]
    assert _unwaited(lines) == {16}
    lines[2] = (8, "s_nop 0")
    assert _unwaited(lines) == set()
    lines[2] = (8, "s_cbranch_vccnz 1")  # one that all lanes take
    assert _unwaited(lines) == set()
