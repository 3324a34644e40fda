"""The loads to LDS of csrc/mfma_tile.h are written in assembly, where the
compiler inserts no wait states.  gfx950 wants five between a vector
instruction that writes a scalar register and a buffer load that reads it, and
one after a write of m0: both are looked for in the assembly that hipcc makes
of the kernels, along every way to each load."""
import os
import re
import subprocess

import pytest

from bsscl_gbm import _build

WANTED = 5


def _scalars(operand):
    m = re.fullmatch(r"s\[(\d+):(\d+)\]", operand)
    if m:
        return set(range(int(m.group(1)), int(m.group(2)) + 1))
    m = re.fullmatch(r"s(\d+)", operand)
    return {int(m.group(1))} if m else set()


def _functions(text):
    """Each kernel's instructions and labels, comments and directives left out."""
    code = []
    for line in text.splitlines():
        line = line.split(";")[0].strip()
        m = re.match(r"(\S+):$", line)
        if m and not m.group(1).startswith(".L"):
            if code:
                yield code
            code = []
        elif m or (line and not line.startswith(".")):
            code.append(line)
    if code:
        yield code


def _faults(code):
    into = {}
    for i, t in enumerate(code):
        if t.startswith(("s_branch", "s_cbranch")):
            into.setdefault(t.split()[-1], []).append(i)
    for at, t in enumerate(code):
        if not (t.startswith("buffer_load") and t.endswith("lds")):
            continue
        reads = _scalars(re.split(r",\s*", t.split(None, 1)[1])[1])
        assert len(reads) == 4, t
        if not code[at - 1].startswith("s_nop") or not code[at - 2].startswith("s_mov_b32 m0"):
            yield "m0", t
        ways, seen = [(at - 1, 0)], set()
        while ways:
            i, states = ways.pop()
            if i < 0 or states >= WANTED or (i, states) in seen:
                continue
            seen.add((i, states))
            op = code[i].split()
            if op[0].endswith(":"):
                ways += [(j - 1, states + 1) for j in into.get(op[0][:-1], [])]
                if not code[i - 1].startswith(("s_branch", "s_endpgm", "s_setpc")):
                    ways.append((i - 1, states))
                continue
            if op[0].startswith("v_") and len(op) > 1 and _scalars(op[1].rstrip(",")) & reads:
                yield code[i], t
            states += int(op[1], 0) + 1 if op[0] == "s_nop" else 1
            ways.append((i - 1, states))


def test_the_search_finds_what_it_is_for():
    load = ["s_mov_b32 m0, s9", "s_nop 0", "buffer_load_dwordx4 v1, s[4:7], 0 offen lds"]
    assert not list(_faults(["v_readlane_b32 s3, v0, 1"] + load))
    assert list(_faults(["v_readlane_b32 s5, v0, 1", "s_nop 1"] + load))
    assert not list(_faults(["v_readlane_b32 s5, v0, 1", "s_nop 2"] + load))
    assert list(_faults([".LBB0_1:"] + load + ["v_readfirstlane_b32 s6, v2",
                                               "s_cbranch_scc1 .LBB0_1"]))
    away = ["v_readfirstlane_b32 s6, v2", "s_branch .LBB0_2"]
    assert list(_faults(away + [".LBB0_1:", "s_nop 7", ".LBB0_2:"] + load))
    assert not list(_faults(away + [".LBB0_1:"] + load + [".LBB0_2:"]))
    assert list(_faults(load[1:]))


def test_loads_to_lds_have_their_wait_states(tmp_path):
    try:
        cc = _build.hipcc()
    except RuntimeError:
        pytest.skip("no hipcc")
    out = os.path.join(tmp_path, "head.s")
    subprocess.run([cc, *[f for f in _build.flags() if f != "-fPIC"], "-S", "--cuda-device-only",
                    os.path.join(_build.CSRC, "softmax_head.hip"), "-o", out], check=True,
                   stderr=subprocess.DEVNULL)
    with open(out) as f:
        functions = list(_functions(f.read()))
    loads = sum(t.startswith("buffer_load") and t.endswith("lds") for c in functions for t in c)
    assert loads > 100, "the kernels hold no loads to LDS"
    faults = [f for c in functions for f in _faults(c)]
    assert not faults, faults[:5]


def test_each_load_brings_its_wait_states_along():
    """Whatever the compiler puts before a load: the move to m0 and the s_nop
    between them are the five states by themselves."""
    with open(os.path.join(_build.CSRC, "mfma_tile.h")) as f:
        found = re.findall(r's_mov_b32 m0, %0\\n\\ts_nop (\d+)\\n\\tbuffer_load\w+ .* lds"', f.read())
    assert found and all(1 + int(n) + 1 >= WANTED for n in found)
