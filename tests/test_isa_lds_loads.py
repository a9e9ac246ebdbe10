"""The generated ISA around the loads that go straight into LDS, which csrc/dense_gemm_kernel.hpp writes as inline assembly: the
compiler keeps the distances that the hardware asks for between its own instructions, but does not look into such a string.
- m0 (the load's place in LDS) may be read one wait state after a scalar write of it at the earliest;
- a scalar register of the load (descriptor, offset) may be read five wait states after a vector instruction wrote it.
The sources are compiled to assembly (hipcc cross-compiles without a GPU) and scanned."""
import concurrent.futures
import glob
import os
import re

import pytest

from test_isa_store_hazard import CSRC, HIPCC, _compile


def _scalars(tok):
    m = re.match(r"s\[(\d+):(\d+)\]$", tok)
    if m:
        return set(range(int(m.group(1)), int(m.group(2)) + 1))
    m = re.match(r"s(\d+)$", tok)
    return {int(m.group(1))} if m else set()


def _states(instruction):
    m = re.match(r"s_nop (\d+)", instruction)
    return int(m.group(1)) + 1 if m else 1


def lds_load_sites(asm_text):
    """(number of loads into LDS, those that come too early after a write of a register they read)."""
    lines = [l.split(";")[0].strip() for l in asm_text.splitlines()]
    ins = [l for l in lines if l and not l.startswith((".", "//")) and not l.endswith(":")]
    loads, sites = 0, []
    for k, l in enumerate(ins):
        if not re.match(r"buffer_load_\w+ .*\blds$", l):
            continue
        loads += 1
        if re.match(r"s_\w+ m0\b", ins[k - 1]):
            sites.append((ins[k - 1], l))
        used = set().union(*(_scalars(t) for t in re.findall(r"\bs\[\d+:\d+\]|\bs\d+\b", l)))
        before, j = 0, k - 1
        while j >= 0 and before < 5:
            m = re.match(r"v_\w+ (s\[\d+:\d+\]|s\d+)", re.sub(r"\s+", " ", ins[j]))
            if m and _scalars(m.group(1)) & used:
                sites.append((ins[j], l))
                break
            before += _states(ins[j])
            j -= 1
    return loads, sites


def test_scanner_sees_the_patterns():
    load = "buffer_load_dwordx4 v1, s[8:11], 0 offen lds\n"
    assert lds_load_sites("s_mov_b32 m0, s4\n" + load) == (1, [("s_mov_b32 m0, s4", load.strip())])
    assert lds_load_sites("s_mov_b32 m0, s4\ns_nop 0\n" + load) == (1, [])
    assert len(lds_load_sites("v_readfirstlane_b32 s9, v3\ns_mov_b32 m0, s4\ns_nop 0\n" + load)[1]) == 1
    assert lds_load_sites("v_readfirstlane_b32 s9, v3\ns_nop 2\ns_mov_b32 m0, s4\ns_nop 0\n" + load) == (1, [])
    assert lds_load_sites("v_readfirstlane_b32 s4, v3\ns_mov_b32 m0, s4\ns_nop 0\n" + load) == (1, [])
    assert lds_load_sites("buffer_load_dwordx4 v[1:4], v1, s[8:11], 0 offen\n") == (0, [])


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not found")
def test_no_load_into_lds_comes_too_early(tmp_path):
    srcs = sorted(glob.glob(os.path.join(CSRC, "dense_gemm_*.hip")))
    assert len(srcs) == 4, srcs
    with concurrent.futures.ThreadPoolExecutor(max_workers=4) as ex:
        results = list(ex.map(lambda s: _compile(s, str(tmp_path)), srcs))
    for src, asm in results:
        loads, sites = lds_load_sites(asm)
        assert loads >= 50, src
        assert not sites, "%s: %d sites, first: %s || %s" % (os.path.basename(src), len(sites), sites[0][0], sites[0][1])
