"""The read-back kernel's waits, from its compiled code (CPU only).

``mx4_unrotate_kernel`` copies a tile's rows into LDS asynchronously and reads them
behind a barrier, where other waves' copies are read too: a wave has to have waited
for its own before it gets there. The waits count operations in flight (``s_waitcnt
vmcnt(n)``: all but the newest n are done), so whether one covers the copies depends on
what was issued behind them on every path that leads there. This walks those paths.
"""

import re
import subprocess

from mla_kv_quant_amd import build

VMEM = re.compile(r"(global|buffer|scratch|flat)_(load|store|atomic)")
MOST = 64  # past what a wait can count


def listing(source, out):
    cmd = [build.hipcc(), *build.common_flags(), "-w", "-x", "hip", "--cuda-device-only", "-S",
           str(build.CSRC / source), "-o", str(out)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-2000:]
    return out.read_text()


def kernels_of(text, name):
    """{symbol: instructions and labels} of the kernels whose symbol holds ``name``."""
    out, lines = {}, None
    for raw in text.splitlines():
        line = raw.split(";")[0].strip()
        if re.match(r"_Z\w+:$", line):
            lines = out.setdefault(line[:-1], []) if name in line else None
        elif line.startswith(".Lfunc_end"):
            lines = None
        elif lines is not None and line and (line.startswith(".LBB") or not line.startswith(".")):
            lines.append(line)
    return out


def copies_in_flight_at_barriers(lines):
    """Indices of barriers that a path reaches with an LDS copy that no wait has covered.

    The state in front of an instruction is the least number, over the paths there, of
    operations issued behind the newest copy that may be in flight; MOST + 1: none is.
    """
    at = {ln[:-1]: i for i, ln in enumerate(lines) if ln.endswith(":")}
    none = MOST + 1
    state = [None] * (len(lines) + 1)
    todo, bad = [(0, none)], set()
    while todo:
        i, new = todo.pop()
        if i >= len(lines) or (state[i] is not None and state[i] <= new):
            continue
        state[i] = s = new if state[i] is None else min(new, state[i])
        ln = lines[i]
        if "_load_lds_" in ln:
            s = 0
        elif VMEM.match(ln):
            s = s if s == none else min(s + 1, MOST)
        elif ln.startswith("s_waitcnt"):
            n = re.search(r"vmcnt\((\d+)\)", ln)
            if n and s >= int(n[1]):
                s = none
        elif ln.startswith("s_barrier"):
            if s != none:
                bad.add(i)
        elif ln.startswith("s_endpgm"):
            continue
        m = re.match(r"s_c?branch\w*\s+(\.LBB\w+)", ln)
        if m:
            todo.append((at[m[1]], s))
            if ln.startswith("s_branch"):
                continue
        todo.append((i + 1, s))
    return sorted(bad)


def test_the_walk_itself():
    copy, load, store = "global_load_lds_dwordx4 v[0:1], off", "global_load_dword v2, v[0:1], off", \
        "global_store_dword v[0:1], v2, off"
    assert copies_in_flight_at_barriers([copy, "s_waitcnt vmcnt(0)", "s_barrier", "s_endpgm"]) == []
    assert copies_in_flight_at_barriers([copy, "s_barrier", "s_endpgm"]) == [1]
    assert copies_in_flight_at_barriers([copy, load, store, "s_waitcnt vmcnt(2)", "s_barrier", "s_endpgm"]) == []
    assert copies_in_flight_at_barriers([copy, load, "s_waitcnt vmcnt(2)", "s_barrier", "s_endpgm"]) == [3]
    # the store is on one of two paths; and a loop whose first turn has none before it
    assert copies_in_flight_at_barriers([copy, "s_cbranch_scc1 .LBB0_1", store, ".LBB0_1:", "s_waitcnt vmcnt(1)",
                                         "s_barrier", "s_endpgm"]) == [5]
    loop = [copy, ".LBB0_1:", "s_waitcnt vmcnt(1)", "s_barrier", copy, store, "s_cbranch_scc1 .LBB0_1", "s_endpgm"]
    assert copies_in_flight_at_barriers(loop) == [3]
    assert copies_in_flight_at_barriers([copy, "s_waitcnt vmcnt(0)"] + loop[1:]) == []


def test_no_barrier_is_passed_with_a_tile_on_its_way(tmp_path):
    found = kernels_of(listing("mx4_unrotate.hip", tmp_path / "k.s"), "mx4_unrotate_kernel")
    blocks = {s: lines for s, lines in found.items() if "Li8ELi2E" in s}  # eight waves, both widths
    assert len(blocks) == 2
    for symbol, lines in blocks.items():
        barriers = [i for i, ln in enumerate(lines) if ln.startswith("s_barrier")]
        assert len(barriers) >= 2 and any("_load_lds_" in ln for ln in lines)
        bad = copies_in_flight_at_barriers(lines)
        assert not bad, f"{symbol}: barriers {[barriers.index(i) for i in bad]} of {len(barriers)}"
