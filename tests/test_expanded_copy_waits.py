"""The expanded attention's counted waits, from its compiled code (CPU only).

A step of ``expanded_kernel`` issues five asynchronous copies into LDS and waits, before it meets the other waves, for all
operations but the newest ten (``s_waitcnt vmcnt(10)``): what was issued two steps before is there. That holds while at
least five operations lie between one such wait and the next, on every path, or a wait for all of them does.
"""

import re

from tests.test_lds_copy_waits import VMEM, kernels_of, listing

STEP, WAIT = 5, "s_waitcnt vmcnt(10) lgkmcnt(0)"  # (the compiler's own waits name one counter at a time there)


def few_between_waits(lines):
    """{index of a counted wait: the least number of operations, over the paths there, since the counted wait before it},
    where that is below ``STEP``."""
    at = {ln[:-1]: i for i, ln in enumerate(lines) if ln.endswith(":")}
    waits = {i for i, ln in enumerate(lines) if ln == WAIT}
    state, bad, todo = {}, {}, [(i + 1, 0) for i in waits]
    while todo:
        i, n = todo.pop()
        if i >= len(lines) or state.get(i, STEP) <= n:  # (STEP and more are enough)
            continue
        state[i] = n
        ln = lines[i]
        if i in waits:
            bad[i] = min(n, bad.get(i, n))
            continue
        if VMEM.match(ln):
            n += 1
        elif ln.startswith("s_endpgm") or (ln.startswith("s_waitcnt") and "vmcnt(0)" in ln):
            continue
        m = re.match(r"s_c?branch\w*\s+(\.LBB\w+)", ln)
        if m:
            todo.append((at[m[1]], n))
            if ln.startswith("s_branch"):
                continue
        todo.append((i + 1, n))
    return bad


def test_the_walk_itself():
    copy, wait, end = "global_load_lds_dwordx4 v1, s[0:1]", WAIT, "s_endpgm"
    assert few_between_waits([wait, *[copy] * 5, wait, end]) == {}
    assert few_between_waits([wait, *[copy] * 4, wait, end]) == {5: 4}
    assert few_between_waits([wait, copy, "s_waitcnt vmcnt(0)", wait, end]) == {}
    # a path past one of the copies, and a loop
    assert few_between_waits([wait, *[copy] * 4, "s_cbranch_vccnz .LBB0_1", copy, ".LBB0_1:", wait, end]) == {8: 4}
    assert few_between_waits([".LBB0_1:", copy, copy, wait, copy, copy, "s_cbranch_scc1 .LBB0_1", end]) == {3: 4}
    assert few_between_waits([".LBB0_1:", copy, copy, wait, *[copy] * 3, "s_cbranch_scc1 .LBB0_1", end]) == {}


def test_every_step_issues_what_its_waits_count_on(tmp_path):
    found = kernels_of(listing("expanded.hip", tmp_path / "k.s"), "expanded_kernel")
    assert len(found) == 4  # two widths, with and without the LSE
    for symbol, lines in found.items():
        waits = [i for i, ln in enumerate(lines) if ln == WAIT]
        # four steps and the one that only copies, in the plain pass and in the careful one
        assert len(waits) >= 10, symbol
        for i in waits:  # (what other waves' copies brought is read behind the barrier)
            ahead = lines[i + 1:i + 12]
            ahead = ahead[:[ln.startswith("s_barrier") for ln in ahead].index(True)]
            assert not any(ln.startswith("ds_") or VMEM.match(ln) for ln in ahead), (symbol, ahead)
        assert few_between_waits(lines) == {}, symbol
