"""Bounded waits inside loops that meet at a named barrier.  A warp that gives up its wait and leaves such a loop by itself makes the others wait at
the barrier without a bound, which no test can provoke without hanging a GPU: the sources are read instead.  Runs without a GPU."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ml-recurrent-drafter_b200", "csrc")


def blocks(source):
    """The bodies of all loops, the innermost and outer ones alike, without comments."""
    text = re.sub(r"//[^\n]*", "", source)
    for m in re.finditer(r"\bfor \(", text):
        depth, i = 0, m.end() - 1
        while True:  # past the loop's head
            depth += {"(": 1, ")": -1}.get(text[i], 0)
            i += 1
            if depth == 0:
                break
        rest = text[i:].lstrip()
        if not rest.startswith("{"):
            continue
        i, start = text.index("{", i), text.index("{", i)
        while True:
            depth += {"{": 1, "}": -1}.get(text[i], 0)
            i += 1
            if depth == 0:
                break
        yield text[start:i]


def left_alone(body):
    """Conditions under which a thread leaves a loop that holds a named barrier, where these were not agreed upon."""
    if not re.search(r"bar\.sync 1|epilogue_agrees\(", body):
        return []
    return [m.group(0) for m in re.finditer(r"if \(([^;{}]*wait[^;{}]*)\) \{[^{}]*\b(?:break|return)\b[^{}]*\}", body) if "epilogue_agrees(" not in m.group(1)]


@pytest.mark.parametrize("name", ["gemm_int8.cu", "gemm_tc.cu"])
def test_epilogue_warps_leave_a_loop_together(name):
    with open(os.path.join(CSRC, name)) as f:
        source = f.read()
    assert "epilogue_agrees(" in source
    found = [leave for body in blocks(source) for leave in left_alone(body)]
    assert not found, found


def test_the_reading_finds_one_that_leaves_alone():
    good = "for (;;) { stage(); if (!rd::epilogue_agrees(warp_wait(&full, 0, stop))) { ok = false; break; } use(); }"
    bad = 'for (int t = 0; t < n; ++t) { asm volatile("bar.sync 1, 128;" ::: "memory"); if (!warp_wait(&full, 0, stop)) { ok = false; break; } use(); }'
    assert not any(left_alone(b) for b in blocks(good)) and any(left_alone(b) for b in blocks(bad))


@pytest.mark.parametrize("name, kernels", [("gemm_int8.cu", 2), ("attention_quant_many.cuh", 1)])
def test_a_kernel_that_gave_up_lets_its_work_land(name, kernels):
    """Copies and products in flight have time to land before tensor memory is given back and the CTA leaves its shared memory."""
    with open(os.path.join(CSRC, name)) as f:
        source = f.read()
    ends = re.findall(r"__syncthreads\(\);\n  if \(\*stop\)\n    for \(int i = 0; i < 2000; \+\+i\) __nanosleep\(1000\);[^}]*?dealloc", source)
    assert len(ends) == len(re.findall(r"tmem_dealloc\(|tcgen05\.dealloc", source)) == kernels
