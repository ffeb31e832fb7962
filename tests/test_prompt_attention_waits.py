"""The tensor-core prompt kernel's waits all end.  Its mbarrier waits have a
limit; the meeting of the two softmax warps that share 32 rows (a named
barrier) has none, so the two must come to it equally often whatever their
waits come to.  Shown here on the CPU: over every outcome of the waits for a
walk written as the kernel writes it, and on the kernel's source for the form
that the walk stands for."""

import itertools
import os
import re

import pytest

from conftest import REPO

GONE = "gone"


def walk(items):
    """One softmax warp: yields "wait" (sent: whether it came in time) and
    ("meet", value) (sent: the partner's value).  items: chunks per item."""
    for n_it in items:
        ok = True
        for _ in range(n_it):
            if not (yield "wait"):
                yield ("meet", GONE)
                ok = False
                break
            if (yield ("meet", "max")) == GONE:
                ok = False
                break
        if not ok:
            return
        if n_it > 0:
            yield ("meet", "sum")
            if not (yield "wait"):
                continue  # no output, on to the next item


def walk_that_leaves(items):
    """The form it must not have: leaving as soon as a wait has run out."""
    for n_it in items:
        for _ in range(n_it):
            if not (yield "wait"):
                return
            yield ("meet", "max")
        if n_it > 0:
            yield ("meet", "sum")
            if not (yield "wait"):
                return


class Warp:
    def __init__(self, walk, items, outcomes):
        self.g, self.outcomes = walk(items), iter(outcomes)
        self.at = next(self.g, None)

    def run(self):  # up to the next meeting, or the end
        while self.at == "wait":
            self.send(next(self.outcomes))

    def send(self, x):
        try:
            self.at = self.g.send(x)
        except StopIteration:
            self.at = None


def both_end(walk, items, a, b):
    x, y = Warp(walk, items, a), Warp(walk, items, b)
    while True:
        x.run(), y.run()
        if x.at is None or y.at is None:
            return x.at is None and y.at is None
        x_value, y_value = x.at[1], y.at[1]
        # a meeting is of two values of one kind, or with a warp that leaves
        assert x_value == y_value or GONE in (x_value, y_value)
        x.send(y_value), y.send(x_value)


ITEMS = [(1,), (2,), (0, 1), (1, 1), (2, 0, 1), (1, 2)]


@pytest.mark.parametrize("items", ITEMS)
def test_partners_meet_equally_often(items):
    waits = sum(n + (n > 0) for n in items)
    for a in itertools.product((True, False), repeat=waits):
        for b in itertools.product((True, False), repeat=waits):
            assert both_end(walk, items, a, b), (a, b)


def test_leaving_at_once_strands_the_partner():
    assert both_end(walk_that_leaves, (2,), (True,) * 3, (True,) * 3)
    assert not both_end(walk_that_leaves, (2,), (True, False, True), (True,) * 3)


def softmax_source():
    src = open(os.path.join(REPO, "mtp-engine_b200", "csrc", "mtp_promptattn_tc.cuh")).read()
    kernel = src[src.index("prompt_attention_tc_kernel(const"):src.index("prompt_merge_kernel(Params p)")]
    code = re.sub(r"//[^\n]*", "", kernel)
    role = code[code.index("ex_mine ="):]
    assert code.count("bar.sync") == role.count("bar.sync") == 1  # the exchange's own
    return role


def test_the_kernel_has_that_form():
    role = softmax_source()
    loop = role[role.index("for (int r = 0"):]
    # a wait that ran out never ends the walk by itself ...
    assert not re.search(r"wait_bar\([^;{]*\)\)\)\s*break", loop)
    # ... the one inside the chunk loop meets the partner first
    assert re.search(r"if \(!__all_sync\(0xffffffffu, wait_bar\(&s_full[^;{]*\{\s*"
                     r"exchange\(__uint_as_float\(kGone\)\);\s*ok = false;\s*break;\s*\}", loop)
    # ... and the partner leaves when it hears of it
    assert re.search(r"other = exchange\(mx\);\s*if \(__any_sync\(0xffffffffu, __float_as_uint\(other\) == kGone\)\) "
                     r"\{\s*ok = false;\s*break;\s*\}", loop)
    assert re.search(r"got = __all_sync\(0xffffffffu, wait_bar\(&pv_done[^;]*;[^{}]*if \(!got\) continue;", loop)
    # every other way out is one that both warps take: no more items, or the two above
    assert loop.count("wait_bar(") == 2 and loop.count("exchange(") == 3
    assert sorted(re.findall(r"(?:if \([^\n]*\) )?break;", loop)) == \
        ["break;", "break;", "if (!more) break;", "if (!ok) break;"]
    assert "return" not in loop[:loop.index("tc_fence_before();\n  __syncthreads();")]


def test_loads_land_before_the_block_ends():
    """After a wait ran out, page loads may still be under way into shared
    memory that the SM's next block will own: each producer waits (with a
    limit) for the loads it has issued, a full ring of chunks and the queries.
    `chunks` and `queries` count issued loads only."""
    src = open(os.path.join(REPO, "mtp-engine_b200", "csrc", "mtp_promptattn_tc.cuh")).read()
    code = re.sub(r"//[^\n]*|/\*.*?\*/ *", "", src)
    role = code[code.index("if (warp == kWarpK || warp == kWarpV)"):code.index("} else if (warp == kWarpMma) {")]
    tail = role[role.index("attn::cp_async_wait_all();\n      if (lane == 0)"):]
    assert re.search(r"for \(int j = max\(0, chunks - kRing\); j < chunks; \+\+j\)\s*"
                     r"mbar_wait\(&buf_full\[2 \* \(j % kRing\) \+ kv\], \(j / kRing\) & 1, abort_flag, false\);", tail)
    assert re.search(r"if \(queries > 0\) mbar_wait\(q_full, \(queries - 1\) & 1, abort_flag, false\);", tail)
    # counted behind the wait that may give up
    assert re.search(r"if \(!__shfl_sync\(0xffffffffu, got, 0\)\) break;\s*\+\+queries;", role)
    assert role.count("++queries") == 1 and role.count("++chunks") == 1
    assert re.search(r"for \(int i = 0; i < n_it && ok; \+\+i, \+\+chunks\)", role)
    # the fills of one buffer: chunk j is fill j / ring, and nothing is filled again behind the last ring
    for ring in (2, 4):
        for chunks in range(12):
            last = {}
            for j in range(chunks):
                last[j % ring] = j // ring
            waited = {j % ring: j // ring for j in range(max(0, chunks - ring), chunks)}
            assert waited == last
