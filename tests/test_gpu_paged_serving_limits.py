"""The paged-cache serving operators on the GPU at the ends of their argument
ranges (bounds as in tests/paged_reference.py)."""

import sys

import pytest
import torch

import paged_reference as R
from test_gpu_paged_serving import clean_status, dev, mk, pools, randn, status, within  # noqa: F401

pytestmark = pytest.mark.gpu


# --------------------------------------------------------------------------- #
# windows and sinks near 2^63
# --------------------------------------------------------------------------- #
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 40)])
def test_far_windows_are_no_window(mk, dtype, D):
    """window=sys.maxsize is a usual way to say "everything": the same bits as
    no window, totals included, and nothing outside the scratch (a neighbour
    of the workspace keeps its bits)."""
    g = torch.Generator().manual_seed(4)
    B, Hq, Hkv, ps, n, S = 2, 8, 2, 16, 700, 20
    table = dev(R.make_table(B, n, -(-n // ps), ps, 3))
    kp, vp = (dev(t) for t in pools(g, -(-n // ps), B, Hkv, ps, D, dtype))
    q = dev(randn(g, B, S, Hq, D, dtype=dtype))
    lens = torch.tensor([n, 55]).cuda()

    def calls(**kw):
        w = torch.zeros(B, Hkv, n, device="cuda")
        out = mk.fused_paged_decode_attention(q[:, 0], kp, vp, table, lens, key_weights=w, **kw)
        return out, w, mk.fused_paged_prompt_attention(q, kp, vp, table, lens, **kw)

    want = calls()
    assert float(want[1].sum()) > 0
    for window in ((1 << 30) + 1, 1 << 62, sys.maxsize):
        for sinks in (0, 4, sys.maxsize):
            for a, b in zip(calls(window=window, sinks=sinks), want):
                assert torch.equal(a, b), (window, sinks)
    # a small window and every earlier key a sink: all keys again, numbered otherwise (sinks first)
    ref, tol, w, wtol = R.attention(q[:, :1].cpu(), kp.cpu(), vp.cpu(), table.cpu(), [n, 55], [1, 1], None, 0)
    out, got, _ = calls(window=5, sinks=sys.maxsize)
    within(out, ref[:, 0], tol[:, 0])
    within(got, w, wtol + w * 2.0 ** -23)


# --------------------------------------------------------------------------- #
# lengths outside their range
# --------------------------------------------------------------------------- #
@pytest.mark.parametrize("S,Hq,D,dtype,width", [
    (5, 2, 64, torch.bfloat16, 40),     # 16-row tiles
    (40, 2, 64, torch.bfloat16, 40),    # 128-row tiles
    (40, 4, 128, torch.float16, 3000),  # pieces of the key axis, joined
    (40, 2, 64, torch.float32, 40),     # row by row
])
def test_bad_lengths_are_recorded_on_every_path(mk, S, Hq, D, dtype, width):
    """Lengths are forced into [0, table width] and [0, min(S, length)], and
    recorded whichever kernel serves the call."""
    g = torch.Generator().manual_seed(4)
    B, ps = 40, 16  # more sequences than lanes; the bad ones lie behind the first 32
    P = -(-width // ps)
    kp, vp = (dev(t) for t in pools(g, P, B, 1, ps, D, dtype))
    table = dev(R.make_table(B, width, P, ps, 3))
    q = dev(randn(g, B, S, Hq, D, dtype=dtype))

    def call(lens, new=None):
        t = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32).cuda()
        out = mk.fused_paged_prompt_attention(q, kp, vp, table, t(lens), t(new))
        return out, status()

    ok = [min(width, 7 * b) for b in range(B)]
    good, code = call(ok)  # a sequence shorter than S has that many rows: in range
    assert code == 0
    for b, bad, forced in ((35, width + 1, width), (38, -2, 0), (39, 2 ** 31 - 1, width)):
        want, code = call(ok[:b] + [forced] + ok[b + 1:])
        assert code == 0
        got, code = call(ok[:b] + [bad] + ok[b + 1:])
        assert code == 7 and torch.equal(got, want), b
    new = [min(S, n) for n in ok]
    out, code = call(ok, new)
    assert code == 0 and torch.equal(out, good)
    for b, bad, forced in ((1, 8, min(S, 7)), (34, S + 1, S), (37, -1, 0), (39, -2 ** 31, 0)):
        want, code = call(ok, new[:b] + [forced] + new[b + 1:])
        assert code == 0
        got, code = call(ok, new[:b] + [bad] + new[b + 1:])
        assert code == 7 and torch.equal(got, want), b


# --------------------------------------------------------------------------- #
# NaN queries
# --------------------------------------------------------------------------- #
@pytest.mark.parametrize("S,Hq,D,dtype,n", [
    (1, 4, 128, torch.bfloat16, 60), (1, 4, 128, torch.bfloat16, 5000), (1, 20, 64, torch.float16, 3000),
    (4, 4, 128, torch.float16, 4000), (40, 4, 128, torch.bfloat16, 60), (40, 4, 128, torch.bfloat16, 5000),
    (70, 7, 80, torch.float16, 3000), (1, 2, 40, torch.float32, 500), (3, 2, 40, torch.float32, 500),
])
def test_nan_queries_stay_nan(mk, S, Hq, D, dtype, n):
    """A NaN in a query makes that row NaN, in one piece or in joined pieces,
    and leaves every other row's bits alone."""
    g = torch.Generator().manual_seed(4)
    B, ps = 2, 16
    P = -(-n // ps)
    kp, vp = (dev(t) for t in pools(g, P, B, 1, ps, D, dtype))
    table = dev(R.make_table(B, n, P, ps, 3))
    q = dev(randn(g, B, S, Hq, D, dtype=dtype))
    lens = torch.tensor([n, n // 2]).cuda()

    def call(x):
        out = [mk.fused_paged_prompt_attention(x, kp, vp, table, lens)]
        if S == 1:
            out.append(mk.fused_paged_decode_attention(x[:, 0], kp, vp, table, lens)[:, None])
        return out

    bad = q.clone()
    hit = torch.zeros(B, S, Hq, dtype=torch.bool)
    for b, s, h in ((0, S - 1, 1), (1, 0, Hq - 1), (1, S // 2, 0)):
        bad[b, s, h, 3] = float("nan")
        hit[b, s, h] = True
    for good, got in zip(call(q), call(bad)):
        assert torch.isfinite(good).all()
        assert got.cpu()[hit].isnan().all()
        assert torch.equal(got.cpu()[~hit], good.cpu()[~hit])
    if S > 1:
        return
    w = [torch.zeros(B, 1, n, device="cuda") for _ in range(2)]
    bad[1] = q[1]
    for x, t in zip((q, bad), w):
        mk.fused_paged_decode_attention(x[:, 0], kp, vp, table, lens, key_weights=t)
    assert w[1][0, 0].isnan().all() and torch.equal(w[0][1], w[1][1])  # that key head's totals alone


# --------------------------------------------------------------------------- #
# page ids outside the pool
# --------------------------------------------------------------------------- #
@pytest.mark.parametrize("S,Hq,D,dtype,n", [
    (5, 2, 64, torch.bfloat16, 90), (40, 4, 128, torch.bfloat16, 90), (300, 4, 64, torch.float16, 300),
    (40, 4, 128, torch.float16, 3000), (40, 2, 40, torch.float32, 90),
])
def test_bad_pages_in_prompts(mk, S, Hq, D, dtype, n):
    """A page id outside the pool is recorded where a row sees it; rows in
    front of it keep their bits, and ids that no row sees are not looked at."""
    g = torch.Generator().manual_seed(4)
    B, ps = 2, 16
    P = -(-n // ps)
    kp, vp = (dev(t) for t in pools(g, P, B, 1, ps, D, dtype))
    table = R.make_table(B, n, P, ps, 3)
    q = dev(randn(g, B, S, Hq, D, dtype=dtype))
    lens = torch.tensor([n, n - 20]).cuda()
    call = lambda t: mk.fused_paged_prompt_attention(q, kp, vp, dev(t), lens)
    good = call(table)
    behind = table.clone()
    behind[1, n - 20:] = 1 << 30  # behind the sequence
    assert torch.equal(call(behind), good) and status() == 0
    at = n - 2  # the last rows of sequence 0 see it
    for bad in (P, -P - 1, 2 ** 31 - 1, -2 ** 31):
        t = table.clone()
        t[0, at] = bad
        out = call(t)
        assert status() == 7
        assert torch.equal(out[1], good[1]) and torch.equal(out[0, :S - 2], good[0, :S - 2])
        assert torch.isfinite(out).all()
