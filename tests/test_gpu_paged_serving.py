"""The paged-cache serving operators on the GPU against their 64-bit
restatement (tests/paged_reference.py, where the error bounds are derived):
query/key norm with rotation and cache write, prompt and decode attention
with windows, eviction; each alone and all of them in a row, as a server with
a bounded cache runs them."""

import math

import pytest
import torch

import paged_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mk():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import mtp_kernels
    return mtp_kernels


@pytest.fixture(autouse=True)
def clean_status():
    """Every test starts and ends with a clean device error word."""
    if not torch.cuda.is_available():
        yield
        return
    import _mtp_native
    d = torch.device("cuda", 0)
    _mtp_native.device_status(d)
    yield
    assert _mtp_native.device_status(d) == 0


def status():
    import _mtp_native
    return _mtp_native.device_status(torch.device("cuda", 0))


def dev(t):
    return t.cuda() if t is not None else None


def randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (scale * torch.randn(*shape, generator=g)).to(dtype)


def within(got, ref, tol):
    err = (got.double().cpu() - ref).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values outside; worst {float((err - tol).max()):.3g} over"


def pools(g, P, B, H, ps, D, dtype):
    return randn(g, P, B, H, ps, D, dtype=dtype), randn(g, P, B, H, ps, D, dtype=dtype)


def wipe_unused(pages, table, lens, ps, low=None):
    """NaN in every slot that no visible position owns."""
    keep = torch.zeros(pages.shape[0], pages.shape[1], ps, dtype=torch.bool)
    for b, n in enumerate(lens):
        for j in range(n):
            if low is None or j >= low[b][0] or j < low[b][1]:
                keep[int(table[b, j]), b, j % ps] = True
    return torch.where(keep[:, :, None, :, None], pages, torch.full_like(pages, float("nan")))


# --------------------------------------------------------------------------- #
# decode
# --------------------------------------------------------------------------- #
DECODE = [
    # B, Hq, Hkv, D, ps, lens, window, sinks, dtype, per_token
    (1, 1, 1, 64, 16, [1], None, 0, torch.bfloat16, False),
    (2, 8, 2, 128, 16, [0, 17], None, 0, torch.bfloat16, False),
    (3, 14, 2, 64, 16, [16, 333, 50], None, 0, torch.float16, False),
    (4, 10, 2, 128, 8, [1, 2, 700, 15], None, 0, torch.float16, True),
    (2, 20, 1, 128, 16, [300, 31], None, 0, torch.bfloat16, False),  # 20 rows: two tiles
    (3, 4, 4, 80, 32, [129, 128, 127], None, 0, torch.bfloat16, False),
    (2, 6, 3, 96, 24, [100, 257], None, 0, torch.bfloat16, True),
    (2, 4, 2, 256, 16, [90, 5], None, 0, torch.bfloat16, False),
    (2, 4, 2, 8, 16, [90, 5], None, 0, torch.float16, False),
    (3, 8, 2, 128, 16, [500, 64, 3], 64, 4, torch.bfloat16, False),
    (3, 8, 2, 128, 16, [500, 64, 3], 1, 0, torch.bfloat16, False),
    (2, 8, 2, 64, 16, [400, 70], 33, 200, torch.float16, True),  # more sinks than the window
    (2, 6, 2, 128, 16, [200, 9], None, 0, torch.float32, False),
    (2, 6, 2, 40, 7, [200, 9], 50, 3, torch.float32, True),
    (2, 6, 2, 20, 16, [100, 0], None, 0, torch.bfloat16, False),  # rows of 40 bytes
    (40, 2, 1, 64, 16, list(range(0, 120, 3)), None, 0, torch.bfloat16, False),  # more sequences than lanes
]


@pytest.mark.parametrize("B,Hq,Hkv,D,ps,lens,window,sinks,dtype,per_token", DECODE)
def test_decode(mk, B, Hq, Hkv, D, ps, lens, window, sinks, dtype, per_token):
    g = torch.Generator().manual_seed(B * 1000 + D)
    L = max(1, max(lens)) + 5
    P = -(-L // ps) + 3
    table = R.make_table(B, L, P, ps, 3, per_token)
    kp, vp = pools(g, P, B, Hkv, ps, D, dtype)
    q = randn(g, B, Hq, D, dtype=dtype, scale=1.5)
    low = None
    if window:
        low = [(max(0, n - window), sinks) for n in lens]
    kn, vn = wipe_unused(kp, table, lens, ps, low), wipe_unused(vp, table, lens, ps, low)
    ref, tol, w, wtol = R.attention(q[:, None], kp, vp, table, lens, [min(1, n) for n in lens], window, sinks)
    kw0 = torch.rand(B, Hkv, L + 2, generator=g)
    kw = dev(kw0.clone())
    args = (dev(q), dev(kn), dev(vn), dev(table), dev(torch.tensor(lens)))
    out = mk.fused_paged_decode_attention(*args, window=window, sinks=sinks)
    within(out, ref[:, 0], tol[:, 0])
    out2 = mk.fused_paged_decode_attention(*args, window=window, sinks=sinks, key_weights=kw)
    assert torch.equal(out, out2)
    want = kw0.double()
    want[:, :, :L] += w
    seen = torch.zeros_like(want, dtype=torch.bool)
    seen[:, :, :L] = w > 0
    bound = torch.zeros_like(want)
    bound[:, :, :L] = wtol
    assert torch.equal(kw.cpu()[~seen], kw0[~seen])  # what no query saw keeps its bits
    within(kw, want, bound + want.abs() * 2.0 ** -23 + 1e-30)


def test_decode_many_pieces(mk):
    """One sequence over the whole GPU (hundreds of pieces to join), values at
    growing scores so that the running maximum moves in every piece."""
    g = torch.Generator().manual_seed(5)
    B, Hq, Hkv, D, ps, n = 1, 4, 1, 128, 16, 20011
    P = -(-n // ps)
    table = R.make_table(B, n, P, ps, 1)
    kp, vp = pools(g, P, B, Hkv, ps, D, torch.bfloat16)
    q = randn(g, B, Hq, D, dtype=torch.bfloat16)
    grow = torch.linspace(0.0, 2.0, n).sqrt()
    for j in range(n):
        kp[int(table[0, j]), 0, 0, j % ps] = (kp[int(table[0, j]), 0, 0, j % ps].float() * grow[j]).to(torch.bfloat16)
    ref, tol, _, _ = R.attention(q[:, None], kp, vp, table, [n], [1], None, 0)
    args = (dev(q), dev(kp), dev(vp), dev(table), torch.tensor([n]).cuda())
    out = mk.fused_paged_decode_attention(*args)
    within(out, ref[:, 0], tol[:, 0])
    for _ in range(3):  # fixed order of the joins: the same bits every time
        assert torch.equal(out, mk.fused_paged_decode_attention(*args))


def test_decode_extreme_scores(mk):
    """Scores of +-10^4: one key takes everything, and nothing overflows."""
    g = torch.Generator().manual_seed(8)
    B, Hq, Hkv, D, ps, n = 2, 4, 2, 64, 16, 100
    table = R.make_table(B, n, 9, ps, 1)
    kp, vp = pools(g, 9, B, Hkv, ps, D, torch.bfloat16)
    q = randn(g, B, Hq, D, dtype=torch.bfloat16, scale=1000.0)
    out = mk.fused_paged_decode_attention(dev(q), dev(kp), dev(vp), dev(table), torch.tensor([n, n]).cuda(),
                                          scale=10.0)
    ref, _, _, _ = R.attention(q[:, None], kp, vp, table, [n, n], [1, 1], None, 0, scale=10.0)
    # the gap between the greatest scores is far above their rounding: the weights are 0 and 1
    assert torch.isfinite(out).all()
    within(out, ref[:, 0], 2.0 ** -7 * ref[:, 0].abs() + 1e-20)


# --------------------------------------------------------------------------- #
# prompt
# --------------------------------------------------------------------------- #
PROMPT = [
    # B, S, Hq, Hkv, D, ps, past, new, window, sinks, dtype, per_token
    (1, 1, 4, 2, 128, 16, [0], [1], None, 0, torch.bfloat16, False),
    (2, 3, 4, 2, 128, 16, [0, 61], [3, 1], None, 0, torch.bfloat16, False),
    (2, 8, 2, 2, 64, 16, [5, 0], [0, 8], None, 0, torch.float16, False),  # nothing new in a sequence
    (1, 200, 8, 2, 128, 16, [0], [200], None, 0, torch.bfloat16, False),
    (2, 130, 14, 2, 64, 16, [70, 0], [130, 33], None, 0, torch.float16, False),
    (2, 70, 8, 2, 128, 16, [301, 128], [70, 64], 48, 4, torch.bfloat16, False),
    (1, 300, 4, 4, 128, 32, [0], [300], 100, 130, torch.bfloat16, False),
    (1, 150, 4, 1, 80, 16, [33], [150], None, 0, torch.bfloat16, True),
    (2, 90, 6, 2, 96, 24, [10, 0], [90, 50], 64, 1, torch.float16, False),
    (1, 140, 5, 1, 128, 8, [260], [140], 1, 0, torch.bfloat16, True),
    (1, 129, 2, 2, 128, 128, [127], [129], None, 0, torch.bfloat16, False),
    (1, 64, 2, 1, 128, 256, [500], [64], None, 0, torch.bfloat16, False),
    (1, 60, 2, 1, 256, 16, [20], [60], None, 0, torch.bfloat16, False),
    (1, 40, 2, 1, 32, 16, [20], [40], 16, 2, torch.bfloat16, False),
    (1, 50, 2, 1, 64, 16, [20], [50], 30, 2, torch.float32, False),
    (1, 30, 3, 1, 20, 16, [20], [30], None, 0, torch.float16, False),
    (1, 20, 16, 1, 128, 16, [1500], [20], None, 0, torch.bfloat16, False),  # few rows, a long cache
    (1, 9, 130, 1, 64, 16, [40], [9], None, 0, torch.bfloat16, False),  # more heads than a tile has rows
    (1, 20, 2, 2, 128, 16, [3], [20], None, 0, torch.bfloat16, False),  # fewer positions than a tile has
    (2, 17, 1, 1, 64, 3, [0, 2], [17, 5], None, 0, torch.float16, False),  # pages of three tokens
    (2, 600, 2, 1, 96, 64, [0, 200], [333, 600], 130, 2, torch.bfloat16, False),  # several items, a short window
    (1, 300, 8, 1, 64, 16, [900], [300], 256, 300, torch.float16, True),  # sinks over whole chunks, scattered tokens
]


@pytest.mark.parametrize("B,S,Hq,Hkv,D,ps,past,new,window,sinks,dtype,per_token", PROMPT)
def test_prompt(mk, B, S, Hq, Hkv, D, ps, past, new, window, sinks, dtype, per_token):
    g = torch.Generator().manual_seed(S * 100 + D)
    lens = [p + n for p, n in zip(past, new)]
    L = max(lens) + 3
    P = -(-L // ps) + 3
    table = R.make_table(B, L, P, ps, 7, per_token)
    kp, vp = pools(g, P, B, Hkv, ps, D, dtype)
    q = randn(g, B, S, Hq, D, dtype=dtype, scale=1.5)
    low = None
    if window:  # what the first new row's window has left behind
        low = [(max(0, p - window + 1), sinks) for p in past]
    used = [n if m else 0 for n, m in zip(lens, new)]
    kn, vn = wipe_unused(kp, table, used, ps, low), wipe_unused(vp, table, used, ps, low)
    for b in range(B):  # padding rows hold anything
        q[b, new[b]:] = float("nan")
    ref, tol, _, _ = R.attention(q, kp, vp, table, lens, new, window, sinks)
    out = mk.fused_paged_prompt_attention(dev(q), dev(kn), dev(vn), dev(table), dev(torch.tensor(lens)),
                                          dev(torch.tensor(new)), window=window, sinks=sinks)
    within(out, ref, tol)


def test_prompt_all_rows_new(mk):
    """q_lens left out: all S rows are new."""
    g = torch.Generator().manual_seed(2)
    B, S, Hq, Hkv, D, ps = 2, 37, 4, 2, 128, 16
    table = R.make_table(B, 50, 6, ps, 7)
    kp, vp = pools(g, 6, B, Hkv, ps, D, torch.bfloat16)
    q = randn(g, B, S, Hq, D, dtype=torch.bfloat16)
    ref, tol, _, _ = R.attention(q, kp, vp, table, [37, 50], [37, 37], None, 0)
    out = mk.fused_paged_prompt_attention(dev(q), dev(kp), dev(vp), dev(table), torch.tensor([37, 50]).cuda())
    within(out, ref, tol)


def test_prompt_matches_decode(mk):
    """The last row of a prompt is the decode of that token."""
    g = torch.Generator().manual_seed(4)
    B, S, Hq, Hkv, D, ps, n = 2, 200, 8, 2, 128, 16, 260
    table = R.make_table(B, n, 20, ps, 7)
    kp, vp = (dev(x) for x in pools(g, 20, B, Hkv, ps, D, torch.float16))
    q = dev(randn(g, B, S, Hq, D, dtype=torch.float16))
    lens = torch.tensor([n, n - 40]).cuda()
    kw = dict(window=100, sinks=4)
    a = mk.fused_paged_prompt_attention(q, kp, vp, dev(table), lens, **kw)[:, -1]
    b = mk.fused_paged_decode_attention(q[:, -1], kp, vp, dev(table), lens, **kw)
    # both are within half a step and the weights' half step of the same value; |v| < 6
    assert (a.double() - b.double()).abs().max() <= 4 * 2.0 ** -11 * 6


def test_bad_lengths_and_pages_are_recorded(mk):
    g = torch.Generator().manual_seed(4)
    kp, vp = (dev(x) for x in pools(g, 4, 2, 1, 16, 64, torch.bfloat16))
    q = dev(randn(g, 2, 2, 64, dtype=torch.bfloat16))
    table = torch.zeros(2, 40, dtype=torch.int32).cuda()
    table[1, 3] = 9  # outside the pool, in sequence 1
    good = mk.fused_paged_decode_attention(q, kp, vp, table, torch.tensor([40, 3]).cuda())
    assert status() == 0
    out = mk.fused_paged_decode_attention(q, kp, vp, table, torch.tensor([40, 4]).cuda())
    assert status() == 7
    assert torch.equal(out[0], good[0])
    out = mk.fused_paged_decode_attention(q, kp, vp, table, torch.tensor([41, -2]).cuda())
    assert status() == 7
    assert torch.equal(out[0], good[0]) and not out[1].any()  # forced into [0, 40]
    qp = dev(randn(g, 2, 5, 2, 64, dtype=torch.bfloat16))
    out = mk.fused_paged_prompt_attention(qp, kp, vp, table, torch.tensor([3, 3]).cuda(),
                                          torch.tensor([4, -1]).cuda())
    assert status() == 7
    assert not out[0, 3:].any() and not out[1].any()


# --------------------------------------------------------------------------- #
# norm, rotation, cache write
# --------------------------------------------------------------------------- #
def angles(n, R_, far=0):
    t = torch.arange(far, far + n, dtype=torch.float64)[:, None] * 10000.0 ** (
        -torch.arange(0, R_, 2, dtype=torch.float64) / R_)
    return t.cos().float(), t.sin().float()


ROPE = [
    # B, S, Hq, Hkv, D, rot, interleaved, dtype, weights, eps, packed
    (1, 1, 1, 1, 64, 64, False, torch.bfloat16, True, 1e-6, False),
    (2, 5, 8, 2, 128, 128, False, torch.bfloat16, True, 1e-6, True),
    (2, 5, 8, 2, 128, 128, True, torch.float16, True, 1e-6, True),
    (3, 9, 7, 1, 96, 48, False, torch.float16, False, 1e-6, True),
    (3, 9, 7, 1, 96, 24, True, torch.bfloat16, True, None, True),
    (1, 11, 3, 3, 80, 80, False, torch.float32, True, 1e-5, True),  # half = 40
    (1, 11, 3, 2, 80, 40, False, torch.float32, True, 1e-5, False),  # half = 20: value by value
    (2, 4, 2, 1, 20, 10, True, torch.bfloat16, True, 1e-6, True),
    (2, 4, 2, 1, 256, 128, False, torch.bfloat16, True, 1e-6, True),
    (2, 3, 2, 1, 320, 64, False, torch.bfloat16, True, 1e-6, False),
    (2, 3, 2, 1, 64, 0, False, torch.bfloat16, True, 1e-6, False),  # nothing turns
    (4, 700, 4, 2, 64, 64, False, torch.bfloat16, True, 1e-6, True),  # eight tokens to a block
]


@pytest.mark.parametrize("B,S,Hq,Hkv,D,rot,interleaved,dtype,weights,eps,packed", ROPE)
@pytest.mark.parametrize("paged", [False, True])
def test_qk_norm_rope(mk, B, S, Hq, Hkv, D, rot, interleaved, dtype, weights, eps, packed, paged):
    g = torch.Generator().manual_seed(S * 10 + D)
    cos, sin = angles(S + 60, rot) if rot else (torch.zeros(S + 60, 0), torch.zeros(S + 60, 0))
    qkv = randn(g, B, S, Hq + 2 * Hkv, D, dtype=dtype, scale=2.0)
    q, k, v = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hkv], qkv[:, :, Hq + Hkv:]
    if not packed:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    qw = randn(g, D, dtype=torch.float32) if weights else None
    kw = randn(g, D, dtype=dtype) if weights else None
    pos = torch.randint(0, S + 60, (B, S), generator=g)
    rq, tq = R.norm_rope(q, qw, cos, sin, pos, eps, interleaved)
    rk, tk = R.norm_rope(k, kw, cos, sin, pos, eps, interleaved)
    gq, gk, gv = (dev(qkv)[:, :, a:b] for a, b in ((0, Hq), (Hq, Hq + Hkv), (Hq + Hkv, Hq + 2 * Hkv)))
    if not packed:
        gq, gk, gv = gq.contiguous(), gk.contiguous(), gv.contiguous()
    if not paged:
        oq, ok = mk.fused_qk_norm_rope(gq, gk, dev(pos), dev(cos), dev(sin), dev(qw), dev(kw), eps,
                                       interleaved=interleaved)
        assert oq.shape == (B, S, Hq, D) and ok.shape == (B, Hkv, S, D)
        within(oq, rq, tq)
        within(ok.transpose(1, 2), rk, tk)
        return
    ps = 16
    start = [7 * b for b in range(B)]
    count = [max(0, S - 2 * b) for b in range(B)]
    L = max(s + S for s in start)
    P = -(-L // ps) + 2
    table = R.make_table(B, L, P, ps, 3)
    kp0, vp0 = pools(g, P, B, Hkv, ps, D, dtype)
    kp, vp = dev(kp0), dev(vp0)
    oq = mk.fused_qk_norm_rope_paged(gq, gk, gv, dev(pos), dev(cos), dev(sin), kp, vp, dev(table),
                                     dev(torch.tensor(start)), dev(qw), dev(kw), eps,
                                     count=dev(torch.tensor(count)), interleaved=interleaved)
    wk, wv = kp0.double(), vp0.clone()
    tolk = torch.zeros_like(wk)
    for b in range(B):
        rq[b, count[b]:] = 0
        for s in range(count[b]):
            at = (int(table[b, start[b] + s]), b, slice(None), (start[b] + s) % ps)
            wk[at], tolk[at], wv[at] = rk[b, s], tk[b, s], v[b, s]
    within(oq, rq, tq)
    within(kp, wk, tolk)  # bound 0 where nothing was written: the same bits
    assert torch.equal(vp.cpu(), wv)


def test_rope_default_positions_and_far_angles(mk):
    """positions=None turns by start + s; far positions keep the tables' precision."""
    g = torch.Generator().manual_seed(3)
    B, S, H, D, ps = 2, 6, 2, 64, 16
    cos, sin = angles(40, D, far=1000000)
    start = torch.tensor([3, 20])
    x = randn(g, B, S, 3 * H, D, dtype=torch.float32)
    pos = start[:, None] + torch.arange(S)
    table = R.make_table(B, 40, 4, ps, 3)
    kp, vp = (dev(t) for t in pools(g, 4, B, H, ps, D, torch.float32))
    gx = dev(x)
    oq = mk.fused_qk_norm_rope_paged(gx[:, :, :H], gx[:, :, H:2 * H], gx[:, :, 2 * H:], None, dev(cos), dev(sin), kp,
                                     vp, dev(table), dev(start))
    within(oq, *R.norm_rope(x[:, :, :H], None, cos, sin, pos, 1e-6, False))


@pytest.mark.parametrize("D", [64, 20])
def test_rope_paged_same_slot_keeps_the_later_token(mk, D):
    """A table whose columns alias one page (a -1 column is page P - 1): the
    later token of the call stays, as in paged_kv_write."""
    g = torch.Generator().manual_seed(3)
    B, S, H, ps, P = 1, 50, 2, 8, 4
    table = torch.tensor([[-1, 3, 0, 1] * 16])[:, :60].to(torch.int32).contiguous()  # odd columns of period 4
    cos, sin = angles(80, D)
    x = randn(g, B, S, 3 * H, D, dtype=torch.bfloat16)
    kp0, vp0 = pools(g, P, B, H, ps, D, torch.bfloat16)
    for count in (S, 21):
        kp, vp = dev(kp0), dev(vp0)
        gx = dev(x)
        mk.fused_qk_norm_rope_paged(gx[:, :, :H], gx[:, :, H:2 * H], gx[:, :, 2 * H:], None, dev(cos), dev(sin), kp,
                                    vp, dev(table), torch.tensor([2]).cuda(), count=torch.tensor([count]).cuda())
        want = vp0.clone()
        for s in range(count):
            want[int(table[0, 2 + s]), 0, :, (2 + s) % ps] = x[0, s, 2 * H:]
        assert torch.equal(vp.cpu(), want)


def test_rope_bad_positions_are_recorded(mk):
    g = torch.Generator().manual_seed(3)
    B, S, H, D, ps = 1, 4, 1, 64, 16
    cos, sin = (dev(t) for t in angles(10, D))
    x = dev(randn(g, B, S, 3 * H, D, dtype=torch.bfloat16))
    q, k, v = x[:, :, :1], x[:, :, 1:2], x[:, :, 2:]
    pos = torch.tensor([[0, 10, -1, 9]]).cuda()
    oq, ok = mk.fused_qk_norm_rope(q, k, pos, cos, sin)
    assert status() == 7
    assert not oq[0, 1:3].any() and not ok[0, :, 1:3].any() and oq[0, 0].any() and oq[0, 3].any()
    kp0, vp0 = pools(g, 2, B, H, ps, D, torch.bfloat16)
    kp, vp = dev(kp0), dev(vp0)
    table = torch.tensor([[0, 0, 5, 1]], dtype=torch.int32).cuda()  # page 5 is outside; the table ends at 4
    mk.fused_qk_norm_rope_paged(q, k, v, torch.zeros_like(pos), cos, sin, kp, vp, table, torch.tensor([1]).cuda())
    assert status() == 7
    want = vp0.clone()
    want[0, 0, 0, 1], want[1, 0, 0, 3] = v[0, 0, 0].cpu(), v[0, 2, 0].cpu()
    assert torch.equal(vp.cpu(), want)


# --------------------------------------------------------------------------- #
# eviction
# --------------------------------------------------------------------------- #
EVICT = [
    # B, Hkv, D, ps, lens, budget, sinks, recent, dtype, ties
    (1, 1, 64, 16, [1], 1, 0, 0, torch.bfloat16, False),
    (2, 2, 128, 16, [40, 10], 20, 2, 5, torch.bfloat16, False),
    (3, 2, 64, 16, [100, 0, 33], 32, 0, 0, torch.float16, True),
    (2, 3, 80, 24, [257, 500], 100, 4, 96, torch.float32, True),  # nothing but the ends
    (2, 1, 20, 16, [90, 64], 64, 1, 3, torch.bfloat16, True),  # rows of 40 bytes
    (2, 1, 9, 16, [90, 64], 10, 1, 3, torch.float16, False),
    (1, 2, 128, 16, [9000], 4100, 4, 64, torch.bfloat16, True),  # two numbering steps
    (1, 1, 64, 16, [17000], 16999, 0, 0, torch.bfloat16, False),  # one token goes
    (20, 4, 128, 32, list(range(10, 410, 20)), 130, 3, 20, torch.bfloat16, False),
    (2, 1, 64, 16, [30, 12], 0, 0, 0, torch.bfloat16, False),  # everything goes
]


@pytest.mark.parametrize("B,Hkv,D,ps,lens,budget,sinks,recent,dtype,ties", EVICT)
def test_evict(mk, B, Hkv, D, ps, lens, budget, sinks, recent, dtype, ties):
    g = torch.Generator().manual_seed(budget + D)
    L = max(lens) + 3
    P = -(-L // ps) + 2
    table = R.make_table(B, L, P, ps, 3)
    kp0, vp0 = pools(g, P, B, Hkv, ps, D, dtype)
    w0 = torch.rand(B, Hkv, L + 1, generator=g) - 0.2
    if ties:
        w0 = (w0 * 4).round() / 4  # exact ties, zeros of both signs
        w0 = torch.where((w0 == 0) & (torch.rand(w0.shape, generator=g) < 0.5), torch.full_like(w0, -0.0), w0)
        w0[:, :, 5::11] = float("nan")
        w0[:, :, 7::13] = float("inf")
        w0[:, :, 3::17] = -float("inf")
    kp, vp, w = dev(kp0), dev(vp0), dev(w0)
    kept, new_lens = mk.paged_kv_evict(kp, vp, dev(table), dev(torch.tensor(lens)), w, budget, sinks=sinks,
                                       recent=recent)
    want = R.evict(lens, w0, budget, sinks, recent)
    wk, wv, ww = kp0.clone(), vp0.clone(), w0.clone()
    for b in range(B):
        for h in range(Hkv):
            src = torch.tensor(want[b][h], dtype=torch.long)
            got = kept[b, h].cpu().tolist()
            assert got == want[b][h] + [-1] * (budget - len(want[b][h])), (b, h)
            to = torch.arange(len(src))
            for new, old in ((wk, kp0), (wv, vp0)):
                new[table[b, to].long(), b, h, to % ps] = old[table[b, src].long(), b, h, src % ps]
            if lens[b] > budget:
                ww[b, h, :len(src)] = w0[b, h, src]
                ww[b, h, len(src):lens[b]] = 0
    assert new_lens.cpu().tolist() == [min(n, budget) for n in lens]
    assert torch.equal(kp.cpu(), wk) and torch.equal(vp.cpu(), wv)
    assert torch.equal(w.cpu().view(torch.int32), ww.view(torch.int32))


def test_evict_bad_pages_are_recorded(mk):
    """A page id outside the pool: that row is skipped, the others move."""
    kp = torch.arange(4 * 16, dtype=torch.float32).view(4, 1, 1, 16, 1).cuda()
    vp = kp.clone()
    table = (torch.arange(64) // 16).view(1, 64).to(torch.int32)
    table[0, 40] = 7
    w = torch.zeros(1, 1, 64)
    w[0, 0, 40] = 5.0
    kept, _ = mk.paged_kv_evict(kp, vp, dev(table), torch.tensor([64]).cuda(), dev(w), 10, recent=4)
    assert status() == 7
    assert kept[0, 0].tolist() == [0, 1, 2, 3, 4, 40, 60, 61, 62, 63]
    assert kp.view(-1)[:10].tolist() == [0, 1, 2, 3, 4, 5, 60, 61, 62, 63]


# --------------------------------------------------------------------------- #
# together
# --------------------------------------------------------------------------- #
def test_server_with_a_bounded_cache(mk):
    """Two ragged prompts, decode steps that keep the totals, an eviction, more
    decode steps: against the same steps in 64 bits on lists of keys."""
    g = torch.Generator().manual_seed(11)
    B, Hq, Hkv, D, ps, S = 2, 8, 2, 64, 16, 90
    G = Hq // Hkv
    dt = torch.bfloat16
    n0, budget, steps = [90, 47], 40, 3
    L = 100
    P = -(-L // ps) + 1
    table = R.make_table(B, L, P, ps, 5)
    cos, sin = angles(200, D)
    qw, kw = 1 + 0.1 * torch.randn(D, generator=g), 1 + 0.1 * torch.randn(D, generator=g)
    kp, vp = (dev(torch.full((P, B, Hkv, ps, D), float("nan"), dtype=dt)) for _ in range(2))
    totals = torch.zeros(B, Hkv, L).cuda()
    dtab, dcos, dsin, dqw, dkw = dev(table), dev(cos), dev(sin), dev(qw), dev(kw)

    def cached(lens):
        """what the cache holds, head by head (its own rounded keys and values)"""
        K, V = kp.cpu(), vp.cpu()
        return [[(R.gather(K, table, b, h, torch.arange(lens[b]), ps), R.gather(V, table, b, h, torch.arange(lens[b]),
                                                                                  ps)) for h in range(Hkv)]
                for b in range(B)]

    # prompts
    x = randn(g, B, S, Hq + 2 * Hkv, D, dtype=dt)
    gx = dev(x)
    new = torch.tensor(n0, dtype=torch.int32)
    q = mk.fused_qk_norm_rope_paged(gx[:, :, :Hq], gx[:, :, Hq:Hq + Hkv], gx[:, :, Hq + Hkv:], None, dcos, dsin, kp,
                                    vp, dtab, torch.zeros(B, dtype=torch.int32).cuda(), dqw, dkw, count=dev(new))
    pos = torch.arange(S).expand(B, S)
    rk, tk = R.norm_rope(x[:, :, Hq:Hq + Hkv], kw, cos, sin, pos, 1e-6, False)
    for b, heads in enumerate(cached(n0)):
        for h, (K, V) in enumerate(heads):
            assert ((K - rk[b, :n0[b], h]).abs() <= tk[b, :n0[b], h]).all()
            assert torch.equal(V, x[b, :n0[b], Hq + Hkv + h].double())
    out = mk.fused_paged_prompt_attention(q, kp, vp, dtab, dev(new), dev(new), window=32, sinks=4)
    ref, tol, _, _ = R.attention(q.cpu(), kp.cpu(), vp.cpu(), table, n0, n0, 32, 4)
    within(out, ref, tol)

    # decode, eviction, decode
    lens, true_pos = list(n0), list(n0)
    kept_before = None
    for step in range(2 * steps):
        if step == steps:
            before, w0 = cached(lens), totals.cpu().clone()
            kept, nl = mk.paged_kv_evict(kp, vp, dtab, torch.tensor(lens).cuda(), totals, budget, sinks=2, recent=8)
            want = R.evict(lens, w0, budget, 2, 8)
            lens = [min(n, budget) for n in lens]
            assert nl.cpu().tolist() == lens
            after = cached(lens)
            for b in range(B):
                for h in range(Hkv):
                    assert kept[b, h].cpu().tolist() == want[b][h]
                    for x0, x1 in zip(before[b][h], after[b][h]):
                        assert torch.equal(x0[want[b][h]], x1)
            kept_before = lens
        y = randn(g, B, 1, Hq + 2 * Hkv, D, dtype=dt)
        gy = dev(y)
        start = torch.tensor(lens, dtype=torch.int32)
        pos = torch.tensor(true_pos)[:, None]
        q = mk.fused_qk_norm_rope_paged(gy[:, :, :Hq], gy[:, :, Hq:Hq + Hkv], gy[:, :, Hq + Hkv:], dev(pos), dcos,
                                        dsin, kp, vp, dtab, dev(start), dqw, dkw)
        within(q, *R.norm_rope(y[:, :, :Hq], qw, cos, sin, pos, 1e-6, False))
        lens, true_pos = [n + 1 for n in lens], [n + 1 for n in true_pos]
        w0 = totals.cpu().double()
        out = mk.fused_paged_decode_attention(q[:, 0], kp, vp, dtab, torch.tensor(lens).cuda(), key_weights=totals)
        ref, tol, w, wtol = R.attention(q.cpu(), kp.cpu(), vp.cpu(), table, lens, [1] * B, None, 0)
        within(out, ref[:, 0], tol[:, 0])
        within(totals, w0 + w, wtol + (w0 + w) * 2.0 ** -23)
    assert kept_before == [budget, budget]
    # every decode step handed out G of weight per key head
    assert math.isclose(float(w.sum()), B * Hkv * G, rel_tol=1e-9)


def test_capture_replay_and_streams(mk):
    """All of them in one captured graph, replayed on another stream after the
    inputs changed, equal to the eager calls; two graphs replayed at the same
    time on two streams do not meet in a workspace."""
    g = torch.Generator().manual_seed(2)
    B, S, Hq, Hkv, D, ps, L = 2, 33, 8, 2, 128, 16, 400
    P = -(-L // ps)
    table = dev(R.make_table(B, L, P, ps, 5))
    cos, sin = (dev(t) for t in angles(L, D))

    def state(seed):
        h = torch.Generator().manual_seed(seed)
        return dict(x=dev(randn(h, B, S, Hq + 2 * Hkv, D, dtype=torch.bfloat16)),
                    kp=dev(randn(h, P, B, Hkv, ps, D, dtype=torch.bfloat16)),
                    vp=dev(randn(h, P, B, Hkv, ps, D, dtype=torch.bfloat16)),
                    w=dev(torch.rand(B, Hkv, L, generator=h)),
                    start=torch.tensor([300, 61], dtype=torch.int32).cuda())

    def step(s):
        x, lens = s["x"], s["start"] + S
        q = mk.fused_qk_norm_rope_paged(x[:, :, :Hq], x[:, :, Hq:Hq + Hkv], x[:, :, Hq + Hkv:], None, cos, sin,
                                        s["kp"], s["vp"], table, s["start"])
        a = mk.fused_paged_prompt_attention(q, s["kp"], s["vp"], table, lens, window=90, sinks=3)
        d = mk.fused_paged_decode_attention(q[:, -1], s["kp"], s["vp"], table, lens, key_weights=s["w"])
        kept, nl = mk.paged_kv_evict(s["kp"], s["vp"], table, lens, s["w"], 70, sinks=2, recent=9)
        return q, a, d, kept, nl

    def copy(dst, src):
        for k in dst:
            dst[k].copy_(src[k])

    want = []
    for seed in (1, 2):
        s = state(seed)
        want.append([t.clone() for t in step(s)] + [s["kp"].clone(), s["vp"].clone(), s["w"].clone()])
    torch.cuda.synchronize()
    graphs, states, outs = [], [], []
    for _ in range(2):
        s = state(9)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = step(s)
        graphs.append(graph), states.append(s), outs.append(o)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for i in range(2):
            copy(states[i], state(1 + i))
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            got = list(outs[i]) + [states[i]["kp"], states[i]["vp"], states[i]["w"]]
            for a, b in zip(got, want[i]):
                assert torch.equal(a, b)


def test_side_stream(mk):
    """A call on a side stream runs there, behind what that stream already holds."""
    g = torch.Generator().manual_seed(2)
    B, Hq, Hkv, D, ps, L = 2, 4, 2, 128, 16, 200
    table = dev(R.make_table(B, L, 13, ps, 5))
    kp, vp = (dev(x) for x in pools(g, 13, B, Hkv, ps, D, torch.bfloat16))
    q0 = dev(randn(g, B, Hq, D, dtype=torch.bfloat16))
    lens = torch.tensor([200, 77]).cuda()
    want = mk.fused_paged_decode_attention(q0, kp, vp, table, lens)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        q = torch.zeros_like(q0)
        big = torch.randn(4000, 4000, device="cuda")
        for _ in range(10):
            big = big @ big * 1e-4
        q.copy_(q0)
        out = mk.fused_paged_decode_attention(q, kp, vp, table, lens)
    st.synchronize()
    assert torch.equal(out, want)


def test_offsets_past_32_bits(mk):
    """Pools of more than 2^31 elements: pages behind that mark give the same
    bits as the same pages in a small pool."""
    B, Hq, Hkv, D, ps, S, n = 1, 4, 1, 128, 16, 40, 300
    dt = torch.bfloat16
    used = -(-n // ps)
    big = (1 << 31) // (ps * D) + used + 8
    if torch.cuda.mem_get_info()[0] < 3 * big * ps * D * 2:
        pytest.skip("not enough memory")
    g = torch.Generator().manual_seed(6)
    small = [dev(x) for x in pools(g, used, B, Hkv, ps, D, dt)]
    order = torch.randperm(used, generator=g)
    small_table = order[torch.arange(n) // ps][None].to(torch.int32)
    huge = [torch.empty(big, B, Hkv, ps, D, dtype=dt, device="cuda") for _ in range(2)]
    for a, b in zip(huge, small):
        a[big - used:] = b
    x = dev(randn(g, B, S, Hq + 2 * Hkv, D, dtype=dt))
    cos, sin = (dev(t) for t in angles(n, D))
    lens, new = torch.tensor([n]).cuda(), torch.tensor([S]).cuda()
    results = []
    for (kp, vp), table in ((small, dev(small_table)), (huge, dev(small_table + (big - used)))):
        w = torch.linspace(0, 1, n).view(1, 1, n).cuda().contiguous()
        q = mk.fused_qk_norm_rope_paged(x[:, :, :Hq], x[:, :, Hq:Hq + Hkv], x[:, :, Hq + Hkv:], None, cos, sin, kp, vp,
                                        table, lens - S)
        a = mk.fused_paged_prompt_attention(q, kp, vp, table, lens, new)
        d = mk.fused_paged_decode_attention(q[:, -1], kp, vp, table, lens, key_weights=w)
        kept, _ = mk.paged_kv_evict(kp, vp, table, lens, w, 100, sinks=3, recent=10)
        results.append((q, a, d, w, kept, kp[-used:], vp[-used:]))
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_rows_of_a_batch_do_not_depend_on_it(mk):
    """A sequence gives the same bits of queries and caches alone and in a
    padded batch, and the same attention up to the joins' order."""
    g = torch.Generator().manual_seed(9)
    B, S, Hq, Hkv, D, ps = 3, 150, 8, 2, 128, 16
    lens, new = [150, 400, 9], [150, 30, 9]
    L = 400
    P = L // ps
    table = R.make_table(B, L, P, ps, 5)
    kp, vp = (dev(x) for x in pools(g, P, B, Hkv, ps, D, torch.bfloat16))
    q = dev(randn(g, B, S, Hq, D, dtype=torch.bfloat16))
    out = mk.fused_paged_prompt_attention(q, kp, vp, dev(table), torch.tensor(lens).cuda(), torch.tensor(new).cuda())
    for b in range(B):
        one = mk.fused_paged_prompt_attention(q[b:b + 1, :new[b]], kp[:, b:b + 1], vp[:, b:b + 1], dev(table[b:b + 1]),
                                              torch.tensor(lens[b:b + 1]).cuda())
        # either is within half a step of the output and half a step of every weight; |v| < 6
        assert (one[0].double() - out[b, :new[b]].double()).abs().max() <= 4 * 2.0 ** -8 * 6
        assert not out[b, new[b]:].any()


def test_two_streams_at_once(mk):
    """Calls that overlap on two streams do not meet in scratch memory."""
    g = torch.Generator().manual_seed(3)
    B, Hq, Hkv, D, ps, n = 1, 8, 2, 128, 16, 3000
    P = -(-n // ps)
    table, lens = dev(R.make_table(B, n, P, ps, 5)), torch.tensor([n]).cuda()
    data = []
    for _ in range(2):
        kp, vp = (dev(x) for x in pools(g, P, B, Hkv, ps, D, torch.bfloat16))
        data.append((dev(randn(g, B, Hq, D, dtype=torch.bfloat16)), dev(randn(g, B, 50, Hq, D, dtype=torch.bfloat16)),
                     kp, vp))
    call = lambda q, p, kp, vp: (mk.fused_paged_decode_attention(q, kp, vp, table, lens),
                                 mk.fused_paged_prompt_attention(p, kp, vp, table, lens))
    want = [call(*d) for d in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(call(*data[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for pair in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(pair, want[i]))


def test_empty_calls(mk):
    z = torch.zeros
    kp = z(2, 0, 1, 16, 64, dtype=torch.bfloat16).cuda()
    t0, l0 = z(0, 4, dtype=torch.int32).cuda(), z(0, dtype=torch.int32).cuda()
    assert mk.fused_paged_decode_attention(z(0, 2, 64, dtype=torch.bfloat16).cuda(), kp, kp, t0, l0).shape == (0, 2, 64)
    assert mk.fused_paged_prompt_attention(z(0, 3, 2, 64, dtype=torch.bfloat16).cuda(), kp, kp, t0, l0).numel() == 0
    kept, nl = mk.paged_kv_evict(kp, kp, t0, l0, z(0, 1, 4).cuda(), 3)
    assert kept.shape == (0, 1, 3) and nl.shape == (0,)
    # a cache of no columns: nothing to see
    kp = z(2, 1, 1, 16, 64, dtype=torch.bfloat16).cuda()
    t0, l0 = z(1, 0, dtype=torch.int32).cuda(), z(1, dtype=torch.int32).cuda()
    out = mk.fused_paged_decode_attention(torch.ones(1, 2, 64, dtype=torch.bfloat16).cuda(), kp, kp, t0, l0)
    assert not out.any()
    out = mk.fused_paged_prompt_attention(torch.ones(1, 40, 2, 64, dtype=torch.bfloat16).cuda(), kp, kp, t0, l0, l0)
    assert out.shape == (1, 40, 2, 64) and not out.any()
    cos, sin = (dev(t) for t in angles(4, 64))
    q, k = mk.fused_qk_norm_rope(z(1, 0, 2, 64).cuda(), z(1, 0, 1, 64).cuda(), z(1, 0, dtype=torch.int32).cuda(), cos,
                                 sin)
    assert q.shape == (1, 0, 2, 64) and k.shape == (1, 1, 0, 64)
