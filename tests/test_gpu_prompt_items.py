"""The tensor-core prompt kernel over more items than the GPU has SMs: every
block goes from item to item (rings, barrier phases, the queries' buffer and
the accumulators run on), in ragged batches with empty sequences, whole and in
pieces, for each head size and type that it is built for.  All rows are held
to 64 bits; the bound is that of tests/paged_reference.py."""

import math

import pytest
import torch

import paged_reference as R
from test_gpu_paged_serving import clean_status, dev, mk, pools, randn, wipe_unused, within  # noqa: F401

pytestmark = pytest.mark.gpu


def reference(q, kp, vp, table, lens, new, window, sinks):
    """R.attention for every row at once, a (sequence, key head) at a time."""
    B, S, Hq, D = q.shape
    Hkv, ps = kp.shape[2], kp.shape[3]
    G, dt, scale = Hq // Hkv, q.dtype, 1.0 / math.sqrt(D)
    out = torch.zeros(B, S, Hq, D, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for b in range(B):
        if new[b] == 0:
            continue
        j = torch.arange(lens[b])
        p = torch.arange(lens[b] - new[b], lens[b])
        seen = j <= p[:, None]
        if window:
            seen &= (j > p[:, None] - window) | (j < sinks)
        used = seen.any(0)
        seen, rows = seen[:, used].cuda(), j[used]
        for h in range(Hkv):
            K, V = (R.gather(x, table, b, h, rows, ps).cuda() for x in (kp, vp))
            x = q[b, :new[b], h * G:(h + 1) * G].double().cuda()  # [n, G, D]
            score = (x @ K.T * scale).masked_fill(~seen[:, None], -math.inf)
            smag = (x.abs() @ K.abs().T * scale).masked_fill(~seen[:, None], 0).amax(-1, keepdim=True)
            w = score.softmax(-1)
            o, mag, n = w @ V, w @ V.abs(), seen.sum(-1)[:, None, None]
            rel = 2 * (D + 4) * 2.0 ** -24 * smag + (n + 8) * 2.0 ** -23
            t = R.HALF[dt] * o.abs() + mag * (R.HALF[dt] + rel)
            if dt == torch.float16:
                t = t + 2.0 ** -25 + n * 2.0 ** -25 * V.abs().amax(0)
            out[b, :new[b], h * G:(h + 1) * G] = o.cpu()
            tol[b, :new[b], h * G:(h + 1) * G] = (1.01 * t + 1e-30).cpu()
    return out, tol


# B, S, Hq, Hkv, D, ps, most cached, window, sinks, dtype, per_token, least items
ITEMS = [
    (40, 200, 8, 2, 128, 16, 190, None, 0, torch.bfloat16, False, 300),
    (24, 300, 32, 4, 64, 16, 40, None, 0, torch.float16, False, 900),
    (30, 260, 8, 4, 80, 32, 150, 100, 5, torch.float16, False, 300),
    (20, 150, 14, 2, 96, 8, 300, None, 0, torch.bfloat16, True, 200),
    (33, 129, 20, 4, 128, 64, 140, 64, 2, torch.float16, False, 300),
    (28, 310, 4, 4, 64, 24, 100, 130, 140, torch.bfloat16, True, 224),
    # long caches behind few rows: pieces
    (6, 100, 16, 4, 128, 16, 3900, None, 0, torch.float16, False, 48),
    (8, 90, 20, 4, 64, 16, 2500, 1500, 4, torch.bfloat16, False, 64),
    (5, 70, 14, 2, 80, 16, 3000, None, 0, torch.bfloat16, True, 20),
]


@pytest.mark.parametrize("B,S,Hq,Hkv,D,ps,most,window,sinks,dtype,per_token,items", ITEMS)
def test_many_items(mk, B, S, Hq, Hkv, D, ps, most, window, sinks, dtype, per_token, items):
    import _mtp_native as N
    g = torch.Generator().manual_seed(B * 100 + D)
    tpt = 128 // (Hq // Hkv)
    assert B * Hkv * -(-S // (2 * tpt)) >= items
    # full, empty and single-row sequences, and ends at and around the tiles' borders
    ends = [S, 0, 1, S - 1, tpt, tpt + 1, 2 * tpt, 2 * tpt + 1, S // 2]
    new = [min(S, ends[b % len(ends)]) for b in range(B)]
    past = [(most * ((b * 7) % 11)) // 10 if b % 5 else 0 for b in range(B)]
    past[-1] = most
    lens = [a + b for a, b in zip(past, new)]
    L = max(lens)
    P = -(-L // ps) + 2
    table = R.make_table(B, L, P, ps, 7, per_token)
    kp, vp = pools(g, P, B, Hkv, ps, D, dtype)
    q = randn(g, B, S, Hq, D, dtype=dtype, scale=1.5)
    for b in range(B):
        q[b, new[b]:] = float("nan")
    low = [(max(0, p - window + 1), sinks) for p in past] if window else None
    used = [n if m else 0 for n, m in zip(lens, new)]
    kn, vn = wipe_unused(kp, table, used, ps, low), wipe_unused(vp, table, used, ps, low)
    args = (dev(q), dev(kn), dev(vn))
    t32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    ref, tol = reference(q, kp, vp, table, lens, new, window, sinks)
    pieces = []
    for wide in (0, 30000):  # a table as wide as the longest sequence, and a wide one: other pieces
        tab = torch.nn.functional.pad(table, (0, wide), value=1 << 30)  # ids that no position may use
        pieces.append(N.lib().mtp_paged_window_attention_workspace(B, S, Hq, Hkv, D, L + wide, window or 0, sinks,
                                                                   N.dtype_code(q), 0) > 256)
        out = mk.fused_paged_prompt_attention(*args, dev(tab), t32(lens), t32(new), window=window, sinks=sinks)
        within(out, ref, tol)
        for _ in range(2):
            assert torch.equal(out, mk.fused_paged_prompt_attention(*args, dev(tab), t32(lens), t32(new),
                                                                    window=window, sinks=sinks))
    assert pieces[0] == (most > 2000)
