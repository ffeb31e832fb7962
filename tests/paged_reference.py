"""64-bit restatement of the paged-cache serving operators (query/key norm with
rotation, windowed attention over the cache, eviction) and the error bounds
their GPU results are held to.  Test infrastructure: plain loops on the CPU."""

import math

import torch

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step, relative


def make_table(B, L, P, ps, seed, per_token=False):
    """[B, L] int32: every sequence's pages in an order of its own; per_token
    shifts them so that no page slot of the table lies in one page."""
    g = torch.Generator().manual_seed(seed)
    rows = []
    for _ in range(B):
        order = torch.randperm(P, generator=g)
        t = torch.arange(L)
        rows.append(order[(t + (ps // 2 if per_token else 0)) // ps % P])
    return torch.stack(rows).to(torch.int32)


def gather(pages, table, b, h, j, ps):
    """Rows of key head h at positions j (int64 tensor), in 64 bits."""
    return pages[table[b, j].long(), b, h, j % ps].double()


def attention(q, k_pages, v_pages, table, lens, n_new, window, sinks, scale=None):
    """q [B,S,Hq,D] -> (out, bound) in 64 bits, and the per-key weights
    [B,Hkv,L] of the last row with their bound.  Bound of an output: half a step of
    its type; the weights' rounding to the type of V (16-bit types), half a
    step of each product p v; the error of a score, at most (D + 4) fp32
    roundings of its products, moves a weight by twice that, and a sum of n
    terms and the exponential cost another n + 8 roundings."""
    B, S, Hq, D = q.shape
    _, _, Hkv, ps, _ = k_pages.shape
    L = table.shape[1]
    G = Hq // Hkv
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    dt = q.dtype
    out = torch.zeros(B, S, Hq, D, dtype=torch.float64)
    tol = torch.zeros_like(out)
    weights = torch.zeros(B, Hkv, L, dtype=torch.float64)
    wtol = torch.zeros_like(weights)
    qd = q.double()
    for b in range(B):
        for s in range(n_new[b]):
            p = lens[b] - n_new[b] + s
            j = torch.arange(p + 1)
            if window:
                j = j[(j > p - window) | (j < sinks)]
            for h in range(Hkv):
                K, V = gather(k_pages, table, b, h, j, ps), gather(v_pages, table, b, h, j, ps)
                for g in range(h * G, h * G + G):
                    x = K @ qd[b, s, g] * scale
                    smag = float((K.abs() @ qd[b, s, g].abs()).max() * abs(scale))
                    w = torch.softmax(x, 0)
                    o, mag = w @ V, w @ V.abs()
                    out[b, s, g] = o
                    rel = 2 * (D + 4) * 2.0 ** -24 * smag + (len(j) + 8) * 2.0 ** -23
                    up = HALF[dt] if dt != torch.float32 else 0.0
                    t = HALF[dt] * o.abs() + mag * (up + rel)
                    if dt == torch.float16:  # outputs and weights below f16's normal range
                        t = t + 2.0 ** -25 + len(j) * 2.0 ** -25 * V.abs().max(0).values
                    tol[b, s, g] = 1.01 * t + 1e-30
                    if s == n_new[b] - 1:
                        weights[b, h, j] += w
                        wtol[b, h, j] += w * (rel + 2.0 ** -20) + 1e-30
    return out, tol, weights, wtol


def norm_rope(x, w, cos, sin, pos, eps, interleaved):
    """x [B,S,H,D], pos [B,S] -> (values, bound) in 64 bits: half a step of the
    type, and D / 2 + 10 fp32 roundings of the two terms of a turned value."""
    B, S, H, D = x.shape
    half = cos.shape[1]
    y = x.double()
    if eps is not None:
        y = y / (y.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    if w is not None:
        y = y * w.double()
    c, s = cos.double()[pos.long()][:, :, None], sin.double()[pos.long()][:, :, None]
    i = torch.arange(half)
    ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    out, mag = y.clone(), y.abs()
    a, b = y[..., ia], y[..., ib]
    out[..., ia], out[..., ib] = a * c - b * s, b * c + a * s
    mag[..., ia], mag[..., ib] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    tol = HALF[x.dtype] * out.abs() + mag * (D / 2 + 10) * 2.0 ** -24
    if x.dtype == torch.float16:
        tol = tol + 2.0 ** -25
    return out, 1.01 * tol + 1e-30


def evict(lens, weights, budget, sinks, recent):
    """kept [B][Hkv] lists of positions."""
    B, H, _ = weights.shape
    kept = []
    for b in range(B):
        kept.append([])
        for h in range(H):
            n = lens[b]
            if n <= budget:
                kept[b].append(list(range(n)))
                continue
            ends = set(range(sinks)) | set(range(n - recent, n))
            w = [(-math.inf if math.isnan(x) else x) for x in weights[b, h, :n].tolist()]
            nan = [math.isnan(x) for x in weights[b, h, :n].tolist()]
            middle = [j for j in range(n) if j not in ends]
            middle.sort(key=lambda j: (-w[j], nan[j], j))
            kept[b].append(sorted(ends | set(middle[:budget - len(ends)])))
    return kept
