"""Cases, plain forms and exact values of the paged-cache serving operators of
``mtp_kernels``:

  rope     fused_qk_norm_rope / fused_qk_norm_rope_paged: RMSNorm of every
           query and key head, the position rotation, and (paged) the write of
           the keys and values into the page pool, in one pass
  prompt   fused_paged_prompt_attention: causal attention of new tokens over a
           paged cache, with a sliding window and first tokens that stay visible
  decode   fused_paged_decode_attention: attention of one new token per
           sequence, ragged lengths, optionally adding every key's attention
           weight to a running total
  evict    paged_kv_evict: keep the first, the last and the heaviest tokens of
           every (sequence, key head) and close the gaps in the pool

A case is a dict of plain values; ``prepare`` builds its tensors from a seed,
``run`` makes one pass (``own``: through the framework, else in elementary
torch operations in 32 bits), ``exact`` gives the result in 64 bits.
"""

import math
import os
import sys

import numpy as np
import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}
_BASE = 500000.0  # base of the rotation's frequencies
_EPS = 1e-5


# --------------------------------------------------------------------------- #
# cases
# --------------------------------------------------------------------------- #
def _rope(name, **kw):
    c = dict(name=name, kind="rope", B=1, S=1, new_min=1, past=0, Hq=32, Hkv=8, D=128, rot=128, interleaved=False,
             paged=True, ps=16, dtype="bf16")
    c.update(kw)
    return c


def _prompt(name, **kw):
    c = dict(name=name, kind="prompt", B=1, S=64, new_min=64, past_min=0, past_max=0, Hq=32, Hkv=8, D=128, ps=16,
             window=0, sinks=0, dtype="bf16")
    c.update(kw)
    return c


def _decode(name, **kw):
    c = dict(name=name, kind="decode", B=1, len_min=1, len_max=4096, Hq=32, Hkv=8, D=128, ps=16, window=0, sinks=0,
             weights=False, dtype="bf16")
    c.update(kw)
    return c


def _evict(name, **kw):
    c = dict(name=name, kind="evict", B=1, len_min=1, len_max=2048, budget=1024, sinks=4, recent=64, Hkv=8, D=128,
             ps=16, dtype="bf16")
    c.update(kw)
    return c


def listed():
    return [
        # one generated token for each of 16 sequences with 4096 tokens behind it: latency
        _rope("rope, one token each", B=16, S=1, new_min=1, past=4095),
        # the 64 nodes of a draft tree, half of each head rotated, pairs side by side; nothing enters the cache yet
        _rope("rope, draft tree", B=16, S=64, new_min=64, past=4096, rot=64, interleaved=True, paged=False,
              dtype="f16"),
        # four ragged prompts into an empty cache: bandwidth
        _rope("rope, prompts", B=4, S=4093, new_min=2500),
        # short turns of a conversation, 7 query heads to a key head, small heads: latency
        _prompt("prompt, short turns", B=3, S=77, new_min=1, past_min=100, past_max=500, Hq=14, Hkv=2, D=64,
                dtype="f16"),
        # a 512-token piece of a prompt behind 32,000 cached tokens: few rows against a long axis
        _prompt("prompt, piece of a long one", S=512, new_min=512, past_min=32000, past_max=32000),
        # two prompts through a layer that sees 1024 tokens back and the first four
        _prompt("prompt, window", B=2, S=5501, new_min=2750, window=1024, sinks=4),
        # one prompt of 8192 tokens through a layer that sees everything: matrix-product bound
        _prompt("prompt, causal", S=8192, new_min=8192),
        # one conversation: latency, few (sequence, head) pairs
        _decode("decode, one sequence", len_min=4096, len_max=4096),
        # a served batch with lengths from 1 to 32,768: bandwidth and balance
        _decode("decode, ragged batch", B=16, len_max=32768),
        # the same with 5 query heads to a key head, keeping the totals that an eviction goes by
        _decode("decode, with key weights", B=8, len_min=9001, len_max=16000, Hq=40, Hkv=8, weights=True, dtype="f16"),
        # one conversation cut from 2048 to 1024 tokens: latency
        _evict("evict, one sequence", len_min=2048, len_max=2048),
        # a served batch cut to half; the shortest sequences stay as they are
        _evict("evict, batch", B=16, len_min=2000, len_max=8192, budget=4096, recent=512),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "prompt", "decode", "evict"])
    Hkv = rng.choice([1, 2, 4, 8])
    G = rng.choice([1, 2, 4, 5, 7, 8])
    D = rng.choice([64, 80, 96, 128])
    ps = rng.choice([8, 16, 32, 64])
    d16 = rng.choice(["bf16", "f16"])
    any_type = rng.choice(["bf16", "f16", "f32"])
    window, sinks = rng.choice([(0, 0), (_log(rng, 64, 4096), rng.randrange(0, 9))])
    if kind == "rope":
        while True:
            B, S = _log(rng, 1, 64), _log(rng, 1, 4096)
            # no more than the listed prompts move
            if B * S * Hkv * (G + 2) * D * _SIZE[any_type] <= 4 * 4093 * 48 * 128 * 2:
                break
        c = _rope("", B=B, S=S, new_min=rng.randint(1, S), past=_log(rng, 1, 4096), Hq=Hkv * G, Hkv=Hkv, D=D,
                  rot=rng.choice([D, D // 2]), interleaved=rng.random() < 0.3, paged=rng.random() < 0.7, ps=ps,
                  dtype=any_type)
    elif kind == "prompt":
        while True:
            B, S, past = _log(rng, 1, 16), _log(rng, 1, 8192), rng.choice([0, _log(rng, 1, 16384)])
            if B * S * (past + S) * Hkv * G * D <= 8192 * 8192 * 32 * 128 // 2:
                break
        c = _prompt("", B=B, S=S, new_min=rng.randint(1, S), past_min=past // 2, past_max=past, Hq=Hkv * G, Hkv=Hkv,
                    D=D, ps=ps, window=window, sinks=sinks, dtype=d16)
    elif kind == "decode":
        while True:
            B, n = _log(rng, 1, 64), _log(rng, 1, 32768)
            if B * n * Hkv * D <= 16 * 16384 * 8 * 128:
                break
        c = _decode("", B=B, len_min=rng.randint(0, n), len_max=n, Hq=Hkv * G, Hkv=Hkv, D=D, ps=ps, window=window,
                    sinks=sinks, weights=rng.random() < 0.4, dtype=d16)
    else:
        while True:
            B, n = _log(rng, 1, 64), _log(rng, 64, 16384)
            if B * n * Hkv * D * _SIZE[any_type] <= 16 * 8192 * 8 * 128 * 2:
                break
        budget = rng.randint(n // 4, n)
        s = rng.randrange(0, 9)
        c = _evict("", B=B, len_min=rng.randint(0, n), len_max=n, budget=budget, sinks=s,
                   recent=rng.randint(0, max(0, budget - s) // 2), Hkv=Hkv, D=D, ps=ps, dtype=any_type)
    del c["name"]
    return c


# --------------------------------------------------------------------------- #
# inputs
# --------------------------------------------------------------------------- #
def _spread(lo, hi, n):
    """n lengths from lo to hi, evenly spread: the same sum for every seed."""
    return [int(round(hi - (hi - lo) * i / max(1, n - 1))) for i in range(n)]


def _lens(case):
    """(new, total) tokens of each sequence."""
    k, B = case["kind"], case["B"]
    if k == "rope":
        new = _spread(case["new_min"], case["S"], B)
        return new, [case["past"] + n for n in new]
    if k == "prompt":
        new = _spread(case["new_min"], case["S"], B)
        past = _spread(case["past_min"], case["past_max"], B)[::-1]
        return new, [p + n for p, n in zip(past, new)]
    total = _spread(case["len_min"], case["len_max"], B)
    return [1] * B, total


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _pool(case, g, width, dtype):
    """Page pools and a table that scatters every sequence's pages over them."""
    pages = -(-width // case["ps"]) + 3
    shape = (pages, case["B"], case["Hkv"], case["ps"], case["D"])
    k, v = (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype) for _ in range(2))
    order = torch.rand(case["B"], pages, generator=g, device="cuda").argsort(1)
    token = torch.arange(width, device="cuda") // case["ps"]
    return k, v, order[:, token].to(torch.int32).contiguous()


def prepare(case, seed):
    g = _generator(seed)
    dtype = _TYPES[case["dtype"]]
    B, D, Hkv = case["B"], case["D"], case["Hkv"]
    new, total = _lens(case)
    perm = np.random.RandomState(int(seed) % (1 << 31)).permutation(B)
    st = {"case": dict(case)}
    st["new"] = torch.tensor(np.array(new)[perm], dtype=torch.int32, device="cuda")
    st["lens"] = torch.tensor(np.array(total)[perm], dtype=torch.int32, device="cuda")

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)

    if case["kind"] == "rope":
        S, Hq, R = case["S"], case["Hq"], case["rot"]
        # the projection's output: queries, keys and values side by side
        qkv = (1.5 * randn(B, S, Hq + 2 * Hkv, D)).to(dtype)
        st["q"], st["k"], st["v"] = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hkv], qkv[:, :, Hq + Hkv:]
        st["qw"], st["kw"] = (1.0 + 0.2 * randn(D)).to(dtype), (1.0 + 0.2 * randn(D)).to(dtype)
        width = case["past"] + S
        angle = torch.arange(width, dtype=torch.float64, device="cuda")[:, None] * _BASE ** (
            -torch.arange(0, R, 2, dtype=torch.float64, device="cuda") / R)
        st["cos"], st["sin"] = angle.cos().float(), angle.sin().float()
        st["start"] = torch.full((B,), case["past"], dtype=torch.int32, device="cuda")
        if case["paged"]:
            step = torch.arange(S, device="cuda")
            st["kp"], st["vp"], st["table"] = _pool(case, g, width, dtype)
        else:  # tree nodes: the position is the depth behind the cache
            step = (torch.rand(B, S, generator=g, device="cuda") * min(S, 16)).long().sort(1).values
        st["positions"] = (st["start"][:, None] + step).to(torch.int32)
    elif case["kind"] == "evict":
        st["kp"], st["vp"], st["table"] = _pool(case, g, max(1, case["len_max"]), dtype)
        # totals of attention: a few heavy tokens, many light ones, some that no query looked at
        w = -torch.log(torch.rand(B, Hkv, st["table"].shape[1], generator=g, device="cuda").clamp(min=1e-7)) ** 3
        seen = torch.rand(w.shape, generator=g, device="cuda") > 0.1
        st["w"] = torch.where(seen, w.abs(), torch.zeros_like(w))
    else:
        width = max(1, max(total))
        st["kp"], st["vp"], st["table"] = _pool(case, g, width, dtype)
        shape = (B, case["Hq"], D) if case["kind"] == "decode" else (B, case["S"], case["Hq"], D)
        st["q"] = (1.5 * randn(*shape)).to(dtype)
        if case.get("weights"):
            st["w"] = torch.rand(B, Hkv, width, generator=g, device="cuda")
    st["window"] = case.get("window") or None
    return st


# --------------------------------------------------------------------------- #
# one pass
# --------------------------------------------------------------------------- #
def _kernels():
    pkg = os.path.join(_ROOT, "mtp-engine_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import mtp_kernels
    return mtp_kernels


def run(st):
    return (_run_own if own else _run_plain)[st["case"]["kind"]](st)


def _own_rope(st):
    K, c = _kernels(), st["case"]
    if not c["paged"]:
        return K.fused_qk_norm_rope(st["q"], st["k"], st["positions"], st["cos"], st["sin"], st["qw"], st["kw"], _EPS,
                                    interleaved=c["interleaved"])
    q = K.fused_qk_norm_rope_paged(st["q"], st["k"], st["v"], st["positions"], st["cos"], st["sin"], st["kp"],
                                   st["vp"], st["table"], st["start"], st["qw"], st["kw"], _EPS, count=st["new"],
                                   interleaved=c["interleaved"])
    return q, st["kp"], st["vp"]


def _own_prompt(st):
    return _kernels().fused_paged_prompt_attention(st["q"], st["kp"], st["vp"], st["table"], st["lens"], st["new"],
                                                   window=st["window"], sinks=st["case"]["sinks"])


def _own_decode(st):
    out = _kernels().fused_paged_decode_attention(st["q"], st["kp"], st["vp"], st["table"], st["lens"],
                                                  window=st["window"], sinks=st["case"]["sinks"],
                                                  key_weights=st.get("w"))
    return (out, st["w"]) if "w" in st else out


def _own_evict(st):
    c = st["case"]
    kept, lens = _kernels().paged_kv_evict(st["kp"], st["vp"], st["table"], st["lens"], st["w"], c["budget"],
                                           sinks=c["sinks"], recent=c["recent"])
    return kept, lens, st["kp"], st["vp"], st["w"]


def _norm_rotate(x, w, cos, sin, interleaved):
    """[B, S, H, D] in 32 bits: RMSNorm over each head, then the rotation of its first 2 * cos.shape[-1] values."""
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * w.float()
    h = cos.shape[-1]
    cos, sin = cos[:, :, None], sin[:, :, None]
    r, rest = x[..., :2 * h], x[..., 2 * h:]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :h], r[..., h:])
    a, b = a * cos - b * sin, b * cos + a * sin
    r = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((r, rest), -1)


def _plain_rope(st):
    c = st["case"]
    B, S, dtype = c["B"], c["S"], st["q"].dtype
    pos = st["positions"].long()
    cos, sin = st["cos"][pos], st["sin"][pos]
    q = _norm_rotate(st["q"], st["qw"], cos, sin, c["interleaved"]).to(dtype)
    k = _norm_rotate(st["k"], st["kw"], cos, sin, c["interleaved"]).to(dtype)
    if not c["paged"]:
        return q, k.transpose(1, 2).contiguous()
    live = torch.arange(S, device="cuda")[None] < st["new"][:, None]
    slot = st["start"].long()[:, None] + torch.arange(S, device="cuda")
    page, slot = st["table"].gather(1, slot).long(), slot % c["ps"]
    seq = torch.arange(B, device="cuda")[:, None].expand(B, S)
    at = (page, seq, slice(None), slot)
    keep = live[:, :, None, None]
    st["kp"][at] = torch.where(keep, k, st["kp"][at])
    st["vp"][at] = torch.where(keep, st["v"], st["vp"][at])
    return torch.where(keep, q, torch.zeros_like(q)), st["kp"], st["vp"]


def _cached(pages, table, ps):
    """[B, Hkv, L, D] in 32 bits: the cache in the order of its positions."""
    B, L = table.shape
    slot = (torch.arange(L, device="cuda") % ps).expand(B, L)
    seq = torch.arange(B, device="cuda")[:, None].expand(B, L)
    return pages[table.long(), seq, :, slot].permute(0, 2, 1, 3).float()


def _attend(q, k, v, seen):
    """q [B, Hkv, R, D], k, v [B, Hkv, L, D], seen [B, 1, R, L] -> the mix of values and the weights, in 32 bits."""
    p = torch.matmul(q, k.transpose(-1, -2)).mul_(1.0 / math.sqrt(q.shape[-1])).masked_fill_(~seen, -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True).clamp_(min=-1e30)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total > 0, total, torch.ones_like(total)))
    # positions that no query sees may hold anything
    v = torch.where(seen.any(-2)[..., None], v, torch.zeros_like(v))
    return torch.matmul(p, v), p


def _visible(pos, L, window, sinks):
    """pos [B, R] (-1: nothing) -> [B, 1, R, L]."""
    j = torch.arange(L, device="cuda")
    seen = j <= pos[..., None]
    if window:
        seen = seen & ((j > pos[..., None] - window) | (j < sinks))
    return seen[:, None]


def _plain_prompt(st):
    c = st["case"]
    B, S, Hkv, D = c["B"], c["S"], c["Hkv"], c["D"]
    G = c["Hq"] // Hkv
    s = torch.arange(S, device="cuda")
    pos = (st["lens"] - st["new"])[:, None] + s
    pos = torch.where(s < st["new"][:, None], pos, torch.full_like(pos, -1))
    seen = _visible(pos, st["table"].shape[1], st["window"], c["sinks"])
    seen = seen[:, :, None].expand(-1, -1, G, -1, -1).flatten(2, 3)
    q = st["q"].float().view(B, S, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * S, D)
    o, _ = _attend(q, _cached(st["kp"], st["table"], c["ps"]), _cached(st["vp"], st["table"], c["ps"]), seen)
    return o.view(B, Hkv, G, S, D).permute(0, 3, 1, 2, 4).reshape(B, S, c["Hq"], D).to(st["q"].dtype)


def _plain_decode(st):
    c = st["case"]
    B, Hkv, D = c["B"], c["Hkv"], c["D"]
    seen = _visible((st["lens"] - 1)[:, None], st["table"].shape[1], st["window"], c["sinks"])
    q = st["q"].float().view(B, Hkv, c["Hq"] // Hkv, D)
    o, p = _attend(q, _cached(st["kp"], st["table"], c["ps"]), _cached(st["vp"], st["table"], c["ps"]), seen)
    o = o.reshape(B, c["Hq"], D).to(st["q"].dtype)
    if "w" not in st:
        return o
    st["w"].add_(p.sum(2))
    return o, st["w"]


def _plain_evict(st):
    c = st["case"]
    B, Hkv, n, ps = c["B"], c["Hkv"], c["budget"], c["ps"]
    w, table, lens = st["w"], st["table"].long(), st["lens"].long()
    L = w.shape[-1]
    j = torch.arange(L, device="cuda")
    size = lens[:, None, None]
    must = (j < c["sinks"]) | (j >= size - c["recent"])
    rank = torch.where(must, torch.full_like(w, math.inf), w)
    rank = torch.where(j < size, rank, torch.full_like(w, -math.inf))
    order = rank.sort(dim=-1, descending=True, stable=True).indices
    place = torch.empty_like(order).scatter_(-1, order, j.expand_as(order))  # 0 = the heaviest
    keep = (place < n) & (j < size)
    src = torch.where(keep, j.expand_as(place), torch.full_like(place, L)).sort(-1).values[..., :n]
    live = src < L
    kept = torch.where(live, src, torch.full_like(src, -1))
    kept = torch.nn.functional.pad(kept, (0, n - kept.shape[-1]), value=-1).to(torch.int32)
    to = j[:src.shape[-1]].expand_as(src)
    src = torch.where(live, src, to)  # a place that nothing moves to keeps its row
    b = torch.arange(B, device="cuda")[:, None, None].expand_as(src)
    h = torch.arange(Hkv, device="cuda")[None, :, None].expand_as(src)
    for pages in (st["kp"], st["vp"]):
        pages[table[b, to], b, h, to % ps] = pages[table[b, src], b, h, src % ps]
    moved = torch.where(live, w.gather(-1, src), torch.zeros_like(w[..., :1]))
    moved = torch.nn.functional.pad(moved, (0, L - moved.shape[-1]))
    w.copy_(torch.where(j < size, moved, w))
    return kept, lens.clamp(max=n).to(torch.int32), st["kp"], st["vp"], w


_run_own = {"rope": _own_rope, "prompt": _own_prompt, "decode": _own_decode, "evict": _own_evict}
_run_plain = {"rope": _plain_rope, "prompt": _plain_prompt, "decode": _plain_decode, "evict": _plain_evict}


# --------------------------------------------------------------------------- #
# what a pass cannot do without
# --------------------------------------------------------------------------- #
def _pairs(case):
    """(visible (query, key) pairs, keys that some query sees), over the sequences."""
    window, sinks = case.get("window", 0), case.get("sinks", 0)
    pairs = keys = 0
    for n, total in zip(*_lens(case)):
        if total < 1:
            continue
        pos = np.arange(total - n, total, dtype=np.int64)
        if window:
            pairs += int((np.minimum(pos + 1, window) + np.minimum(sinks, np.maximum(pos + 1 - window, 0))).sum())
            low = max(0, total - n + 1 - window)
            keys += total - low + min(sinks, low)
        else:
            pairs += int((pos + 1).sum())
            keys += total
    return pairs, keys


def work(case):
    e, D, Hkv = _SIZE[case["dtype"]], case["D"], case["Hkv"]
    new, total = _lens(case)
    if case["kind"] == "rope":
        n = sum(new) if case["paged"] else case["B"] * case["S"]
        heads = case["Hq"] + (2 if case["paged"] else 1) * Hkv
        out = case["B"] * case["S"] * case["Hq"] * D * e + n * (heads - case["Hq"]) * D * e
        angles = min(n, case["past"] + case["S"]) * case["rot"] * 4
        return {"bytes": n * heads * D * e + out + angles + n * 8,
                "flops": n * (case["Hq"] + Hkv) * (4 * D + 3 * case["rot"])}
    if case["kind"] == "evict":
        cut = [t for t in total if t > case["budget"]]
        moved = len(cut) * case["budget"] * Hkv
        return {"bytes": moved * 2 * D * e * 2 + sum(cut) * (8 * Hkv + 4) + case["B"] * case["budget"] * Hkv * 4,
                "flops": sum(cut) * Hkv}
    pairs, keys = _pairs(case)
    rows = sum(new) if case["kind"] == "prompt" else case["B"]
    size = keys * (Hkv * 2 * D * e + 4) + 2 * rows * case["Hq"] * D * e
    if case.get("weights"):
        size += keys * Hkv * 8
    return {"bytes": size, "flops": 4 * D * case["Hq"] * pairs}


# --------------------------------------------------------------------------- #
# in 64 bits, from the definitions
# --------------------------------------------------------------------------- #
def exact(case, seed):
    st = prepare(case, seed)
    return {"rope": _exact_rope, "prompt": _exact_attention, "decode": _exact_attention,
            "evict": _exact_evict}[case["kind"]](case, st)


def _exact_rope(case, st):
    S, half, inter = case["S"], case["rot"] // 2, case["interleaved"]
    i = torch.arange(half, device="cuda")
    first, second = (2 * i, 2 * i + 1) if inter else (i, i + half)
    angle = torch.complex(st["cos"].double(), st["sin"].double())[st["positions"].long()].unsqueeze(2)

    def turned(x, w):
        x = x.double()
        x = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + _EPS).sqrt() * w.double()
        z = torch.complex(x[..., first], x[..., second]) * angle
        y = x.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    q, k = turned(st["q"], st["qw"]), turned(st["k"], st["kw"])
    if not case["paged"]:
        return q, k.permute(0, 2, 1, 3).contiguous()
    kp, vp = st["kp"].double(), st["vp"].double()
    for b, (n, start) in enumerate(zip(st["new"].tolist(), st["start"].tolist())):
        q[b, n:] = 0
        at = torch.arange(start, start + n, device="cuda")
        page = st["table"][b, at].long()
        kp[page, b, :, at % case["ps"]] = k[b, :n]
        vp[page, b, :, at % case["ps"]] = st["v"][b, :n].double()
    return q, kp, vp


def _exact_attention(case, st):
    decode = case["kind"] == "decode"
    q = (st["q"][:, None] if decode else st["q"]).double()
    G = case["Hq"] // case["Hkv"]
    out = torch.zeros_like(q)
    weights = st["w"].double() if "w" in st else None
    for b, (n, total) in enumerate(zip(st["new"].tolist(), st["lens"].tolist())):
        if total == 0 or n == 0:
            continue
        at = torch.arange(total, device="cuda")
        page = st["table"][b, :total].long()
        pos = at[total - n:, None]
        hidden = at > pos
        if st["window"]:
            hidden |= (at <= pos - st["window"]) & (at >= case["sinks"])
        for h in range(case["Hkv"]):
            keys = st["kp"][page, b, h, at % case["ps"]].double()
            vals = st["vp"][page, b, h, at % case["ps"]].double()
            for g in range(h * G, h * G + G):
                score = (q[b, :n, g] @ keys.T / math.sqrt(case["D"])).masked_fill(hidden, -math.inf)
                p = torch.softmax(score, -1)
                out[b, :n, g] = p @ vals
                if weights is not None:
                    weights[b, h, :total] += p[0]
    if not decode:
        return out
    return out[:, 0] if weights is None else (out[:, 0], weights)


def _exact_evict(case, st):
    n, kp, vp, w = case["budget"], st["kp"].clone(), st["vp"].clone(), st["w"].clone()
    total, weights = st["lens"].tolist(), st["w"].cpu().numpy()
    kept = np.full((case["B"], case["Hkv"], n), -1, np.int32)
    for b in range(case["B"]):
        size = total[b]
        for h in range(case["Hkv"]):
            if size <= n:
                kept[b, h, :size] = np.arange(size)
                continue
            ends = np.r_[0:case["sinks"], size - case["recent"]:size]
            middle = np.arange(case["sinks"], size - case["recent"])
            heavy = middle[np.lexsort((middle, -weights[b, h, middle]))][:n - ends.size]
            kept[b, h] = np.sort(np.r_[ends, heavy])
            src = torch.from_numpy(kept[b, h].astype(np.int64)).cuda()
            to = torch.arange(n, device="cuda")
            ps, row = case["ps"], st["table"][b].long()
            for new, old in ((kp, st["kp"]), (vp, st["vp"])):
                new[row[to], b, h, to % ps] = old[row[src], b, h, src % ps]
            w[b, h, :n] = st["w"][b, h, src]
            w[b, h, n:size] = 0
    lens = torch.tensor([min(t, n) for t in total], dtype=torch.int32)
    return torch.from_numpy(kept), lens, kp, vp, w
