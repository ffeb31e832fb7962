"""Refusals of the paged-cache serving operators: the C entry points answer bad
sizes, dtypes, pointers and workspaces on the host before any launch, and the
Python operators check shapes, strides, dtypes and devices.  CPU only."""

import math

import pytest
import torch

import paged_reference as R

OK, SHAPE, DTYPE, WORKSPACE, ARG = 0, 1, 2, 6, 8
P = 256  # an address that is never dereferenced: every call below returns before a launch


def rope_args(**kw):
    a = dict(q=P, q_sb=64, q_ss=64, q_sh=64, k=P, k_sb=64, k_ss=64, k_sh=64, v=P, v_sb=64, v_ss=64, v_sh=64, dtype=1,
             positions=P, cos=P, sin=P, max_pos=10, rot=64, qw=None, qwd=0, kw=None, kwd=0, eps=1e-6, norm=1, inter=0,
             q_out=P, k_out=P, k_pages=None, v_pages=None, table=None, stride=0, pages=0, ps=0, start=None,
             count=None, B=2, S=3, Hq=4, Hkv=2, D=64, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return [0 if x is None else x for x in a.values()]


def attn_args(**kw):
    a = dict(q=P, k=P, v=P, table=P, stride=64, lens=P, q_lens=None, out=P, dtype=1, B=2, S=3, Hq=4, Hkv=2, D=64,
             pages=8, ps=16, scale=0.1, window=0, sinks=0, weights=None, weight_ld=0, ws=P, ws_bytes=1 << 40,
             stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return [0 if x is None else x for x in a.values()]


def evict_args(**kw):
    a = dict(k=P, v=P, dtype=1, table=P, stride=64, pages=8, ps=16, lens=P, weights=P, weight_ld=64, kept=P,
             new_lens=P, B=2, H=2, D=64, budget=10, sinks=1, recent=2, ws=P, ws_bytes=1 << 40, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return [0 if x is None else x for x in a.values()]


PAGED = dict(k_pages=P, v_pages=P, table=P, stride=64, pages=8, ps=16, start=P)


@pytest.mark.parametrize("kw,status", [
    (dict(B=0), OK), (dict(S=0), OK), (dict(D=0), SHAPE), (dict(Hq=-1), SHAPE), (dict(rot=63), SHAPE),
    (dict(rot=66), SHAPE), (dict(dtype=3), DTYPE), (dict(dtype=7), DTYPE), (dict(qw=P, qwd=3), DTYPE),
    (dict(q=None), ARG), (dict(q_out=None), ARG), (dict(k=None), ARG), (dict(k_out=None), ARG), (dict(cos=None), ARG),
    (dict(positions=None), ARG), (dict(PAGED, ps=0), SHAPE), (dict(PAGED, start=None), ARG),
    (dict(PAGED, v=None), ARG), (dict(PAGED, v_pages=None), ARG), (dict(B=1 << 40), SHAPE),
    (dict(B=1 << 20, S=1 << 12), SHAPE),
])
def test_rope_entry_refuses(kw, status):
    import _mtp_native as N
    before = N.lib().mtp_launch_count()
    assert N.lib().mtp_qk_norm_rope(N.QK_NORM_ROPE_ARGS.pack(*rope_args(**kw))) == status
    assert N.lib().mtp_launch_count() == before


@pytest.mark.parametrize("kw,status", [
    (dict(B=0), OK), (dict(S=0), OK), (dict(D=0), SHAPE), (dict(D=264), SHAPE), (dict(Hq=5), SHAPE),
    (dict(Hkv=0), SHAPE), (dict(ps=0), SHAPE), (dict(window=-1), SHAPE), (dict(sinks=-1), SHAPE),
    (dict(dtype=3), DTYPE), (dict(q=None), ARG), (dict(lens=None), ARG), (dict(table=None), ARG), (dict(k=None), ARG),
    (dict(ws=None), WORKSPACE), (dict(ws_bytes=16), WORKSPACE), (dict(ws=264), WORKSPACE),
    (dict(weights=P, weight_ld=64), SHAPE),  # key weights with three rows a sequence
    (dict(weights=P, weight_ld=63, S=1), SHAPE), (dict(pages=1 << 31), SHAPE), (dict(stride=1 << 31), SHAPE),
    (dict(B=1 << 30), SHAPE),
])
def test_attention_entry_refuses(kw, status):
    import _mtp_native as N
    before = N.lib().mtp_launch_count()
    assert N.lib().mtp_paged_window_attention(N.WINDOW_ATTENTION_ARGS.pack(*attn_args(**kw))) == status
    assert N.lib().mtp_launch_count() == before


@pytest.mark.parametrize("kw,status", [
    (dict(B=0), OK), (dict(D=0), SHAPE), (dict(H=0), SHAPE), (dict(budget=-1), SHAPE), (dict(sinks=11), SHAPE),
    (dict(sinks=5, recent=6), SHAPE), (dict(recent=1 << 62), SHAPE), (dict(dtype=3), DTYPE), (dict(lens=None), ARG),
    (dict(kept=None), ARG), (dict(weights=None), ARG), (dict(new_lens=None), ARG), (dict(ws=None), WORKSPACE),
    (dict(ws_bytes=10), WORKSPACE), (dict(pages=1 << 40), SHAPE),
])
def test_evict_entry_refuses(kw, status):
    import _mtp_native as N
    before = N.lib().mtp_launch_count()
    assert N.lib().mtp_paged_kv_evict(N.KV_EVICT_ARGS.pack(*evict_args(**kw))) == status
    assert N.lib().mtp_launch_count() == before


def test_null_arguments_are_refused():
    import _mtp_native as N
    for f in (N.lib().mtp_qk_norm_rope, N.lib().mtp_paged_window_attention, N.lib().mtp_paged_kv_evict):
        assert f(None) == ARG


def test_argument_structs_match_the_header(tmp_path):
    """The packed structs have the sizes and member offsets that a C compiler
    gives the header's."""
    import os
    import re
    import shutil
    import subprocess
    import _mtp_native as N
    from conftest import REPO
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    header = open(os.path.join(REPO, "include", "mtp_b200.h")).read()
    src = '#include <stddef.h>\n#include <stdio.h>\n#include "mtp_b200.h"\nint main(void) {\n'
    names = {"mtp_qk_norm_rope_args": N.QK_NORM_ROPE_ARGS, "mtp_paged_window_attention_args": N.WINDOW_ATTENTION_ARGS,
             "mtp_paged_kv_evict_args": N.KV_EVICT_ARGS}
    for name in names:
        src += f'  printf("%zu %zu\\n", sizeof({name}), offsetof({name}, stream));\n'
    src += "  return 0;\n}\n"
    (tmp_path / "s.c").write_text(src)
    subprocess.run([cc, "-std=c99", "-I", os.path.join(REPO, "include"), str(tmp_path / "s.c"), "-o",
                    str(tmp_path / "s")], check=True)
    out = subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split()
    for i, (name, packed) in enumerate(names.items()):
        assert int(out[2 * i]) == packed.size and int(out[2 * i + 1]) == packed.size - 8, name
        body = re.search(r"typedef struct \{([^}]*)\} " + name, header).group(1)
        doubles = [d for d in re.findall(r"double (\w+);", body)]
        assert packed.format.replace("=", "").count("d") == len(doubles)


def tensors():
    B, S, Hq, Hkv, D, ps, L = 2, 3, 4, 2, 64, 16, 40
    bf = torch.bfloat16
    return dict(q=torch.zeros(B, S, Hq, D, dtype=bf), k=torch.zeros(B, S, Hkv, D, dtype=bf),
                v=torch.zeros(B, S, Hkv, D, dtype=bf), pos=torch.zeros(B, S, dtype=torch.int32),
                cos=torch.zeros(50, D // 2), sin=torch.zeros(50, D // 2), kp=torch.zeros(4, B, Hkv, ps, D, dtype=bf),
                vp=torch.zeros(4, B, Hkv, ps, D, dtype=bf), table=torch.zeros(B, L, dtype=torch.int32),
                lens=torch.ones(B, dtype=torch.int32), w=torch.zeros(B, Hkv, L))


def test_operators_refuse_shapes_and_devices():
    import mtp_kernels as mk
    t = tensors()
    rope = lambda **kw: mk.fused_qk_norm_rope(*[{**t, **kw}[n] for n in ("q", "k", "pos", "cos", "sin")])
    paged = lambda **kw: mk.fused_qk_norm_rope_paged(
        *[{**t, **kw}[n] for n in ("q", "k", "v", "pos", "cos", "sin", "kp", "vp", "table", "lens")])
    prompt = lambda opt={}, **kw: mk.fused_paged_prompt_attention(
        *[{**t, **kw}[n] for n in ("q", "kp", "vp", "table", "lens")], **opt)
    decode = lambda opt={}, **kw: mk.fused_paged_decode_attention(
        {**t, **kw}["q"][:, 0], *[{**t, **kw}[n] for n in ("kp", "vp", "table", "lens")], **opt)
    evict = lambda opt={}, budget=5, **kw: mk.paged_kv_evict(
        *[{**t, **kw}[n] for n in ("kp", "vp", "table", "lens", "w")], budget, **opt)
    for call in (rope, paged, prompt, decode, evict):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    bad = [
        (rope, dict(k=t["k"][:, :2])), (rope, dict(k=t["k"].float())), (rope, dict(cos=t["cos"].double())),
        (rope, dict(cos=t["cos"][:, :5])), (rope, dict(pos=t["pos"][:1])), (rope, dict(pos=None)),
        (paged, dict(v=t["v"].float())), (paged, dict(kp=t["kp"].transpose(0, 1))), (paged, dict(kp=t["kp"].float())),
        (paged, dict(table=t["table"][:1])), (paged, dict(lens=t["lens"][:1])),
        (prompt, dict(kp=t["kp"].half())), (prompt, dict(table=t["table"][0])), (prompt, dict(lens=t["lens"][:1])),
        (prompt, dict(opt=dict(window=0))), (prompt, dict(opt=dict(sinks=-1))), (prompt, dict(q=t["q"][:, :, :3])),
        (prompt, dict(opt=dict(q_lens=t["lens"][:1]))), (decode, dict(opt=dict(window=-3))),
        (decode, dict(opt=dict(key_weights=t["w"].half()))), (decode, dict(opt=dict(key_weights=t["w"][:, :, :30]))),
        (decode, dict(opt=dict(key_weights=t["w"].transpose(0, 1)))),
        (evict, dict(opt=dict(sinks=3, recent=3))), (evict, dict(budget=-1)), (evict, dict(w=t["w"].double())),
        (evict, dict(w=t["w"][:, :, :39].contiguous())), (evict, dict(vp=t["vp"].float())),
        (evict, dict(kp=t["kp"].transpose(3, 4))),
    ]
    for call, kw in bad:
        with pytest.raises(AssertionError):
            call(**kw)


def test_reference_attention_against_dense_softmax():
    """The 64-bit restatement itself: one sequence in page order, causal, is the
    textbook formula."""
    g = torch.Generator().manual_seed(1)
    B, S, H, D, ps = 1, 7, 2, 16, 4
    kp, vp, q = (torch.randn(*s, generator=g) for s in ((2, B, H, ps, D), (2, B, H, ps, D), (B, S, H, D)))
    table = (torch.arange(8) // ps)[None].to(torch.int32)
    out, tol, w, _ = R.attention(q, kp, vp, table, [7], [7], None, 0)
    K = kp.permute(1, 2, 0, 3, 4).reshape(B, H, 8, D)[:, :, :7].double()
    V = vp.permute(1, 2, 0, 3, 4).reshape(B, H, 8, D)[:, :, :7].double()
    x = torch.einsum("bshd,bhjd->bhsj", q.double(), K) / math.sqrt(D)
    x = x.masked_fill(torch.ones(S, S).triu(1).bool(), -math.inf)
    want = torch.einsum("bhsj,bhjd->bshd", x.softmax(-1), V)
    assert (out - want).abs().max() < 1e-12 and (tol > 0).all()
    assert (w[0, :, :7] - x.softmax(-1)[0, :, -1]).abs().max() < 1e-12


def test_reference_evict_against_sort():
    g = torch.Generator().manual_seed(1)
    w = torch.rand(1, 1, 30, generator=g)
    kept = R.evict([30], w, 12, 2, 3)[0][0]
    middle = w[0, 0, 2:27].sort(descending=True, stable=True).indices[:7] + 2
    assert kept == sorted([0, 1, 27, 28, 29] + middle.tolist())
