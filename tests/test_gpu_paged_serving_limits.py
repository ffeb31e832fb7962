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
