"""Host arithmetic of the paged-cache serving entries at the ends of their
argument ranges: sizes are worked out in 64 bits without wrapping, so that no
call passes its workspace check with less memory than its kernels write.  CPU
only: nothing here reaches a launch."""

import pytest

import test_paged_serving as T

FAR = (1 << 30, (1 << 30) + 1, 1 << 62, (1 << 63) - 1)  # "everything", as callers write it


def workspace(window, sinks, weights, S=1, D=128, dtype=1, width=4096):
    import _mtp_native as N
    return N.lib().mtp_paged_window_attention_workspace(2, S, 8, 2, D, width, window, sinks, dtype, weights)


@pytest.mark.parametrize("S,D,dtype", [(1, 128, 1), (3, 128, 2), (200, 128, 1), (20, 256, 1), (1, 128, 0)])
@pytest.mark.parametrize("weights", [0, 1])
def test_workspace_of_far_windows_and_sinks(S, D, dtype, weights):
    """A window past the table is no window, and sinks past it are all keys."""
    if weights and S > 1:
        pytest.skip("key weights go with one row per sequence")
    kw = dict(weights=weights, S=S, D=D, dtype=dtype)
    everything = workspace(0, 0, **kw)
    for window in FAR:
        for sinks in (0, 4) + FAR:
            assert workspace(window, sinks, **kw) == everything, (window, sinks)
    for sinks in FAR:
        assert workspace(5, sinks, **kw) == everything, sinks
        assert workspace(0, sinks, **kw) == everything, sinks


@pytest.mark.parametrize("window,sinks", [((1 << 63) - 1, 4), (1 << 62, 1 << 62), (5, (1 << 63) - 1)])
def test_far_windows_need_the_whole_workspace(window, sinks):
    import _mtp_native as N
    need = workspace(0, 0, 1, D=64, width=4096)
    args = T.attn_args(S=1, stride=4096, window=window, sinks=sinks, weights=T.P, weight_ld=4096, ws_bytes=need - 1,
                       B=2, Hq=8, Hkv=2, D=64)
    before = N.lib().mtp_launch_count()
    assert N.lib().mtp_paged_window_attention(N.WINDOW_ATTENTION_ARGS.pack(*args)) == T.WORKSPACE
    assert N.lib().mtp_launch_count() == before


@pytest.mark.parametrize("kw", [
    dict(B=1 << 32, S=1 << 32), dict(B=1 << 40, S=1 << 40), dict(S=1 << 62, B=4), dict(Hq=1 << 62, Hkv=1 << 62),
    dict(Hq=(1 << 63) - 1, Hkv=1),
])
def test_sizes_whose_products_wrap_are_refused(kw):
    """B * S = 2^64 is not an empty call."""
    import _mtp_native as N
    before = N.lib().mtp_launch_count()
    assert N.lib().mtp_qk_norm_rope(N.QK_NORM_ROPE_ARGS.pack(*T.rope_args(k_out=T.P, **kw))) == T.SHAPE
    assert N.lib().mtp_qk_norm_rope(N.QK_NORM_ROPE_ARGS.pack(*T.rope_args(**dict(T.PAGED, **kw)))) == T.SHAPE
    assert N.lib().mtp_paged_window_attention(N.WINDOW_ATTENTION_ARGS.pack(*T.attn_args(**kw))) == T.SHAPE
    assert N.lib().mtp_launch_count() == before


@pytest.mark.parametrize("window", [0.5, 1.5, 0, -1, float("inf"), float("nan")])
def test_windows_of_no_whole_number_are_refused(window):
    """0.5 positions must not come out as 0, which is no window."""
    import mtp_kernels as mk
    t = T.tensors()
    with pytest.raises(AssertionError, match="window"):
        mk.fused_paged_prompt_attention(t["q"], t["kp"], t["vp"], t["table"], t["lens"], window=window)
    with pytest.raises(AssertionError, match="window"):
        mk.fused_paged_decode_attention(t["q"][:, 0], t["kp"], t["vp"], t["table"], t["lens"], window=window)


@pytest.mark.parametrize("window", [1, 7, 2.0, 1 << 62])
def test_whole_windows_are_taken(window):
    import mtp_kernels as mk
    t = T.tensors()
    with pytest.raises(ValueError, match="CUDA"):  # past the window's check
        mk.fused_paged_prompt_attention(t["q"], t["kp"], t["vp"], t["table"], t["lens"], window=window)
