"""Positions, head norms and window attention without a GPU: the scaled
frequencies against their formulas, and the calls that are refused before any
CUDA call."""
import ctypes

import numpy as np
import pytest

from arm_ai_b200 import prims
from arm_ai_b200._lib import QkNormRopeArgs, RopeArgs, WindowAttentionArgs, load_cuda
from arm_ai_b200.native import NifError


def plain(rot, base=10000.0):
    return base ** (-np.arange(0, rot, 2, dtype=np.float64) / rot)


@pytest.mark.parametrize("rot", [2, 20, 64, 128])
def test_frequencies(built, rot):
    f = plain(rot)
    # one rounding to f32 of a power that libm gives to an ulp or two of f64
    tol = 2.0 ** -24 * 1.001
    np.testing.assert_allclose(prims.rope_frequencies(rot), f, rtol=tol)
    np.testing.assert_allclose(prims.rope_frequencies(rot, scaling="linear", factor=8.0), f / 8, rtol=tol)
    np.testing.assert_allclose(prims.rope_frequencies(rot, base=5e5), plain(rot, 5e5), rtol=tol)
    if rot > 2:
        got = prims.rope_frequencies(rot, scaling="base", factor=4.0)
        np.testing.assert_allclose(got, plain(rot, 10000.0 * 4.0 ** (rot / (rot - 2))), rtol=tol)
        np.testing.assert_allclose(got[[0, -1]], [1.0, f[-1] / 4], rtol=tol)  # the ends: kept, divided
    got = prims.rope_frequencies(rot, scaling="turns", factor=8.0, orig_ctx=8192, low=1.0, high=4.0)
    turns = 8192 * f / (2 * np.pi)
    exact = np.where(turns >= 4, f, np.where(turns <= 1, f / 8, 0.0))
    mid = exact == 0
    g = (turns[mid] - 1) / 3
    exact[mid] = (1 - g) * f[mid] / 8 + g * f[mid]
    np.testing.assert_allclose(got, exact, rtol=tol)
    assert prims.rope_frequencies(0).size == 0


def test_frequency_refusals(built):
    for kw, msg in ((dict(base=0.0), "base must be positive"), (dict(base=float("nan")), "base must be positive"),
                    (dict(scaling="linear", factor=0.0), "factor must be positive"),
                    (dict(scaling="turns", factor=2.0), "orig_ctx > 0 and low < high"),
                    (dict(scaling="turns", factor=2.0, orig_ctx=10, low=4, high=4), "low < high"),
                    (dict(scaling="cubic"), "rope scaling 'cubic' is not one of")):
        with pytest.raises(NifError, match=msg):
            prims.rope_frequencies(64, **kw)
    with pytest.raises(NifError, match="needs rot_dim above 2"):
        prims.rope_frequencies(2, scaling="base", factor=2.0)
    with pytest.raises(NifError, match="rot_dim 5 must be even"):
        prims.rope_frequencies(5)


def refused(fn, args, msg):
    lib = load_cuda()
    assert getattr(lib, fn)(ctypes.byref(args), None) == -1
    assert msg in lib.armai_last_error().decode(), lib.armai_last_error()


def test_rope_refusals(built):
    ok = dict(n_tokens=2, n_heads=3, head_dim=64, rot_dim=64, dtype=0, layout=0)
    for change, msg in ((dict(dtype=3), "unknown dtype 3"), (dict(layout=2), "unknown layout 2"),
                        (dict(n_tokens=-1), "n_tokens -1"), (dict(n_tokens=1 << 31), "n_tokens"),
                        (dict(n_heads=65536), "heads"), (dict(head_dim=257, rot_dim=0), "head_dim 257"),
                        (dict(head_dim=0, rot_dim=0), "head_dim 0"), (dict(rot_dim=63), "rot_dim 63"),
                        (dict(rot_dim=66), "rot_dim 66"), (dict(rot_dim=-2), "rot_dim -2"),
                        (dict(x=64, out=64, x_token_stride=1, out_token_stride=2), "same strides")):
        refused("armai_dev_rope", RopeArgs(**{**ok, **change}), msg)
    lib = load_cuda()
    assert lib.armai_dev_rope(None, None) == -1
    for change in (dict(n_tokens=0), dict(n_heads=0)):  # nothing to do: no pointer is looked at
        assert lib.armai_dev_rope(ctypes.byref(RopeArgs(**{**ok, **change})), None) == 0


def test_qk_norm_rope_refusals(built):
    ok = dict(n_tokens=2, n_q_heads=4, n_kv_heads=2, head_dim=64, rot_dim=64, dtype=1, kv_dtype=1, layout=1, n_rows=9)
    for change, msg in ((dict(kv_dtype=2), "kv_dtype 2"), (dict(dtype=0, kv_dtype=5), "kv_dtype 5"),
                        (dict(dtype=9), "unknown dtype 9"), (dict(rot_dim=65), "rot_dim 65"),
                        (dict(n_q_heads=-1), "head counts"), (dict(n_kv_heads=40000), "80004 heads"),
                        (dict(n_rows=-1), "n_rows"),
                        (dict(q=64, q_out=64, head_stride=64, q_out_head_stride=128), "q and q_out must have the same"),
                        (dict(k=64, k_out=64, q=1, q_out=2, kv_rows=128), "in place, k and v")):
        refused("armai_dev_qk_norm_rope", QkNormRopeArgs(**{**ok, **change}), msg)
    lib = load_cuda()
    assert lib.armai_dev_qk_norm_rope(ctypes.byref(QkNormRopeArgs(**{**ok, "n_tokens": 0})), None) == 0
    with pytest.raises(NifError, match=r"qk_norm_rope: q_gamma len 3 != head_dim = 4"):
        prims.qk_norm_rope_f32_op(np.zeros(8), np.zeros(4), np.zeros(3), np.zeros(4), [0], np.zeros(2), 2, 1, 4)
    with pytest.raises(NifError, match=r"qk_norm_rope: k len 4 != T\*Hkv\*D = 8"):
        prims.qk_norm_rope_f32_op(np.zeros(8), np.zeros(4), np.zeros(4), np.zeros(4), [0], np.zeros(2), 2, 2, 4)
    with pytest.raises(NifError, match=r"inv_freq len 3 exceeds head_dim/2 = 2"):
        prims.rope_ext_f32_op(np.zeros(4), [0], np.zeros(3), 1, 4, 1)
    with pytest.raises(NifError, match=r"rope_ext: n_rows 2 != n_tokens \* heads_per_token = 1"):
        prims.rope_ext_f32_op(np.zeros(8), [0], np.zeros(2), 2, 4, 1)


def test_window_attention_refusals(built):
    ok = dict(n_seq=2, max_q=1, n_tokens=2, n_q_heads=8, n_kv_heads=2, head_dim=64, n_slots=2, kv_rows=100, window=50,
              n_sink=4, ring=0, scale=1.0, dtype=2)
    for change, msg in ((dict(dtype=-1), "unknown dtype -1"), (dict(n_seq=65536), "n_seq 65536"),
                        (dict(max_q=-1), "max_q"), (dict(n_tokens=1 << 30), "n_tokens"),
                        (dict(n_q_heads=7), "n_q_heads 7 must be a multiple of n_kv_heads 2"),
                        (dict(n_kv_heads=0), "multiple of n_kv_heads 0"), (dict(head_dim=0), "head_dim 0"),
                        (dict(head_dim=300), "head_dim 300"), (dict(window=0), "window must be at least 1"),
                        (dict(n_sink=-1), "n_sink"), (dict(kv_rows=0), "kv_rows"), (dict(n_slots=0), "n_slots"),
                        (dict(ring=2), "ring must be 0 or 1"),
                        (dict(ring=1, window=97), "window + max_q - 1 = 97, got 96"),
                        (dict(ring=1, max_q=48), "window + max_q - 1 = 97"),
                        (dict(ring=1, n_sink=100), "a ring needs")):
        refused("armai_dev_window_attention", WindowAttentionArgs(**{**ok, **change}), msg)
    lib = load_cuda()
    for change in (dict(n_seq=0), dict(max_q=0), dict(n_tokens=0), dict(n_q_heads=0)):
        assert lib.armai_dev_window_attention(ctypes.byref(WindowAttentionArgs(**{**ok, **change})), None) == 0
    with pytest.raises(NifError, match=r"window_attn: k len 3 != B\*Hkv\*Sk\*D = 4"):
        prims.window_attention_f32_op(np.zeros(4), np.zeros(3), np.zeros(4), 1.0, 1, 1, 1, 1, 1, 4, 8)
