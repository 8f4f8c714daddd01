"""Addresses that are no multiple of their values' size are refused by the
device entry points of the rotation, the head norms and window attention
before any CUDA call (no GPU is needed: the addresses are never looked at)."""
import ctypes

import pytest

from arm_ai_b200._lib import QkNormRopeArgs, RopeArgs, WindowAttentionArgs, load_cuda


def refusal(fn, args):
    lib = load_cuda()
    assert getattr(lib, fn)(ctypes.byref(args), None) == -1
    return lib.armai_last_error().decode()


@pytest.mark.parametrize("dtype,size", [(0, 4), (1, 2), (2, 2)])
def test_first_tensor_off_its_type(built, dtype, size):
    """The first tensor of each call, one byte and (f32) two bytes off."""
    for off in {1, size // 2, size - 1}:
        p = 4096 + off
        want = f"is not aligned to its values of {size} bytes"
        r = RopeArgs(x=p, out=8192, positions=256, inv_freq=256, n_tokens=2, n_heads=3, head_dim=64, rot_dim=64, dtype=dtype)
        assert f"rope: x {want}" in refusal("armai_dev_rope", r)
        qk = dict(k=8192, q_out=512, k_out=1024, n_tokens=2, head_dim=64, dtype=dtype, kv_dtype=dtype, n_rows=9)
        assert f"qk_norm_rope: q {want}" in refusal("armai_dev_qk_norm_rope", QkNormRopeArgs(q=p, n_q_heads=4, **qk))
        assert f"qk_norm_rope: k {want}" in refusal("armai_dev_qk_norm_rope",
                                                    QkNormRopeArgs(q=p, n_kv_heads=4, **{**qk, "k": p}))
        w = WindowAttentionArgs(q=p, k=512, v=512, out=512, kv_len=256, n_seq=1, max_q=1, n_tokens=1, n_q_heads=2,
                                n_kv_heads=1, head_dim=64, n_slots=1, kv_rows=9, window=5, scale=1.0, dtype=dtype)
        assert f"window_attn: q {want}" in refusal("armai_dev_window_attention", w)
