"""Plain 64-bit forms of the position, head-norm and window-attention
operators, from their definitions, and the argument blocks of their
device entry points for torch tensors (shared by the tests)."""
import ctypes
import math

import torch

from arm_ai_b200._lib import QkNormRopeArgs, RopeArgs, WindowAttentionArgs, check, load_cuda

CODE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
LAYOUT = {"interleaved": 0, "half": 1}


def half_step(dtype):
    """Largest relative error of one rounding to dtype."""
    return torch.finfo(dtype).eps / 2


def stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def rotate64(x, pos, inv_freq, layout, mscale=1.0):
    """x [t, h, d] -> f64, the first 2 * len(inv_freq) values turned; and the
    length of each value's pair (itself behind the rotated part)."""
    x = x.double()
    r = inv_freq.numel()
    ang = pos.double()[:, None] * inv_freq.double()
    c, s = (ang.cos() * mscale)[:, None], (ang.sin() * mscale)[:, None]
    out, size = x.clone(), x.abs()
    for i in range(r):
        a, b = (2 * i, 2 * i + 1) if layout == "interleaved" else (i, i + r)
        out[..., a] = x[..., a] * c[..., i] - x[..., b] * s[..., i]
        out[..., b] = x[..., a] * s[..., i] + x[..., b] * c[..., i]
        size[..., a] = size[..., b] = torch.hypot(x[..., a], x[..., b])
    return out, size


def norm64(x, gamma, eps):
    x = x.double()
    return x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * gamma.double()


def rope_args(x, out, pos, inv_freq, layout, mscale=1.0):
    return RopeArgs(x=x.data_ptr(), out=out.data_ptr(), positions=pos.data_ptr(), inv_freq=inv_freq.data_ptr(),
                    n_tokens=x.shape[0], n_heads=x.shape[1], head_dim=x.shape[2], rot_dim=2 * inv_freq.numel(),
                    x_token_stride=x.stride(0), x_head_stride=x.stride(1), out_token_stride=out.stride(0),
                    out_head_stride=out.stride(1), mscale=mscale, dtype=CODE[x.dtype], layout=LAYOUT[layout])


def rope(x, out, pos, inv_freq, layout, mscale=1.0):
    a = rope_args(x, out, pos, inv_freq, layout, mscale)
    check(load_cuda().armai_dev_rope(ctypes.byref(a), stream()))


def qk_args(q, k, v, q_out, k_cache, v_cache, gq, gk, pos, inv_freq, rows, layout, eps=1e-5, mscale=1.0):
    """k_cache [slots, hkv, cap, d] (strided as a cache) or k_out [t, hkv, d]."""
    if k_cache.dim() == 4:
        row, head, n_rows = k_cache.stride(2), k_cache.stride(1), (k_cache.shape[0] - 1) * (
            k_cache.stride(0) // k_cache.stride(2)) + k_cache.shape[2]
    else:
        row, head, n_rows = k_cache.stride(0), k_cache.stride(1), k_cache.shape[0]
    p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    return QkNormRopeArgs(
        q=p(q), k=p(k), v=p(v), q_out=p(q_out), k_out=p(k_cache), v_out=p(v_cache), q_gamma=p(gq), k_gamma=p(gk),
        positions=p(pos), inv_freq=p(inv_freq), kv_rows=p(rows), n_tokens=q.shape[0], n_q_heads=q.shape[1],
        n_kv_heads=k.shape[1], head_dim=q.shape[2], rot_dim=2 * inv_freq.numel(), token_stride=q.stride(0),
        head_stride=q.stride(1), q_out_token_stride=q_out.stride(0), q_out_head_stride=q_out.stride(1),
        kv_row_stride=row, kv_head_stride=head, n_rows=n_rows, eps=eps, mscale=mscale, dtype=CODE[q.dtype],
        kv_dtype=CODE[k_cache.dtype], layout=LAYOUT[layout])


def qk_norm_rope(*a, **kw):
    args = qk_args(*a, **kw)
    check(load_cuda().armai_dev_qk_norm_rope(ctypes.byref(args), stream()))


def attn_args(q, k, v, out, kv_len, window, n_sink=0, ring=False, q_start=None, slots=None, max_q=None, scale=None):
    """q / out [tokens, hq, d]; k / v [slots, hkv, rows, d] of any strides."""
    return WindowAttentionArgs(
        q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), out=out.data_ptr(),
        q_start=None if q_start is None else q_start.data_ptr(), kv_len=kv_len.data_ptr(),
        slots=None if slots is None else slots.data_ptr(), n_seq=kv_len.numel(),
        max_q=q.shape[0] // kv_len.numel() if max_q is None else max_q, n_tokens=q.shape[0], n_q_heads=q.shape[1],
        n_kv_heads=k.shape[1], head_dim=q.shape[2], q_token_stride=q.stride(0), q_head_stride=q.stride(1),
        out_token_stride=out.stride(0), out_head_stride=out.stride(1), kv_slot_stride=k.stride(0),
        kv_head_stride=k.stride(1), kv_row_stride=k.stride(2), n_slots=k.shape[0], kv_rows=k.shape[2], window=window,
        n_sink=n_sink, ring=int(ring), scale=q.shape[2] ** -0.5 if scale is None else scale, dtype=CODE[q.dtype])


def window_attention(*a, **kw):
    args = attn_args(*a, **kw)
    check(load_cuda().armai_dev_window_attention(ctypes.byref(args), stream()))


def attention64(q, k, v, q_lens, kv_len, window, n_sink=0, ring=False, slots=None, scale=None):
    """(exact, bound): the definition per sequence and head in f64, and how far
    an element may be off: the weights and the output are each rounded once to
    q's type (weights of f32 inputs are not), and the scores, the exponentials
    and the sums are f32 with errors bounded by their lengths."""
    d, group = q.shape[2], q.shape[1] // k.shape[1]
    scale = d ** -0.5 if scale is None else scale
    u, u32 = half_step(q.dtype), 2.0 ** -24
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    at = 0
    for s, n in enumerate(q_lens):
        slot, length = s if slots is None else slots[s], kv_len[s]
        p = torch.arange(length - n, length, device=q.device)
        j = torch.arange(max(length, 0), device=q.device)
        seen = (j[None] <= p[:, None]) & ((j[None] > p[:, None] - window) | (j[None] < n_sink))
        used = seen.any(0)
        j, seen = j[used], seen[:, used]
        rows = torch.where(j < n_sink, j, n_sink + (j - n_sink) % (k.shape[2] - n_sink)) if ring else j
        for h in range(q.shape[1]) if j.numel() and 0 <= slot < k.shape[0] else ():
            qd = q[at:at + n, h].double()
            kd, vd = k[slot, h // group][rows].double(), v[slot, h // group][rows].double()
            sc = (qd @ kd.T * scale).masked_fill(~seen, -math.inf)
            top = sc.amax(-1, keepdim=True)
            e = torch.exp(sc - torch.where(top == -math.inf, 0.0, top))
            tot = e.sum(-1, keepdim=True)
            w = torch.where(tot > 0, e / tot, 0.0)
            out[at:at + n, h] = w @ vd
            # a score's error: d products and the scale in f32; a weight's: twice that (itself and the sum's)
            # and two steps of the exponential; the sums': their length
            ds = ((d + 4) * u32 * (qd.abs() @ kd.abs().T * scale)).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
            mass = w @ vd.abs()
            rel = 2 * ds + (math.log2(j.numel() + 1) + j.numel() / 16 + 24) * u32 + (u if q.dtype != torch.float32 else 0.0)
            tol[at:at + n, h] = rel * mass + u * out[at:at + n, h].abs() + torch.finfo(q.dtype).tiny
        at += n
    return out, tol


def close(got, exact, tol):
    """Largest error in units of its bound; asserts that it is at most 1."""
    err = (got.double() - exact).abs()
    assert torch.isfinite(got.double()).all()
    worst = (err / tol.clamp(min=1e-300)).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"error {err.max().item():.3e}, {worst:.2f} of its bound"
    return worst
