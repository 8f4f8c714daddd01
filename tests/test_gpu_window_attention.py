"""Attention with a sliding window and visible first tokens
(armai_dev_window_attention) against its definition in f64: ragged prompts,
chunks behind a cache, single tokens; linear and ring caches; grouped heads;
every type. The bound of each element's error is derived in
window_reference.attention64 from the roundings that the kernels make."""
import ctypes
import math

import pytest

torch = pytest.importorskip("torch")

import window_reference as wr
from arm_ai_b200 import prims
from arm_ai_b200._lib import check, load_cuda

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rnd(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def starts(q_lens):
    s = [0]
    for n in q_lens:
        s.append(s[-1] + n)
    return i32(s)


def run(g, dtype, hq, hkv, d, q_lens, kv_len, window, n_sink=0, ring=False, extra=0, slots=None, n_slots=None,
        hide=True, scale=None):
    """One call on random data; the cache rows that nobody may look at hold NaN."""
    t, n = sum(q_lens), len(q_lens)
    rows = n_sink + window + max(q_lens) - 1 + extra if ring else max(max(kv_len), 1) + extra
    n_slots = n if n_slots is None else n_slots
    q = rnd(g, t, hq, d, dtype=dtype)
    k, v = rnd(g, n_slots, hkv, rows, d, dtype=dtype), rnd(g, n_slots, hkv, rows, d, dtype=dtype)
    if hide:
        for s in range(n_slots):
            at = slots.index(s) if slots is not None and s in slots else s if slots is None else None
            seen = torch.zeros(rows, dtype=torch.bool, device="cuda")
            if at is not None:
                p0, p1 = kv_len[at] - q_lens[at], kv_len[at]
                j = torch.arange(max(p1, 0), device="cuda")
                j = j[(j < n_sink) | (j > p0 - window)]
                seen[torch.where(j < n_sink, j, n_sink + (j - n_sink) % (rows - n_sink)) if ring else j] = True
            k[s, :, ~seen] = float("nan")
            v[s, :, ~seen] = float("nan")
    out = torch.full((t + 3, hq, d), 5.0, dtype=dtype, device="cuda")
    wr.window_attention(q, k, v, out[:t], i32(kv_len), window, n_sink, ring, q_start=starts(q_lens),
                        slots=None if slots is None else i32(slots), max_q=max(q_lens), scale=scale)
    exact, tol = wr.attention64(q, k, v, q_lens, kv_len, window, n_sink, ring, slots, scale)
    wr.close(out[:t], exact, tol)
    assert (out[t:] == 5.0).all()
    return out[:t]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 64), (4, 4, 128), (16, 1, 128), (7, 1, 64), (6, 2, 80), (3, 3, 17),
                                      (2, 1, 256), (64, 2, 128)])
@pytest.mark.parametrize("kv_len,window,n_sink,ring", [
    ([1, 2, 63, 64, 65], 1000, 0, False),
    ([1, 130, 700, 33], 100, 4, False),
    ([5, 104, 105, 999], 100, 4, True),
    ([40, 41, 2000], 33, 0, True),
    ([3, 77], 1, 0, False),
    ([500], 1, 3, True),
])
def test_single_tokens(built, dtype, hq, hkv, d, kv_len, window, n_sink, ring):
    run(gen(d + hq), dtype, hq, hkv, d, [1] * len(kv_len), kv_len, window, n_sink, ring, extra=5)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (4, 4, 64), (8, 1, 64), (6, 2, 64), (5, 1, 128), (4, 2, 96)])
@pytest.mark.parametrize("q_lens,past,window,n_sink,ring", [
    ([1, 127, 128, 129, 300], [0, 0, 0, 0, 0], 10000, 0, False),    # prompts, no window
    ([300, 5, 513], [0, 0, 0], 70, 4, False),                       # prompts longer than the window
    ([257, 64], [100, 1000], 128, 0, False),                        # behind a cache
    ([33, 2, 17], [1000, 0, 90], 64, 4, True),                      # ring, wrapping inside the call
    ([260], [777], 500, 1, True),
    ([130, 140], [3, 500], 1, 0, False),                            # only itself
    ([200], [300], 1, 5, True),                                     # itself and the first ones
])
def test_prompts_and_chunks(built, dtype, hq, hkv, d, q_lens, past, window, n_sink, ring):
    kv_len = [a + b for a, b in zip(past, q_lens)]
    # NaN only where no query of the sequence looks
    run(gen(sum(q_lens) + d), dtype, hq, hkv, d, q_lens, kv_len, window, n_sink, ring, extra=3)


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 64), (F32, 64)])
def test_long_single_tokens(built, dtype, d):
    """Contexts of many tiles per CTA: a long linear cache, and a long window in a ring."""
    run(gen(1), dtype, 8, 2, d, [1, 1], [20000, 12345], 1 << 40, 0, False)
    run(gen(2), dtype, 4, 1, d, [1], [100001], 30000, 4, True)


@pytest.mark.parametrize("dtype,hq,hkv", [(BF16, 32, 8), (F16, 8, 8)])
def test_long_prompt(built, dtype, hq, hkv):
    run(gen(3), dtype, hq, hkv, 128, [2049], [2049], 1024, 4, False)
    run(gen(4), dtype, hq, hkv, 64, [1500], [4000], 2000, 4, True)


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 64), (F32, 80)])
@pytest.mark.parametrize("q_lens,kv_len", [([1, 1, 1, 1], [0, 5, 9, -3]), ([4, 4, 200], [2, 0, 150]), ([3, 3], [7, 9])])
def test_rows_that_see_nothing(built, dtype, d, q_lens, kv_len):
    """Sequences without keys, queries before the first position, slots that do not exist: zeros."""
    slots = [2, 0, 7, 1][:len(q_lens)]
    out = run(gen(6), dtype, 4, 2, d, q_lens, kv_len, 50, 2, False, extra=4, slots=slots, n_slots=3)
    at = 0
    for n, length, s in zip(q_lens, kv_len, slots):
        dead = n if s >= 3 else min(max(n - length, 0), n)
        assert (out[at:at + dead] == 0).all()
        at += n


@pytest.mark.parametrize("dtype,d,q", [(BF16, 128, 1), (F16, 64, 150), (F32, 64, 1), (F32, 64, 70)])
def test_uniform_queries_without_starts(built, dtype, d, q):
    g = gen(7)
    n, kv_len = 3, [q + 9, q, q + 40]
    qq = rnd(g, n * q, 4, d, dtype=dtype)
    k, v = rnd(g, n, 2, q + 40, d, dtype=dtype), rnd(g, n, 2, q + 40, d, dtype=dtype)
    out = torch.empty_like(qq)
    wr.window_attention(qq, k, v, out, i32(kv_len), 25, 2, False)
    wr.close(out, *wr.attention64(qq, k, v, [q] * n, kv_len, 25, 2))


@pytest.mark.parametrize("dtype,d,q_lens,past", [(BF16, 128, [200, 31], [0, 50]), (F16, 64, [1, 1], [300, 70]),
                                                 (F32, 64, [1, 1], [300, 70]), (F32, 80, [90, 31], [0, 50])])
def test_strides_and_unaligned_rows(built, dtype, d, q_lens, past):
    """q packed with k and v behind it; a cache with the heads inside the rows; rows off 16-byte
    boundaries: the same values as contiguous tensors, to the bound."""
    g = gen(8)
    hq, hkv, n, t = 6, 2, len(q_lens), sum(q_lens)
    kv_len = [a + b for a, b in zip(past, q_lens)]
    rows = max(kv_len)
    packed = rnd(g, t, hq + 2 * hkv, d, dtype=dtype)
    cache = rnd(g, 2, n, rows, hkv, d, dtype=dtype)
    odd = torch.zeros(2 * n * rows * hkv * (d + 1) + 9, dtype=dtype, device="cuda")
    odd = odd[3:3 + 2 * n * rows * hkv * (d + 1)].view(2, n, rows, hkv, d + 1)[..., :d]
    odd.copy_(cache)
    for kv in (cache, odd):
        q, k, v = packed[:, :hq], kv[0].transpose(1, 2), kv[1].transpose(1, 2)
        out = torch.zeros(t, 2 * hq, d, dtype=dtype, device="cuda")
        wr.window_attention(q, k, v, out[:, hq:], i32(kv_len), 60, 3, False, q_start=starts(q_lens), max_q=max(q_lens))
        wr.close(out[:, hq:], *wr.attention64(q, k, v, q_lens, kv_len, 60, 3))
        assert not out[:, :hq].any()


@pytest.mark.parametrize("dtype,d", [(BF16, 64), (F16, 128), (F32, 64)])
def test_growing_and_extreme_scores(built, dtype, d):
    """Scores of up to a few hundred whose maximum moves from tile to tile, both ways; and all equal."""
    g = gen(9)
    for q_lens, kv_len in (([300], [600]), ([1], [3000])):
        t, rows = q_lens[0], kv_len[0]
        for ramp in (torch.linspace(0.05, 6.0, rows), torch.linspace(6.0, 0.05, rows), torch.zeros(rows)):
            q = rnd(g, t, 4, d, dtype=dtype)
            k = (rnd(g, 1, 2, rows, d) * ramp.cuda()[:, None]).to(dtype)
            v = rnd(g, 1, 2, rows, d, dtype=dtype)
            out = torch.empty_like(q)
            wr.window_attention(q, k, v, out, i32(kv_len), 100000, 0, False, scale=1.0)
            wr.close(out, *wr.attention64(q, k, v, q_lens, kv_len, 100000, scale=1.0))


@pytest.mark.parametrize("dtype,d,q", [(BF16, 128, 1), (F16, 64, 1), (F32, 64, 1), (BF16, 64, 300), (F32, 80, 90)])
def test_infinite_keys(built, dtype, d, q):
    """A key that makes its score -inf has weight 0; where every visible score is -inf the row is 0."""
    g = gen(10)
    rows = q + 200
    qq = rnd(g, q, 2, d, dtype=dtype).abs()
    k, v = rnd(g, 1, 1, rows, d, dtype=dtype), rnd(g, 1, 1, rows, d, dtype=dtype)
    k[0, 0, ::3] = float("-inf")
    out = torch.empty_like(qq)
    wr.window_attention(qq, k, v, out, i32([rows]), 90, 0, False)
    finite = torch.arange(rows, device="cuda") % 3 != 0
    # the definition over the finite keys alone
    exact = torch.zeros(q, 2, d, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(exact)
    j = torch.arange(rows, device="cuda")
    for i in range(0, q, max(1, q // 7)):
        p = rows - q + i
        keep = finite & (j <= p) & (j > p - 90)
        e, b = wr.attention64(qq[i:i + 1], k[:, :, keep].contiguous(), v[:, :, keep].contiguous(), [1],
                              [int(keep.sum())], 1000)
        wr.close(out[i:i + 1], e, b)
    k.fill_(float("-inf"))
    wr.window_attention(qq, k, v, out, i32([rows]), 90, 0, False)
    assert (out == 0).all()


def test_offsets_past_32_bits(built):
    """The second slot of a cache starts beyond 2^31 elements."""
    g = gen(11)
    stride = (1 << 31) + 128
    flat = torch.empty(2, stride + 2 * 300 * 128, dtype=BF16, device="cuda")
    for q_len in (1, 200):
        kv = []
        for f in flat:
            c = f.as_strided((2, 2, 300, 128), (stride, 300 * 128, 128, 1))
            c[1] = rnd(g, 2, 300, 128, dtype=BF16)
            kv.append(c)
        q = rnd(g, q_len, 4, 128, dtype=BF16)
        out = torch.empty_like(q)
        wr.window_attention(q, *kv, out, i32([290]), 128, 2, False, slots=i32([1]))
        wr.close(out, *wr.attention64(q, *kv, [q_len], [290], 128, 2, slots=[1]))


def test_garbage_starts_stay_in_bounds(built):
    """q_start values outside 0 .. n_tokens are clamped: nothing is read or written beyond the tensors."""
    g = gen(12)
    q = rnd(g, 10, 2, 64, dtype=BF16)
    k, v = rnd(g, 2, 1, 50, 64, dtype=BF16), rnd(g, 2, 1, 50, 64, dtype=BF16)
    out = torch.zeros(14, 2, 64, dtype=BF16, device="cuda")
    wr.window_attention(q, k, v, out[2:12], i32([40, 40]), 16, 0, False, q_start=i32([-7, 6, 99]), max_q=10)
    assert not out[:2].any() and not out[12:].any()


@pytest.mark.parametrize("dtype,d,q", [(BF16, 128, 1), (BF16, 128, 256), (F32, 64, 1), (F16, 64, 40)])
def test_captured_and_replayed(built, dtype, d, q):
    """Two graphs over the same buffers, replayed in turn with lengths that change between replays, on
    a side stream; each replay equals the eager call bit for bit, and repeats itself."""
    g = gen(13)
    n, rows = 2, q + 300
    qq = rnd(g, n * q, 8, d, dtype=dtype)
    k, v = rnd(g, n, 2, rows, d, dtype=dtype), rnd(g, n, 2, rows, d, dtype=dtype)
    kv_len, outs = i32([q + 200, q + 10]), [torch.zeros_like(qq) for _ in range(3)]
    s = torch.cuda.Stream()
    graphs = []
    torch.cuda.synchronize()
    for o in outs[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            wr.window_attention(qq, k, v, o, kv_len, 64, 4, False)
        graphs.append(graph)
    for lens in ([q + 200, q + 10], [q, q + 299], [q + 7, 0]):
        kv_len.copy_(i32(lens))
        for graph in graphs:
            graph.replay()
        wr.window_attention(qq, k, v, outs[2], kv_len, 64, 4, False)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[2])
        wr.close(outs[2], *wr.attention64(qq, k, v, [q] * n, lens, 64, 4))


def test_two_streams_at_once(built):
    g = gen(14)
    calls = []
    for i in range(4):
        q = rnd(g, 8, 16, 128, dtype=BF16)
        k, v = rnd(g, 8, 4, 2000, 128, dtype=BF16), rnd(g, 8, 4, 2000, 128, dtype=BF16)
        calls.append((q, k, v, torch.empty_like(q), i32([2000 - i * 100] * 8)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for i, (q, k, v, o, n) in enumerate(calls):
            with torch.cuda.stream(streams[i % 2]):
                wr.window_attention(q, k, v, o, n, 1500, 4, False)
    torch.cuda.synchronize()
    for i, (q, k, v, o, _) in enumerate(calls):
        wr.close(o, *wr.attention64(q, k, v, [1] * 8, [2000 - i * 100] * 8, 1500, 4))


def test_host_form(built):
    g = gen(15)
    q, k, v = rnd(g, 2, 4, 30, 48), rnd(g, 2, 2, 70, 48), rnd(g, 2, 2, 70, 48)
    got = prims.window_attention_f32_op(*(t.cpu().numpy() for t in (q, k, v)), 0.2, 2, 4, 2, 30, 70, 48, 20, 3)
    rows = q.transpose(1, 2).reshape(60, 4, 48)
    exact, tol = wr.attention64(rows, k, v, [30, 30], [70, 70], 20, 3, scale=0.2)
    back = torch.from_numpy(got).cuda().view(2, 4, 30, 48).transpose(1, 2).reshape(60, 4, 48)
    wr.close(back, exact, tol)
    empty = prims.window_attention_f32_op(q.cpu().numpy(), k[:, :, :0].cpu().numpy(), v[:, :, :0].cpu().numpy(), 0.2, 2,
                                          4, 2, 30, 0, 48, 20)
    assert not empty.any()


@pytest.mark.parametrize("dtype,layout", [(BF16, "half"), (F32, "interleaved"), (F16, "half")])
def test_stream_through_a_ring(built, dtype, layout):
    """A prompt, a chunk and single tokens of two sequences through norm, rotation, append and
    attention over one ring cache, as a serving loop runs them; every output against the same tokens
    attended to at once in f64 from what the cache was given."""
    g = gen(16)
    hq, hkv, d, window, n_sink, longest = 8, 2, 64, 90, 3, 40
    ring = window + longest - 1
    cap = n_sink + ring
    n, total = 2, 40 + 17 + 150
    qkv = rnd(g, n, total, hq + 2 * hkv, d, dtype=dtype)
    gq, gk = 1 + 0.1 * rnd(g, d), 1 + 0.1 * rnd(g, d)
    f = torch.from_numpy(prims.rope_frequencies(32, scaling="turns", factor=4.0, orig_ctx=64)).cuda()
    kc = torch.full((n, hkv, cap, d), float("nan"), dtype=dtype, device="cuda")
    vc = torch.full_like(kc, float("nan"))
    k_all, v_all = (torch.zeros(n, hkv, total, d, dtype=dtype, device="cuda") for _ in range(2))
    q_all, out_all = (torch.zeros(n, total, hq, d, dtype=dtype, device="cuda") for _ in range(2))
    at = 0
    for step in [40, 17] + [1] * 150:
        x = qkv[:, at:at + step].reshape(n * step, hq + 2 * hkv, d)
        pos = torch.arange(at, at + step, device="cuda").repeat(n)
        row = torch.where(pos < n_sink, pos, n_sink + (pos - n_sink) % ring)
        slot = torch.arange(n, device="cuda").repeat_interleave(step)
        q_out, out = (torch.empty(n * step, hq, d, dtype=dtype, device="cuda") for _ in range(2))
        wr.qk_norm_rope(x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], q_out, kc, vc, gq, gk, pos, f,
                        slot * (hkv * cap) + row, layout)
        wr.window_attention(q_out, kc, vc, out, i32([at + step] * n), window, n_sink, True)
        k_all[:, :, at:at + step] = kc[slot, :, row].view(n, step, hkv, d).transpose(1, 2)
        v_all[:, :, at:at + step] = vc[slot, :, row].view(n, step, hkv, d).transpose(1, 2)
        q_all[:, at:at + step], out_all[:, at:at + step] = q_out.view(n, step, hq, d), out.view(n, step, hq, d)
        at += step
    for s in range(n):
        pos = torch.arange(total, device="cuda")
        for got, x, gam in ((q_all[s], qkv[s, :, :hq], gq), (k_all[s].transpose(0, 1), qkv[s, :, hq:hq + hkv], gk)):
            exact, size = wr.rotate64(wr.norm64(x, gam, 1e-5), pos, f, layout)
            wr.close(got, exact, (6e-7 + 1.5e-6) * size + wr.half_step(dtype) * exact.abs() + torch.finfo(dtype).tiny)
        wr.close(out_all[s], *wr.attention64(q_all[s], k_all[s:s + 1], v_all[s:s + 1], [total], [total], window, n_sink))


def test_device_checks_refuse_host_tensors(built):
    q, k = torch.zeros(1, 2, 64, device="cuda"), torch.zeros(1, 1, 8, 64, device="cuda")
    a = wr.attn_args(q, k, k.cpu(), q, i32([3]), 4)
    lib = load_cuda()
    assert lib.armai_dev_window_attention(ctypes.byref(a), None) == -1
    assert b"window_attn: v is not device memory" in lib.armai_last_error()
    a = wr.attn_args(q, k, k, torch.empty_like(q), i32([3]), 4)
    a.n_seq = 0
    check(lib.armai_dev_window_attention(ctypes.byref(a), None))


# ---- many queries: more rows than the split form takes (its reads would pass
# 80 MB, or 36 f32 rows per SM and round of tiles) ---------------------------
MANY = [
    ([1, 127, 128, 129, 300], [0, 0, 0, 0, 0], 10000, 0, False),
    ([300, 5, 513], [0, 0, 0], 70, 4, False),
    ([257, 64], [100, 1000], 128, 0, False),
    ([333, 2, 170], [1000, 0, 90], 64, 4, True),
    ([260], [777], 500, 1, True),
    ([330, 340], [3, 500], 1, 0, False),
    ([400], [300], 1, 5, True),
]


@pytest.mark.parametrize("dtype,hq,hkv,d", [(BF16, 64, 16, 128), (F16, 64, 16, 64), (BF16, 48, 16, 64), (F16, 48, 8, 128),
                                            (F16, 64, 16, 96), (BF16, 80, 16, 80), (F16, 64, 32, 8), (F32, 64, 16, 64),
                                            (F32, 96, 32, 80)])
@pytest.mark.parametrize("q_lens,past,window,n_sink,ring", MANY)
def test_many_queries(built, dtype, hq, hkv, d, q_lens, past, window, n_sink, ring):
    run(gen(sum(q_lens) + d), dtype, hq, hkv, d, q_lens, [a + b for a, b in zip(past, q_lens)], window, n_sink, ring,
        extra=3)


@pytest.mark.parametrize("dtype,hq,hkv,d", [(BF16, 16, 4, 256), (F16, 6, 2, 160), (BF16, 4, 4, 136)])
@pytest.mark.parametrize("q_lens,past,window,n_sink,ring", MANY)
def test_many_queries_of_wide_heads(built, dtype, hq, hkv, d, q_lens, past, window, n_sink, ring):
    run(gen(sum(q_lens) + d), dtype, hq, hkv, d, q_lens, [a + b for a, b in zip(past, q_lens)], window, n_sink, ring,
        extra=3)


def test_more_than_65536_blocks_of_rows(built):
    """One call with many heads gives what calls with parts of the heads give."""
    g = gen(31)
    q, hq, hkv, d = 1100, 1024, 16, 136
    qq, k, v = (rnd(g, *s, dtype=BF16) for s in ((q, hq, d), (1, hkv, q, d), (1, hkv, q, d)))
    out, part = torch.empty_like(qq), torch.empty_like(qq)
    wr.window_attention(qq, k, v, out, i32([q]), 300, 2, False)
    for i in range(0, hkv, 4):
        h = slice(i * (hq // hkv), (i + 4) * (hq // hkv))
        wr.window_attention(qq[:, h], k[:, i:i + 4], v[:, i:i + 4], part[:, h], i32([q]), 300, 2, False)
    assert torch.equal(out, part)
    h = slice(hq - hq // hkv, hq)
    wr.close(out[:, h], *wr.attention64(qq[:, h], k[:, -1:], v[:, -1:], [q], [q], 300, 2))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 256), (5, 1, 192), (3, 3, 160), (12, 4, 132), (4, 1, 248)])
@pytest.mark.parametrize("q_lens,past,window,n_sink,ring", [
    ([1, 1, 1, 1], [0, 62, 700, 4099], 1000, 4, False),
    ([1, 1], [5000, 1030], 1024, 0, True),
    ([1], [40000], 1 << 40, 0, False),   # clusters of every size the keys are divided over
    ([3, 1, 8], [300, 0, 2], 90, 2, True),
])
def test_few_queries_of_wide_heads(built, dtype, hq, hkv, d, q_lens, past, window, n_sink, ring):
    run(gen(sum(past) + d), dtype, hq, hkv, d, q_lens, [a + b for a, b in zip(past, q_lens)], window, n_sink, ring,
        extra=2)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("seqs,hkv", [(1, 7), (1, 8), (1, 24), (3, 16), (2, 33), (7, 21)])
def test_divisions_of_the_keys(built, dtype, d, seqs, hkv):
    """Head and stream counts around those at which clusters of 16, 8, 4 and 2 CTAs no longer run all at once."""
    run(gen(hkv), dtype, hkv, hkv, d, [1] * seqs, [2100 - 300 * i for i in range(seqs)], 2000, 1, False)


@pytest.mark.parametrize("group,q", [(96, 700), (33, 2000)])
def test_more_than_65536_rows_of_a_head(built, group, q):
    """Pairs of a token and a head beyond 2^16, a key / value head of width 136."""
    run(gen(group), F16, group, 1, 136, [q], [q + 3], 70, 2, False)


@pytest.mark.parametrize("dtype,hq,hkv,d", [(BF16, 32, 8, 128), (F16, 32, 8, 64), (F16, 16, 2, 96)])
@pytest.mark.parametrize("q_lens,past,window,n_sink,ring", [
    ([64], [4000], 3000, 4, False),      # eight tiles, the keys divided over clusters
    ([100, 90, 97], [5000, 1300, 0], 2048, 4, True),
    ([200], [2500], 1 << 40, 0, False),
    ([129, 80], [2100, 30], 1000, 3, True),
])
def test_chunks_divided_over_clusters(built, dtype, hq, hkv, d, q_lens, past, window, n_sink, ring):
    out = run(gen(sum(q_lens) + d), dtype, hq, hkv, d, q_lens, [a + b for a, b in zip(past, q_lens)], window, n_sink, ring,
              extra=1)
    again = run(gen(sum(q_lens) + d), dtype, hq, hkv, d, q_lens, [a + b for a, b in zip(past, q_lens)], window, n_sink,
                ring, extra=1)
    assert torch.equal(out, again)


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 64), (F32, 80)])
def test_many_queries_that_see_nothing(built, dtype, d):
    """Queries before the first position, a sequence without keys, a slot that does not exist."""
    q_lens, kv_len, slots = [300, 260, 290, 280], [150, 0, 290, 400], [2, 0, 9, 1]
    out = run(gen(21), dtype, 64, 16, d, q_lens, kv_len, 50, 2, False, extra=4, slots=slots, n_slots=3)
    assert (out[:150] == 0).all() and (out[300:850] == 0).all()


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 64), (F32, 80)])
def test_many_queries_infinite_keys(built, dtype, d):
    g = gen(22)
    q, rows = 300, 500
    qq = rnd(g, q, 128, d, dtype=dtype).abs()
    k, v = rnd(g, 1, 32, rows, d, dtype=dtype), rnd(g, 1, 32, rows, d, dtype=dtype)
    k[0, :, ::3] = float("-inf")
    out = torch.empty_like(qq)
    wr.window_attention(qq, k, v, out, i32([rows]), 90, 0, False)
    finite = torch.arange(rows, device="cuda") % 3 != 0
    j = torch.arange(rows, device="cuda")
    for i in range(0, q, 37):
        p = rows - q + i
        keep = finite & (j <= p) & (j > p - 90)
        e, b = wr.attention64(qq[i:i + 1], k[:, :, keep].contiguous(), v[:, :, keep].contiguous(), [1],
                              [int(keep.sum())], 1000)
        wr.close(out[i:i + 1], e, b)
    k.fill_(float("-inf"))
    wr.window_attention(qq, k, v, out, i32([rows]), 90, 0, False)
    assert (out == 0).all()


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 64), (F32, 64)])
def test_many_queries_growing_scores(built, dtype, d):
    """The maximum moves from tile to tile, both ways: the output is rescaled many times."""
    g = gen(23)
    q, rows = 260, 700
    for ramp in (torch.linspace(0.05, 6.0, rows), torch.linspace(6.0, 0.05, rows)):
        qq = rnd(g, q, 128, d, dtype=dtype)
        k = (rnd(g, 1, 32, rows, d) * ramp.cuda()[:, None]).to(dtype)
        v = rnd(g, 1, 32, rows, d, dtype=dtype)
        out = torch.empty_like(qq)
        wr.window_attention(qq, k, v, out, i32([rows]), 100000, 0, False, scale=1.0)
        wr.close(out, *wr.attention64(qq, k, v, [q], [rows], 100000, scale=1.0))


@pytest.mark.parametrize("dtype,d,q,hq,hkv", [(BF16, 128, 256, 64, 16), (F16, 64, 64, 64, 8), (F32, 64, 256, 64, 16)])
def test_many_queries_captured_and_on_two_streams(built, dtype, d, q, hq, hkv):
    """Graphs on two streams replayed at once, with lengths that change between replays."""
    g = gen(24)
    n, rows = 2, q + 1200
    qq = rnd(g, n * q, hq, d, dtype=dtype)
    k, v = rnd(g, n, hkv, rows, d, dtype=dtype), rnd(g, n, hkv, rows, d, dtype=dtype)
    kv_len, outs = i32([q + 200, q + 10]), [torch.zeros_like(qq) for _ in range(3)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs = []
    torch.cuda.synchronize()
    for o, s in zip(outs, streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            for _ in range(4):
                wr.window_attention(qq, k, v, o, kv_len, 900, 4, False)
        graphs.append(graph)
    for lens in ([q + 1200, q + 10], [q, q + 299], [q + 7, 0]):
        kv_len.copy_(i32(lens))
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        wr.window_attention(qq, k, v, outs[2], kv_len, 900, 4, False)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[2])
        wr.close(outs[2], *wr.attention64(qq, k, v, [q] * n, lens, 900, 4))


@pytest.mark.parametrize("dtype,d,q,hq", [(BF16, 128, 300, 64), (F16, 64, 1, 8), (F32, 64, 1, 8), (F32, 64, 300, 64)])
def test_broadcast_cache_and_negative_scale(built, dtype, d, q, hq):
    """One cache expanded over slots and heads (strides of 0), keys in descending rows of memory
    (a negative row stride is no torch tensor: the argument block is changed by hand), and a scale
    below 0."""
    g = gen(25)
    rows = q + 100
    qq = rnd(g, 2 * q, hq, d, dtype=dtype)
    k1, v1 = rnd(g, 1, 1, rows, d, dtype=dtype), rnd(g, 1, 1, rows, d, dtype=dtype)
    k, v = k1.expand(2, hq // 4, rows, d), v1.expand(2, hq // 4, rows, d)
    out = torch.empty_like(qq)
    for scale in (0.1, -0.1):
        wr.window_attention(qq, k, v, out, i32([rows, rows - 5]), 70, 2, False, scale=scale)
        wr.close(out, *wr.attention64(qq, k, v, [q, q], [rows, rows - 5], 70, 2, scale=abs(scale))
                 if scale > 0 else wr.attention64(-qq, k, v, [q, q], [rows, rows - 5], 70, 2, scale=-scale))
    back_k, back_v = k1.flip(2).contiguous(), v1.flip(2).contiguous()
    a = wr.attn_args(qq, back_k.expand(2, hq // 4, rows, d), back_v.expand(2, hq // 4, rows, d), out,
                     i32([rows, rows - 5]), 70, 2)
    last = (rows - 1) * d * qq.element_size()
    a.k, a.v, a.kv_row_stride = a.k + last, a.v + last, -d
    check(load_cuda().armai_dev_window_attention(ctypes.byref(a), wr.stream()))
    wr.close(out, *wr.attention64(qq, k, v, [q, q], [rows, rows - 5], 70, 2))


def test_scale_zero_averages(built):
    """A scale of 0 weighs every visible key alike."""
    g = gen(26)
    for dtype in (BF16, F32):
        qq, k, v = rnd(g, 40, 4, 64, dtype=dtype), rnd(g, 1, 2, 100, 64, dtype=dtype), rnd(g, 1, 2, 100, 64, dtype=dtype)
        out = torch.empty_like(qq)
        wr.window_attention(qq, k, v, out, i32([100]), 30, 2, False, scale=0.0)
        wr.close(out, *wr.attention64(qq, k, v, [40], [100], 30, 2, scale=0.0))


# ---- heads and rows of no whole 16 bytes -------------------------------
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 100), (3, 3, 98), (16, 2, 36), (4, 1, 130), (2, 2, 250), (5, 1, 2), (4, 2, 63)])
@pytest.mark.parametrize("q_lens,past,window,n_sink,ring", [
    ([1, 1, 1, 1], [0, 62, 700, 3099], 1000, 4, False),
    ([1, 1], [5000, 1030], 1024, 0, True),
    ([3, 1, 8], [300, 0, 2], 90, 2, True),
    ([40, 7, 150], [0, 1000, 31], 64, 1, False),
])
def test_heads_of_no_whole_vectors(built, dtype, hq, hkv, d, q_lens, past, window, n_sink, ring):
    run(gen(sum(past) + d), dtype, hq, hkv, d, q_lens, [a + b for a, b in zip(past, q_lens)], window, n_sink, ring,
        extra=2)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d,shift,pad", [(64, 2, 2), (128, 1, 1), (96, 0, 4), (64, 4, 12)])
@pytest.mark.parametrize("q", [1, 90])
def test_tensors_that_are_less_aligned(built, dtype, d, shift, pad, q):
    """Every tensor starts `shift` values behind an aligned address, its rows `pad` values apart."""
    g = gen(d + shift)
    rows = 400

    def view(*shape):
        n = math.prod(shape) * (d + pad) + shift
        return rnd(g, n, dtype=dtype)[shift:].view(*shape, d + pad)[..., :d]

    qq, k, v, out = view(2 * q, 8), view(2, 2, rows), view(2, 2, rows), view(2 * q, 8)
    around = out._base.clone()
    wr.window_attention(qq, k, v, out, i32([rows, 123]), 150, 3, False)
    wr.close(out, *wr.attention64(qq, k, v, [q, q], [rows, 123], 150, 3))
    out.copy_(around[shift:].view(2 * q, 8, d + pad)[..., :d])
    assert torch.equal(out._base, around)  # nothing between the rows was touched
