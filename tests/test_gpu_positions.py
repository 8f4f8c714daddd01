"""Rotary positions (armai_dev_rope) and the head norms of q and k with the
rotation and the cache append (armai_dev_qk_norm_rope) against their
definitions in f64.

Tolerances. A turned pair of length L: cos and sin are off by at most the f32
rounding of a remainder below half a turn (pi * 2^-24 = 1.9e-7) plus two steps
of sincospi (1.2e-7), the products and their sum by 3 * 2^-24: together below
6e-7 L. A norm multiplies by an inverse root whose sum of at most 256 squares
is added in a tree of at most 8 + 5 levels (13 * 2^-24, halved by the root),
with a root, a division and two products: below 1.5e-6. Then one rounding to
the output's type.
"""
import ctypes

import pytest

torch = pytest.importorskip("torch")

import window_reference as wr
from arm_ai_b200 import prims
from arm_ai_b200._lib import load_cuda

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TURN, NORM = 6e-7, 1.5e-6


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rnd(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def freqs(rot, **kw):
    return torch.from_numpy(prims.rope_frequencies(rot, **kw)).cuda()


def rope_close(got, exact, size, mscale=1.0, more=0.0):
    tol = (TURN + more) * size * mscale + wr.half_step(got.dtype) * exact.abs() + torch.finfo(got.dtype).tiny
    return wr.close(got, exact, tol)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("tokens,heads,dim,rot", [
    (1, 1, 2, 2), (1, 40, 128, 128), (5, 3, 64, 32), (700, 9, 128, 64), (33, 2, 80, 80), (7, 5, 96, 48),
    (3, 7, 50, 18), (4, 2, 256, 256), (2, 1, 7, 6), (6, 33, 64, 0), (1200, 40, 64, 64), (2, 3, 1, 0)])
def test_rope_matches_definition(built, dtype, layout, tokens, heads, dim, rot):
    g = gen(tokens * 1000 + dim + rot)
    x = rnd(g, tokens, heads, dim, dtype=dtype)
    pos = torch.randint(0, 200000, (tokens,), generator=g, device="cuda")
    f = freqs(rot)
    out = torch.empty_like(x)
    wr.rope(x, out, pos, f, layout, mscale=1.2)
    exact, size = wr.rotate64(x, pos, f, layout, 1.2)
    rope_close(out, exact, size, 1.2)
    assert torch.equal(out[..., rot:], x[..., rot:])


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype,dim,rot", [(BF16, 128, 128), (F32, 50, 20), (F16, 80, 80)])
def test_rope_in_place_strided_and_back(built, layout, dtype, dim, rot):
    """Heads of a packed projection turned in place (their neighbours untouched), and back by
    negated positions."""
    g = gen(3)
    packed = rnd(g, 77, 9, dim, dtype=dtype)
    before = packed.clone()
    x = packed[:, 2:7]
    pos = torch.randint(0, 5000, (77,), generator=g, device="cuda")
    f = freqs(rot)
    wr.rope(x, x, pos, f, layout)
    exact, size = wr.rotate64(before[:, 2:7], pos, f, layout)
    rope_close(x, exact, size)
    assert torch.equal(packed[:, :2], before[:, :2]) and torch.equal(packed[:, 7:], before[:, 7:])
    turned = x.clone()
    wr.rope(x, x, -pos, f, layout)
    exact, size = wr.rotate64(turned, -pos, f, layout)
    rope_close(x, exact, size)
    # there and back: two roundings of the type and two turns
    tol = 2 * (TURN + wr.half_step(dtype)) * size * 1.5 + torch.finfo(dtype).tiny
    wr.close(x, before[:, 2:7].double(), tol)


def test_rope_unaligned_rows(built):
    """Rows that start off a 16-byte boundary, or whose pitch is odd, give the same values."""
    g = gen(4)
    f, pos = freqs(64), torch.arange(9, device="cuda") * 1000
    x = rnd(g, 9, 3, 64, dtype=BF16)
    want = torch.empty_like(x)
    wr.rope(x, want, pos, f, "half")
    flat = torch.zeros(9 * 3 * 67 + 8, dtype=BF16, device="cuda")
    y = flat[1:1 + 9 * 3 * 67].view(9, 3, 67)[..., :64]
    y.copy_(x)
    wr.rope(y, y, pos, f, "half")
    assert (y.double() - want.double()).abs().max().item() <= 2 * wr.half_step(BF16) * want.abs().max().item()


def test_rope_far_positions(built):
    """Positions up to 2^40: the angle is reduced in f64, not rounded to f32."""
    g = gen(5)
    x = rnd(g, 6, 2, 128)
    pos = torch.tensor([0, 1, 1 << 20, (1 << 24) + 1, (1 << 31) + 12345, -(1 << 20)], device="cuda")
    f = freqs(128)
    out = torch.empty_like(x)
    wr.rope(x, out, pos, f, "half")
    exact, size = wr.rotate64(x, pos, f, "half")
    # the f64 angle itself: 2^-53 of up to 2^31 rad on both sides
    rope_close(out, exact, size, more=2.0 ** -20)
    near = pos.abs() <= (1 << 24) + 1
    rope_close(out[near], exact[near], size[near])


def test_rope_host_form(built):
    g = gen(6)
    x, pos, f = rnd(g, 5, 3, 48), torch.tensor([0, 7, 100, 5, 9]), freqs(20)
    got = prims.rope_ext_f32_op(x.cpu().numpy(), pos.numpy(), f.cpu().numpy(), 15, 48, 3, layout="half", mscale=0.5)
    exact, size = wr.rotate64(x, pos.cuda(), f, "half", 0.5)
    rope_close(torch.from_numpy(got).cuda().view(5, 3, 48), exact, size, 0.5)
    # the plain form of the reference, where it computes the same: interleaved, whole heads, near positions
    want = prims.rope_f32_op(x.cpu().numpy(), pos.numpy(), freqs(48).cpu().numpy(), 15, 48, 3)
    got = prims.rope_ext_f32_op(x.cpu().numpy(), pos.numpy(), freqs(48).cpu().numpy(), 15, 48, 3)
    # its angle is rounded to f32: 2^-24 of up to 100 rad, on pairs below 5
    assert abs(got - want).max() <= 5 * (100 * 2.0 ** -24 + 1e-6)


@pytest.mark.parametrize("dtype,kv", [(F32, F32), (F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("tokens,hq,hkv,dim,rot", [
    (1, 32, 4, 64, 64), (32, 32, 8, 128, 128), (3, 6, 2, 80, 40), (2, 3, 1, 33, 10), (900, 8, 8, 128, 64),
    (5, 2, 2, 256, 256), (4, 7, 0, 64, 64), (4, 0, 3, 64, 32)])
def test_qk_norm_rope_matches_definition(built, dtype, kv, layout, tokens, hq, hkv, dim, rot):
    g = gen(tokens + dim + hq)
    qkv = rnd(g, tokens, hq + 2 * hkv, dim, dtype=dtype)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    gq, gk = 1 + 0.1 * rnd(g, dim), 1 + 0.1 * rnd(g, dim)
    pos = torch.randint(0, 100000, (tokens,), generator=g, device="cuda")
    f = freqs(rot)
    slots, cap = 3, tokens + 2
    kc = torch.full((slots, max(hkv, 1), cap, dim), 7.0, dtype=kv, device="cuda")
    vc = torch.full_like(kc, 7.0)
    # tokens in a random order of slots and rows; every third is padding
    where = torch.randperm(slots * cap, generator=g, device="cuda")[:tokens]
    slot, row = where // cap, where % cap
    rows = slot * (max(hkv, 1) * cap) + row
    pad = torch.arange(tokens, device="cuda") % 3 == 2
    rows = torch.where(pad, -1, rows)
    q_out = torch.empty(tokens, hq, dim, dtype=dtype, device="cuda")
    wr.qk_norm_rope(q, k, v, q_out, kc, vc, gq, gk, pos, f, rows, layout)
    for got, x, gam in ((q_out, q, gq), (None, k, gk)):
        if x.shape[1] == 0:
            continue
        exact, size = wr.rotate64(wr.norm64(x, gam, 1e-5), pos, f, layout)
        if got is None:
            got, exact, size = kc[slot, :, row][~pad], exact[~pad], size[~pad]
        rope_close(got, exact, size, more=NORM)
    if hkv:
        assert torch.equal(vc[slot, :, row][~pad], v[~pad].to(kv))
    written = torch.zeros(slots, cap, dtype=torch.bool, device="cuda")
    if hkv:
        written[slot[~pad], row[~pad]] = True
    for c in (kc, vc):  # every other row as it was
        assert (c.transpose(1, 2)[~written] == 7.0).all()


def test_qk_rows_outside_the_cache_are_skipped(built):
    g = gen(8)
    qkv = rnd(g, 4, 4, 64, dtype=BF16)
    out = torch.zeros(3, 1, 64, dtype=BF16, device="cuda")
    spare = torch.zeros(64, 1, 64, dtype=BF16, device="cuda")  # rows behind n_rows, inside the allocation
    whole = torch.cat((out, spare))
    vw = torch.zeros_like(whole)
    rows = torch.tensor([0, 3, -5, 50], device="cuda")
    q_out = torch.empty(4, 2, 64, dtype=BF16, device="cuda")
    wr.qk_norm_rope(qkv[:, :2], qkv[:, 2:3], qkv[:, 3:], q_out, whole[:3], vw[:3], None, None,
                    torch.arange(4, device="cuda"), freqs(64), rows, "half")
    assert torch.equal(vw[0], qkv[0, 3:]) and not vw[1:].any() and not whole[1:].any()


@pytest.mark.parametrize("scale", [1e-30, 1.0, 1e15])
def test_qk_norm_of_tiny_zero_and_large_rows(built, scale):
    g = gen(9)
    x = rnd(g, 3, 2, 64) * scale
    x[1] = 0
    one = torch.ones(64, device="cuda")
    pos, f = torch.arange(3, device="cuda"), freqs(64)
    q_out, k_out = torch.empty(3, 1, 64, device="cuda"), torch.empty(3, 1, 64, device="cuda")
    wr.qk_norm_rope(x[:, :1], x[:, 1:], None, q_out, k_out, None, one, one, pos, f, None, "half")
    exact, size = wr.rotate64(wr.norm64(x, one, 1e-5), pos, f, "half")
    rope_close(torch.cat((q_out, k_out), 1), exact, size, more=NORM)


def test_qk_host_form(built):
    g = gen(10)
    q, k = rnd(g, 6, 4, 64), rnd(g, 6, 2, 64)
    gq, gk, pos, f = 1 + rnd(g, 64) * 0.1, 1 + rnd(g, 64) * 0.1, torch.arange(6) * 11, freqs(32)
    got = prims.qk_norm_rope_f32_op(*(t.cpu().numpy() for t in (q, k, gq, gk, pos, f)), 4, 2, 64)
    for o, x, gam in zip(got, (q, k), (gq, gk)):
        exact, size = wr.rotate64(wr.norm64(x, gam, 1e-5), pos.cuda(), f, "half")
        rope_close(torch.from_numpy(o).cuda().view(x.shape), exact, size, more=NORM)


def test_rope_captured_on_another_stream(built):
    """Captured into a graph on a side stream and replayed on new data."""
    g = gen(11)
    x = rnd(g, 16, 8, 128, dtype=BF16)
    pos, f = torch.arange(16, device="cuda"), freqs(128)
    out = torch.zeros_like(x)
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        wr.rope(x, out, pos, f, "half")
    x.copy_(rnd(g, 16, 8, 128, dtype=BF16))
    pos.add_(100)
    graph.replay()
    exact, size = wr.rotate64(x, pos, f, "half")
    rope_close(out, exact, size)


def test_device_checks_refuse_host_tensors(built):
    x = torch.zeros(1, 1, 64)
    a = wr.rope_args(x, x, torch.zeros(1, dtype=torch.int64), torch.zeros(32), "half")
    lib = load_cuda()
    assert lib.armai_dev_rope(ctypes.byref(a), None) == -1
    assert b"rope: x is not device memory" in lib.armai_last_error()
    d = torch.zeros(1, 1, 64, device="cuda")
    a = wr.rope_args(d, d, torch.zeros(1, dtype=torch.int64), torch.zeros(32), "half")
    assert lib.armai_dev_rope(ctypes.byref(a), None) == -1
    assert b"rope: positions is not device memory" in lib.armai_last_error()


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype,dim,rot", [(F32, 64, 32), (BF16, 128, 64), (F16, 128, 20), (F32, 33, 10)])
def test_infinities_stay_in_their_pair(built, layout, dtype, dim, rot):
    """An infinity or NaN reaches its own pair (its head, through the norm) and nothing else."""
    g = gen(30)
    x = rnd(g, 5, 4, dim, dtype=dtype)
    x[1, 2, 0], x[2, 1, dim - 1], x[3, 0, 1] = float("inf"), float("-inf"), float("nan")
    pos, f = torch.arange(5, device="cuda") + 3, freqs(rot)
    out = torch.empty_like(x)
    wr.rope(x, out, pos, f, layout)
    clean = torch.where(torch.isfinite(x.float()), x, 0.0)
    want = torch.empty_like(x)
    wr.rope(clean, want, pos, f, layout)
    partner = {0: 1, 1: 0} if layout == "interleaved" else {0: rot // 2, 1: 1 + rot // 2}
    touched = torch.zeros(x.shape, dtype=torch.bool, device="cuda")
    touched[1, 2, 0] = touched[1, 2, partner[0]] = touched[2, 1, dim - 1] = touched[3, 0, 1] = True
    touched[3, 0, partner[1]] = True
    assert torch.equal(out[~touched], want[~touched])
    assert not torch.isfinite(out[touched].float()).any()
    one = torch.ones(dim, device="cuda")
    q_out, k_out = torch.empty(5, 2, dim, dtype=dtype, device="cuda"), torch.empty(5, 2, dim, dtype=dtype, device="cuda")
    wr.qk_norm_rope(x[:, :2], x[:, 2:], None, q_out, k_out, None, one, one, pos, f, None, layout)
    bad = ~torch.isfinite(x.float()).all(-1)
    assert torch.isfinite(torch.cat((q_out, k_out), 1)[~bad].float()).all()


def test_many_tokens_share_the_warps(built):
    """More tokens than the device's warps, odd counts: each warp goes through several tokens."""
    g = gen(31)
    for tokens, hq, hkv, dim, layout in ((9001, 5, 3, 64, "half"), (3999, 9, 1, 96, "interleaved"), (5000, 2, 2, 256, "half")):
        qkv = rnd(g, tokens, hq + 2 * hkv, dim, dtype=BF16)
        gq, gk = 1 + 0.1 * rnd(g, dim), 1 + 0.1 * rnd(g, dim)
        pos, f = torch.randint(0, 1 << 20, (tokens,), generator=g, device="cuda"), freqs(dim)
        q_out = torch.empty(tokens, hq, dim, dtype=BF16, device="cuda")
        k_out, v_out = (torch.empty(tokens, hkv, dim, dtype=BF16, device="cuda") for _ in range(2))
        q, k, v = qkv.split([hq, hkv, hkv], 1)
        wr.qk_norm_rope(q, k, v, q_out, k_out, v_out, gq, gk, pos, f, None, layout)
        for got, x, gam in ((q_out, q, gq), (k_out, k, gk)):
            exact, size = wr.rotate64(wr.norm64(x, gam, 1e-5), pos, f, layout)
            rope_close(got, exact, size, more=NORM)
        assert torch.equal(v_out, v)


# ---- vectors narrower than 16 bytes ------------------------------------
NARROW = [(9, 5, 80, 40), (3000, 3, 80, 40), (5, 2, 100, 100), (1100, 9, 100, 36), (4, 3, 52, 20), (2, 1, 4, 4),
          (3, 2, 12, 8), (600, 7, 132, 132), (70, 3, 248, 124), (65, 33, 18, 10)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("tokens,heads,dim,rot", NARROW)
def test_rope_of_narrow_vectors(built, dtype, layout, tokens, heads, dim, rot):
    test_rope_matches_definition(built, dtype, layout, tokens, heads, dim, rot)


@pytest.mark.parametrize("dtype,kv", [(F32, F32), (F32, F16), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("tokens,hq,hkv,dim,rot", [(700, 6, 2, 80, 40), (5, 3, 1, 100, 100), (333, 4, 4, 100, 36),
                                                  (40, 2, 1, 52, 20), (3, 2, 2, 248, 124)])
def test_qk_norm_rope_of_narrow_vectors(built, dtype, kv, layout, tokens, hq, hkv, dim, rot):
    test_qk_norm_rope_matches_definition(built, dtype, kv, layout, tokens, hq, hkv, dim, rot)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("shift,pad", [(4, 4), (2, 2), (1, 1), (0, 6), (8, 4)])
@pytest.mark.parametrize("tokens", [3, 800])
def test_rope_of_tensors_that_are_less_aligned(built, dtype, layout, shift, pad, tokens):
    """Heads that start `shift` values behind an aligned address, `pad` values apart, in and out of place."""
    g = gen(shift + pad)
    buf = rnd(g, tokens * 3 * (64 + pad) + shift, dtype=dtype)
    x = buf[shift:].view(tokens, 3, 64 + pad)[..., :64]
    pos = torch.randint(0, 9000, (tokens,), generator=g, device="cuda")
    f = freqs(48)
    exact, size = wr.rotate64(x, pos, f, layout)
    before = buf.clone()
    out = torch.empty(tokens, 3, 64, dtype=dtype, device="cuda")
    wr.rope(x, out, pos, f, layout)
    rope_close(out, exact, size)
    wr.rope(x, x, pos, f, layout)
    assert torch.equal(x, out)
    x.copy_(before[shift:].view(tokens, 3, 64 + pad)[..., :64])
    assert torch.equal(buf, before)  # nothing between the heads was touched
