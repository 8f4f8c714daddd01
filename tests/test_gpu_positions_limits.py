"""Rotary positions and head norms at the limits of their arguments, against
their definitions in f64 (tolerances as in test_gpu_positions)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import window_reference as wr
from test_gpu_positions import NORM, freqs, gen, rnd, rope_close

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("tokens,hq,hkv,dim,rot", [(3000, 3, 0, 64, 64), (3000, 0, 3, 64, 32), (2500, 1, 0, 128, 64),
                                                  (5, 1, 0, 64, 64), (2, 0, 1, 128, 128), (2600, 0, 2, 100, 36),
                                                  (2600, 5, 0, 33, 10)])
def test_tensors_without_heads(built, dtype, layout, tokens, hq, hkv, dim, rot):
    """q alone or k alone, by few tokens and by many; nothing of the other tensor is needed."""
    g = gen(tokens + hq)
    x = rnd(g, tokens, max(hq, hkv), dim, dtype=dtype)
    none = x[:, :0]
    gam = 1 + 0.1 * rnd(g, dim)
    pos, f = torch.randint(0, 50000, (tokens,), generator=g, device="cuda"), freqs(rot)
    out, spare = torch.empty_like(x), torch.empty(tokens, 0, dim, dtype=dtype, device="cuda")
    rows = torch.randperm(tokens, generator=g, device="cuda")
    a = wr.qk_args(*((x, none, none, out, spare, spare) if hq else (none, x, None, spare, out, None)), gam, gam, pos, f,
                   rows if hkv else None, layout)
    if not hq:  # strides of the tensor that has heads
        a.token_stride, a.head_stride = x.stride(0), x.stride(1)
    wr.check(wr.load_cuda().armai_dev_qk_norm_rope(wr.ctypes.byref(a), wr.stream()))
    exact, size = wr.rotate64(wr.norm64(x, gam, 1e-5), pos, f, layout)
    rope_close(out if hq else out[rows], exact, size, more=NORM)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype,dim", [(F32, 64), (BF16, 128), (F16, 33)])
@pytest.mark.parametrize("tokens", [3, 2000])
def test_frequencies_that_are_no_numbers(built, layout, dtype, dim, tokens):
    """A NaN or infinite frequency makes its own pair NaN at every position (0 times infinity too), as
    the definition does, and no other value."""
    g = gen(dim)
    x = rnd(g, tokens, 3, dim, dtype=dtype)
    pos, f = torch.arange(tokens, device="cuda"), freqs(32)
    bad = f.clone()
    bad[[1, 6, 15]] = torch.tensor([float("nan"), float("inf"), float("-inf")], device="cuda")
    out, want = torch.empty_like(x), torch.empty_like(x)
    wr.rope(x, out, pos, bad, layout)
    wr.rope(x, want, pos, f, layout)
    pairs = torch.zeros(dim, dtype=torch.bool, device="cuda")
    for i in (1, 6, 15):
        pairs[[2 * i, 2 * i + 1] if layout == "interleaved" else [i, i + 16]] = True
    assert torch.isnan(out[..., pairs]).all()
    assert torch.equal(out[..., ~pairs], want[..., ~pairs])


@pytest.mark.parametrize("layout,dim", [("half", 128), ("interleaved", 64), ("half", 33)])
@pytest.mark.parametrize("base,factor", [(10000.0, 1.0), (5e5, 8.0), (10000.0, 0.125)])
def test_positions_up_to_2_40(built, layout, dim, base, factor):
    """The product of a 40-bit position and a 24-bit frequency is exact in 64 bits, where its cosine
    and sine are taken; the kernel's angle may be off by 2^-60 rad per position on top of a turn's
    other roundings."""
    assert np.finfo(np.longdouble).nmant >= 63
    g = gen(dim)
    pos = [0, 1, -1, 1 << 24, (1 << 31) + 12345, -(1 << 33) - 7, (1 << 36) + 1, (1 << 39) + 987654321, (1 << 40) - 1,
           1 - (1 << 40)]
    f = freqs(dim // 2 * 2, base=base, scaling="linear", factor=factor)
    x = rnd(g, len(pos), 2, dim)
    pos = torch.tensor(pos, device="cuda")
    out = torch.empty_like(x)
    wr.rope(x, out, pos, f, layout)
    ang = pos.cpu().numpy().astype(np.longdouble)[:, None] * f.cpu().numpy().astype(np.longdouble)
    c, s = (torch.from_numpy(t.astype(np.float64)).cuda()[:, None] for t in (np.cos(ang), np.sin(ang)))
    r = dim // 2
    a, b = ((x[..., 0:2 * r:2], x[..., 1:2 * r:2]) if layout == "interleaved" else (x[..., :r], x[..., r:2 * r]))
    a, b = a.double(), b.double()
    want, size = torch.stack((a * c - b * s, a * s + b * c), -1), torch.hypot(a, b)[..., None].expand(-1, -1, -1, 2)
    got = (torch.stack((out[..., 0:2 * r:2], out[..., 1:2 * r:2]), -1) if layout == "interleaved"
           else torch.stack((out[..., :r], out[..., r:2 * r]), -1))
    rope_close(got, want, size, more=pos.abs().double()[:, None, None, None] * 2.0 ** -60)
