"""Rotary positions and head norms at the limits of their arguments, against
their definitions in f64 (tolerances as in test_gpu_positions)."""
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
