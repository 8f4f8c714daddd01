"""Window attention at the limits of its types and lengths, against its
definition in f64 (window_reference.attention64): weights far below a row's
largest."""
import pytest

torch = pytest.importorskip("torch")

import window_reference as wr
from arm_ai_b200._lib import check, load_cuda

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("q,hq,hkv,d", [(1, 8, 2, 64), (1, 8, 8, 128), (1, 2, 1, 100), (20, 4, 2, 256), (300, 128, 32, 64),
                                        (300, 128, 32, 128), (70, 32, 4, 128), (200, 8, 2, 256)])
@pytest.mark.parametrize("gap", [8.0, 12.0, 14.5, 17.0])
def test_first_token_far_above_the_rest(built, dtype, q, hq, hkv, d, gap):
    """The first token's score stands `gap` nats above all others and its value is 0, so the output
    is made of weights of e^-gap alone. They count as the definition has them, to the rounding of
    the weights: half a step of the type, and for f16, whose exponents end, 2^-25 where the row's
    largest weight is 2^7 or more: 2^-32 of the largest."""
    g = gen(int(gap) + d)
    rows = 1300 + q
    k = torch.zeros(1, hkv, rows, d, device="cuda")
    k[..., 0] = 0.01 * torch.randn(1, hkv, rows, generator=g, device="cuda")
    k[:, :, 0, 0] = gap
    v = 1024 * (1 + torch.rand(1, hkv, rows, d, generator=g, device="cuda"))
    v[:, :, 0] = 0
    qq = torch.zeros(q, hq, d, device="cuda")
    qq[..., 0] = 1
    qq, k, v = qq.to(dtype), k.to(dtype), v.to(dtype)
    out = torch.empty_like(qq)
    wr.window_attention(qq, k, v, out, i32([rows]), 1000, 1, False, scale=1.0)
    exact, tol = wr.attention64(qq, k, v, [q], [rows], 1000, 1, scale=1.0)
    assert exact.abs().min().item() > 0.01  # far above the type's smallest values
    if dtype == F16:
        tol += 2.0 ** -32 * v.double().sum(2).amax(1)[0]
    wr.close(out, exact, tol)


def test_status_after_calls(built):
    """No wait has given up in calls of every form: the question is answered, and answered again."""
    lib = load_cuda()
    check(lib.armai_dev_window_attention_status())
    for dtype, q, hq, hkv, d in ((BF16, 400, 64, 16, 128), (F16, 40, 64, 8, 64), (BF16, 1, 8, 2, 128), (F32, 300, 64, 16, 64)):
        g = gen(q)
        qq = torch.randn(q, hq, d, generator=g, device="cuda").to(dtype)
        k, v = (torch.randn(1, hkv, q + 2000, d, generator=g, device="cuda").to(dtype) for _ in range(2))
        out = torch.empty_like(qq)
        wr.window_attention(qq, k, v, out, i32([q + 2000]), 1500, 4, False)
        torch.cuda.synchronize()
        check(lib.armai_dev_window_attention_status())
        assert torch.isfinite(out.float()).all()


@pytest.mark.parametrize("dtype,q,hq,hkv,d", [(BF16, 1, 8, 2, 128), (F32, 1, 4, 2, 64), (F16, 1, 4, 2, 100),
                                              (F16, 300, 64, 16, 64), (BF16, 300, 64, 16, 128), (F32, 300, 64, 16, 80),
                                              (BF16, 90, 8, 2, 256), (F32, 20, 4, 2, 64), (F16, 50, 2, 1, 33)])
@pytest.mark.parametrize("rows,past,window,n_sink", [(400, 90, 100, 2), (400, 390, 64, 0), (310, 900, 200, 3),
                                                     (64, 1500, 70, 0)])
def test_positions_behind_a_linear_cache(built, dtype, q, hq, hkv, d, rows, past, window, n_sink):
    """A linear cache has no row for positions from kv_rows on: they are seen by nobody, the queries
    there see what the cache holds, and nothing is read beyond it."""
    g = gen(rows + d)
    length = past + q
    qq = torch.randn(q, hq, d, generator=g, device="cuda").to(dtype)
    # the cache between rows that nobody may look at
    whole = torch.full((2, 1, hkv, rows + 128, d), float("nan"), dtype=dtype, device="cuda")
    whole[..., 64:64 + rows, :] = torch.randn(2, 1, hkv, rows, d, generator=g, device="cuda").to(dtype)
    k, v = whole[:, :, :, 64:64 + rows]
    out = torch.empty_like(qq)
    wr.window_attention(qq, k, v, out, i32([length]), window, n_sink, False)
    j = torch.arange(rows, device="cuda")
    for i in range(0, q, max(1, q // 9)):
        p = past + i
        keep = (j <= p) & ((j > p - window) | (j < n_sink))
        wr.close(out[i:i + 1], *wr.attention64(qq[i:i + 1], k[:, :, keep].contiguous(), v[:, :, keep].contiguous(), [1],
                                              [int(keep.sum())], 1 << 40))


@pytest.mark.parametrize("dtype,q,hq,hkv,d", [(BF16, 1, 8, 2, 128), (F32, 1, 4, 2, 64), (F16, 1, 4, 2, 100),
                                              (F16, 300, 64, 16, 64), (BF16, 300, 64, 16, 128), (BF16, 40, 64, 8, 128),
                                              (F32, 300, 64, 16, 80), (BF16, 90, 8, 2, 256), (F16, 50, 2, 1, 33)])
@pytest.mark.parametrize("ring", [True, False])
def test_positions_up_to_2_31(built, dtype, q, hq, hkv, d, ring):
    """Sequences as long as kv_len can say: in a ring the same rows, so bit for bit the same output,
    as a whole number of turns before; in a linear cache, far behind its rows, the first tokens."""
    g = gen(d)
    window, n_sink = 700, 3
    turn = window + q + 40
    rows = n_sink + turn
    qq = torch.randn(2 * q, hq, d, generator=g, device="cuda").to(dtype)
    k, v = (torch.randn(2, hkv, rows, d, generator=g, device="cuda").to(dtype) for _ in range(2))
    longest = (1 << 31) - 1
    near = [longest - (longest // turn - 5) * turn, longest - 7 - (longest // turn - 5) * turn]
    outs = []
    for lens in ([longest, longest - 7], near):
        out = torch.full_like(qq, 9.0)
        wr.window_attention(qq, k, v, out, i32(lens), window, n_sink, ring)
        outs.append(out)
    assert torch.equal(*outs) and torch.isfinite(outs[0].float()).all()
    if not ring:
        wr.close(outs[0][:1], *wr.attention64(qq[:1], k[:1, :, :n_sink].contiguous(), v[:1, :, :n_sink].contiguous(), [1],
                                             [n_sink], 100))


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("ctas", [14, 15, 16, 30, 33, 34, 37, 63, 72, 74, 75])
def test_clusters_that_fit_at_once(built, dtype, d, ctas):
    """CTA counts (of four tokens of 64 heads) around those up to which clusters of 8, 4 and 2 run
    all at once; the last CTA has fewer tokens."""
    g = gen(ctas)
    q, past, window, n_sink = 4 * ctas - 1, 1800, 2040, 3
    rows = n_sink + window + q - 1
    qq = torch.randn(q, 64, d, generator=g, device="cuda").to(dtype)
    k, v = (torch.randn(1, 1, rows, d, generator=g, device="cuda").to(dtype) for _ in range(2))
    out = torch.empty_like(qq)
    for length, ring in ((past + q, False), (5000, True)):
        wr.window_attention(qq, k, v, out, i32([length]), window, n_sink, ring)
        wr.close(out, *wr.attention64(qq, k, v, [q], [length], window, n_sink, ring))
