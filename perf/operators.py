"""The position, head-norm and window-attention operators: the cases they are
measured on, their plain forms and the framework's calls.

  rope    rotary positions: both pair layouts, part of the head, scaled frequencies
  qk      head norms of q and k, the rotation and the append to the key / value cache
  attn    attention with a sliding window and first tokens that stay visible, over
          prompts, chunks and single tokens, from a linear or a ring cache
"""
import ctypes
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 2}
LAYOUTS = {"interleaved": 0, "half": 1}


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------
def _rope(tokens, heads, dim, rot, layout, dtype, first, scaling="none", factor=1.0):
    return dict(op="rope", tokens=tokens, heads=heads, dim=dim, rot=rot, layout=layout, dtype=dtype, first=first,
                scaling=scaling, factor=factor)


def _qk(seqs, q_len, hq, hkv, dim, rot, layout, dtype, kv, first):
    return dict(op="qk", seqs=seqs, q_len=q_len, hq=hq, hkv=hkv, dim=dim, rot=rot, layout=layout, dtype=dtype, kv=kv,
                first=first)


def _attn(seqs, q_min, q_max, hq, hkv, dim, dtype, window, sinks, past, ring):
    return dict(op="attn", seqs=seqs, q_min=q_min, q_max=q_max, hq=hq, hkv=hkv, dim=dim, dtype=dtype, window=window,
                sinks=sinks, past=past, ring=ring)


def listed():
    named = {
        # one token's q and k heads of a 7B-class model, f32 activations as the decode chain keeps them
        "rope_token_f32": _rope(1, 40, 128, 128, "interleaved", "f32", 1500),
        # a long document's q and k, half of each head rotated, context stretched eightfold
        "rope_prompt_bf16": _rope(8191, 40, 128, 64, "half", "bf16", 100000, "turns", 8.0),
        # one token of a 1.1B-class model into its f16 cache
        "qk_token_f32": _qk(1, 1, 32, 4, 64, 64, "interleaved", "f32", "f16", 700),
        # a decode step of a batch of 32
        "qk_batch_bf16": _qk(32, 1, 32, 8, 128, 128, "half", "bf16", "bf16", 6000),
        # a long prompt of odd length
        "qk_prompt_bf16": _qk(1, 16381, 32, 8, 128, 128, "half", "bf16", "bf16", 0),
        # a single stream, its window full, ring cache
        "attn_token_f16": _attn(1, 1, 1, 32, 8, 128, "f16", 4096, 4, 5000, True),
        # a batch of 32 streams at different places, ring cache
        "attn_batch_bf16": _attn(32, 1, 1, 32, 8, 128, "bf16", 4096, 4, 12000, True),
        # a batch of 16 short sequences over the f32 cache (the framework's default cache type)
        "attn_batch_f32": _attn(16, 1, 1, 32, 4, 64, "f32", 512, 4, 640, False),
        # chunks of a few dozen tokens behind a filled window (a turn of a conversation)
        "attn_chunk_f16": _attn(3, 33, 61, 64, 8, 128, "f16", 2048, 4, 6000, True),
        # five ragged prompts of a 1.1B-class model in one call
        "attn_prompts_f16": _attn(5, 37, 1021, 32, 4, 64, "f16", 256, 4, 0, False),
        # a prompt of twice the window
        "attn_prompt_bf16": _attn(1, 8192, 8192, 32, 8, 128, "bf16", 4096, 4, 0, False),
        # f32, a head width that is no power of two
        "attn_prompt_f32": _attn(2, 333, 1000, 8, 2, 80, "f32", 300, 2, 0, False),
    }
    return [{**c, "name": n} for n, c in named.items()]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    dim = rng.choice([64, 128, 128, 80, 96])
    layout = rng.choice(["interleaved", "half"])
    rot = rng.choice([dim, dim, dim // 2])
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([1, 2, 3, 4, 8])
    kind = rng.choice(["rope", "qk", "attn", "attn", "attn"])
    if kind == "rope":
        most = 8191 * 40 * 128 * 2 // (hq * dim * (4 if dtype == "f32" else 2))
        scaling = rng.choice(["none", "linear", "base", "turns"])
        return _rope(_log(rng, 1, min(8191, most)), hq, dim, rot, layout, dtype, _log(rng, 1, 200000), scaling,
                     1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0]))
    if kind == "qk":
        kv = dtype if dtype != "f32" else rng.choice(["f32", "f16"])
        if rng.random() < 0.5:
            return _qk(_log(rng, 1, 64), 1, hq, hkv, dim, rot, layout, dtype, kv, _log(rng, 1, 6000))
        most = 16381 * 48 * 128 * 2 // ((hq + 2 * hkv) * dim * (4 if dtype == "f32" else 2))
        return _qk(1, _log(rng, 16, min(8000, most)), hq, hkv, dim, rot, layout, dtype, kv, rng.choice([0, 100]))
    dim = dim if dtype == "f32" else rng.choice([64, 128])
    window, sinks = _log(rng, 64, 4096), rng.choice([0, 1, 4, 8])
    form = rng.choice(["token", "chunk", "prompt"])
    if form == "token":
        return _attn(_log(rng, 1, 32), 1, 1, hq, hkv, dim, dtype, window, sinks, _log(rng, 1, 12000),
                     rng.choice([True, False]))
    if form == "chunk":
        q = _log(rng, 2, 100)
        return _attn(_log(rng, 1, 8), max(1, q // 2), q, hq, hkv, dim, dtype, window, sinks, _log(rng, 64, 6000), True)
    q = _log(rng, 16, 1024 if dtype == "f32" else 4096)
    return _attn(_log(rng, 1, max(1, min(6, 4096 // q))), max(1, q // 3), q, hq, hkv, dim, dtype, window, sinks, 0,
                 False)


# --------------------------------------------------------------------------
# inputs: what a serving program holds before the call
# --------------------------------------------------------------------------
def _frequencies(case):
    """f32 [rot / 2]; the scaled forms of a longer context than the model was made for."""
    rot, factor, kind = case["rot"], case.get("factor", 1.0), case.get("scaling", "none")
    i = torch.arange(0, rot, 2, dtype=torch.float64)
    base = 10000.0 if kind != "base" else 10000.0 * factor ** (rot / (rot - 2))
    f = base ** (-i / rot)
    if kind == "linear":
        f = f / factor
    if kind == "turns":  # by the turns over the 8192 tokens that the model was made for
        keep = ((8192 * f / (2 * math.pi) - 1.0) / (4.0 - 1.0)).clamp(0.0, 1.0)
        f = f * keep + f / factor * (1.0 - keep)
    return f.float().to(DEV)


def _randn(g, *shape, dtype):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    cg = torch.Generator().manual_seed(seed)
    make = {"rope": _prepare_rope, "qk": _prepare_qk, "attn": _prepare_attn}[case["op"]]
    s = make(case, g, cg)
    s["case"] = case
    s["plan"] = None  # the framework's argument block, filled at the first call and kept beside these buffers
    return s


def _prepare_rope(case, g, cg):
    t, h, d = case["tokens"], case["heads"], case["dim"]
    dt = TYPES[case["dtype"]]
    packed = _randn(g, t, h + 8, d, dtype=dt)  # q and k heads of a packed projection, the values behind them
    pos = case["first"] + int(torch.randint(0, 100, (1,), generator=cg))
    return dict(x=packed[:, :h], pos=pos + torch.arange(t, device=DEV), inv_freq=_frequencies(case),
                mscale=1.0 + 0.1 * math.log(case["factor"]), out=torch.empty(t, h, d, dtype=dt, device=DEV))


def _prepare_qk(case, g, cg):
    n, ql, hq, hkv, d = case["seqs"], case["q_len"], case["hq"], case["hkv"], case["dim"]
    dt, kv = TYPES[case["dtype"]], TYPES[case["kv"]]
    t = n * ql
    qkv = _randn(g, t, hq + 2 * hkv, d, dtype=dt)
    # each sequence somewhere behind `first` tokens; a cache slot of a ring of 256 rows more than a call brings
    past = case["first"] + torch.randint(0, 50, (n, 1), generator=cg)
    pos = past + torch.arange(ql)
    cap = 256 + ql
    rows = torch.arange(n)[:, None] * (hkv * cap) + pos % cap
    k_cache = torch.zeros(n, hkv, cap, d, dtype=kv, device=DEV)
    return dict(qkv=qkv, pos=pos.reshape(-1).to(DEV), rows=rows.reshape(-1).to(DEV), inv_freq=_frequencies(case),
                gq=1.0 + 0.1 * _randn(g, d, dtype=torch.float32), gk=1.0 + 0.1 * _randn(g, d, dtype=torch.float32),
                q_out=torch.empty(t, hq, d, dtype=dt, device=DEV), k_cache=k_cache, v_cache=torch.zeros_like(k_cache))


def _lengths(case):
    """Query counts of the sequences: of the case alone, so that its outputs keep their shapes."""
    pick = random.Random(1000 * case["seqs"] + case["q_max"])
    return [case["q_max"]] + [pick.randint(case["q_min"], case["q_max"]) for _ in range(case["seqs"] - 1)]


def _prepare_attn(case, g, cg):
    n, hq, hkv, d = case["seqs"], case["hq"], case["hkv"], case["dim"]
    dt, w, ns = TYPES[case["dtype"]], case["window"], case["sinks"]
    q_len = torch.tensor(_lengths(case))
    past = torch.randint(case["past"] // 2, case["past"] + 1, (n,), generator=cg)
    past[-1] = case["past"]
    kv_len = past + q_len
    if case["ring"]:
        cap = ns + -(-(w + case["q_max"]) // 64) * 64
    else:
        cap = -(-(case["past"] + case["q_max"]) // 64) * 64
    q_start = torch.zeros(n + 1, dtype=torch.int64)
    q_start[1:] = q_len.cumsum(0)
    t = int(q_start[-1])
    return dict(q=_randn(g, t, hq, d, dtype=dt), k=_randn(g, n, hkv, cap, d, dtype=dt),
                v=_randn(g, n, hkv, cap, d, dtype=dt), q_start=q_start.to(DEV, torch.int32),
                kv_len=kv_len.to(DEV, torch.int32), out=torch.empty(t, hq, d, dtype=dt, device=DEV),
                scale=d ** -0.5)


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        return {"rope": _own_rope, "qk": _own_qk, "attn": _own_attn}[case["op"]](state, case)
    return {"rope": _plain_rope, "qk": _plain_qk, "attn": _plain_attn}[case["op"]](state, case)


def _rotate(x, pos, inv_freq, layout, mscale):
    """x f32 [t, h, d]: the first 2 * len(inv_freq) values of each head rotated."""
    angle = pos.double()[:, None] * inv_freq.double()
    c, s = (angle.cos() * mscale).float()[:, None], (angle.sin() * mscale).float()[:, None]
    rot = 2 * inv_freq.numel()
    part = x[..., :rot]
    a, b = (part[..., 0::2], part[..., 1::2]) if layout == "interleaved" else part.chunk(2, -1)
    a, b = a * c - b * s, a * s + b * c
    part = torch.stack((a, b), -1).flatten(-2) if layout == "interleaved" else torch.cat((a, b), -1)
    return torch.cat((part, x[..., rot:]), -1)


def _plain_rope(st, case):
    return _rotate(st["x"].float(), st["pos"], st["inv_freq"], case["layout"], st["mscale"]).to(st["x"].dtype)


def _plain_qk(st, case):
    hq, hkv, d = case["hq"], case["hkv"], case["dim"]
    x = st["qkv"].float()
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + 1e-5) * st["gq"]
    k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + 1e-5) * st["gk"]
    q = _rotate(q, st["pos"], st["inv_freq"], case["layout"], 1.0).to(st["qkv"].dtype)
    k = _rotate(k, st["pos"], st["inv_freq"], case["layout"], 1.0)
    cap = st["k_cache"].shape[2]
    rows = st["rows"][:, None] + torch.arange(hkv, device=DEV) * cap
    st["k_cache"].view(-1, d)[rows] = k.to(st["k_cache"].dtype)
    st["v_cache"].view(-1, d)[rows] = v.to(st["v_cache"].dtype)
    return q, st["k_cache"], st["v_cache"]


def _plain_attn(st, case):
    n, hq, hkv, d = case["seqs"], case["hq"], case["hkv"], case["dim"]
    w, ns, lq = case["window"], case["sinks"], case["q_max"]
    k, v, q_start, kv_len = st["k"], st["v"], st["q_start"].long(), st["kv_len"].long()
    cap = k.shape[2]
    # queries padded to [n, lq]
    q_len = q_start[1:] - q_start[:-1]
    i = torch.arange(lq, device=DEV)
    tok = (q_start[:-1, None] + i).clamp(max=st["q"].shape[0] - 1)
    q_pos = (kv_len - q_len)[:, None] + i
    q = st["q"][tok].float().view(n, lq, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(n, hkv, -1, d)
    # the positions that any query of a sequence can see: all, or the first ones and the last w + lq - 1
    if case["past"] + lq <= ns + w + lq - 1:
        k_pos = torch.arange(case["past"] + lq, device=DEV).expand(n, -1)
    else:
        first = torch.arange(ns, device=DEV).expand(n, -1)
        last = (kv_len - q_len)[:, None] - w + 1 + torch.arange(w + lq - 1, device=DEV)
        k_pos = torch.cat((first, torch.where(last < ns, 1 << 40, last)), 1)
    row = torch.where(k_pos < ns, k_pos, ns + (k_pos - ns) % (cap - ns)) if case["ring"] else k_pos
    row = row.clamp(max=cap - 1)
    seq = torch.arange(n, device=DEV)[:, None]
    kk = k.transpose(1, 2)[seq, row].float().transpose(1, 2)
    vv = v.transpose(1, 2)[seq, row].float().transpose(1, 2)
    s = (torch.matmul(q, kk.transpose(-1, -2)) * st["scale"]).view(n, hkv, hq // hkv, lq, -1)
    kp, qp = k_pos[:, None, :], q_pos[:, :, None]
    seen = (kp <= qp) & ((kp > qp - w) | (kp < ns)) & (kp < kv_len[:, None, None])
    s = s.masked_fill(~seen[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == float("-inf"), 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n, hkv, -1, p.shape[-1]), vv).view(n, hkv, hq // hkv, lq, d)
    o = torch.where(total > 0, o / total, 0.0)
    o = o.permute(0, 3, 1, 2, 4).reshape(n, lq, hq, d)
    # back to the ragged rows
    t = torch.arange(st["q"].shape[0], device=DEV)
    b = torch.searchsorted(q_start[1:], t, right=True)
    return o[b, t - q_start[b]].to(st["q"].dtype)


# ---- the framework's calls -------------------------------------------------
def _call(fn, plan):
    from arm_ai_b200._lib import check
    check(fn(ctypes.byref(plan), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))


def _own_rope(st, case):
    from arm_ai_b200._lib import RopeArgs, load_cuda
    x, out = st["x"], st["out"]
    if st["plan"] is None:
        st["plan"] = RopeArgs(
            x=x.data_ptr(), out=out.data_ptr(), positions=st["pos"].data_ptr(), inv_freq=st["inv_freq"].data_ptr(),
            n_tokens=case["tokens"], n_heads=case["heads"], head_dim=case["dim"], rot_dim=case["rot"],
            x_token_stride=x.stride(0), x_head_stride=x.stride(1), out_token_stride=out.stride(0),
            out_head_stride=out.stride(1), mscale=st["mscale"], dtype=CODES[case["dtype"]],
            layout=LAYOUTS[case["layout"]])
    _call(load_cuda().armai_dev_rope, st["plan"])
    return out


def _own_qk(st, case):
    from arm_ai_b200._lib import QkNormRopeArgs, load_cuda
    qkv, q_out, kc, vc = st["qkv"], st["q_out"], st["k_cache"], st["v_cache"]
    if st["plan"] is None:
        hq, hkv, d = case["hq"], case["hkv"], case["dim"]
        es = qkv.element_size()
        st["plan"] = QkNormRopeArgs(
            q=qkv.data_ptr(), k=qkv.data_ptr() + hq * d * es, v=qkv.data_ptr() + (hq + hkv) * d * es,
            q_out=q_out.data_ptr(), k_out=kc.data_ptr(), v_out=vc.data_ptr(), q_gamma=st["gq"].data_ptr(),
            k_gamma=st["gk"].data_ptr(), positions=st["pos"].data_ptr(), inv_freq=st["inv_freq"].data_ptr(),
            kv_rows=st["rows"].data_ptr(), n_tokens=qkv.shape[0], n_q_heads=hq, n_kv_heads=hkv, head_dim=d,
            rot_dim=case["rot"], token_stride=qkv.stride(0), head_stride=qkv.stride(1),
            q_out_token_stride=q_out.stride(0), q_out_head_stride=q_out.stride(1), kv_row_stride=d,
            kv_head_stride=kc.stride(1), n_rows=(case["seqs"] - 1) * hkv * kc.shape[2] + kc.shape[2], eps=1e-5,
            mscale=1.0, dtype=CODES[case["dtype"]], kv_dtype=CODES[case["kv"]], layout=LAYOUTS[case["layout"]])
    _call(load_cuda().armai_dev_qk_norm_rope, st["plan"])
    return q_out, kc, vc


def _own_attn(st, case):
    from arm_ai_b200._lib import WindowAttentionArgs, load_cuda
    q, k, out = st["q"], st["k"], st["out"]
    if st["plan"] is None:
        st["plan"] = WindowAttentionArgs(
            q=q.data_ptr(), k=k.data_ptr(), v=st["v"].data_ptr(), out=out.data_ptr(),
            q_start=st["q_start"].data_ptr(), kv_len=st["kv_len"].data_ptr(), slots=None, n_seq=case["seqs"],
            max_q=case["q_max"], n_tokens=q.shape[0], n_q_heads=case["hq"], n_kv_heads=case["hkv"],
            head_dim=case["dim"], q_token_stride=q.stride(0), q_head_stride=q.stride(1),
            out_token_stride=out.stride(0), out_head_stride=out.stride(1), kv_slot_stride=k.stride(0),
            kv_head_stride=k.stride(1), kv_row_stride=k.stride(2), n_slots=k.shape[0], kv_rows=k.shape[2],
            window=case["window"], n_sink=case["sinks"], ring=int(case["ring"]), scale=st["scale"],
            dtype=CODES[case["dtype"]])
    _call(load_cuda().armai_dev_window_attention, st["plan"])
    return out


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------
def _size(name):
    return 4 if name == "f32" else 2


def work(case):
    if case["op"] == "rope":
        values = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 2 * values * _size(case["dtype"]) + 8 * case["tokens"] + 2 * case["rot"],
                "flops": 3 * case["tokens"] * case["heads"] * case["rot"]}
    if case["op"] == "qk":
        t, d, hq, hkv = case["seqs"] * case["q_len"], case["dim"], case["hq"], case["hkv"]
        es, kv = _size(case["dtype"]), _size(case["kv"])
        return {"bytes": t * d * ((2 * hq + 2 * hkv) * es + 2 * hkv * kv) + 16 * t + 2 * case["rot"] + 8 * d,
                "flops": t * (hq + hkv) * (4 * d + 3 * case["rot"])}
    # attention: the keys before the call at the middle of their range
    n, w, ns, es, d = case["seqs"], case["window"], case["sinks"], _size(case["dtype"]), case["dim"]
    past = case["past"] * 0.75 if n > 1 else case["past"]
    keys = pairs = 0
    for q in _lengths(case):
        full = max(0, min(q, past + q - ns - w))  # queries whose window is full
        grow = q - full
        keys += min(past + q, ns + w + q - 1)
        pairs += full * (w + ns) + grow * (past + (grow + 1) / 2)
    return {"bytes": es * d * (2 * sum(_lengths(case)) * case["hq"] + 2 * keys * case["hkv"]),
            "flops": 4 * d * pairs * case["hq"]}


# --------------------------------------------------------------------------
# the definitions in 64 bits
# --------------------------------------------------------------------------
def _turn64(x, pos, inv_freq, layout, mscale):
    """Each pair as a complex number, turned by its angle."""
    rot = 2 * inv_freq.numel()
    unit = mscale * torch.exp(1j * (pos.double()[:, None] * inv_freq.double()[None, :]))
    out = x.double().clone()
    first, second = ((slice(0, rot, 2), slice(1, rot, 2)) if layout == "interleaved"
                     else (slice(0, rot // 2), slice(rot // 2, rot)))
    z = torch.complex(out[..., first].contiguous(), out[..., second].contiguous()) * unit[:, None, :]
    out[..., first], out[..., second] = z.real, z.imag
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "rope":
        return _turn64(st["x"], st["pos"], st["inv_freq"], case["layout"], st["mscale"])
    if case["op"] == "qk":
        hq, hkv = case["hq"], case["hkv"]
        q, k, v = st["qkv"].double().split([hq, hkv, hkv], 1)
        q, k = (y / torch.linalg.vector_norm(y, dim=-1, keepdim=True).square().div(y.shape[-1]).add(1e-5).sqrt() * g
                for y, g in ((q, st["gq"].double()), (k, st["gk"].double())))
        q, k = (_turn64(y, st["pos"], st["inv_freq"], case["layout"], 1.0) for y in (q, k))
        kc, vc = st["k_cache"].double(), st["v_cache"].double()
        cap = kc.shape[2]
        slot, row = st["rows"] // (hkv * cap), st["rows"] % cap
        for h in range(hkv):
            kc[slot, h, row], vc[slot, h, row] = k[:, h], v[:, h]
        return q, kc, vc
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    w, ns, cap, group = case["window"], case["sinks"], st["k"].shape[2], case["hq"] // case["hkv"]
    starts, lens = st["q_start"].tolist(), st["kv_len"].tolist()
    for b in range(case["seqs"]):
        a, e = starts[b], starts[b + 1]
        p = torch.arange(lens[b] - (e - a), lens[b], device=DEV)
        j = torch.arange(lens[b], device=DEV)
        j = j[(j < ns) | (j > int(p[0]) - w)]
        rows = torch.where(j < ns, j, (j - ns) % (cap - ns) + ns) if case["ring"] else j
        hidden = (j[None] > p[:, None]) | ((j[None] <= p[:, None] - w) & (j[None] >= ns))
        for h in range(case["hq"]):
            kd, vd = st["k"][b, h // group, rows].double(), st["v"][b, h // group, rows].double()
            s = st["q"][a:e, h].double() @ kd.T * st["scale"]
            s[hidden] = -math.inf
            out[a:e, h] = torch.softmax(s, -1) @ vd
    return out
