"""Performance cases of the 4-bit paged KV cache (quant_mode "affine4_g64"): a cache
quantized to 4 bits as it is written, read back, and attended over in place.

The cache holds, per token, KV head and group of 64 dims, an fp16 scale s, an fp16 bias b
and 64 codes c of 4 bits; the values they stand for are s c + b:

    b = f16(min w), s = f16((max w - b) / 15), at least 0
    c = clip(rint((w - b) / s), 0, 15), 0 where s = 0

with w the group's elements limited to +-65504.  Kinds of call:

* write   new K/V rows (K rotated by its position first where `rope`) quantized into the
          slots reserved for them, and the stored rows read back from those slots
* read    whole sequences read back as fp16, left- or right-aligned
* step    one decode step: the new token's K/V written and every query attended over its
          sequence's whole cache, that token included; the stored token read back
* chunk   causal attention of the last `new` tokens of every sequence over its cache
          (speculative drafts, a prefill chunk, a whole prompt); with `window`, over the
          last `window` keys of each row in a sliding-window pool
"""
import math

import numpy as np
import torch

own = False

BF16, F16, F32 = "bf16", "f16", "f32"
_TORCH = {BF16: torch.bfloat16, F16: torch.float16, F32: torch.float32}

_DEFAULT = dict(B=1, lo=1, hi=1, new=1, rope=False, dt=BF16, out=BF16, window=0, left=False)


def _case(kind, Hq, Hkv, D, **kw):
    c = dict(kind=kind, Hq=Hq, Hkv=Hkv, D=D, **_DEFAULT)
    c.update(kw)
    return c


def listed():
    return [
        # one user's chat on a small model: latency
        _case("step", 32, 8, 64, name="step_chat", lo=512, hi=512, rope=True),
        # a serving batch at mixed contexts
        _case("step", 40, 8, 128, name="step_batch", B=32, lo=512, hi=8192),
        # few very long contexts
        _case("step", 32, 4, 128, name="step_long", B=8, lo=98304, hi=131072),
        # a batch on layers of head_dim 512, fp16 model, the default output type
        _case("step", 16, 2, 512, name="step_wide", B=32, lo=512, hi=4096, dt=F16, out=F32),
        # speculative decoding: 8 drafted rows per sequence verified
        _case("chunk", 32, 8, 128, name="verify", B=16, lo=1024, hi=8192, new=8),
        # chunked prefill of a batch on top of its contexts
        _case("chunk", 40, 8, 128, name="prefill_chunk", B=8, lo=2048, hi=6144, new=512),
        # a whole prompt from scratch, fp16 model
        _case("chunk", 32, 8, 64, name="prefill_prompt", lo=0, hi=0, new=3900, dt=F16, out=F16),
        # a prefill chunk of sliding-window layers
        _case("chunk", 16, 8, 256, name="prefill_window", B=4, lo=300, hi=5000, new=512, window=1024),
        # a decode step's tokens written
        _case("write", 8, 8, 128, name="write_step", B=64, lo=100, hi=8000, rope=True),
        # a prefill chunk written
        _case("write", 8, 8, 128, name="write_chunk", B=8, lo=0, hi=4000, new=512),
        # a batch's caches read back, left-aligned to the end as a stacked batch takes them
        _case("read", 8, 8, 128, name="read_batch", B=8, lo=512, hi=8192, left=True),
        # a few short sequences read back
        _case("read", 2, 2, 256, name="read_short", B=3, lo=1, hi=200, dt=F16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["step", "step", "step", "chunk", "chunk", "chunk", "window", "write", "read"])
    dt = rng.choice([BF16, BF16, F16])
    out = rng.choice([dt, F32])
    D = rng.choice([64, 128, 128, 256, 512])
    Hkv = rng.choice([1, 2, 4, 8])
    R = rng.choice([1, 2, 3, 4, 5, 7, 8])
    c = dict(dt=dt, out=out)
    if kind == "step":
        B = _log(rng, 1, 64)
        hi = _log(rng, 1, max(2, min(131072, (1 << 28) // (B * Hkv * D))))
        return _case(kind, Hkv * R, Hkv, D, B=B, lo=max(1, hi // rng.choice([1, 2, 16])), hi=hi,
                     rope=rng.random() < 0.4, **c)
    if kind == "chunk":
        new = _log(rng, 2, 3900 if D <= 256 else 512)
        hi = _log(rng, 1, 8192)
        # (at most the work of the listed prefill chunk)
        B = min(_log(rng, 1, 16), max(1, (1 << 28) // (Hkv * R * D * new // 64 * (hi + new // 2 + 1))))
        if Hkv * R * D * new * (hi + new // 2) > 1 << 36:
            new = max(2, (1 << 36) // (Hkv * R * D * (hi + 2000)))
        return _case(kind, Hkv * R, Hkv, D, B=B, lo=hi // rng.choice([1, 2, 16]), hi=hi, new=new, **c)
    if kind == "window":
        new = _log(rng, 2, 700)
        hi = _log(rng, 16, 8192)
        return _case("chunk", Hkv * R, Hkv, min(D, 256), B=max(1, min(_log(rng, 1, 8), 2048 // new)), lo=hi // 4, hi=hi,
                     new=new, window=rng.choice([100, 512, 1024, 2048]), **c)
    if kind == "write":
        new = _log(rng, 1, 2000)
        hi = _log(rng, 1, 8000)
        return _case(kind, Hkv, Hkv, D, B=max(1, min(_log(rng, 1, 64), 8192 // new)), lo=hi // 4, hi=hi, new=new,
                     rope=rng.random() < 0.5, dt=dt)
    hi = _log(rng, 2, 8192)
    return _case(kind, Hkv, Hkv, D, B=_log(rng, 1, 8), lo=max(1, hi // rng.choice([1, 4, 16])), hi=hi,
                 left=rng.random() < 0.5, dt=dt)


# ------------------------------------------------------------------ inputs


def _rng(seed, *what):
    return np.random.default_rng([int(seed) & 0x7FFFFFFF, *what])


def _lens(c, seed):
    """Tokens of each sequence before the call's new rows, spread evenly over the range so that
    one seed's work is another's."""
    u = (np.arange(c["B"]) + _rng(seed, 1).random(c["B"])) / c["B"]
    if c["B"] == 1:
        u = u * 0.1 + 0.45
    return [int(x) for x in _rng(seed, 2).permutation(np.floor(c["lo"] + u * (c["hi"] - c["lo"] + 1)).astype(np.int64))]


def _total(c, ctx):
    """Tokens of the sequence when the call attends or reads it (a step's new token is the last
    of its context)."""
    return ctx + (c["new"] if c["kind"] in ("chunk", "write") else 0)


def _first(c, T):
    """First token that a windowed sequence of T tokens still needs (0 without a window)."""
    return max(0, T - c["new"] - c["window"] + 1) if c["window"] else 0


def _randn(c, seed, shape, *what):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(_rng(seed, 7, *what).integers(1 << 62)))
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _kv(c, seed, b, T):
    """K and V [Hkv, T, D] of sequence b in the case's input type: N(0, 1), each channel of K
    about a mean of its own, as keys are."""
    shape = (c["Hkv"], T, c["D"])
    k = _randn(c, seed, shape, 11, b) + _randn(c, seed, (c["Hkv"], 1, c["D"]), 14)
    return k.to(_TORCH[c["dt"]]), _randn(c, seed, shape, 12, b).to(_TORCH[c["dt"]])


def _q(c, seed):
    return (1.5 * _randn(c, seed, (c["B"], c["Hq"], c["new"], c["D"]), 13)).to(_TORCH[c["dt"]])


def _angles(max_pos, D):
    """fp32 [max_pos, D]: cosines of the pair angles p 10000^(-2i/D), then their sines."""
    inv = 10000.0 ** (-2.0 * np.arange(D // 2, dtype=np.float64) / D)
    ang = np.arange(max_pos, dtype=np.float64)[:, None] * inv[None, :]
    return torch.from_numpy(np.concatenate([np.cos(ang), np.sin(ang)], axis=1).astype(np.float32)).cuda()


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()


def prepare(case, seed):
    return _prepare_own(case, seed) if own else _prepare_plain(case, seed)


def _prepare_own(c, seed):
    import krill_amd
    from krill_amd import _lib as KL

    lens = _lens(c, seed)
    total = [_total(c, t) for t in lens]
    blocks = sum((t + 63) // 64 + 1 for t in total) + c["B"]
    pool = krill_amd.KVPool(1, c["Hkv"], c["D"], blocks, "affine4_g64", c["dt"], free_list_seed=5)
    if c["window"]:
        pool.set_option(KL.OPT_WINDOW, c["window"])
    st = dict(c=c, pool=pool, scale=1.0 / math.sqrt(c["D"]))
    seqs, slots, kn, vn = [], [], [], []
    write, step = c["kind"] == "write", c["kind"] == "step"
    for b, T in enumerate(total):
        s = pool.seq_create()
        seqs.append(s)
        k, v = _kv(c, seed, b, T)
        # what the sequence holds before the call: all but a step's or a write's new rows
        held = T - (c["new"] if write or step else 0)
        # (a windowed pool drops what the rows appended next do not see: the chunk comes in one append)
        chunk = held - c["new"] if c["window"] else 0
        at = [*range(0, chunk, 512), *([chunk] if held else []), held]
        for t, n in zip(at, np.diff(at).tolist()):
            sl = _i32(pool.reserve_append(s, n).reshape(1, n))
            pool.quantize_append(0, k[None, :, t:t + n].contiguous(), v[None, :, t:t + n].contiguous(), sl)
        if write or step:
            slots.append(pool.reserve_append(s, c["new"]).copy())
            kn.append(k[:, held:])
            vn.append(v[:, held:])
    if write or step:
        st.update(slots=_i32(np.stack(slots)), k=torch.stack(kn).contiguous(), v=torch.stack(vn).contiguous())
    if c["rope"]:
        st["cos_sin"] = _angles(max(total), c["D"])
        if write:
            st["positions"] = _i32(np.stack([np.arange(t - c["new"], t) for t in total]))
    width = max((t + 63) // 64 for t in total)
    tables, n = pool.batch_tables(seqs, width)
    st.update(tables=_i32(tables), lens=_i32(n), max_len=max(total))
    if c["kind"] in ("step", "chunk"):
        st["q"] = _q(c, seed)
        st["o"] = torch.empty_like(st["q"], dtype=_TORCH[c["out"]])
        if c["window"]:
            st["starts"] = _i32(pool.batch_starts(seqs))
        else:
            need = pool.workspace_size(c["B"], c["Hq"], c["new"], st["max_len"])
            st["ws"] = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    return st


def _prepare_plain(c, seed):
    lens = _lens(c, seed)
    total = [_total(c, t) for t in lens]
    st = dict(c=c, scale=1.0 / math.sqrt(c["D"]), total=total)
    write, step = c["kind"] == "write", c["kind"] == "step"
    cache, kn, vn = [], [], []
    for b, T in enumerate(total):
        k, v = _kv(c, seed, b, T)
        if write or step:
            kn.append(k[:, T - c["new"]:])
            vn.append(v[:, T - c["new"]:])
        if not write:
            f = _first(c, T)
            cache.append((_quantize(k[:, f:]), _quantize(v[:, f:])))
    if write or step:
        st.update(k=torch.stack(kn), v=torch.stack(vn))
    st["cache"] = cache
    if c["rope"]:
        st["cos_sin"] = _angles(max(total), c["D"])
    if c["kind"] in ("step", "chunk"):
        st["q"] = _q(c, seed)
    return st


# ------------------------------------------------------------------ one pass


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(st):
    c, pool = st["c"], st["pool"]
    if c["kind"] == "write":
        if c["rope"]:
            pool.quantize_append_rope(0, st["k"], st["v"], st["slots"], st["positions"], st["cos_sin"])
        else:
            pool.quantize_append(0, st["k"], st["v"], st["slots"])
        return list(pool.read_slots(0, st["slots"]))
    if c["kind"] == "read":
        return list(pool.gather_dequant(0, st["tables"], st["lens"], c["hi"], c["left"]))
    if c["kind"] == "step":
        args = (0, st["q"], st["k"], st["v"], st["tables"], st["lens"], st["max_len"], st["scale"])
        kw = dict(out_dtype=_TORCH[c["out"]], ws=st["ws"], out=st["o"])
        if c["rope"]:
            o = pool.decode_append_attention_rope(*args, st["cos_sin"], **kw)
        else:
            o = pool.decode_append_attention(*args, **kw)
        return [o, *pool.read_slots(0, st["slots"])]
    if c["window"]:
        return pool.attention_windowed(0, st["q"], st["tables"], st["lens"], st["starts"], c["window"], st["max_len"],
                                       st["scale"], out_dtype=_TORCH[c["out"]], out=st["o"])
    return pool.attention(0, st["q"], st["tables"], st["lens"], st["max_len"], st["scale"],
                          out_dtype=_TORCH[c["out"]], ws=st["ws"], out=st["o"])


def _quantize(x):
    """Codes [..., D/64, 64] u8, scales and biases [..., D/64, 1] f16 of rows [..., D]."""
    w = x.float().clamp(-65504.0, 65504.0).unflatten(-1, (-1, 64))
    lo, hi = w.amin(-1, keepdim=True), w.amax(-1, keepdim=True)
    b = lo.half()
    # (a division by a tensor is rounded once; by a number torch multiplies by its inverse)
    s = ((hi - b.float()).clamp(min=0.0) / torch.full_like(hi, 15.0)).half()
    q = torch.where(s > 0, (w - b.float()) / s.float(), torch.zeros_like(w))
    return q.round().clamp(0.0, 15.0).to(torch.uint8), s, b


def _value(q):
    """The fp32 rows [..., D] that codes, scales and biases stand for."""
    c, s, b = q
    return (s.float() * c.float() + b.float()).flatten(-2)


def _f16(x):
    return x.clamp(-65504.0, 65504.0).half()


def _turn(x, cs):
    """Rows [..., D] rotated by the angles cs [..., D], in the rows' type."""
    h = x.shape[-1] // 2
    a, b, cos, sin = x[..., :h].float(), x[..., h:].float(), cs[..., :h], cs[..., h:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1).to(x.dtype)


def _rope_rows(st, x):
    """Rows [B, H, new, D] at the last positions of their sequences."""
    if not st["c"]["rope"]:
        return x
    n = x.shape[2]
    cs = torch.stack([st["cos_sin"][t - n:t] for t in st["total"]])
    return _turn(x, cs[:, None])


def _attend(q, k, v, scale, window):
    """q [Hq, n, D] at the last n positions of k, v [Hkv, T, D], all fp32."""
    (Hq, n, D), (Hkv, T, _) = q.shape, k.shape
    s = torch.matmul(q.reshape(Hkv, Hq // Hkv * n, D), k.transpose(1, 2).contiguous()) * scale
    s = s.view(Hkv, Hq // Hkv, n, T)
    if n > 1 or window:
        pos = torch.arange(T - n, T, device=q.device)[:, None]
        key = torch.arange(T, device=q.device)[None, :]
        hide = key > pos
        if window:
            hide = hide | (key <= pos - window)
        s = s.masked_fill(hide, float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    return torch.matmul(p.view(Hkv, Hq // Hkv * n, T), v).view(Hq, n, D)


def _run_plain(st):
    c = st["c"]
    if c["kind"] == "write":
        return [_f16(_value(_quantize(_rope_rows(st, st["k"])))), _f16(_value(_quantize(st["v"])))]
    if c["kind"] == "read":
        shape = (c["B"], c["Hkv"], c["hi"], c["D"])
        k, v = (torch.zeros(shape, dtype=torch.float16, device="cuda") for _ in range(2))
        for b, T in enumerate(st["total"]):
            at = slice(shape[2] - T, shape[2]) if c["left"] else slice(0, T)
            k[b, :, at], v[b, :, at] = (_f16(_value(x)) for x in st["cache"][b])
        return [k, v]
    out = torch.empty(c["B"], c["Hq"], c["new"], c["D"], dtype=_TORCH[c["out"]], device="cuda")
    q, back = st["q"], []
    if c["kind"] == "step":
        q = _rope_rows(st, q)
        for i, new in enumerate((_quantize(_rope_rows(st, st["k"])), _quantize(st["v"]))):
            for b in range(c["B"]):
                for held, row in zip(st["cache"][b][i], new):
                    held[:, -1:] = row[b]
            back.append(_f16(_value(new)))
    for b in range(c["B"]):
        k, v = (_value(x) for x in st["cache"][b])
        out[b] = _attend(q[b].float(), k, v, st["scale"], c["window"])
    return [out, *back] if back else out


# ------------------------------------------------------------------ what it costs


def work(case):
    c = case
    G = c["D"] // 64
    ctx = 0.5 * (c["lo"] + c["hi"])
    size = {BF16: 2, F16: 2, F32: 4}
    row4 = c["Hkv"] * (c["D"] + 8 * G)  # bytes of a token's K and V in the cache
    row16 = c["Hkv"] * c["D"] * 4       # the same in 16 bits
    new = c["B"] * c["new"]
    if c["kind"] == "write":
        return dict(bytes=new * (2 * row16 + 2 * row4), flops=new * c["Hkv"] * c["D"] * 2 * 8)
    if c["kind"] == "read":
        return dict(bytes=c["B"] * (ctx * row4 + c["hi"] * row16), flops=c["B"] * ctx * c["Hkv"] * c["D"] * 4)
    qo = new * c["Hq"] * c["D"] * (2 + size[c["out"]])
    if c["kind"] == "step":
        return dict(bytes=c["B"] * ctx * row4 + qo + new * (2 * row16 + row4), flops=4 * c["B"] * c["Hq"] * c["D"] * ctx)
    keys, pairs = ctx + c["new"], c["new"] * (ctx + 0.5 * (c["new"] + 1))
    if c["window"]:
        keys = min(keys, c["new"] + c["window"] - 1)
        pairs = min(pairs, c["new"] * c["window"])
    return dict(bytes=c["B"] * keys * row4 + qo, flops=4 * c["B"] * c["Hq"] * c["D"] * pairs)


# ------------------------------------------------------------------ in 64 bits


def _exact_rows(x):
    """What the cache holds for rows [..., D], in 64 bits from the definition (the stored scale
    and bias are fp16 numbers by definition)."""
    w = x.double().clamp(-65504.0, 65504.0)
    w = w.view(*w.shape[:-1], w.shape[-1] // 64, 64)
    bias = w.min(dim=-1, keepdim=True).values.half().double()
    step = ((w.max(dim=-1, keepdim=True).values - bias) / 15.0).clamp(min=0.0).half().double()
    code = torch.round((w - bias) / torch.where(step > 0, step, torch.ones_like(step)))
    code = torch.minimum(code.clamp(min=0.0), torch.full_like(code, 15.0)) * (step > 0)
    return (bias + step * code).reshape(x.shape)


def _exact_turn(x, T):
    """Rows [H, n, D] at positions T - n .. T - 1, rotated, in the rows' type."""
    H, n, D = x.shape
    ang = torch.arange(T - n, T, device="cuda", dtype=torch.float64)[:, None] * torch.pow(
        torch.tensor(10000.0, device="cuda", dtype=torch.float64),
        torch.arange(D // 2, device="cuda", dtype=torch.float64) * (-2.0 / D))[None]
    cos, sin = ang.cos().float().double(), ang.sin().float().double()  # the table holds 32 bits
    z = x.double()
    lo, hi = z[..., :D // 2], z[..., D // 2:]
    return torch.cat((lo * cos - hi * sin, hi * cos + lo * sin), dim=-1).to(x.dtype)


def exact(case, seed):
    c = case
    n, D, R = c["new"], c["D"], c["Hq"] // c["Hkv"]
    total = [_total(c, t) for t in _lens(c, seed)]
    if c["kind"] == "write":
        ks, vs = [], []
        for b, T in enumerate(total):
            k, v = (x[:, T - n:] for x in _kv(c, seed, b, T))
            ks.append(_exact_rows(_exact_turn(k, T) if c["rope"] else k))
            vs.append(_exact_rows(v))
        return [torch.stack(ks), torch.stack(vs)]
    if c["kind"] == "read":
        S = c["hi"]
        k64, v64 = (torch.zeros(c["B"], c["Hkv"], S, D, dtype=torch.float64, device="cuda") for _ in range(2))
        for b, T in enumerate(total):
            k, v = _kv(c, seed, b, T)
            o = S - T if c["left"] else 0
            k64[b, :, o:o + T] = _exact_rows(k)
            v64[b, :, o:o + T] = _exact_rows(v)
        return [k64, v64]
    q = _q(c, seed)
    out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    back_k, back_v = [], []
    for b, T in enumerate(total):
        k, v = _kv(c, seed, b, T)
        qb = q[b]
        if c["kind"] == "step" and c["rope"]:
            # (only the step's own token is rotated here: the context was given as it is)
            k = torch.cat((k[:, :-1], _exact_turn(k[:, -1:], T)), dim=1)
            qb = _exact_turn(qb, T)
        f = _first(c, T)
        for h in range(c["Hkv"]):
            kh, vh = _exact_rows(k[h, f:]), _exact_rows(v[h, f:])
            if c["kind"] == "step":
                back_k.append(kh[-1:])
                back_v.append(vh[-1:])
            # rows in pieces, so that a piece's scores fit
            step = max(1, (1 << 28) // (R * (T - f)))
            for j in range(0, n, step):
                m = min(step, n - j)
                z = qb[h * R:(h + 1) * R, j:j + m].double().reshape(R * m, D) @ kh.T / math.sqrt(D)
                z = z.view(R, m, T - f)
                pos = torch.arange(T - n + j, T - n + j + m, device="cuda").view(1, m, 1)
                key = torch.arange(f, T, device="cuda").view(1, 1, T - f)
                seen = key <= pos
                if c["window"]:
                    seen = seen & (key > pos - c["window"])
                w = torch.softmax(torch.where(seen, z, torch.full_like(z, -math.inf)), dim=-1)
                out[b, h * R:(h + 1) * R, j:j + m] = (w.view(R * m, T - f) @ vh).view(R, m, D)
    if c["kind"] != "step":
        return out
    shape = (c["B"], c["Hkv"], 1, D)
    return [out, torch.stack(back_k).view(shape), torch.stack(back_v).view(shape)]
