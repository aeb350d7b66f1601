"""The 4-bit storage mode on the GPU: append, read-back and attention against 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import oracle as O

import q4util as Q
from kvutil import i32, rand_bits, to_dev

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


def make_pool(H, D, blocks, dt="bf16", layers=1, **kw):
    import krill_amd

    return krill_amd.KVPool(layers, H, D, blocks, "affine4_g64", dt, free_list_seed=kw.pop("seed", 3), **kw)


class Cache:
    """Sequences of `lens` tokens in a pool, with their input bits."""

    def __init__(self, pool, lens, rng, dt, chunk=None, scale=1.0, k=None, v=None):
        self.pool, self.lens, self.dt = pool, list(lens), dt
        H, D = pool.num_kv_heads, pool.head_dim
        self.k = [rand_bits(rng, (H, T, D), dt, scale) for T in lens] if k is None else k
        self.v = [rand_bits(rng, (H, T, D), dt, scale) for T in lens] if v is None else v
        self.seqs = [pool.seq_create() for _ in lens]
        for b, T in enumerate(lens):
            t = 0
            while t < T:
                n = min(T - t, chunk or T)
                slots = pool.reserve_append(self.seqs[b], n)
                pool.quantize_append(0, to_dev(self.k[b][None, :, t:t + n], dt), to_dev(self.v[b][None, :, t:t + n], dt),
                                     i32(slots.reshape(1, n)))
                t += n

    def tables(self, extra=0):
        mb = max(1, max((T + 63) // 64 for T in self.lens) + extra)
        t, n = self.pool.batch_tables(self.seqs, mb)
        return i32(t), i32(n)

    def check(self, got, qbits, scale, out, window=0, upto=None, long=False):
        """got [B, Hq, Lq, D] against 64 bits, queries at the sequences' last positions."""
        B, Hq, Lq, D = qbits.shape
        H = self.pool.num_kv_heads
        R = Hq // H
        qf = O.bits_to_f32(qbits, Q.DT[self.dt]).astype(np.float64)
        got = got.float().cpu().numpy().astype(np.float64)
        for b in range(B):
            T = self.lens[b]
            for h in range(H):
                kd, vd = Q.stored(self.k[b][h], self.dt), Q.stored(self.v[b][h], self.dt)
                rows = qf[b, h * R:(h + 1) * R].reshape(R * Lq, D)
                hi = np.tile(np.arange(T - Lq + 1, T + 1), R)
                if upto is not None:
                    hi = np.minimum(hi, upto)
                lo = np.maximum(0, hi - window) if window else np.zeros_like(hi)
                want = Q.attention(rows, kd, vd, lo, np.maximum(hi, 0), scale)
                g = got[b, h * R:(h + 1) * R].reshape(R * Lq, D)
                if T == 0:
                    assert not g.any()
                    continue
                err, lim = np.abs(g - want), Q.bound(rows, kd, vd, scale, want, out, *(
                    Q.quantize(x[b][h], self.dt)[1].max(initial=0) for x in (self.k, self.v)), long=long)
                assert np.all(err <= lim), f"b {b} h {h}: {np.nanmax(err / lim):.3g} times the bound"
                # errors of the weights are independent, as the values they weigh: both sum alike
                x = np.abs(rows @ kd.T).max() * abs(scale) * np.log2(np.e)
                if out == "f32" and x <= 8 and T >= 64:
                    rms = [np.sqrt((y ** 2).mean()) for y in (err, want)]
                    assert rms[0] <= Q.weight_error(D // 64) * rms[1], f"b {b} h {h}: rms {rms[0] / rms[1]:.3g} of the result"


def all_slots(pool):
    return i32(np.arange(pool.num_blocks * 64).reshape(1, -1))


def same(a, b):
    """Equal values, NaN where NaN."""
    np.testing.assert_array_equal(a, b)


# ------------------------------------------------------------ write and read


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_append_reads_back(D, dt):
    rng = np.random.default_rng(D)
    H, B = 3, 3
    pool = make_pool(H, D, 40, dt)
    cap = pool.num_blocks * 64
    want_k = np.zeros((H, cap, D), np.float16)
    want_v = np.zeros_like(want_k)
    seqs = [pool.seq_create() for _ in range(B)]
    for L in (1, 5, 58, 64, 1, 63, 130, 200):
        kb, vb = rand_bits(rng, (B, H, L, D), dt), rand_bits(rng, (B, H, L, D), dt)
        slots = np.stack([pool.reserve_append(s, L) for s in seqs])
        slots[1, L // 3] = -1  # a skipped row
        pool.quantize_append(0, to_dev(kb, dt), to_dev(vb, dt), i32(slots))
        for b in range(B):
            ok = slots[b] >= 0
            want_k[:, slots[b][ok]] = Q.read_back(Q.stored(kb[b][:, ok], dt))
            want_v[:, slots[b][ok]] = Q.read_back(Q.stored(vb[b][:, ok], dt))
        k, v = pool.read_slots(0, i32(slots))
        ok = slots >= 0
        for b in range(B):
            same(k[b].cpu().numpy()[:, ok[b]], want_k[:, slots[b][ok[b]]])
            same(v[b].cpu().numpy()[:, ok[b]], want_v[:, slots[b][ok[b]]])
            assert not k[b].cpu().numpy()[:, ~ok[b]].any() and not v[b].cpu().numpy()[:, ~ok[b]].any()
    # the whole pool: rows never written are as they were
    k, v = pool.read_slots(0, all_slots(pool))
    same(k[0].cpu().numpy(), want_k)
    same(v[0].cpu().numpy(), want_v)
    # and by sequences, from either end, in more and in fewer rows than tokens
    n = pool.seq_length(seqs[0])
    t, lens = pool.batch_tables(seqs, (n + 63) // 64)
    for S in (n + 70, n, n - 100, 1):
        for left in (False, True):
            k, v = pool.gather_dequant(0, i32(t), i32(lens), S, left)
            for b in range(B):
                pos = np.arange(n)
                sl = t[b][pos // 64] * 64 + pos % 64
                row = pos + (S - n if left else 0)
                ok = (row >= 0) & (row < S)
                for got, want in ((k, want_k), (v, want_v)):
                    full = np.zeros((H, S, D), np.float16)
                    full[:, row[ok]] = want[:, sl[ok]]
                    same(got[b].cpu().numpy(), full)
    pool.close()


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128, 512])
def test_slots_in_any_order_and_strides(D, dt):
    rng = np.random.default_rng(7 * D)
    H, B, L = 2, 2, 150
    pool = make_pool(H, D, 12, dt)
    slots = rng.permutation(12 * 64)[:B * L].reshape(B, L).astype(np.int32)
    slots[0, 3] = 12 * 64 + 5  # past the pool: skipped
    # a projection's layout [B][L][Hkv][D] at a row stride that is no multiple of 16 bytes, one element in
    for pad, first in ((0, 0), (1, 1), (8, 0)):
        raw = rand_bits(rng, (2, B * L * (H * D + pad) + 8), dt)
        kt, vt = to_dev(raw[0], dt), to_dev(raw[1], dt)
        sl = H * D + pad
        pool.quantize_append_strided(0, kt[first:], vt[first:], (L * sl, D, sl), i32(slots), B, L)
        got_k, got_v = (x.cpu().numpy() for x in pool.read_slots(0, i32(slots)))
        for b in range(B):
            for h in range(H):
                at = first + b * L * sl + np.arange(L)[:, None] * sl + h * D + np.arange(D)[None]
                for got, x in ((got_k, raw[0]), (got_v, raw[1])):
                    want = Q.read_back(Q.stored(x[at], dt))
                    want[slots[b] >= 12 * 64] = 0
                    same(got[b, h], want)
    pool.close()


def special_groups(dt):
    """Groups of 64 where the quantizer can go wrong."""
    f = np.float32
    g = []
    g.append(np.zeros(64, f))
    g.append(np.full(64, -0.0, f))
    g.append(np.full(64, 3.25, f))
    g.append(np.full(64, 1e-9, f))
    g.append(np.linspace(-65504, 65504, 64, dtype=f))
    g.append(np.linspace(1e-7, 9e-7, 64, dtype=f))
    g.append(np.where(np.arange(64) == 7, 1.0, 1e-6).astype(f))
    g.append((np.arange(64) % 16).astype(f))                       # exact codes
    g.append((np.arange(64) % 31 / 2).astype(f))                   # ties
    g.append((100 + np.arange(64) * 2.0 ** -5).astype(f))          # bias rounds
    g.append(np.where(np.arange(64) == 0, np.inf, np.arange(64)).astype(f))
    g.append(np.where(np.arange(64) == 63, -np.inf, np.arange(64)).astype(f))
    x = np.arange(64).astype(f)
    x[5] = np.nan
    g.append(x)
    x = np.full(64, np.nan, f)
    g.append(x)
    if dt == "bf16":
        g.append(np.linspace(-3e38, 3e38, 64, dtype=f))
        g.append(np.linspace(65500, 66000, 64, dtype=f))
    return np.stack(g)


@pytest.mark.parametrize("L", [1, 64])
@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_special_values(dt, L):
    D, H = 128, 1
    g = special_groups(dt)
    rows = np.concatenate([g, np.roll(g, 1, 0)], 1)  # every group as the first and as the second of a row
    bits = (O.f32_to_bf16_bits if dt == "bf16" else O.f32_to_f16_bits)(rows)
    pool = make_pool(H, D, 2, dt)
    bits = bits[np.arange(64) % len(rows)]
    slots = np.arange(64, dtype=np.int32)
    v = bits[::-1].copy()
    for a in range(0, 64, L):
        pool.quantize_append(0, to_dev(bits[None, None, a:a + L], dt), to_dev(v[None, None, a:a + L], dt),
                             i32(slots[None, a:a + L]))
    k_got, v_got = (x.cpu().numpy()[0, 0] for x in pool.read_slots(0, i32(slots[None])))
    same(k_got, Q.read_back(Q.stored(bits, dt)))
    same(v_got, Q.read_back(Q.stored(v, dt)))
    pool.close()


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("L", [1, 130])
def test_append_with_rope(D, dt, L):
    from krill_amd.pool import rope_table

    rng = np.random.default_rng(D + L)
    H, B, P = 2, 2, 300
    pool = make_pool(H, D, 12, dt)
    kb, vb = rand_bits(rng, (B, H, L, D), dt), rand_bits(rng, (B, H, L, D), dt)
    pos = rng.integers(0, P, (B, L)).astype(np.int32)
    pos[1, 0] = P  # outside the table: not written
    slots = np.stack([pool.reserve_append(pool.seq_create(), L) for _ in range(B)])
    cs = rope_table(P, D)
    pool.quantize_append_rope(0, to_dev(kb, dt), to_dev(vb, dt), i32(slots), i32(pos), torch.from_numpy(cs).cuda())
    k, v = (x.cpu().numpy() for x in pool.read_slots(0, i32(slots)))
    for b in range(B):
        for h in range(H):
            turned = O.rope_rows(kb[b, h], Q.DT[dt], np.minimum(pos[b], P - 1), cs)
            want_k, want_v = Q.read_back(Q.stored(turned, dt)), Q.read_back(Q.stored(vb[b, h], dt))
            want_k[pos[b] >= P] = 0
            want_v[pos[b] >= P] = 0
            same(k[b, h], want_k)
            same(v[b, h], want_v)
    pool.close()


@pytest.mark.parametrize("quant", ["ref_row", "affine_g64"])
@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_read_slots_of_int8_pools(quant, D):
    import krill_amd

    rng = np.random.default_rng(D)
    H, T = 2, 150
    pool = krill_amd.KVPool(1, H, D, 6, quant, "bf16", free_list_seed=5)
    seq = pool.seq_create()
    slots = pool.reserve_append(seq, T)
    pool.quantize_append(0, to_dev(rand_bits(rng, (1, H, T, D), "bf16"), "bf16"),
                         to_dev(rand_bits(rng, (1, H, T, D), "bf16"), "bf16"), i32(slots.reshape(1, T)))
    t, n = pool.batch_tables([seq], 3)
    k, v = pool.gather_dequant(0, i32(t), i32(n), T)
    ask = slots.copy().reshape(2, -1)
    ask[1, 4] = -1
    ks, vs = pool.read_slots(0, i32(ask))
    for got, want in ((ks, k), (vs, v)):
        want = want[0].cpu().numpy().reshape(H, 2, -1, D).swapaxes(0, 1).copy()
        want[1, :, 4] = 0
        same(got.cpu().numpy(), want)
    pool.close()


# ------------------------------------------------------------ attention

LENS = [1, 0, 63, 64, 65, 300, 129, 2]


@pytest.mark.parametrize("out", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("R", [1, 4, 5, 8, 17])
@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_decode(D, R, out):
    rng = np.random.default_rng(R)
    dt = "f16" if R == 4 else "bf16"
    H = 2
    pool = make_pool(H, D, 40, dt)
    c = Cache(pool, LENS, rng, dt, chunk=70)
    qb = rand_bits(rng, (len(LENS), H * R, 1, D), dt)
    t, n = c.tables(extra=1)
    o = pool.attention(0, to_dev(qb, dt), t, n, max(LENS), 1 / np.sqrt(D), out_dtype=getattr(
        torch, {"f32": "float32", "bf16": "bfloat16", "f16": "float16"}[out]))
    c.check(o, qb, 1 / np.sqrt(D), out)
    pool.close()


@pytest.mark.parametrize("path", [0, 1, 2])
@pytest.mark.parametrize("Lq,R", [(2, 1), (3, 4), (8, 4), (9, 5), (70, 2)])
@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_several_rows(D, Lq, R, path):
    from krill_amd import _lib as L

    rng = np.random.default_rng(100 * Lq + R)
    dt = "bf16" if Lq % 2 else "f16"
    H = 2
    lens = [Lq, Lq + 1, Lq + 63, 300, 64 * ((Lq + 63) // 64)]
    pool = make_pool(H, D, 40, dt)
    pool.set_option(L.OPT_ATTN_PATH, path)
    c = Cache(pool, lens, rng, dt)
    qb = rand_bits(rng, (len(lens), H * R, Lq, D), dt)
    t, n = c.tables()
    o = pool.attention(0, to_dev(qb, dt), t, n, max(lens), 1 / np.sqrt(D))
    c.check(o, qb, 1 / np.sqrt(D), "f32")
    pool.close()


def rope(D, P=2000):
    from krill_amd.pool import rope_table

    cs = rope_table(P, D)
    return cs, torch.from_numpy(cs).cuda()


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("R", [1, 5, 20])
@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_fused_step_equals_append_then_attention(D, R, dt):
    """Pool and output of the fused step, plain and with RoPE, are those of the calls it joins."""
    rng = np.random.default_rng(R + D)
    H, scale = 2, 1 / np.sqrt(D)
    lens = [1, 0, 64, 65, 200, 17, 128]
    kb, vb, qb = (rand_bits(rng, (len(lens), h, 1, D), dt) for h in (H, H, H * R))
    cs, cs_d = rope(D)
    pos = np.array([max(T - 1, 0) for T in lens])
    turned_k, turned_q = (np.stack([np.stack([O.rope_rows(x[b, h], Q.DT[dt], [pos[b]], cs) for h in range(x.shape[1])])
                                    for b in range(len(lens))]) for x in (kb, qb))
    for turn in (False, True):
        outs, pools = [], []
        for fused in (False, True):
            pool = make_pool(H, D, 24, dt)
            c = Cache(pool, [max(T - 1, 0) for T in lens], np.random.default_rng(1), dt)
            slots = np.array([pool.reserve_append(s, 1)[0] if T else -1 for s, T in zip(c.seqs, lens)], np.int32)
            c.lens = lens
            t, n = c.tables()
            if fused:
                args = (0, to_dev(qb, dt), to_dev(kb, dt), to_dev(vb, dt), t, n, max(lens), scale)
                o = pool.decode_append_attention_rope(*args, cs_d) if turn else pool.decode_append_attention(*args)
            else:
                k, q = (turned_k, turned_q) if turn else (kb, qb)
                pool.quantize_append(0, to_dev(k, dt), to_dev(vb, dt), i32(slots[:, None]))
                o = pool.attention(0, to_dev(q, dt), t, n, max(lens), scale)
                for b, T in enumerate(lens):
                    if T:
                        c.k[b] = np.concatenate([c.k[b], k[b]], 1)
                        c.v[b] = np.concatenate([c.v[b], vb[b]], 1)
                c.check(o, q, scale, "f32")
            outs.append(o.cpu().numpy())
            pools.append([x.cpu().numpy() for x in pool.read_slots(0, all_slots(pool))])
            pool.close()
        same(outs[0], outs[1])
        for a, b in zip(*pools):
            same(a, b)


def test_step_without_allocation_equals_the_step():
    import ctypes

    from krill_amd import _lib as L

    rng = np.random.default_rng(5)
    H, R, D, dt = 2, 4, 128, "bf16"
    lens = [100, 1, 400]
    pool = make_pool(H, D, 24, dt)
    c = Cache(pool, [T - 1 for T in lens], rng, dt)
    for s in c.seqs:
        pool.reserve_append(s, 1)
    c.lens = lens
    t, n = c.tables()
    kb, vb, qb = (to_dev(rand_bits(rng, (3, h, 1, D), dt), dt) for h in (H, H, H * R))
    want = pool.decode_append_attention(0, qb, kb, vb, t, n, max(lens), 0.1)
    got = torch.empty_like(want)
    L.check(L.lib().krill_decode_append_attention_noalloc(
        pool.handle, 0, qb.data_ptr(), kb.data_ptr(), vb.data_ptr(), H * D, D, t.data_ptr(), n.data_ptr(), 3, t.shape[1],
        max(lens), H * R, ctypes.c_float(0.1), got.data_ptr(), L.DTYPE_F32, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
    same(got.cpu().numpy(), want.cpu().numpy())
    pool.close()


@pytest.mark.parametrize("Lq,R", [(1, 1), (1, 8), (5, 2), (40, 4)])
@pytest.mark.parametrize("window", [2, 64, 100])
@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_windows(D, window, Lq, R):
    from krill_amd import _lib as L

    rng = np.random.default_rng(window + Lq)
    H, dt, scale = 2, "bf16", 1 / np.sqrt(D)
    lens = [Lq, 130, 64 + Lq, 331]
    pool = make_pool(H, D, 30, dt)
    pool.set_option(L.OPT_WINDOW, window)
    kb = [rand_bits(rng, (H, T, D), dt) for T in lens]
    vb = [rand_bits(rng, (H, T, D), dt) for T in lens]
    seqs = [pool.seq_create() for _ in lens]
    for b, T in enumerate(lens):
        t = 0
        while t < T:  # the last Lq rows in one append
            m = min(37, T - Lq - t) if t < T - Lq else Lq
            sl = pool.reserve_append(seqs[b], m)
            pool.quantize_append(0, to_dev(kb[b][None, :, t:t + m], dt), to_dev(vb[b][None, :, t:t + m], dt), i32(sl[None]))
            t += m
    tab, n = pool.batch_tables(seqs, 6)
    starts = i32(pool.batch_starts(seqs))
    qb = rand_bits(rng, (len(lens), H * R, Lq, D), dt)
    o = pool.attention_windowed(0, to_dev(qb, dt), i32(tab), i32(n), starts, window, max(lens), scale)
    c = Cache.__new__(Cache)
    c.pool, c.lens, c.dt, c.k, c.v = pool, lens, dt, kb, vb
    c.check(o, qb, scale, "f32", window)
    if Lq == 1:  # and the fused step: the same token again, then turned by its absolute position
        cs, cs_d = rope(D)
        last = [to_dev(np.stack([x[b][:, -1:] for b in range(len(lens))]), dt) for x in (kb, vb)]
        got = pool.decode_append_attention_windowed(0, to_dev(qb, dt), *last, i32(tab), i32(n), starts, window, max(lens), scale)
        same(got.cpu().numpy(), o.cpu().numpy())
        got = pool.decode_append_attention_windowed(0, to_dev(qb, dt), *last, i32(tab), i32(n), starts, window, max(lens),
                                                    scale, cos_sin=cs_d)
        for b, T in enumerate(lens):
            for h in range(H):
                kb[b][h, -1:] = O.rope_rows(kb[b][h, -1:], Q.DT[dt], [T - 1], cs)
            for h in range(H * R):
                qb[b, h] = O.rope_rows(qb[b, h], Q.DT[dt], [T - 1], cs)
        c.check(got, qb, scale, "f32", window)
    pool.close()


@pytest.mark.parametrize("B,R", [(3, 2), (30, 4)])
@pytest.mark.parametrize("D", [64, 128, 512])
def test_shared_prefix(D, B, R):
    """Sequences forked from one prefix: the cascade, with the step's append fused, against 64 bits; a fork's
    append copies the shared tail block and leaves the other sequences alone."""
    rng = np.random.default_rng(B)
    H, dt, scale, P = 2, "bf16", 1 / np.sqrt(D), 130  # two shared blocks and a shared tail
    pool = make_pool(H, D, 100, dt)
    src = Cache(pool, [P], rng, dt)
    before = [x.cpu().numpy() for x in pool.gather_dequant(0, *src.tables(), P)]
    lens = [P + 1 + int(x) for x in rng.integers(0, 140, B)]
    seqs, ks, vs = [], [], []
    for T in lens:
        s = pool.seq_fork(src.seqs[0], P)
        seqs.append(s)
        m = T - P
        kb, vb = rand_bits(rng, (H, m, D), dt), rand_bits(rng, (H, m, D), dt)
        sl = pool.reserve_append(s, m)
        if m > 1:
            pool.quantize_append(0, to_dev(kb[None, :, :-1], dt), to_dev(vb[None, :, :-1], dt), i32(sl[None, :-1]))
        ks.append(np.concatenate([src.k[0], kb], 1))
        vs.append(np.concatenate([src.v[0], vb], 1))
    tab, n = pool.batch_tables(seqs, 6)
    qb = rand_bits(rng, (B, H * R, 1, D), dt)
    last = [to_dev(np.stack([x[:, -1:] for x in y]), dt) for y in (ks, vs)]
    o = pool.attention_shared_prefix(0, to_dev(qb, dt), i32(tab[0, :2]), i32(np.ascontiguousarray(tab[:, 2:])),
                                     i32(n - 128), max(lens) - 128, scale, k_new=last[0], v_new=last[1])
    c = Cache.__new__(Cache)
    c.pool, c.lens, c.dt, c.k, c.v = pool, lens, dt, ks, vs
    c.check(o, qb, scale, "f32")
    c.check(pool.attention(0, to_dev(qb, dt), i32(tab), i32(n), max(lens), scale), qb, scale, "f32")
    for a, b in zip(before, pool.gather_dequant(0, *src.tables(), P)):
        same(a, b.cpu().numpy())
    pool.close()


@pytest.mark.parametrize("Lq,path", [(1, 0), (6, 0), (6, 2)])
@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_rows_behind_a_sequence_do_not_matter(D, Lq, path):
    """Slots behind a sequence's end that hold NaN, infinities and large numbers from a longer past; stale table
    entries; lengths beyond max_seq_len are read up to it."""
    from krill_amd import _lib as L

    rng = np.random.default_rng(D)
    H, R, dt, scale, T, keep = 2, 3, "f16", 1 / np.sqrt(D), 200, 70
    pool = make_pool(H, D, 8, dt)
    pool.set_option(L.OPT_ATTN_PATH, path)
    kb, vb = rand_bits(rng, (H, T, D), dt), rand_bits(rng, (H, T, D), dt)
    for x in (kb, vb):
        x[:, keep:] = np.array([0x7e00, 0x7c00, 0xfc00, 0x7bff], np.uint16)[rng.integers(0, 4, (H, T - keep, D))]
    c = Cache(pool, [T], rng, dt, k=[kb], v=[vb])
    pool.seq_truncate(c.seqs[0], keep)
    c.lens, c.k, c.v = [keep], [kb[:, :keep]], [vb[:, :keep]]
    qb = rand_bits(rng, (1, H * R, Lq, D), dt)
    t, n = pool.batch_tables(c.seqs, 4)
    t[0, 2:] = [-1, 1 << 30]
    c.check(pool.attention(0, to_dev(qb, dt), i32(t), i32(n), 256, scale), qb, scale, "f32")
    pool.close()


@pytest.mark.parametrize("Lq,path", [(1, 0), (9, 0), (9, 2)])
def test_large_numbers(Lq, path):
    """Queries over the whole range of their type, V of the fp16 range, scores that rise block by block, one
    NaN row among others."""
    from krill_amd import _lib as L

    rng = np.random.default_rng(Lq)
    H, R, D, T = 1, 2, 128, 400
    for dt, qscale, kscale, rise in (("bf16", 1e30, 1e-3, 0.0), ("bf16", 1e-30, 1.0, 0.0), ("bf16", 3e38, 1.0, 0.0),
                                     ("f16", 1.0, 0.01, 3.0), ("f16", 1.0, 0.01, 7.9), ("f16", 1.0, 0.01, 40.0),
                                     ("f16", 30000.0, 1.0, 0.0), ("f16", 1e-6, 100.0, 0.0)):
        pool = make_pool(H, D, 8, dt)
        pool.set_option(L.OPT_ATTN_PATH, path)
        enc = O.f32_to_bf16_bits if dt == "bf16" else O.f32_to_f16_bits
        k = rng.standard_normal((H, T, D)).astype(np.float32) * kscale
        k[..., 0] += rise * (np.arange(T) // 64)
        v = rng.uniform(-60000, 60000, (H, T, D)).astype(np.float32)
        c = Cache(pool, [T], rng, dt, k=[enc(k)], v=[enc(v)])
        q = rng.uniform(-1, 1, (1, H * R, Lq, D)).astype(np.float32) * np.float32(qscale)
        if rise:
            q[..., 0] = 1.0
        qb = enc(q)
        scale = np.log(2.0) if rise else 1 / np.sqrt(D)
        t, n = c.tables()
        got = pool.attention(0, to_dev(qb, dt), t, n, T, float(np.float32(scale)))
        if qscale < 1e20:
            c.check(got, qb, float(np.float32(scale)), "f32")
        else:  # one key has all the weight: the row is that key's V, within rounding
            kd, vd = Q.stored(c.k[0][0], dt), Q.stored(c.v[0][0], dt)
            lo = O.bits_to_f32(qb, Q.DT[dt]).astype(np.float64)[0].reshape(-1, D)
            for i, row in enumerate(lo):
                upto = T - Lq + i % Lq + 1
                want = vd[int(np.argmax(kd[:upto] @ row))]
                np.testing.assert_allclose(got[0].reshape(-1, D)[i].cpu().numpy(), want, rtol=2.0 ** -19, atol=2.0 ** -4)
        if Lq > 1:
            clean = got.clone()
            qb[0, 0, 3, 5] = 0x7fc0 if dt == "bf16" else 0x7e00
            got = pool.attention(0, to_dev(qb, dt), t, n, T, float(np.float32(scale)))
            assert torch.isnan(got[0, 0, 3]).all()
            got[0, 0, 3] = clean[0, 0, 3]
            same(got.cpu().numpy(), clean.cpu().numpy())
        pool.close()


@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_results_repeat_and_do_not_depend_on_the_workspace(D):
    rng = np.random.default_rng(1)
    H, R, dt = 2, 4, "bf16"
    lens = [3000, 10, 700]
    pool = make_pool(H, D, 80, dt)
    c = Cache(pool, lens, rng, dt)
    t, n = c.tables()
    for Lq in (1, 8, 80):
        qb = to_dev(rand_bits(rng, (3, H * R, Lq, D), dt), dt)
        need = pool.workspace_size(3, H * R, Lq, 3000)
        outs = []
        for fill in (0, 0x7f, 0xff):
            ws = torch.full((need + 16,), fill, dtype=torch.uint8, device="cuda")
            outs.append(pool.attention(0, qb, t, n, 3000, 0.1, ws=ws).cpu().numpy())
            assert (ws[need:] == fill).all()
        same(outs[0], outs[1])
        same(outs[0], outs[2])
    pool.close()


@pytest.mark.parametrize("split", [1, 3, 64])
def test_chosen_splits(split):
    from krill_amd import _lib as L

    rng = np.random.default_rng(split)
    H, R, D, dt = 2, 5, 128, "bf16"
    lens = [900, 0, 64, 129]
    pool = make_pool(H, D, 40, dt)
    pool.set_option(L.OPT_SPLIT_BLOCKS, split)
    c = Cache(pool, lens, rng, dt)
    t, n = c.tables()
    for Lq in (1, 20):
        if Lq > 1:
            c.lens = [900, 30, 64, 129]
            c.k[1], c.v[1] = rand_bits(rng, (H, 30, D), dt), rand_bits(rng, (H, 30, D), dt)
            sl = pool.reserve_append(c.seqs[1], 30)
            pool.quantize_append(0, to_dev(c.k[1][None], dt), to_dev(c.v[1][None], dt), i32(sl[None]))
            t, n = c.tables()
        qb = rand_bits(rng, (4, H * R, Lq, D), dt)
        c.check(pool.attention(0, to_dev(qb, dt), t, n, 900, 0.1), qb, 0.1, "f32")
    pool.close()


def test_many_sequences():
    rng = np.random.default_rng(2)
    H, R, D, dt = 1, 4, 64, "bf16"
    lens = [int(x) for x in rng.integers(0, 200, 150)]
    pool = make_pool(H, D, 500, dt)
    c = Cache(pool, lens, rng, dt)
    t, n = c.tables()
    qb = rand_bits(rng, (150, H * R, 1, D), dt)
    c.check(pool.attention(0, to_dev(qb, dt), t, n, max(lens), 0.125), qb, 0.125, "f32")
    pool.close()


def test_step_in_a_graph_on_another_stream():
    """A captured step replayed over a growing sequence, eager work between the replays; two graphs share a
    workspace."""
    rng = np.random.default_rng(3)
    H, R, D, dt, scale = 2, 4, 128, "bf16", 0.1
    pool = make_pool(H, D, 24, dt, layers=2)
    start = [100, 62, 5]
    c = Cache(pool, start, rng, dt)
    for b, T in enumerate(start):  # layer 1 holds the same tokens
        t, n = pool.batch_tables([c.seqs[b]], 3)
        sl = t[0][np.arange(T) // 64] * 64 + np.arange(T) % 64
        pool.quantize_append(1, to_dev(c.k[b][None], dt), to_dev(c.v[b][None], dt), i32(sl[None]))
    steps = 4
    kb, vb, qb = (rand_bits(rng, (steps, 3, h, 1, D), dt) for h in (H, H, H * R))
    kd, vd, qd = (to_dev(x[0], dt) for x in (kb, vb, qb))
    tabs, lens = i32(np.zeros((3, 4))), i32(np.zeros(3))
    outs = [torch.empty((3, H * R, 1, D), dtype=torch.float32, device="cuda") for _ in range(2)]
    ws = torch.empty(pool.workspace_size(3, H * R, 1, 256), dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    graphs = []

    def one(layer):
        pool.decode_append_attention(layer, qd, kd, vd, tabs, lens, 256, scale, ws=ws, out=outs[layer])

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one(0)  # (lengths of zero: nothing is written)
        for layer in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                one(layer)
            graphs.append(g)
    torch.cuda.synchronize()
    for i in range(steps):
        for s in c.seqs:
            pool.reserve_append(s, 1)
        pool.flush()
        t, n = pool.batch_tables(c.seqs, 4)
        for dst, src in ((kd, kb), (vd, vb), (qd, qb)):
            dst.copy_(to_dev(src[i], dt))
        tabs.copy_(i32(t))
        lens.copy_(i32(n))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for g in graphs:
                g.replay()
        torch.cuda.synchronize()
        c.lens = [int(x) for x in n]
        for b in range(3):
            c.k[b] = np.concatenate([c.k[b], kb[i][b]], 1)
            c.v[b] = np.concatenate([c.v[b], vb[i][b]], 1)
        for o in outs:
            c.check(o, qb[i], scale, "f32")
        eager = pool.attention(0, qd, tabs, lens, 256, scale)
        same(eager.cpu().numpy(), outs[0].cpu().numpy())
    pool.close()


def test_prefix_entries_and_the_cache_api():
    from krill_amd.cache import PrefixCache, make_quantized_kv_caches

    rng = np.random.default_rng(9)
    H, D, dt, T = 2, 128, "bf16", 90
    pool = make_pool(H, D, 24, dt, layers=2)
    caches = make_quantized_kv_caches(pool)
    kb, vb = rand_bits(rng, (1, H, T, D), dt), rand_bits(rng, (1, H, T, D), dt)
    for layer in caches:
        k, v = layer.update(to_dev(kb, dt), to_dev(vb, dt))
        same(k[0].cpu().numpy(), Q.read_back(Q.stored(kb[0], dt)))
        same(v[0].cpu().numpy(), Q.read_back(Q.stored(vb[0], dt)))
        assert layer.memory_size_bytes == T * H * (D + 8 * (D // 64))
    assert pool.seq_memory_bytes(caches[0].s.seq) == T * H * (D + 8 * (D // 64))
    assert pool.stats()["block_bytes"] == 64 * H * (D + 8 * (D // 64))
    pc = PrefixCache(pool)
    tokens = list(range(T))
    assert pc.store_quantized(tokens, caches[0].s.seq)
    n, entry = pc.lookup_longest_prefix_quantized(tokens[:70] + [-1])
    assert n == 70
    f = pool.seq_fork(entry, n)
    t, ln = pool.batch_tables([f], 2)
    k, v = pool.gather_dequant(1, i32(t), i32(ln), n)
    same(k[0].cpu().numpy(), Q.read_back(Q.stored(kb[0][:, :70], dt)))
    pool.close()


def test_refusals():
    import krill_amd
    from krill_amd import _lib as L
    from krill_amd._lib import KrillError

    pool = make_pool(1, 128, 4)
    Cache(pool, [10], np.random.default_rng(0), "bf16")
    t, n = i32(np.zeros((1, 1))), i32(np.array([10]))
    with pytest.raises(KrillError) as e:
        pool.gather(0, t, n, 10)
    assert e.value.code == L.KRILL_E_UNSUPPORTED
    with pytest.raises(KrillError) as e:
        z = torch.zeros((1, 1, 4, 128), dtype=torch.uint8, device="cuda")
        m = torch.zeros((1, 1, 4, 2), dtype=torch.float16, device="cuda")
        pool.scatter(0, dict(keys=z, values=z, key_scales=m, key_zeros=m, value_scales=m, value_zeros=m), i32([0]),
                     i32(np.arange(4)[None]))
    assert e.value.code == L.KRILL_E_UNSUPPORTED
    with pytest.raises(KrillError):
        pool.read_slots(1, i32([[0]]))
    with pytest.raises(ValueError):
        pool.read_slots(0, i32([0]))
    q = torch.zeros((1, 3, 1, 128), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(KrillError) as e:  # max_seq_len past the table
        pool.attention(0, q, t, n, 100, 1.0)
    assert e.value.code == L.KRILL_E_RANGE
    with pytest.raises(KrillError) as e:
        pool.attention(0, q, t, n, 64, float("nan"))
    assert e.value.code == L.KRILL_E_INVAL
    two = krill_amd.KVPool(1, 2, 128, 4, "affine4_g64", "bf16")
    with pytest.raises(KrillError) as e:  # 3 heads over 2
        two.attention(0, q, t, n, 64, 1.0)
    assert e.value.code == L.KRILL_E_INVAL
    two.close()
    pool.close()


@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("Lq,R,window", [(2, 1, 0), (70, 3, 0), (200, 1, 0), (70, 2, 50), (70, 1, 100)])
def test_long_windows_with_bf16_outputs(D, Lq, R, window):
    """The long-window kernel's form for bf16 outputs; slots behind the sequences hold NaN and infinities, one
    row of the queries a NaN."""
    from krill_amd import _lib as L

    rng = np.random.default_rng(Lq + window)
    H, dt, scale = 2, "bf16", 1 / np.sqrt(D)
    lens = [Lq, Lq + 100, 64 * ((Lq + 63) // 64) + 1, 333]
    pool = make_pool(H, D, 40, dt)
    pool.set_option(L.OPT_ATTN_PATH, 2)
    junk = np.array([0x7fc0, 0x7f80, 0xff80, 0x7f7f], np.uint16)[rng.integers(0, 4, (1, H, pool.num_blocks * 64, D))]
    pool.quantize_append(0, to_dev(junk, dt), to_dev(junk, dt), all_slots(pool))
    c = Cache(pool, lens, rng, dt)
    qb = rand_bits(rng, (len(lens), H * R, Lq, D), dt)
    t, n = c.tables()

    def run():
        if window:
            return pool.attention_windowed(0, to_dev(qb, dt), t, n, None, window, max(lens), scale, out_dtype=torch.bfloat16)
        return pool.attention(0, to_dev(qb, dt), t, n, max(lens), scale, out_dtype=torch.bfloat16)

    clean = run()
    c.check(clean, qb, scale, "bf16", window, long=True)
    qb[1, 0, Lq // 2, 3] = 0x7fc0
    got = run()
    assert torch.isnan(got[1, 0, Lq // 2]).all()
    got[1, 0, Lq // 2] = clean[1, 0, Lq // 2]
    same(got.float().cpu().numpy(), clean.float().cpu().numpy())
    pool.close()


@pytest.mark.parametrize("L", [1, 17])
def test_append_of_more_sequences_than_a_grid_dimension(L):
    """A batch past 65535 rows of slots, nearly all of them skipped."""
    rng = np.random.default_rng(L)
    B, H, D, blocks = 65536 + 5, 1, 64, 4
    pool = make_pool(H, D, blocks)
    kb = np.zeros((B, H, L, D), np.uint16)
    vb = np.zeros_like(kb)
    slots = np.full((B, L), -1, np.int32)
    for i, b in enumerate((0, 40000, 65535, 65536, B - 1)):
        kb[b], vb[b] = rand_bits(rng, (H, L, D), "bf16"), rand_bits(rng, (H, L, D), "bf16")
        slots[b] = 1 + 40 * i + np.arange(L)
    pool.quantize_append(0, to_dev(kb, "bf16"), to_dev(vb, "bf16"), i32(slots))
    want = np.zeros((2, H, blocks * 64, D), np.float16)
    for b in np.flatnonzero(slots[:, 0] >= 0):
        want[0][:, slots[b]] = Q.read_back(Q.stored(kb[b], "bf16"))
        want[1][:, slots[b]] = Q.read_back(Q.stored(vb[b], "bf16"))
    k, v = pool.read_slots(0, all_slots(pool))
    same(k[0].cpu().numpy(), want[0])
    same(v[0].cpu().numpy(), want[1])
    pool.close()


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("D,R,chunk", [(64, 4, 96), (128, 5, 64), (256, 2, 33)])
def test_batcher_over_a_4bit_pool(D, R, chunk, out):
    """Requests that come and go: chunked prefill, batched decode steps, blocks given back and reused; every
    output of every request and layer against 64 bits over that request's own tokens."""
    from krill_amd.batcher import ContinuousBatcher, Request

    H, layers, dt = 2, 2, "bf16"
    reqs = [Request(rid, T, g) for rid, T, g in [(0, 70, 5), (1, 5, 9), (2, 130, 3), (3, 64, 6), (4, 1, 4), (5, 200, 2)]]
    arrivals = {0: reqs[:2], 1: reqs[2:3], 4: reqs[3:5], 6: reqs[5:]}

    class Model:
        def __init__(self):
            self.x, self.out = {}, {}
            for r in reqs:
                rng, T = np.random.default_rng(r.rid + D), r.prompt_len + r.max_new_tokens
                for l in range(layers):
                    self.x[r.rid, l] = [rand_bits(rng, (n, T, D), dt) for n in (H * R, H, H)]
                    self.out[r.rid, l] = np.full((H * R, T, D), np.nan)

        def prefill(self, req, start, n, layer):
            return tuple(to_dev(a[None, :, start:start + n], dt) for a in self.x[req.rid, layer])

        def decode(self, rs, positions, layer):
            return tuple(to_dev(np.stack([self.x[r.rid, layer][i][:, p:p + 1] for r, p in zip(rs, positions)]), dt)
                         for i in range(3))

        def consume(self, rs, layer, positions, o):
            o = o.float().cpu().numpy()
            if len(rs) == 1:
                self.out[rs[0].rid, layer][:, positions] = o[0]
            else:
                for b, (r, p) in enumerate(zip(rs, positions)):
                    self.out[r.rid, layer][:, p] = o[b, :, 0]

    pool = make_pool(H, D, 16, dt, layers)
    model, scale = Model(), D ** -0.5
    cb = ContinuousBatcher(pool, model, 3, H * R, scale, prefill_chunk=chunk,
                           out_dtype=torch.float32 if out == "f32" else torch.bfloat16)
    for step in range(100):
        for r in arrivals.get(step, []):
            cb.submit(r)
        if cb.idle and step > max(arrivals):
            break
        cb.step()
    torch.cuda.synchronize()
    assert cb.idle
    for r in reqs:
        T = r.prompt_len + r.max_new_tokens
        for l in range(layers):
            qb, kb, vb = model.x[r.rid, l]
            qf = O.bits_to_f32(qb, Q.DT[dt]).astype(np.float64)
            for h in range(H):
                kd, vd = Q.stored(kb[h], dt), Q.stored(vb[h], dt)
                rows, hi = qf[h * R:(h + 1) * R].reshape(R * T, D), np.tile(np.arange(1, T + 1), R)
                want = Q.attention(rows, kd, vd, np.zeros_like(hi), hi, scale)
                got = model.out[r.rid, l][h * R:(h + 1) * R].reshape(R * T, D)
                lim = Q.bound(rows, kd, vd, scale, want, out, *(Q.quantize(x[h], dt)[1].max() for x in (kb, vb)), long=True)
                assert np.all(np.abs(got - want) <= lim), f"request {r.rid} layer {l} head {h}"
    pool.close()


@pytest.mark.parametrize("out", ["bf16", "f16"])
@pytest.mark.parametrize("Lq,R,path,split", [(2, 1, 2, 0), (9, 5, 2, 0), (9, 5, 2, 1), (70, 2, 1, 0), (70, 2, 0, 1)])
@pytest.mark.parametrize("window", [2, 100])
@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_windows_on_chosen_paths(D, window, Lq, R, path, split, out):
    """Sliding windows on the kernel and the block ranges a caller asks for."""
    from krill_amd import _lib as L

    rng = np.random.default_rng(window * Lq + D)
    H, dt, scale = 2, "bf16", 1 / np.sqrt(D)
    lens = [Lq, 130 + Lq, 331]
    pool = make_pool(H, D, 30, dt)
    for o, x in ((L.OPT_WINDOW, window), (L.OPT_ATTN_PATH, path), (L.OPT_SPLIT_BLOCKS, split)):
        pool.set_option(o, x)
    kb = [rand_bits(rng, (H, T, D), dt) for T in lens]
    vb = [rand_bits(rng, (H, T, D), dt) for T in lens]
    seqs = [pool.seq_create() for _ in lens]
    for b, T in enumerate(lens):
        for t0, t1 in ((0, T - Lq), (T - Lq, T)):
            if t1 > t0:
                sl = pool.reserve_append(seqs[b], t1 - t0)
                pool.quantize_append(0, to_dev(kb[b][None, :, t0:t1], dt), to_dev(vb[b][None, :, t0:t1], dt), i32(sl[None]))
    tab, n = pool.batch_tables(seqs, 6)
    starts = i32(pool.batch_starts(seqs))
    qb = rand_bits(rng, (len(lens), H * R, Lq, D), dt)
    c = Cache.__new__(Cache)
    c.pool, c.lens, c.dt, c.k, c.v = pool, lens, dt, kb, vb
    got = pool.attention_windowed(0, to_dev(qb, dt), i32(tab), i32(n), starts, window, max(lens), scale,
                                  out_dtype={"bf16": torch.bfloat16, "f16": torch.float16}[out])
    c.check(got, qb, scale, out, window, long=True)
    pool.close()
