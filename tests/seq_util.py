"""What the tests of the paged cache and of attention over packed sequences share: the operators written out in numpy
(64 bits, one request and one row after the other, straight from the definitions in include/hodu_rocm_kernels.h), and
the bound that an attention output may be off by."""
import numpy as np
import torch

import helpers as H
from hodu_amd import ffi

TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f8e4m3": torch.float8_e4m3fn}
HALF_STEP = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f8e4m3": 2.0 ** -4}  # of a rounding, relative to the value


def to_bits(x, dt):
    """float64 values rounded to dt (nearest even), as storage words"""
    t = torch.from_numpy(np.ascontiguousarray(x, dtype=np.float64)).to(torch.float32)
    if dt == "f8e4m3":
        return t.clamp(-448, 448).to(TORCH[dt]).view(torch.uint8).numpy()
    return t.to(TORCH[dt]).view(torch.int16).numpy().view(np.uint16)


def widen(bits, dt):
    t = torch.from_numpy(np.ascontiguousarray(bits).view(np.uint8 if dt == "f8e4m3" else np.int16))
    return t.view(TORCH[dt]).to(torch.float64).numpy()


# ---- block tables and slot maps ---------------------------------------------------------------------------------------
def plan_reference(cached, added, free, table, page, capacity):
    """(table, lens, offsets, slots, used), one request after the other"""
    table, width = table.copy(), table.shape[1] if table.ndim == 2 else 0
    lens, offsets, slots = [], [0], np.full(capacity, -1, np.int64)
    taken = total = refused = 0
    list_out = capacity_out = False  # dealt out in order: whoever needs one after it ran out is refused too
    for r, (c, n) in enumerate(zip(cached.tolist(), added.tolist())):
        fits = c >= 0 and n >= 0 and c + n <= width * page
        held, need = (-(-c // page), -(-(c + n) // page)) if fits else (0, 0)
        fresh = need - held
        ok = fits
        if ok and fresh and (list_out or taken + fresh > len(free)):
            ok, list_out = False, True
        if ok and n and (capacity_out or total + n > capacity):
            ok, capacity_out = False, True
        if not ok:
            refused += 1
            lens.append(max(c, 0))
            offsets.append(total)
            continue
        for i in range(fresh):
            table[r, held + i] = free[taken + i]
        for i in range(n):
            slots[total + i] = int(table[r, (c + i) // page]) * page + (c + i) % page
        taken += fresh
        total += n
        lens.append(c + n)
        offsets.append(total)
    return table, np.array(lens, np.int32), np.array(offsets, np.int32), slots.astype(np.int32), np.array([taken, refused], np.int32)


# ---- attention --------------------------------------------------------------------------------------------------------
def attend(q, k, v, scale, causal):
    """q [n, Hq, D], k, v [m, Hkv, D] float64 -> (o [n, Hq, D], weighted |v| [n, Hq, D], largest sum of |q k| scale [n, Hq],
    1 / sum of p relative to the largest [n, Hq])"""
    n, hq, d = q.shape
    m, hk, _ = k.shape
    o, a = np.zeros((n, hq, d)), np.zeros((n, hq, d))
    size, inv = np.zeros((n, hq)), np.zeros((n, hq))
    for h in range(hq):
        kk, vv = k[:, h // (hq // hk)], v[:, h // (hq // hk)]
        for i in range(n):
            open_ = max(0, i + m - n + 1) if causal else m
            if open_ == 0:
                continue
            s = kk[:open_] @ q[i, h] * scale
            p = np.exp(s - s.max())
            inv[i, h] = 1.0 / p.sum()
            p *= inv[i, h]
            o[i, h] = p @ vv[:open_]
            a[i, h] = p @ np.abs(vv[:open_])
            size[i, h] = (np.abs(kk[:open_]) @ np.abs(q[i, h])).max() * scale
    return o, a, size, inv


def allowed(dt, o, a, size, inv, m, vmax, d):
    """How far an output may be from o.  With u half a step of dt and e = 2^-24:
      * P is rounded to dt as the second product's operand: u of every term, u a in all (a = sum of p |v|); an f16 P below
        its normal range is off by 2^-25 of the largest P each, of which the row has m and the sum l = 1 / inv: m 2^-25 inv vmax
      * the scores are sums of D products in f32, off by (D + 2) e of the sum of their terms' sizes; through the
        exponential that is a relative error of P, and of l: 2 (D + 2) e size; base-2 exponential, its argument's
        fused multiply-add (|argument| e) and the rescalings 8 e + size e, twice
      * sums over the keys in f32: (m + 8) e a
      * the row sum is taken over the rounded P: off by u of itself at most, u |o|
      * the result is rounded once: u |o|, in f16 at least 2^-25"""
    u, e = HALF_STEP[dt], 2.0 ** -24
    rel = u + 2 * ((d + 2) * e * size + 8 * e + 2 * size * e) + (m + 8) * e
    tol = a * rel[..., None] + 2 * np.abs(o) * u
    if dt == "f16":
        tol = tol + (m * 2.0 ** -25 * inv * vmax)[..., None] + 2.0 ** -25
    return tol * (1 + 2 * u) + 1e-30


def assert_attention(got, parts, dt, m, vmax, d, what=""):
    o, a, size, inv = parts
    tol = allowed(dt, o, a, size, inv, m, vmax, d)
    off = np.abs(got - o)
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} outputs, worst {np.nanmax(np.where(bad, off / tol, 0)):.3g} times the bound, " \
                          f"first at {np.argwhere(bad)[0].tolist()}: got {got[tuple(np.argwhere(bad)[0])]}, want {o[tuple(np.argwhere(bad)[0])]}"


POISON = 0x7E57  # a bit pattern that outputs are filled with: a finite bf16 and an f16 NaN


class Side:
    """a [d0, .., D] operand laid out in memory with the given order of axes (innermost: the last of `order`, D always dense),
    a gap behind the tensor axis and an offset: element strides and the flat storage"""

    def __init__(self, values, dt, order=None, gap=0, offset=0, fill=0):
        nd = values.ndim
        order = list(range(nd)) if order is None else list(order) + [nd - 1]
        shape = values.shape
        strides, acc = [0] * nd, 1
        for n, ax in enumerate(reversed(order)):
            strides[ax] = acc
            acc *= shape[ax]
            if n == 0:
                acc += gap
        self.strides, self.offset, self.dt = strides, offset, dt
        bits = to_bits(values, dt)
        self.flat = np.full(offset + acc + gap, fill, bits.dtype)
        np.lib.stride_tricks.as_strided(self.flat[offset:], shape, [s * bits.itemsize for s in strides])[...] = bits
        self.values = widen(bits, dt).reshape(shape)

    def view(self, flat):
        shape = self.values.shape
        return np.lib.stride_tricks.as_strided(flat[self.offset:], shape, [s * flat.itemsize for s in self.strides])


def scalar(d, dt):
    bits = to_bits(np.array([d ** -0.5]), dt)
    return bits, float(widen(bits, dt)[0])


def run_varlen(ctx, dt, lens_q, lens_k, hq, hk, d, causal, seed=0, q_order=None, k_order=None, gap=0, offset=0, spare=0, qscale=1.0,
               expect=None, edit=None, shared_offsets=False):
    """one hodu_rocm_attention_varlen call against the definition; spare: packed rows behind the last sequence"""
    g = np.random.default_rng(seed)
    tq, tk = sum(lens_q) + spare, sum(lens_k) + spare
    q = g.standard_normal((tq, hq, d)) * qscale
    k, v = g.standard_normal((tk, hk, d)), g.standard_normal((tk, hk, d))
    if edit is not None:
        edit(q, k, v)
    q, k, v = Side(q, dt, q_order, gap, offset), Side(k, dt, k_order, gap, offset), Side(v, dt, k_order, gap, 2 * offset)
    qo, ko = np.cumsum([0] + lens_q).astype(np.int32), np.cumsum([0] + lens_k).astype(np.int32)
    bits, scale = scalar(d, dt)
    out = ctx.upload(np.full(tq * hq * d, POISON, np.uint16))
    md = ffi.varlen_md(len(lens_q), tq, tk, hq, hk, d, q.strides[:2], k.strides[:2], v.strides[:2], q.offset, k.offset, v.offset)
    dqo = ctx.upload(qo)
    ctx.attention_varlen(dt, ctx.upload(q.flat), ctx.upload(k.flat), ctx.upload(v.flat), out, dqo, dqo if shared_offsets else ctx.upload(ko), md,
                         bits, causal)
    if expect:
        assert expect in ctx.last_kernel(), ctx.last_kernel()
    raw = ctx.download(out, np.uint16).reshape(tq, hq, d)
    got = widen(raw, dt).reshape(raw.shape)
    for b, (n, m) in enumerate(zip(lens_q, lens_k)):
        kb, vb = k.values[ko[b]:ko[b + 1]], v.values[ko[b]:ko[b + 1]]
        parts = attend(q.values[qo[b]:qo[b + 1]], kb, vb, scale, causal)
        assert_attention(got[qo[b]:qo[b + 1]], parts, dt, m, np.abs(vb).max() if m else 0.0, d, f"sequence {b}: {n} rows, {m} keys")
    assert np.all(raw[qo[-1]:] == POISON)  # rows behind the last sequence
    return raw


def make_cache(g, dt, pages, page, hk, d, order=None, gap=0, offset=0, garbage=None):
    """a cache side; garbage: the storage word that slots nobody wrote hold"""
    x = g.standard_normal((pages, page, hk, d)) * (16.0 if dt == "f8e4m3" else 1.0)
    return Side(x, dt, order, gap, offset)


def run_paged(ctx, dt, new, lens, hq, hk, d, page, cache_dt=None, seed=0, order=None, gap=0, offset=0, spare=0, width_extra=1, qscale=1.0,
              expect=None, garbage=None, q_order=None):
    """one hodu_rocm_attention_paged call against the definition; garbage: a storage word for every slot that is not in use"""
    cache_dt = cache_dt or dt
    g = np.random.default_rng(seed)
    counts = [-(-n // page) for n in lens]
    pages, width = sum(counts) + 2, max(counts + [0]) + width_extra
    order_of = g.permutation(pages)
    table, at = np.full((len(lens), width), -1, np.int32), 0
    used = np.zeros((pages, page), bool)
    for b, n in enumerate(counts):
        table[b, :n] = order_of[at:at + n]
        at += n
        for t in range(lens[b]):
            used[table[b, t // page], t % page] = True
    kc, vc = make_cache(g, cache_dt, pages, page, hk, d, order, gap, offset), make_cache(g, cache_dt, pages, page, hk, d, order, gap, 2 * offset)
    if garbage is not None:
        for side in (kc, vc):
            side.view(side.flat)[~used] = garbage
    tq = sum(new) + spare
    q = Side(g.standard_normal((tq, hq, d)) * qscale, dt, q_order)
    qo = np.cumsum([0] + new).astype(np.int32)
    bits, scale = scalar(d, dt)
    ks = vs = np.ones(hk)
    scales = {}
    if cache_dt == "f8e4m3":
        ks, vs = (np.linspace(0.05, 0.1, hk).astype(np.float32), np.linspace(0.03, 0.07, hk).astype(np.float32))
        scales = dict(k_scale=ctx.upload(ks), v_scale=ctx.upload(vs))
    out = ctx.upload(np.full(tq * hq * d, POISON, np.uint16))
    md = ffi.paged_attention_md(len(lens), tq, hq, hk, d, pages, page, width, q.strides[:2], kc.strides[:3], vc.strides[:3], q.offset, kc.offset,
                                vc.offset)
    ctx.attention_paged(dt, ctx.upload(q.flat), ctx.upload(kc.flat), ctx.upload(vc.flat), out, ctx.upload(qo), ctx.upload(table),
                        ctx.upload(np.array(lens, np.int32)), md, bits, cache_dt=cache_dt, **scales)
    if expect:
        assert expect in ctx.last_kernel(), ctx.last_kernel()
    raw = ctx.download(out, np.uint16).reshape(tq, hq, d)
    got = widen(raw, dt).reshape(raw.shape)
    for b, (n, m) in enumerate(zip(new, lens)):
        t = np.arange(m)
        kb = kc.values[table[b, t // page], t % page] * ks.astype(np.float64)[:, None]
        vb = vc.values[table[b, t // page], t % page] * vs.astype(np.float64)[:, None]
        parts = attend(q.values[qo[b]:qo[b + 1]], kb, vb, scale, True)
        assert_attention(got[qo[b]:qo[b + 1]], parts, dt, m, np.abs(vb).max() if m else 0.0, d, f"request {b}: {n} rows, {m} keys")
    assert np.all(raw[qo[-1]:] == POISON)
    return raw
