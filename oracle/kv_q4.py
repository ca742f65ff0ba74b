"""Oracle of the 4-bit KV cache (test infrastructure only): numpy, 64 bits.

Restates the record format of include/b200_attn.h (80 bytes per (token, kv head): codes of
four groups of 32 dimensions, then scale and minimum of each group as 16-bit floats) and
attention over the values the records stand for.
"""
import numpy as np

D, GROUP, RECORD = 128, 32, 80
MIN_SCALE = 2.0 ** -100


def float_bits(x, bf16):
    """uint16 patterns of float64 values rounded to bf16 / fp16 (nearest even); NaN -> 0x7fff."""
    x = np.asarray(x, np.float64)
    if bf16:
        # Through fp32 rounded to odd (an inexact value ends in a one), which no second rounding can tell
        # from the value itself.
        with np.errstate(over="ignore", invalid="ignore"):
            f = x.astype(np.float32)
            even = (f.view(np.uint32) & 1 == 0) & (f != x) & np.isfinite(f)
            f = np.where(even, np.nextafter(f, np.where(x > f, np.float32(np.inf), np.float32(-np.inf))), f)
            u = f.view(np.uint32).astype(np.uint64)
        r = ((u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    else:
        with np.errstate(over="ignore"):
            r = x.astype(np.float16).view(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7fff), r)


def bits_float(b, bf16):
    b = np.asarray(b, np.uint16)
    if bf16:
        return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return b.view(np.float16).astype(np.float64)


def quantise(x, bf16):
    """x float64 [..., 128] of 16-bit values -> (codes uint8 [..., 4, 32], scale bits, min bits uint16 [..., 4])."""
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        g = np.asarray(x, np.float64).reshape(*x.shape[:-1], D // GROUP, GROUP)
        lo = g.min(-1)
        span = (g.max(-1) - lo).astype(np.float32)  # differences are fp32
        ok = np.isfinite(span)
        s_bits = float_bits(np.where(ok, span.astype(np.float64) / 15, np.nan), bf16)
        s = bits_float(s_bits, bf16)
        tiny = ok & (s < MIN_SCALE)
        s_bits = np.where(tiny, 0, s_bits).astype(np.uint16)
        s = np.where(tiny, 0.0, s)
        use = ok & (s > 0)
        q = np.rint((g - lo[..., None]).astype(np.float32).astype(np.float64) / np.where(use, s, 1.0)[..., None])
        codes = np.where(use[..., None], np.clip(q, 0, 15), 0).astype(np.uint8)
        m_bits = np.where(ok, float_bits(np.where(ok, lo, np.nan), bf16), 0x7fff).astype(np.uint16)
    return codes, s_bits, m_bits


def pack(codes, s_bits, m_bits):
    """Records uint8 [..., 80]."""
    lead = codes.shape[:-2]
    rec = np.zeros((*lead, RECORD), np.uint8)
    for d in range(D):
        i = d % 8
        nib = i // 2 + 4 * (i % 2)
        rec[..., 4 * (d // 8) + nib // 2] |= (codes[..., d // GROUP, d % GROUP] << (4 * (nib % 2))).astype(np.uint8)
    for j in range(D // GROUP):
        for o, b in ((0, s_bits), (2, m_bits)):
            rec[..., 64 + 4 * j + o] = b[..., j] & 0xff
            rec[..., 64 + 4 * j + o + 1] = b[..., j] >> 8
    return rec


def unpack(rec, bf16):
    """(codes [..., 4, 32], s [..., 4], m [..., 4]) in float64."""
    codes = np.empty((*rec.shape[:-1], D // GROUP, GROUP), np.float64)
    for d in range(D):
        i = d % 8
        nib = i // 2 + 4 * (i % 2)
        codes[..., d // GROUP, d % GROUP] = (rec[..., 4 * (d // 8) + nib // 2] >> (4 * (nib % 2))) & 15
    w = rec[..., 64:].astype(np.uint16)
    s = bits_float(w[..., 0::4] | (w[..., 1::4] << 8), bf16)
    m = bits_float(w[..., 2::4] | (w[..., 3::4] << 8), bf16)
    return codes, s, m


def values(rec, bf16):
    """float64 [..., 128], unrounded."""
    codes, s, m = unpack(rec, bf16)
    return (codes * s[..., None] + m[..., None]).reshape(*rec.shape[:-1], D)


def attention(q, k_rec, v_rec, block_tables, context_lens, scale, bf16):
    """q float64 [B, Lq, Hq, 128]; caches uint8 [NB, Hkv, bs, 80]; float64 [B, Lq, Hq, 128].

    Also returns a bound on the error a kernel with fp32 scores and fp16 probabilities may make
    before it rounds its output, per element (see tolerance())."""
    B, lq, hq, d = q.shape
    nb, hkv, bs, _ = k_rec.shape
    g = hq // hkv
    out = np.zeros(q.shape)
    bound = np.zeros(q.shape)
    for b in range(B):
        n = min(int(context_lens[b]), block_tables.shape[1] * bs)
        if n <= 0:
            continue
        pages = np.asarray(block_tables[b, :(n + bs - 1) // bs])
        inside = (pages >= 0) & (pages < nb)
        safe = np.where(inside, pages, 0)
        kr = np.where(inside[:, None, None, None], k_rec[safe], 0).transpose(1, 0, 2, 3).reshape(hkv, -1, RECORD)[:, :n]
        vr = np.where(inside[:, None, None, None], v_rec[safe], 0).transpose(1, 0, 2, 3).reshape(hkv, -1, RECORD)[:, :n]
        K, V = values(kr.astype(np.uint8), bf16), values(vr.astype(np.uint8), bf16)
        _, sv, mv = unpack(vr.astype(np.uint8), bf16)
        _, sk, mk = unpack(kr.astype(np.uint8), bf16)
        for i in range(lq):
            m = n - lq + i + 1
            if m <= 0:
                continue
            qi = q[b, i].reshape(hkv, g, d)
            s = np.einsum("hgd,hnd->hgn", qi, K[:, :m]) * scale
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            out[b, i] = np.einsum("hgn,hnd->hgd", p, V[:, :m]).reshape(hq, d)
            # scores: sums of the magnitudes |q| (15 s + |m|), held to 2^-20
            mag = np.einsum("hgjd,hnj->hgn", np.abs(qi).reshape(hkv, g, 4, 32),
                            15 * np.abs(sk[:, :m]) + np.abs(mk[:, :m])) * scale
            delta = mag.max(-1) * 2.0 ** -20                                          # [hkv, g]
            reach = np.maximum((15 * np.abs(sv[:, :m]) + np.abs(mv[:, :m])).max((1, 2)),
                               np.maximum(16 * np.abs(sv[:, :m]), np.abs(mv[:, :m])).max((1, 2)))  # [hkv]
            span = (15 * np.abs(sv[:, :m])).max((1, 2)) if bf16 else np.zeros(hkv)
            e = (2 * delta * reach[:, None]
                 + (reach * (2.0 ** -11 + m * 2.0 ** -24 + m * 2.0 ** -27 + 2.0 ** -20) + span * 2.0 ** -11)[:, None])
            bound[b, i] = np.repeat(e.reshape(hq, 1), d, 1)
    return out, bound


def tolerance(want, bound, bf16):
    """Largest error of an output: half a step of its 16-bit type, and the kernel's own bound.

    The bound's terms, with R the largest |value| a row may meet:
      * a relative error of 2^-20 of the scores' magnitude changes a weighted mean of values by at
        most twice that times R;
      * probabilities rounded to fp16, in the numerator and the sum alike: a mean over changed
        weights moves by at most sum |change| |v - mean| / sum p.  Half a step of fp16 is 2^-11
        of p, and the mean absolute deviation of values in [-R, R] is at most R: 2^-11 R.  Below
        2^-14 the step is absolute, half of it 2^-25, each of m tokens off the mean by at most
        2 R, the sum at least 1 (the running maximum's own p): m 2^-24 R;
      * p s rounded to fp16 before it meets codes up to 15 (bf16 models; fp16 ones keep the rest):
        2^-11 of at most 15 s, and below 2^-14 half of 2^-24 in units of at most R / 64: m 2^-27 R;
      * 2^-20 R for the fp32 sums and exponentials."""
    return np.abs(want) * (2.0 ** -8 if bf16 else 2.0 ** -11) + bound + (2.0 ** -130 if bf16 else 2.0 ** -25)
