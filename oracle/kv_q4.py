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


def attention_bound(q, k_rec, v_rec, block_tables, context_lens, scale, bf16):
    """As attention(), with a bound that is each element's own: its group's parameters under the
    row's own probabilities, in place of the largest value that the row may meet.

    With w_t a row's probabilities, o its output, and s_t, m_t, n_t the scale and minimum of the element's
    group and its code at token t (v_t = n_t s_t + m_t), N tokens seen, R the group's largest max(16 s, |m|):
      * scores off by d_t move a weighted mean by sum w_t d_t (v_t - o).  Products of 16-bit
        operands are exact, sums fp32, and sum(q) is held to 2^-23 of sum |q|: d_t is 2^-20 of
        scale * sum |q| (n s + |m|).  Queries are 16-bit operands in units of a power of two in which the
        row's largest is at least 1/2: below 2^-14 half a step is 2^-25, so each element adds 2^-24 max|q| n s;
      * a matrix product of 16 terms cuts each term (and the running sum) at 2^-25 of the largest exponent
        sum among its operands, in which a code that is a subnormal counts as 2^-14: 16 cuts of 2^-25 2^-14 are
        2^-11 of what code 1, 2^-24, makes of the largest other operand.  Scores: 2^-11 s max|q| for each of a
        group's two products.  Values: 2^-11 of the largest p s among each 16 tokens;
      * exponentials: 2^-18 of p (ex2.approx, and a fused exponent rounded at a magnitude below 64);
      * p to fp16, the same in numerator and sum: 2^-11 of p (fp16 models carry the rest: 2^-21), and
        half of 2^-24 below 2^-14 where the row's largest p is at least 2^8: 2^-33 of the sum per token;
      * p s to fp16: 2^-11 of p s n (2^-21); below 2^-14 half of 2^-24 times a code of 15, in units
        of at most R / 8, of a sum that is at least 2^8: 2^-32 R per token;
      * s and m in fp16 units of at most R / 8: exact but for 2^-25 of a unit: (15 + 1) 2^-28 R < 2^-23 R;
      * fp32 sums, truncated at each step by at most 2^-23 of the sum of their terms' magnitudes (n s + |m|):
        a warp meets a quarter of the tokens, 16 (fp16 models: 8) at a time, and up to eight more steps
        join the parts."""
    B, lq, hq, d = q.shape
    nb, hkv, bs, _ = k_rec.shape
    g = hq // hkv
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    rel = 2.0 ** -11 if bf16 else 2.0 ** -21
    for b in range(B):
        n = min(int(context_lens[b]), block_tables.shape[1] * bs)
        if n <= 0:
            continue
        pages = np.asarray(block_tables[b, :(n + bs - 1) // bs])
        inside = (pages >= 0) & (pages < nb)
        safe = np.where(inside, pages, 0)
        for h in range(hkv):
            kr, vr = (np.where(inside[:, None, None], c[safe, h], 0).astype(np.uint8).reshape(-1, RECORD)[:n]
                      for c in (k_rec, v_rec))
            (nk, sk, mk), (nv, sv, mv) = unpack(kr, bf16), unpack(vr, bf16)
            ks, vs = (nk * sk[..., None]).reshape(n, d), (nv * sv[..., None]).reshape(n, d)  # n s
            K, V = values(kr, bf16), values(vr, bf16)
            km, vm = np.repeat(np.abs(mk), GROUP, 1), np.repeat(np.abs(mv), GROUP, 1)
            for i in range(lq):
                m = n - lq + i + 1
                if m <= 0:
                    continue
                qi = q[b, i, h * g:(h + 1) * g]                                   # [g, d]
                s = (qi @ K[:m].T) * scale
                w = np.exp(s - s.max(-1, keepdims=True))
                w /= w.sum(-1, keepdims=True)
                o = w @ V[:m]
                dt = scale * (2.0 ** -20 * (np.abs(qi) @ (ks[:m] + km[:m]).T)
                              + 2.0 ** -24 * np.abs(qi).max(-1, keepdims=True) * ks[:m].sum(-1)
                              + 2.0 ** -10 * np.abs(qi).reshape(g, 4, GROUP).max(-1) @ sk[:m].T)
                we = w * (1.1 * dt + rel + 2.0 ** -18)
                R = np.repeat(np.maximum(16 * sv[:n], np.abs(mv[:n])).max(0), GROUP)
                steps = 8 + m / (64 if bf16 else 32)
                e = we @ np.abs(V[:m]) + we.sum(-1, keepdims=True) * np.abs(o)
                e += 2.0 ** -33 * (np.abs(V[:m]).sum(0) + m * np.abs(o))
                e += rel * (w @ vs[:m]) + (m * 2.0 ** -32 + 2.0 ** -23) * R
                e += steps * 2.0 ** -23 * (w @ (vs[:m] + vm[:m]))
                ps = np.pad(w[:, :, None] * sv[:m], ((0, 0), (0, -m % 16), (0, 0))).reshape(g, -1, 16, 4)
                e += 2.0 ** -11 * np.repeat(ps.max(2).sum(1), GROUP, -1)
                out[b, i, h * g:(h + 1) * g], bound[b, i, h * g:(h + 1) * g] = o, e
    return out, bound
