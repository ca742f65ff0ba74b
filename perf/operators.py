"""Cases, plain forms and 64-bit definitions of the 4-bit KV cache operators.

A 4-bit cache keeps one record of 80 bytes for every (token, kv head): 128 codes
of 4 bits, then a scale s and a minimum m in the model's type for each of the
four groups of 32 head dimensions; a value is s * code + m.  The cache of one
layer is uint8 [num_blocks, num_kv_heads, block_size, 80], once for the keys and
once for the values.  Three operators work on it:

  write   store the keys and values of new tokens at their slots, quantised as
          they are written, and read the same slots back;
  read    read the pages of whole sequences back as packed rows (what a prefill
          that continues a cached prefix attends to);
  attend  causal attention of one or a few query tokens per sequence over the
          pages of the cache (decode and speculative verification).

`own` selects the side: False computes each operator with elementary torch
operations, True calls the package.
"""
import math

import numpy as np
import torch

own = False

D = 128        # head dimension
GROUP = 32     # head dimensions that share a scale and a minimum
RECORD = 80    # bytes of one (token, kv head): 64 of codes, 16 of scales and minima
MIN_SCALE = 2.0 ** -100
_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _package():
    import __graft_entry__
    return __graft_entry__.load_package()


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one new token of each of 8 sequences: the write of a small decode step (latency)
        {"name": "write_decode_8", "op": "write", "type": "bf16", "tokens": 8, "run": 1, "hq": 16, "hkv": 8,
         "block": 256},
        # the write of the largest decode batch the engine captures; values are a view of the fused projection
        {"name": "write_decode_512", "op": "write", "type": "bf16", "tokens": 512, "run": 1, "hq": 32, "hkv": 8,
         "block": 256},
        # one rank of two: an odd number of prompt tokens in chunks of odd length, half precision
        {"name": "write_prompt_4133_fp16", "op": "write", "type": "fp16", "tokens": 4133, "run": 311, "hq": 8, "hkv": 4,
         "block": 128},
        # the largest prefill batch of the engine (max_num_batched_tokens)
        {"name": "write_prompt_16384", "op": "write", "type": "bf16", "tokens": 16384, "run": 400, "hq": 16, "hkv": 8,
         "block": 256},
        # the second chunk of one short prompt reads the first one back
        {"name": "read_one_700", "op": "read", "type": "bf16", "lens": "list:700", "seqs": 1, "hkv": 8, "block": 256,
         "shared": 0},
        # 64 sequences that share a cached prefix of 768 tokens, with suffixes of 64 to 512
        {"name": "read_prefix_64", "op": "read", "type": "bf16", "lens": "uniform:832:1280", "seqs": 64, "hkv": 8,
         "block": 256, "shared": 3},
        # chunked prefill of four long documents, half precision
        {"name": "read_long_4_fp16", "op": "read", "type": "fp16", "lens": "uniform:20000:32768", "seqs": 4, "hkv": 8,
         "block": 256, "shared": 0},
        # one short chat: the latency of a single sequence
        {"name": "attend_1_short", "op": "attend", "type": "bf16", "lens": "list:293", "seqs": 1, "lq": 1, "hq": 16,
         "hkv": 8, "block": 256},
        # eight short chats in a batch padded to 16 rows for a captured graph
        {"name": "attend_8_padded", "op": "attend", "type": "bf16", "lens": "uniform:100:1024", "seqs": 8, "pad": 8,
         "lq": 1, "hq": 16, "hkv": 8, "block": 256},
        # one long document: the work has to be split along the context
        {"name": "attend_1_long_fp16", "op": "attend", "type": "fp16", "lens": "list:32768", "seqs": 1, "lq": 1,
         "hq": 32, "hkv": 8, "block": 256},
        # verification of four draft tokens: five queries per sequence
        {"name": "attend_verify_128", "op": "attend", "type": "bf16", "lens": "uniform:512:4096", "seqs": 128, "lq": 5,
         "hq": 16, "hkv": 8, "block": 256},
        # the serving batch: 512 sequences of very different lengths
        {"name": "attend_512", "op": "attend", "type": "bf16", "lens": "lognormal:2048:0.5", "seqs": 512, "lq": 1,
         "hq": 32, "hkv": 8, "block": 256},
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], its logarithm uniform."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["write", "read", "attend", "attend"])
    case = {"op": op, "type": rng.choice(["bf16", "bf16", "fp16"]), "block": rng.choice([128, 256, 256, 512])}
    if op == "write":
        case["hq"], case["hkv"] = rng.choice([(16, 8), (32, 8), (8, 4), (16, 2), (4, 1), (16, 16)])
        case["tokens"] = _log(rng, 1, 16384 * 8 // max(8, case["hkv"]))
        case["run"] = rng.choice([1, _log(rng, 1, 700)])
    elif op == "read":
        case["hkv"] = rng.choice([8, 8, 4, 2, 1, 16])
        case["seqs"] = _log(rng, 1, 96)
        longest = _log(rng, 2, min(32768, 100000 * 8 // (case["seqs"] * max(8, case["hkv"]))))
        case["lens"] = f"uniform:{_log(rng, 1, longest)}:{longest}"
        case["shared"] = rng.choice([0, 0, 1, 2])
    else:
        case["hq"], case["hkv"] = rng.choice([(16, 8), (32, 8), (16, 16), (16, 4), (8, 1), (64, 8)])
        case["lq"] = rng.choice([1, 1, 1, rng.randint(2, 16 * case["hkv"] // case["hq"])])
        case["seqs"] = _log(rng, 1, 512)
        longest = _log(rng, case["lq"] + 1, min(32768, 1000000 * 8 // (case["seqs"] * max(8, case["hkv"]))))
        case["lens"] = f"uniform:{_log(rng, case['lq'], longest)}:{longest}"
        case["pad"] = rng.choice([0, 0, rng.randint(1, 16)])
    return case


def _lens(case):
    """Sequence lengths of a case: host integers, the same for every seed (the plan of a step)."""
    kind, *args = case["lens"].split(":")
    n = case["seqs"]
    rng = np.random.default_rng(n)
    if kind == "list":
        return [int(a) for a in args]
    if kind == "uniform":
        return [int(x) for x in rng.integers(int(args[0]), int(args[1]) + 1, size=n)]
    x = np.exp(rng.normal(math.log(float(args[0])), float(args[1]), size=n))
    return [int(v) for v in np.clip(np.rint(x), 1, 32768)]


# ---------------------------------------------------------------- the records
def _quantise(x):
    """Records uint8 [..., 80] of rows [..., 128] of 16-bit floats: within each group of 32,
    m = min, s = (max - min) / 15 rounded to the rows' type (0 below 2^-100), code = (x - m) / s
    rounded to the nearest integer (ties to even), at most 15.  A group whose max - min is not
    finite gets s = m = NaN and codes 0."""
    g = x.float().unflatten(-1, (D // GROUP, GROUP))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    span = hi - lo
    s = (span / 15).to(x.dtype).float()
    s = torch.where(s < MIN_SCALE, torch.zeros_like(s), s)
    code = torch.round((g - lo) / torch.where(s > 0, s, torch.ones_like(s))).clamp(0, 15)
    finite = torch.isfinite(span)
    code = torch.where((s > 0) & finite, code, torch.zeros_like(code)).to(torch.uint8)
    nan = torch.full_like(s, math.nan)
    par = torch.cat([torch.where(finite, s, nan), torch.where(finite, lo, nan)], -1).to(x.dtype)
    # Eight codes make a 32-bit word: the even dimensions in its low half, the odd ones in its high half.
    w = code.unflatten(-1, (4, 4, 2)).transpose(-1, -2)                 # [..., group, word, half, 4]
    byte = w[..., 0::2] | (w[..., 1::2] << 4)                            # [..., group, word, half, 2]
    return torch.cat([byte.flatten(-4), par.flatten(-2).contiguous().view(torch.uint8)], -1)


def _codes(rec):
    """Codes [..., 4, 32] of records."""
    b = rec[..., :64].unflatten(-1, (4, 4, 2, 2))
    n = torch.stack([b & 15, b >> 4], -1).flatten(-2)                    # [..., group, word, half, 4]
    return n.transpose(-1, -2).flatten(-3)


def _values(rec, dtype, work):
    """Rows [..., 128] of records in the type `work`."""
    par = rec[..., 64:].contiguous().view(dtype).unflatten(-1, (4, 2)).to(work)
    return (_codes(rec).to(work) * par[..., :1] + par[..., 1:]).flatten(-2)


# ----------------------------------------------------------------- the inputs
def _rows(gen, shape, dtype, spread):
    """Rows of a layer's keys or values: normal, each head dimension with its own spread."""
    x = torch.randn(shape, generator=gen, device="cuda")
    return (x * spread).to(dtype)


def _spread(gen, hkv, sigma):
    return torch.exp(torch.randn(hkv, D, generator=gen, device="cuda") * sigma)


def _cache(gen, blocks, case, dtype, sigma):
    """A cache of `blocks` pages full of quantised rows."""
    hkv, bs = case["hkv"], case["block"]
    cache = torch.empty(blocks, hkv, bs, RECORD, dtype=torch.uint8, device="cuda")
    spread = _spread(gen, hkv, sigma).unsqueeze(1)
    step = max(1, (1 << 26) // (hkv * bs * D))
    for i in range(0, blocks, step):
        n = min(step, blocks - i)
        cache[i:i + n] = _quantise(_rows(gen, (n, hkv, bs, D), dtype, spread))
    return cache


def _tables(gen, lens, case, shared=0):
    """Block tables of sequences whose first `shared` pages are the same; returns (table, number of pages)."""
    bs = case["block"]
    need = [-(-n // bs) for n in lens]
    own_pages = [max(0, n - shared) for n in need]
    pages = shared + sum(own_pages) + 2
    perm = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32).cpu().tolist()
    bt = np.full((len(lens), max(max(need), 1)), -1, np.int32)
    used = shared
    for b, n in enumerate(need):
        bt[b, :min(n, shared)] = perm[:min(n, shared)]
        if n > shared:
            bt[b, shared:n] = perm[used:used + n - shared]
            used += n - shared
    return torch.from_numpy(bt).cuda(), pages


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _TYPES[case["type"]]
    st = {"case": case, "dtype": dtype, "own": _package() if own else None}
    hkv, bs = case["hkv"], case["block"]
    if case["op"] == "write":
        n, run_len = case["tokens"], case["run"]
        seqs = -(-n // run_len)
        pages_each = -(-(run_len + bs - 1) // bs)
        blocks = seqs * pages_each + 1
        perm = torch.randperm(blocks, generator=gen, device="cuda").to(torch.int32).cpu().numpy()
        start = np.random.default_rng(seed).integers(0, bs, size=seqs)
        t = np.arange(n)
        pos = start[t // run_len] + t % run_len
        slots = perm[(t // run_len) * pages_each + pos // bs] * bs + pos % bs
        st["slots"] = torch.from_numpy(slots.astype(np.int32)).cuda()
        # keys come contiguous out of the rotary embedding, values as a view of the fused projection
        st["k"] = _rows(gen, (n, hkv, D), dtype, _spread(gen, hkv, 0.5))
        qkv = torch.randn(n, (case["hq"] + 2 * hkv) * D, generator=gen, device="cuda").to(dtype)
        st["v"] = qkv[:, -hkv * D:].view(n, hkv, D)
        st["kc"] = torch.zeros(blocks, hkv, bs, RECORD, dtype=torch.uint8, device="cuda")
        st["vc"] = torch.zeros_like(st["kc"])
        return st
    lens = _lens(case)
    st["lens"] = lens
    if case["op"] == "read":
        st["bt"], pages = _tables(gen, lens, case, case["shared"])
        st["cu"] = torch.tensor([0] + np.cumsum(lens).tolist(), dtype=torch.int32, device="cuda")
        st["total"] = sum(lens)
    else:
        lens = lens + [0] * case.get("pad", 0)  # rows of a captured batch that hold no sequence
        st["lens"] = lens
        st["bt"], pages = _tables(gen, lens, case)
        st["ctx"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        st["q"] = _rows(gen, (len(lens), case["lq"], case["hq"], D), dtype, 1.0)
        st["scale"] = D ** -0.5
    st["kc"] = _cache(gen, pages, case, dtype, 0.5)
    st["vc"] = _cache(gen, pages, case, dtype, 0.3)
    return st


# --------------------------------------------------------------- the operators
def run(st):
    case, dtype, pkg = st["case"], st["dtype"], st["own"]
    if case["op"] == "write":
        if pkg is not None:
            pkg.store_kvcache_q4(st["k"], st["v"], st["kc"], st["vc"], st["slots"])
            return pkg.load_kvcache_q4(st["kc"], st["vc"], st["slots"], dtype)
        return _plain_write(st, case["block"])
    if case["op"] == "read":
        if pkg is not None:
            return pkg.gather_kvcache_q4(st["kc"], st["vc"], st["cu"], st["bt"], st["total"], dtype)
        return _plain_read(st)
    if pkg is not None:
        return pkg.flash_attn_with_kvcache_q4(st["q"], st["kc"], st["vc"], cache_seqlens=st["ctx"],
                                              block_table=st["bt"], softmax_scale=st["scale"], causal=True)
    return _plain_attend(st)


def _plain_write(st, bs):
    slots = st["slots"].long()
    live = slots >= 0
    page, pos = slots[live] // bs, slots[live] % bs
    out = []
    for x, cache in ((st["k"], st["kc"]), (st["v"], st["vc"])):
        cache[page, :, pos] = _quantise(x[live])
        y = torch.zeros(x.shape, dtype=x.dtype, device=x.device)
        y[live] = _values(cache[page, :, pos], x.dtype, torch.float32).to(x.dtype)
        out.append(y)
    return tuple(out)


def _plain_read(st):
    out = []
    for cache in (st["kc"], st["vc"]):
        rows = []
        for b, n in enumerate(st["lens"]):
            pages = st["bt"][b, :-(-n // cache.shape[2])].long()
            rec = cache[pages].transpose(1, 2).flatten(0, 1)[:n]  # [n, Hkv, 80]
            rows.append(_values(rec, st["dtype"], torch.float32).to(st["dtype"]))
        out.append(torch.cat(rows))
    return tuple(out)


def _plain_attend(st):
    q, scale = st["q"], st["scale"]
    B, Lq, Hq, _ = q.shape
    hkv, bs = st["kc"].shape[1], st["kc"].shape[2]
    out = torch.zeros_like(q)
    for b, n in enumerate(st["lens"]):
        if n == 0:
            continue
        pages = st["bt"][b, :-(-n // bs)].long()
        k, v = (_values(c[pages].transpose(0, 1).flatten(1, 2)[:, :n], st["dtype"], torch.float32)
                for c in (st["kc"], st["vc"]))                                    # [Hkv, n, D]
        x = q[b].float().view(Lq, hkv, Hq // hkv, D).permute(1, 0, 2, 3)          # [Hkv, Lq, G, D]
        s = (x.flatten(1, 2) @ k.transpose(1, 2)).view(hkv, Lq, Hq // hkv, n) * scale
        if Lq > 1:  # query i of the last Lq tokens sees tokens up to n - Lq + i
            last = n - Lq + torch.arange(Lq, device=q.device)
            hidden = torch.arange(n, device=q.device)[None] > last[:, None]
            s = s.masked_fill(hidden[None, :, None], -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
        den = p.sum(-1, keepdim=True)
        o = (p.flatten(1, 2) @ v).view(hkv, Lq, Hq // hkv, D) / torch.where(den > 0, den, torch.ones_like(den))
        out[b] = o.permute(1, 0, 2, 3).reshape(Lq, Hq, D).to(q.dtype)
    return out


# ------------------------------------------------------------------- the work
def work(case):
    """Bytes and operations of one pass."""
    hkv = case["hkv"]
    if case["op"] == "write":
        n = case["tokens"]
        # keys and values in, records out, the values they stand for out, and the slots
        return {"bytes": n * hkv * (2 * 2 * D + 2 * RECORD + 2 * 2 * D) + 4 * n, "flops": n * hkv * 2 * D * 8}
    lens = _lens(case)
    tokens, pages = sum(lens), sum(-(-n // case["block"]) for n in lens)
    if case["op"] == "read":
        shared = case["shared"] * case["block"]
        distinct = tokens - sum(min(n, shared) for n in lens) + min(max(lens), shared)
        return {"bytes": distinct * hkv * 2 * RECORD + tokens * hkv * 2 * 2 * D + 4 * (pages + len(lens) + 1),
                "flops": tokens * hkv * 2 * D * 2}
    rows = len(lens) + case.get("pad", 0)
    io = rows * case["lq"] * case["hq"] * D * 2 * 2
    return {"bytes": tokens * hkv * 2 * RECORD + io + 4 * (pages + rows),
            "flops": tokens * case["lq"] * case["hq"] * D * 4}


# ------------------------------------------------------- the definition, 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "write":
        return tuple(_exact_round_trip(st[n], st["slots"]) for n in ("k", "v"))
    if case["op"] == "read":
        return tuple(torch.cat([_exact_rows(c, st["bt"][b], n, st["dtype"]) for b, n in enumerate(st["lens"]) if n])
                     for c in (st["kc"], st["vc"]))
    q = st["q"].double()
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    Lq, Hq = q.shape[1:3]
    for b, n in enumerate(st["lens"]):
        if n == 0:
            continue
        k = _exact_rows(st["kc"], st["bt"][b], n, st["dtype"])  # [n, Hkv, D]
        v = _exact_rows(st["vc"], st["bt"][b], n, st["dtype"])
        group = Hq // k.shape[1]
        for i in range(Lq):
            m = n - Lq + i + 1  # visible tokens
            if m <= 0:
                continue
            qi = q[b, i].view(k.shape[1], group, D)
            logits = torch.einsum("hgd,nhd->hgn", qi, k[:m]) * st["scale"]
            out[b, i] = torch.einsum("hgn,nhd->hgd", torch.softmax(logits, -1), v[:m]).reshape(Hq, D)
    return out


def _exact_round_trip(x, slots):
    """The value nearest to x on its group's grid of 16 levels."""
    y = x.double().reshape(*x.shape[:-1], -1, GROUP)
    low = y.min(-1, keepdim=True).values
    step = ((y.max(-1, keepdim=True).values - low) / 15).to(x.dtype).double()
    step = step * (step >= MIN_SCALE)
    level = torch.clamp(torch.round((y - low) / step), max=15)
    y = torch.where(step > 0, low + step * level, low.expand_as(y))
    return (y * (slots >= 0)[:, None, None, None]).reshape(x.shape)


def _exact_rows(cache, table, n, dtype):
    """Rows [n, Hkv, D] of a sequence, straight from the words of its records."""
    bs = cache.shape[2]
    t = torch.arange(n, device=cache.device)
    rec = cache[table.long()[t // bs], :, t % bs]
    words = rec[..., :64].contiguous().view(torch.int32)                 # 16 words of 8 codes
    par = rec[..., 64:].contiguous().view(torch.int16).view(dtype).double()
    d = torch.arange(D, device=cache.device)
    shift = (d % 8) // 2 * 4 + (d % 2) * 16
    level = (words[..., d // 8] >> shift.to(torch.int32)) & 15
    return par[..., 2 * (d // GROUP)] * level.double() + par[..., 2 * (d // GROUP) + 1]
