"""Performance cases of the operators on a cache held in 4 or 8 bits: its
writer and reader, attention with score forms (capped scores, a bias by
distance, a window, a prefix that stays visible), the accumulation of
attention weights per cached token, and the eviction by those weights.

Every case is one pass of one operator on a synthetic paged cache in GPU
memory.  With `own` true run() calls the library; with it false it computes
the same in elementary torch operations in fp32.  Keys, values and new rows
are N(0,1) (a fraction of the tokens eight times that where the case has
outliers), queries N(0,1) rounded to their type, page tables random
permutations of the pool.

A 4-bit block is 32 consecutive dims of one token and kv head: bf16 minimum
mn, bf16 step sc = (max - mn) / 15, code = clamp(rint((x - mn) / sc), 0, 15),
value code * sc + mn.  Row byte n * G + g (G = dim / 32) holds dims 32g + 2n
(low nibble) and 32g + 2n + 1; parameter word g is sc << 16 | mn.
"""
import math
import random

import numpy as np
import torch

own = False

DEVICE = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---- cases -------------------------------------------------------------------

def _attend(name, bits, batch, rows, heads, page, shortest, longest, kind, *, cap=0.0, window=0, slopes=False, prefix=0,
            outliers=0.0, length_seed=0x4B56423, op="attend", fresh=0):
    q_heads, kv_heads, dim = heads
    case = {"op": op, "bits": bits, "batch": batch, "rows": rows, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim,
            "page": page, "shortest": shortest, "longest": longest, "length_seed": length_seed, "type": kind, "cap": cap,
            "window": window, "slopes": slopes, "prefix": prefix, "outliers": outliers}
    if op == "weights":
        case["fresh"] = fresh
    return dict(case, name=name) if name else case


def _write(name, tokens, kv_heads, dim, page, kind, layout, pad):
    case = {"op": "write", "tokens": tokens, "kv_heads": kv_heads, "dim": dim, "page": page, "type": kind,
            "layout": layout, "pad": pad}
    return dict(case, name=name) if name else case


def _evict(name, bits, batch, kv_heads, dim, page, shortest, longest, keep, sink, recent, *, length_seed=0x4B56423):
    case = {"op": "evict", "bits": bits, "batch": batch, "kv_heads": kv_heads, "dim": dim, "page": page,
            "shortest": shortest, "longest": longest, "length_seed": length_seed, "keep": keep, "sink": sink,
            "recent": recent}
    return dict(case, name=name) if name else case


def listed():
    return [
        # One decode step of 64 sequences written to the 4-bit cache out of a fused QKV buffer (and read back as values).
        _write("write_step_64", 64, 8, 128, 16, "bf16", "step", 0),
        # A long prompt's prefill written to the 4-bit cache, its last chunk padded.
        _write("write_prefill_16k", 16389, 8, 128, 64, "f16", "prefill", 5),
        # A short chat turn on a small model: launch and latency are all there is.
        _attend("attend4_short_512", 4, 1, 1, (8, 2, 64), 16, 512, 512, "f16"),
        # One long sequence, the geometry of the benchmark's call.
        _attend("attend4_long_64k", 4, 1, 1, (32, 8, 128), 64, 65536, 65536, "bf16"),
        # Ragged serving batch over a shared pool.
        _attend("attend4_ragged_16", 4, 16, 1, (32, 8, 128), 64, 1024, 32768, "bf16"),
        # The largest: four 128K-token contexts, wide GQA, outlier tokens.
        _attend("attend4_batch_128k", 4, 4, 1, (64, 8, 128), 64, 131072, 131072, "f16", outliers=0.01),
        # Drafted tokens of a model with a bias by distance, dim 256, 32-token pages, fp32 in and out.
        _attend("attend4_distance_rows8", 4, 2, 8, (24, 4, 256), 32, 4001, 8191, "f32", slopes=True),
        # An int8 cache under capped scores in a sliding window with the first tokens kept visible.
        _attend("attend8_capped_window", 8, 32, 1, (16, 8, 256), 64, 500, 16384, "bf16", cap=50.0, window=4096, prefix=4),
        # Attention weights of a decode step added to what the tokens have, ragged batch.
        _attend("weights4_ragged_16", 4, 16, 1, (32, 8, 128), 64, 1024, 32768, "bf16", op="weights", fresh=1),
        # The first weights after a prompt, by its last rows' queries, int8 cache, capped scores.
        _attend("weights8_prompt", 8, 2, 16, (8, 2, 64), 16, 3001, 7000, "f16", cap=30.0, op="weights", fresh=1 << 20),
        # A ragged batch cut down to 4,096 tokens a sequence.
        _evict("evict4_ragged_16", 4, 16, 8, 128, 64, 1024, 32768, 4096, 4, 512),
        # Two short conversations on an int8 cache, odd sizes.
        _evict("evict8_short", 8, 2, 2, 64, 16, 700, 1999, 501, 1, 64),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _fit(rng, lo, hi, unit, most):
    """A size of [lo, hi], spread over its logarithm, whose cost at `unit` each is at most `most`."""
    return _log_int(rng, lo, max(lo, min(hi, int(most // unit))))


def draw(rng):
    heads = rng.choice([(8, 2, 64), (32, 8, 128), (16, 4, 128), (8, 8, 128), (64, 8, 128), (24, 4, 256), (16, 8, 256)])
    page = rng.choice([8, 16, 32, 48, 64, 128])
    kind = rng.randrange(8)
    bits = rng.choice([4, 4, 8])
    seed = rng.randrange(1 << 20)
    row = heads[1] * heads[2]  # elements of a token's K
    if kind == 0:
        layout = rng.choice(["step", "prefill"])
        tokens = _fit(rng, 1, 16384 if layout == "prefill" else 1024, row, 16384 * 1024)
        return _write("", tokens, heads[1], heads[2], page, rng.choice(list(TYPES)), layout,
                      rng.choice([0, min(tokens - 1, rng.randrange(8))]))
    if kind == 1:
        longest = _log_int(rng, 64, 32768)
        keep = _fit(rng, max(1, longest // 16), longest, row, 65536 * 1024)
        sink = rng.randrange(min(8, keep))
        batch = rng.randint(1, max(1, min(16, 65536 * 1024 // (keep * row))))
        return _evict("", bits, batch, heads[1], heads[2], page, max(1, longest // 16), longest, keep, sink,
                      rng.randrange(keep - sink), length_seed=seed)
    # at most the largest listed call: its bytes, and its products of rows and tokens
    rows = rng.choice([1, 1, 4, 16] if kind < 4 else [1, 1, 1, 3, 8])
    unit = max(2 * heads[1] * _token_bytes(bits, heads[2]), 1280 * rows)
    longest = _fit(rng, 1, 131072, unit, 524288 * 2560)
    batch = _fit(rng, 1, 32, unit * longest, 524288 * 2560)
    forms = {"cap": rng.choice([0.0, 0.0, 20.0, 50.0]), "slopes": rng.random() < 0.25,
             "window": rng.choice([0, 0, _log_int(rng, 1, longest)]), "prefix": rng.choice([0, 0, rng.randint(1, 64)])}
    if kind < 4:
        return _attend("", bits, batch, rows, heads, page, max(1, longest // 16), longest, rng.choice(list(TYPES)),
                       length_seed=seed, op="weights", fresh=rng.choice([0, 1, 1 << 20]), **forms)
    if kind < 6:
        forms = {}
    return _attend("", bits, batch, rows, heads, page, max(1, longest // 16), longest, rng.choice(list(TYPES)),
                   outliers=rng.choice([0.0, 0.01]), length_seed=seed, **forms)


def _lengths(case):
    """Tokens of each sequence, the longest among them (wherever the seed puts it)."""
    rng = np.random.default_rng(case["length_seed"])
    lengths = rng.integers(case["shortest"], case["longest"], size=case["batch"], endpoint=True)
    lengths[int(rng.integers(case["batch"]))] = case["longest"]
    return lengths.astype(np.int64)


def _token_bytes(bits, dim):
    """Bytes of one token's K (or V) row of one kv head with its scales."""
    return dim // 2 + dim // 32 * 4 if bits == 4 else dim + 4


def _seen(case):
    """(cached tokens that some row of the sequence sees, row-token pairs) over the batch."""
    tokens = pairs = 0
    R, W, pre = case["rows"], case["window"], case["prefix"]
    for T in _lengths(case):
        T, per, low = int(T), 0, None
        for r in range(R):
            last = T - R + r
            first = 0 if W == 0 else max(0, last - W + 1)
            per += max(0, last + 1 - first) + (min(pre, T) - max(0, min(pre, T, last + 1) - first) if pre else 0)
            low = first if low is None else min(low, first)
        tokens += (T - low) + min(pre, low, T)
        pairs += per
    return tokens, pairs


def work(case):
    if case["op"] == "write":
        t, h, d = case["tokens"] - case["pad"], case["kv_heads"], case["dim"]
        src = 4 if case["type"] == "f32" else 2
        # rows in, rows of the cache out and in again, values out (padding writes zeros)
        return {"bytes": 2 * h * (t * d * src + 2 * t * _token_bytes(4, d) + case["tokens"] * d * 4), "flops": t * h * d * 12}
    if case["op"] == "evict":
        T, h, d = _lengths(case), case["kv_heads"], case["dim"]
        kept = int(np.minimum(T, case["keep"]).sum())
        row = 2 * h * _token_bytes(case["bits"], d) + 4 * h + 8
        return {"bytes": int(T.sum()) * 4 * h + kept * (3 * row + 4) + case["batch"] * case["keep"] * 2 * h * d * 2,
                "flops": int(T.sum()) * h}
    tokens, pairs = _seen(case)
    h, d, rows = case["kv_heads"], case["dim"], case["batch"] * case["rows"]
    el = 4 if case["type"] == "f32" else 2
    q = rows * case["q_heads"] * (d * el + 8)
    if case["op"] == "weights":
        every = int(_lengths(case).sum()) * h * 4  # tokens that no row sees are set or kept too
        return {"bytes": tokens * h * _token_bytes(case["bits"], d) + q + 2 * every, "flops": 2 * pairs * case["q_heads"] * d}
    return {"bytes": 2 * tokens * h * _token_bytes(case["bits"], d) + q + rows * case["q_heads"] * d * el,
            "flops": 4 * pairs * case["q_heads"] * d}


# ---- the 4-bit rows ------------------------------------------------------------

def _encode4(x):
    """Rows [..., dim] (fp32) -> packed codes uint8 [..., dim / 2], parameter words int32 [..., dim / 32]."""
    G = x.shape[-1] // 32
    b = x.reshape(*x.shape[:-1], G, 32)
    lo, hi = b.amin(-1), b.amax(-1)
    mn = lo.to(torch.bfloat16).float()
    fifteen = torch.full((), 15.0, device=x.device)  # a tensor: torch divides by a plain number as a product
    sc = (torch.clamp(hi - mn, min=0.0) / fifteen).to(torch.bfloat16).float()
    bad = ~(torch.isfinite(b).all(-1) & torch.isfinite(mn) & torch.isfinite(sc))
    flat = bad | (sc == 0)
    c = torch.clamp(torch.round((b - mn[..., None]) / torch.where(flat, torch.ones_like(sc), sc)[..., None]), 0, 15)
    c = torch.where(flat[..., None], torch.zeros_like(c), c).to(torch.uint8).reshape(*x.shape[:-1], G, 16, 2)
    nan = torch.full_like(sc, float("nan"))
    sc, mn = torch.where(bad, nan, sc), torch.where(bad, nan, mn)
    words = (sc.to(torch.bfloat16).view(torch.int16).to(torch.int32) << 16) | \
        (mn.to(torch.bfloat16).view(torch.int16).to(torch.int32) & 0xffff)
    packed = (c[..., 0] | (c[..., 1] << 4)).transpose(-1, -2)
    return packed.reshape(*x.shape[:-1], 16 * G).contiguous(), words.contiguous()


def _decode4(packed, words):
    """The values that packed rows stand for, fp32 [..., dim]."""
    G = words.shape[-1]
    b = packed.reshape(*packed.shape[:-1], 16, G).transpose(-1, -2)
    c = torch.stack((b & 15, b >> 4), -1).reshape(*packed.shape[:-1], G, 32).float()
    sc = (words & -65536).view(torch.float32)
    mn = (words << 16).view(torch.float32)
    return (c * sc[..., None] + mn[..., None]).reshape(*packed.shape[:-1], 32 * G)


def _encode8(x):
    absmax = x.abs().amax(-1)
    sc = torch.where(absmax == 0, torch.ones_like(absmax), absmax / 127.0)
    return torch.clamp(torch.round(x / sc[..., None]), -127, 127).to(torch.int8), sc


# ---- inputs ----------------------------------------------------------------------

def _pool(g, bits, pages, kv_heads, page, dim, outliers):
    """A filled page pool: k, v, k_scales, v_scales in the library's layouts."""
    out = {}
    for name in ("k", "v"):
        codes, scales = [], []
        step = max(1, (1 << 26) // (kv_heads * page * dim))
        for p0 in range(0, pages, step):
            n = min(step, pages - p0)
            x = torch.randn((n, kv_heads, page, dim), generator=g, device=DEVICE)
            if outliers:
                hit = torch.rand((n, 1, page, 1), generator=g, device=DEVICE) < outliers
                x = torch.where(hit, x * 8.0, x)
            c, s = (_encode4 if bits == 4 else _encode8)(x)
            codes.append(c.transpose(2, 3).contiguous() if bits == 8 and name == "v" else c)
            scales.append(s)
        out[name], out[name + "_scales"] = torch.cat(codes), torch.cat(scales)
    return out


def _ragged(g, lengths, page, spare):
    """Token offsets, page lists out of a shuffled pool (and `spare` pages more of it), flat (sequence, token) lists."""
    npages = -(-lengths // page)
    pool = int(npages.sum()) + spare
    table = torch.randperm(pool, generator=g, device=DEVICE).to(torch.int32)
    starts = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    offsets = np.concatenate([[0], np.cumsum(npages)[:-1]]).astype(np.int32)
    seq = np.repeat(np.arange(len(lengths)), lengths)
    at = np.arange(int(lengths.sum())) - np.repeat(starts[:-1].astype(np.int64), lengths)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(DEVICE)  # noqa: E731
    return {"pages": pool, "table": table[:pool - spare].contiguous(), "spare": table[pool - spare:].contiguous(),
            "starts": dev(starts), "offsets": dev(offsets), "seq": dev(seq), "at": dev(at), "kpos": dev(at.astype(np.int64)),
            "lengths": dev(lengths), "max_tokens": int(lengths.max())}


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    s = {"case": dict(case)}
    if case["op"] == "write":
        tokens, h, d, page = case["tokens"], case["kv_heads"], case["dim"], case["page"]
        kind = TYPES[case["type"]]
        pages = -(-tokens // page) + 2 if case["layout"] == "prefill" else max(4, tokens * 2)
        if case["layout"] == "prefill":  # whole pages in random order, filled in turn
            order = torch.randperm(pages, generator=g, device=DEVICE)
            t = torch.arange(tokens, device=DEVICE)
            slots = order[t // page] * page + t % page
        else:  # one slot of a page of each sequence
            order = torch.randperm(pages, generator=g, device=DEVICE)[torch.arange(tokens, device=DEVICE) % pages]
            slots = order * page + torch.randint(0, page, (tokens,), generator=g, device=DEVICE)
        if case["pad"]:
            slots[tokens - case["pad"]:] = pages * page
        # K and V as columns of one buffer, behind two query columns, as a fused projection writes them
        s["qkv"] = torch.randn((tokens, 4, h * d), generator=g, device=DEVICE).to(kind)
        s["slots"], s["pages"] = slots.to(torch.int32), pages
        s["k"], s["v"] = (torch.zeros((pages, h, page, d // 2), dtype=torch.uint8, device=DEVICE) for _ in range(2))
        s["k_scales"], s["v_scales"] = (torch.zeros((pages, h, page, d // 32), dtype=torch.int32, device=DEVICE) for _ in range(2))
        return s
    lengths = _lengths(case)
    batch, h, d, page = case["batch"], case["kv_heads"], case["dim"], case["page"]
    if case["op"] == "evict":
        kept = np.minimum(lengths, case["keep"])
        npages = -(-kept // page)
        s.update(_ragged(g, lengths, page, int(npages.sum())))
        s.update(_pool(g, case["bits"], s["pages"], h, page, d, 0.0))
        # weights as decode steps leave them: most tokens little, a few much
        s["weights"] = torch.empty((s["pages"], h, page), device=DEVICE).exponential_(1.0, generator=g).pow_(3.0)
        doff = np.concatenate([[0], np.cumsum(npages)[:-1]]).astype(np.int32)
        s["dst_offsets"] = torch.from_numpy(doff).to(DEVICE)
        seq = np.repeat(np.arange(batch), kept)
        at = np.arange(int(kept.sum())) - np.repeat(np.cumsum(kept) - kept, kept)
        s["to_seq"], s["to_at"] = (torch.from_numpy(a).to(DEVICE) for a in (seq, at))
        s["kept_counts"] = torch.from_numpy(kept).to(DEVICE)
        slots = torch.full((batch * case["keep"],), s["pages"] * page, dtype=torch.int64, device=DEVICE)
        dpage = s["spare"].long()[s["dst_offsets"].long()[s["to_seq"]] + s["to_at"] // page]
        slots[s["to_seq"] * case["keep"] + s["to_at"]] = dpage * page + s["to_at"] % page
        s["to_slots"] = slots.to(torch.int32)
        return s
    s.update(_ragged(g, lengths, page, 0))
    s.update(_pool(g, case["bits"], s["pages"], h, page, d, case["outliers"]))
    R, H = case["rows"], case["q_heads"]
    s["q"] = torch.randn((batch, R, H, d), generator=g, device=DEVICE).to(torch.float16).to(TYPES[case["type"]])
    s["qpos"] = s["lengths"][:, None] - R + torch.arange(R, device=DEVICE)
    s["slopes"] = torch.exp2(-8.0 * torch.arange(1, H + 1, device=DEVICE) / H) if case["slopes"] else None
    s["prefix"] = torch.full((batch,), case["prefix"], dtype=torch.int64, device=DEVICE) if case["prefix"] else None
    if case["op"] == "weights":
        scores = _scores(s)
        s["m"] = scores.amax(-1)
        s["l"] = torch.exp(scores - torch.where(torch.isfinite(s["m"]), s["m"], torch.zeros_like(s["m"]))[..., None]).sum(-1)
        s["m"], s["l"] = (x.reshape(-1) for x in (s["m"], s["l"]))
        del scores
        s["weights"] = torch.rand((s["pages"], h, page), generator=g, device=DEVICE)
    return s


# ---- plain forms -------------------------------------------------------------------

def _cached(s, name):
    """K or V of every (sequence, token) of the batch, padded to the longest: fp32 [batch, kv_heads, tokens, dim]."""
    case = s["case"]
    t = torch.arange(s["max_tokens"], device=DEVICE)
    inside = t < s["lengths"][:, None]
    at = s["offsets"].long()[:, None] + torch.where(inside, t // case["page"], torch.zeros_like(t))
    page, slot = s["table"].long()[at], (t % case["page"]).expand(at.shape)
    codes, scales = s[name], s[name + "_scales"][page, :, slot]
    if case["bits"] == 4:
        x = _decode4(codes[page, :, slot], scales)
    else:
        x = (codes[page, :, :, slot] if name == "v" else codes[page, :, slot]).float() * scales[..., None]
    return x.transpose(1, 2).contiguous()


def _scores(s):
    """Masked scores fp32 [batch, rows, q_heads, tokens] in the order of the outputs."""
    case = s["case"]
    B, R, H, d, h = case["batch"], case["rows"], case["q_heads"], case["dim"], case["kv_heads"]
    q = s["q"].float().reshape(B, R, h, H // h, d).permute(0, 2, 1, 3, 4).reshape(B, h, R * (H // h), d)
    x = torch.matmul(q, _cached(s, "k").transpose(-1, -2)) * (1.0 / math.sqrt(d))
    x = x.reshape(B, h, R, H // h, -1).permute(0, 2, 1, 3, 4).reshape(B, R, H, -1)
    if case["cap"]:
        x = case["cap"] * torch.tanh(x / case["cap"])
    kpos = torch.arange(s["max_tokens"], device=DEVICE)
    far = (kpos - s["qpos"][..., None])[:, :, None, :]
    if s["slopes"] is not None:
        x = x + s["slopes"][:, None] * far.float()
    seen = far <= 0
    if case["window"]:
        seen = seen & (-far < case["window"])
    if s["prefix"] is not None:
        seen = seen | (kpos < s["prefix"][:, None])[:, None, None, :]
    seen = seen & (kpos < s["lengths"][:, None])[:, None, None, :]
    return torch.where(seen, x, torch.full_like(x, -math.inf))


def _plain_attend(s):
    case = s["case"]
    B, R, H, d, h = case["batch"], case["rows"], case["q_heads"], case["dim"], case["kv_heads"]
    x = _scores(s)
    m = x.amax(-1)
    p = torch.exp(x - torch.where(torch.isfinite(m), m, torch.zeros_like(m))[..., None])
    l = p.sum(-1)
    p = p.reshape(B, R, h, H // h, -1).permute(0, 2, 1, 3, 4).reshape(B, h, R * (H // h), -1)
    n = torch.matmul(p, _cached(s, "v")).reshape(B, h, R, H // h, d).permute(0, 2, 1, 3, 4).reshape(B, R, H, d)
    out = torch.where(l[..., None] > 0, n / l[..., None], torch.zeros_like(n))
    return {"out": out.to(TYPES[case["type"]]), "m": m, "l": l}


def _plain_weights(s):
    case = s["case"]
    B, R, H, h = case["batch"], case["rows"], case["q_heads"], case["kv_heads"]
    m, l = (s[x].reshape(B, R, H, 1) for x in ("m", "l"))
    p = torch.exp(_scores(s) - torch.where(l > 0, m, torch.zeros_like(m))) / torch.where(l > 0, l, torch.ones_like(l))
    mass = p.reshape(B, R, h, H // h, -1).sum((1, 3)).transpose(1, 2)[s["seq"], s["at"]]
    page = s["table"].long()[s["offsets"].long()[s["seq"]] + s["at"] // case["page"]]
    slot = s["at"] % case["page"]
    old = (s["at"] < s["lengths"][s["seq"]] - case["fresh"])[:, None]
    w = s["weights"]
    w[page, :, slot] = torch.where(old, w[page, :, slot], torch.zeros_like(mass)) + mass
    return w


def _plain_write(s):
    case = s["case"]
    tokens, h, d, page = case["tokens"], case["kv_heads"], case["dim"], case["page"]
    n = tokens - case["pad"]
    slots = s["slots"].long()[:n]
    got = {}
    for i, name in ((2, "k"), (3, "v")):
        codes, words = _encode4(s["qkv"][:n, i].float().reshape(n, h, d))
        s[name][slots // page, :, slots % page] = codes
        s[name + "_scales"][slots // page, :, slots % page] = words
        x = _decode4(s[name][slots // page, :, slots % page], s[name + "_scales"][slots // page, :, slots % page])
        got[name] = torch.cat((x, x.new_zeros((tokens - n, h, d))))
    return got


def _plain_evict(s):
    case = s["case"]
    keep, page, batch = case["keep"], case["page"], case["batch"]
    T, n = s["max_tokens"], s["kept_counts"]
    t = torch.arange(T, device=DEVICE)
    inside = t < s["lengths"][:, None]
    pid = s["table"].long()[s["offsets"].long()[:, None] + torch.where(inside, t // page, torch.zeros_like(t))]
    key = s["weights"][pid, :, (t % page).expand(pid.shape)].double().sum(-1).float()
    always = (t < case["sink"]) | (t >= s["lengths"][:, None] - case["recent"])
    key = torch.where(always, torch.full_like(key, math.inf), key)
    key = torch.where(inside, key, torch.full_like(key, -math.inf))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    stays = torch.zeros_like(inside).scatter(-1, order, t.expand(order.shape) < n[:, None])
    ids = torch.where(stays, t, torch.full_like(t, T)).sort(-1).values
    at = torch.arange(keep, device=DEVICE)
    ids = torch.where(at < n[:, None], ids[:, torch.clamp(at, max=T - 1)], torch.full_like(at, -1))
    starts = torch.cat((n.new_zeros(1), n.cumsum(0)))
    b, j = s["to_seq"], s["to_at"]
    src = ids[b, j]
    sp, ss = s["table"].long()[s["offsets"].long()[b] + src // page], src % page
    dp, ds = s["spare"].long()[s["dst_offsets"].long()[b] + j // page], j % page
    got = {}
    for name in ("k", "v"):
        c, w = s[name], s[name + "_scales"]
        w[dp, :, ds] = w[sp, :, ss]
        if case["bits"] == 4:
            c[dp, :, ds] = c[sp, :, ss]
            x = _decode4(c[dp, :, ds], w[dp, :, ds])
        elif name == "k":
            c[dp, :, ds] = c[sp, :, ss]
            x = c[dp, :, ds].float() * w[dp, :, ds][..., None]
        else:
            c[dp, :, :, ds] = c[sp, :, :, ss]
            x = c[dp, :, :, ds].float() * w[dp, :, ds][..., None]
        got[name] = torch.zeros((batch * keep, *x.shape[1:]), dtype=torch.bfloat16, device=DEVICE)
        got[name][b * keep + j] = x.to(torch.bfloat16)
    s["weights"][dp, :, ds] = s["weights"][sp, :, ss]
    positions = torch.full((batch * keep,), -1, dtype=torch.int64, device=DEVICE)
    positions[starts[b] + j] = s["kpos"][s["starts"].long()[b] + src]
    return {"kept": ids.to(torch.int32), "starts": starts.to(torch.int32), "positions": positions,
            "weights": s["weights"], **got}


# ---- the library's calls -------------------------------------------------------------

def _plan(s):
    """Descriptors, workspaces and output buffers of a state, as a serving loop holds them."""
    import kvbridge_amd as kvb

    case = s["case"]
    source = {"f32": kvb.KVB_SRC_F32, "f16": kvb.KVB_SRC_F16, "bf16": kvb.KVB_SRC_BF16}
    empty = lambda *shape, dtype=torch.float32: torch.empty(shape, dtype=dtype, device=DEVICE)  # noqa: E731
    h, d, page = case["kv_heads"], case["dim"], case["page"]
    cache = [s[x] for x in ("k", "v", "k_scales", "v_scales")]
    if case["op"] == "write":
        tokens = case["tokens"]
        k, v = s["qkv"][:, 2], s["qkv"][:, 3]
        shape = kvb.append_shape(tokens, h, d, page, s["pages"], source[case["type"]], k.stride(0), v.stride(0))
        back = kvb.read_shape(tokens, h, d, page, s["pages"], 4, kvb.KVB_OUT_F32)
        got = {"k": empty(tokens, h, d), "v": empty(tokens, h, d)}

        def call():
            kvb.append_kv_i4(shape, k, v, s["slots"], *cache)
            kvb.read_kv(back, s["slots"], *cache, got["k"], got["v"])
            return got

        return call
    batch = case["batch"]
    total, entries = s["kpos"].numel(), s["table"].numel()
    if case["op"] == "evict":
        keep = case["keep"]
        shape = kvb.make_evict_shape(batch, h, d, page, s["pages"], s["max_tokens"], total, entries, s["spare"].numel(),
                                     keep, case["sink"], case["recent"], case["bits"])
        scratch = empty(kvb.evict_scratch_elements(shape), dtype=torch.int32)
        got = {"kept": torch.full((batch, keep), -1, dtype=torch.int32, device=DEVICE),
               "starts": empty(batch + 1, dtype=torch.int32),
               "positions": torch.full((batch * keep,), -1, dtype=torch.int64, device=DEVICE), "weights": s["weights"],
               "k": empty(batch * keep, h, d, dtype=torch.bfloat16), "v": empty(batch * keep, h, d, dtype=torch.bfloat16)}
        source_io = kvb.evict_input(s["starts"], s["offsets"], s["table"], s["kpos"])
        moved = kvb.evict_cache(*cache, s["weights"], s["dst_offsets"], s["spare"], got["positions"])
        back = kvb.read_shape(batch * keep, h, d, page, s["pages"], case["bits"], kvb.KVB_OUT_BF16)

        def call():
            kvb.evict_select(shape, source_io, s["weights"], scratch, got["kept"], got["starts"])
            kvb.evict_move(shape, source_io, moved, got["kept"], got["starts"])
            kvb.read_kv(back, s["to_slots"], *cache, got["k"], got["v"])
            return got

        return call
    R, H = case["rows"], case["q_heads"]
    shape = kvb.make_scored_shape(batch, R, H, h, d, page, s["pages"], s["max_tokens"], total, entries, 1.0 / math.sqrt(d),
                                  kv_bits=case["bits"], q_type=source[case["type"]], window=case["window"], cap=case["cap"])
    given = kvb.scored_input(s["q"], s["qpos"], s["starts"], s["offsets"], s["kpos"], s["table"], *cache, s["slopes"],
                             s["prefix"])
    if case["op"] == "weights":
        def call():
            kvb.accumulate_weights(shape, given, s["m"], s["l"], s["weights"], case["fresh"])
            return s["weights"]

        return call
    result = {"f32": kvb.KVB_OUT_F32, "f16": kvb.KVB_OUT_F16, "bf16": kvb.KVB_OUT_BF16}[case["type"]]
    scratch = empty(kvb.scored_scratch_elements(shape))
    counters = torch.zeros(kvb.scored_counter_elements(shape), dtype=torch.int32, device=DEVICE)
    got = {"out": empty(batch, R, H, d, dtype=TYPES[case["type"]]), "m": empty(batch, R, H), "l": empty(batch, R, H)}

    def call():
        kvb.decode_attention_scored(shape, given, scratch, got["m"], got["l"], got["out"], result, counters)
        return got

    return call


def run(state):
    if own:
        if "call" not in state:
            state["call"] = _plan(state)
        return state["call"]()
    return {"write": _plain_write, "attend": _plain_attend, "weights": _plain_weights,
            "evict": _plain_evict}[state["case"]["op"]](state)


# ---- in 64 bits ------------------------------------------------------------------------

def _value4(packed, words):
    """Values of 4-bit rows in fp64, by the definition: one group of dims after the other."""
    G = words.shape[-1]
    raw = words.to(torch.int64) & 0xffffffff
    step = (raw >> 16 << 16).to(torch.int32).view(torch.float32).double()
    least = ((raw & 0xffff) << 16).to(torch.int32).view(torch.float32).double()
    x = torch.empty((*packed.shape[:-1], 32 * G), dtype=torch.float64, device=packed.device)
    for g in range(G):
        byte = packed[..., g::G].to(torch.int64)
        x[..., 32 * g:32 * g + 32:2] = (byte % 16) * step[..., g:g + 1] + least[..., g:g + 1]
        x[..., 32 * g + 1:32 * g + 32:2] = (byte // 16) * step[..., g:g + 1] + least[..., g:g + 1]
    return x


def _rows_of(s, b, name):
    """Cached K or V of sequence b in fp64, [tokens, kv_heads, dim]."""
    case = s["case"]
    T, P = int(s["lengths"][b]), case["page"]
    first = int(s["offsets"][b])
    pages = s["table"][first:first + -(-T // P)].long()
    codes, scales = s[name][pages], s[name + "_scales"][pages]
    if case["bits"] == 8:
        codes = codes.transpose(2, 3) if name == "v" else codes
        x = codes.double() * scales.double()[..., None]
    else:
        x = _value4(codes, scales)
    return x.transpose(1, 2).reshape(-1, case["kv_heads"], case["dim"])[:T]


def _scores_of(s, b):
    """Scores of sequence b in fp64, [rows, q_heads, tokens], -inf where masked."""
    case = s["case"]
    K = _rows_of(s, b, "k")
    group = case["q_heads"] // case["kv_heads"]
    q = s["q"][b].double()
    x = torch.stack([q[:, i] @ K[:, i // group].t() for i in range(case["q_heads"])], 1) / math.sqrt(case["dim"])
    if case["cap"]:
        x = torch.tanh(x / case["cap"]) * case["cap"]
    kpos = torch.arange(x.shape[-1], device=x.device)
    qpos = s["qpos"][b][:, None, None]
    if s["slopes"] is not None:
        x = x + s["slopes"].double()[:, None] * (kpos - qpos).double()
    hidden = kpos > qpos
    if case["window"]:
        hidden = hidden | (qpos - kpos >= case["window"])
    if case["prefix"]:
        hidden = hidden & (kpos >= case["prefix"])
    return x.masked_fill(hidden, -math.inf)


def _bf16(x):
    """fp32 array rounded to bfloat16, half to even, as fp32."""
    u = x.astype(np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7fff + ((u >> 16) & 1)) >> 16 << 16).astype(np.uint32).view(np.float32)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "write":
        # the definition's own fp32 steps (IEEE on the host) give the codes; the values they stand for in fp64
        h, d = case["kv_heads"], case["dim"]
        got = {}
        for i, name in ((2, "k"), (3, "v")):
            x = s["qkv"][:, i].float().cpu().numpy().reshape(-1, h, d // 32, 32)
            least = _bf16(x.min(-1, keepdims=True))
            step = _bf16(np.maximum(x.max(-1, keepdims=True) - least, np.float32(0)) / np.float32(15))
            code = np.clip(np.rint((x - least) / np.where(step > 0, step, np.float32(1))), 0, 15) * (step > 0)
            value = code.astype(np.float64) * step + least
            value[case["tokens"] - case["pad"]:] = 0.0
            got[name] = value.reshape(-1, h, d)
        return got
    if case["op"] == "evict":
        batch, keep, P = case["batch"], case["keep"], case["page"]
        k, v = (torch.zeros((batch * keep, case["kv_heads"], case["dim"]), dtype=torch.float64, device=DEVICE) for _ in range(2))
        weights = s["weights"].clone()
        for b in range(batch):
            T, first, to = int(s["lengths"][b]), int(s["offsets"][b]), int(s["dst_offsets"][b])
            n = min(T, keep)
            w = weights[s["table"][first:first + -(-T // P)].long()].transpose(1, 2).reshape(-1, case["kv_heads"])[:T]
            total = w.double().sum(1).float().cpu().numpy()
            rank = [(-math.inf if t < case["sink"] or t >= T - case["recent"] else -float(total[t]), t) for t in range(T)]
            ids = torch.tensor(sorted(t for _, t in sorted(rank)[:n]), device=DEVICE)
            k[b * keep:b * keep + n], v[b * keep:b * keep + n] = _rows_of(s, b, "k")[ids], _rows_of(s, b, "v")[ids]
            for j0 in range(0, n, P):
                c = min(P, n - j0)
                weights[int(s["spare"][to + j0 // P]), :, :c] = w[ids[j0:j0 + c]].t()
        return {"kept": None, "starts": None, "positions": None, "weights": weights.double(), "k": k, "v": v}
    batch, R, H, h = case["batch"], case["rows"], case["q_heads"], case["kv_heads"]
    if case["op"] == "weights":
        total = s["weights"].double()
        P = case["page"]
        for b in range(batch):
            T, first = int(s["lengths"][b]), int(s["offsets"][b])
            m, l = (s[x].reshape(batch, R, H)[b].double() for x in ("m", "l"))
            p = torch.exp(_scores_of(s, b) - torch.where(l > 0, m, torch.zeros_like(m))[..., None])
            p = p / torch.where(l > 0, l, torch.ones_like(l))[..., None]
            mass = p.reshape(R, h, H // h, T).sum((0, 2))
            pages = s["table"][first:first + -(-T // P)].long()
            have = total[pages].transpose(0, 1).reshape(h, -1)
            have[:, max(0, T - case["fresh"]):T] = 0.0
            have[:, :T] += mass
            total[pages] = have.reshape(h, -1, P).transpose(0, 1)
        return total
    out = torch.zeros((batch, R, H, case["dim"]), dtype=torch.float64, device=DEVICE)
    m, l = (torch.zeros((batch, R, H), dtype=torch.float64, device=DEVICE) for _ in range(2))
    for b in range(batch):
        x = _scores_of(s, b)
        m[b] = x.max(-1).values
        p = torch.exp(x - torch.where(torch.isinf(m[b]), torch.zeros_like(m[b]), m[b])[..., None])
        l[b] = p.sum(-1)
        V = _rows_of(s, b, "v")
        for i in range(H):
            out[b, :, i] = (p[:, i] @ V[:, i // (H // h)]) / torch.where(l[b, :, i] > 0, l[b, :, i], torch.ones_like(l[b, :, i]))[:, None]
    return {"out": out, "m": m, "l": l}


if __name__ == "__main__":
    for c in listed() + [draw(random.Random(i)) for i in range(6)]:
        print(c, work(c))
