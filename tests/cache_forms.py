"""Plain 64-bit implementations of the operators on a 4- or 8-bit cache, and
builders of small cases, for the tests (numpy, host only)."""
import math

import numpy as np

import kvbridge_amd as kvb

NP_SRC = {"f32": kvb.KVB_SRC_F32, "f16": kvb.KVB_SRC_F16, "bf16": kvb.KVB_SRC_BF16}
OUT = {"f32": kvb.KVB_OUT_F32, "f16": kvb.KVB_OUT_F16, "bf16": kvb.KVB_OUT_BF16}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def bf16_round(x):
    """fp32 -> nearest bfloat16 (half to even) as fp32; overflow gives infinity."""
    u = np.asarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16 << 16).astype(np.uint32).view(np.float32)


def encode4(x):
    """Rows [..., dim] fp32 -> (packed uint8 [..., dim / 2], words uint32 [..., dim / 32]), in IEEE fp32."""
    x = np.asarray(x, np.float32)
    G = x.shape[-1] // 32
    b = x.reshape(*x.shape[:-1], G, 32)
    with np.errstate(all="ignore"):
        least = bf16_round(b.min(-1))
        step = bf16_round(np.maximum(b.max(-1) - least, np.float32(0)) / np.float32(15))
        bad = ~(np.isfinite(b).all(-1) & np.isfinite(least) & np.isfinite(step))
        flat = bad | (step == 0)
        c = np.rint((b - least[..., None]) / np.where(flat, np.float32(1), step)[..., None])
        c = np.where(flat[..., None], 0, np.clip(c, 0, 15)).astype(np.uint8)
    step_b = np.where(bad, np.uint32(0x7FC0), step.view(np.uint32) >> 16).astype(np.uint32)
    least_b = np.where(bad, np.uint32(0x7FC0), least.view(np.uint32) >> 16).astype(np.uint32)
    c = c.reshape(*x.shape[:-1], G, 16, 2)
    packed = np.swapaxes(c[..., 0] | (c[..., 1] << 4), -1, -2)
    return np.ascontiguousarray(packed.reshape(*x.shape[:-1], 16 * G)), (step_b << 16 | least_b)


def decode4(packed, words):
    """Values of packed rows in fp64."""
    G = words.shape[-1]
    b = np.swapaxes(packed.reshape(*packed.shape[:-1], 16, G), -1, -2)
    c = np.stack((b & 15, b >> 4), -1).reshape(*packed.shape[:-1], G, 32).astype(np.float64)
    step = (words & np.uint32(0xFFFF0000)).view(np.float32).astype(np.float64)
    least = (words << np.uint32(16)).view(np.float32).astype(np.float64)
    return (c * step[..., None] + least[..., None]).reshape(*packed.shape[:-1], 32 * G)


class Case:
    """A ragged batch over a shuffled pool in either format (host arrays)."""

    def __init__(self, bits, lengths, rows, q_heads, kv_heads, dim, page, *, seed=0, kind="f32", cap=0.0, window=0,
                 slopes=False, prefix=None, scale=None, spare=0, qpos=None, kpos=None, q_pad=0, split_tokens=0):
        rng = np.random.default_rng(seed)
        self.bits, self.lengths, self.rows, self.q_heads, self.kv_heads, self.dim, self.page = \
            bits, [int(t) for t in lengths], rows, q_heads, kv_heads, dim, page
        self.kind, self.cap, self.window, self.split_tokens = kind, cap, window, split_tokens
        batch = self.batch = len(lengths)
        npages = [-(-t // page) for t in self.lengths]
        self.pages = max(1, sum(npages)) + spare
        perm = rng.permutation(self.pages).astype(np.uint32)
        self.table, self.free = perm[:max(1, sum(npages))], perm[max(1, sum(npages)):]
        self.offsets = np.concatenate([[0], np.cumsum(npages)[:-1]]).astype(np.uint32)
        self.starts = np.concatenate([[0], np.cumsum(self.lengths)]).astype(np.uint32)
        total = max(1, int(self.starts[-1]))
        if kpos is None:
            kpos = np.concatenate([np.arange(t) for t in self.lengths] + [np.zeros(total - int(self.starts[-1]))])
        self.kpos = np.asarray(kpos, np.int64)
        if qpos is None:
            qpos = np.stack([np.arange(rows) + t - rows for t in self.lengths])
        self.qpos = np.asarray(qpos, np.int64).reshape(batch, rows)
        self.q_stride = q_heads * dim + q_pad
        q = rng.standard_normal((batch * rows, self.q_stride)).astype(np.float32)
        self.q = {"f32": lambda: q, "f16": lambda: q.astype(np.float16).astype(np.float32), "bf16": lambda: bf16_round(q)}[kind]()
        kx = rng.standard_normal((self.pages, kv_heads, page, dim)).astype(np.float32)
        vx = rng.standard_normal((self.pages, kv_heads, page, dim)).astype(np.float32)
        if bits == 4:
            (self.k, self.ks), (self.v, self.vs) = encode4(kx), encode4(vx)
        else:
            def enc(x):
                s = np.abs(x).max(-1) / np.float32(127)
                return np.clip(np.rint(x / s[..., None]), -127, 127).astype(np.int8), s
            self.k, self.ks = enc(kx)
            v, self.vs = enc(vx)
            self.v = np.ascontiguousarray(np.swapaxes(v, 2, 3))
        self.weights = rng.random((self.pages, kv_heads, page), dtype=np.float32)
        self.slopes = (2.0 ** (-8.0 * np.arange(1, q_heads + 1) / q_heads)).astype(np.float32) if slopes else None
        self.prefix = None if prefix is None else np.full(batch, prefix, np.int64)
        self.scale = np.float32(1 / math.sqrt(dim) if scale is None else scale)
        self.max_tokens = max(1, max(self.lengths))

    # -- plain forms --
    def rows_of(self, b, name):
        """K or V of sequence b in fp64, [tokens, kv_heads, dim]."""
        T, P = self.lengths[b], self.page
        pg = self.table[self.offsets[b]:self.offsets[b] + -(-T // P)]
        return self.pool_values(name)[pg].transpose(0, 2, 1, 3).reshape(-1, self.kv_heads, self.dim)[:T]

    def pool_values(self, name):
        """Every slot's K or V as fp64 values, [pages, kv_heads, page, dim]."""
        codes, scales = (self.k, self.ks) if name == "k" else (self.v, self.vs)
        if self.bits == 4:
            return decode4(codes, scales)
        codes = np.swapaxes(codes, 2, 3) if name == "v" else codes
        return codes.astype(np.float64) * scales.astype(np.float64)[..., None]

    def scores(self, b):
        """(masked scores fp64 [rows, q_heads, tokens], largest sum of the magnitudes of a score's terms)."""
        K = self.rows_of(b, "k")
        T, group = K.shape[0], self.q_heads // self.kv_heads
        q = self.q.reshape(self.batch, self.rows, self.q_stride)[b, :, :self.q_heads * self.dim]
        q = q.reshape(self.rows, self.q_heads, self.dim).astype(np.float64)
        x = np.stack([q[:, h] @ K[:, h // group].T for h in range(self.q_heads)], 1) * float(self.scale)
        bound = float(np.abs(q).sum(-1).max() * abs(float(self.scale)) * 2 * (np.abs(K).max() if T else 0.0))
        if self.cap:
            x = self.cap * np.tanh(x / self.cap)
        far = self.kpos[self.starts[b]:self.starts[b] + T][None, :] - self.qpos[b][:, None]
        if self.slopes is not None:
            x = x + self.slopes.astype(np.float64)[None, :, None] * far[:, None, :]
        seen = far <= 0
        if self.window:
            seen &= -far < self.window
        if self.prefix is not None:
            seen |= (self.kpos[self.starts[b]:self.starts[b] + T] < self.prefix[b])[None, :]
        return np.where(seen[:, None, :], x, -np.inf), bound

    def attention(self):
        """m, l [batch, rows, q_heads], out [.., dim] in fp64, and the score bound and largest value of each sequence."""
        R, H, D, group = self.rows, self.q_heads, self.dim, self.q_heads // self.kv_heads
        m, l = np.full((self.batch, R, H), -np.inf), np.zeros((self.batch, R, H))
        out, bounds, tops = np.zeros((self.batch, R, H, D)), [], []
        for b in range(self.batch):
            x, bound = self.scores(b)
            V = self.rows_of(b, "v")
            bounds.append(bound)
            tops.append(float(np.abs(V).max()) if len(V) else 0.0)
            if x.shape[-1] == 0:
                continue
            m[b] = x.max(-1)
            p = np.where(np.isfinite(x), np.exp(x - np.where(np.isfinite(m[b]), m[b], 0)[..., None]), 0)
            l[b] = p.sum(-1)
            for h in range(H):
                out[b, :, h] = (p[:, h] @ np.where(np.isfinite(V[:, h // group]), V[:, h // group], 0)) / \
                    np.where(l[b, :, h] > 0, l[b, :, h], 1)[:, None]
        return m, l, out, np.asarray(bounds), np.asarray(tops)

    def mass(self, b):
        """Attention weight of each token and kv head, summed over rows and query heads: fp64 [tokens, kv_heads]."""
        x, _ = self.scores(b)
        if x.shape[-1] == 0:
            return np.zeros((0, self.kv_heads))
        m = x.max(-1, keepdims=True)
        p = np.where(np.isfinite(x), np.exp(x - np.where(np.isfinite(m), m, 0)), 0)
        l = p.sum(-1, keepdims=True)
        p = p / np.where(l > 0, l, 1)
        return p.reshape(self.rows, self.kv_heads, -1, x.shape[-1]).sum((0, 2)).T

    # -- device side --
    def shape(self, **changes):
        s = kvb.make_scored_shape(self.batch, self.rows, self.q_heads, self.kv_heads, self.dim, self.page, self.pages,
                                  self.max_tokens, len(self.kpos), len(self.table), float(self.scale), kv_bits=self.bits,
                                  q_type=NP_SRC[self.kind], q_stride=self.q_stride, window=self.window, cap=self.cap,
                                  split_tokens=self.split_tokens)
        return s.copy(**changes)

    def to_device(self, device="cuda:0"):
        import torch

        def dev(a):
            if a is None:
                return None
            a = np.ascontiguousarray(a)
            return torch.from_numpy(a.view(np.int32) if a.dtype == np.uint32 else a).to(device)

        q = torch.from_numpy(self.q).to({"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[self.kind])
        return {"q": q.to(device), **{n: dev(getattr(self, n)) for n in
                ("qpos", "starts", "offsets", "kpos", "table", "k", "v", "ks", "vs", "slopes", "prefix", "weights", "free")}}


def scored_input(t):
    return kvb.scored_input(t["q"], t["qpos"], t["starts"], t["offsets"], t["kpos"], t["table"], t["k"], t["v"], t["ks"],
                            t["vs"], t["slopes"], t["prefix"])


class Attend:
    """Workspaces and outputs of a case's attention call, and the call."""

    def __init__(self, case, t, out_kind=None, fused=True, **changes):
        import torch

        self.s, self.t, self.kind = case.shape(**changes), t, out_kind or case.kind
        dev = t["q"].device
        self.inp = scored_input(t)
        self.scratch = torch.full((kvb.scored_scratch_elements(self.s),), float("nan"), device=dev)
        self.counters = torch.zeros(kvb.scored_counter_elements(self.s), dtype=torch.int32, device=dev) if fused else None
        shape = (case.batch, case.rows, case.q_heads)
        self.m, self.l = (torch.full(shape, float("nan"), device=dev) for _ in range(2))
        dt = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[self.kind]
        self.out = torch.full((*shape, case.dim), float("nan"), dtype=dt, device=dev)

    def __call__(self, stream=None):
        kvb.decode_attention_scored(self.s, self.inp, self.scratch, self.m, self.l, self.out, OUT[self.kind], self.counters,
                                    stream)
        return self

    def read(self):
        import torch

        torch.cuda.synchronize()
        if self.counters is not None:
            assert int(torch.count_nonzero(self.counters)) == 0
        return (self.m.double().cpu().numpy(), self.l.double().cpu().numpy(), self.out.double().cpu().numpy())


def check_attention(case, got, out_kind=None, want=None):
    """m, l, out against fp64.

    A score is a sum of fewer than 2 * 8 + 16 fp32 roundings of partial sums
    that are at most `bound`, the sum of its terms' magnitudes (the value of a
    4-bit element is a difference of two terms, each at most twice the largest
    value's magnitude): delta = 32 * 2^-24 * bound, plus 8 * 2^-24 of the cap
    and 4 * 2^-24 of a visible bias.  e^s moves by delta relative, the quotient
    by twice that; its sums carry at most 2^-19 of the largest value (two
    digits of 11 bits, a few roundings per tile), or half an fp16 step of each
    weight, 2^-11, where the output is bf16 with a 16-bit q; and the output
    half a step of its type."""
    kind = out_kind or case.kind
    m, l, out = got
    wm, wl, wout, bounds, tops = want if want is not None else case.attention()
    empty = wl == 0
    assert np.array_equal(np.isneginf(m), empty) and np.array_equal(l == 0, empty)
    assert np.all(out[empty] == 0)
    bias = 0.0
    if case.slopes is not None:
        bias = 4 * 2.0 ** -24 * float(case.slopes.max()) * 64  # farther keys have no weight left at these slopes
    delta = 32 * 2.0 ** -24 * bounds[:, None, None] + 8 * 2.0 ** -24 * case.cap + bias + 2.0 ** -22
    seen = ~empty
    err_m = np.abs(np.where(seen, m, 0) - np.where(seen, wm, 0))
    assert np.all(err_m <= delta), (err_m.max(), delta.min())
    err_l = np.abs(l - wl) / np.where(seen, wl, 1)
    assert np.all(err_l <= 2 * delta + 2.0 ** -20), (err_l.max(), delta.min())
    digits = 2.0 ** -11 if kind == "bf16" and case.kind != "f32" else 0.0
    tol = (2 * delta + 2.0 ** -19 + digits)[..., None] * tops[:, None, None, None] + HALF_STEP[kind] * np.abs(wout)
    if kind == "f16":
        tol = tol + 2.0 ** -25  # half a subnormal step
    assert np.all(np.abs(out - wout) <= tol), (np.abs(out - wout).max(), tol.min())
