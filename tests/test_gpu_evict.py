"""evict_select and evict_move on the GPU against plain forms, and a serving
step of all the operators together: write, attend, weigh, evict, attend."""
import numpy as np
import pytest

import kvbridge_amd as kvb

from cache_forms import Attend, Case, check_attention, encode4

pytestmark = pytest.mark.gpu


def select_plain(case, weights, keep, sink, recent):
    kept = []
    for b in range(case.batch):
        T = case.lengths[b]
        pg = case.table[case.offsets[b]:case.offsets[b] + -(-T // case.page)]
        w = weights[pg].transpose(0, 2, 1).reshape(-1, case.kv_heads)[:T].astype(np.float64)
        with np.errstate(invalid="ignore"):
            key = w.sum(1).astype(np.float32)
        order = sorted(range(T), key=lambda t: (not (t < sink or t >= T - recent), np.isnan(key[t]),
                                                -float(key[t]) if not np.isnan(key[t]) else 0.0, t))
        kept.append(sorted(order[:min(T, keep)]))
    return kept


class Evict:
    def __init__(self, case, t, keep, sink, recent):
        import torch

        self.case, self.t, self.keep = case, t, keep
        self.s = kvb.make_evict_shape(case.batch, case.kv_heads, case.dim, case.page, case.pages, case.max_tokens,
                                      len(case.kpos), len(case.table), len(case.free), keep, sink, recent, case.bits)
        self.inp = kvb.evict_input(t["starts"], t["offsets"], t["table"], t["kpos"])
        dev = t["k"].device
        self.scratch = torch.empty(kvb.evict_scratch_elements(self.s), dtype=torch.int32, device=dev)
        self.kept = torch.full((case.batch, keep), -7, dtype=torch.int32, device=dev)
        self.starts = torch.empty(case.batch + 1, dtype=torch.int32, device=dev)
        self.positions = torch.full((case.batch * keep,), -7, dtype=torch.int64, device=dev)
        counts = [-(-min(n, keep) // case.page) for n in case.lengths]
        self.doff = np.concatenate([[0], np.cumsum(counts)[:-1]]).astype(np.int32)
        self.cache = kvb.evict_cache(t["k"], t["v"], t["ks"], t["vs"], t["weights"], torch.from_numpy(self.doff).to(dev),
                                     t["free"], self.positions)
        self._keep_alive = torch.from_numpy(self.doff).to(dev)
        self.cache.dst_offsets = self._keep_alive.data_ptr()

    def select(self, stream=None):
        kvb.evict_select(self.s, self.inp, self.t["weights"], self.scratch, self.kept, self.starts, stream)

    def move(self, stream=None):
        kvb.evict_move(self.s, self.inp, self.cache, self.kept, self.starts, stream)


SELECT = [
    # lengths, kv_heads, page, keep, sink, recent, weights
    ([300, 1, 0, 64, 65], 2, 16, 64, 2, 10, "random"),
    ([5000, 4097, 3], 8, 64, 1000, 4, 100, "random"),
    ([700], 3, 24, 699, 0, 0, "random"),
    ([700, 33], 1, 8, 1, 0, 0, "random"),
    ([700, 500], 2, 8, 10, 4, 6, "random"),      # nothing but the ends
    ([2500], 2, 16, 777, 1, 1, "equal"),         # every weight the same: the earliest
    ([2500, 1300], 1, 16, 500, 0, 8, "few"),     # many ties
    ([900, 400], 2, 16, 300, 3, 5, "odd"),       # NaN, infinities, zeros of both signs, negative values
]


def weights_of(case, how, rng):
    shape = case.weights.shape
    if how == "equal":
        return np.full(shape, 0.25, np.float32)
    if how == "few":
        return rng.integers(0, 4, shape).astype(np.float32) / 4
    w = rng.exponential(1.0, shape).astype(np.float32) ** 3
    if how == "odd":
        pick = rng.integers(0, 40, shape)
        for i, x in enumerate((np.nan, np.inf, 0.0, -0.0, -1.5, 1e-42)):
            w[pick == i] = x
    return w


@pytest.mark.parametrize("case", SELECT, ids=lambda c: f"{c[0]}-{c[3]}-{c[6]}")
def test_select(gpu, case):
    import torch

    lengths, kvh, page, keep, sink, recent, how = case
    c = Case(4, lengths, 1, kvh, kvh, 64, page, seed=2, spare=1)
    c.weights = weights_of(c, how, np.random.default_rng(3))
    e = Evict(c, c.to_device(), keep, sink, recent)
    e.select()
    torch.cuda.synchronize()
    want = select_plain(c, c.weights, keep, sink, recent)
    got = e.kept.cpu().numpy()
    for b, ids in enumerate(want):
        assert got[b, :len(ids)].tolist() == ids, b
        assert np.all(got[b, len(ids):] == -7)  # behind the count: as it was
    assert e.starts.cpu().tolist() == np.concatenate([[0], np.cumsum([len(x) for x in want])]).tolist()


MOVE = [
    # bits, dim, page, kv_heads, lengths, keep
    (4, 64, 16, 2, [300, 5, 0, 70], 67),
    (4, 128, 24, 1, [200, 130], 129),
    (4, 256, 8, 3, [90, 20], 33),
    (8, 64, 16, 2, [300, 5, 0, 70], 67),
    (8, 128, 24, 1, [200, 130], 130),
    (8, 256, 64, 2, [190, 66], 65),
]


@pytest.mark.parametrize("case", MOVE)
def test_move_keeps_every_bit_and_touches_nothing_else(gpu, case):
    import torch

    bits, dim, page, kvh, lengths, keep = case
    need = sum(-(-min(n, keep) // page) for n in lengths)
    c = Case(bits, lengths, 1, kvh, kvh, dim, page, seed=5, spare=need + 2, kpos=np.cumsum(np.arange(sum(lengths)) % 3))
    t = c.to_device()
    e = Evict(c, t, keep, 1, 2)
    e.select()
    before = {n: t[n].cpu().numpy().copy() for n in ("k", "v", "ks", "vs", "weights")}
    e.move()
    torch.cuda.synchronize()
    kept, starts = e.kept.cpu().numpy(), e.starts.cpu().numpy()
    for b in range(c.batch):
        n = min(c.lengths[b], keep)
        for j in range(n):
            src = int(kept[b, j])
            sp, ss = int(c.table[c.offsets[b] + src // page]), src % page
            dp, ds = int(c.free[e.doff[b] + j // page]), j % page
            for name in before:
                if name == "v" and bits == 8:
                    before[name][dp, :, :, ds] = before[name][sp, :, :, ss]
                else:
                    before[name][dp, :, ds] = before[name][sp, :, ss]
            assert int(e.positions[starts[b] + j]) == int(c.kpos[c.starts[b] + src])
    for name, w in before.items():
        assert np.array_equal(t[name].cpu().numpy().view(np.uint8), w.view(np.uint8)), name
    assert np.all(e.positions.cpu().numpy()[starts[-1]:] == -7)


def test_move_skips_bad_pages_and_optional_buffers(gpu):
    """A destination id past the pool, too few destination entries, and neither
    weights nor positions: nothing outside the named pages changes."""
    import torch

    c = Case(4, [100], 1, 2, 2, 64, 16, seed=6, spare=6)
    t = c.to_device()
    t["free"][1] = -1
    e = Evict(c, t, 80, 0, 0)
    e.s.dst_entries = 3
    e.cache.weights = e.cache.positions = None
    e.select()
    before = {n: t[n].clone() for n in ("k", "v", "ks", "vs", "weights")}
    e.move()
    torch.cuda.synchronize()
    touched = [int(c.free[0]), int(c.free[2])]
    others = [p for p in range(c.pages) if p not in touched]
    for n in ("k", "v", "ks", "vs"):
        assert torch.equal(t[n][others], before[n][others])
        assert not torch.equal(t[n][touched], before[n][touched])
    assert torch.equal(t["weights"], before["weights"])


@pytest.mark.parametrize("bits", [4, 8])
def test_serving_step_of_all_operators(gpu, bits):
    """Prefill written through the writer, decode steps with attention and
    weights, then eviction and attention over what is left, each against its
    plain form; the steps captured and replayed give the eager bits."""
    import torch

    kvh, qh, D, P, lengths, keep, sink, recent = 2, 8, 64, 16, [90, 40], 48, 2, 6
    total = [n + 3 for n in lengths]
    c = Case(bits, total, 1, qh, kvh, D, P, seed=20, kind="f32", spare=6)
    rng = np.random.default_rng(21)
    x = rng.standard_normal((2, sum(total), kvh, D)).astype(np.float32)
    slot_of = lambda b, tok: int(c.table[c.offsets[b] + tok // P]) * P + tok % P  # noqa: E731
    # the host's copy of what the writer stores
    for b in range(2):
        for tok in range(total[b]):
            i = int(c.starts[b]) + tok
            pg, sl = divmod(slot_of(b, tok), P)
            if bits == 4:
                (c.k[pg, :, sl], c.ks[pg, :, sl]), (c.v[pg, :, sl], c.vs[pg, :, sl]) = encode4(x[0, i]), encode4(x[1, i])
            else:
                sk, sv = (np.abs(x[n, i]).max(-1) / np.float32(127) for n in range(2))
                c.k[pg, :, sl], c.ks[pg, :, sl] = np.rint(x[0, i] / sk[:, None]).astype(np.int8), sk
                c.v[pg, :, :, sl], c.vs[pg, :, sl] = np.rint(x[1, i] / sv[:, None]).astype(np.int8), sv
    t = c.to_device()
    used = torch.from_numpy(c.table.astype(np.int64)).to(gpu)
    full = {n: t[n].clone() for n in ("k", "v", "ks", "vs")}
    for n in ("k", "v", "ks", "vs"):
        t[n][used] = 0
    write = kvb.append_kv_i4 if bits == 4 else kvb.append_kv
    rows = [torch.from_numpy(np.ascontiguousarray(x[n])).to(gpu) for n in range(2)]

    def append(tokens_of):
        ids = [int(c.starts[b]) + tok for b in range(2) for tok in tokens_of[b]]
        slots = torch.tensor([slot_of(b, tok) for b in range(2) for tok in tokens_of[b]], dtype=torch.int32, device=gpu)
        k, v = (r[ids].contiguous() for r in rows)
        write(kvb.append_shape(len(ids), kvh, D, P, c.pages), k, v, slots, t["k"], t["v"], t["ks"], t["vs"])
        torch.cuda.synchronize()

    append([range(n) for n in lengths])
    w = torch.full_like(t["weights"], 1e9)  # stale: every token is set before it is added to
    plain_w = np.zeros(c.weights.shape)
    steps, q = [], rng.standard_normal((3, 2, qh * D)).astype(np.float32)
    for step in range(3):
        now = [n + step + 1 for n in lengths]
        append([[n - 1] for n in now])
        view = Case(bits, total, 1, qh, kvh, D, P, seed=20, kind="f32", spare=6)
        view.__dict__.update({k: v for k, v in c.__dict__.items() if k not in ("q", "qpos")})
        view.q, view.lengths = q[step].reshape(2, qh * D), now
        view.qpos = np.asarray([[n - 1] for n in now], np.int64)
        view.starts = np.asarray([0, now[0], sum(now)], np.uint32)
        view.kpos = np.concatenate([np.arange(n) for n in now]).astype(np.int64)
        view.max_tokens = max(now)
        tv = {**t, **{n: d for n, d in view.to_device().items() if n in ("q", "qpos", "starts", "kpos")}}
        call = Attend(view, tv)()
        check_attention(view, call.read())
        fresh = max(now) if step == 0 else 1
        kvb.accumulate_weights(call.s, call.inp, call.m, call.l, w, fresh)
        for b in range(2):
            for tok, mass in enumerate(view.mass(b)):
                pg, sl = divmod(slot_of(b, tok), P)
                plain_w[pg, :, sl] = (0 if tok >= now[b] - fresh else plain_w[pg, :, sl]) + mass
        steps.append((view, tv, call))
    torch.cuda.synchronize()
    for n in full:
        if not (bits == 8 and n == "v"):
            for b in range(2):
                for tok in range(total[b]):
                    pg, sl = divmod(slot_of(b, tok), P)
                    assert torch.equal(t[n][pg, :, sl], full[n][pg, :, sl])
    for b in range(2):
        for tok in range(total[b]):
            pg, sl = divmod(slot_of(b, tok), P)
            # three steps' weights, each within a few 2^-20
            assert np.allclose(w[pg, :, sl].cpu().numpy(), plain_w[pg, :, sl], rtol=2.0 ** -17, atol=2.0 ** -28)
    t["weights"] = w
    view = steps[-1][0]
    tv = {**steps[-1][1], "weights": w}
    view.weights = w.cpu().numpy()
    ev = Evict(view, tv, keep, sink, recent)
    ev.select()
    ev.move()
    torch.cuda.synchronize()
    ids = select_plain(view, view.weights, keep, sink, recent)
    assert [ev.kept[b, :len(ids[b])].tolist() for b in range(2)] == ids
    after = Case(bits, [len(i) for i in ids], 1, qh, kvh, D, P, seed=20, kind="f32", spare=6)
    after.pages, after.table, after.offsets = c.pages, np.ascontiguousarray(c.free), ev.doff.astype(np.uint32)
    after.q, after.qpos, after.kpos = view.q, view.qpos, ev.positions[:sum(len(i) for i in ids)].cpu().numpy()
    for n, d in (("k", t["k"]), ("v", t["v"]), ("ks", t["ks"]), ("vs", t["vs"])):
        a = d.cpu().numpy()
        setattr(after, n, a.view(np.uint32) if bits == 4 and n in ("ks", "vs") else a)
    td = {**tv, "starts": ev.starts, "kpos": ev.positions, "table": t["free"], "offsets": ev._keep_alive}
    call = Attend(after, td)
    check_attention(after, call().read())
    eager = [y.clone() for y in (call.m, call.l, call.out, ev.kept, t["k"], w)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ev.select()
        ev.move()
        call()
    for _ in range(3):
        call.out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, (call.m, call.l, call.out, ev.kept, t["k"], w)))
