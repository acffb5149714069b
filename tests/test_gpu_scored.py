"""decode_attention_scored and accumulate_weights on the GPU against plain
64-bit implementations: formats, head layouts, page sizes, lengths from none to
several splits, score forms, rows that see nothing, what masked places hold,
strides, streams, graphs and pools past 4 GiB."""
import numpy as np
import pytest

import kvbridge_amd as kvb

from cache_forms import Attend, Case, check_attention, scored_input

pytestmark = pytest.mark.gpu

LENGTHS = [517, 1, 0, 33, 260, 32, 7, 31]

# bits, rows, q_heads, kv_heads, dim, page, kind, out, forms
LAYOUTS = [
    (4, 1, 8, 2, 64, 16, "f16", "f16", {}),
    (4, 1, 8, 8, 128, 64, "bf16", "bf16", {}),
    (4, 1, 16, 1, 128, 8, "f32", "f32", {}),            # one full block, smallest pages
    (4, 3, 16, 2, 128, 24, "bf16", "f32", {}),          # 24 head-rows: two blocks, 24-token pages
    (4, 2, 24, 4, 256, 32, "f32", "bf16", {}),
    (4, 5, 10, 2, 64, 40, "f16", "bf16", {}),           # 25 head-rows
    (8, 1, 8, 2, 64, 16, "f16", "f16", {}),
    (8, 1, 32, 8, 128, 64, "bf16", "bf16", {}),
    (8, 3, 16, 2, 128, 24, "f32", "f32", {}),
    (8, 2, 24, 4, 256, 8, "f16", "f32", {}),
    (4, 1, 8, 2, 128, 16, "bf16", "bf16", {"cap": 5.0}),
    (4, 2, 8, 2, 64, 48, "f32", "f32", {"cap": 50.0, "window": 37}),
    (8, 2, 8, 2, 256, 64, "bf16", "f32", {"cap": 2.0, "window": 70, "prefix": 5}),
    (4, 4, 8, 2, 128, 32, "f32", "f32", {"slopes": True}),
    (8, 2, 12, 2, 64, 16, "f16", "f16", {"slopes": True, "window": 100}),
    (4, 1, 8, 2, 64, 16, "f32", "f32", {"window": 1}),
    (4, 2, 8, 2, 128, 16, "f32", "f32", {"window": 3, "prefix": 40}),
    (8, 7, 8, 2, 128, 16, "f32", "f32", {"prefix": 300}),  # rows before the prefix's end see ahead
    (4, 2, 8, 2, 256, 64, "f32", "f32", {"slopes": True, "cap": 20.0, "window": 200, "prefix": 3}),
]


@pytest.mark.parametrize("layout", LAYOUTS, ids=lambda x: "-".join(str(y) for y in x[:8]) + "-" + "-".join(x[8]))
@pytest.mark.parametrize("split", [0, 32, 96])
def test_attention_matches_64_bits(gpu, layout, split):
    bits, rows, qh, kvh, dim, page, kind, out, forms = layout
    case = Case(bits, LENGTHS, rows, qh, kvh, dim, page, seed=dim + rows, kind=kind, split_tokens=split, **forms)
    t = case.to_device()
    want = case.attention()
    for fused in (True, False):
        check_attention(case, Attend(case, t, out, fused)().read(), out, want)


@pytest.mark.parametrize("bits", [4, 8])
def test_long_context(gpu, bits):
    """Several splits of many tiles, page lookups past the first window, and a
    second call on the same workspaces."""
    case = Case(bits, [5003, 2999], 1, 8, 2, 128, 16, seed=3, kind="f16", split_tokens=1536)
    call = Attend(case, case.to_device(), "f32")
    check_attention(case, call().read(), "f32")
    first = [x.clone() for x in (call.m, call.l, call.out)]
    call().read()
    assert all(bool((a == b).all()) for a, b in zip(first, (call.m, call.l, call.out)))  # the same bits


@pytest.mark.parametrize("bits", [4, 8])
def test_rows_that_see_nothing_and_odd_positions(gpu, bits):
    """Duplicate and sparse key positions, query positions before every key,
    between keys and after all, and far beyond 32 bits."""
    lengths = [40, 65]
    far = 1 << 40
    kpos = np.concatenate([np.repeat(np.arange(20), 2) * 3, far + np.sort(np.arange(65) * 7 // 3)])
    qpos = [[-1, 0, 29, 57], [far - 1, far, far + 71, far + (1 << 35)]]
    for forms in ({}, {"window": 10}, {"prefix": 4}, {"prefix": far + 9, "window": 5}):
        case = Case(bits, lengths, 4, 8, 2, 64, 16, seed=9, qpos=qpos, kpos=kpos, **forms)
        check_attention(case, Attend(case, case.to_device())().read())


def poison(case, t):
    """NaN scales (4 bits: both parameters; 8 bits: the scale) and full codes in
    every slot that no row of its sequence sees."""
    import torch

    need = np.zeros((case.pages, case.page), bool)
    for b in range(case.batch):
        x, _ = case.scores(b)
        seen = np.isfinite(x).any((0, 1))
        for tok in np.nonzero(seen)[0]:
            need[case.table[case.offsets[b] + tok // case.page], tok % case.page] = True
    bad = torch.from_numpy(~need).to(t["k"].device)
    nan = 0x7FC07FC0 if case.bits == 4 else float("nan")
    for n in ("ks", "vs"):
        mask = bad[:, None, :, None] if case.bits == 4 else bad[:, None, :]
        t[n] = torch.where(mask, torch.full_like(t[n], nan), t[n])
    return int((~need).sum())


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("forms", [{}, {"window": 9, "prefix": 2}, {"slopes": True}])
def test_masked_places_have_no_effect(gpu, bits, forms):
    case = Case(bits, [45, 3, 100], 2, 8, 2, 128, 16, seed=4, kind="f32", spare=2, qpos=[[20, 30], [0, 1], [50, 98]], **forms)
    t = case.to_device()
    clean = Attend(case, t)().read()
    check_attention(case, clean)
    assert poison(case, t) > 0
    dirty = Attend(case, t)().read()
    assert all(np.array_equal(a, b) for a, b in zip(clean, dirty))


@pytest.mark.parametrize("bits", [4, 8])
def test_a_row_is_not_touched_by_what_only_others_see(gpu, bits):
    """A NaN token that the last row sees and the first does not."""
    import torch

    case = Case(bits, [40], 2, 4, 1, 64, 8, seed=5, qpos=[[30, 39]])
    t = case.to_device()
    want = Attend(case, t)().read()
    page, slot = int(case.table[35 // 8]), 35 % 8
    t["vs"][page, :, slot] = 0x7FC07FC0 if bits == 4 else float("nan")
    m, l, out = Attend(case, t)().read()
    assert np.array_equal(out[0, 0], want[2][0, 0]) and np.isnan(out[0, 1]).all()
    t["ks"][page, :, slot] = 0x7FC07FC0 if bits == 4 else float("nan")
    m, l, out = Attend(case, t)().read()
    assert np.array_equal(out[0, 0], want[2][0, 0]) and np.isnan(l[0, 1]).all() and np.isnan(out[0, 1]).all()
    torch.cuda.synchronize()


def test_extreme_scales(gpu):
    """Steps and values from 2^-100 to 2^100 in one context, with weights that
    single out either end: fp16 digits neither overflow nor lose the small ones
    where those carry the weight."""
    rng = np.random.default_rng(0)
    case = Case(4, [96], 1, 4, 1, 64, 16, seed=6, kind="f32")
    size = np.where(np.arange(96) < 48, 2.0 ** -60, 2.0 ** 60)
    vx = rng.standard_normal((96, 64)) * size[:, None]
    from cache_forms import encode4
    packed, words = encode4(vx.astype(np.float32))
    for tok in range(96):
        pg, sl = int(case.table[tok // 16]), tok % 16
        case.v[pg, 0, sl], case.vs[pg, 0, sl] = packed[tok], words[tok]
    for qpos in (47, 95):  # only small values; both
        case.qpos[:] = qpos
        m, l, out = Attend(case, case.to_device())().read()
        wm, wl, wout, _, _ = case.attention()
        top = np.abs(case.rows_of(0, "v")[:qpos + 1]).max()
        # sums of terms of magnitude `top`: as in check_attention
        assert np.all(np.abs(out - wout) <= 2.0 ** -16 * top)
    # a large token that has next to no weight does not cost the others' digits
    big = Case(4, [64], 1, 2, 1, 64, 16, seed=7, kind="f32", scale=4.0)
    x, _ = big.scores(0)
    tok = int(np.argmin(x.max((0, 1))))
    gap = float((x.max(-1) - x[..., tok]).min())
    pg, sl = int(big.table[tok // 16]), tok % 16
    p2, w2 = encode4((rng.standard_normal(64) * 2.0 ** 12).astype(np.float32))
    big.v[pg, 0, sl], big.vs[pg, 0, sl] = p2, w2
    m, l, out = Attend(big, big.to_device())().read()
    wm, wl, wout, bounds, tops = big.attention()
    carried = max(4.0, float(np.exp(-gap)) * tops[0])  # largest term of a sum
    delta = 32 * 2.0 ** -24 * bounds[0] + 2.0 ** -22
    assert np.all(np.abs(out - wout) <= (2 * delta + 2.0 ** -19) * carried)


def test_strided_queries_other_stream_and_zero_scale(gpu):
    import torch

    case = Case(4, [70, 20], 2, 8, 2, 64, 16, seed=8, kind="bf16", q_pad=72, scale=0.0)
    t = case.to_device()
    side = torch.cuda.Stream()
    call = Attend(case, t, "f32")
    side.wait_stream(torch.cuda.current_stream())
    call(side)
    side.synchronize()
    check_attention(case, call.read(), "f32")
    # a negative scale reverses the order
    neg = Case(4, [70, 20], 2, 8, 2, 64, 16, seed=8, kind="bf16", q_pad=72, scale=-0.3)
    check_attention(neg, Attend(neg, neg.to_device(), "f32")().read(), "f32")


@pytest.mark.parametrize("bits", [4, 8])
def test_graph_with_changing_lengths(gpu, bits):
    """One captured call and weight accumulation, replayed while lengths and
    positions in device memory change, against the eager calls."""
    import torch

    case = Case(bits, [700, 300], 1, 8, 2, 128, 64, seed=11, kind="bf16", split_tokens=128)
    t = case.to_device()
    call = Attend(case, t)
    w = torch.zeros_like(t["weights"])
    call()
    kvb.accumulate_weights(call.s, call.inp, call.m, call.l, w, 0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
        kvb.accumulate_weights(call.s, call.inp, call.m, call.l, w, 0)
    for lengths in ([700, 300], [650, 1], [17, 0], [700, 300]):
        t["starts"].copy_(torch.tensor([0, lengths[0], lengths[0] + lengths[1]], dtype=torch.int32))
        t["kpos"][:sum(lengths)] = torch.cat([torch.arange(n) for n in lengths]).to(gpu)
        t["qpos"].copy_(torch.tensor([[n - 1] for n in lengths]))
        w.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in (call.m, call.l, call.out, w)]
        w.zero_()
        call()
        kvb.accumulate_weights(call.s, call.inp, call.m, call.l, w, 0)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (call.m, call.l, call.out, w))), lengths


@pytest.mark.parametrize("bits", [4, 8])
def test_bad_metadata_stays_inside(gpu, bits):
    """Page ids past the pool, falling and oversized starts, offsets past the
    table: every index is clamped, the call ends and a sound sequence beside
    them is right (also shown on the host: every address formed is that of a
    clamped page, run and position)."""
    import torch

    case = Case(bits, [50, 40, 30], 1, 4, 2, 64, 16, seed=12)
    t = case.to_device()
    t["table"][case.offsets[0]] = -1          # a page id of 2^32 - 1
    t["starts"].copy_(torch.tensor([0, 50, 90, 1 << 30], dtype=torch.int32))  # past total_tokens
    t["offsets"][2] = 1 << 20                 # past the table: no tokens
    m, l, out = Attend(case, t)().read()
    wm, wl, wout, _, _ = case.attention()
    assert np.allclose(out[1], wout[1], atol=1e-4) and np.all(l[2] == 0)


# ---- accumulated weights ---------------------------------------------------------

def expected_weights(case, before, fresh):
    w = before.astype(np.float64)
    for b in range(case.batch):
        T = case.lengths[b]
        mass = case.mass(b)
        for tok in range(T):
            pg, sl = int(case.table[case.offsets[b] + tok // case.page]), tok % case.page
            w[pg, :, sl] = (0 if tok >= T - fresh else w[pg, :, sl]) + mass[tok]
    return w


@pytest.mark.parametrize("layout", LAYOUTS, ids=lambda x: "-".join(str(y) for y in x[:8]) + "-" + "-".join(x[8]))
@pytest.mark.parametrize("fresh", [0, 5, 1 << 31])
def test_weights_match_64_bits(gpu, layout, fresh):
    import torch

    bits, rows, qh, kvh, dim, page, kind, _, forms = layout
    case = Case(bits, LENGTHS, rows, qh, kvh, dim, page, seed=dim + rows, kind=kind, spare=1, **forms)
    t = case.to_device()
    call = Attend(case, t)()
    kvb.accumulate_weights(call.s, call.inp, call.m, call.l, t["weights"], fresh)
    torch.cuda.synchronize()
    got = t["weights"].cpu().numpy()
    want = expected_weights(case, case.weights, fresh)
    _, _, _, bounds, _ = case.attention()
    bias = 4 * 2.0 ** -24 * 64 if case.slopes is not None else 0.0
    # score and m by delta each, l by 2 delta (check_attention), the sums of at most rows * group terms of at most 1
    delta = 32 * 2.0 ** -24 * bounds.max() + 8 * 2.0 ** -24 * case.cap + bias + 2.0 ** -22
    tol = (4 * delta + 2.0 ** -20) * np.abs(want) + 2.0 ** -30
    assert np.all(np.abs(got - want) <= tol), np.abs(got - want).max()
    # without V: its buffers are not read
    inp = scored_input({**t, "v": None, "vs": None})
    before = t["weights"].clone()
    kvb.accumulate_weights(call.s, inp, call.m, call.l, t["weights"], 0)
    torch.cuda.synchronize()
    assert float((t["weights"] - before).sum()) == pytest.approx(sum(case.mass(b).sum() for b in range(case.batch)), rel=1e-4)


def test_weights_of_a_shared_page_are_both_sequences(gpu):
    import torch

    case = Case(4, [32, 32], 1, 4, 2, 64, 16, seed=13)
    case.table[case.offsets[1]] = case.table[case.offsets[0]]  # a common first page
    t = case.to_device()
    call = Attend(case, t)()
    check_attention(case, call.read())
    kvb.accumulate_weights(call.s, call.inp, call.m, call.l, t["weights"], 0)
    torch.cuda.synchronize()
    assert np.allclose(t["weights"].cpu().numpy(), expected_weights(case, case.weights, 0), rtol=1e-5, atol=1e-6)


def test_pool_past_4_gib(gpu):
    """Pages whose rows begin past 2^32 bytes (4-bit rows of 64 bytes) through
    the writer, the reader, attention, weights and the move."""
    import torch

    P, kvh, D = 64, 8, 128
    pages = (1 << 32) // (P * kvh * 64) + 64
    lengths = [150, 64]
    small = Case(4, lengths, 1, 16, kvh, D, P, seed=14, kind="f16")
    t = small.to_device()
    high = torch.tensor([pages - 1, pages - 5, pages - 9, pages - 40], dtype=torch.int32)
    big = {n: torch.empty((pages, *t[n].shape[1:]), dtype=t[n].dtype, device=gpu) for n in ("k", "v", "ks", "vs", "weights")}
    assert big["k"].numel() > 1 << 32
    for n in big:
        for i, pg in enumerate(small.table):
            big[n][int(high[i])] = t[n][int(pg)]
    want = Attend(small, t)().read()
    tb = {**t, **{n: big[n] for n in ("k", "v", "ks", "vs")}, "table": high.to(gpu)}
    call = Attend(small, tb, pages=pages)
    assert all(np.array_equal(a, b) for a, b in zip(want, call().read()))
    kvb.accumulate_weights(call.s, call.inp, call.m, call.l, big["weights"], 0)
    kvb.accumulate_weights(small.shape(), scored_input(t), call.m, call.l, t["weights"], 0)
    for i, pg in enumerate(small.table):
        assert torch.equal(big["weights"][int(high[i])], t["weights"][int(pg)])
    # write and read back at the last page
    x = torch.randn((3, 2, kvh * D), device=gpu)
    slots = torch.tensor([(pages - 2) * P, (pages - 2) * P + 63, pages * P], dtype=torch.int64).to(torch.int32).to(gpu)
    kvb.append_kv_i4(kvb.append_shape(3, kvh, D, P, pages, k_stride=2 * kvh * D, v_stride=2 * kvh * D), x[:, 0], x[:, 1],
                     slots, big["k"], big["v"], big["ks"], big["vs"])
    k, v = (torch.full((3, kvh, D), float("nan"), device=gpu) for _ in range(2))
    kvb.read_kv(kvb.read_shape(3, kvh, D, P, pages, 4), slots, big["k"], big["v"], big["ks"], big["vs"], k, v)
    torch.cuda.synchronize()
    from cache_forms import decode4, encode4
    for got, src in ((k, x[:, 0]), (v, x[:, 1])):
        rows = decode4(*encode4(src.reshape(3, kvh, D).cpu().numpy()))
        rows[2] = 0
        assert np.array_equal(got.double().cpu().numpy(), rows.astype(np.float32).astype(np.float64))
    # the move, out of and into pages past 4 GiB
    e = kvb.make_evict_shape(2, kvh, D, P, pages, 150, 214, 4, 2, 60, 2, 8)
    inp = kvb.evict_input(tb["starts"], tb["offsets"], tb["table"], tb["kpos"])
    kept = torch.full((2, 60), -1, dtype=torch.int32, device=gpu)
    starts = torch.empty(3, dtype=torch.int32, device=gpu)
    scratch = torch.empty(kvb.evict_scratch_elements(e), dtype=torch.int32, device=gpu)
    kvb.evict_select(e, inp, big["weights"], scratch, kept, starts)
    dst = torch.tensor([pages - 20, pages - 21], dtype=torch.int32, device=gpu)
    pos = torch.empty(120, dtype=torch.int64, device=gpu)
    kvb.evict_move(e, inp, kvb.evict_cache(big["k"], big["v"], big["ks"], big["vs"], big["weights"],
                                           torch.tensor([0, 1], dtype=torch.int32, device=gpu), dst, pos), kept, starts)
    torch.cuda.synchronize()
    for b in range(2):
        ids = kept[b].long().cpu()
        for n in big:
            src = torch.stack([big[n][int(high[int(small.offsets[b]) + int(i) // P])][:, int(i) % P] for i in ids], 1)
            assert torch.equal(big[n][int(dst[b])][:, :60], src), n
