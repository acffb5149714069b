"""Calls on a 4- or 8-bit cache at their ends, on the GPU against the plain
64-bit forms: many head-rows, every column layout over long contexts, one
sequence over more items than a merge holds at once, hundreds of sequences,
graphs captured before any eager call, two streams at a time, and selections
over more tokens than a work-group holds."""
import numpy as np
import pytest

import kvbridge_amd as kvb

from cache_forms import Attend, Case, check_attention, encode4
from test_gpu_evict import Evict, select_plain, weights_of
from test_gpu_scored import expected_weights

pytestmark = pytest.mark.gpu


def check_weights(case, t, call, fresh):
    """Tolerance: score and m off by delta each and l by 2 delta (check_attention),
    fewer than 2^5 fp32 roundings of sums of positive terms."""
    import torch

    kvb.accumulate_weights(call.s, call.inp, call.m, call.l, t["weights"], fresh)
    torch.cuda.synchronize()
    want = expected_weights(case, case.weights, fresh)
    _, _, _, bounds, _ = case.attention()
    delta = 32 * 2.0 ** -24 * bounds.max() + 8 * 2.0 ** -24 * case.cap + 2.0 ** -22
    got = t["weights"].cpu().numpy()
    assert np.all(np.abs(got - want) <= (4 * delta + 2.0 ** -18) * np.abs(want) + 2.0 ** -30), np.abs(got - want).max()


MANY = [
    # bits, rows, q_heads, kv_heads, dim, page, kind: the weights' Q operands take more than one pass at the last sizes
    (4, 9, 8, 1, 256, 16, "f32"),
    (4, 16, 16, 2, 128, 32, "bf16"),
    (4, 30, 8, 1, 64, 8, "f32"),
    (8, 9, 8, 1, 256, 32, "f32"),
    (8, 16, 16, 2, 128, 24, "f16"),
    (8, 70, 4, 1, 64, 16, "f32"),
]


@pytest.mark.parametrize("case", MANY)
@pytest.mark.parametrize("forms", [{}, {"window": 40, "prefix": 3}])
def test_many_head_rows(gpu, case, forms):
    bits, rows, qh, kvh, dim, page, kind = case
    c = Case(bits, [75, 300, 0, 131], rows, qh, kvh, dim, page, seed=31, kind=kind, **forms)
    c.qpos[2] = -1
    t = c.to_device()
    want = c.attention()
    for fused in (True, False):
        call = Attend(c, t, "f32", fused)()
        check_attention(c, call.read(), "f32", want)
    check_weights(c, t, call, 7)


COLUMNS = [
    # bits, q_heads, kv_heads, dim: head-rows over 8, 4, 2 and 1 columns each
    (4, 4, 2, 256), (4, 8, 2, 256), (4, 16, 2, 256),
    (4, 4, 4, 128), (4, 16, 2, 128), (4, 32, 2, 128),
    (4, 16, 2, 64), (4, 32, 2, 64),
    (8, 8, 2, 64), (8, 8, 2, 128), (8, 8, 2, 256),
]


@pytest.mark.parametrize("case", COLUMNS)
@pytest.mark.parametrize("page", [16, 64])
def test_shared_out_items(gpu, case, page):
    """Items by length (no split size named): one long sequence beside short ones."""
    bits, qh, kvh, dim = case
    c = Case(bits, [4001, 20, 9000, 641], 1, qh, kvh, dim, page, seed=32, kind="f16")
    t = c.to_device()
    want = c.attention()
    for fused in (True, False):
        call = Attend(c, t, "f32", fused)
        check_attention(c, call().read(), "f32", want)
        first = [x.clone() for x in (call.m, call.l, call.out)]
        call().read()  # the same workspaces: the same bits
        assert all(bool((a == b).all()) for a, b in zip(first, (call.m, call.l, call.out)))
    check_weights(c, t, call, 0)


@pytest.mark.parametrize("qh,kvh,dim,tokens", [(2, 2, 64, 33000), (8, 1, 128, 70000)])
def test_one_sequence_over_more_items_than_a_merge_takes_at_once(gpu, qh, kvh, dim, tokens):
    c = Case(4, [tokens], 1, qh, kvh, dim, 64, seed=33, kind="f16")
    t = c.to_device()
    want = c.attention()
    for fused in (True, False):
        call = Attend(c, t, "f32", fused)
        assert kvb.scored_item_count(call.s) > 64
        check_attention(c, call().read(), "f32", want)
    check_weights(c, t, call, 0)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("batch", [70, 256, 300])
def test_hundreds_of_sequences(gpu, bits, batch):
    """Up to 256 sequences share the items out, above them every one gets the same number."""
    lengths = np.random.default_rng(batch).integers(0, 150, batch)
    lengths[batch // 2] = 1500
    c = Case(bits, lengths, 1, 4, 2, 64, 16, seed=34, kind="bf16", window=100)
    t = c.to_device()
    want = c.attention()
    for fused in (True, False):
        call = Attend(c, t, "f32", fused)()
        check_attention(c, call.read(), "f32", want)
    check_weights(c, t, call, 1)


@pytest.mark.parametrize("bits,qh,kvh,dim", [(4, 32, 2, 128), (8, 16, 2, 256), (4, 4, 2, 128), (4, 32, 2, 256)])
def test_capture_without_an_eager_call(gpu, bits, qh, kvh, dim):
    """After preloading, the first call of a shape may be a captured one, also
    where a work-group needs more than 64 KiB of LDS."""
    import torch

    assert kvb.preload_attention_kernels() == 0
    c = Case(bits, [3000], 1, qh, kvh, dim, 64, seed=35, kind="f32")
    t = c.to_device()
    calls = [Attend(c, t, "f32", fused) for fused in (True, False)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in calls:
            call()
    want = c.attention()
    for _ in range(3):
        for call in calls:
            call.out.fill_(float("nan"))
        graph.replay()
        for call in calls:
            check_attention(c, call.read(), "f32", want)


def test_two_streams_at_a_time(gpu):
    """Calls on two streams with workspaces of their own, and captured graphs of
    each replayed beside each other, give the bits of calls alone."""
    import torch

    cases = [Case(4, [2000, 900], 1, 8, 2, 128, 32, seed=36, kind="f16"), Case(8, [1700, 1200], 2, 8, 2, 64, 16, seed=37)]
    ts = [c.to_device() for c in cases]
    calls = [Attend(c, t, "f32")() for c, t in zip(cases, ts)]
    alone = [call.read() for call in calls]
    for c, got in zip(cases, alone):
        check_attention(c, got, "f32")
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(5):
        for call, s in zip(calls, streams):
            s.wait_stream(torch.cuda.current_stream())
            call(s)
            call(s)
    for call, want in zip(calls, alone):
        assert all(np.array_equal(a, b) for a, b in zip(call.read(), want))
    graphs = []
    for call in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call()
        graphs.append(g)
    for _ in range(5):
        for g, s in zip(graphs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for call, want in zip(calls, alone):
            assert all(np.array_equal(a, b) for a, b in zip(call.read(), want))


@pytest.mark.parametrize("lengths,keep,how", [([70001, 32769, 32768], 5000, "random"), ([66000], 33000, "equal"),
                                              ([40000, 100], 39999, "few")])
def test_select_over_more_tokens_than_a_work_group_holds(gpu, lengths, keep, how):
    import torch

    c = Case(4, lengths, 1, 1, 1, 64, 64, seed=38, spare=1)
    c.weights = weights_of(c, how, np.random.default_rng(39))
    e = Evict(c, c.to_device(), keep, 3, 17)
    e.select()
    torch.cuda.synchronize()
    got = e.kept.cpu().numpy()
    for b, ids in enumerate(select_plain(c, c.weights, keep, 3, 17)):
        assert got[b, :len(ids)].tolist() == ids, b


def test_select_from_weights_off_16_bytes(gpu):
    """The weights are floats: no alignment beyond theirs is asked for."""
    import torch

    c = Case(4, [700, 33, 9], 1, 3, 3, 64, 24, seed=43, spare=1)
    c.weights = weights_of(c, "odd", np.random.default_rng(44))
    t = c.to_device()
    e = Evict(c, t, 65, 1, 9)
    want = select_plain(c, c.weights, 65, 1, 9)
    room = torch.empty(t["weights"].numel() + 1, device=gpu)
    off = room[1:].view(t["weights"].shape)
    off.copy_(t["weights"])
    kvb.evict_select(e.s, e.inp, off, e.scratch, e.kept, e.starts)
    torch.cuda.synchronize()
    got = e.kept.cpu().numpy()
    assert [got[b, :len(w)].tolist() for b, w in enumerate(want)] == want


def test_one_token_kept_of_one(gpu):
    """The smallest eviction: every sequence one token, kept and moved."""
    import torch

    c = Case(8, [1, 1], 1, 1, 1, 64, 8, seed=40, spare=2)
    t = c.to_device()
    e = Evict(c, t, 1, 0, 0)
    e.select()
    e.move()
    torch.cuda.synchronize()
    assert e.kept.tolist() == [[0], [0]] and e.starts.tolist() == [0, 1, 2]
    for b in range(2):
        src, dst = int(c.table[b]), int(c.free[b])
        assert torch.equal(t["k"][src][:, 0], t["k"][dst][:, 0]) and torch.equal(t["v"][src][..., 0], t["v"][dst][..., 0])


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim,heads", [(64, 16), (128, 16), (128, 8), (256, 16), (256, 4)])
@pytest.mark.parametrize("at", [0, 12, 28])
def test_head_rows_of_different_value_scales(gpu, bits, dim, heads, at):
    """Head-rows of a block that meet their largest weights at values 2^14 apart,
    then large values in four tokens of a tile: head h looks at dim h of K only.
    Going backwards, head 0's best token of every tile holds tiny values, the
    other heads weigh all tokens alike; in the first half the tokens from `at` on
    have values of 1 and scores for head 0 that are 5 higher, the rest tiny ones."""
    T = 2048
    c = Case(bits, [T], 1, heads, 1, dim, 32, seed=41, kind="f32", scale=1.0)
    rng = np.random.default_rng(42)
    c.q[:] = 0
    for h in range(heads):
        c.q[0, h * dim + h] = 1.0
    k, v = np.zeros((T, dim), np.float32), rng.standard_normal((T, dim)).astype(np.float32)
    k[:, 0], k[:, heads:] = -30.0, 0.01
    best = np.arange(T // 2, T, 32) + rng.integers(0, 32, T // 64)
    k[best, 0] = 0.0
    v[best] *= 2.0 ** -14
    large = np.arange(0, T // 2).reshape(-1, 32)[:, at:at + 4].ravel()
    k[large, 0] = 5.0
    v[np.setdiff1d(np.arange(T // 2), large)] *= 2.0 ** -14
    for i in range(T):
        pg, sl = int(c.table[i // 32]), i % 32
        for rows, codes, scales in ((k, c.k, c.ks), (v, c.v, c.vs)):
            if bits == 4:
                codes[pg, 0, sl], scales[pg, 0, sl] = encode4(rows[i])
            else:
                s = np.abs(rows[i]).max() / np.float32(127)
                x = np.clip(np.rint(rows[i] / s), -127, 127).astype(np.int8)
                scales[pg, 0, sl] = s
                if codes is c.v:
                    codes[pg, 0, :, sl] = x
                else:
                    codes[pg, 0, sl] = x
    t = c.to_device()
    for split in (0, T):
        c.split_tokens = split
        check_attention(c, Attend(c, t, "f32")().read(), "f32")


@pytest.mark.parametrize("bits,heads,dim", [(4, 4, 128), (4, 16, 64), (4, 4, 256), (8, 8, 128)])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_head_that_is_not_finite_stays_alone(gpu, bits, heads, dim, value):
    """One query head with a NaN or an infinity: its own l and output are NaN, the
    other heads of its kv head are as without it.  Their scores are the same; their
    weights may be scaled at other tiles, 2^-19 of the largest value either way
    (check_attention)."""
    c = Case(bits, [900, 33], 1, heads, 1, dim, 16, seed=45, kind="f32")
    t = c.to_device()
    want = Attend(c, t, "f32")().read()
    t["q"].view(2, heads, dim)[0, 1, 5] = value
    got = Attend(c, t, "f32")().read()
    keep = np.ones((2, 1, heads), bool)
    keep[0, 0, 1] = False
    assert np.array_equal(want[0][keep], got[0][keep])
    assert np.all(np.abs(want[1] - got[1])[keep] <= 2.0 ** -19 * want[1][keep])
    top = max(np.abs(c.rows_of(b, "v")).max() for b in range(2))
    assert np.all(np.abs(want[2] - got[2])[keep] <= 2.0 ** -18 * top)
    assert np.isnan(got[1][0, 0, 1]) and np.isnan(got[2][0, 0, 1]).all()
