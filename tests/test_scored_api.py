"""Host-side contract of the calls on a 4- or 8-bit cache (no GPU): validation
order and messages, sizes, and argument rejection before any launch."""
import math

import pytest

import kvbridge_amd as kvb

FAKE = 0x1000


def shape(**chg):
    s = kvb.make_scored_shape(4, 1, 32, 8, 128, 64, 8192, 131072, 4 * 131072, 8192, 1 / math.sqrt(128), q_type=kvb.KVB_SRC_F16)
    return s.copy(**chg)


def given(**chg):
    names = ("q", "q_positions", "seq_starts", "page_offsets", "k_positions", "page_table", "k", "v", "k_scales", "v_scales")
    return kvb.scored_input(*(chg.get(n, FAKE) for n in names))


def test_valid_shapes_and_sizes():
    s = shape()
    assert kvb.scored_shape_error(s) is None
    n = kvb.scored_item_count(s)
    assert 4 <= n <= 4096
    assert kvb.scored_scratch_elements(s) == n * 32 * 130
    assert kvb.scored_counter_elements(s) == 4 * 8
    assert kvb.scored_counter_elements(s.copy(rows=5)) == 4 * 8 * 2  # 20 head-rows: two blocks of 16
    # with a split size: every sequence the splits of max_tokens
    assert kvb.scored_item_count(shape(split_tokens=2048)) == 4 * 64
    assert kvb.scored_item_count(shape(max_tokens=1)) == 4
    # a window bounds the tokens that are cut
    assert kvb.scored_item_count(shape(split_tokens=512, window=1000)) == 4 * -(-(1000 + 1 + 32 + 31) // 32 // 16)
    # more sequences than the kernel shares items out for
    assert kvb.scored_item_count(shape(batch=300, max_tokens=4000)) >= 300


@pytest.mark.parametrize("change,msg", [
    (dict(batch=0), "batch must be in [1,65535]"),
    (dict(batch=65536), "batch must be in [1,65535]"),
    (dict(rows=0), "rows and head counts must be positive"),
    (dict(kv_heads=0), "rows and head counts must be positive"),
    (dict(q_heads=60), "q_heads must be divisible by kv_heads"),
    (dict(kv_bits=3), "kv_bits must be 4 or 8"),
    (dict(dim=96), "dim must be 64, 128 or 256"),
    (dict(page_tokens=12), "page_tokens must be a positive multiple of 8"),
    (dict(page_tokens=0), "page_tokens must be a positive multiple of 8"),
    (dict(pages=0), "pages must be positive"),
    (dict(pages=1 << 30), "page and kv head product exceeds 32 bits"),
    (dict(max_tokens=0), "max_tokens must be in [1,2^31-1]"),
    (dict(max_tokens=1 << 31), "max_tokens must be in [1,2^31-1]"),
    (dict(max_tokens=8192 * 64 + 1), "tokens exceed allocated page capacity"),
    (dict(total_tokens=0), "total_tokens and table_entries must be positive"),
    (dict(table_entries=0), "total_tokens and table_entries must be positive"),
    (dict(split_tokens=33), "split_tokens must be a multiple of 32"),
    (dict(q_type=0), "unknown query element type"),
    (dict(q_stride=32 * 128 - 1), "row stride must cover q_heads * dim elements"),
    (dict(scale=float("nan")), "score scale must be finite"),
    (dict(cap=-1.0), "score cap must be finite and not negative"),
    (dict(cap=float("inf")), "score cap must be finite and not negative"),
    (dict(rows=1 << 20), "batch row/head product exceeds the grid limit"),
    (dict(pages=1 << 20, max_tokens=1 << 26, split_tokens=32), "split count exceeds 65535"),
    (dict(batch=65535, rows=8, split_tokens=32), "split and head product exceeds the grid limit"),
])
def test_scored_rejections_in_order(change, msg):
    s = shape(**change)
    assert kvb.scored_shape_error(s) == msg
    for f in (kvb.scored_item_count, kvb.scored_scratch_elements, kvb.scored_counter_elements):
        with pytest.raises(kvb.KvbInvalidArgument) as e:
            f(s)
        assert str(e.value) == msg


def test_scored_calls_rejected_before_launch():
    s = shape()

    def call(s=s, inp=None, scratch=FAKE, m=FAKE, l=FAKE, out=FAKE, kind=kvb.KVB_OUT_F16):
        kvb.decode_attention_scored(s, inp or given(), scratch, m, l, out, kind, stream=0)

    bad = [
        (dict(scratch=None), "scratch, m, l and out"),
        (dict(m=None), "scratch, m, l and out"),
        (dict(l=None), "scratch, m, l and out"),
        (dict(out=None), "scratch, m, l and out"),
        (dict(inp=given(seq_starts=None)), "attention input device buffers"),
        (dict(inp=given(q=FAKE + 1)), "aligned to their element size"),
        (dict(inp=given(v=None)), "cache buffers must be non-null"),
        (dict(inp=given(k=FAKE + 8)), "16-byte aligned"),
        (dict(inp=given(k_scales=FAKE + 4)), "cache scales must be aligned"),
        (dict(kind=kvb.KVB_OUT_NONE), "unknown output type"),
        (dict(kind=7), "unknown output type"),
        (dict(out=FAKE + 2), "16-byte aligned"),
        (dict(s=shape(batch=0)), "batch must be"),
    ]
    for args, msg in bad:
        with pytest.raises(kvb.KvbInvalidArgument, match=msg):
            call(**args)
    for args, msg in [(dict(m=None), "m, l and weights"), (dict(w=None), "m, l and weights"),
                      (dict(inp=given(k=None, v=None)), "cache buffers"), (dict(s=shape(dim=65)), "dim must be")]:
        a = {"s": s, "inp": given(v=None, v_scales=None), "m": FAKE, "w": FAKE, **args}
        with pytest.raises(kvb.KvbInvalidArgument, match=msg):
            kvb.accumulate_weights(a["s"], a["inp"], a["m"], FAKE, a["w"], 0, stream=0)


@pytest.mark.parametrize("change,msg", [
    (dict(dim=32), "dim must be 64, 128 or 256"),
    (dict(page_tokens=4), "page_tokens must be a positive multiple of 8"),
    (dict(kv_heads=0), "kv_heads must be in [1,65535]"),
    (dict(src_type=9), "unknown source element type"),
    (dict(k_stride=1023), "token stride must cover kv_heads * dim elements"),
    (dict(tokens=1 << 31), "token and kv head product exceeds the grid limit"),
])
def test_append_rejections(change, msg):
    s = kvb.append_shape(64, 8, 128, 16, 100, kvb.KVB_SRC_BF16)
    assert kvb.append_i4_shape_error(s) is None
    for k, v in change.items():
        setattr(s, k, v)
    assert kvb.append_i4_shape_error(s) == msg


def test_append_and_read_rejected_before_launch():
    s = kvb.append_shape(64, 8, 128, 16, 100, kvb.KVB_SRC_BF16)
    ok = [FAKE] * 7
    for i, x, msg in [(0, None, "append buffers"), (2, None, "append buffers"), (3, None, "cache buffers"),
                      (0, FAKE + 1, "aligned to their element size"), (4, FAKE + 4, "16-byte aligned"),
                      (5, FAKE + 8, "cache scales must be aligned")]:
        a = list(ok)
        a[i] = x
        with pytest.raises(kvb.KvbInvalidArgument, match=msg):
            kvb.append_kv_i4(s, *a, stream=0)
    s.tokens = 0
    kvb.append_kv_i4(s, *[None] * 7, stream=0)  # nothing to write
    r = kvb.read_shape(10, 8, 128, 16, 100, 4, kvb.KVB_OUT_F16)
    assert kvb.read_shape_error(r) is None
    for i, x, msg in [(0, None, "read buffers"), (5, None, "read buffers"), (1, None, "cache buffers"), (6, FAKE + 8, "16-byte aligned")]:
        a = list(ok)
        a[i] = x
        with pytest.raises(kvb.KvbInvalidArgument, match=msg):
            kvb.read_kv(r, *a, stream=0)
    for name, x, msg in [("kv_bits", 5, "kv_bits must be 4 or 8"), ("out_type", 0, "unknown output type"),
                         ("page_tokens", 9, "page_tokens must be"), ("tokens", 0xFFFFFFFF, "grid limit")]:
        bad = kvb.read_shape(10, 8, 128, 16, 100, 4, kvb.KVB_OUT_F16)
        setattr(bad, name, x)
        assert msg in kvb.read_shape_error(bad)


@pytest.mark.parametrize("change,msg", [
    (dict(batch=0), "batch must be in [1,65535]"),
    (dict(kv_bits=16), "kv_bits must be 4 or 8"),
    (dict(max_tokens=0), "max_tokens must be in [1,2^31-1]"),
    (dict(dst_entries=0), "total_tokens, table_entries and dst_entries must be positive"),
    (dict(keep=0), "keep must be in [1,2^30]"),
    (dict(sink=60, recent=41), "sink and recent exceed keep"),
    (dict(sink=0xFFFFFFFF, recent=0xFFFFFFFF), "sink and recent exceed keep"),
    (dict(keep=1 << 30, batch=8), "batch and keep product exceeds 32 bits"),
])
def test_evict_rejections(change, msg):
    s = kvb.make_evict_shape(2, 8, 128, 16, 500, 4000, 8000, 500, 100, 100, 4, 20)
    assert kvb.evict_shape_error(s) is None and kvb.evict_scratch_elements(s) >= 2 * 4000
    s = s.copy(**change)
    assert kvb.evict_shape_error(s) == msg
    with pytest.raises(kvb.KvbInvalidArgument):
        kvb.evict_scratch_elements(s)


def test_evict_calls_rejected_before_launch():
    s = kvb.make_evict_shape(2, 8, 128, 16, 500, 4000, 8000, 500, 100, 100, 4, 20)
    inp = kvb.evict_input(FAKE, FAKE, FAKE, FAKE)
    with pytest.raises(kvb.KvbInvalidArgument, match="eviction buffers"):
        kvb.evict_select(s, inp, None, FAKE, FAKE, FAKE, stream=0)
    with pytest.raises(kvb.KvbInvalidArgument, match="eviction buffers"):
        kvb.evict_select(s, kvb.evict_input(FAKE, None, FAKE, None), FAKE, FAKE, FAKE, FAKE, stream=0)
    with pytest.raises(kvb.KvbInvalidArgument, match="16-byte aligned"):
        kvb.evict_select(s, inp, FAKE, FAKE + 4, FAKE, FAKE, stream=0)
    cache = [FAKE] * 8
    for i, x, msg in [(5, None, "eviction buffers"), (6, None, "eviction buffers"), (1, None, "cache buffers"),
                      (0, FAKE + 2, "16-byte aligned"), (3, FAKE + 4, "cache scales")]:
        a = list(cache)
        a[i] = x
        with pytest.raises(kvb.KvbInvalidArgument, match=msg):
            kvb.evict_move(s, inp, kvb.evict_cache(*a), FAKE, FAKE, stream=0)
    with pytest.raises(kvb.KvbInvalidArgument, match="positions need k_positions"):
        kvb.evict_move(s, kvb.evict_input(FAKE, FAKE, FAKE, None), kvb.evict_cache(*cache), FAKE, FAKE, stream=0)
