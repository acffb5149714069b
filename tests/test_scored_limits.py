"""Grid limits of the scored attention (no GPU): threads of a launch are counted
in 32 bits, with as many waves per work-group as the call would launch."""
import kvbridge_amd as kvb


def test_threads_of_a_launch_fit_32_bits():
    # 16 kv heads x 4,096 blocks of 16 head-rows x 100 items of eight or more waves
    s = kvb.make_scored_shape(1, 65536, 16, 16, 128, 32, 1 << 20, 512 * 100, 512 * 100, 1600, 0.1, split_tokens=512)
    assert kvb.scored_shape_error(s) == "split and head product exceeds the grid limit"
    assert kvb.scored_shape_error(s.copy(split_tokens=51200)) is None


def test_sizes_follow_the_splits():
    for bits in (4, 8):
        for dim in (64, 128, 256):
            for page in (8, 32):
                s = kvb.make_scored_shape(1, 1, 8, 8, dim, page, 1 << 17, 1 << 17, 1 << 17, 1 << 17, 0.1, kv_bits=bits)
                n = kvb.scored_item_count(s)
                assert 1 <= n <= 256 and kvb.scored_scratch_elements(s) == n * 8 * (dim + 2)


def test_work_groups_of_an_eviction():
    s = kvb.make_evict_shape(65535, 8, 128, 16, 500, 1 << 20, 8000, 500, 100, 100, 4, 20)
    assert kvb.evict_shape_error(s) is None
    assert kvb.evict_shape_error(s.copy(max_tokens=(1 << 31) - 1)) == "batch, tokens and heads exceed the grid limit"
    wide = kvb.make_evict_shape(4096, 4096, 64, 8, 1000, 1 << 20, 8000, 500, 100, 1 << 19, 4, 20)
    assert kvb.evict_shape_error(wide) == "batch, tokens and heads exceed the grid limit"
    assert kvb.evict_shape_error(wide.copy(keep=4096)) is None
