"""append_kv_i4 and read_kv on the GPU: the stored bits against an IEEE fp32
restatement, values against it in 64 bits rounded once, skipped and untouched
slots, strides, source and output types, non-finite blocks."""
import numpy as np
import pytest

import kvbridge_amd as kvb

from cache_forms import OUT, NP_SRC, Case, bf16_round, decode4, encode4

pytestmark = pytest.mark.gpu


def torch_type(kind):
    import torch

    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[kind]


CASES = [
    # tokens, kv_heads, dim, page, source, extra stride, output
    (1, 8, 128, 16, "bf16", 0, "f32"),
    (64, 8, 128, 16, "bf16", 4096, "bf16"),
    (77, 3, 64, 8, "f16", 0, "f16"),
    (300, 2, 256, 24, "f32", 0, "f32"),
    (129, 1, 128, 64, "f32", 5, "bf16"),   # rows off the 16-byte grid
    (1030, 2, 64, 40, "bf16", 3, "f32"),
    (515, 5, 256, 64, "f16", 8, "f32"),
]


def sources(tokens, kvh, dim, kind, extra, seed):
    """K, V rows [tokens, stride]: ordinary ones, zeros, constants, huge, tiny and outlying values."""
    import torch

    rng = np.random.default_rng(seed)
    rows = []
    for _ in range(2):
        x = rng.standard_normal((tokens, kvh * dim + extra)).astype(np.float32)
        x[0, :dim] = 0
        x[-1, :32] = 1.2345
        x[-1, 32:64] = -3.3
        x[tokens // 2, :kvh * dim] *= 1e-3
        x[tokens // 3, 5] = 300
        rows.append(torch.from_numpy(x).to(torch_type(kind)))
    return rows


@pytest.mark.parametrize("case", CASES)
def test_write_and_read(gpu, case):
    import torch

    tokens, kvh, D, P, kind, extra, out = case
    rng = np.random.default_rng(tokens)
    pages = -(-tokens // P) + 2
    slots = rng.permutation(pages * P)[:tokens].astype(np.uint32)
    if tokens > 20:
        slots[7], slots[11] = pages * P, 0xFFFFFFFF  # padding
    k, v = sources(tokens, kvh, D, kind, extra, tokens + D)
    pool = [rng.integers(0, 256, (pages, kvh, P, D // 2), dtype=np.uint8) for _ in range(2)] + \
           [rng.integers(0, 1 << 32, (pages, kvh, P, D // 32), dtype=np.uint32) for _ in range(2)]
    want = [a.copy() for a in pool]
    for i, src in ((0, k), (1, v)):
        codes, words = encode4(src.float().numpy()[:, :kvh * D].reshape(tokens, kvh, D))
        for t, s in enumerate(slots):
            if s < pages * P:
                want[i][s // P, :, s % P], want[2 + i][s // P, :, s % P] = codes[t], words[t]
    dev = [torch.from_numpy(a.view(np.int32) if a.dtype == np.uint32 else a).to(gpu) for a in pool]
    ds = torch.from_numpy(slots.view(np.int32)).to(gpu)
    shape = kvb.append_shape(tokens, kvh, D, P, pages, NP_SRC[kind], kvh * D + extra, kvh * D + extra)
    kvb.append_kv_i4(shape, k.to(gpu), v.to(gpu), ds, *dev)
    torch.cuda.synchronize()
    for name, g, w in zip(("k", "v", "k words", "v words"), dev, want):
        assert np.array_equal(g.cpu().numpy().view(w.dtype), w), name
    got = [torch.full((tokens, kvh, D), float("nan"), dtype=torch_type(out), device=gpu) for _ in range(2)]
    kvb.read_kv(kvb.read_shape(tokens, kvh, D, P, pages, 4, OUT[out]), ds, *dev, *got)
    torch.cuda.synchronize()
    for i in range(2):
        vals = np.zeros((tokens, kvh, D), np.float32)
        for t, s in enumerate(slots):
            if s < pages * P:
                vals[t] = decode4(want[i][s // P, :, s % P], want[2 + i][s // P, :, s % P]).astype(np.float32)
        assert torch.equal(got[i].cpu(), torch.from_numpy(vals).to(torch_type(out)))


def test_blocks_that_are_not_finite_or_extreme(gpu):
    import torch

    x = np.zeros((10, 64), np.float32)
    x[:, :32] = np.linspace(-1, 1, 32)
    x[0, 3] = np.nan
    x[1, 31] = np.inf
    x[2, 0] = -np.inf
    x[3, 9] = 3.4e38
    x[4, :32] = np.linspace(-3.4e38, 3.4e38, 32)  # the spread is past fp32
    x[5, :32] = -3.4028235e38                     # rounds past bfloat16
    x[6, :32] = np.linspace(0, 1e-37, 32)
    x[7, :32] = np.float32(1e-39)                 # subnormal
    x[8, :32] = -0.0
    x[9, :32] = np.float32(1 / 3)
    pool = [torch.zeros((2, 1, 8, 32), dtype=torch.uint8, device=gpu) for _ in range(2)] + \
           [torch.zeros((2, 1, 8, 2), dtype=torch.int32, device=gpu) for _ in range(2)]
    slots = torch.arange(10, dtype=torch.int32, device=gpu)
    src = torch.from_numpy(x).to(gpu)
    kvb.append_kv_i4(kvb.append_shape(10, 1, 64, 8, 2), src, src, slots, *pool)
    torch.cuda.synchronize()
    codes, words = encode4(x)
    for i in range(2):
        assert np.array_equal(pool[i].cpu().numpy().reshape(16, 32)[:10], codes)
        assert np.array_equal(pool[2 + i].cpu().numpy().view(np.uint32).reshape(16, 2)[:10], words)
    assert np.all(words[[0, 1, 2, 4, 5], 0] == 0x7FC07FC0) and np.all(words[:, 1] == 0)
    # a value is off by at most half a step and the parameters' own rounding (2^-8 of them, 15 steps)
    fine = decode4(codes, words)[[6, 9]][:, :32]
    assert np.all(np.abs(fine - x[[6, 9], :32]) <= np.abs(x[[6, 9], :32]).max() / 15)


@pytest.mark.parametrize("dim,page,out", [(64, 16, "f32"), (128, 24, "bf16"), (256, 64, "f16")])
def test_read_int8(gpu, dim, page, out):
    import torch

    case = Case(8, [130, 61], 1, 2, 2, dim, page, seed=1)
    t = case.to_device()
    rng = np.random.default_rng(5)
    slots = rng.permutation(case.pages * page)[:97].astype(np.uint32)
    slots[3] = case.pages * page
    ds = torch.from_numpy(slots.view(np.int32)).to(gpu)
    got = [torch.full((97, 2, dim), float("nan"), dtype=torch_type(out), device=gpu) for _ in range(2)]
    kvb.read_kv(kvb.read_shape(97, 2, dim, page, case.pages, 8, OUT[out]), ds, t["k"], t["v"], t["ks"], t["vs"], *got)
    torch.cuda.synchronize()
    for g, name in zip(got, "kv"):
        vals = case.pool_values(name).astype(np.float32)  # one product: rounded once
        want = np.stack([vals[s // page, :, s % page] if s < case.pages * page else np.zeros((2, dim), np.float32) for s in slots])
        assert torch.equal(g.cpu(), torch.from_numpy(want).to(torch_type(out)))


def test_quantization_error_of_ordinary_rows():
    """The format's own error on N(0, 1) rows: half a step, and the rounding of step and least."""
    x = np.random.default_rng(0).standard_normal((64, 4, 128)).astype(np.float32)
    codes, words = encode4(x)
    y = decode4(codes, words)
    step = (words & np.uint32(0xFFFF0000)).view(np.float32)
    least = (words << np.uint32(16)).view(np.float32)
    # the top code falls short by up to 15 half steps of the step's rounding, 15 * 2^-9 of a step
    tol = np.repeat(step * (0.5 + 15 * 2.0 ** -8) + np.abs(least) * 2.0 ** -8, 32, axis=-1)
    assert np.all(np.abs(x - y) <= tol)
    assert np.array_equal(bf16_round(step), step)
