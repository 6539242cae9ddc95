"""Ciphertexts held in fewer bits and contractions with 4-bit weights.  Everything is integer
arithmetic mod 2^64, so every word must equal the plain restatement here (numpy u64 and the CPU
oracle's contraction)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

MARK = 0x5A5A5A5A5A5A5A5A  # what untouched words hold


def words(rng, *shape):
    return rng.integers(0, 1 << 64, shape, dtype=np.uint64)


def dev(a):
    a = np.ascontiguousarray(a)
    return torch.tensor(a.view(np.int64) if a.dtype == np.uint64 else a, device="cuda")


def host(t):
    return t.cpu().numpy().view(np.uint64)


def marked(*shape):
    return torch.full(shape, MARK, dtype=torch.int64, device="cuda")


def quantise(x, bits):
    return (x + np.uint64(1 << (63 - bits))) >> np.uint64(64 - bits)


def as_bytes(q, n):
    """u64 [.., L] below 2^(8n) as little-endian bytes [.., L * n]."""
    q = np.ascontiguousarray(q)
    return q.view(np.uint8).reshape(*q.shape, 8)[..., :n].reshape(*q.shape[:-1], -1)


def as_words(b, L, bits):
    """Cache rows [.., row_bytes] as u64 [.., L]."""
    n = bits // 8
    wide = np.zeros((*b.shape[:-1], L, 8), np.uint8)
    wide[..., 8 - n:] = b[..., :L * n].reshape(*b.shape[:-1], L, n)
    return wide.view(np.uint64)[..., 0]


def plain_write(cache, slots, X, L, bits):
    """What `cache` (uint8 [slots, features, row_bytes]) holds in its words afterwards."""
    out = cache.copy()
    for t, s in enumerate(slots):
        if 0 <= s < len(cache):
            out[s, :, :L * (bits // 8)] = as_bytes(quantise(X[t, :, :L], bits), bits // 8)
    return out[:, :, :L * (bits // 8)]


class Weights:
    """Random 4-bit weights, the matrix that they stand for, and the binding's object."""

    def __init__(self, pnb, rng, M, K, group, zeros=True, q=None, scales=None):
        G = -(-K // group)
        q = rng.integers(0, 16, (M, K)) if q is None else q
        s = rng.integers(-128, 128, (M, G)) if scales is None else scales
        # zero points' upper bits say nothing
        z = rng.integers(0, 256, (M, G)) if zeros else None
        at = np.arange(K) // group
        self.dense = s[:, at] * (q - ((z[:, at] & 15) if zeros else 8))
        packed = pnb.pack_int4(torch.tensor(q))
        if K % 2:  # so does the last nibble of an odd row
            packed[:, -1] |= torch.tensor(rng.integers(0, 16, M) << 4, dtype=torch.uint8)
        self.own = pnb.GroupWeights(packed.cuda(), dev(s.astype(np.int8)), group, K,
                                    dev(z.astype(np.uint8)) if zeros else None)


# ---- the cache ----------------------------------------------------------------------------------
ROWS = [  # features, L, ld
    (1, 1, 1), (1, 1, 2), (3, 2, 2), (2, 3, 5), (5, 4, 4), (3, 5, 6), (7, 15, 15), (2, 16, 16),
    (3, 17, 18), (2, 835, 835), (3, 835, 836), (1, 2048, 2048), (3, 2049, 2049), (4, 2049, 2050),
    (2, 2049, 2052), (2, 8193, 8193), (40, 33, 33), (513, 5, 5), (1, 511, 511), (2, 512, 513),
    (2, 513, 513), (1, 1 << 20, 1 << 20), (2, (1 << 20) - 1, (1 << 20) - 1),
]


@pytest.mark.parametrize("bits", [16, 24, 32])
@pytest.mark.parametrize("F,L,ld", ROWS)
def test_write_and_read(pnb, F, L, ld, bits):
    rng = np.random.default_rng(F * 7 + L * 3 + ld + bits)
    slots = np.array([3, -1, 0, 5, 8, 3, 7, -2147483648, 2147483647, 3], np.int32)
    X = words(rng, len(slots), F, ld)
    X[0] = (1 << 64) - 1  # rounds up, around to 0
    X[2, 0, 0] = (1 << (63 - bits)) - 1  # just below the first tie, and the tie itself
    X[3, 0, 0] = 1 << (63 - bits)
    cache = pnb.CiphertextCache(8, F, L, bits)
    before = rng.integers(0, 256, cache.data.shape, dtype=np.uint8)
    cache.data.copy_(torch.tensor(before))
    assert pnb.cache_write(cache, dev(X), dev(slots)) is cache
    got = cache.data.cpu().numpy()
    assert np.array_equal(got[:, :, :L * (bits // 8)], plain_write(before, slots, X, L, bits))
    # back, at the same pitch, with words behind L and unused tokens left as they were
    want = np.full((len(slots), F, ld), MARK, np.uint64)
    for t, s in enumerate(slots):
        if 0 <= s < 8:
            want[t, :, :L] = as_words(got[s], L, bits)
    out = marked(len(slots), F, ld)
    assert pnb.cache_read(cache, dev(slots), out=out) is out
    assert np.array_equal(host(out), want)
    packed = host(pnb.cache_read(cache, dev(slots)))
    used = (slots >= 0) & (slots < 8)
    assert packed.shape == (len(slots), F, L)
    assert np.array_equal(packed[used], want[used][:, :, :L])


@pytest.mark.parametrize("bits", [16, 24, 32])
def test_rounding_is_to_nearest(pnb, bits):
    rng = np.random.default_rng(bits)
    X = words(rng, 2, 3, 100)
    cache = pnb.CiphertextCache(2, 3, 100, bits)
    slots = dev(np.array([1, 0], np.int32))
    back = host(pnb.cache_read(pnb.cache_write(cache, dev(X), slots), slots))
    assert np.all(np.abs((X - back).view(np.int64)) <= 1 << (63 - bits))
    again = host(pnb.cache_read(pnb.cache_write(cache, dev(back), slots), slots))
    assert np.array_equal(back, again)  # what has been rounded stays


def test_the_last_of_many_tokens_with_one_slot_stays(pnb):
    rng = np.random.default_rng(1)
    T = 3000
    slots = rng.integers(-1, 5, T).astype(np.int32)
    X = words(rng, T, 2, 70)
    for bits in (16, 24, 32):
        cache = pnb.CiphertextCache(5, 2, 70, bits)
        pnb.cache_write(cache, dev(X), dev(slots))
        want = plain_write(np.zeros(cache.data.shape, np.uint8), slots, X, 70, bits)
        assert np.array_equal(cache.data.cpu().numpy()[:, :, :70 * bits // 8], want)


@pytest.mark.parametrize("rows,words", [(1, 1), (1, 5_000_001), (3, 2047), (2368, 2048),
                                        (3000, 2050), (70_000, 3)])
def test_zero_skipped(pnb, rows, words):
    rng = np.random.default_rng(rows + words)
    index = rng.integers(-1, 7, rows).astype(np.int32)
    index[0], index[-1] = -2147483648, 2147483647
    out = marked(rows + 1, words)  # (the last row is nobody's)
    i = dev(index)
    torch.cuda.synchronize()
    assert pnb.lib().pnb_zero_skipped(i.data_ptr(), rows, 5, out.data_ptr(), words, None) == 0
    torch.cuda.synchronize()
    want = marked(rows + 1, words)
    want[:rows][(i < 0) | (i >= 5)] = 0
    assert torch.equal(out, want)


@pytest.mark.parametrize("ld", [64, 65])
def test_results_made_here_hold_zeros_where_a_token_is_skipped(pnb, ld):
    rng = np.random.default_rng(15)
    F, L = 8, 64
    cache = pnb.CiphertextCache(4, F, L, 32)
    cache.data.copy_(torch.tensor(rng.integers(0, 256, cache.data.shape, dtype=np.uint8)))
    slots = dev(np.array([1, -1, 2, 9], np.int32))
    W = Weights(pnb, rng, F, F, F)
    route = pnb.expert_route(dev(np.array([[0], [-1], [1], [-1]], np.int32)), 2)
    X = dev(words(rng, 4, F, ld))
    We = torch.ones(2, F, F, dtype=torch.int8, device="cuda")
    for skipped, call in [
            ([1, 3], lambda **o: pnb.cache_read(cache, slots, ld=ld, **o)),
            ([1, 3], lambda **o: pnb.group_contract_cached(W.own, None, 0, cache, slots, ld=ld, **o)),
            ([2, 3], lambda **o: pnb.expert_dispatch(route, X, L, **o)),
            ([2, 3], lambda **o: pnb.expert_contract(route, We, None, 0, X, L, **o))]:
        want = marked(4, F, ld)
        call(out=want)
        assert bool((want[skipped] == MARK).all())
        want[skipped] = 0
        want[..., L:] = 0
        used = marked(4, F, ld)  # memory that the next buffer of its size gets
        del used
        assert torch.equal(call(), want)


def test_most_tokens(pnb):
    T = 65536
    X = torch.arange(T, device="cuda").view(T, 1, 1) << 40
    slots = torch.arange(T, device="cuda", dtype=torch.int32).flip(0)
    cache = pnb.cache_write(pnb.CiphertextCache(T, 1, 1, 32), X, slots)
    assert torch.equal(pnb.cache_read(cache, slots), X)


def test_offsets_past_32_bits(pnb):
    # slots at 6.6 GB of the cache, rows at 4.3 GB of the words
    cache = pnb.CiphertextCache(100, 8000, 2049, 32, data=torch.empty(
        100, 8000, 8208, dtype=torch.uint8, device="cuda"))
    X = torch.empty(35, 8000, 2049, dtype=torch.int64, device="cuda")
    X[0], X[34] = 0, 0
    X[34, 7999] = torch.arange(2049, device="cuda") << 35
    slots = torch.full((35,), -1, dtype=torch.int32, device="cuda")
    slots[34], slots[0] = 99, 0
    pnb.cache_write(cache, X, slots)
    X.fill_(MARK)
    pnb.cache_read(cache, slots, out=X)
    assert torch.equal(X[34, 7999], torch.arange(2049, device="cuda") << 35)
    assert not X[34, :7999].any() and not X[0].any() and bool((X[1:34] == MARK).all())
    W = Weights(pnb, np.random.default_rng(0), 16, 8000, 8000)
    Y = marked(35, 16, 2049)
    pnb.group_contract_cached(W.own, None, 0, cache, slots, out=Y)
    want = torch.tensor(W.dense[:, 7999:], device="cuda") * (torch.arange(2049, device="cuda") << 35)
    assert torch.equal(Y[34], want) and not Y[0].any() and bool((Y[1:34] == MARK).all())


# ---- contractions -------------------------------------------------------------------------------
SHAPES = [  # batch, K, M, group, L, ld
    (1, 1, 1, 1, 1, 1), (2, 1, 3, 5, 7, 7), (3, 2, 1, 1, 9, 10), (1, 31, 17, 8, 33, 34),
    (2, 33, 15, 16, 65, 65), (4, 64, 64, 64, 64, 64), (3, 65, 65, 32, 63, 66),
    (2, 130, 200, 32, 2049, 2049), (2, 130, 200, 32, 2049, 2050), (5, 128, 10, 48, 2049, 2050),
    (1, 784, 128, 128, 2049, 2050), (1, 784, 128, 784, 2049, 2049), (3, 257, 129, 17, 835, 836),
    (2, 257, 384, 48, 835, 835), (1, 1000, 40, 128, 8193, 8194), (1, 90, 70, 3, 8193, 8193),
    # last weight slots of 32 inputs and of more; on both sides of each way of computing
    (3, 32, 20, 32, 40, 41), (3, 160, 150, 16, 40, 42), (3, 161, 150, 16, 40, 40),
    (2, 384, 130, 64, 35, 36), (2, 384, 130, 64, 35, 35), (2, 385, 130, 64, 35, 36),
    (2, 385, 130, 64, 35, 35), (2, 896, 130, 896, 35, 36), (2, 897, 130, 16, 35, 36),
    (2, 128, 128, 16, 35, 36), (2, 129, 128, 16, 35, 36), (2, 128, 129, 16, 35, 36),
    (1, 24, 16, 8, 35, 36), (1, 25, 16, 8, 35, 36), (1, 100, 4800, 20, 20, 20),
    # enough tiles of X for a block to have all tiles of outputs
    (320, 130, 200, 32, 70, 71), (320, 130, 200, 32, 70, 72), (320, 30, 300, 7, 70, 70),
    (320, 257, 140, 48, 66, 66),
    # the longest ciphertexts
    (1, 3, 2, 2, 1 << 20, 1 << 20), (1, 40, 20, 16, 1 << 20, (1 << 20) + 1),
    (7, 16, 10, 16, 2049, 2049), (70, 40, 24, 8, 100, 100), (2, 2100, 66, 64, 70, 70),
    (2, 2100, 300, 100, 70, 72), (300, 16, 4, 16, 33, 34), (2, 300, 1000, 64, 40, 40),
]


def check(pnb, oracle, W, X, L, ld, rng, bias=None, transposed=False, out=None):
    B = len(X)
    w = W.dense.T if transposed else W.dense
    delta = 1 << 45
    want = np.full((B, len(w), ld), MARK, np.uint64)
    want[:, :, :L] = oracle.contract(np.ascontiguousarray(w), bias, delta,
                                     np.ascontiguousarray(X[:, :, :L]))
    got = marked(B, len(w), ld) if out is None else out
    pnb.group_contract(W.own, None if bias is None else dev(bias), delta, dev(X), L,
                       transposed=transposed, out=got)
    assert np.array_equal(host(got), want)
    assert pnb.device_status(0) == 0


@pytest.mark.parametrize("B,K,M,group,L,ld", SHAPES)
def test_contract(pnb, oracle, B, K, M, group, L, ld):
    rng = np.random.default_rng(B + K * 5 + M * 11 + L)
    W = Weights(pnb, rng, M, K, group, zeros=(B + K) % 2 == 0)
    bias = rng.integers(-1000, 1000, M) if M % 2 else None
    check(pnb, oracle, W, words(rng, B, K, ld), L, ld, rng, bias)


@pytest.mark.parametrize("B,K,M,group,L,ld", SHAPES)
def test_transposed(pnb, oracle, B, K, M, group, L, ld):
    rng = np.random.default_rng(B + K * 5 + M * 11 + L + 1)
    W = Weights(pnb, rng, M, K, group, zeros=(B + M) % 2 == 0)
    check(pnb, oracle, W, words(rng, B, M, ld), L, ld, rng, transposed=True)


@pytest.mark.parametrize("bits", [16, 24, 32])
@pytest.mark.parametrize("B,K,M,group,L,ld", SHAPES)
def test_cached(pnb, oracle, B, K, M, group, L, ld, bits):
    rng = np.random.default_rng(B + K * 5 + M * 11 + L + bits)
    W = Weights(pnb, rng, M, K, group, zeros=(B + K) % 2 == 0)
    bias = rng.integers(-1000, 1000, M) if M % 2 else None
    n = B + 2
    cache = pnb.CiphertextCache(n, K, L, bits)
    data = rng.integers(0, 256, cache.data.shape, dtype=np.uint8)  # padding that must not count
    cache.data.copy_(torch.tensor(data))
    slots = rng.permutation(n)[:B].astype(np.int32)
    if B > 2:
        slots[B // 2] = (-1, n, 2147483647)[B % 3]
        slots[0] = slots[-1]  # one slot for two requests
    want = np.full((B, M, ld), MARK, np.uint64)
    for b, s in enumerate(slots):
        if 0 <= s < n:
            want[b, :, :L] = oracle.contract(W.dense, bias, 3, as_words(data[s], L, bits)[None])[0]
    got = marked(B, M, ld)
    pnb.group_contract_cached(W.own, None if bias is None else dev(bias), 3, cache, dev(slots),
                              out=got)
    assert np.array_equal(host(got), want)
    assert pnb.device_status(0) == 0


@pytest.mark.parametrize("K,M", [(784, 128), (100, 200), (240, 130), (241, 130), (384, 70),
                                 (61440, 70)])
@pytest.mark.parametrize("sign", [1, -1])
def test_extreme_sums(pnb, K, M, sign):
    # every product as large as it can be: 128 * 15 times words of all ones
    q = np.full((M, K), 0 if sign > 0 else 15)
    W = Weights(pnb, np.random.default_rng(0), M, K, K, False, q, np.full((M, 1), -128))
    W.own.zeros = dev(np.full((M, 1), 15 if sign > 0 else 0, np.uint8))
    L = 40
    X = np.full((1, K, L), (1 << 64) - 1, np.uint64)
    want = -sign * 1920 * K  # times -1
    want = np.full((1, M, L), want % (1 << 64), np.uint64)
    assert np.array_equal(host(pnb.group_contract(W.own, None, 0, dev(X))), want)
    for bits in (16, 24, 32):
        cache = pnb.CiphertextCache(1, K, L, bits)
        cache.data.fill_(255)
        y = pnb.group_contract_cached(W.own, None, 0, cache, dev(np.zeros(1, np.int32)))
        assert np.array_equal(host(y), want << np.uint64(64 - bits))


def test_gradient_is_the_transpose(pnb):
    # <W x, g> = <x, W^T g> in every word, and a unit step of one input moves the outputs by its column
    rng = np.random.default_rng(2)
    W = Weights(pnb, rng, 21, 77, 16)
    x, g = words(rng, 1, 77, 9), words(rng, 1, 21, 9)
    y = host(pnb.group_contract(W.own, None, 0, dev(x)))
    dx = host(pnb.group_contract(W.own, None, 0, dev(g), transposed=True))
    g1, x1 = g[0, :, :1], x[0, :, :1]
    assert (y[0, :, 0] * g1[:, 0]).sum() == (x1[:, 0] * dx[0, :, 0]).sum()
    for i in (0, 40, 76):
        step = x.copy()
        step[0, i] += np.uint64(1)
        moved = host(pnb.group_contract(W.own, None, 0, dev(step))) - y
        assert np.array_equal(moved[0].view(np.int64), np.repeat(W.dense[:, i:i + 1], 9, 1))


@pytest.mark.parametrize("K,M", [(70, 90), (200, 150), (500, 90)])
@pytest.mark.parametrize("off_x,off_y,ldx,ldy", [
    (0, 0, 66, 66), (1, 0, 66, 66), (0, 1, 66, 66), (1, 1, 67, 67), (0, 0, 67, 66), (0, 0, 66, 67),
    (1, 0, 67, 70), (0, 1, 70, 65),
])
def test_every_alignment_through_the_c_abi(pnb, oracle, off_x, off_y, ldx, ldy, K, M):
    import ctypes as C
    rng = np.random.default_rng(off_x + 2 * off_y + 4 * ldx + ldy)
    B, L = 3, 65
    W = Weights(pnb, rng, M, K, 32)
    x = torch.zeros(B * K * ldx + 2, dtype=torch.int64, device="cuda")
    X = words(rng, B, K, ldx)
    x[off_x:off_x + X.size] = dev(X).reshape(-1)
    y = marked(B * M * ldy + 2)
    at = lambda t, off=0: C.c_void_p(t.data_ptr() + 8 * off)
    torch.cuda.synchronize()
    assert pnb.lib().pnb_group_contract(
        at(W.own.q), at(W.own.scales), at(W.own.zeros), 32, None, 0, M, K, 0, at(x, off_x), ldx,
        at(y, off_y), ldy, B, L, None, 0, None) == 0
    torch.cuda.synchronize()
    want = np.full((B, M, ldy), MARK, np.uint64)
    want[:, :, :L] = oracle.contract(W.dense, None, 0, np.ascontiguousarray(X[:, :, :L]))
    got = host(y)
    assert np.array_equal(got[off_y:off_y + want.size].reshape(want.shape), want)
    assert np.all(np.delete(got, np.s_[off_y:off_y + want.size]) == MARK)
    # (without a workspace of the caller's) and over a cache
    cache = pnb.CiphertextCache(B, K, L, 32)
    slots = dev(np.arange(B, dtype=np.int32))
    pnb.cache_write(cache, dev(X), slots)
    y.fill_(MARK)
    torch.cuda.synchronize()
    assert pnb.lib().pnb_group_contract_cached(
        at(W.own.q), at(W.own.scales), at(W.own.zeros), 32, None, 0, M, K, at(slots),
        at(cache.data), B, 32, at(y, off_y), ldy, B, L, None, 0, None) == 0
    torch.cuda.synchronize()
    want[:, :, :L] = oracle.contract(
        W.dense, None, 0, quantise(X[:, :, :L], 32) << np.uint64(32))
    got = host(y)
    assert np.array_equal(got[off_y:off_y + want.size].reshape(want.shape), want)
    assert np.all(np.delete(got, np.s_[off_y:off_y + want.size]) == MARK)


# Pairs of blocks (385 to 896 inputs, an even pitch) with 5 to 40 tiles a pair: the second accumulator, its
# hand-back across the blocks, and the inputs' slots from tile to tile.
PAIRED = [(12, 500, 140), (9, 385, 300), (10, 896, 128), (5, 784, 1000)]


@pytest.mark.parametrize("ldy", [2050, 2049])
@pytest.mark.parametrize("B,K,M", PAIRED)
def test_many_tiles_of_a_pair(pnb, oracle, B, K, M, ldy):
    import ctypes as C
    rng = np.random.default_rng(B + K + M)
    L, ldx = 2049, 2050
    W = Weights(pnb, rng, M, K, 64)
    X = words(rng, B, K, ldx)
    bias = rng.integers(-1000, 1000, M)
    x, y, b = dev(X), marked(B, M, ldy), dev(bias)
    at = lambda t: C.c_void_p(t.data_ptr())
    torch.cuda.synchronize()
    assert pnb.lib().pnb_group_contract(
        at(W.own.q), at(W.own.scales), at(W.own.zeros), 64, at(b), 1 << 45, M, K, 0, at(x), ldx, at(y),
        ldy, B, L, None, 0, None) == 0
    torch.cuda.synchronize()
    want = np.full((B, M, ldy), MARK, np.uint64)
    want[:, :, :L] = oracle.contract(W.dense, bias, 1 << 45, np.ascontiguousarray(X[:, :, :L]))
    assert np.array_equal(host(y), want)
    # and transposed, from as many inputs
    T = Weights(pnb, rng, K, M, 64)
    check(pnb, oracle, T, X, L, ldx, rng, transposed=True)


@pytest.mark.parametrize("bits", [16, 24, 32])
@pytest.mark.parametrize("B,K,M", PAIRED)
@pytest.mark.parametrize("ld", [2050, 2049])
def test_many_tiles_of_a_pair_over_a_cache(pnb, oracle, B, K, M, bits, ld):
    rng = np.random.default_rng(B + K + M + bits)
    B, L = 3 * B, 2049
    W = Weights(pnb, rng, M, K, 48)
    cache = pnb.CiphertextCache(2 * B, K, L, bits)
    cache.data.copy_(torch.randint(0, 256, cache.data.shape, dtype=torch.uint8,
                                   generator=torch.Generator().manual_seed(bits)))
    slots = rng.permutation(2 * B)[:B].astype(np.int32)
    slots[1::4] = -1
    slots[2::8] = 2 * B
    bias = rng.integers(-1000, 1000, M)
    got = marked(B, M, ld)
    pnb.group_contract_cached(W.own, dev(bias), 3, cache, dev(slots), out=got)
    used = np.flatnonzero((slots >= 0) & (slots < 2 * B))
    x = as_words(cache.data[slots[used].astype(np.int64)].cpu().numpy(), L, bits)
    want = np.full((B, M, ld), MARK, np.uint64)
    want[used, :, :L] = oracle.contract(W.dense, bias, 3, x)
    assert np.array_equal(host(got), want)
    assert pnb.device_status(0) == 0


def test_pairs_captured_and_in_one_workspace(pnb, oracle):
    import ctypes as C
    rng = np.random.default_rng(16)
    B, K, M, L, ld = 6, 700, 140, 2049, 2050
    W = [Weights(pnb, rng, M, K, 64) for _ in range(2)]
    X = words(rng, B, K, ld)
    x = dev(X)
    y = [marked(B, M, ld) for _ in range(2)]
    at = lambda t: C.c_void_p(t.data_ptr())

    def wanted(X):
        want = np.full((2, B, M, ld), MARK, np.uint64)
        for i in range(2):
            want[i, :, :, :L] = oracle.contract(W[i].dense, None, 0, np.ascontiguousarray(X[:, :, :L]))
        return want

    # one call after the other in one workspace
    ws = torch.empty(2 * M * ((K + 15) & -16), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    for _ in range(3):
        for w, out in zip(W, y):
            assert pnb.lib().pnb_group_contract(
                at(w.own.q), at(w.own.scales), at(w.own.zeros), 64, None, 0, M, K, 0, at(x), ld,
                at(out), ld, B, L, at(ws), ws.numel(), None) == 0
    torch.cuda.synchronize()
    assert np.array_equal(np.stack([host(t) for t in y]), wanted(X))
    # two graphs of a call each, replayed in turn with new inputs
    graphs = []
    for w, out in zip(W, y):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            pnb.group_contract(w.own, None, 0, x, L, out=out)
    for _ in range(3):
        X = words(rng, B, K, ld)
        x.copy_(dev(X))
        for t in y:
            t.fill_(MARK)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(np.stack([host(t) for t in y]), wanted(X))
    assert pnb.device_status(0) == 0


# ---- together, as a server uses them ------------------------------------------------------------
def test_layers_over_a_cache_decrypt(pnb):
    # two requests' encrypted inputs are kept in 32 bits, go through a 4-bit layer from the cache and
    # through another from words, and decrypt to the integers
    rng = np.random.default_rng(5)
    keys = pnb.keygen(seed=11)
    K, H, M = 36, 12, 4
    x = rng.integers(0, 4, (2, K))
    W1 = Weights(pnb, rng, H, K, 16, False, rng.integers(7, 10, (H, K)), rng.integers(1, 4, (H, 3)))
    W2 = Weights(pnb, rng, M, H, 4, False, rng.integers(7, 10, (M, H)), rng.integers(1, 3, (M, 3)))
    scale = 1 << 46
    ct = pnb.encrypt(keys, torch.tensor(x.reshape(-1)), seed=3, delta=scale).view(2, K, -1)
    L = ct.shape[2]
    cache = pnb.CiphertextCache(5, K, L, 32)
    slots = dev(np.array([4, 1], np.int32))
    pnb.cache_write(cache, ct, slots)
    b1 = rng.integers(-50, 50, H)
    h = pnb.group_contract_cached(W1.own, dev(b1), scale, cache, slots)
    y = pnb.group_contract(W2.own, None, 0, h)
    want = (x @ W1.dense.T + b1) @ W2.dense.T
    ph = pnb.phase(keys, y.reshape(-1, L)).cpu().numpy().astype(np.int64).reshape(2, M)
    # rounding moves a phase by 2^35.2 (standard deviation); the layers multiply that by the norms of
    # the products' rows
    norm = np.linalg.norm(W2.dense @ W1.dense, axis=1).max()
    assert 8 * norm * 2 ** 35.2 < scale / 2
    assert np.array_equal((ph + scale // 2) >> 46, want)
    g = pnb.group_contract(W1.own, None, 0, pnb.group_contract(W2.own, None, 0, y, transposed=True),
                           transposed=True)
    assert g.shape == ct.shape
    keys.free()


@pytest.mark.parametrize("K,M", [(150, 140), (500, 140), (90, 500), (1000, 60)])
def test_on_another_stream_and_captured(pnb, oracle, K, M):
    rng = np.random.default_rng(6)
    B, L = 3, 2049
    W = Weights(pnb, rng, M, K, 32)
    X = words(rng, B, K, L)
    slots = dev(np.array([2, 0, 1], np.int32))
    cache = pnb.CiphertextCache(3, K, L, 24)
    x, y, z, r, g = dev(X), marked(B, M, L), marked(B, M, L), marked(B, K, L), marked(B, K, L)

    def run():
        pnb.cache_write(cache, x, slots)
        pnb.group_contract(W.own, None, 0, x, out=y)
        pnb.group_contract_cached(W.own, None, 0, cache, slots, out=z)
        pnb.cache_read(cache, slots, out=r)
        pnb.group_contract(W.own, None, 0, y, transposed=True, out=g)

    def check_all(X):
        back = quantise(X, 24) << np.uint64(40)
        want = oracle.contract(W.dense, None, 0, X)
        assert np.array_equal(host(y), want)
        assert np.array_equal(host(z), oracle.contract(W.dense, None, 0, back))
        assert np.array_equal(host(r), back)
        assert np.array_equal(host(g), oracle.contract(np.ascontiguousarray(W.dense.T), None, 0, want))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    side.synchronize()
    check_all(X)
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    for graph in graphs:
        with torch.cuda.graph(graph):
            run()
    for i in range(3):
        X = words(rng, B, K, L)
        x.copy_(dev(X))
        for t in (y, z, r, g):
            t.fill_(0)
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        check_all(X)


@pytest.mark.parametrize("K", [100, 500, 1000])
def test_two_host_threads(pnb, oracle, K):
    import threading
    rng = np.random.default_rng(7)
    W = [Weights(pnb, rng, 130, K, 32) for _ in range(2)]
    X = [words(rng, 2, K, 300) for _ in range(2)]
    got = [[], []]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            x = dev(X[i])
            for _ in range(20):
                got[i].append(pnb.group_contract(W[i].own, None, 0, x))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(2):
        want = oracle.contract(W[i].dense, None, 0, X[i])
        assert len(got[i]) == 20 and all(np.array_equal(host(y), want) for y in got[i])


def test_weights_at_any_address_and_other_types_of_words(pnb, oracle):
    import ctypes as C
    rng = np.random.default_rng(12)
    K, M, L = 160, 70, 40
    W = Weights(pnb, rng, M, K, 32)
    X = words(rng, 2, K, L)
    want = oracle.contract(W.dense, None, 0, X)
    # unsigned words, and inputs that are a view
    x = dev(X)
    assert np.array_equal(host(pnb.group_contract(W.own, None, 0, x.view(torch.uint64))), want)
    wide = torch.zeros(2, 2 * K, L, dtype=torch.int64, device="cuda")
    wide[:, ::2] = x
    assert np.array_equal(host(pnb.group_contract(W.own, None, 0, wide[:, ::2])), want)
    # packed weights, scales and zero points that start anywhere
    for off in (1, 2, 3):
        at = []
        for t in (W.own.q, W.own.scales, W.own.zeros):
            moved = torch.zeros(t.numel() + 4, dtype=t.dtype, device="cuda")
            moved[off:off + t.numel()] = t.reshape(-1)
            at.append(moved)
        y = marked(2, M, L)
        torch.cuda.synchronize()
        assert pnb.lib().pnb_group_contract(
            *(C.c_void_p(t.data_ptr() + off) for t in at), 32, None, 0, M, K, 0,
            C.c_void_p(x.data_ptr()), L, C.c_void_p(y.data_ptr()), L, 2, L, None, 0, None) == 0
        torch.cuda.synchronize()
        assert np.array_equal(host(y), want)


@pytest.mark.parametrize("group", [41, (1 << 32) + 16, 1 << 40])
def test_a_group_past_the_inputs_is_one_group(pnb, oracle, group):
    rng = np.random.default_rng(14)
    W = Weights(pnb, rng, 20, 40, 40)
    wide = pnb.GroupWeights(W.own.q, W.own.scales, group, 40, W.own.zeros)
    X, G = words(rng, 2, 40, 30), words(rng, 2, 20, 30)
    assert np.array_equal(host(pnb.group_contract(wide, None, 0, dev(X))),
                          oracle.contract(W.dense, None, 0, X))
    assert np.array_equal(host(pnb.group_contract(wide, None, 0, dev(G), transposed=True)),
                          oracle.contract(np.ascontiguousarray(W.dense.T), None, 0, G))


def test_calls_one_after_the_other_in_one_workspace(pnb, oracle):
    # the second call's weights are laid out only when the first is done with its own
    import ctypes as C
    rng = np.random.default_rng(13)
    K, M, L = 700, 100, 2049
    W = [Weights(pnb, rng, M, K, 64) for _ in range(2)]
    X = words(rng, 4, K, L)
    x = dev(X)
    ws = torch.empty(2 * M * ((K + 15) & -16), dtype=torch.uint8, device="cuda")
    y = [marked(4, M, L) for _ in range(2)]
    at = lambda t: C.c_void_p(t.data_ptr())
    torch.cuda.synchronize()
    for _ in range(3):
        for w, out in zip(W, y):
            assert pnb.lib().pnb_group_contract(
                at(w.own.q), at(w.own.scales), at(w.own.zeros), 64, None, 0, M, K, 0, at(x), L,
                at(out), L, 4, L, at(ws), ws.numel(), None) == 0
    torch.cuda.synchronize()
    for w, out in zip(W, y):
        assert np.array_equal(host(out), oracle.contract(w.dense, None, 0, X))


def test_refusals_on_the_device(pnb):
    rng = np.random.default_rng(8)
    W = Weights(pnb, rng, 6, 5, 4)
    X = torch.zeros(4, 5, 10, dtype=torch.int64, device="cuda")
    G = torch.zeros(4, 6, 10, dtype=torch.int64, device="cuda")
    bias = torch.zeros(6, dtype=torch.int64, device="cuda")
    cache = pnb.CiphertextCache(3, 5, 10, 32)
    slots = torch.zeros(4, dtype=torch.int32, device="cuda")
    for bad, err in [
            (lambda: pnb.group_contract(W.own, None, 0, G), ValueError),
            (lambda: pnb.group_contract(W.own, None, 0, X, transposed=True), ValueError),
            (lambda: pnb.group_contract(W.own, bias, 0, G, transposed=True), ValueError),
            (lambda: pnb.group_contract(W.own, bias[:5], 0, X), ValueError),
            (lambda: pnb.group_contract(W.own, bias.int(), 0, X), TypeError),
            (lambda: pnb.group_contract(W.own, bias.cpu(), 0, X), ValueError),
            (lambda: pnb.group_contract(W.own, None, 0, X, 11), ValueError),
            (lambda: pnb.group_contract(W.own, None, 0, X, out=X), ValueError),
            (lambda: pnb.group_contract(W.own, None, 0, X, out=G[:, :, :9]), ValueError),
            (lambda: pnb.cache_write(cache, X[:3], slots), ValueError),
            (lambda: pnb.cache_write(cache, G, slots), ValueError),
            (lambda: pnb.cache_write(cache, X[:, :, :9], slots), ValueError),
            (lambda: pnb.cache_write(cache, X, slots.long()), TypeError),
            (lambda: pnb.cache_write(cache, X, slots.cpu()), ValueError),
            (lambda: pnb.cache_read(cache, slots, ld=9), ValueError),
            (lambda: pnb.cache_read(cache, slots, ld=11, out=X), ValueError),
            (lambda: pnb.cache_read(cache, slots, out=G), ValueError),
            (lambda: pnb.group_contract_cached(W.own, None, 0, cache, slots, out=X), ValueError),
            (lambda: pnb.group_contract_cached(W.own, bias[:3], 0, cache, slots), ValueError),
    ]:
        with pytest.raises(err):
            bad()
    whole = torch.zeros(3 * 5 * 48 // 8, dtype=torch.int64, device="cuda")
    inside = pnb.CiphertextCache(3, 5, 10, 32, data=whole.view(torch.uint8).view(3, 5, 48))
    with pytest.raises(ValueError, match="overlaps"):
        pnb.cache_write(inside, whole[:50].view(1, 5, 10), slots[:1])
    with pytest.raises(ValueError, match="overlaps"):
        pnb.cache_read(inside, slots[:1], out=whole[40:90].view(1, 5, 10))
    with pytest.raises(ValueError, match="overlaps"):
        pnb.group_contract_cached(W.own, None, 0, inside, slots[:1], out=whole[:60].view(1, 6, 10))


def test_nothing(pnb):
    W = Weights(pnb, np.random.default_rng(9), 6, 5, 4)
    X = torch.zeros(0, 5, 10, dtype=torch.int64, device="cuda")
    cache = pnb.CiphertextCache(3, 5, 10, 32)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert pnb.group_contract(W.own, None, 0, X).shape == (0, 6, 10)
    assert pnb.cache_read(pnb.cache_write(cache, X, none), none).shape == (0, 5, 10)
    assert pnb.group_contract_cached(W.own, None, 0, cache, none, ld=12).shape == (0, 6, 12)
