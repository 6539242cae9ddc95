"""Per-request contractions with every word of every row compared: calls of many rows, in which a
block walks through many groups, slots and turns.  The plain form runs on the GPU: 16-bit limbs of the
words as doubles, whose products with int8 weights stay below 2^53 and so are whole numbers."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

MARK = 0x5A5A5A5A5A5A5A5A  # what untouched words hold


def source(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def words(g, *shape):
    return torch.randint(-(1 << 63), (1 << 63) - 1, shape, dtype=torch.int64, device="cuda",
                         generator=g)


def weights(g, *shape):
    return torch.randint(-128, 128, shape, dtype=torch.int8, device="cuda", generator=g)


def bias_of(g, *shape):
    return torch.randint(-(1 << 40), 1 << 40, shape, device="cuda", generator=g)


def times(W, X):
    """W [.., M, K] (int8) times X [.., K, L] mod 2^64."""
    w, y = W.double(), 0
    for i in range(4):
        limb = ((X >> (16 * i)) & 0xFFFF).double()
        y = y + (torch.matmul(w, limb).long() << (16 * i))
    return y


def rows_of(ids, E):
    """The choices of the rows: used ones by expert, ties in order."""
    flat = ids.reshape(-1).long()
    used = torch.nonzero((flat >= 0) & (flat < E)).reshape(-1)
    return used[torch.sort(flat[used], stable=True).indices]


def check_experts(pnb, ids, W, bias, delta, X, L, sorted_rows=False, step=64):
    """Runs the contraction and compares all of its output with the plain form."""
    E, M, _ = W.shape
    n, ld = ids.numel(), X.shape[2]
    out = torch.full((n, M, ld), MARK, dtype=torch.int64, device="cuda")
    pnb.expert_contract(pnb.expert_route(ids, E), W, bias, delta, X, L, sorted_rows=sorted_rows,
                        out=out)
    choice = rows_of(ids, E)
    for r in range(0, len(choice), step):
        c = choice[r:r + step]
        e = ids.reshape(-1)[c].long()
        want = times(W[e], X[r:r + len(c), :, :L] if sorted_rows else X[c // ids.shape[1], :, :L])
        if bias is not None:
            want[:, :, -1] += bias[e] * delta
        assert torch.equal(out[r:r + len(c), :, :L], want), r
    assert bool((out[:, :, L:] == MARK).all()) and bool((out[len(choice):] == MARK).all())
    assert pnb.device_status(0) == 0


def check_adapters(pnb, W, bias, delta, A, B, which, X, L, shift, step=64):
    n, M, ld = A.shape[0], W.shape[0], X.shape[2]
    out = torch.full((X.shape[0], M, ld), MARK, dtype=torch.int64, device="cuda")
    pnb.adapter_contract(W, bias, delta, A, B, which, X, L, base_shift=shift, out=out)
    for b in range(0, X.shape[0], step):
        x, a = X[b:b + step, :, :L], which[b:b + step].long()
        has = ((a >= 0) & (a < n)).view(-1, 1, 1)
        a = a.clamp(0, n - 1)
        want = (times(W, x) << shift) + torch.where(has, times(B[a], times(A[a], x)), 0)
        if bias is not None:
            want[:, :, -1] += bias * delta
        assert torch.equal(out[b:b + step, :, :L], want), b
    assert bool((out[:, :, L:] == MARK).all())
    assert pnb.device_status(0) == 0


def which_of(g, batch, n, without):
    """Adapters of the requests: runs of those without one between others, all of them, or none."""
    a = torch.randint(0, n, (batch,), dtype=torch.int32, device="cuda", generator=g)
    if without == "runs":
        a[(torch.arange(batch, device="cuda") // 9) % 2 == 1] = -1
    elif without == "all":
        a.fill_(-1)
    return a


# ---- rows at an odd pitch -----------------------------------------------------------------------
# A raw slot holds 32 rows of X (64 beside adapters), an operand slot two of them, and four warps take
# the raw slots in turn: from one raw slot, which leaves three warps idle, to several operand slots.
@pytest.mark.parametrize("K", [25, 32, 33, 64, 65, 97, 129, 200])
@pytest.mark.parametrize("M,L,T,k", [(40, 257, 150, 2), (140, 70, 130, 3)])
def test_experts_at_an_odd_pitch(pnb, K, M, L, T, k):
    g = source(K + M)
    E, ld = 5, L | 1
    ids = torch.randint(-1, E, (T, k), dtype=torch.int32, device="cuda", generator=g)
    check_experts(pnb, ids, weights(g, E, M, K), bias_of(g, E, M), (1 << 45) + 3,
                  words(g, T, K, ld), L)
    check_experts(pnb, ids, weights(g, E, M, K), None, 0, words(g, T * k, K, ld), L, sorted_rows=True)


@pytest.mark.parametrize("K", [33, 64, 65, 128, 129, 300])
@pytest.mark.parametrize("without", ["no", "runs", "all"])
@pytest.mark.parametrize("M,rank,L,batch", [(60, 17, 257, 150), (260, 40, 70, 150)])
def test_adapters_at_an_odd_pitch(pnb, K, without, M, rank, L, batch):
    g = source(K + M + rank)
    n, ld = 4, L | 1
    check_adapters(pnb, weights(g, M, K), bias_of(g, M), (1 << 45) + 3,
                   weights(g, n, rank, K), weights(g, n, M, rank), which_of(g, batch, n, without),
                   words(g, batch, K, ld), L, 6)


# ---- requests without an adapter, and several tiles to a group ------------------------------------
# The warps that issue a tile's products must stay in step also over tiles for which one of them
# issues nothing: those of requests without an adapter, and a group's second and later tiles.
@pytest.mark.parametrize("K,M", [(128, 33), (48, 130), (200, 128), (64, 300), (128, 700)])
@pytest.mark.parametrize("without", ["no", "runs", "all"])
@pytest.mark.parametrize("rank,L", [(17, 258), (64, 70)])
def test_adapters_here_and_there(pnb, K, M, without, rank, L):
    g = source(K + M + rank)
    n, batch, ld = 4, 250, L + 2
    check_adapters(pnb, weights(g, M, K), bias_of(g, M), (1 << 45) + 3, weights(g, n, rank, K),
                   weights(g, n, M, rank), which_of(g, batch, n, without), words(g, batch, K, ld), L, 6)
