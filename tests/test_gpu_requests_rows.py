"""Per-request contractions with every word of every row compared: calls of many rows, in which a
block walks through many groups, slots and turns.  The plain form runs on the GPU: 16-bit limbs of the
words as doubles, whose products with int8 weights stay below 2^53 and so are whole numbers."""
from __future__ import annotations

import math

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


# ---- what small calls no longer reach --------------------------------------------------------------
# Calls of few products take plain multiply-adds; these are above that: the tiles' own range checks of
# indices, their padded copies of weights, and whole blocks that decrypt.
@pytest.mark.parametrize("sorted_rows", [False, True])
@pytest.mark.parametrize("ld", [40, 41])
def test_damaged_route_in_tiles(pnb, ld, sorted_rows):
    g = source(50 + ld)
    T, k, E, M, K, L = 6, 2, 3, 33, 65, 40
    ids = torch.randint(0, E, (T, k), dtype=torch.int32, device="cuda", generator=g)
    W, X = weights(g, E, M, K), words(g, T * k if sorted_rows else T, K, ld)
    route = pnb.expert_route(ids, E)
    big, low = 2147483647, -2147483648
    choice = torch.tensor([T * k, -3, big, low, 4, 5, 6, 7, 8, 9, 10, 11], dtype=torch.int32)
    expert = torch.tensor([0, 1, 2, 0, E, -1, big, low, 2, 1, 0, 2], dtype=torch.int32)
    route.row_choice.copy_(choice)
    route.row_expert.copy_(expert)
    out = torch.full((T * k, M, ld), MARK, dtype=torch.int64, device="cuda")
    pnb.expert_contract(route, W, None, 0, X, L, sorted_rows=sorted_rows, out=out)
    assert bool((out[:8] == MARK).all())
    for r in range(8, 12):
        x = X[r if sorted_rows else r // k, :, :L]
        assert torch.equal(out[r, :, :L], times(W[int(expert[r])], x)), r
    assert pnb.device_status(0) == 0


@pytest.mark.parametrize("ld", [40, 41])
@pytest.mark.parametrize("off", [0, 3])  # weights at an aligned address, and at an odd one
def test_padded_weights_of_the_c_abi(pnb, ld, off):
    # rows of 65 and 17 bytes are copied to the caller's memory or, without it, to the call's own
    g = source(60 + ld)
    E, M, K, rank, L, batch = 3, 33, 65, 17, 40, 5
    place = lambda t: torch.zeros(t.numel() + off, dtype=torch.int8, device="cuda")[off:].view(  # noqa: E731
        t.shape).copy_(t)
    W, A, B = (place(weights(g, *s)) for s in ((E, M, K), (E, rank, K), (E, M, rank)))
    X, lib = words(g, batch, K, ld), pnb.lib()
    a = torch.tensor([2, -1, 0, 1, 1], dtype=torch.int32, device="cuda")
    route = pnb.expert_route(a.view(-1, 1), E)
    x = X[:, :, :L]
    low = torch.stack([times(B[i], times(A[i], x[b])) if i >= 0 else torch.zeros_like(x[0, :M])
                       for b, i in enumerate(a.tolist())])
    choice = rows_of(a, E)
    want = {"adapter": (times(W[0], x) << 2) + low, "expert": times(W[a[choice].long()], x[choice])}
    p = lambda t: t.data_ptr()  # noqa: E731
    stream = torch.cuda.current_stream().cuda_stream

    def call(op, out, ws, size, at):
        if op == "adapter":
            return lib.pnb_adapter_contract(p(W), None, 0, 2, M, K, p(A), p(B), E, rank, p(a), p(X), ld,
                                            p(out), ld, batch, L, ws, size, at)
        return lib.pnb_expert_contract(p(route.row_choice), p(route.row_expert), batch, 1, E, 0, p(W),
                                       None, 0, M, K, p(X), ld, p(out), ld, L, ws, size, at)

    need = {"adapter": lib.pnb_adapter_contract_workspace_bytes(p(W), M, K, p(A), p(B), E, rank),
            "expert": lib.pnb_expert_contract_workspace_bytes(p(W), E, M, K)}
    assert need == {"adapter": (M + E * rank) * 80 + E * M * 32, "expert": E * M * 80}
    new = lambda: torch.full((batch, M, ld), MARK, dtype=torch.int64, device="cuda")  # noqa: E731
    for op in ("adapter", "expert"):
        n, y = need[op], want[op]
        ws = torch.full((n + 256,), 7, dtype=torch.uint8, device="cuda")
        for at, size in ((p(ws), n), (None, 0), (p(ws), n + 256), (None, 0)):
            out = new()
            assert call(op, out, at, size, stream) == 0, pnb.lib().pnb_last_error()
            assert torch.equal(out[:len(y), :, :L], y)
            assert bool((out[len(y):] == MARK).all()) and bool((out[:, :, L:] == MARK).all())
        assert bool((ws[n:] == 7).all())  # nothing behind the bytes asked for
        for at, size in ((p(ws), n - 1), (p(ws) + 8, n)):
            out = new()
            assert call(op, out, at, size, stream) == 1
            assert b"workspace" in lib.pnb_last_error()
            assert bool((out == MARK).all())
        # the call's own memory inside a graph
        out = new()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            rc = call(op, out, None, 0, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        for _ in range(2):
            out.fill_(MARK)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out[:len(y), :, :L], y)
            assert bool((out[len(y):] == MARK).all())
    assert pnb.device_status(0) == 0


@pytest.mark.parametrize("ld", [2049, 2050])
def test_routed_block_of_tiles_decrypts(pnb, ld):
    """route -> expert layer -> Requant -> expert layer on the sorted rows -> weighted combine, each
    layer above the few products: the decrypted outputs are the integer block's."""
    ring = pnb.KeyRing(seed=78)
    g = torch.Generator().manual_seed(33)
    T, k, E, K, H, M, scale, L = 6, 2, 3, 40, 20, 20, 50, 2049
    draw = lambda lo, hi, *s: torch.randint(lo, hi, s, generator=g)  # noqa: E731
    ids = draw(0, E, T, k)
    ids[1, 1] = -1
    x, W1, b1 = draw(0, 4, T, K), draw(-1, 2, E, H, K), draw(-5, 6, E, H)
    W2, w = draw(-1, 2, E, M, H), draw(1, 4, T, k)

    def at_pitch(rows):
        out = torch.zeros(*rows.shape[:2], ld, dtype=torch.int64, device="cuda")
        out[:, :, :L] = rows
        return out

    X = at_pitch(ring.encrypt(x.reshape(-1), scale, seed=5).reshape(T, K, L))
    route = pnb.expert_route(ids.int().cuda(), E)
    R = int(route.offsets[-1])
    h = pnb.expert_contract(route, W1.to(torch.int8).cuda(), b1.cuda(), 1 << scale, X, L)[:R, :, :L]
    reach = int(W1.abs().sum(2).max() * 3 + 5)
    fresh = math.log2(ring.params.glwe_std) + 64
    sigma = fresh + 0.5 * math.log2(float((W1 ** 2).sum(2).max()))
    hd = pnb.TensorDesc.make(H, -reach, reach, scale, sigma)
    q, _ = pnb.requant_batch(ring, h.contiguous(), hd, shift=2, mult=1, round_bias=2, out_scale=52,
                             out_sigma=43.0)
    # noise of the outputs: 2^43 * sqrt(sum W2^2) * sqrt(sum w^2) <= 2^43 * 4.5 * 4.3 < 2^47.3, thirteen
    # of them below half a step of 2^52
    rows = torch.zeros(T * k, H, ld, dtype=torch.int64, device="cuda")
    rows[:R] = at_pitch(q.reshape(R, H, L))
    y = pnb.expert_contract(route, W2.to(torch.int8).cuda(), None, 0, rows, L, sorted_rows=True)
    out = pnb.expert_combine(route, y, L, weights=w.int().cuda())
    got = ring.decrypt(out[:, :, :L].contiguous(), 52).cpu()
    want = torch.zeros(T, M, dtype=torch.int64)
    for t in range(T):
        for i in range(k):
            if ids[t, i] >= 0:
                a = W1[ids[t, i]] @ x[t] + b1[ids[t, i]]
                a = ((a.clamp(min=0) + 2) >> 2).clamp(0, 3)
                want[t] += w[t, i] * (W2[ids[t, i]] @ a)
    assert int(want.abs().max()) < 1 << 10  # what a scale of 2^52 holds with the padding bit
    assert torch.equal(got, want)


@pytest.mark.parametrize("ld", [2049, 2050])
def test_adapters_in_tiles_of_clients_with_different_keys(pnb, ld):
    keys = [pnb.keygen(seed=s, device=0) for s in (43, 44)]
    g = torch.Generator().manual_seed(34)
    K, M, rank, delta, shift, L = 70, 40, 20, 1 << 40, 4, 2049
    draw = lambda lo, hi, *s: torch.randint(lo, hi, s, generator=g)  # noqa: E731
    W, A, B, x = draw(-8, 9, M, K), draw(-3, 4, 2, rank, K), draw(-3, 4, 2, M, rank), draw(0, 4, 2, K)
    X = torch.zeros(2, K, ld, dtype=torch.int64, device="cuda")
    for i in range(2):
        X[i, :, :L] = pnb.encrypt(keys[i], x[i], seed=60 + i, delta=delta)
    Y = pnb.adapter_contract(W.to(torch.int8).cuda(), None, 0, A.to(torch.int8).cuda(),
                             B.to(torch.int8).cuda(),
                             torch.tensor([1, 0], dtype=torch.int32, device="cuda"), X, L,
                             base_shift=shift)
    for i in range(2):
        ph = pnb.phase(keys[i], Y[i, :, :L].contiguous()).cpu().double()
        want = ((W @ x[i]) << shift) + B[1 - i] @ (A[1 - i] @ x[i])
        assert torch.equal(torch.round(ph / delta).long(), want)


# ---- every way of sharing out a block's memory, every row ------------------------------------------
# Weights kept or streamed, X kept for several tiles of rows or read again: a slot let go too early, or
# weights kept over a change of expert, shows in a few rows and tiles, and in no status.
PLANS = [(600, 700, 64, 34), (600, 700, 64, 33), (1100, 130, 20, 34), (260, 1500, 40, 34),
         (260, 1500, 40, 33), (128, 5000, 3, 34), (128, 784, 16, 33), (128, 784, 64, 34)] + [
    (M, K, rank, ld) for M, K, rank in ((896, 128, 16), (800, 97, 16), (769, 128, 33), (640, 128, 64),
                                        (1537, 128, 8), (1664, 64, 1), (256, 256, 48)) for ld in (33, 34)]


@pytest.mark.parametrize("M,K,rank,ld", PLANS)
def test_every_row_of_every_plan(pnb, M, K, rank, ld):
    g = source(M + K + rank)
    n, batch, L = 3, 170, 33
    W, X = weights(g, n, M, K), words(g, batch, K, ld)
    check_adapters(pnb, W[0], None, 0, weights(g, n, rank, K), weights(g, n, M, rank),
                   which_of(g, batch, n, "runs"), X, L, 9, step=16)
    ids = torch.randint(-1, n, (batch, 1), dtype=torch.int32, device="cuda", generator=g)
    check_experts(pnb, ids, W, None, 0, X, L, step=16)


# Words across the tiles of 32 (16 beside adapters), among them a last one of a single word.
@pytest.mark.parametrize("L,ld", [(2049, 2050), (2049, 2049), (835, 838), (97, 98), (1, 1), (16, 18)])
def test_every_row_of_a_wide_call(pnb, L, ld):
    g = source(L + ld)
    E, T, k, K, M, rank = 7, 90, 2, 130, 200, 24
    ids = torch.randint(-1, E, (T, k), dtype=torch.int32, device="cuda", generator=g)
    check_experts(pnb, ids, weights(g, E, M, K), bias_of(g, E, M), 12345, words(g, T, K, ld), L, step=16)
    check_adapters(pnb, weights(g, M, K), bias_of(g, M), 12345, weights(g, E, rank, K),
                   weights(g, E, M, rank), which_of(g, T, E, "runs"), words(g, T, K, ld), L, 4, step=16)


# ---- the largest limb sums --------------------------------------------------------------------------
# 65536 weights of -128 against bytes of 255 reach -2139095040, 0.4% from the end of 32 bits; both for
# the contraction and for the low product of an adapter.
@pytest.mark.parametrize("L,ld", [(33, 34), (33, 33)])
@pytest.mark.parametrize("value", [-128, 127])
def test_largest_limb_sums(pnb, L, ld, value):
    E, T, M, K, rank = 2, 3, 20, 65536, 17
    W = torch.full((E, M, K), value, dtype=torch.int8, device="cuda")
    X = torch.full((T, K, ld), -1, dtype=torch.int64, device="cuda")  # words of all ones
    ids = torch.tensor([[1], [0], [1]], dtype=torch.int32, device="cuda")
    check_experts(pnb, ids, W, None, 0, X, L)
    A = torch.full((E, rank, K), value, dtype=torch.int8, device="cuda")
    B = torch.full((E, M, rank), -128, dtype=torch.int8, device="cuda")
    B[1] = 127
    which = torch.tensor([1, -1, 0], dtype=torch.int32, device="cuda")
    check_adapters(pnb, W[0], None, 0, A, B, which, X, L, 3)
    if value == -128:  # -128 * 65536 * (2^64 - 1) = 2^23 mod 2^64
        out = pnb.expert_contract(pnb.expert_route(ids, E), W, None, 0, X, L)
        assert bool((out[:, :, :L] == 1 << 23).all())


# ---- inputs and outputs at different pitches, through the C ABI ------------------------------------
@pytest.mark.parametrize("L", [33, 34, 257])
@pytest.mark.parametrize("dx,dy", [(0, 1), (1, 0), (0, 3), (3, 1), (1, 2), (2, 0)])
@pytest.mark.parametrize("K,M,rank", [(3, 4, 2), (70, 40, 20), (65, 200, 33)])  # few products, tiles
def test_pitches_apart(pnb, L, dx, dy, K, M, rank):
    g = source(L + 10 * dx + dy)
    lib, E, T, k = pnb.lib(), 3, 9, 2
    ldx, ldy, n = L + dx, L + dy, T * k
    stream = torch.cuda.current_stream().cuda_stream
    p = lambda t: t.data_ptr()  # noqa: E731
    ids = torch.randint(-1, E, (T, k), dtype=torch.int32, device="cuda", generator=g)
    w = torch.randint(-99, 99, (T, k), dtype=torch.int32, device="cuda", generator=g)
    route = pnb.expert_route(ids, E)
    choice = rows_of(ids, E)
    R = len(choice)
    W, X, Y = weights(g, E, M, K), words(g, T, K, ldx), words(g, n, K, ldx)
    A, B = weights(g, E, rank, K), weights(g, E, M, rank)
    a = which_of(g, T, E, "runs")

    def same(out, rows, want):
        assert torch.equal(out[:rows, :, :L], want)
        assert bool((out[rows:] == MARK).all()) and bool((out[:, :, L:] == MARK).all())

    new = lambda *s: torch.full((*s, ldy), MARK, dtype=torch.int64, device="cuda")  # noqa: E731
    out = new(n, M)
    assert lib.pnb_expert_contract(p(route.row_choice), p(route.row_expert), T, k, E, 0, p(W), None, 0, M,
                                   K, p(X), ldx, p(out), ldy, L, None, 0, stream) == 0
    same(out, R, times(W[ids.reshape(-1)[choice].long()], X[choice // k, :, :L]))
    out = new(T, M)
    assert lib.pnb_adapter_contract(p(W), None, 0, 5, M, K, p(A), p(B), E, rank, p(a), p(X), ldx, p(out),
                                    ldy, T, L, None, 0, stream) == 0
    x, i = X[:, :, :L], a.long().clamp(min=0)
    same(out, T, (times(W[0], x) << 5) +
         torch.where((a >= 0).view(-1, 1, 1), times(B[i], times(A[i], x)), 0))
    out = new(n, K)
    assert lib.pnb_expert_dispatch(p(route.choice_row), T, k, p(w), p(X), K, ldx, p(out), ldy, L,
                                   stream) == 0
    same(out, R, X[choice // k, :, :L] * w.reshape(-1)[choice].long().view(-1, 1, 1))
    out = new(T, K)
    assert lib.pnb_expert_combine(p(route.choice_row), T, k, p(w), p(Y), K, ldx, p(out), ldy, L,
                                  stream) == 0
    want = torch.zeros(T, K, L, dtype=torch.int64, device="cuda")
    want.index_add_(0, choice // k, Y[:R, :, :L] * w.reshape(-1)[choice].long().view(-1, 1, 1))
    same(out, T, want)
    torch.cuda.synchronize()
    assert pnb.device_status(0) == 0


# ---- two host threads at once -----------------------------------------------------------------------
def test_two_threads_at_once(pnb):
    # each on a stream of its own, through tiles with padded weights, few products and both pitches
    import threading

    def work(seed, ld, errors):
        try:
            torch.cuda.set_device(0)
            with torch.cuda.stream(torch.cuda.Stream()):
                g = source(seed)
                E, T, L = 4, 60, 130
                for K, M, rank in ((70, 40, 20), (3, 4, 2), (130, 200, 33)) * 3:
                    ids = torch.randint(-1, E, (T, 2), dtype=torch.int32, device="cuda", generator=g)
                    route = pnb.expert_route(ids, E)
                    W, X = weights(g, E, M, K), words(g, T, K, ld)
                    A, B, a = weights(g, E, rank, K), weights(g, E, M, rank), which_of(g, T, E, "runs")
                    y = pnb.expert_contract(route, W, None, 0, X, L)
                    z = pnb.adapter_contract(W[0], None, 0, A, B, a, X, L)
                    c, x, i = rows_of(ids, E), X[:, :, :L], a.long().clamp(min=0)
                    assert torch.equal(y[:len(c), :, :L], times(W[ids.reshape(-1)[c].long()], x[c // 2]))
                    assert torch.equal(z[:, :, :L], times(W[0], x) + torch.where(
                        (a >= 0).view(-1, 1, 1), times(B[i], times(A[i], x)), 0))
        except BaseException as e:  # handed to the test's own thread
            errors.append(e)

    errors = []
    threads = [threading.Thread(target=work, args=(90 + ld, ld, errors)) for ld in (131, 132)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    assert pnb.device_status(0) == 0
