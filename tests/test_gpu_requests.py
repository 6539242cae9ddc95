"""Per-request weights over LWE ciphertexts: routing, dispatch, per-expert contraction, combine and
low-rank adapters.  Everything is integer arithmetic mod 2^64, so every word must equal the plain
restatement here (numpy u64 and the CPU oracle's contraction)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

MARK = 0x5A5A5A5A5A5A5A5A  # what untouched words hold


def words(rng, *shape):
    return rng.integers(0, 1 << 64, shape, dtype=np.uint64)


def dev(a, dtype=None):
    a = np.ascontiguousarray(a)
    return torch.tensor(a.view(np.int64) if a.dtype == np.uint64 else a, device="cuda", dtype=dtype)


def host(t):
    return t.cpu().numpy().view(np.uint64)


def marked(*shape):
    return torch.full(shape, MARK, dtype=torch.int64, device="cuda")


def draw_ids(rng, T, k, E, unused):
    ids = rng.integers(0, E, (T, k)).astype(np.int32)
    ids[rng.random((T, k)) < unused] = -1
    return ids


def plain_route(ids, E):
    flat = ids.reshape(-1)
    rows = [c for e in range(E) for c in np.nonzero(flat == e)[0]]
    n = flat.size
    row_choice = np.full(n, -1, np.int32)
    row_choice[:len(rows)] = rows
    row_expert = np.full(n, -1, np.int32)
    row_expert[:len(rows)] = flat[rows]
    choice_row = np.full(n, -1, np.int32)
    choice_row[rows] = np.arange(len(rows))
    offsets = np.array([int(np.sum((flat >= 0) & (flat < e))) for e in range(E + 1)], np.int32)
    return offsets, row_choice, row_expert, choice_row.reshape(ids.shape)


def wt(w, c):
    return np.uint64(1) if w is None else w.reshape(-1)[c].astype(np.int64).astype(np.uint64)


def plain_dispatch(ids, E, X, w, out):
    for r, c in enumerate(plain_route(ids, E)[1]):
        if c >= 0:
            out[r] = X[c // ids.shape[1]] * wt(w, c)
    return out


def plain_combine(ids, E, Y, w):
    out = np.zeros((ids.shape[0],) + Y.shape[1:], np.uint64)
    for r, c in enumerate(plain_route(ids, E)[1]):
        if c >= 0:
            out[c // ids.shape[1]] += Y[r] * wt(w, c)
    return out


def plain_contract(oracle, ids, E, W, bias, delta, X, sorted_rows, out):
    for r, c in enumerate(plain_route(ids, E)[1]):
        if c >= 0:
            e = ids.reshape(-1)[c]
            x = X[r if sorted_rows else c // ids.shape[1]]
            out[r] = oracle.contract(W[e].astype(np.int64), None if bias is None else bias[e], delta,
                                     np.ascontiguousarray(x)[None])[0]
    return out


def plain_adapter(oracle, W, bias, delta, A, B, which, X, shift):
    out = []
    for b, a in enumerate(which):
        x = np.ascontiguousarray(X[b])[None]
        y = oracle.contract(W.astype(np.int64), None, 0, x)[0] << np.uint64(shift)
        if 0 <= a < len(A):
            low = oracle.contract(A[a].astype(np.int64), None, 0, x)
            y = y + oracle.contract(B[a].astype(np.int64), None, 0, low)[0]
        if bias is not None:
            y[:, -1] += bias.astype(np.int64).astype(np.uint64) * np.uint64(delta)
        out.append(y)
    return np.stack(out)


# ---- route --------------------------------------------------------------------------------------
@pytest.mark.parametrize("T,k,E,unused", [
    (1, 1, 1, 0.0), (1, 4, 3, 0.5), (7, 3, 5, 0.2), (32, 1, 8, 0.0), (33, 1, 8, 0.0),
    (128, 8, 64, 0.1), (341, 3, 1024, 0.0), (1025, 1, 2, 0.3), (8191, 4, 64, 0.1),
    (40000, 1, 200, 0.0), (64, 2, 8, 1.0), (513, 2, 1, 0.0), (1024, 1, 7, 0.1), (257, 4, 7, 0.1),
    (2000, 1, 1000, 0.2),
])
def test_route(pnb, T, k, E, unused):
    rng = np.random.default_rng(T * 31 + k * 7 + E)
    ids = draw_ids(rng, T, k, E, unused)
    got = pnb.expert_route(dev(ids), E)
    for name, want in zip(("offsets", "row_choice", "row_expert", "choice_row"),
                          plain_route(ids, E)):
        assert np.array_equal(getattr(got, name).cpu().numpy(), want), name


def test_route_any_value_outside_is_unused(pnb):
    ids = np.array([[0, 4], [-7, 3], [2147483647, -2147483648], [3, 3]], np.int32)
    got = pnb.expert_route(dev(ids), 4)
    assert got.offsets.tolist() == [0, 1, 1, 1, 4]
    assert got.row_choice.tolist() == [0, 3, 6, 7, -1, -1, -1, -1]
    assert got.choice_row.tolist() == [[0, -1], [-1, 1], [-1, -1], [2, 3]]


def test_route_of_nothing(pnb):
    got = pnb.expert_route(torch.zeros(0, 2, dtype=torch.int32, device="cuda"), 5)
    assert got.offsets.tolist() == [0] * 6
    X = torch.zeros(0, 3, 9, dtype=torch.int64, device="cuda")
    assert pnb.expert_dispatch(got, X).shape == (0, 3, 9)
    assert pnb.expert_combine(got, X).shape == (0, 3, 9)


def test_route_largest(pnb):
    ids = (torch.arange(1 << 20, device="cuda") * 2654435761 % 1021).int().reshape(-1, 1)
    got = pnb.expert_route(ids, 1024)
    key, order = torch.sort(ids.reshape(-1), stable=True)
    assert torch.equal(got.row_choice.long(), order)
    assert torch.equal(got.row_expert, key)
    assert torch.equal(got.choice_row.reshape(-1)[order].long(),
                       torch.arange(1 << 20, device="cuda"))


# ---- dispatch and combine -----------------------------------------------------------------------
MOVES = [  # T, k, E, unused, features, L, ld
    (1, 1, 1, 0.0, 1, 1, 1), (1, 1, 1, 0.0, 1, 1, 2), (5, 3, 4, 0.3, 3, 7, 7),
    (5, 3, 4, 0.3, 3, 7, 10), (4, 2, 3, 0.0, 2, 2049, 2049), (4, 2, 3, 0.2, 3, 2049, 2050),
    (9, 4, 6, 0.1, 5, 835, 838), (3, 1, 2, 0.5, 2, 8193, 8193), (6, 2, 4, 1.0, 2, 33, 34),
    (33, 2, 5, 0.1, 17, 64, 64), (2, 16, 16, 0.2, 2, 130, 130),
]


@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("T,k,E,unused,F,L,ld", MOVES)
def test_dispatch_and_combine(pnb, T, k, E, unused, F, L, ld, weighted):
    rng = np.random.default_rng(T * 131 + k * 17 + L + ld)
    ids = draw_ids(rng, T, k, E, unused)
    w = rng.integers(-(1 << 31), 1 << 31, (T, k)).astype(np.int32) if weighted else None
    route = pnb.expert_route(dev(ids), E)
    wd = None if w is None else dev(w)
    X = words(rng, T, F, ld)
    got = host(pnb.expert_dispatch(route, dev(X), L, weights=wd, out=marked(T * k, F, ld)))
    want = plain_dispatch(ids, E, X[:, :, :L], w, np.full((T * k, F, L), MARK, np.uint64))
    assert np.array_equal(got[:, :, :L], want)
    assert np.all(got[:, :, L:] == MARK)
    Y = words(rng, T * k, F, ld)
    got = host(pnb.expert_combine(route, dev(Y), L, weights=wd, out=marked(T, F, ld)))
    assert np.array_equal(got[:, :, :L], plain_combine(ids, E, Y[:, :, :L], w))
    assert np.all(got[:, :, L:] == MARK)


def test_dispatch_and_combine_are_each_others_gradient(pnb):
    # <combine(Y, w), G> = <Y, dispatch(G, w)> mod 2^64, and, the map being linear, the difference
    # of two combines is the combine of the difference.
    rng = np.random.default_rng(3)
    T, k, E, F, L = 11, 3, 6, 4, 300
    ids = draw_ids(rng, T, k, E, 0.2)
    w = rng.integers(-255, 256, (T, k)).astype(np.int32)
    route = pnb.expert_route(dev(ids), E)
    R = int(route.offsets[-1])
    Y, D, G = words(rng, T * k, F, L), words(rng, T * k, F, L), words(rng, T, F, L)
    out = pnb.expert_combine(route, dev(Y), weights=dev(w))
    back = pnb.expert_dispatch(route, dev(G), weights=dev(w))
    assert np.sum(host(out) * G) == np.sum(Y[:R] * host(back)[:R])
    moved = pnb.expert_combine(route, dev(Y + D), weights=dev(w))
    assert torch.equal(moved - out, pnb.expert_combine(route, dev(D), weights=dev(w)))
    out = pnb.expert_dispatch(route, dev(G))
    back = pnb.expert_combine(route, dev(Y))
    assert np.sum(host(out)[:R] * Y[:R]) == np.sum(G * host(back))


def test_rows_outside_the_route_are_not_addresses(pnb):
    # a damaged route: places outside the rows count as unused
    rng = np.random.default_rng(4)
    T, k, E, F, L = 3, 2, 4, 2, 9
    route = pnb.expert_route(dev(draw_ids(rng, T, k, E, 0.0)), E)
    route.choice_row.copy_(torch.tensor([[6, -2], [2147483647, -2147483648], [5, 5]]))
    X = words(rng, T, F, L)
    got = host(pnb.expert_dispatch(route, dev(X), out=marked(T * k, F, L)))
    assert np.all(got[:5] == MARK) and np.array_equal(got[5], X[2])
    Y = words(rng, T * k, F, L)
    got = host(pnb.expert_combine(route, dev(Y)))
    assert not got[:2].any() and np.array_equal(got[2], Y[5] * np.uint64(2))


# ---- per-expert contraction ---------------------------------------------------------------------
CONTRACTS = [  # T, k, E, unused, M, K, L, ld
    (1, 1, 1, 0.0, 1, 1, 1, 1),
    (2, 2, 3, 0.0, 3, 5, 40, 40),
    (3, 2, 4, 0.3, 10, 36, 2049, 2050),
    (3, 2, 4, 0.3, 10, 36, 2049, 2049),
    (2, 1, 2, 0.0, 128, 784, 2049, 2050),
    (2, 1, 2, 0.0, 128, 784, 2049, 2049),
    (5, 2, 3, 0.1, 33, 65, 301, 302),
    (3, 3, 4, 0.1, 200, 130, 300, 300),
    (4, 2, 3, 0.0, 129, 127, 130, 133),
    (4, 2, 3, 0.0, 129, 128, 130, 132),
    (2, 2, 2, 0.0, 257, 144, 835, 836),
    (40, 2, 5, 0.2, 16, 72, 2049, 2050),
    (40, 2, 5, 0.2, 16, 72, 2049, 2049),
    (2, 1, 2, 0.0, 128, 256, 8193, 8194),
    (1, 1, 2, 0.0, 20, 256, 8193, 8193),
    (3, 2, 2, 0.0, 64, 1000, 2049, 2050),
    (2, 1, 2, 1.0, 4, 8, 64, 64),
    (2, 1, 1, 0.0, 2, 3001, 66, 66),
]


@pytest.mark.parametrize("sorted_rows", [False, True])
@pytest.mark.parametrize("T,k,E,unused,M,K,L,ld", CONTRACTS)
def test_expert_contract(pnb, oracle, T, k, E, unused, M, K, L, ld, sorted_rows):
    rng = np.random.default_rng(M * 1009 + K * 13 + ld)
    ids = draw_ids(rng, T, k, E, unused)
    W = rng.integers(-128, 128, (E, M, K)).astype(np.int8)
    bias = rng.integers(-(1 << 40), 1 << 40, (E, M)) if K % 2 else None
    X = words(rng, T * k if sorted_rows else T, K, ld)
    delta = (1 << 45) + 3
    route = pnb.expert_route(dev(ids), E)
    got = host(pnb.expert_contract(route, dev(W), None if bias is None else dev(bias), delta, dev(X),
                                   L, sorted_rows=sorted_rows, out=marked(T * k, M, ld)))
    want = plain_contract(oracle, ids, E, W, bias, delta, X[:, :, :L], sorted_rows,
                          np.full((T * k, M, L), MARK, np.uint64))
    assert np.array_equal(got[:, :, :L], want)
    assert np.all(got[:, :, L:] == MARK)
    assert pnb.device_status(0) == 0


def test_expert_contract_extremes(pnb, oracle):
    # the largest limb sums: all weights -128 or 127 against words of all ones
    W = np.stack([np.full((130, 1024), -128), np.full((130, 1024), 127)]).astype(np.int8)
    X = np.full((2, 1024, 70), (1 << 64) - 1, np.uint64)
    ids = np.array([[1], [0]], np.int32)
    for ld in (70, 71):
        Xp = np.zeros((2, 1024, ld), np.uint64)
        Xp[:, :, :70] = X
        got = host(pnb.expert_contract(pnb.expert_route(dev(ids), 2), dev(W), None, 0, dev(Xp), 70))
        want = plain_contract(oracle, ids, 2, W, None, 0, X, False, np.zeros((2, 130, 70), np.uint64))
        assert np.array_equal(got[:, :, :70], want)


def test_expert_contract_damaged_route(pnb, oracle):
    rng = np.random.default_rng(8)
    T, k, E, M, K, L = 4, 1, 2, 5, 6, 40
    ids = draw_ids(rng, T, k, E, 0.0)
    W = rng.integers(-128, 128, (E, M, K)).astype(np.int8)
    X = words(rng, T, K, L)
    route = pnb.expert_route(dev(ids), E)
    route.row_choice.copy_(torch.tensor([4, -3, 2, 1]))
    route.row_expert.copy_(torch.tensor([0, 0, 2, 1]))
    got = host(pnb.expert_contract(route, dev(W), None, 0, dev(X), out=marked(T, M, L)))
    assert np.all(got[:3] == MARK)
    assert np.array_equal(got[3], oracle.contract(W[1].astype(np.int64), None, 0, X[1:2])[0])


def test_unaligned_base(pnb, oracle):
    # rows at an even pitch whose first word is only 8-byte aligned
    rng = np.random.default_rng(9)
    T, E, M, K, L, ld = 2, 2, 20, 33, 60, 62
    ids = np.array([[1], [0]], np.int32)
    W = rng.integers(-128, 128, (E, M, K)).astype(np.int8)
    flat = dev(words(rng, T * K * ld + 1))
    X = flat[1:].view(T, K, ld)
    out = marked(T * M * ld + 1)[1:].view(T, M, ld)
    route = pnb.expert_route(dev(ids), E)
    got = host(pnb.expert_contract(route, dev(W), None, 0, X, L, out=out))
    want = plain_contract(oracle, ids, E, W, None, 0, host(X)[:, :, :L], False,
                          np.zeros((T, M, L), np.uint64))
    assert np.array_equal(got[:, :, :L], want)
    moved = marked(T * K * ld + 1)[1:].view(T, K, ld)
    pnb.expert_dispatch(route, X, L, out=moved)
    assert np.array_equal(host(moved)[:, :, :L], host(X)[::-1, :, :L])
    Wu = torch.zeros(E * M * K + 5, dtype=torch.int8, device="cuda")[5:].view(E, M, K)
    Wu.copy_(dev(W))  # weights at an odd address
    got = host(pnb.expert_contract(route, Wu, None, 0, X, L))
    assert np.array_equal(got[:, :, :L], want)


# ---- low-rank adapters --------------------------------------------------------------------------
ADAPTERS = [  # batch, n, rank, M, K, L, ld, shift
    (1, 1, 1, 1, 1, 1, 1, 0),
    (3, 2, 2, 3, 5, 40, 40, 63),
    (2, 3, 8, 128, 784, 2049, 2050, 7),
    (2, 3, 8, 128, 784, 2049, 2049, 7),
    (5, 3, 16, 33, 65, 301, 302, 1),
    (4, 2, 33, 200, 130, 300, 300, 10),
    (4, 5, 64, 129, 127, 130, 133, 0),
    (4, 5, 64, 129, 128, 130, 132, 5),
    (3, 2, 17, 257, 144, 835, 836, 3),
    (40, 7, 5, 16, 72, 2049, 2050, 12),
    (40, 7, 5, 16, 72, 2049, 2049, 12),
    (2, 2, 31, 384, 257, 2049, 2049, 10),
    (2, 2, 64, 300, 512, 8193, 8194, 9),
    (1, 2, 7, 10, 128, 8193, 8193, 8),
    (3, 2, 48, 64, 1000, 2049, 2050, 8),
]


@pytest.mark.parametrize("batch,n,rank,M,K,L,ld,shift", ADAPTERS)
def test_adapter_contract(pnb, oracle, batch, n, rank, M, K, L, ld, shift):
    rng = np.random.default_rng(M * 1009 + K * 13 + ld)
    W = rng.integers(-128, 128, (M, K)).astype(np.int8)
    A = rng.integers(-128, 128, (n, rank, K)).astype(np.int8)
    B = rng.integers(-128, 128, (n, M, rank)).astype(np.int8)
    bias = rng.integers(-(1 << 40), 1 << 40, M) if K % 2 else None
    which = rng.integers(-1, n, batch).astype(np.int32)
    which[0] = n - 1
    if batch > 3:
        which[1:4] = (n, -2147483648, 2147483647)  # none of them an adapter
    X = words(rng, batch, K, ld)
    delta = (1 << 45) + 3
    got = host(pnb.adapter_contract(dev(W), None if bias is None else dev(bias), delta, dev(A),
                                    dev(B), dev(which), dev(X), L, base_shift=shift,
                                    out=marked(batch, M, ld)))
    want = plain_adapter(oracle, W, bias, delta, A, B, which, X[:, :, :L], shift)
    assert np.array_equal(got[:, :, :L], want)
    assert np.all(got[:, :, L:] == MARK)
    assert pnb.device_status(0) == 0


def test_adapter_without_any_equals_the_shared_contraction(pnb):
    rng = np.random.default_rng(12)
    W = dev(rng.integers(-128, 128, (40, 70)).astype(np.int8))
    A = dev(rng.integers(-128, 128, (2, 4, 70)).astype(np.int8))
    B = dev(rng.integers(-128, 128, (2, 40, 4)).astype(np.int8))
    bias = dev(rng.integers(-100, 100, 40))
    X = dev(words(rng, 3, 70, 2049))
    none = torch.full((3,), -1, dtype=torch.int32, device="cuda")
    assert torch.equal(pnb.adapter_contract(W, bias, 1 << 40, A, B, none, X),
                       pnb.lwe_contract(W, bias, 1 << 40, X))


def test_adapter_extremes(pnb, oracle):
    n, rank, M, K, L = 2, 64, 130, 1024, 70
    W = np.full((M, K), -128, np.int8)
    A = np.stack([np.full((rank, K), -128), np.full((rank, K), 127)]).astype(np.int8)
    B = np.stack([np.full((M, rank), 127), np.full((M, rank), -128)]).astype(np.int8)
    X = np.full((2, K, L), (1 << 64) - 1, np.uint64)
    which = np.array([0, 1], np.int32)
    got = host(pnb.adapter_contract(dev(W), None, 0, dev(A), dev(B), dev(which), dev(X)))
    assert np.array_equal(got, plain_adapter(oracle, W, None, 0, A, B, which, X, 0))


def test_workspace_of_the_c_abi(pnb, oracle):
    # rows of 13 and 5 bytes are copied first: to the caller's memory, or to the call's own
    rng = np.random.default_rng(14)
    n, rank, M, K, L = 2, 5, 6, 13, 40
    W = rng.integers(-128, 128, (M, K)).astype(np.int8)
    A = rng.integers(-128, 128, (n, rank, K)).astype(np.int8)
    B = rng.integers(-128, 128, (n, M, rank)).astype(np.int8)
    X, which = words(rng, 2, K, L), np.array([1, 0], np.int32)
    want = plain_adapter(oracle, W, None, 0, A, B, which, X, 2)
    Wd, Ad, Bd, wd, Xd = dev(W), dev(A), dev(B), dev(which), dev(X)
    need = pnb.lib().pnb_adapter_contract_workspace_bytes(Wd.data_ptr(), M, K, Ad.data_ptr(),
                                                          Bd.data_ptr(), n, rank)
    assert need == (M + n * rank + n * M) * 16
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    for p, size, rc in ((ws.data_ptr(), need, 0), (None, 0, 0), (ws.data_ptr(), need - 1, 1),
                        (ws.data_ptr() + 8, need, 1)):
        out = marked(2, M, L)
        got = pnb.lib().pnb_adapter_contract(
            Wd.data_ptr(), None, 0, 2, M, K, Ad.data_ptr(), Bd.data_ptr(), n, rank, wd.data_ptr(),
            Xd.data_ptr(), L, out.data_ptr(), L, 2, L, p, size, stream)
        assert got == rc
        if rc == 0:
            assert np.array_equal(host(out), want)
        else:
            assert b"workspace" in pnb.lib().pnb_last_error()
            assert np.all(host(out) == MARK)


@pytest.mark.parametrize("ld", [44, 45])
@pytest.mark.parametrize("x_off,y_off", [(0, 1), (1, 0), (1, 1)])
def test_every_alignment_of_rows(pnb, oracle, ld, x_off, y_off):
    # inputs, outputs or both start at an address that is only 8-byte aligned, at either pitch
    rng = np.random.default_rng(16)
    n, rank, M, K, L, batch = 2, 16, 20, 96, 43, 3
    at = lambda off, *shape: torch.zeros(int(np.prod(shape)) + off, dtype=torch.int64,  # noqa: E731
                                         device="cuda")[off:].view(*shape)
    W = rng.integers(-128, 128, (2, M, K)).astype(np.int8)
    A = rng.integers(-128, 128, (n, rank, K)).astype(np.int8)
    B = rng.integers(-128, 128, (n, M, rank)).astype(np.int8)
    X = words(rng, batch, K, ld)
    which, ids = np.array([1, -1, 0], np.int32), np.array([[1], [0], [1]], np.int32)
    Xd = at(x_off, batch, K, ld).copy_(dev(X))
    bytes_at = lambda a: torch.zeros(a.size + 3, dtype=torch.int8, device="cuda")[3:].view(  # noqa: E731
        *a.shape).copy_(dev(a))
    for place in (dev, bytes_at):  # weights 16-byte aligned, and at odd addresses
        out = at(y_off, batch, M, ld).fill_(MARK)
        got = host(pnb.adapter_contract(place(W[0]), None, 0, place(A), place(B), dev(which), Xd, L,
                                        base_shift=3, out=out))
        assert np.array_equal(got[:, :, :L], plain_adapter(oracle, W[0], None, 0, A, B, which,
                                                           X[:, :, :L], 3))
        assert np.all(got[:, :, L:] == MARK)
        out = at(y_off, batch, M, ld).fill_(MARK)
        route = pnb.expert_route(dev(ids), 2)
        got = host(pnb.expert_contract(route, place(W), None, 0, Xd, L, out=out))
        assert np.array_equal(got[:, :, :L], plain_contract(oracle, ids, 2, W, None, 0, X[:, :, :L],
                                                            False, np.zeros((3, M, L), np.uint64)))
        assert np.all(got[:, :, L:] == MARK)
    out = at(y_off, batch, K, ld).fill_(MARK)
    got = host(pnb.expert_dispatch(route, Xd, L, out=out))
    assert np.array_equal(got[:, :, :L], X[[1, 0, 2], :, :L]) and np.all(got[:, :, L:] == MARK)
    back = at(x_off, batch, K, ld).fill_(MARK)
    got = host(pnb.expert_combine(route, out, L, out=back))
    assert np.array_equal(got[:, :, :L], X[:, :, :L]) and np.all(got[:, :, L:] == MARK)
    assert pnb.device_status(0) == 0


@pytest.mark.parametrize("M,K,rank,ld", [(600, 700, 64, 34), (600, 700, 64, 33), (1100, 130, 20, 34),
                                         (260, 1500, 40, 34), (260, 1500, 40, 33), (128, 5000, 3, 34)])
def test_shapes_whose_operands_do_not_stay(pnb, oracle, M, K, rank, ld):
    # every way of sharing out a block's memory: weights kept or streamed, X kept for several tiles of
    # rows or read again
    rng = np.random.default_rng(M + K)
    L, batch, n = 33, 40, 5
    W = rng.integers(-128, 128, (n, M, K)).astype(np.int8)
    A = rng.integers(-128, 128, (n, rank, K)).astype(np.int8)
    B = rng.integers(-128, 128, (n, M, rank)).astype(np.int8)
    X = torch.randint(-(1 << 63), (1 << 63) - 1, (batch, K, ld), device="cuda")
    which = rng.integers(-1, n, batch).astype(np.int32)
    ids = rng.integers(-1, n, (batch, 1)).astype(np.int32)
    got = pnb.adapter_contract(dev(W[0]), None, 0, dev(A), dev(B), dev(which), X, L, base_shift=9)
    rows = [0, 1, batch // 2, batch - 1]
    Xh = host(X[rows])[:, :, :L]
    want = plain_adapter(oracle, W[0], None, 0, A, B, which[rows], Xh, 9)
    assert np.array_equal(host(got[rows])[:, :, :L], want)
    route = pnb.expert_route(dev(ids), n)
    got = pnb.expert_contract(route, dev(W), None, 0, X, L)
    choice_row = route.choice_row.cpu().numpy()[:, 0]
    for i, t in enumerate(rows):
        if ids[t, 0] >= 0:
            want = oracle.contract(W[ids[t, 0]].astype(np.int64), None, 0,
                                   np.ascontiguousarray(Xh[i])[None])[0]
            assert np.array_equal(host(got[choice_row[t]])[:, :L], want), t
    assert pnb.device_status(0) == 0


@pytest.mark.parametrize("ld", [33, 34])
@pytest.mark.parametrize("M,K,rank", [(896, 128, 16), (800, 97, 16), (769, 128, 33), (640, 128, 64),
                                      (1537, 128, 8), (1664, 64, 1), (256, 256, 48)])
def test_short_k_of_many_tiles(pnb, oracle, M, K, rank, ld):
    # all tiles' weights stay, and take the memory that X is left with
    rng = np.random.default_rng(M + K + rank)
    L, batch, n = 33, 80, 3
    W = rng.integers(-128, 128, (n, M, K)).astype(np.int8)
    A = rng.integers(-128, 128, (n, rank, K)).astype(np.int8)
    B = rng.integers(-128, 128, (n, M, rank)).astype(np.int8)
    X = words(rng, batch, K, ld)
    which = rng.integers(-1, n, batch).astype(np.int32)
    ids = rng.integers(-1, n, (batch, 1)).astype(np.int32)
    rows = [0, 7, batch - 1]
    got = pnb.adapter_contract(dev(W[0]), None, 0, dev(A), dev(B), dev(which), dev(X), L,
                               base_shift=2)
    assert np.array_equal(host(got[rows])[:, :, :L],
                          plain_adapter(oracle, W[0], None, 0, A, B, which[rows], X[rows][:, :, :L], 2))
    route = pnb.expert_route(dev(ids), n)
    got = pnb.expert_contract(route, dev(W), None, 0, dev(X), L)
    for t in rows:
        if ids[t, 0] >= 0:
            want = oracle.contract(W[ids[t, 0]].astype(np.int64), None, 0,
                                   np.ascontiguousarray(X[t, :, :L])[None])[0]
            at = route.choice_row[t, 0].item()
            assert np.array_equal(host(got[at])[:, :L], want), t
    assert pnb.device_status(0) == 0


@pytest.mark.parametrize("K,M,rank,L,ld", [(1, 1, 1, 1, 1), (24, 16, 16, 257, 257), (12, 32, 3, 256, 258),
                                           (25, 16, 17, 300, 301), (8, 48, 1, 835, 835),
                                           (57, 3, 9, 70, 72), (3, 65, 5, 40, 41)])
def test_few_products(pnb, oracle, K, M, rank, L, ld):
    # both sides of the change to plain multiply-adds, with extreme weights, bias and unused rows
    rng = np.random.default_rng(K * 100 + M)
    T, k, E = 5, 2, 3
    ids = draw_ids(rng, T, k, E, 0.3)
    W = rng.choice([-128, 127, 0, 5], (E, M, K)).astype(np.int8)
    bias = rng.integers(-9, 9, (E, M))
    X = words(rng, T, K, ld)
    X[0] = np.uint64(2**64 - 1)
    route = pnb.expert_route(dev(ids), E)
    got = host(pnb.expert_contract(route, dev(W), dev(bias), 1 << 40, dev(X), L,
                                   out=marked(T * k, M, ld)))
    want = host(marked(T * k, M, ld))
    want[:, :, :L] = plain_contract(oracle, ids, E, W, bias, 1 << 40, X[:, :, :L], False,
                                    want[:, :, :L].copy())
    assert np.array_equal(got, want)
    A = rng.choice([-128, 127], (E, rank, K)).astype(np.int8)
    B = rng.choice([-128, 127, 1], (E, M, rank)).astype(np.int8)
    which = np.array([0, -1, 2, 3, 1], np.int32)
    got = host(pnb.adapter_contract(dev(W[0]), dev(bias[0]), 3, dev(A), dev(B), dev(which), dev(X), L,
                                    base_shift=11, out=marked(T, M, ld)))
    assert np.array_equal(got[:, :, :L], plain_adapter(oracle, W[0], bias[0], 3, A, B, which,
                                                       X[:, :, :L], 11))
    assert np.all(got[:, :, L:] == MARK)


def test_strided_inputs(pnb):
    # tensors that are not contiguous are used as the values they hold
    rng = np.random.default_rng(15)
    T, k, E, M, K, L = 4, 2, 3, 10, 12, 30
    ids = dev(draw_ids(rng, T, 2 * k, E, 0.1))[:, ::2]
    route = pnb.expert_route(ids, E)
    assert torch.equal(route.row_choice, pnb.expert_route(ids.contiguous(), E).row_choice)
    X = dev(words(rng, K, T, L)).transpose(0, 1)
    W = dev(rng.integers(-128, 128, (E, K, M)).astype(np.int8)).mT
    got = pnb.expert_contract(route, W, None, 0, X, out=marked(T * k, M, L))
    assert torch.equal(got, pnb.expert_contract(route, W.contiguous(), None, 0, X.contiguous(),
                                                out=marked(T * k, M, L)))
    assert torch.equal(pnb.expert_dispatch(route, X, out=marked(T * k, K, L)),
                       pnb.expert_dispatch(route, X.contiguous(), out=marked(T * k, K, L)))


# ---- refusals of the binding --------------------------------------------------------------------
def test_binding_refusals(pnb):
    i32, i8 = dict(dtype=torch.int32, device="cuda"), dict(dtype=torch.int8, device="cuda")
    route = pnb.expert_route(torch.zeros(4, 2, **i32), 3)
    X = torch.zeros(4, 5, 10, dtype=torch.int64, device="cuda")
    rows = torch.zeros(8, 5, 10, dtype=torch.int64, device="cuda")
    W = torch.zeros(3, 6, 5, **i8)
    with pytest.raises(TypeError, match="int32"):
        pnb.expert_route(torch.zeros(4, 2, dtype=torch.int64, device="cuda"), 3)
    with pytest.raises(pnb.LibraryError, match="experts"):
        pnb.expert_route(torch.zeros(4, 2, **i32), 5000)
    with pytest.raises(ValueError, match="route of"):
        pnb.expert_route(torch.zeros(4, 1, **i32), 3, out=route)
    for call in (lambda: pnb.expert_dispatch(route, rows),
                 lambda: pnb.expert_combine(route, X),
                 lambda: pnb.expert_dispatch(route, X, weights=torch.zeros(4, 1, **i32)),
                 lambda: pnb.expert_dispatch(route, X, out=X),
                 lambda: pnb.expert_dispatch(route, X, 11),
                 lambda: pnb.expert_dispatch(route, X, 0),
                 lambda: pnb.expert_contract(route, W[:2], None, 0, X),
                 lambda: pnb.expert_contract(route, W[0], None, 0, X),
                 lambda: pnb.expert_contract(route, W, None, 0, X, sorted_rows=True),
                 lambda: pnb.expert_contract(route, W, None, 0, rows),
                 lambda: pnb.expert_contract(route, W, None, 0, X[:, :4]),
                 lambda: pnb.expert_contract(route, W.cpu(), None, 0, X),
                 lambda: pnb.adapter_contract(W[0], None, 0, W, W, torch.zeros(4, **i32), X),
                 lambda: pnb.adapter_contract(W[0], None, 0, W, W.mT, torch.zeros(3, **i32), X)):
        with pytest.raises(ValueError):
            call()
    one = pnb.expert_route(torch.zeros(4, 1, **i32), 3)
    buf = torch.zeros(5, 5, 10, dtype=torch.int64, device="cuda")
    for call in (lambda: pnb.expert_dispatch(one, X, out=X),
                 lambda: pnb.expert_combine(one, buf[:4], out=buf[1:]),
                 lambda: pnb.expert_contract(one, torch.zeros(3, 5, 5, **i8), None, 0, buf[1:],
                                             out=buf[:4]),
                 lambda: pnb.adapter_contract(torch.zeros(5, 5, **i8), None, 0, W[:, :2], W[:, :5, :2],
                                              torch.zeros(4, **i32), X, out=X)):
        with pytest.raises(ValueError, match="overlaps"):
            call()
    with pytest.raises(TypeError, match="int8"):
        pnb.expert_contract(route, W.int(), None, 0, X)
    with pytest.raises(pnb.LibraryError, match="rank"):
        pnb.adapter_contract(W[0], None, 0, torch.zeros(3, 65, 5, **i8),
                             torch.zeros(3, 6, 65, **i8), torch.zeros(4, **i32), X)


# ---- streams and graphs -------------------------------------------------------------------------
def _set(pnb, rng, T, k, E, M, K, L, ld, rank):
    s = {"ids": dev(draw_ids(rng, T, k, E, 0.1)), "E": E, "L": L,
         "W": dev(rng.integers(-128, 128, (E, M, K)).astype(np.int8)),
         "w": dev(rng.integers(-9, 9, (T, k)).astype(np.int32)),
         "V": dev(rng.integers(-128, 128, (M, M)).astype(np.int8)),
         "A": dev(rng.integers(-128, 128, (3, rank, M)).astype(np.int8)),
         "B": dev(rng.integers(-128, 128, (3, M, rank)).astype(np.int8)),
         "a": dev(rng.integers(-1, 3, T).astype(np.int32)), "X": dev(words(rng, T, K, ld))}
    return s


def _layer(pnb, s):
    r = pnb.expert_route(s["ids"], s["E"])
    y = pnb.expert_contract(r, s["W"], None, 0, s["X"], s["L"])
    z = pnb.expert_combine(r, y, s["L"], weights=s["w"])
    return pnb.adapter_contract(s["V"], None, 0, s["A"], s["B"], s["a"], z, s["L"], base_shift=3)


def test_two_streams_at_once(pnb):
    rng = np.random.default_rng(21)
    sets = [_set(pnb, rng, 7, 2, 4, 40, 65, 2049, ld, 9) for ld in (2050, 2049)]
    want = [_layer(pnb, s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(_layer(pnb, sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert torch.equal(g[:, :, :2049], want[i][:, :, :2049])


def test_captured_and_replayed(pnb):
    rng = np.random.default_rng(22)
    sets = [_set(pnb, rng, 5, 2, 4, 33, 65, 301, ld, 5) for ld in (302, 301)]
    other = [_set(pnb, rng, 5, 2, 4, 33, 65, 301, ld, 5) for ld in (302, 301)]
    want = [[_layer(pnb, s)[:, :, :301].clone() for s in pair] for pair in zip(sets, other)]
    graphs, outs = [], []
    for s in sets:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _layer(pnb, s)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_layer(pnb, s))
        graphs.append(g)
    for rep in range(3):
        for i, g in enumerate(graphs):
            if rep == 1:  # new inputs in the captured buffers
                for n in ("ids", "W", "w", "V", "A", "B", "a", "X"):
                    sets[i][n].copy_(other[i][n])
            g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i][:, :, :301], want[i][1 if rep else 0]), (rep, i)


def test_large_route_captured_and_replayed(pnb):  # several blocks, and more shared memory than usual
    rng = np.random.default_rng(23)
    T, k, E = 3000, 2, 700
    ids = [draw_ids(rng, T, k, E, 0.2) for _ in range(2)]
    at = dev(ids[0])
    route = pnb.expert_route(at, E)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        pnb.expert_route(at, E, out=route)
    for want in ids[::-1]:
        at.copy_(dev(want))
        g.replay()
        torch.cuda.synchronize()
        for name, w in zip(("offsets", "row_choice", "row_expert", "choice_row"),
                           plain_route(want, E)):
            assert np.array_equal(getattr(route, name).cpu().numpy(), w), name


# ---- sizes past 32 bits -------------------------------------------------------------------------
@pytest.fixture
def room():
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("ld", [1026, 1025])
def test_inputs_past_32_bit_offsets(pnb, oracle, room, ld):
    # 67 requests of the longest K: 4.5e9 words; the first, and the last two, hold something
    rng = np.random.default_rng(41)
    batch, K, M, L, rank = 67, 65536, 3, 1025, 2
    X = torch.empty(batch, K, ld, dtype=torch.int64, device="cuda")
    assert X.numel() > 1 << 32
    rows = [0, batch - 2, batch - 1]
    for b in rows:
        X[b] = torch.randint(-(1 << 63), (1 << 63) - 1, (K, ld), device="cuda")
    W = rng.integers(-128, 128, (2, M, K)).astype(np.int8)
    A = rng.integers(-128, 128, (2, rank, K)).astype(np.int8)
    B = rng.integers(-128, 128, (2, M, rank)).astype(np.int8)
    ids = np.full((batch, 1), -1, np.int32)
    which = np.full(batch, -1, np.int32)
    ids[rows, 0], which[rows] = [1, 0, 1], [1, -1, 0]
    route = pnb.expert_route(dev(ids), 2)
    y = host(pnb.expert_contract(route, dev(W), None, 0, X, L)[:3])
    z = host(pnb.adapter_contract(dev(W[0]), None, 0, dev(A), dev(B), dev(which), X, L)[rows])
    for i, b in enumerate(rows):
        x = np.ascontiguousarray(host(X[b])[:, :L])[None]
        at = route.choice_row[b, 0].item()
        assert np.array_equal(y[at, :, :L], oracle.contract(W[ids[b, 0]].astype(np.int64), None, 0,
                                                            x)[0])
        assert np.array_equal(z[i, :, :L], plain_adapter(oracle, W[0], None, 0, A, B, which[b:b + 1],
                                                         x, 0)[0])
    assert pnb.device_status(0) == 0


@pytest.mark.parametrize("ld", [1026, 1025])
def test_outputs_past_32_bit_offsets(pnb, oracle, room, ld):
    rng = np.random.default_rng(42)
    M, K, L, batch = 262144, 32, 1025, 17
    W = rng.integers(-128, 128, (M, K)).astype(np.int8)
    A, B = np.zeros((1, 1, K), np.int8), np.zeros((1, M, 1), np.int8)
    which = np.full(batch, -1, np.int32)
    X = words(rng, batch, K, ld)
    y = pnb.adapter_contract(dev(W), None, 0, dev(A), dev(B), dev(which), dev(X), L)
    assert y.numel() > 1 << 32
    pick = np.array([0, 1, 131071, M - 129, M - 1])
    got = host(y[-1][torch.tensor(pick, device="cuda")])[:, :L]
    assert np.array_equal(got, oracle.contract(W[pick].astype(np.int64), None, 0,
                                               np.ascontiguousarray(X[-1:, :, :L]))[0])
    # the same rows moved: one token in, one row out, and back
    route = pnb.expert_route(torch.zeros(1, 1, dtype=torch.int32, device="cuda"), 1)
    whole = y.view(1, batch * M, ld)
    moved = pnb.expert_dispatch(route, whole, L)
    assert torch.equal(moved[0, -M:, :L], y[-1, :, :L])
    assert torch.equal(moved[0, :M, :L], y[0, :, :L])
    back = pnb.expert_combine(route, moved, L, out=whole.zero_())
    assert torch.equal(back[0, -M:, :L], moved[0, -M:, :L])
    assert pnb.device_status(0) == 0


@pytest.mark.parametrize("K", [65536, 65535])  # read in place, and padded in the workspace
def test_weights_past_32_bit_offsets(pnb, oracle, room, K):
    rng = np.random.default_rng(43)
    E, M, L = 1024, 65, 33
    W = torch.empty(E, M, K, dtype=torch.int8, device="cuda")
    assert W.numel() > 1 << 32
    for e in (0, 511, E - 1):
        W[e] = torch.randint(-128, 128, (M, K), device="cuda", dtype=torch.int8)
    ids = np.array([[E - 1], [0], [511]], np.int32)
    X = words(rng, 3, K, L + 1)
    route = pnb.expert_route(dev(ids), E)
    got = host(pnb.expert_contract(route, W, None, 0, dev(X), L))
    for r, (t, e) in enumerate([(1, 0), (2, 511), (0, E - 1)]):
        want = oracle.contract(W[e].cpu().numpy().astype(np.int64), None, 0,
                               np.ascontiguousarray(X[t:t + 1, :, :L]))[0]
        assert np.array_equal(got[r, :, :L], want), e
    assert pnb.device_status(0) == 0


# ---- the operators together, as they are used ----------------------------------------------------
def test_routed_block_decrypts_to_the_integer_block(pnb):
    """route -> first expert layer -> Requant (bootstraps) -> second expert layer on the sorted rows
    -> weighted combine: the decrypted outputs are the integer block's."""
    ring = pnb.KeyRing(seed=77)
    rng = np.random.default_rng(31)
    T, k, E, K, H, M, scale = 3, 2, 3, 12, 6, 4, 50
    ids = draw_ids(rng, T, k, E, 0.0)
    ids[1, 1] = -1
    x = rng.integers(0, 4, (T, K))
    W1 = rng.integers(-3, 4, (E, H, K))
    b1 = rng.integers(-5, 6, (E, H))
    W2 = rng.integers(-3, 4, (E, M, H))
    w = rng.integers(1, 4, (T, k)).astype(np.int32)
    X = ring.encrypt(x.reshape(-1), scale, seed=5).reshape(T, K, -1)
    route = pnb.expert_route(dev(ids), E)
    R = int(route.offsets[-1])
    h = pnb.expert_contract(route, dev(W1.astype(np.int8)), dev(b1), 1 << scale, X)[:R]
    reach = int(np.abs(W1).sum(2).max() * 3 + 5)
    fresh = float(np.log2(ring.params.glwe_std) + 64)
    sigma = fresh + 0.5 * np.log2(float((W1 ** 2).sum(2).max()))
    hd = pnb.TensorDesc.make(H, -reach, reach, scale, sigma)
    q, qd = pnb.requant_batch(ring, h.contiguous(), hd, shift=2, mult=1, round_bias=2, out_scale=52,
                              out_sigma=43.0)
    # noise of the outputs: 2^43 * sqrt(sum W2^2) * sqrt(sum w^2) <= 2^43 * 7.4 * 4.3 < 2^48, seven of
    # them below half a step of 2^52
    rows = torch.zeros(T * k, H, q.shape[-1], dtype=torch.int64, device="cuda")
    rows[:R] = q
    y = pnb.expert_contract(route, dev(W2.astype(np.int8)), None, 0, rows, sorted_rows=True)
    out = pnb.expert_combine(route, y, weights=dev(w))
    got = ring.decrypt(out, 52).cpu().numpy()
    want = np.zeros((T, M), np.int64)
    for t in range(T):
        for i in range(k):
            if ids[t, i] >= 0:
                a = W1[ids[t, i]] @ x[t] + b1[ids[t, i]]
                a = np.clip((np.maximum(a, 0) + 2) >> 2, 0, 3)
                want[t] += w[t, i] * (W2[ids[t, i]] @ a)
    assert np.abs(want).max() < 1 << 10  # what a scale of 2^52 holds with the padding bit
    assert np.array_equal(got, want)


def test_adapters_of_clients_with_different_keys(pnb):
    """One call over requests encrypted under two clients' keys, each with its own adapter."""
    keys = [pnb.keygen(seed=s, device=0) for s in (41, 42)]
    rng = np.random.default_rng(32)
    K, M, rank, delta, shift = 30, 9, 4, 1 << 40, 4
    W = rng.integers(-8, 9, (M, K))
    A = rng.integers(-3, 4, (2, rank, K))
    B = rng.integers(-3, 4, (2, M, rank))
    x = rng.integers(0, 4, (2, K))
    X = torch.stack([pnb.encrypt(keys[i], torch.tensor(x[i]), seed=50 + i, delta=delta)
                     for i in range(2)])
    Y = pnb.adapter_contract(dev(W.astype(np.int8)), None, 0, dev(A.astype(np.int8)),
                             dev(B.astype(np.int8)), dev(np.array([1, 0], np.int32)), X,
                             base_shift=shift)
    for i in range(2):
        ph = pnb.phase(keys[i], Y[i].contiguous()).cpu().numpy().astype(np.float64)
        want = (W @ x[i] << shift) + B[1 - i] @ (A[1 - i] @ x[i])
        assert np.array_equal(np.round(ph / delta).astype(np.int64), want)
