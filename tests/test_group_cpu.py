"""Refusals of the ciphertext cache and of the 4-bit contractions: decided before any device work."""
from __future__ import annotations

import ctypes as C
from types import SimpleNamespace

import pytest
import torch

P = C.c_void_p(4096)  # never dereferenced: every call here is refused on the host
ODD8, ODD4, ODD2 = C.c_void_p(4104), C.c_void_p(4100), C.c_void_p(4098)
NUL = C.c_void_p(0)

WRITE = [P, 4, P, 3, 10, 10, P, 8, 32, NUL]
READ = [P, 4, P, 8, 32, 3, P, 10, 10, NUL]
GROUP = [P, P, P, 16, P, 1, 3, 5, 0, P, 10, P, 10, 4, 10, NUL, 0, NUL]
CACHED = [P, P, P, 16, P, 1, 3, 5, P, P, 8, 32, P, 10, 4, 10, NUL, 0, NUL]


def _refused(pnb, fn, args, change, text):
    args = list(args)
    for i, v in change.items():
        args[i] = v
    assert getattr(pnb.lib(), fn)(*args) == 1
    assert text in pnb.lib().pnb_last_error()


@pytest.mark.parametrize("change,text", [
    ({1: -1}, b"tokens=-1"), ({1: 65537}, b"tokens=65537"), ({7: 0}, b"cache_slots=0"),
    ({8: 8}, b"8 bits"), ({8: 64}, b"64 bits"), ({8: 20}, b"20 bits"), ({3: 0}, b"0 ciphertexts"),
    ({4: 9}, b"at pitches 9"), ({5: 0}, b" 0 words"),
    ({4: 1 << 21, 5: (1 << 20) + 1}, b"1048577 words"), ({0: NUL}, b"NULL"), ({2: NUL}, b"NULL"),
    ({6: NUL}, b"NULL"), ({6: ODD8}, b"16-byte"), ({2: ODD4}, b"64-bit words"),
    ({0: ODD2}, b"32-bit integers"),
])
def test_write_refuses(pnb, change, text):
    _refused(pnb, "pnb_cache_write", WRITE, change, text)


@pytest.mark.parametrize("change,text", [
    ({1: -1}, b"tokens=-1"), ({1: 65537}, b"tokens=65537"), ({3: 0}, b"cache_slots=0"),
    ({4: 0}, b"0 bits"), ({4: 40}, b"40 bits"), ({5: 0}, b"0 ciphertexts"), ({7: 9}, b"and 9"),
    ({8: 0}, b" 0 words"), ({0: NUL}, b"NULL"), ({2: NUL}, b"NULL"), ({6: NUL}, b"NULL"),
    ({2: ODD8}, b"16-byte"), ({6: ODD4}, b"64-bit words"), ({0: ODD2}, b"32-bit integers"),
])
def test_read_refuses(pnb, change, text):
    _refused(pnb, "pnb_cache_read", READ, change, text)


@pytest.mark.parametrize("change,text", [
    ({3: 0}, b"group=0"), ({6: 0}, b"M=0"), ({6: 524161}, b"M=524161"), ({7: 0}, b"K=0"),
    ({7: 61441}, b"K=61441"), ({8: 1, 4: NUL, 6: 61441}, b"M=61441"),
    ({8: 1, 4: NUL, 7: 524161}, b"K=524161"), ({8: 1}, b"no bias"), ({10: 9}, b"at pitches 9"),
    ({12: 9}, b"and 9"), ({13: -1}, b"batch=-1"), ({14: 0}, b" 0 words"), ({0: NUL}, b"NULL"),
    ({1: NUL}, b"NULL"), ({9: NUL}, b"NULL"), ({11: NUL}, b"NULL"), ({9: ODD4}, b"64-bit words"),
    ({11: ODD4}, b"64-bit words"), ({4: ODD4}, b"64-bit words"),
    ({7: 1000, 15: P, 16: 6047}, b"6047 bytes"), ({7: 1000, 15: ODD8, 16: 6048}, b"16-byte"),
])
def test_group_contract_refuses(pnb, change, text):
    _refused(pnb, "pnb_group_contract", GROUP, change, text)


@pytest.mark.parametrize("change,text", [
    ({3: -2}, b"group=-2"), ({6: 0}, b"M=0"), ({6: 524161}, b"M=524161"), ({7: 61441}, b"K=61441"),
    ({10: 0}, b"cache_slots=0"), ({11: 12}, b"12 bits"), ({13: 9}, b"and 9"),
    ({14: -1}, b"batch=-1"), ({15: 0}, b" 0 words"), ({0: NUL}, b"NULL"), ({1: NUL}, b"NULL"),
    ({8: NUL}, b"NULL"), ({9: NUL}, b"NULL"), ({12: NUL}, b"NULL"), ({9: ODD8}, b"16-byte"),
    ({8: ODD2}, b"32-bit integers"), ({12: ODD4}, b"64-bit words"), ({4: ODD4}, b"64-bit words"),
    ({7: 1000, 16: P, 17: 6047}, b"6047 bytes"), ({7: 1000, 16: ODD8, 17: 6048}, b"16-byte"),
])
def test_group_contract_cached_refuses(pnb, change, text):
    _refused(pnb, "pnb_group_contract_cached", CACHED, change, text)


@pytest.mark.parametrize("change,text", [
    ({1: -1}, b"rows=-1"), ({2: -1}, b"limit=-1"), ({0: NUL}, b"NULL"), ({3: NUL}, b"NULL"),
    ({0: ODD2}, b"32-bit integers"), ({3: ODD4}, b"64-bit words"),
])
def test_zero_skipped_refuses(pnb, change, text):
    _refused(pnb, "pnb_zero_skipped", [P, 4, 8, P, 10, NUL], change, text)


def test_empty_batches_run_nothing(pnb):
    L = pnb.lib()
    assert L.pnb_zero_skipped(NUL, 0, 8, NUL, 10, NUL) == 0
    assert L.pnb_zero_skipped(NUL, 4, 8, NUL, 0, NUL) == 0
    assert L.pnb_cache_write(NUL, 0, NUL, 3, 10, 10, NUL, 8, 32, NUL) == 0
    assert L.pnb_cache_read(NUL, 0, NUL, 8, 32, 3, NUL, 10, 10, NUL) == 0
    assert L.pnb_group_contract(NUL, NUL, NUL, 16, NUL, 1, 3, 5, 0, NUL, 10, NUL, 10, 0, 10, NUL, 0,
                                NUL) == 0
    assert L.pnb_group_contract_cached(NUL, NUL, NUL, 16, NUL, 1, 3, 5, NUL, NUL, 8, 32, NUL, 10, 0,
                                       10, NUL, 0, NUL) == 0


@pytest.mark.parametrize("L", [1, 7, 8, 9, 835, 2049, 8193, 1 << 20])
@pytest.mark.parametrize("bits", [16, 24, 32])
def test_row_bytes(pnb, L, bits):
    want = -(-L * bits // 8 // 16) * 16
    assert pnb.lib().pnb_cache_row_bytes(L, bits) == want
    assert pnb.CiphertextCache(1, 1, L, bits, device="cpu").data.shape == (1, 1, want)


def test_row_bytes_of_nothing(pnb):
    assert pnb.lib().pnb_cache_row_bytes(0, 32) == 0
    assert pnb.lib().pnb_cache_row_bytes((1 << 20) + 1, 32) == 0
    assert pnb.lib().pnb_cache_row_bytes(10, 48) == 0


@pytest.mark.parametrize("M,K", [(1, 1), (3, 5), (10, 128), (128, 784), (33, 17), (16, 16),
                                 (896, 897), (4736, 100), (4737, 100), (1, 61440),
                                 (16, 24), (16, 25), (384, 1), (4737, 1),
                                 (128, 128), (129, 128), (128, 129)])
def test_binding_and_library_agree_on_workspaces(pnb, M, K):
    L = pnb.lib()
    assert L.pnb_group_contract_workspace_bytes(M, K, 0) == pnb._group_bytes(K, M)
    assert L.pnb_group_contract_workspace_bytes(M, K, 1) == pnb._group_bytes(M, K)


def test_pack_int4(pnb):
    q = torch.tensor([[0, 15, 7], [8, 1, 14]])
    assert pnb.pack_int4(q).tolist() == [[0xF0, 0x07], [0x18, 0x0E]]
    assert pnb.pack_int4(q[:, :2].to(torch.int8)).tolist() == [[0xF0], [0x18]]
    for bad in (q - 1, q + 1, q.float(), q[0]):
        with pytest.raises(ValueError):
            pnb.pack_int4(bad)


def test_binding_refuses(pnb):
    q = torch.zeros(3, 3, dtype=torch.uint8)
    scales = torch.zeros(3, 2, dtype=torch.int8)
    zeros = torch.zeros(3, 2, dtype=torch.uint8)
    W = pnb.GroupWeights(q, scales, 4, 5, zeros)
    for bad in (dict(K=7), dict(K=0), dict(group=0), dict(group=2), dict(scales=scales[:2]),
                dict(zeros=zeros[:, :1]), dict(q=q[0])):
        with pytest.raises(ValueError):
            pnb.GroupWeights(**{**dict(q=q, scales=scales, group=4, K=5, zeros=zeros), **bad})
    for bad in (dict(q=q.to(torch.int8)), dict(scales=zeros), dict(zeros=scales)):
        with pytest.raises(TypeError):
            pnb.GroupWeights(**{**dict(q=q, scales=scales, group=4, K=5, zeros=zeros), **bad})
    for bad in (dict(bits=8), dict(slots=0), dict(features=0), dict(lwe_len=0),
                dict(lwe_len=(1 << 20) + 1), dict(data=torch.zeros(2, 5, 32, dtype=torch.uint8))):
        with pytest.raises(ValueError):
            pnb.CiphertextCache(**{**dict(slots=2, features=5, lwe_len=10, device="cpu"), **bad})
    with pytest.raises(TypeError):
        pnb.CiphertextCache(2, 5, 8, data=torch.zeros(2, 5, 32, dtype=torch.int8))
    cache = pnb.CiphertextCache(2, 5, 10, device="cpu")
    slots = torch.zeros(4, dtype=torch.int32)
    X = torch.zeros(4, 5, 10, dtype=torch.int64)
    for call in (lambda: pnb.cache_write(cache, X, slots), lambda: pnb.cache_read(cache, slots),
                 lambda: pnb.group_contract(W, None, 0, X),
                 lambda: pnb.group_contract_cached(W, None, 0, cache, slots)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    with pytest.raises(ValueError, match="ciphertexts a token"):
        pnb.group_contract_cached(W, None, 0, pnb.CiphertextCache(2, 4, 10, device="cpu"), slots)
    with pytest.raises(TypeError, match="64-bit"):
        pnb.group_contract(W, None, 0, X.to(torch.int32))


def test_sizes_past_32_bits_are_not_cut_short(pnb):
    # ctypes passes the low 32 bits of a longer integer, which the library cannot tell from a size
    long = 1 << 32
    q = torch.zeros(3, 3, dtype=torch.uint8)
    scales = torch.zeros(3, 1, dtype=torch.int8)
    for group in (5, 6, long, long + 4):  # one group of all K
        assert pnb.GroupWeights(q, scales, group, 5).group == 5
    meta = dict(device="meta")
    for M, K in ((1, long + 8), (1, 1 << 31), (long + 8, 1)):
        shape = (M, (K + 1) // 2)
        with pytest.raises(ValueError, match="below 2"):
            pnb.GroupWeights(torch.empty(shape, dtype=torch.uint8, **meta),
                             torch.empty(M, 1, dtype=torch.int8, **meta), K, K)
    for size in ((long + 2, 1), (1 << 31, 1), (1, long + 2)):
        with pytest.raises(ValueError, match="a cache of"):
            pnb.CiphertextCache(*size, 1, **meta)
    cache = pnb.CiphertextCache(2, 1, 3, device="cpu")
    for ld in (long + 3, 1 << 31):
        with pytest.raises(ValueError, match="do not fit a pitch"):
            pnb._pitch(cache, ld, None)
    for n, features, ld in ((long + 2, 1, 3), (2, long + 1, 3), (2, 1, long + 3), (2, 1, 1 << 31)):
        X = SimpleNamespace(dtype=torch.int64, shape=(n, features, ld), is_cuda=True, device=None,
                            is_contiguous=lambda: True)
        with pytest.raises(ValueError, match="below 2"):
            pnb._want_words("X", X, 3, None, (None, features))
    held = SimpleNamespace(data=SimpleNamespace(is_cuda=True), device=torch.device("meta"))
    with pytest.raises(ValueError, match="below 2"):
        pnb.CiphertextCache._slots(held, torch.empty(long + 2, dtype=torch.int32, **meta))
