"""Refusals of the per-request-weight entry points: decided before any device work."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

P = C.c_void_p(4096)  # never dereferenced: every call here is refused on the host
ODD4, ODD2 = C.c_void_p(4100), C.c_void_p(4098)
NUL = C.c_void_p(0)


def _refused(pnb, rc, text):
    assert rc == 1
    assert text in pnb.lib().pnb_last_error()


@pytest.mark.parametrize("tokens,top_k,experts,text", [
    (-1, 1, 4, b"tokens=-1"), (4, 0, 4, b"top_k=0"), (1 << 20, 2, 4, b"choices"),
    (1 << 30, 1 << 30, 4, b"choices"), (4, 2, 0, b"0 experts"), (4, 2, 1025, b"1025 experts"),
])
def test_route_refuses(pnb, tokens, top_k, experts, text):
    _refused(pnb, pnb.lib().pnb_expert_route(P, tokens, top_k, experts, P, P, P, P, NUL), text)


@pytest.mark.parametrize("hole", [0, 4, 5, 6, 7])
def test_route_refuses_null(pnb, hole):
    args = [P, 4, 2, 4, P, P, P, P, NUL]
    args[hole] = NUL
    _refused(pnb, pnb.lib().pnb_expert_route(*args), b"NULL")


@pytest.mark.parametrize("fn,args,words,indices", [
    ("pnb_expert_route", [P, 4, 2, 4, P, P, P, P, NUL], (), (0, 4, 5, 6, 7)),
    ("pnb_expert_dispatch", [P, 4, 2, P, P, 3, 10, P, 10, 10, NUL], (4, 7), (0, 3)),
    ("pnb_expert_combine", [P, 4, 2, P, P, 3, 10, P, 10, 10, NUL], (4, 7), (0, 3)),
    ("pnb_expert_contract", [P, P, 4, 2, 4, 0, P, P, 1, 3, 5, P, 10, P, 10, 10, NUL, 0, NUL],
     (7, 11, 13), (0, 1)),
    ("pnb_adapter_contract", [P, P, 1, 0, 3, 5, P, P, 2, 2, P, P, 10, P, 10, 4, 10, NUL, 0, NUL],
     (1, 11, 13), (10,)),
])
def test_misaligned_addresses_are_refused(pnb, fn, args, words, indices):
    for i in words:
        _refused(pnb, getattr(pnb.lib(), fn)(*args[:i], ODD4, *args[i + 1:]), b"64-bit words")
    for i in indices:
        _refused(pnb, getattr(pnb.lib(), fn)(*args[:i], ODD2, *args[i + 1:]), b"32-bit integers")


@pytest.mark.parametrize("fn", ["pnb_expert_dispatch", "pnb_expert_combine"])
@pytest.mark.parametrize("change,text", [
    ({1: -1}, b"tokens=-1"), ({2: 0}, b"top_k=0"), ({5: 0}, b"0 ciphertexts"),
    ({9: 0}, b" 0 words"), ({6: 9}, b"at pitches 9"), ({8: 9}, b"and 9"), ({0: NUL}, b"NULL"),
    ({4: NUL}, b"NULL"), ({7: NUL}, b"NULL"),
    ({6: 1 << 22, 8: 1 << 22, 9: (1 << 20) + 1}, b"1048577 words"),
])
def test_moves_refuse(pnb, fn, change, text):
    args = [P, 4, 2, NUL, P, 3, 10, P, 10, 10, NUL]
    for i, v in change.items():
        args[i] = v
    _refused(pnb, getattr(pnb.lib(), fn)(*args), text)


@pytest.mark.parametrize("change,text", [
    ({2: -1}, b"tokens=-1"), ({3: 0}, b"top_k=0"), ({4: 0}, b"0 experts"),
    ({4: 2000}, b"2000 experts"), ({9: 0}, b"M=0"), ({9: 524161}, b"M=524161"), ({10: 0}, b"K=0"), ({10: 65537}, b"K=65537"),
    ({12: 9}, b"at pitches 9"), ({14: 9}, b"and 9"), ({15: 0}, b" 0 words"),
    ({12: 1 << 21, 14: 1 << 21, 15: (1 << 20) + 1}, b"1048577 words"), ({0: NUL}, b"NULL"),
    ({1: NUL}, b"NULL"), ({6: NUL}, b"NULL"), ({11: NUL}, b"NULL"), ({13: NUL}, b"NULL"),
])
def test_contract_refuses(pnb, change, text):
    args = [P, P, 4, 2, 4, 0, P, P, 1, 3, 5, P, 10, P, 10, 10, NUL, 0, NUL]
    for i, v in change.items():
        args[i] = v
    _refused(pnb, pnb.lib().pnb_expert_contract(*args), text)


@pytest.mark.parametrize("change,text", [
    ({3: -1}, b"base_shift=-1"), ({3: 64}, b"base_shift=64"), ({4: 0}, b"M=0"),
    ({4: 524161}, b"M=524161"), ({5: 0}, b"K=0"),
    ({5: 65537}, b"K=65537"), ({8: 0}, b"adapters=0"), ({9: 0}, b"rank=0"), ({9: 65}, b"rank=65"),
    ({12: 9}, b"at pitches 9"), ({14: 9}, b"and 9"), ({15: -1}, b"batch=-1"), ({16: 0}, b" 0 words"),
    ({0: NUL}, b"NULL"), ({6: NUL}, b"NULL"), ({7: NUL}, b"NULL"), ({10: NUL}, b"NULL"),
    ({11: NUL}, b"NULL"), ({13: NUL}, b"NULL"),
])
def test_adapter_refuses(pnb, change, text):
    args = [P, P, 1, 0, 3, 5, P, P, 2, 2, P, P, 10, P, 10, 4, 10, NUL, 0, NUL]
    for i, v in change.items():
        args[i] = v
    _refused(pnb, pnb.lib().pnb_adapter_contract(*args), text)


def test_workspace_bytes(pnb):
    L = pnb.lib()
    at = [C.c_void_p(a) for a in (4096, 4104)]
    assert L.pnb_expert_contract_workspace_bytes(at[0], 3, 5, 32) == 0  # read in place
    assert L.pnb_expert_contract_workspace_bytes(at[1], 3, 5, 32) == 15 * 32
    assert L.pnb_expert_contract_workspace_bytes(at[0], 3, 5, 33) == 15 * 48
    assert L.pnb_adapter_contract_workspace_bytes(at[0], 5, 32, at[0], at[0], 2, 16) == 0
    assert L.pnb_adapter_contract_workspace_bytes(at[0], 5, 33, at[0], at[0], 2, 7) == \
        5 * 48 + 14 * 48 + 10 * 16
    assert L.pnb_adapter_contract_workspace_bytes(at[0], 5, 32, at[0], at[1], 2, 16) == 10 * 16


def test_empty_batches_run_nothing(pnb):
    L = pnb.lib()
    assert L.pnb_expert_dispatch(NUL, 0, 2, NUL, NUL, 3, 10, NUL, 10, 10, NUL) == 0
    assert L.pnb_expert_combine(NUL, 0, 2, NUL, NUL, 3, 10, NUL, 10, 10, NUL) == 0
    assert L.pnb_expert_contract(NUL, NUL, 0, 2, 4, 0, NUL, NUL, 1, 3, 5, NUL, 10, NUL, 10, 10,
                                 NUL, 0, NUL) == 0
    assert L.pnb_adapter_contract(NUL, NUL, 1, 0, 3, 5, NUL, NUL, 2, 2, NUL, NUL, 10, NUL, 10, 0,
                                  10, NUL, 0, NUL) == 0


def test_binding_refuses_host_tensors(pnb):
    ids = torch.zeros(4, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        pnb.expert_route(ids, 4)
    route = pnb.ExpertRoute(4, 2, 4, "cpu")
    X = torch.zeros(4, 5, 10, dtype=torch.int64)
    W = torch.zeros(4, 3, 5, dtype=torch.int8)
    with pytest.raises(ValueError, match="CUDA"):
        pnb.expert_dispatch(route, X)
    with pytest.raises(ValueError, match="CUDA"):
        pnb.expert_combine(route, X)
    with pytest.raises(ValueError, match="CUDA"):
        pnb.expert_contract(route, W, None, 0, X)
    with pytest.raises(ValueError, match="CUDA"):
        pnb.adapter_contract(W[0], None, 0, W, W, ids[:, 0], X)
    with pytest.raises(TypeError, match="64-bit"):
        pnb.expert_dispatch(route, X.to(torch.int32))


@pytest.mark.parametrize("off", [0, 1, 8, 16])
@pytest.mark.parametrize("rows,cols", [(3, 16), (3, 17), (1, 1), (7, 32), (5, 784), (5, 785), (2, 33)])
def test_binding_and_library_agree_on_workspaces(pnb, off, rows, cols):
    # the binding works them out by itself, and the library refuses one that is too small
    base = torch.zeros(rows * cols + 64, dtype=torch.int8)
    t = base[-base.data_ptr() % 16 + off:][:rows * cols].view(rows, cols)
    at, L = C.c_void_p(t.data_ptr()), pnb.lib()
    one = pnb._padded(t, rows, cols)
    assert one == L.pnb_expert_contract_workspace_bytes(at, 1, rows, cols)
    assert one == L.pnb_expert_contract_workspace_bytes(at, rows, 1, cols)
    if cols <= 64:  # W [rows][cols], two adapters of rank cols over cols inputs
        three = one + pnb._padded(t, 2 * cols, cols) + pnb._padded(t, 2 * rows, cols)
        assert three == L.pnb_adapter_contract_workspace_bytes(at, rows, cols, at, at, 2, cols)
