"""Timed cases of the per-request-weight operators over LWE ciphertexts.

A ciphertext is a row of ``lwe_len`` u64 words (held as int64, arithmetic mod 2^64) at a pitch of
``ld`` words; a token is ``features`` such rows.  The operators:

  route     choices [tokens, top_k] of experts -> rows sorted by expert, and back
  dispatch  the tokens' ciphertexts laid out in row order (optionally weighted)
  contract  every row by its own expert's int8 matrix
  combine   a token's rows back together, with integer weights
  adapter   a shared int8 matrix plus a low-rank adapter per request

``run`` computes them from elementary torch operations, or calls the library when ``own`` is set.
"""
from __future__ import annotations

import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_SHIFT_MAX = 16


def _pnb():
    if "penumbra_b200" not in sys.modules:
        d = os.path.join(_ROOT, "penumbra-fhe_b200")
        spec = importlib.util.spec_from_file_location(
            "penumbra_b200", os.path.join(d, "__init__.py"), submodule_search_locations=[d])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["penumbra_b200"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["penumbra_b200"]


# ---- cases ------------------------------------------------------------------------------------
def listed():
    return [
        # the choices of a handful of requests: launch latency only
        {"name": "route 8x2 of 8", "op": "route", "tokens": 8, "top_k": 2, "experts": 8,
         "unused": 0.0},
        # a full queue of requests, some of whose choices were dropped by a capacity limit
        {"name": "route 8191x4 of 64", "op": "route", "tokens": 8191, "top_k": 4, "experts": 64,
         "unused": 0.1},
        # hidden layer of the MLP configuration (128 values), two experts a token, evaluator pitch
        {"name": "dispatch 96x2, 128 cts", "op": "dispatch", "tokens": 96, "top_k": 2,
         "experts": 8, "unused": 0.0, "features": 128, "lwe_len": 2049, "ld": 2050,
         "weighted": False},
        # gradient of a combine: weighted rows of logits, contiguous rows as encryption makes them
        {"name": "dispatch 37x3, 10 cts, weights", "op": "dispatch", "tokens": 37, "top_k": 3,
         "experts": 5, "unused": 0.2, "features": 10, "lwe_len": 2049, "ld": 2049,
         "weighted": True},
        # one request through its expert's 784 -> 128 layer
        {"name": "contract 1x1, 784->128", "op": "contract", "tokens": 1, "top_k": 1,
         "experts": 8, "unused": 0.0, "sorted": False, "K": 784, "M": 128, "lwe_len": 2049,
         "ld": 2050},
        # 256 requests, each with its tenant's 784 -> 128 layer
        {"name": "contract 256x1, 784->128", "op": "contract", "tokens": 256, "top_k": 1,
         "experts": 16, "unused": 0.0, "sorted": False, "K": 784, "M": 128, "lwe_len": 2049,
         "ld": 2050},
        # second layer: sorted rows, ragged sizes, contiguous ciphertexts at an odd pitch
        {"name": "contract 61x2, 130->200, odd", "op": "contract", "tokens": 61, "top_k": 2,
         "experts": 7, "unused": 0.1, "sorted": True, "K": 130, "M": 200, "lwe_len": 2049,
         "ld": 2049},
        # hidden layer back in token order
        {"name": "combine 96x2, 128 cts", "op": "combine", "tokens": 96, "top_k": 2,
         "experts": 8, "unused": 0.0, "features": 128, "lwe_len": 2049, "ld": 2050,
         "weighted": True},
        # logits of the N = 8192 set, a few requests, contiguous
        {"name": "combine 7x3, 10 cts, N=8192", "op": "combine", "tokens": 7, "top_k": 3,
         "experts": 5, "unused": 0.2, "features": 10, "lwe_len": 8193, "ld": 8193,
         "weighted": True},
        # one request with an adapter beside the shared 784 -> 128 layer
        {"name": "adapter 1, 784->128 r8", "op": "adapter", "batch": 1, "adapters": 4, "rank": 8,
         "K": 784, "M": 128, "lwe_len": 2049, "ld": 2050, "without": 0.0, "shift": 7},
        # 256 requests of 32 tenants, one in eight without an adapter
        {"name": "adapter 256, 784->128 r16", "op": "adapter", "batch": 256, "adapters": 32,
         "rank": 16, "K": 784, "M": 128, "lwe_len": 2049, "ld": 2050, "without": 0.125,
         "shift": 7},
        # a wide layer at a ragged rank, contiguous ciphertexts at an odd pitch
        {"name": "adapter 45, 257->384 r33, odd", "op": "adapter", "batch": 45, "adapters": 9,
         "rank": 33, "K": 257, "M": 384, "lwe_len": 2049, "ld": 2049, "without": 0.2,
         "shift": 10},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# u64 words read and written by the largest listed contraction
_MOST_WORDS = 256 * (784 + 128) * 2050


def draw(rng):
    op = rng.choice(["route", "dispatch", "contract", "contract", "combine", "adapter",
                     "adapter"])
    lwe_len = rng.choice([835, 2049, 2049, 2049, 8193])  # small key, N = 2048, N = 8192
    ld = lwe_len + (0 if rng.random() < 0.35 else 1 + 2 * rng.randint(0, 1))
    unused = rng.choice([0.0, 0.0, 0.1, 0.3])
    if op == "route":
        return {"op": op, "tokens": _log_int(rng, 1, 8191), "top_k": rng.randint(1, 4),
                "experts": _log_int(rng, 1, 256), "unused": unused}
    if op in ("dispatch", "combine"):
        top_k, features = rng.randint(1, 4), _log_int(rng, 1, 512)
        most = max(1, _MOST_WORDS // ((1 + top_k) * features * ld))
        return {"op": op, "tokens": _log_int(rng, 1, min(512, most)), "top_k": top_k,
                "experts": _log_int(rng, 1, 64), "unused": unused, "features": features,
                "lwe_len": lwe_len, "ld": ld, "weighted": rng.random() < 0.6}
    K, M = _log_int(rng, 8, 1024), _log_int(rng, 4, 512)
    # no more words, and no more products, than the largest listed case
    per_token = max((K + M) * ld / _MOST_WORDS, (K + 64) * M * ld / (256 * 864 * 128 * 2050))
    most = max(1, int(1 / per_token))
    if op == "contract":
        top_k = rng.randint(1, 3)
        return {"op": op, "tokens": _log_int(rng, 1, max(1, min(256, most // top_k))),
                "top_k": top_k, "experts": _log_int(rng, 1, 32), "unused": unused,
                "sorted": rng.random() < 0.4, "K": K, "M": M, "lwe_len": lwe_len, "ld": ld}
    return {"op": op, "batch": _log_int(rng, 1, min(256, most)),
            "adapters": _log_int(rng, 1, 64), "rank": _log_int(rng, 1, 64), "K": K, "M": M,
            "lwe_len": lwe_len, "ld": ld, "without": rng.choice([0.0, 0.0, 0.125, 0.5]),
            "shift": rng.randint(0, _SHIFT_MAX)}


# ---- inputs -----------------------------------------------------------------------------------
def _words(g, rows, case):
    """Ciphertext rows: uniform words (LWE masks are uniform), zeros behind lwe_len."""
    x = torch.randint(-(1 << 63), (1 << 63) - 1, (*rows, case["ld"]), dtype=torch.int64,
                      device="cuda", generator=g)
    x[..., case["lwe_len"]:] = 0
    return x


def _int8(g, *shape):
    return torch.randint(-127, 128, shape, dtype=torch.int8, device="cuda", generator=g)


def _ids(g, case):
    """Choices per token, skewed towards the low experts as real routers are; some unused."""
    T, k, E = case["tokens"], case["top_k"], case["experts"]
    u = torch.rand(T, k, device="cuda", generator=g)
    ids = (u * u.sqrt() * E).to(torch.int32).clamp_(0, E - 1)
    drop = torch.rand(T, k, device="cuda", generator=g) < case["unused"]
    return ids.masked_fill_(drop, -1).contiguous()


def _plain_route(ids, E):
    """Rows of the used choices, sorted by expert; ties keep the order of the choices."""
    flat = ids.reshape(-1).long()
    n = flat.numel()
    used = (flat >= 0) & (flat < E)
    key = torch.where(used, flat, torch.full_like(flat, E))
    order = torch.sort(key, stable=True).indices
    per = torch.zeros(E + 1, dtype=torch.int64, device=ids.device)
    per.scatter_add_(0, key, torch.ones_like(key))
    offsets = torch.cat([torch.zeros_like(per[:1]), per[:E].cumsum(0)])
    at = torch.arange(n, device=ids.device)
    row_choice = torch.where(at < offsets[E], order, torch.full_like(order, -1))
    choice_row = torch.empty_like(order).scatter_(0, order, at)
    choice_row = torch.where(used, choice_row, torch.full_like(choice_row, -1))
    return offsets.int(), row_choice.int(), choice_row.int()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op = case["op"]
    s = {"case": case, "op": op}
    if op == "adapter":
        B, K, M = case["batch"], case["K"], case["M"]
        n, r = case["adapters"], case["rank"]
        which = torch.randint(0, n, (B,), dtype=torch.int32, device="cuda", generator=g)
        none = torch.rand(B, device="cuda", generator=g) < case["without"]
        s.update(W=_int8(g, M, K), A=_int8(g, n, r, K), B=_int8(g, n, M, r),
                 bias=torch.randint(-1000, 1000, (M,), device="cuda", generator=g),
                 adapter=which.masked_fill_(none, -1), X=_words(g, (B, K), case))
        s["out"] = torch.zeros(B, M, case["ld"], dtype=torch.int64, device="cuda")
        return s
    ids = _ids(g, case)
    T, k, E = case["tokens"], case["top_k"], case["experts"]
    s["ids"] = ids
    if own:  # a program's buffers, used again by every call
        s["route"] = _pnb().ExpertRoute(T, k, E, ids.device)
    if op == "route":
        return s
    if own:
        _pnb().expert_route(ids, E, out=s["route"])
    else:
        s["offsets"], s["row_choice"], s["choice_row"] = _plain_route(ids, E)
    if op == "contract":
        K, M = case["K"], case["M"]
        s.update(W=_int8(g, E, M, K),
                 bias=torch.randint(-1000, 1000, (E, M), device="cuda", generator=g),
                 X=_words(g, (T * k if case["sorted"] else T, K), case))
        s["out"] = torch.zeros(T * k, M, case["ld"], dtype=torch.int64, device="cuda")
        return s
    F = case["features"]
    s["weights"] = (torch.randint(-255, 256, (T, k), dtype=torch.int32, device="cuda",
                                  generator=g) if case["weighted"] else None)
    rows, outs = (T, T * k) if op == "dispatch" else (T * k, T)
    s["X"] = _words(g, (rows, F), case)
    s["out"] = torch.zeros(outs, F, case["ld"], dtype=torch.int64, device="cuda")
    return s


# ---- one pass ---------------------------------------------------------------------------------
_DELTA = 1 << 45


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    pnb, case, op = _pnb(), s["case"], s["op"]
    if op == "route":
        r = pnb.expert_route(s["ids"], case["experts"], out=s["route"])
        return r.offsets, r.row_choice, r.choice_row.view(-1)
    L = case["lwe_len"]
    if op == "dispatch":
        return pnb.expert_dispatch(s["route"], s["X"], L, weights=s["weights"], out=s["out"])
    if op == "combine":
        return pnb.expert_combine(s["route"], s["X"], L, weights=s["weights"], out=s["out"])
    if op == "contract":
        return pnb.expert_contract(s["route"], s["W"], s["bias"], _DELTA, s["X"], L,
                                   sorted_rows=case["sorted"], out=s["out"])
    return pnb.adapter_contract(s["W"], s["bias"], _DELTA, s["A"], s["B"], s["adapter"], s["X"],
                                L, base_shift=case["shift"], out=s["out"])


def _chunks(n, words_each):
    step = max(1, (1 << 27) // max(1, words_each))  # about 1 GB of 64-bit values at a time
    return [(i, min(n, i + step)) for i in range(0, n, step)]


def _times(W, X):
    """W [.., M, K] (int8) times X [.., K, L] mod 2^64: 16-bit limbs of the words as doubles, whose
    products and sums stay below 2^53 and so are whole numbers."""
    w = W.double()
    y = None
    for limb in range(4):
        part = torch.matmul(w, ((X >> (16 * limb)) & 0xFFFF).double()).long() << (16 * limb)
        y = part if y is None else y + part
    return y


def _run_plain(s):
    case, op = s["case"], s["op"]
    if op == "route":
        return _plain_route(s["ids"], case["experts"])
    L, ld, X = case["lwe_len"], case["ld"], s["X"]
    if op == "adapter":
        n, M, K = case["adapters"], case["M"], case["K"]
        which = s["adapter"].long()
        has = ((which >= 0) & (which < n)).view(-1, 1, 1)
        which = which.clamp(0, n - 1)
        out = torch.zeros(X.shape[0], M, ld, dtype=torch.int64, device=X.device)
        for a, b in _chunks(X.shape[0], (K + M) * ld):
            x = X[a:b, :, :L]
            low = _times(s["A"][which[a:b]], x)
            y = (_times(s["W"], x) << case["shift"]) + torch.where(
                has[a:b], _times(s["B"][which[a:b]], low), 0)
            y[:, :, L - 1] += s["bias"] * _DELTA
            out[a:b, :, :L] = y
        return out
    k, E = case["top_k"], case["experts"]
    if op == "combine":
        row = s["choice_row"].long().view(-1, k)
        used = row >= 0
        w = used.long() if s["weights"] is None else s["weights"].long() * used
        out = torch.zeros(row.shape[0], X.shape[1], ld, dtype=torch.int64, device=X.device)
        for i in range(k):
            out[:, :, :L] += X[row[:, i].clamp(min=0), :, :L] * w[:, i].view(-1, 1, 1)
        return out
    choice = s["row_choice"].long()
    used = choice >= 0
    choice = choice.clamp(min=0)
    if op == "dispatch":
        w = used.long() if s["weights"] is None else s["weights"].reshape(-1)[choice].long() * used
        out = torch.zeros(choice.numel(), X.shape[1], ld, dtype=torch.int64, device=X.device)
        out[:, :, :L] = X[choice // k, :, :L] * w.view(-1, 1, 1)
        return out
    M, K = case["M"], case["K"]
    e = s["ids"].reshape(-1).long()[choice].clamp(0, E - 1)
    out = torch.zeros(choice.numel(), M, ld, dtype=torch.int64, device=X.device)
    for a, b in _chunks(choice.numel(), (K + M) * ld):
        x = X[a:b, :, :L] if case["sorted"] else X[choice[a:b] // k, :, :L]
        y = _times(s["W"][e[a:b]], x)
        y[:, :, L - 1] += s["bias"][e[a:b]] * _DELTA
        out[a:b, :, :L] = torch.where(used[a:b].view(-1, 1, 1), y, 0)
    return out


# ---- what a pass cannot do without ---------------------------------------------------------------
def work(case):
    """Each input read once, each output written once; products and sums of 64-bit words.  Expected
    numbers of used choices stand for the counts."""
    op = case["op"]
    if op == "route":
        n = case["tokens"] * case["top_k"]
        return {"bytes": 12 * n + 4 * (case["experts"] + 1), "flops": 0}
    row = 8 * case["lwe_len"]
    if op == "adapter":
        B, K, M, r = case["batch"], case["K"], case["M"], case["rank"]
        with_one = B * (1 - case["without"])
        live = min(case["adapters"], B)
        macs = case["lwe_len"] * (B * M * K + with_one * r * (K + M))
        return {"bytes": B * (K + M) * row + M * K + live * r * (K + M) + 8 * M + 4 * B,
                "flops": 2 * macs}
    T, k = case["tokens"], case["top_k"]
    R = T * k * (1 - case["unused"])
    seen = T * (1 - case["unused"] ** k)  # tokens with a used choice
    if op == "contract":
        K, M, E = case["K"], case["M"], min(case["experts"], T * k)
        rows_in = R if case["sorted"] else seen
        return {"bytes": (rows_in * K + R * M) * row + E * M * (K + 8) + 8 * T * k,
                "flops": 2 * R * M * K * case["lwe_len"]}
    F = case["features"]
    words = R * F * case["lwe_len"]
    side = (8 if case["weighted"] else 4) * T * k
    if op == "dispatch":
        return {"bytes": (seen + R) * F * row + side, "flops": words if case["weighted"] else 0}
    return {"bytes": (R + T) * F * row + side, "flops": (2 if case["weighted"] else 1) * words}


# ---- the definition, in whole numbers on the host ------------------------------------------------
def _np_times(W, X):
    """W [M, K] times X [K, L] (u64) mod 2^64: 8-bit pieces of the words, each product a sum of at
    most K * 2^15 in magnitude, put together by Horner's rule."""
    w = W.astype(np.float64)
    y = np.zeros((W.shape[0], X.shape[1]), dtype=np.uint64)
    for piece in range(7, -1, -1):
        digit = ((X >> np.uint64(8 * piece)) & np.uint64(255)).astype(np.float64)
        y = y * np.uint64(256) + (w @ digit).astype(np.int64).astype(np.uint64)
    return y


def exact(case, seed):
    macs = 0
    if case["op"] == "adapter":
        macs = case["batch"] * case["M"] * case["K"] * case["ld"]
    elif case["op"] == "contract":
        macs = case["tokens"] * case["top_k"] * case["M"] * case["K"] * case["ld"]
    if macs > 6e9:
        return None
    s = prepare(case, seed)
    host = {n: v.cpu().numpy() for n, v in s.items() if isinstance(v, torch.Tensor)}
    op = case["op"]
    if op == "adapter":
        L = case["lwe_len"]
        X = host["X"].view(np.uint64)
        out = np.zeros((case["batch"], case["M"], case["ld"]), dtype=np.uint64)
        for b, a in enumerate(host["adapter"]):
            x = X[b, :, :L]
            y = _np_times(host["W"], x) * np.uint64(1 << case["shift"])
            if 0 <= a < case["adapters"]:
                y += _np_times(host["B"][a], _np_times(host["A"][a], x))
            y[:, L - 1] += (host["bias"] * _DELTA).view(np.uint64)
            out[b, :, :L] = y
        return torch.from_numpy(out.view(np.int64))
    T, k, E = case["tokens"], case["top_k"], case["experts"]
    lists = [[] for _ in range(E)]
    for c, e in enumerate(host["ids"].reshape(-1).tolist()):
        if 0 <= e < E:
            lists[e].append(c)
    rows = [c for one in lists for c in one]
    if op == "route":
        back = [-1] * (T * k)
        for r, c in enumerate(rows):
            back[c] = r
        starts = [0]
        for one in lists:
            starts.append(starts[-1] + len(one))
        return (torch.tensor(starts, dtype=torch.int32),
                torch.tensor(rows + [-1] * (T * k - len(rows)), dtype=torch.int32),
                torch.tensor(back, dtype=torch.int32))
    L = case["lwe_len"]
    X = host["X"].view(np.uint64)
    out = np.zeros(s["out"].shape, dtype=np.uint64)
    w = host.get("weights")
    w = None if w is None else w.reshape(-1).astype(np.int64).view(np.uint64)
    for r, c in enumerate(rows):
        if op == "dispatch":
            v = X[c // k, :, :L]
            out[r, :, :L] = v if w is None else v * w[c]
        elif op == "combine":
            v = X[r, :, :L]
            out[c // k, :, :L] += v if w is None else v * w[c]
        else:
            e = int(host["ids"].reshape(-1)[c])
            y = _np_times(host["W"][e], X[r if case["sorted"] else c // k, :, :L])
            y[:, L - 1] += (host["bias"][e] * _DELTA).view(np.uint64)
            out[r, :, :L] = y
    return torch.from_numpy(out.view(np.int64))
