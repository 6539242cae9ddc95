"""How a 4-bit contraction shares out a device and a block's shared memory: every layer that the calls take
has a plan on every number of multiprocessors."""
from __future__ import annotations

import ctypes as C
import os
import subprocess

import numpy as np
import pytest
from conftest import PKG_DIR

SOURCE = r"""
#include "group_plan.h"
using namespace pnb;

template <int BYTES, bool SHIFTED, GcMode MODE>
static void fill(int n_in, int n_out, int L, int batch, int sms, long long* out) {
  using S = GcShape<BYTES, SHIFTED, MODE>;
  GcPlan a{};
  const long long v[] = {MODE, gc_plan<BYTES, SHIFTED, MODE>(a, n_in, n_out, L, batch, sms),
                         a.m_tiles, a.n_tiles, a.m_group, a.w_tile, a.w_slots, a.x_slots, a.raw_slots,
                         a.x_at, a.out_at, a.raw_at, a.bars_at, S::STAGE, S::RAW_SLOT, S::XK, S::TILE,
                         GC_SMEM - GC_BAR_BYTES, S::THREADS};
  for (int i = 0; i < 19; ++i) out[i] = v[i];
}

template <int BYTES, bool SHIFTED>
static void form(int n_in, int n_out, int L, int batch, int sms, long long* out) {
  switch (gc_mode(n_in, n_out, SHIFTED, sms)) {
    case LONG: return fill<BYTES, SHIFTED, LONG>(n_in, n_out, L, batch, sms, out);
    case SHORT: return fill<BYTES, SHIFTED, SHORT>(n_in, n_out, L, batch, sms, out);
    default: return fill<BYTES, SHIFTED, SHIFTED ? LONG : PAIR>(n_in, n_out, L, batch, sms, out);
  }
}

extern "C" void plan(int bytes, int shifted, int n_in, int n_out, int L, int batch, int sms,
                     long long* out) {
  if (bytes == 8 && shifted) form<8, true>(n_in, n_out, L, batch, sms, out);
  else if (bytes == 8) form<8, false>(n_in, n_out, L, batch, sms, out);
  else if (bytes == 4) form<4, false>(n_in, n_out, L, batch, sms, out);
  else if (bytes == 3) form<3, false>(n_in, n_out, L, batch, sms, out);
  else form<2, false>(n_in, n_out, L, batch, sms, out);
}
"""
NAMES = ("mode grid m_tiles n_tiles m_group w_tile w_slots x_slots raw_slots x_at out_at raw_at bars_at "
         "stage raw_slot xk tile smem threads").split()
LONG, SHORT, PAIR = 0, 1, 2
INPUTS = [1, 31, 32, 33, 96, 97, 128, 129, 160, 161, 256, 257, 288, 289, 383, 384, 385, 512, 513, 784, 895,
          896, 897, 2000, 61440]
OUTPUTS = [1, 127, 128, 129, 384, 385, 1000, 1024, 2305, 2432, 3200, 4608, 4609, 4736, 4737, 524160]


@pytest.fixture(scope="module")
def planner(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-o",
                    str(d / "plan.so"), "-I", os.path.join(PKG_DIR, "csrc"), str(d / "plan.cpp")],
                   check=True)
    lib = C.CDLL(str(d / "plan.so"))
    out = (C.c_longlong * len(NAMES))()

    def plan(*args):
        lib.plan(*args, out)
        return dict(zip(NAMES, out))
    return plan


def check(p, bytes_, shifted, n_in, n_out, L, batch, sms):
    x_tiles = batch * p["n_tiles"]
    kb, kx = -(-n_in // 128), -(-n_in // p["xk"])
    assert p["m_tiles"] == -(-n_out // 128) and p["n_tiles"] == -(-L // p["tile"])
    assert 1 <= p["grid"] <= sms and p["threads"] <= 1024
    if p["mode"] == PAIR:  # whole pairs, and as many for one tile of outputs as for another
        assert p["grid"] % (2 * p["m_tiles"]) == 0 and not shifted
        assert p["grid"] // 2 <= x_tiles * p["m_tiles"] and p["w_slots"] == kb <= 8
    elif p["mode"] == SHORT:  # a block at least for every tile of outputs that a block has alone
        assert p["m_group"] in (1, p["m_tiles"])
        assert p["m_group"] > 1 or p["m_tiles"] <= p["grid"] <= x_tiles * p["m_tiles"]
        assert p["m_group"] == 1 or p["grid"] <= x_tiles and p["x_slots"] > kx
        assert p["w_slots"] == p["m_group"] * kb <= 8
    else:
        assert p["grid"] <= x_tiles * p["m_tiles"] and 2 <= p["w_slots"] <= 8
    # one after the other in shared memory, on the boundaries that the tiles' swizzles want
    assert 2 <= p["x_slots"] <= 12
    assert p["x_at"] >= p["m_group"] * p["w_tile"] and p["x_at"] % 1024 == 0 and p["w_tile"] % 1024 == 0
    assert p["out_at"] == p["x_at"] + p["x_slots"] * 16384
    assert p["raw_at"] == p["out_at"] + 16 * p["stage"] and p["stage"] % 512 == 0
    assert p["bars_at"] == p["raw_at"] + p["raw_slots"] * p["raw_slot"] <= p["smem"]
    assert p["bars_at"] % 8 == 0 and p["raw_slot"] % 256 == 0
    if shifted:  # every copying warp has slots of its own
        assert 4 <= p["raw_slots"] <= 16 and p["raw_slots"] % 4 == 0
    else:
        assert p["raw_slots"] == 0


@pytest.mark.parametrize("sms", [1, 2, 3, 16, 18, 19, 36, 37, 38, 73, 74, 75, 132, 148, 160])
@pytest.mark.parametrize("bytes_,shifted", [(8, 0), (8, 1), (4, 0), (3, 0), (2, 0)])
def test_every_layer_has_a_plan(planner, bytes_, shifted, sms):
    for n_in in INPUTS:
        for n_out in OUTPUTS:
            for L, batch in ((1, 1), (7, 3), (2049, 1), (2049, 61), (1 << 20, 256)):
                args = (bytes_, shifted, n_in, n_out, L, batch, sms)
                check(planner(*args), *args)


@pytest.mark.parametrize("bytes_,shifted", [(8, 0), (8, 1), (4, 0), (3, 0), (2, 0)])
def test_every_number_of_inputs(planner, bytes_, shifted):
    rng = np.random.default_rng(0)
    for n_in in range(1, 1200):
        for n_out in (10, 200, int(rng.integers(1, 5000))):
            args = (bytes_, shifted, n_in, n_out, 2049, 64, 148)
            check(planner(*args), *args)


def test_which_form(planner):
    def mode(n_in, n_out, shifted=0, sms=148):
        return planner(8, shifted, n_in, n_out, 2049, 1, sms)["mode"]
    assert [mode(n, 128) for n in (384, 385, 896, 897)] == [SHORT, PAIR, PAIR, LONG]
    assert [mode(n, 128, 1) for n in (384, 385)] == [SHORT, LONG]
    assert [mode(500, m) for m in (4736, 4737)] == [PAIR, LONG]
    # tiles of outputs whose weights would each want a block, or a pair, of its own on a smaller device
    assert [mode(300, 4736, sms=n) for n in (36, 37)] == [LONG, SHORT]
    assert [mode(500, 4736, sms=n) for n in (73, 74)] == [LONG, PAIR]
