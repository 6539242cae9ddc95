// group_plan.h -- how a 4-bit contraction (group.cu) is computed: one of three forms by the layer's size, the
// grid, and the shares of a block's shared memory.  Plain C++.
#pragma once
#include <algorithm>

namespace pnb {

constexpr int GC_BM = 128;       // outputs per tile
constexpr int GC_WK = 128;       // inputs per weight slot
constexpr int GC_KSTEP = 32;     // inputs per MMA
constexpr int GC_W_HALF = 128 * GC_WK;  // 16 KB: 128 rows of weights
constexpr int GC_X_SLOT = 16 * 1024;
constexpr int GC_COPY_WARPS = 4;
constexpr int GC_EPI_WARPS = 16;  // two groups of two per TMEM lane quarter
// Which way a call goes, by the layer's size.  (The caller's workspace is the same for all.)
constexpr int GC_SHORT = 384;      // most inputs for SHORT,
constexpr int GC_STAYS = 896;      // and for PAIR, whose weights leave X six slots
constexpr int GC_MOST_TILES = 37;  // of outputs: a quarter of 148 multiprocessors
constexpr int GC_MAX_W = 8, GC_MAX_X = 12, GC_MAX_RAW = 16;
constexpr int GC_BARS = 2 * (GC_MAX_W + GC_MAX_X + GC_MAX_RAW) + 4;
constexpr int GC_BAR_BYTES = (8 * GC_BARS + 8 + 127) / 128 * 128;
constexpr int GC_SMEM = 227 * 1024;

// LONG: one block, weights stream, one accumulator of 256 columns for lo and one for hi.
// SHORT: one block, the weights of one tile of outputs stay, or of all, which then take turns at a tile of
//   X; two accumulators of 128 columns for each.
// PAIR: two blocks share a tile, weights stay, two accumulators of 256 columns; every second row of the
//   weights is a hi, in one block those of the first 64 outputs, in the other of the last.
enum GcMode { LONG, SHORT, PAIR };

// BYTES of an X word.
template <int BYTES, bool SHIFTED, GcMode MODE>
struct GcShape {
  static constexpr int STAGES = MODE == LONG ? 1 : 2;
  static constexpr int LOAD = MODE == LONG ? 256 : 128;  // bytes of an X row that one block loads,
  static constexpr int BN = BYTES == 3 ? LOAD / 4 * 3 : LOAD;  // of which these are whole words
  static constexpr int WORDS = BN / BYTES;
  static constexpr int TILE = MODE == PAIR ? 2 * WORDS : WORDS;  // words per tile
  static constexpr int BOXES = LOAD / 128;               // swizzle spans
  static constexpr int XK = GC_X_SLOT / LOAD;            // inputs per X slot
  static constexpr int W_SLOT = (MODE == PAIR ? 1 : 2) * GC_W_HALF;  // 128 rows; 128 of lo, 128 of hi
  static constexpr int W_TAIL = 2 * 128 * GC_KSTEP;      // a last slot of 32 inputs (SHORT)
  static constexpr int RAW_ROWS = XK / 2;                // inputs per raw slot, half of each parity
  static constexpr int RAW_PITCH = LOAD + 16;            // one word of shift, to 16 bytes
  static constexpr int RAW_SLOT = RAW_ROWS * RAW_PITCH;
  static constexpr int COPY = SHIFTED ? GC_COPY_WARPS : 0;
  static constexpr int MMA_WARP = 2 + COPY;  // warp 0 loads X, warp 1 the weights
  static constexpr int ISSUERS = MODE == PAIR ? 1 : 2;   // warps that issue MMAs: by lo, by hi
  static constexpr int EPI_WARP = MMA_WARP + ISSUERS;
  static constexpr int THREADS = 32 * (EPI_WARP + GC_EPI_WARPS);
  static constexpr int EW = TILE / (MODE == LONG ? 4 : 2);  // words per epilogue warp,
  static constexpr int CW = (BYTES == 8 ? 4 : BYTES == 2 ? 16 : 8) / (SHIFTED ? 2 : 1);  // as many
  static constexpr int COLS = CW * BYTES;                // columns of two loads at a time
  static constexpr int HI_AT = MODE == LONG ? 256 : 128;    // columns from lo's sums to hi's
  static constexpr int ROWS = MODE == PAIR ? 16 : 32;    // outputs of a warp
  static constexpr int PART = 8;                         // words of each staged at a time
  static constexpr int STAGE = ROWS * PART * 8;          // of one warp
};

// What a launch does: its tiles, and how a block's shared memory is shared out.
struct GcPlan {
  int n_tiles, m_tiles;  // tiles: outputs fastest, then words, then requests
  int m_group;           // SHORT: tiles of outputs of one block, one or all
  int w_tail;            // of the last weight slot 32 inputs are kept, not 128
  int w_tile;            // bytes of the weights of one tile of outputs
  int w_slots, x_slots, raw_slots;
  int x_at, raw_at, out_at, bars_at;  // shared-memory offsets; weights at 0
};

inline GcMode gc_mode(int n_in, int n_out, bool shifted, int sms) {
  if (n_in > GC_STAYS || n_out > GC_MOST_TILES * GC_BM) return LONG;
  const int m_tiles = (n_out + GC_BM - 1) / GC_BM;  // each wants a block or a pair of its own
  if (n_in <= GC_SHORT) return m_tiles <= sms ? SHORT : LONG;
  // (copying shifted rows costs a pair more than it saves: 64 x 784->128 301 us where LONG took 238)
  return !shifted && m_tiles <= sms / 2 ? PAIR : LONG;
}
// One slot of weights for one tile of outputs is expanded by every block for itself, which saves a launch;
// more by a kernel before.
inline bool gc_in_place(int n_in, int n_out) {
  return n_in <= GC_WK && n_out <= GC_BM;
}

// The grid, and how one block's shared memory is shared out: weights, then X.  Slots of X in flight hide
// memory's latency (64 x 784->128 in pairs: 256, 214 and 199 us with 3, 4 and 5 of them), so a warp
// stages no more than 8 words of its outputs at a time.
template <int BYTES, bool SHIFTED, GcMode MODE>
unsigned gc_plan(GcPlan& a, int n_in, int n_out, int L, int batch, int sms) {
  using S = GcShape<BYTES, SHIFTED, MODE>;
  a.n_tiles = (L + S::TILE - 1) / S::TILE;
  a.m_tiles = (n_out + GC_BM - 1) / GC_BM;
  const int per = MODE == PAIR ? 2 : 1;
  const int kb = (n_in + GC_WK - 1) / GC_WK, kx = (n_in + S::XK - 1) / S::XK;
  unsigned grid =
      (unsigned)std::min<long long>((long long)batch * a.n_tiles * a.m_tiles, sms / per);
  // A block's tiles have the same outputs.  (At some numbers of tiles pairs are left over: 16 x 512->3200
  // takes 50 of 74 and 811 us, its MMAs 523.)
  if (MODE == PAIR) grid = grid / a.m_tiles * a.m_tiles;
  int room = GC_SMEM - GC_BAR_BYTES - GC_EPI_WARPS * S::STAGE;
  a.w_slots = MODE == LONG ? SHIFTED ? 2 : 3 : kb;
  a.m_group = 1;
  a.w_tail = MODE == SHORT && n_in > (kb - 1) * GC_WK && n_in <= (kb - 1) * GC_WK + GC_KSTEP;
  a.w_tile = a.w_slots * S::W_SLOT - (a.w_tail ? S::W_SLOT - S::W_TAIL : 0);
  if (MODE == SHORT) {
    // All tiles of outputs, if their weights leave X its slots and there are tiles of X for all blocks:
    // it is then loaded (and at odd pitches copied) once.  61 x 130->200 88 -> 84 us, at an odd pitch 125
    // -> 95; several of more, so that X is read by fewer groups, 430 -> 600 (96 x 128->784).
    const int x_want = (SHIFTED ? std::max(3, kx + 1) : std::max(4, kx + 2)) * GC_X_SLOT +
                       (SHIFTED ? GC_COPY_WARPS * S::RAW_SLOT : 0);
    const long long x_tiles = (long long)batch * a.n_tiles;
    if (a.m_tiles * a.w_tile <= room - x_want && a.m_tiles * kb <= GC_MAX_W && x_tiles >= 4 * sms)
      a.m_group = a.m_tiles;
    grid = (unsigned)std::min<long long>(sms, x_tiles * (a.m_tiles / a.m_group));
    a.w_slots = a.m_group * kb;
  }
  room -= a.m_group * a.w_tile;
  if (SHIFTED) {
    a.x_slots = a.m_group > 1 ? std::max(3, kx + 1) : 3;
    a.raw_slots = std::min(GC_MAX_RAW, (room - a.x_slots * GC_X_SLOT) / S::RAW_SLOT & ~3);
  } else {
    a.x_slots = std::min(GC_MAX_X, room / GC_X_SLOT);
    a.raw_slots = 0;
  }
  a.x_at = a.m_group * a.w_tile;
  a.out_at = a.x_at + a.x_slots * GC_X_SLOT;
  a.raw_at = a.out_at + GC_EPI_WARPS * S::STAGE;
  a.bars_at = a.raw_at + a.raw_slots * S::RAW_SLOT;
  return grid * per;
}

}  // namespace pnb
