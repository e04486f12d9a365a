// dcn_ffn_layout.h -- the gated feed-forward block on the host: operand form,
// launch plans, workspace and saved-state layouts.
#pragma once

#include <algorithm>

#include "dcn_ffn.h"

#define DCN_HOST_DEVICE __host__ __device__ __forceinline__

namespace dcn {
namespace ffn {

constexpr int kSms = 148;

inline int64_t round_up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }
inline int64_t div_up(int64_t x, int64_t y) { return (x + y - 1) / y; }

constexpr int BM = 128;  // tile rows
constexpr int BK = 64;   // contracted values of a stage (128 bytes)

// Bytes of the saved gate and up values of a 32 x 16 block (dcn_ffn_gemm.cuh).
constexpr size_t saved_block_bytes(bool wide) { return wide ? 4096 : 2048 + 64; }

// Whether the backward computes gate and up again beside dhidden instead of
// reading what the forward saved.  Again: 4 C more operations a hidden value
// (24 C on fp32 data, six passes) at some 1.2 PFLOP/s; saved: 8.25 (16) bytes
// more, written and read at 6.4 TB/s, and kept in between.  The two meet near
// 390 (125) channels; at and below the bounds the saved state is left out, and
// gate and up enter the derivative unrounded.
constexpr bool recompute_gate_up(int64_t channels, bool wide) { return channels <= (wide ? 128 : 256); }

// A matrix as the products read it, in 16-bit planes: row-major [rows][ld], rows
// on 16-byte boundaries; or, for the block's own operands, panels of 8 columns
// (dcn_ffn_gemm.cuh; ld and plane do not apply).
struct Operand {
  const void* base = nullptr;
  int64_t rows = 0, cols = 0, ld = 0, plane = 0;
  int planes = 1;
};

// ---------------------------------------------------------------- plans
// How the last R tiles of a product are cut along their nkb K blocks among W >
// R workers.  a is the even share R nkb / W rounded up, so it is at least 1.
// Worker s R + t, s < S: slice s of tile t, K blocks [s a, s a + a).  The K blocks
// `rest` past S a of each tile go to E workers more, in runs of the units (tile, K
// block >= S a), tile after tile, whose lengths differ by at most one.  No run is
// longer than a slice: R rest <= R nkb - R S a <= (W - R S) a, and where W - R S
// is more than R rest, E is R rest.  So the longest piece is the even share to a
// K block, no piece is empty, and the workers left over are those of the rounding.
// Slots: the worker's index for a slice, S R + e + t for a run (unique, since
// along the runs either e or t grows by one).
struct Cut {
  int R = 0, S = 0, E = 0, a = 0, rest = 0;
  Cut() = default;
  Cut(int R_, int W, int nkb) : R(R_) {
    a = (int)(((int64_t)nkb * R + W - 1) / W);
    S = std::min(W / R, (nkb + a - 1) / a);
    rest = std::max(0, nkb - S * a);
    E = (int)std::min<int64_t>(W - S * R, (int64_t)R * rest);
  }
  DCN_HOST_DEVICE int64_t units() const { return (int64_t)R * rest; }
  size_t slots() const { return (size_t)S * R + (E ? E + R - 1 : 0); }
  // Pieces of tile t: its S slices, then the runs that touch it, from `run` on.
  DCN_HOST_DEVICE int pieces(int t, int& run) const {
    run = 0;
    if (rest == 0) return S;
    run = (int)((((int64_t)t * rest + 1) * E - 1) / units());
    return S + (int)(((int64_t)(t + 1) * rest * E - 1) / units()) - run + 1;
  }
  DCN_HOST_DEVICE int slot(int t, int piece, int run) const {
    return piece < S ? piece * R + t : S * R + run + (piece - S) + t;
  }
};

struct GemmPlan {
  int bn = 256;
  bool pair = false, split = false;
  int workers = 0;  // CTAs, or pairs of them
  int tiles_m = 0, tiles_n = 0;
  int cols = 0;     // output columns of a tile
  Cut cut;          // split: of the tiles past whole rounds of the workers
  size_t partial_bytes() const { return cut.slots() * BM * (pair ? 2 : 1) * bn * 4; }
};

// Column tile and CTA pairing: the choice whose waves of tiles cost least, a
// tile's time being its columns over the relative rate of that form (a narrower
// or unpaired tile reads more operand rows for the same work).  splittable: the
// product stores plain sums, so the tiles of a last wave that would leave many
// SMs idle can be cut along K.  weights: the column operand is a weight in rows
// of the contracted axis; with one row tile 128 columns a stage keep its reads
// long enough (4096 x 14336 in bf16, 16 rows: 64 columns, cut K 33 us; 32 columns
// on 128 SMs, K whole 76 us).
inline GemmPlan plan_gemm(int64_t M, int64_t N, int64_t nkb, int batches, bool gated, bool splittable,
                          bool wide, bool weights) {
  struct Form {
    int bn;
    bool pair;
    double rate;
  };
  static const Form kNarrow[4] = {{256, true, 1.0}, {256, false, 0.8}, {128, false, 0.65}, {64, false, 0.4}};
  static const Form kWide[3] = {{128, true, 1.0}, {128, false, 0.85}, {64, false, 0.65}};  // fp32 sums live in registers
  GemmPlan best;
  double best_cost = 1e300;
  const Form* forms = wide ? kWide : kNarrow;
  const bool stream = weights && !gated && M <= BM;
  for (int i = 0; i < (wide ? 3 : 4); ++i) {
    const Form& f = forms[i];
    if (stream && (f.pair || f.bn == 256)) continue;
    const int cols = gated ? f.bn / 2 : f.bn, rows = f.pair ? 2 * BM : BM, all = f.pair ? kSms / 2 : kSms;
    const int64_t tm = div_up(M, rows), tn = div_up(N, cols), tiles = tm * tn * batches;
    const double tile = f.bn / f.rate * (double)nkb;
    double cost = (double)div_up(tiles, all) * tile;
    bool split = false;
    if (splittable && tiles % all && tiles < 4 * all && tiles * nkb >= 8 * all) {
      // + writing and adding partials, some 10 us
      const double cut = (double)tiles / all * tile + (wide ? 48.0 : 40.0) * f.bn;
      if (cut < 0.95 * cost) {
        split = true;
        cost = cut;
      }
    }
    if (cost < best_cost) {
      best_cost = cost;
      best.bn = f.bn;
      best.pair = f.pair;
      best.split = split;
      best.workers = (int)(split ? all : std::min<int64_t>(tiles, all));
      best.tiles_m = (int)tm;
      best.tiles_n = (int)tn;
      best.cols = cols;
      best.cut = split ? Cut((int)(tiles % all), all, (int)nkb) : Cut();
    }
  }
  if (gated && M <= BM) {
    // one row tile: its time is that of reading the weights, so their rows are
    // spread over the SMs in as few waves as the widest tile allows
    const int most = wide ? 64 : 128;
    const int64_t waves = div_up(N, (int64_t)most * kSms);
    best.pair = best.split = false;
    best.bn = 2 * most;
    best.cols = (int)std::min<int64_t>(most, round_up(div_up(N, kSms * waves), 16));
    best.tiles_m = 1;
    best.tiles_n = (int)div_up(N, best.cols);
    best.workers = std::min(best.tiles_n, kSms);
  }
  return best;
}

inline size_t store_partial_bytes(int64_t M, int64_t N, int64_t K, int nseg, int batches, bool weights = false) {
  return ws_align(plan_gemm(M, N, div_up(K, BK) * nseg, batches, false, true, nseg >= 6, weights).partial_bytes());
}

// ---------------------------------------------------------------- layouts
struct Shape {
  int64_t M, C, F;
  bool wide;        // fp32 data: three planes
  int planes, pair; // planes of an operand, segments of a product
  size_t es;
  explicit Shape(const FfnProblem& p)
      : M(p.M), C(p.C), F(p.F), wide(p.dtype == DCN_FLOAT32), planes(wide ? 3 : 1), pair(wide ? 6 : 1), es(wide ? 4 : 2) {}
  int64_t row_blocks() const { return div_up(M, 2 * BM) * 8; }  // 32-row blocks, to whole tiles of a pair
  bool recompute() const { return recompute_gate_up(C, wide); }
  bool pack_rows_c() const { return wide || C % 8 != 0; }  // x, dy, w_gate, w_up: rows of C
  bool pack_rows_f() const { return wide || F % 8 != 0; }  // w_down: rows of F
  size_t operand_bytes(int64_t rows, int64_t cols) const {
    return ws_align((size_t)planes * (size_t)rows * (size_t)round_up(cols, 8) * 2);
  }
  // the block's own operands: [rows / 128][cols / 8][128][8] a plane
  size_t panel_plane_bytes() const { return (size_t)round_up(M, BM) * (size_t)round_up(F, 8) * 2; }
  size_t panels_bytes() const { return ws_align((size_t)planes * panel_plane_bytes()); }
  Operand operand(const void* base, int64_t rows, int64_t cols) const {
    Operand o;
    o.base = base;
    o.rows = rows;
    o.cols = cols;
    o.ld = round_up(cols, 8);
    o.plane = rows * o.ld;
    o.planes = planes;
    return o;
  }
  size_t blocks_bytes() const {
    if (recompute()) return 0;
    const int64_t m = row_blocks(), c = div_up(F, 16);
    return ws_align((size_t)(m * c) * saved_block_bytes(wide));
  }
};

// Hands out consecutive 256-byte-aligned pieces of a buffer.
struct Carver {
  uint8_t* base;
  size_t at = 0;
  void* take(size_t bytes) {
    void* p = base ? base + at : nullptr;
    at += ws_align(bytes);
    return p;
  }
};

// Few rows and nothing to save: the weights are streamed into registers
// (dcn_ffn_few.cuh).  From 9 rows on the legacy matrix instruction falls behind
// the weights' arrival (4096 x 14336 in bf16, one call: 1 row 68 us, 8 rows 73,
// 16 rows 100, 32 rows 153; the tile products 77 at any of these), but on small
// weights, where launches count, it stays ahead (512 x 2048, 32 rows: 12 us
// against 21).  The bound of 2^22 weights a matrix is near where the two meet: in
// graphs, weights from memory, this form at 1024 x 4096 and 2048 x 2048 against the
// tile products at 8 hidden units more takes, in bf16, 19 : 34 and 23 : 29 us on 16
// rows, 30 : 34 and 37 : 29 on 32; in fp32 109 : 85 and 87 : 118 on 16 rows, 135 :
// 85 and 141 : 118 on 32, where the meeting point lies lower.  fp32 up to 8 rows
// always comes here (4096 x 14336: 1 row 161 us, 8 rows 417); not measured against
// the tile products.
inline bool few_rows(const FfnProblem& p, bool save) {
  if (save || p.M > 32) return false;
  if (p.dtype == DCN_FLOAT32) return p.M <= 8 || p.C * p.F <= (int64_t(1) << 22);
  return p.C % 8 == 0 && p.F % 8 == 0 && (p.M <= 8 || p.C * p.F <= (int64_t(1) << 22));
}

struct ForwardWs {
  Operand x, wg, wu, wd, h;
  void* few = nullptr;  // few rows: the hidden values, row-major
  float* partial = nullptr;
  size_t total = 0;
  bool pack_c = false, pack_f = false;
  ForwardWs(const FfnProblem& p, const FfnTensors& t, void* ws, void* hidden) {
    const Shape s(p);
    Carver c{static_cast<uint8_t*>(ws)};
    if (few_rows(p, hidden != nullptr)) {
      few = c.take((size_t)s.M * (size_t)s.F * s.es);
      total = c.at;
      return;
    }
    pack_c = s.pack_rows_c();
    pack_f = s.pack_rows_f();
    x = s.operand(pack_c ? c.take(s.operand_bytes(s.M, s.C)) : t.x, s.M, s.C);
    wg = s.operand(pack_c ? c.take(s.operand_bytes(s.F, s.C)) : t.w_gate, s.F, s.C);
    wu = s.operand(pack_c ? c.take(s.operand_bytes(s.F, s.C)) : t.w_up, s.F, s.C);
    wd = s.operand(pack_f ? c.take(s.operand_bytes(s.C, s.F)) : t.w_down, s.C, s.F);
    h = s.operand(hidden ? hidden : c.take(s.panels_bytes()), s.M, s.F);
    partial = static_cast<float*>(c.take(store_partial_bytes(s.M, s.C, s.F, s.pair, 1, true)));
    total = c.at;
  }
};

constexpr int kSumSlices = 4 * kSms;  // at most so many rows of partials of the dy column sums

struct BackwardWs {
  Operand x, dy, wg, wu, wd, dg, du;
  float *partial, *colsum, *rowsum;
  size_t total;
  bool pack_c, pack_f;
  BackwardWs(const FfnProblem& p, const FfnTensors& t, const void* grad, void* ws) {
    const Shape s(p);
    Carver c{static_cast<uint8_t*>(ws)};
    pack_c = s.pack_rows_c();
    pack_f = s.pack_rows_f();
    x = s.operand(pack_c ? c.take(s.operand_bytes(s.M, s.C)) : t.x, s.M, s.C);
    dy = s.operand(pack_c ? c.take(s.operand_bytes(s.M, s.C)) : grad, s.M, s.C);
    wg = s.operand(pack_c ? c.take(s.operand_bytes(s.F, s.C)) : t.w_gate, s.F, s.C);
    wu = s.operand(pack_c ? c.take(s.operand_bytes(s.F, s.C)) : t.w_up, s.F, s.C);
    wd = s.operand(pack_f ? c.take(s.operand_bytes(s.C, s.F)) : t.w_down, s.C, s.F);
    dg = s.operand(c.take(s.panels_bytes()), s.M, s.F);
    du = s.operand(c.take(s.panels_bytes()), s.M, s.F);
    const size_t part = std::max({store_partial_bytes(s.C, s.F, s.M, s.pair, 1),
                                  store_partial_bytes(s.F, s.C, s.M, s.pair, 1),
                                  store_partial_bytes(s.F, s.C, s.M, s.pair, 2),
                                  store_partial_bytes(s.M, s.C, s.F, 2 * s.pair, 1)});
    partial = static_cast<float*>(c.take(part));
    colsum = static_cast<float*>(c.take((size_t)s.row_blocks() * 2 * (size_t)s.F * 4));
    rowsum = static_cast<float*>(c.take((size_t)kSumSlices * (size_t)s.C * 4));
    total = c.at;
  }
};

}  // namespace ffn
}  // namespace dcn
