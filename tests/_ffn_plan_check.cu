// Host-side enumeration of the gated feed-forward block's cut products: what the
// workers of a launch write (Work) against what the reduction adds (Cut).  Prints
// one line per fault and ends with their number; nothing runs on a GPU.
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <vector>

#include "dcn_ffn_gemm.cuh"

using namespace dcn;
using namespace dcn::ffn;

static int faults = 0;
#define EXPECT(cond, ...)             \
  do {                                \
    if (!(cond) && ++faults <= 20) {  \
      printf("fault: " __VA_ARGS__);  \
      printf("\n");                   \
    }                                 \
  } while (0)

// `tiles` tiles of nkb K blocks on W workers, the last tiles % W of them cut.
static void check_cut(int tiles, int W, int nkb) {
  const int R = tiles % W;
  GemmArgs a{};
  a.tiles_m = tiles;
  a.tiles_n = a.batches = a.nseg = 1;
  a.nk = nkb;
  a.split = 1;
  a.cut = Cut(R, W, nkb);
  EXPECT(a.cut.a >= 1, "W %d R %d nkb %d: slices of %d K blocks", W, R, nkb, a.cut.a);
  if (a.cut.a < 1) return;
  std::vector<int> whole(tiles, 0), owner(2 * W, -1), covered((size_t)R * nkb, 0);
  long long busiest = 0;
  for (int w = 0; w < W; ++w) {
    Work<true> work(a, w, W);
    long long mine = 0;
    while (work.next(a)) {
      if (work.slot < 0) {
        ++whole[work.tile];
        continue;
      }
      const int t = work.tile - (tiles - R);
      EXPECT(t >= 0 && t < R && work.kb0 >= 0 && work.kb0 < work.kb1 && work.kb1 <= nkb && work.slot < 2 * W,
             "W %d R %d nkb %d: worker %d tile %d blocks %d..%d slot %d", W, R, nkb, w, t, work.kb0, work.kb1, work.slot);
      if (t < 0 || t >= R || work.slot >= 2 * W) return;
      EXPECT(owner[work.slot] == -1, "W %d R %d nkb %d: slot %d twice", W, R, nkb, work.slot);
      owner[work.slot] = t;
      for (int k = work.kb0; k < work.kb1; ++k) ++covered[(size_t)t * nkb + k];
      mine += work.kb1 - work.kb0;
    }
    if (mine > busiest) busiest = mine;
  }
  for (int t = 0; t < tiles - R; ++t) EXPECT(whole[t] == 1, "W %d tiles %d: tile %d dealt %d times", W, tiles, t, whole[t]);
  bool once = true;
  for (int c : covered) once = once && c == 1;
  EXPECT(once, "W %d R %d nkb %d: a K block is not multiplied exactly once", W, R, nkb);
  for (int t = 0; t < R; ++t) {
    int run, written = 0;
    const int n = a.cut.pieces(t, run);
    for (int s = 0; s < 2 * W; ++s) written += owner[s] == t;
    EXPECT(n == written, "W %d R %d nkb %d: tile %d has %d pieces, %d are added", W, R, nkb, t, written, n);
    for (int i = 0; i < n && n == written; ++i) {
      const int s = a.cut.slot(t, i, run);
      EXPECT(s >= 0 && s < 2 * W && owner[s] == t, "W %d R %d nkb %d: tile %d adds slot %d", W, R, nkb, t, s);
      if (s >= 0 && s < 2 * W) owner[s] = -2;  // added once
    }
  }
  const long long even = ((long long)R * nkb + W - 1) / W;
  EXPECT(busiest <= even, "W %d R %d nkb %d: a worker has %lld K blocks, an even share is %lld", W, R, nkb, busiest, even);
}

// The plan of a product M x N over nkb K blocks: what its pieces take of the
// partial buffer, and the longest work of a worker against that without the cut.
static bool check_plan(int64_t M, int64_t N, int64_t nkb, int batches, bool wide, bool weights) {
  const GemmPlan p = plan_gemm(M, N, nkb, batches, false, true, wide, weights);
  if (!p.split) {
    EXPECT(p.partial_bytes() == 0, "%lld x %lld x %lld: a buffer without a cut", (long long)M, (long long)N, (long long)nkb);
    return false;
  }
  GemmArgs a{};
  a.tiles_m = p.tiles_m;
  a.tiles_n = p.tiles_n;
  a.batches = batches;
  a.nseg = 1;
  a.nk = (int)nkb;
  a.split = 1;
  a.cut = p.cut;
  const int tiles = p.tiles_m * p.tiles_n * batches;
  EXPECT(p.cut.R == tiles % p.workers, "%lld x %lld x %lld: %d tiles cut", (long long)M, (long long)N, (long long)nkb, p.cut.R);
  int64_t top = -1, longest = 0;
  for (int w = 0; w < p.workers; ++w) {
    Work<true> work(a, w, p.workers);
    int64_t mine = 0;
    for (; work.next(a); mine += work.kb1 - work.kb0)
      if (work.slot > top) top = work.slot;
    if (mine > longest) longest = mine;
  }
  const int64_t bytes = (top + 1) * BM * (p.pair ? 2 : 1) * p.bn * 4, uncut = div_up(tiles, p.workers) * nkb;
  EXPECT((int64_t)p.partial_bytes() == bytes, "%lld x %lld x %lld: partial sums of %lld bytes in a buffer of %lld",
         (long long)M, (long long)N, (long long)nkb, (long long)bytes, (long long)p.partial_bytes());
  EXPECT(longest < uncut, "%lld x %lld x %lld: the cut takes %lld K blocks, no cut %lld", (long long)M, (long long)N,
         (long long)nkb, (long long)longest, (long long)uncut);
  return true;
}

// Sizes spread over the logarithm; the same every time.
static uint64_t state = 1;
static uint64_t next_random() {
  state = state * 6364136223846793005ull + 1442695040888963407ull;
  return state >> 33;
}
static int64_t size(double lo, double hi) {
  return (int64_t)(lo * exp(log(hi / lo) * (double)(next_random() % 100001) / 1e5) + 0.5);
}
static int check_plans() {
  int cuts = 0;
  for (int i = 0; i < 60000; ++i) {
    const bool wide = next_random() % 4 == 0;
    const int seg = wide ? 6 : 1;
    const int64_t M = size(1, 1e6), C = size(16, 4096), F = C * (1 + (int64_t)(next_random() % 5)) + (int64_t)(next_random() % 3);
    if ((double)M * F > 5e8) continue;
    cuts += check_plan(M, C, div_up(F, BK) * seg, 1, wide, true);        // y
    cuts += check_plan(M, C, div_up(F, BK) * seg * 2, 1, wide, false);   // dx
    cuts += check_plan(C, F, div_up(M, BK) * seg, 1, wide, false);       // dw_down
    cuts += check_plan(F, C, div_up(M, BK) * seg, 2, wide, false);       // dw_gate, dw_up
  }
  return cuts;
}

int main(int argc, char** argv) {
  if (argc > 1 && !strcmp(argv[1], "plans")) {
    const int cuts = check_plans();
    printf("%d cut products, %d faults\n", cuts, faults);
    return faults != 0 || cuts < 1000;
  }
  int combinations = 0;
  for (int W : {kSms / 2, kSms}) {
    for (int R = 1; R < W; ++R) {
      for (int nkb = 1; nkb <= 160; ++nkb, ++combinations) check_cut((nkb & 1 ? W : 0) + R, W, nkb);
      for (int nkb : {257, 333, 400, 768, 1444, 8664}) check_cut(R, W, nkb), ++combinations;
    }
  }
  printf("%d cuts, %d faults\n", combinations, faults);
  return faults != 0;
}
