// The plan of a pass over lines decoded together: block tables, slot map and positions of the pass's new tokens, and
// the work list of its attention, from the lines' lengths on the device, in one launch with no host sync.
//
// Line b has kept_b tokens of its own in pages of p tokens and appends c_b. With have_b = ceil(kept_b / p) and
// need_b = ceil((kept_b + c_b) / p) it takes need_b - have_b pages off the free list, in line order:
//   first_b = sum over b' < b of (need - have),  table[b, have_b + i] = free[used + first_b + i]
// Token t of the pass belongs to the line with cu_b <= t < cu_b+1 (cu the exclusive sum of c), is the line's own
// token s = kept_b + t - cu_b, and goes to slot table[b, s / p] * p + s % p, at position prefix + s.
//
// Bound by latency: the bytes are a few per token. Block 0 scans the lines and writes the work list; every other
// block repeats the scan (B lines, a few hundred nanoseconds) and places PLAN_TOKENS tokens, so nothing waits for
// another block. A page is written into its table by the token that opens it, and read only from entries that
// were there before, so no two threads race. The state that a pass advances (lengths, used) goes to fresh outputs:
// planning the same pass twice gives the same plan.
#pragma once

#include "common.cuh"

namespace d3 {

constexpr int LP_THREADS = 512;
constexpr int LP_WARPS = LP_THREADS / 32;
constexpr int LP_TOKENS = 2048;     // tokens placed by a block
constexpr int LP_MAX_LINES = 8192;  // five int arrays of it fill 160 KB of shared memory
constexpr int LP_MAX_KEPT = 1 << 30;  // lengths are clamped to it, so no index below overflows

// The attention's work list. A unit is a tile of rows, a row being a token and one of the `group` query heads of a KV
// head: la_tile_tokens(group) whole tokens, LA_ROWS rows at most; and the key tiles of LA_KEYS that these rows attend
// to. The list is the same for every KV head. Units lie end to end on a line of costs on which a key tile takes 1 and
// what a unit costs besides (its queries, its results) LA_UNIT_COST; the attention cuts that line into equal runs.
constexpr int LA_ROWS = 128;
constexpr int LA_KEYS = 128;
constexpr int LA_UNIT_COST = 1;
// Most rows of a KV head (T * group) whose prefix and own units may be apart: each row then keeps two fp32 partial
// rows per KV head in the attention's workspace (136 MB at 4 KV heads of 128).
constexpr int LA_APART_ROWS = 32768;
struct __align__(16) LaUnit {
  int line;     // the line, or -1: rows of all lines together against the prefix
  int token0;   // its first token, of the pass
  int rows;     // tokens * group
  int at;       // its first key tile's place; its cost begins LA_UNIT_COST before
  int tiles;    // its key tiles (>= 1)
  int sees;     // own keys that its first token sees (0: prefix unit)
  int own_end;  // own keys that its last token sees
  int lead;     // key tiles of the prefix at its front
};
// work (int32): a header, the own unit of each token [T], then (16-byte aligned) the units
enum {
  LW_TOGETHER = 0,  // 1: a line's unit covers the prefix and then its own keys; 0: prefix units, then own units
  LW_UNITS,         // units
  LW_COST,          // cost of all units (one KV head)
  LW_PREFIX,        // prefix length
  LW_PREFIX_TILES,  // its key tiles
  LW_TOKENS,        // tokens placed (<= T)
  LW_GROUP,
  LW_LINES,
  LW_T,
  LW_HEADER = 16
};
constexpr int LA_UNIT_INTS = sizeof(LaUnit) / 4;
__host__ __device__ inline int la_tile_tokens(int group) { return LA_ROWS / group; }
__host__ __device__ inline size_t la_unit_offset(int T) { return ((size_t)LW_HEADER + T + 3) & ~(size_t)3; }
__host__ __device__ inline long long la_max_units(int B, int T, int group) {
  const int tokens = la_tile_tokens(group);
  return 2 * (((long long)T + tokens - 1) / tokens) + B;
}

struct LinesPlanArgs {
  const int* kept;
  const int* counts;
  int B;
  int* table;
  int W;
  const int* free_pages;
  int F;
  const int* used;
  const int* prefix;  // may be null: 0
  int page;
  int T;
  int group;
  int64_t* slots;
  int64_t* positions;
  int* line;
  int* cu;
  int* lengths;
  int* used_out;
  int* work;
};

// Inclusive sum over the block; `total` the block's. `warp_sums`: LP_WARPS + 1 values of shared memory.
D3_DEV long long lp_block_scan(long long v, long long* warp_sums, long long& total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  long long incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += u;
  }
  if (lane == 31) warp_sums[warp] = incl;
  __syncthreads();
  long long before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < LP_WARPS; ++w) {
    const long long s = warp_sums[w];
    before += w < warp ? s : 0;
    total += s;
  }
  __syncthreads();
  return before + incl;
}

// Exclusive sums of f(b) over the B lines into out[0..B] (shared memory), each clipped to `most`; lines in runs of
// one per thread.
template <class F>
D3_DEV void lp_scan_lines(int B, int* out, long long most, long long* warp_sums, F&& f) {
  long long base = 0;
  for (int b0 = 0; b0 < B; b0 += LP_THREADS) {
    const int b = b0 + threadIdx.x;
    const long long v = b < B ? (long long)f(b) : 0;
    long long total;
    const long long incl = lp_block_scan(v, warp_sums, total);
    if (b < B) out[b] = (int)min(most, base + incl - v);
    base += total;
  }
  if (threadIdx.x == 0) out[B] = (int)min(most, base);
  __syncthreads();
}

D3_DEV int lp_clamped(const int* p, int b) { return min(max(0, p[b]), LP_MAX_KEPT); }

__global__ void __launch_bounds__(LP_THREADS) lines_plan_kernel(LinesPlanArgs a) {
  extern __shared__ int lp_smem[];
  __shared__ long long warp_sums[LP_WARPS];
  int* cu = lp_smem;               // [B + 1] first token of each line, clipped to T
  int* first = cu + a.B + 1;       // [B + 1] pages taken by the lines before
  int* unit0 = first + a.B + 1;    // [B + 1] own units of the lines before
  int* kept_of = unit0 + a.B + 1;  // [B] tokens that the line has
  int* cost_of = kept_of + a.B;    // [B + 1] block 0: cost of the line's units, then of the lines before
  const int tid = threadIdx.x, B = a.B;
  grid_dependency_wait();
  allow_dependents();
  lp_scan_lines(B, cu, a.T, warp_sums, [&](int b) { return lp_clamped(a.counts, b); });
  const int used = max(0, *a.used);
  const int prefix = a.prefix ? max(0, *a.prefix) : 0;
  lp_scan_lines(B, first, 0x7fffffffLL, warp_sums, [&](int b) {
    const int kept = lp_clamped(a.kept, b), p = a.page;
    kept_of[b] = kept;
    return (kept + cu[b + 1] - cu[b] + p - 1) / p - (kept + p - 1) / p;
  });
  const int G = a.group, tile = la_tile_tokens(G), tokens = cu[B];
  lp_scan_lines(B, unit0, 0x7fffffffLL, warp_sums, [&](int b) { return (cu[b + 1] - cu[b] + tile - 1) / tile; });
  const int own_units = unit0[B];
  const int prefix_tiles = (prefix + LA_KEYS - 1) / LA_KEYS;
  const int prefix_units = prefix > 0 ? (tokens + tile - 1) / tile : 0;
  // The prefix is read once for the rows of all lines together, or by each line's units on the way to its own keys.
  // Apart, the rows of short lines share tiles: a decode step of 16 lines x 8 heads needs one tile instead of 16. But
  // each row's parts are then merged through memory, so lines that fill most of their own tiles go together.
  const bool together = prefix_units == 0 || (long long)a.T * G > LA_APART_ROWS ||
                        (long long)own_units * 4 <= (long long)prefix_units * 5;
  const int lead = together ? prefix_tiles : 0;  // key tiles ahead of each own unit's own ones
  const int u0 = together ? 0 : prefix_units;    // the first own unit
  if (blockIdx.x > 0) {
    // ---- tokens
    const int t0 = (blockIdx.x - 1) * LP_TOKENS, t1 = min(a.T, t0 + LP_TOKENS);
    for (int t = t0 + tid; t < t1; t += LP_THREADS) {
      int64_t slot = -1, position = 0;
      int b = -1, unit = -1;
      if (t < tokens) {
        int lo = 0, hi = B;  // the last line with cu <= t has a token there
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (cu[mid] <= t) lo = mid; else hi = mid;
        }
        b = lo;
        const int kept = kept_of[b];
        unit = u0 + unit0[b] + (t - cu[b]) / tile;
        const int s = kept + t - cu[b], j = s / a.page, off = s - j * a.page;
        const int have = (kept + a.page - 1) / a.page;
        int page = -1;
        if (j < a.W) {
          if (j < have) {
            page = a.table[(size_t)b * a.W + j];
          } else {
            const long long at = (long long)used + first[b] + j - have;
            if (at < a.F) page = a.free_pages[at];
            if (off == 0) a.table[(size_t)b * a.W + j] = page;
          }
        }
        if (page < 0) record_fault(FAULT_PAGES);
        else slot = (int64_t)page * a.page + off;
        position = (int64_t)prefix + s;
      }
      a.slots[t] = slot;
      a.positions[t] = position;
      a.line[t] = b;
      a.work[LW_HEADER + t] = unit;
    }
    return;
  }
  // ---- block 0: the state after the pass, and the attention's work list
  int over = 0;
  for (int b = tid; b < B; b += LP_THREADS) {
    const int kept = kept_of[b], n = cu[b + 1] - cu[b];
    over |= n < a.counts[b];
    a.cu[b] = cu[b];
    a.lengths[b] = kept + n;
  }
  if (over) record_fault(FAULT_TOKENS);
  if (tid == 0) {
    a.cu[B] = tokens;
    *a.used_out = (int)min((long long)a.F, (long long)used + first[B]);
  }
  const int warp = tid >> 5, lane = tid & 31;
  // The own units, a warp per line: first what each line costs, then, with the lines' costs summed up, the units
  // themselves. (Written at once and moved to their places afterwards, each unit of a line waited for memory twice.)
  LaUnit* units = (LaUnit*)(a.work + la_unit_offset(a.T));
  auto cost_at = [&](int b, int i, int n, int count, int& from, int& to) {  // of unit i of line b, its tokens
    from = i * tile;
    to = min(from + tile, count);
    return i < n ? lead + (kept_of[b] + to + LA_KEYS - 1) / LA_KEYS + LA_UNIT_COST : 0;
  };
  for (int b = warp; b < B; b += LP_WARPS) {
    const int count = cu[b + 1] - cu[b], n = unit0[b + 1] - unit0[b];
    int sum = 0, from, to;
    for (int i = lane; i < n; i += 32) sum += cost_at(b, i, n, count, from, to);
    sum = __reduce_add_sync(0xffffffffu, sum);
    if (lane == 0) cost_of[b] = sum;
  }
  __syncthreads();
  // in place: a thread's value is read into the scan before its own place is written
  lp_scan_lines(B, cost_of, 0x7fffffffLL, warp_sums, [&](int b) { return cost_of[b]; });
  const int shared_cost = together ? 0 : prefix_units * (prefix_tiles + LA_UNIT_COST);
  for (int b = warp; b < B; b += LP_WARPS) {
    const int count = cu[b + 1] - cu[b], n = unit0[b + 1] - unit0[b];
    int base = shared_cost + cost_of[b];
    for (int i0 = 0; i0 < n; i0 += 32) {
      const int i = i0 + lane;
      int from, to;
      const int cost = cost_at(b, i, n, count, from, to);
      int incl = cost;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      const int tiles = cost - LA_UNIT_COST;
      if (i < n)
        units[u0 + unit0[b] + i] = LaUnit{b, cu[b] + from, (to - from) * G, base + incl - tiles, tiles,
                                          kept_of[b] + from + 1, kept_of[b] + to, lead};
      base += __shfl_sync(0xffffffffu, incl, 31);
    }
  }
  for (int u = tid; u < u0; u += LP_THREADS)
    units[u] = LaUnit{-1, tile * u, min(tile, tokens - tile * u) * G, u * (prefix_tiles + LA_UNIT_COST) + LA_UNIT_COST,
                      prefix_tiles, 0, 0, prefix_tiles};
  if (tid == 0) {
    int* w = a.work;
    w[LW_TOGETHER] = together;
    w[LW_UNITS] = u0 + own_units;
    w[LW_COST] = shared_cost + cost_of[B];
    w[LW_PREFIX] = prefix;
    w[LW_PREFIX_TILES] = prefix_tiles;
    w[LW_TOKENS] = tokens;
    w[LW_GROUP] = G;
    w[LW_LINES] = B;
    w[LW_T] = a.T;
  }
}

}  // namespace d3
