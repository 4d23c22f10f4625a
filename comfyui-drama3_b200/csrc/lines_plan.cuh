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
constexpr int LP_MAX_LINES = 8192;  // three scanned int arrays of it fill 96 KB of shared memory
constexpr int LP_MAX_KEPT = 1 << 30;  // lengths are clamped to it, so no index below overflows

// The attention's work list. A unit is a tile of up to LA_ROWS rows (a row = a token and one of the `group` query
// heads of a KV head, tokens first) and the key tiles of LA_KEYS that these rows attend to. The list is the same for
// every KV head.
constexpr int LA_ROWS = 128;
constexpr int LA_KEYS = 64;
// Most rows of a KV head (T * group) whose prefix and own units may be apart: each row then keeps two fp32 partial
// rows per KV head in the attention's workspace (136 MB at 4 KV heads of 128).
constexpr int LA_APART_ROWS = 32768;
struct LaUnit {
  int line;   // the line, or -1: rows of all lines together against the prefix
  int row0;   // first row: within the line's rows (token - cu[line]) * group + head, or within the pass's
  int start;  // key tiles of the units before this one
  int tiles;  // its key tiles (>= 1)
};
// work (int32): a header, kept [B], the first unit of each line [B], then (16-byte aligned) the units
enum {
  LW_TOGETHER = 0,  // 1: a line's unit covers the prefix and then its own keys; 0: prefix units, then own units
  LW_UNITS,         // units
  LW_TILES,         // key tiles of all units (one KV head)
  LW_PREFIX_UNITS,  // units of the prefix (LW_TOGETHER == 0)
  LW_PREFIX,        // prefix length
  LW_PREFIX_TILES,  // its key tiles
  LW_TOKENS,        // tokens placed (<= T)
  LW_GROUP,
  LW_LINES,
  LW_T,
  LW_HEADER = 16
};
__host__ __device__ inline int la_unit_offset(int B) { return (LW_HEADER + 2 * B + 3) & ~3; }
__host__ __device__ inline long long la_max_units(int B, int T, int group) {
  return 2 * (((long long)T * group + LA_ROWS - 1) / LA_ROWS) + B;
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

// Key tiles that rows [row0, row0 + LA_ROWS) of a line see among its own keys: up to the last of their tokens.
D3_DEV int lp_own_tiles(int kept, int rows, int row0, int group) {
  const int last = (min(row0 + LA_ROWS, rows) - 1) / group;
  return (kept + last + LA_KEYS) / LA_KEYS;  // ceil((kept + last + 1) / LA_KEYS)
}

__global__ void __launch_bounds__(LP_THREADS) lines_plan_kernel(LinesPlanArgs a) {
  extern __shared__ int lp_smem[];
  __shared__ long long warp_sums[LP_WARPS];
  int* cu = lp_smem;               // [B + 1] first token of each line, clipped to T
  int* first = cu + a.B + 1;       // [B + 1] pages taken by the lines before; block 0: then its first unit
  int* tiles_of = first + a.B + 1;  // [B + 1] block 0: key tiles of the line, then of the lines before
  const int tid = threadIdx.x, B = a.B;
  grid_dependency_wait();
  allow_dependents();
  lp_scan_lines(B, cu, a.T, warp_sums, [&](int b) { return lp_clamped(a.counts, b); });
  const int used = max(0, *a.used);
  const int prefix = a.prefix ? max(0, *a.prefix) : 0;
  lp_scan_lines(B, first, 0x7fffffffLL, warp_sums, [&](int b) {
    const int kept = lp_clamped(a.kept, b), p = a.page;
    return (kept + cu[b + 1] - cu[b] + p - 1) / p - (kept + p - 1) / p;
  });
  if (blockIdx.x > 0) {
    // ---- tokens
    const int t0 = (blockIdx.x - 1) * LP_TOKENS, t1 = min(a.T, t0 + LP_TOKENS);
    for (int t = t0 + tid; t < t1; t += LP_THREADS) {
      int64_t slot = -1, position = 0;
      int b = -1;
      if (t < cu[B]) {
        int lo = 0, hi = B;  // the last line with cu <= t has a token there
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (cu[mid] <= t) lo = mid; else hi = mid;
        }
        b = lo;
        const int kept = lp_clamped(a.kept, b);
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
    }
    return;
  }
  // ---- block 0: the state after the pass, and the attention's work list
  const int tokens = cu[B], G = a.group;
  int over = 0;
  for (int b = tid; b < B; b += LP_THREADS) {
    const int kept = lp_clamped(a.kept, b), n = cu[b + 1] - cu[b];
    over |= n < a.counts[b];
    a.cu[b] = cu[b];
    a.lengths[b] = kept + n;
    a.work[LW_HEADER + b] = kept;
  }
  if (over) record_fault(FAULT_TOKENS);
  if (tid == 0) {
    a.cu[B] = tokens;
    *a.used_out = (int)min((long long)a.F, (long long)used + first[B]);
  }
  __syncthreads();  // every read of first[] is done: it becomes the lines' first units
  const int warp = tid >> 5, lane = tid & 31;
  lp_scan_lines(B, first, 0x7fffffffLL, warp_sums,
                [&](int b) { return ((cu[b + 1] - cu[b]) * G + LA_ROWS - 1) / LA_ROWS; });
  const int own_units = first[B];
  const int prefix_tiles = (prefix + LA_KEYS - 1) / LA_KEYS;
  const int prefix_units = prefix > 0 ? (int)(((long long)tokens * G + LA_ROWS - 1) / LA_ROWS) : 0;
  // The prefix is read once for the rows of all lines together, or by each line's units on the way to its own keys.
  // Apart, the rows of short lines share tiles: a decode step of 16 lines x 8 heads needs one tile instead of 16. But
  // each row's parts are then merged through memory, so lines that fill most of their own tiles go together.
  const bool together = prefix_units == 0 || (long long)a.T * G > LA_APART_ROWS ||
                        (long long)own_units * 4 <= (long long)prefix_units * 5;
  const int lead = together ? prefix_tiles : 0;  // key tiles ahead of each own unit's own ones
  // each own unit's key tiles, a warp per line; the units' running sum restarts at each line and is based below
  LaUnit* units = (LaUnit*)(a.work + la_unit_offset(B));
  const int u0 = together ? 0 : prefix_units;
  for (int b = warp; b < B; b += LP_WARPS) {
    const int rows = (cu[b + 1] - cu[b]) * G, n = first[b + 1] - first[b];
    const int kept = lp_clamped(a.kept, b);
    int base = 0;
    for (int i0 = 0; i0 < n; i0 += 32) {
      const int i = i0 + lane;
      const int tiles = i < n ? lead + lp_own_tiles(kept, rows, LA_ROWS * i, G) : 0;
      int incl = tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      if (i < n) units[u0 + first[b] + i] = LaUnit{b, LA_ROWS * i, base + incl - tiles, tiles};
      base += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) {
      a.work[LW_HEADER + B + b] = u0 + first[b];
      tiles_of[b] = base;
    }
  }
  __syncthreads();
  // in place: a thread's value is read into the scan before its own place is written
  lp_scan_lines(B, tiles_of, 0x7fffffffLL, warp_sums, [&](int b) { return tiles_of[b]; });
  const int own_tiles = tiles_of[B], shared_tiles = together ? 0 : prefix_units * prefix_tiles;
  for (int u = tid; u < u0; u += LP_THREADS) units[u] = LaUnit{-1, LA_ROWS * u, u * prefix_tiles, prefix_tiles};
  for (int b = warp; b < B; b += LP_WARPS)
    for (int i = first[b] + lane; i < first[b + 1]; i += 32) units[u0 + i].start += shared_tiles + tiles_of[b];
  if (tid == 0) {
    int* w = a.work;
    w[LW_TOGETHER] = together;
    w[LW_UNITS] = u0 + own_units;
    w[LW_TILES] = shared_tiles + own_tiles;
    w[LW_PREFIX_UNITS] = u0;
    w[LW_PREFIX] = prefix;
    w[LW_PREFIX_TILES] = prefix_tiles;
    w[LW_TOKENS] = tokens;
    w[LW_GROUP] = G;
    w[LW_LINES] = B;
    w[LW_T] = a.T;
  }
}

}  // namespace d3
