// The plan of a pass over lines decoded together: block tables, slot map and positions of the pass's new tokens, and
// the work list of its attention, from the lines' lengths on the device, in one launch with no host sync.
//
// Line b has kept_b tokens of its own in pages of p tokens and appends c_b. With have_b = ceil(kept_b / p) and
// need_b = ceil((kept_b + c_b) / p) it takes need_b - have_b pages off the free list, in line order:
//   first_b = sum over b' < b of (need - have),  table[b, have_b + i] = free[used + first_b + i]
// Token t of the pass belongs to the line with cu_b <= t < cu_b+1 (cu the exclusive sum of c), is the line's own
// token s = kept_b + t - cu_b, and goes to slot table[b, s / p] * p + s % p, at position prefix + s.
//
// Bound by latency: the bytes are a few per token. Every block scans the lines' counts, pages and units for itself (B
// lines, about a microsecond), so that nothing waits for another block; then the first writes the state after the pass,
// each other one places LP_TOKENS tokens, and all write units of the work list, a thread each: a unit's place follows from
// its number by a closed sum. A page is written into its table by the token that opens it, and read only from entries
// that were there before, so no two threads race. The state that a pass advances (lengths, used) goes to fresh outputs:
// planning the same pass twice gives the same plan. Measured (B200, device time in graph replays; a call from Python takes
// the host 19 us): a token each for 16 lines 4.7 us; 1024 lines of up to 512 tokens in pages of 16 (5.4 MB written) 15 us.
#pragma once

#include "common.cuh"

namespace d3 {

constexpr int LP_THREADS = 512;
constexpr int LP_WARPS = LP_THREADS / 32;
constexpr int LP_TOKENS = 2048;     // tokens placed by a block
constexpr int LP_MAX_LINES = 8192;  // four int arrays of it fill 128 KB of shared memory
constexpr int LP_MAX_TOKENS = 1 << 30;          // of a pass
constexpr int LP_MAX_KEPT = LP_MAX_TOKENS - 1;  // lengths are clamped to it: with a pass's tokens they fit 32 bits

// The attention's work list. A unit is a tile of rows, a row being a token and one of the `group` query heads of a KV
// head: la_tile_tokens(group) whole tokens, LA_ROWS rows at most; and the key tiles of LA_KEYS that these rows attend
// to. The list is the same for every KV head. Units lie end to end on a line of costs on which a key tile takes 1 and
// what a unit costs besides (its queries, its results) LA_UNIT_COST; the attention cuts that line into equal runs. (8192
// tokens of a prompt: 680 us with a cost of 1, whose first runs of a head, of many short units, were late; 601 with 2,
// 565 with 3, 556 with 4, which makes 64 lines of a token each behind 32768 2 % slower than 3.)
constexpr int LA_ROWS = 128;
constexpr int LA_KEYS = 128;
constexpr int LA_UNIT_COST = 3;
// Most rows of a KV head (T * group) whose prefix and own units may be apart: each row then keeps two fp32 partial
// rows per KV head in the attention's workspace, whether or not the pass has a prefix (136 MB at 4 KV heads of 128, 1.1 GB
// at 32). Past it every line's units read the prefix for themselves, however few of their rows are taken: 4096 lines of a
// token each behind 4096 (8 heads a KV head, 4 of 128) take 745 us of attention, 4097 take 3800.
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
  LW_PAGE,
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

// Exclusive sums over the B lines of N numbers each, f(b, v) filling v[N], into out[0 .. N - 1][0 .. B] (shared memory),
// clipped to `most`. warp_sums: LP_WARPS x N values of shared memory.
template <int N, class F>
D3_DEV void lp_scan_lines(int B, int* const (&out)[N], long long most, long long (*warp_sums)[N], F&& f) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  long long base[N] = {};
  for (int b0 = 0; b0 < B; b0 += LP_THREADS) {
    const int b = b0 + threadIdx.x;
    long long v[N] = {}, incl[N];
    if (b < B) f(b, v);
#pragma unroll
    for (int k = 0; k < N; ++k) incl[k] = v[k];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const long long u = __shfl_up_sync(0xffffffffu, incl[k], o);
        if (lane >= o) incl[k] += u;
      }
    if (lane == 31)
#pragma unroll
      for (int k = 0; k < N; ++k) warp_sums[warp][k] = incl[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
      long long total = 0, before = base[k];
#pragma unroll
      for (int w = 0; w < LP_WARPS; ++w) {
        const long long s = warp_sums[w][k];
        before += w < warp ? s : 0;
        total += s;
      }
      if (b < B) out[k][b] = (int)min(most, before + incl[k] - v[k]);
      base[k] += total;
    }
    __syncthreads();
  }
  if (threadIdx.x == 0)
#pragma unroll
    for (int k = 0; k < N; ++k) out[k][B] = (int)min(most, base[k]);
  __syncthreads();
}

// Sum over i < n of floor((a i + b) / m), by the widely published method that follows Euclid's algorithm: whole parts of
// a / m and b / m are summed up directly, and what is left counts the lattice points under a line, which turned about its
// diagonal is a sum of the same kind with a and m exchanged.
D3_DEV long long lp_floor_sum(long long n, long long m, long long a, long long b) {
  long long sum = 0;
  while (true) {
    sum += n * (n - 1) / 2 * (a / m) + n * (b / m);
    a %= m;
    b %= m;
    const long long y = a * n + b;
    if (y < m) return sum;
    n = y / m;
    b = y % m;
    const long long t = m;
    m = a;
    a = t;
  }
}

// ceil(n / of): unsigned, since n + of - 1 may pass 2^31 where n and of do not.
D3_DEV int lp_parts(int n, int of) { return (int)(((unsigned)n + (unsigned)of - 1u) / (unsigned)of); }

// What the first i units of a line cost: its tokens in tiles of `tile` (the last one shorter), each tile's key tiles up to
// its last token behind `lead` of the prefix.
D3_DEV long long lp_cost(int i, int n, int kept, int count, int tile, int lead) {
  if (i == 0) return 0;
  const int whole = i == n ? n - 1 : i;
  long long tiles = lp_floor_sum(whole, LA_KEYS, tile, (long long)kept + tile + LA_KEYS - 1);
  if (i == n) tiles += lp_parts(kept + count, LA_KEYS);
  return tiles + (long long)i * (lead + LA_UNIT_COST);
}

__global__ void __launch_bounds__(LP_THREADS) lines_plan_kernel(LinesPlanArgs a) {
  extern __shared__ int lp_smem[];
  __shared__ long long sums1[LP_WARPS][1], sums2[LP_WARPS][2];
  int* cu = lp_smem;                // [B + 1] first token of each line, clipped to T
  int* first = cu + a.B + 1;        // [B + 1] pages taken by the lines before; then what their own units cost
  int* unit0 = first + a.B + 1;     // [B + 1] own units of the lines before
  int* kept_of = unit0 + a.B + 1;   // [B] tokens that the line has
  const int tid = threadIdx.x, B = a.B, G = a.group, tile = la_tile_tokens(G);
  grid_dependency_wait();
  allow_dependents();
  const int used = max(0, *a.used);
  const int prefix = a.prefix ? max(0, *a.prefix) : 0;
  {
    int* const out[1] = {cu};
    lp_scan_lines<1>(B, out, a.T, sums1, [&](int b, long long (&v)[1]) {
      v[0] = max(0, a.counts[b]);
      kept_of[b] = min(max(0, a.kept[b]), LP_MAX_KEPT);
    });
  }
  {
    int* const out[2] = {first, unit0};
    lp_scan_lines<2>(B, out, 0x7fffffffLL, sums2, [&](int b, long long (&v)[2]) {
      const int kept = kept_of[b], n = cu[b + 1] - cu[b], p = a.page;
      v[0] = lp_parts(kept + n, p) - lp_parts(kept, p);
      v[1] = lp_parts(n, tile);
    });
  }
  const int tokens = cu[B], own_units = unit0[B];
  const int prefix_tiles = lp_parts(prefix, LA_KEYS);
  const int prefix_units = prefix > 0 ? lp_parts(tokens, tile) : 0;
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
        const int have = lp_parts(kept, a.page);
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
  } else {
    // ---- the first block: the state after the pass
    int over = 0;
    for (int b = tid; b < B; b += LP_THREADS) {
      const int n = cu[b + 1] - cu[b];
      over |= n < a.counts[b];
      a.cu[b] = cu[b];
      a.lengths[b] = kept_of[b] + n;
    }
    if (over) record_fault(FAULT_TOKENS);
    if (tid == 0) {
      a.cu[B] = tokens;
      *a.used_out = (int)min((long long)a.F, (long long)used + first[B]);
    }
  }
  // ---- all blocks: the attention's work list, a unit per thread
  __syncthreads();  // first is read no more: it becomes what the lines before cost
  {
    int* const out[1] = {first};
    lp_scan_lines<1>(B, out, 0x7fffffffLL, sums1, [&](int b, long long (&v)[1]) {
      const int n = unit0[b + 1] - unit0[b];
      v[0] = lp_cost(n, n, kept_of[b], cu[b + 1] - cu[b], tile, lead);
    });
  }
  LaUnit* units = (LaUnit*)(a.work + la_unit_offset(a.T));
  const long long shared_cost = (long long)u0 * (prefix_tiles + LA_UNIT_COST);
  for (int u = blockIdx.x * LP_THREADS + tid; u < u0 + own_units; u += gridDim.x * LP_THREADS) {
    if (u < u0) {
      units[u] = LaUnit{-1, tile * u, min(tile, tokens - tile * u) * G,
                        (int)((long long)u * (prefix_tiles + LA_UNIT_COST) + LA_UNIT_COST), prefix_tiles, 0, 0, prefix_tiles};
      continue;
    }
    int b = 0, hi = B;  // the last line whose units begin at or before this one: it has it
    while (hi - b > 1) {
      const int mid = (b + hi) >> 1;
      if (unit0[mid] <= u - u0) b = mid; else hi = mid;
    }
    const int i = u - u0 - unit0[b], n = unit0[b + 1] - unit0[b], count = cu[b + 1] - cu[b], kept = kept_of[b];
    const int from = i * tile, to = min(from + tile, count);
    const int at = (int)(shared_cost + first[b] + lp_cost(i, n, kept, count, tile, lead) + LA_UNIT_COST);
    units[u] = LaUnit{b, cu[b] + from, (to - from) * G, at, lead + lp_parts(kept + to, LA_KEYS), kept + from + 1,
                      kept + to, lead};
  }
  if (blockIdx.x == 0 && tid == 0) {
    int* w = a.work;
    w[LW_TOGETHER] = together;
    w[LW_UNITS] = u0 + own_units;
    w[LW_COST] = (int)min(0x7fffffffLL, shared_cost + first[B]);  // the attention refuses 2^30 and more
    w[LW_PREFIX] = prefix;
    w[LW_PREFIX_TILES] = prefix_tiles;
    w[LW_TOKENS] = tokens;
    w[LW_GROUP] = G;
    w[LW_LINES] = B;
    w[LW_T] = a.T;
    w[LW_PAGE] = a.page;
  }
}

}  // namespace d3
