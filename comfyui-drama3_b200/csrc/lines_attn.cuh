// Attention of lines decoded together over a paged key/value cache: every line's tokens see all keys of a prefix that
// the lines share and the line's own keys up to their own.
//   out[t, h] = sum_j p_j V_j / sum_j p_j,   p_j = exp(scale (q_t,h . K_j - max)),   j over prefix, then own keys
// as one pass over the keys with a running maximum and sum per row, all in 32 bits; the products are 16-bit operands
// with 32-bit accumulators on the tensor cores, and p is rounded to the values' type for the second product (its sum
// is taken before the rounding).
//
// A unit (lines_plan.cuh) is a tile of up to 128 rows (whole tokens x the query heads of a KV head) and its key tiles
// of 128. The units of all KV heads, laid end to end by what they cost, are cut into equal runs, one per CTA: every CTA
// has the same work whatever the lengths are. A run crosses units; a unit cut by a run's end leaves parts, which
// lines_join_kernel joins. With few tokens a line the rows of all lines share the prefix's tiles, so that a prefix
// key is read once for all lines.
//
// Per CTA (384 threads, one per SM):
//   warps 0, 11  load by TMA (128-byte swizzle), K and V, each into a ring of stages of its own, a stage being 128
//              columns (64 for heads of 64) of a tile's 128 keys: a box per page and 64 columns, a lane each. A page outside
//              the cache reads as zeros (the map's fill). Warp 0 loads a unit's queries too, into a buffer of their own.
//   warp 1     owns the tensor memory and issues S = Q K^T (128 x 128) into three buffers by turns (two for heads of
//              256, whose O takes half of the tensor memory)
//   warps 2-9  two groups, each with a thread for every row, take the tiles by turns, so that one group's exponentials
//              run under the other's waits: S from tensor memory, mask, maximum, exponentials, P back over S, the row's
//              sum. A row's running maximum goes from group to group through shared memory; O is rescaled only when it
//              has grown by more than 2^8 since the last time (p <= 256 in between, the same value after the division;
//              in float16 p is 2^7 times that, see LA_F16_SHIFT).
//              They also write the results, half of the columns each.
//   warp 10    issues O += P V (128 x D, A = P from tensor memory, B = V as it lies in the cache: keys are its rows, so
//              it is the MN-major operand)
// Loads and first products of a run's next unit go on while the row warps write this one's results.
// Keys of a tile past the end of the prefix or of the line are masked in S, and their V rows are cleared in shared
// memory before the product, since the cache may hold anything there (0 x NaN is NaN).
// Every wait is bounded (2 s) and records FAULT_WAIT_TIMEOUT instead of hanging.
//
// A value that is not finite, at a key that only some rows of its tile see, makes the others of that line's tile NaN too:
// their weight for it is 0, and 0 x NaN is NaN.
//
// Measured (B200, bf16, 32 query heads over 4 KV heads of 128; device time in a few graph replays, in brackets the time of
// a call among many from Python, whose load lowers the clocks): 8192 tokens of a prompt 545 us, 1010 TFLOP/s (614); 16 texts
// of up to 192 tokens behind 4096 123 to 157 us from run to run, 740 to 950 TFLOP/s (143); 64 lines, a token each, behind
// 32768 66 us, 3.0 TB/s (74); 16 lines behind 4096 14.3 us (18, the host's time); one line of 1000 10.1 us (18). Heads of 256
// (16 over 2): the prompt 468 us, 1170 TFLOP/s, the texts 122 us; heads of 64: the prompt 444 us, 620 TFLOP/s. By the
// counters the prompt takes 2080 clocks a tile, units' own cost included, and the tensor cores are active for half of
// them, 1040; the texts the same. L2 and DRAM are a third busy at most: the time is that of the row groups' steps, which the
// products wait for and which wait for them.
// With few keys the time is latency: launch, loads and first product, two or three tiles, the results, then the join.
// Other forms of the same tiles: one warp that loads both K and V, 546 to 578 us for the prompt in turn with 539 to 556 for
// two, heads of 256 (16 lines behind 3001 in pages of 16) 16.6 us against 15.7; two threads a row, one group, 70 us for the
// 64 lines and 153 for the texts; two CTAs per SM with one S buffer each 74 and 165; part of the exponentials as
// polynomials, the same times as without; 216 registers for the row warps and 72 for the others, the texts 139 -> 127 us
// and the prompt 541 -> 535, but 16 lines 14.35 -> 14.7 and heads of 256 15.6 -> 15.8: not kept.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "f32x2.cuh"
#include "lines_plan.cuh"
#include "tcgen05.cuh"

namespace d3 {

constexpr int LA_THREADS = 384;
constexpr int LA_ROW_WARP = 2;        // first of the eight row warps
constexpr int LA_ROW_WARPS = 8;
constexpr int LA_PV_WARP = LA_ROW_WARP + LA_ROW_WARPS;  // issues the products with V
constexpr int LA_V_WARP = LA_PV_WARP + 1;                // loads V
constexpr int LA_SLICE = LA_KEYS * 128;  // 64 columns of a K or V tile
// Growth of the maximum, in powers of two, that rescales O. (That it may lag behind is a published method for attention on
// tensor cores: the division by the row's sum takes out whatever the weights refer to.)
constexpr float LA_RESCALE = 8.0f;
// Where the weights are held in float16 a row's refer to its maximum less this: they are 2^7 to 2^15 times what they
// weigh (float16 ends below 2^16), and float16's smallest steps, 2^-24, are 2^-31 of the largest weight and less. Against
// the maximum itself they were 2^-24 of it, and keys of less weight counted as double or as nothing beside a heavy one.
constexpr float LA_F16_SHIFT = 7.0f;

template <int D>
struct LaShape {
  // Columns of a stage, and of a product with V. Every stage costs the warp that issues the products a wait and a commit:
  // with 64 columns for heads of 128 a pair of tiles took 3850 clocks, with 128 3300.
  static constexpr int COLUMNS = D == 64 ? 64 : 128, PER_STAGE = COLUMNS / 64;
  static constexpr int STAGE = PER_STAGE * LA_SLICE;
  static constexpr int SLICES = D / COLUMNS;  // stages of a tile
  static constexpr int Q_BYTES = LA_ROWS * D * 2;
  static constexpr int K_STAGES = D == 256 ? 2 : D == 128 ? 3 : 6, V_STAGES = D == 64 ? 6 : 3;
  static constexpr int STAGES = K_STAGES + V_STAGES;  // first the ring of K, then that of V
  static constexpr int S_BUFS = D == 256 ? 2 : 3;
  static constexpr int TMEM_COLS = 512;  // O: D columns, then the S buffers of 128
  // Shared memory besides the operands: barriers and the tensor-memory address, the row threads' exchange, and the row
  // warps' copies of plan and walk (which they need only between pieces: kept in registers they were spilled inside the
  // loop over tiles).
  static constexpr int BARRIERS = 2 * STAGES + 3 * S_BUFS + 19;
  static constexpr int EXCHANGE_AT = (BARRIERS * 8 + 4 + 63) / 64 * 64, PLAN_AT = EXCHANGE_AT + LA_ROWS * 16;
  static constexpr int WALK_AT = PLAN_AT + 64, WALK_BYTES = 32;
  static constexpr int SMALL = WALK_AT + LA_ROW_WARPS * WALK_BYTES;
  static constexpr int SMEM = Q_BYTES + STAGES * STAGE + SMALL;
  static_assert(SMEM <= 227 * 1024, "a CTA fits an SM");
};

struct LaArgs {
  int T, Hq, Hkv, G;
  int pages, page, page_box;  // page_box: keys of a TMA box
  const int* table;
  int W;
  const int* prefix_table;
  int PW;
  const int* work;
  int B;
  float scale_log2;  // scale * log2(e)
  void* out;         // [T, Hq, D]
  float* lse;        // [T, Hq] or null
  float4* part_o;    // partial rows, not divided: four columns of 32 rows together, see la_part_at
  float2* part_ml;   // their (maximum * scale_log2, sum)
  int4* joints;      // [runs] the unit that is first cut at this run's start: token0, rows, head, last run; or rows 0
  int units_most;    // units that the plan has room for
  int runs;          // CTAs
};

// Partial rows: LA_ROWS for the part that a run starts in the middle of a unit, LA_ROWS for the part that it leaves
// unfinished, then (prefix and own units apart) the first part of every row's prefix unit and of its own unit, by the
// row's number token * G + head.
D3_DEV long long la_part_rest(int run) { return (long long)run * LA_ROWS; }
D3_DEV long long la_part_open(const LaArgs& a, int run) { return (long long)(a.runs + run) * LA_ROWS; }
__host__ __device__ inline long long la_apart_rows(int T, int G) { return ((long long)T * G + 31) & ~31ll; }
D3_DEV long long la_part_apart(const LaArgs& a, bool own, int h) {
  return (long long)2 * a.runs * LA_ROWS + ((long long)(own ? a.Hkv : 0) + h) * la_apart_rows(a.T, a.G);
}
__host__ __device__ inline long long la_part_rows(int runs, int T, int G, int Hkv) {
  return (long long)2 * runs * LA_ROWS + ((long long)T * G <= LA_APART_ROWS ? 2ll * Hkv * la_apart_rows(T, G) : 0);
}
// Where columns 4c .. 4c + 3 of partial row r are: the same columns of 32 neighbouring rows together, so that a warp
// whose lanes are rows writes and reads them as 512 bytes in a row.
template <int D>
D3_DEV long long la_part_at(long long r, int c) {
  return ((r >> 5) * (D / 4) + c) * 32 + (r & 31);
}

// The header of the work list, and the length of a run.
struct LaPlan {
  bool together;
  int units_n, cost, prefix, prefix_tiles, tokens;
  bool fits;
  int per, total;  // of all KV heads; a plan of 2^30 or more is refused
  int runs;        // with something to do
  const LaUnit* units;
  D3_DEV LaPlan(const LaArgs& a, int& probe) {
    units = (const LaUnit*)(a.work + la_unit_offset(a.T));
    // a first probe for find, on its way with the header: where the first 32 units begin
    probe = __ldg(&units[min((int)threadIdx.x & 31, a.units_most - 1)].at) - LA_UNIT_COST;
    const int4 x = __ldg((const int4*)a.work), y = __ldg((const int4*)a.work + 1);
    const int2 z = __ldg((const int2*)(a.work + LW_T));
    static_assert(LW_GROUP == 6 && LW_LINES == 7 && LW_T == 8 && LW_PAGE == 9, "as they are read");
    together = x.x != 0;
    units_n = x.y;
    cost = x.z;
    prefix = x.w;
    prefix_tiles = y.x;
    tokens = y.y;
    const long long all = (long long)cost * a.Hkv;
    fits = y.z == a.G && y.w == a.B && z.x == a.T && z.y == a.page && all < 0x40000000;
    total = fits ? (int)all : 0;
    per = max((int)((unsigned)(total + a.runs - 1) / (unsigned)a.runs), 1);
    runs = (unsigned)(total + per - 1) / (unsigned)per;
  }
  D3_DEV LaUnit unit(int u) const {
    const int4 x = __ldg((const int4*)(units + u)), y = __ldg((const int4*)(units + u) + 1);
    return LaUnit{x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
  }
  // The last unit that begins at or before `place`, by the whole warp: 32 probes a round.
  D3_DEV int find(int place, int probe) const {
    const int lane = threadIdx.x & 31;
    if (units_n <= 32) return __popc(__ballot_sync(0xffffffffu, lane < units_n && probe <= place)) - 1;
    int lo = 0, n = units_n;  // the answer is in [lo, lo + n)
    while (n > 1) {
      const int step = (n + 31) / 32;
      const bool below = lane * step < n && __ldg(&units[lo + lane * step].at) - LA_UNIT_COST <= place;
      const int hit = __popc(__ballot_sync(0xffffffffu, below)) - 1;
      n = min(step, n - hit * step);
      lo += hit * step;
    }
    return lo;
  }
};

// A CTA's run, piece by piece (a piece: consecutive key tiles of one unit, one at least). Every warp walks it by
// itself; the next unit is on its way while this one is worked on.
struct LaWalk {
  int pos, end;  // where the run goes on and ends
  int head0;     // where the KV head's units begin
  int h, u;
  int j0, n;     // the piece: tiles [j0, j0 + n) of unit u
  int tiles;     // of the unit

  D3_DEV LaWalk(const LaPlan& p, int run, int probe) {
    pos = p.per * run;
    end = p.fits ? min(pos + p.per, p.total) : 0;
    if (pos < end) {
      h = (unsigned)pos / (unsigned)p.cost;
      head0 = h * p.cost;
      u = p.find(pos - head0, probe);
    }
  }
  D3_DEV bool next(const LaPlan& p, LaUnit& unit) {
    while (pos < end) {
      unit = p.unit(u);
      tiles = unit.tiles;
      const int first = head0 + unit.at;
      j0 = max(0, pos - first);
      n = min(end, first + unit.tiles) - first - j0;
      pos = first + j0;
      if (n > 0) {
        asm volatile("prefetch.global.L1 [%0];" ::"l"(p.units + (u + 1 < p.units_n ? u + 1 : 0)));
        return true;
      }
      pos = end;  // it ends before the unit's first tile
    }
    return false;
  }
  D3_DEV void step(const LaPlan& p) {
    pos += n;
    if (j0 + n == tiles && ++u == p.units_n) {
      u = 0;
      ++h;
      head0 += p.cost;
    }
  }
};

// First key of tile j of a unit (of the prefix when own is false) and how many of its LA_KEYS there are.
D3_DEV int la_tile(const LaPlan& p, const LaUnit& u, int j, bool& own, int& valid) {
  own = j >= u.lead;
  const int key0 = (own ? j - u.lead : j) * LA_KEYS;
  valid = min(LA_KEYS, (own ? u.own_end : p.prefix) - key0);
  return key0;
}

// Shared-memory descriptor of V stages as the MMA's B: MN-major (columns contiguous), 128-byte swizzle, atoms of 8
// keys x 64 columns 1024 bytes apart along the keys (SBO) and LA_SLICE apart along the columns (LBO).
D3_DEV uint64_t la_v_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(LA_SLICE >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// The MMA warp runs its loop with all lanes, so that descriptors stay in uniform registers, and issues from the lane
// that elect.sync names. (Issued from a branch on the lane number, each MMA paid about 100 cycles to move its
// operands into uniform registers: twelve a tile, twice the time of the products themselves.)
D3_DEV uint32_t la_elect() {
  uint32_t e;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(e));
  return e;
}
// D (+)= A B, both from shared memory.
D3_DEV void la_mma_ss(uint32_t elected, uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                      uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(elected)
      : "memory");
}
// D (+)= A B with A in tensor memory (16-bit values, two to a column).
D3_DEV void la_mma_ts(uint32_t elected, uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc,
                      uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(elected)
      : "memory");
}
D3_DEV void la_commit(uint32_t elected, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
      "r"(elected)
      : "memory");
}

#define LA_R8(r, o) \
  "=r"(r[o]), "=r"(r[o + 1]), "=r"(r[o + 2]), "=r"(r[o + 3]), "=r"(r[o + 4]), "=r"(r[o + 5]), "=r"(r[o + 6]), "=r"(r[o + 7])
#define LA_V8(r, o) \
  "r"(r[o]), "r"(r[o + 1]), "r"(r[o + 2]), "r"(r[o + 3]), "r"(r[o + 4]), "r"(r[o + 5]), "r"(r[o + 6]), "r"(r[o + 7])

// 32 or 64 columns of this warp's 32 lanes. The wait is part of the statement, so that nothing reads the registers
// ahead of it.
D3_DEV void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : LA_R8(r, 0), LA_R8(r, 8), LA_R8(r, 16), LA_R8(r, 24)
      : "r"(taddr)
      : "memory");
}
D3_DEV void tmem_ld64(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,"
      "%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : LA_R8(r, 0), LA_R8(r, 8), LA_R8(r, 16), LA_R8(r, 24), LA_R8(r, 32), LA_R8(r, 40), LA_R8(r, 48), LA_R8(r, 56)
      : "r"(taddr)
      : "memory");
}
D3_DEV void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"
      "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::LA_V8(r, 0),
      LA_V8(r, 8), LA_V8(r, 16), LA_V8(r, 24), "r"(taddr)
      : "memory");
}
D3_DEV void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::LA_V8(r, 0),
      LA_V8(r, 8), "r"(taddr)
      : "memory");
}
D3_DEV void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Box of the 4-D cache map (column, key in page, head, page).
D3_DEV void tma_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(dst),
      "l"((uint64_t)map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar))
      : "memory");
}

// mbar_wait by a whole warp, with the same answer for all of its lanes, together again afterwards (the tensor-memory
// instructions and shuffles that follow are the warp's).
D3_DEV bool la_warp_wait(uint64_t* bar, uint32_t parity) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  const unsigned long long start = globaltimer();
#pragma unroll 1
  do {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  } while (__any_sync(0xffffffffu, globaltimer() - start < WAIT_LIMIT_NS));
  record_fault(FAULT_WAIT_TIMEOUT);
  return false;
}

D3_DEV float la_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

D3_DEV float la_max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

template <bool F16>
D3_DEV uint32_t la_pack(float lo, float hi) {
  uint32_t r;
  if (F16)
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

struct LaLimited { static constexpr bool value = true; };
struct LaWhole { static constexpr bool value = false; };

template <int D, bool F16>
__global__ void __launch_bounds__(LA_THREADS, 1)
    lines_attn_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                      const __grid_constant__ CUtensorMap vmap, LaArgs a) {
  using S = LaShape<D>;
  extern __shared__ __align__(1024) uint8_t la_smem[];
  uint8_t* q_s = la_smem;
  uint8_t* ring = la_smem + S::Q_BYTES;
  uint64_t* bars = (uint64_t*)(la_smem + S::Q_BYTES + S::STAGES * S::STAGE);
  uint8_t* small = (uint8_t*)bars;
  LaPlan* plan_s = (LaPlan*)(small + S::PLAN_AT);
  LaWalk* walk_s = (LaWalk*)(small + S::WALK_AT) + (threadIdx.x >> 5) - LA_ROW_WARP;
  static_assert(sizeof(LaPlan) <= 64 && sizeof(LaWalk) == S::WALK_BYTES, "layout");
  uint64_t* kv_full = bars;                    // [STAGES]
  uint64_t* kv_empty = kv_full + S::STAGES;    // [STAGES]
  uint64_t* v_full = kv_full + S::K_STAGES;
  uint64_t* q_full = kv_empty + S::STAGES;
  uint64_t* q_empty = q_full + 1;
  uint64_t* s_full = q_empty + 1;              // [S_BUFS]
  uint64_t* p_full = s_full + S::S_BUFS;       // [S_BUFS][2], by halves of the keys
  uint64_t* o_full = p_full + 2 * S::S_BUFS;   // [4], of tiles by turns: a waiter may be up to three products behind
  uint64_t* o_empty = o_full + 4;
  uint64_t* m_full = o_empty + 1;              // [2][4], by group and quarter
  uint64_t* l_full = m_full + 8;               // [4]
  uint32_t* tmem_slot = (uint32_t*)(l_full + 4);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, run = blockIdx.x;
  const bool aligned = (smem_u32(la_smem) & 1023u) == 0;  // the swizzle's atoms
  if (tid == 0) {
    for (int i = 0; i < S::STAGES; ++i) {
      mbar_init(kv_full + i, 1);
      mbar_init(kv_empty + i, 1);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < S::S_BUFS; ++i) {
      mbar_init(s_full + i, 1);
      mbar_init(p_full + 2 * i, LA_ROW_WARPS / 2);
      mbar_init(p_full + 2 * i + 1, LA_ROW_WARPS / 2);
    }
    for (int i = 0; i < 4; ++i) mbar_init(o_full + i, 1);
    mbar_init(o_empty, LA_ROW_WARPS);
    for (int i = 0; i < 8; ++i) mbar_init(m_full + i, 1);
    for (int i = 0; i < 4; ++i) mbar_init(l_full + i, 2);
    fence_mbar_init();
  }
  // tensor memory only once the grids before this one are done: a CTA that held some while it waited for them could
  // keep one of theirs from its own
  grid_dependency_wait();
  if (warp == 1) tmem_alloc(tmem_slot, S::TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  allow_dependents();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tmem_o = tmem, tmem_s = tmem + D;  // S buffer b: columns D + 128 b;
  // P of its keys 32 j .. 32 j + 31 in the first 16 columns of theirs
  int probe;
  LaPlan plan(a, probe);
  if (!plan.fits || !aligned) {
    plan.fits = false;
    if (tid == 0) record_fault(FAULT_PLAN);
  }
  LaWalk w(plan, run, probe);
  const uint32_t type = F16 ? 0u : (1u << 7) | (1u << 10);  // of the products' operands

  if (warp == 0 || warp == LA_V_WARP) {
    // ---- loads: warp 0 a piece's Q and K of its tiles, the other V
    const bool is_v = warp != 0;
    const CUtensorMap* map = is_v ? &vmap : &kmap;
    const uint32_t stages = is_v ? S::V_STAGES : S::K_STAGES, stage0 = is_v ? S::K_STAGES : 0;
    uint32_t st = 0, ph = 0, loads = 0, pieces = 0;
    bool ok = true;
    int win_first = 0, win_page = -1;  // a window of 32 page ids, one per lane
    const int* win_table = nullptr;
    const uint32_t q_bytes = (uint32_t)(la_tile_tokens(a.G) * a.G * 128);  // of a 64-column slice
    for (LaUnit unit; ok && w.next(plan, unit); w.step(plan)) {
      if (!is_v) {
        if (!(ok = la_warp_wait(q_empty, (pieces & 1) ^ 1))) break;
        ++pieces;
        if (lane == 0) mbar_arrive_expect_tx(q_full, q_bytes * (D / 64));
        __syncwarp();
        if (lane < D / 64)
          tma_load_3d(smem_u32(q_s) + lane * (LA_ROWS * 128), &qmap, lane * 64, w.h * a.G, unit.token0, q_full);
      }
      for (int i = 0; ok && i < w.n; ++i) {
        bool own;
        int valid;
        const int key0 = la_tile(plan, unit, w.j0 + i, own, valid);
        const int boxes = (valid + a.page_box - 1) / a.page_box;  // lane l issues box l
        const int key = key0 + lane * a.page_box, first = key0 / a.page, last = (key0 + valid - 1) / a.page;
        const int* table = own ? a.table + (size_t)unit.line * a.W : a.prefix_table;
        const int width = own ? a.W : a.PW;
        if (table != win_table || first < win_first || last >= win_first + 32) {
          win_table = table;
          win_first = first;
          win_page = first + lane < width ? table[first + lane] : -1;
        }
        const int index = key / a.page;
        const int in_page = key - index * a.page;
        int page_id = __shfl_sync(0xffffffffu, win_page, (index - win_first) & 31);
        if (lane < boxes && (page_id < 0 || page_id >= a.pages)) {
          record_fault(FAULT_PAGES);
          page_id = -1;  // outside the map: zeros
        }
#pragma unroll
        for (int sl = 0; ok && sl < S::SLICES; ++sl) {
          uint64_t* full = kv_full + stage0 + st;
          if (!(ok = la_warp_wait(kv_empty + stage0 + st, ph ^ 1))) break;
          if (lane == 0) mbar_arrive_expect_tx(full, boxes * a.page_box * 128 * S::PER_STAGE);
          __syncwarp();
          if (lane < boxes)
#pragma unroll
            for (int y = 0; y < S::PER_STAGE; ++y)
              tma_load_4d(smem_u32(ring) + (stage0 + st) * S::STAGE + y * LA_SLICE + lane * a.page_box * 128, map,
                          sl * S::COLUMNS + y * 64, in_page, w.h, page_id, full);
          ++loads;
          if (++st == stages) {
            st = 0;
            ph ^= 1;
          }
        }
      }
    }
    // nothing may land after the CTA is gone: a stage's last load has arrived once its phase is complete
    if (pieces > 0) mbar_wait(q_full, (pieces - 1) & 1);
    for (uint32_t i = loads < stages ? 0 : loads - stages; i < loads; ++i)
      mbar_wait(kv_full + stage0 + i % stages, (i / stages) & 1);
  } else if (warp == 1) {
    // ---- S = Q K^T, up to S_BUFS - 1 tiles ahead of O
    const uint32_t idesc = (1u << 4) | type | ((LA_KEYS >> 3) << 17) | ((LA_ROWS >> 4) << 24);
    const uint32_t elected = la_elect();
    const uint64_t q_desc = umma_desc_sw128(smem_u32(q_s)), k_desc = umma_desc_sw128(smem_u32(ring));
    uint32_t tile = 0, pieces = 0;
    bool ok = true;
    for (LaUnit unit; ok && w.next(plan, unit); w.step(plan)) {
      if (!(ok = la_warp_wait(q_full, pieces & 1))) break;
      ++pieces;
      for (int i = 0; ok && i < w.n; ++i, ++tile) {
        const uint32_t d = tmem_s + 128 * (tile % S::S_BUFS), done = tile - S::S_BUFS;
        // where P of the tile S_BUFS before was
        if (tile >= (uint32_t)S::S_BUFS && !(ok = la_warp_wait(o_full + done % 4, (done / 4) & 1))) break;
        const uint32_t k0 = S::SLICES * tile;
#pragma unroll
        for (int sl = 0; sl < S::SLICES; ++sl) {
          const uint32_t st = (k0 + sl) % S::K_STAGES;
          if (!ok || !(ok = la_warp_wait(kv_full + st, ((k0 + sl) / S::K_STAGES) & 1))) break;
          tc_fence_after();
          const uint64_t kb = k_desc + st * (S::STAGE >> 4), qb = q_desc + sl * S::PER_STAGE * (LA_ROWS * 128 >> 4);
#pragma unroll
          for (int y = 0; y < S::PER_STAGE; ++y)
#pragma unroll
            for (int c = 0; c < 4; ++c)
              la_mma_ss(elected, d, qb + y * (LA_ROWS * 128 >> 4) + 2 * c, kb + y * (LA_SLICE >> 4) + 2 * c, idesc,
                        sl > 0 || y > 0 || c > 0);
          la_commit(elected, kv_empty + st);
        }
        if (!ok) break;
        if (i + 1 == w.n) la_commit(elected, q_empty);
        la_commit(elected, s_full + tile % S::S_BUFS);
      }
    }
  } else if (warp == LA_PV_WARP) {
    // ---- O += P V
    const uint32_t idesc = (1u << 4) | type | (1u << 16) | ((S::COLUMNS >> 3) << 17) | ((LA_ROWS >> 4) << 24);
    const uint32_t elected = la_elect();
    const uint64_t v_desc = la_v_desc(smem_u32(ring) + S::K_STAGES * S::STAGE);  // in 16-byte units: sums stay within 14 bits
    uint32_t tile = 0, pieces = 0;
    bool ok = true;
    for (LaUnit unit; ok && w.next(plan, unit); w.step(plan)) {
      ++pieces;
      for (int i = 0; ok && i < w.n; ++i, ++tile) {
        const uint32_t buf = tile % S::S_BUFS, v0 = S::SLICES * tile;
#pragma unroll
        for (int sl = 0; sl < S::SLICES; ++sl)
          ok = ok && la_warp_wait(v_full + (v0 + sl) % S::V_STAGES, ((v0 + sl) / S::V_STAGES) & 1);
        if (i == 0) ok = ok && la_warp_wait(o_empty, pieces & 1);  // the rows have read the O before it
        // the product by halves of the keys, as their weights come: keys 64 .. 127, then the others
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          if (!ok || !(ok = la_warp_wait(p_full + 2 * buf + part, (tile / S::S_BUFS) & 1))) break;
          tc_fence_after();
#pragma unroll
          for (int sl = 0; sl < S::SLICES; ++sl) {
            const uint32_t st = (v0 + sl) % S::V_STAGES;
            const uint64_t vb = v_desc + st * (S::STAGE >> 4);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int c = x + 4 * (1 - part);  // 16 keys
              la_mma_ts(elected, tmem_o + S::COLUMNS * sl, tmem_s + 128 * buf + 32 * (c >> 1) + 8 * (c & 1),
                        vb + (c * 2048 >> 4), idesc, i > 0 || part > 0 || x > 0);
            }
            if (part == 1) la_commit(elected, kv_empty + S::K_STAGES + st);
          }
        }
        if (ok) la_commit(elected, o_full + tile % 4);
      }
    }
  } else {
    // ---- rows
    const int quarter = warp & 3, group = (warp - LA_ROW_WARP) >> 2;  // tensor-memory lanes; tiles of its parity
    const uint32_t lanes = (uint32_t)(32 * quarter) << 16;
    const int row = 32 * quarter + lane, tok = row / a.G, g = row - tok * a.G;
    if (lane == 0) {
      if (warp == LA_ROW_WARP) {
        *plan_s = plan;
        a.joints[run] = make_int4(0, 0, 0, 0);
      }
      *walk_s = w;
    }
    named_sync(9, 32 * LA_ROW_WARPS);
    // between a row's two threads: the running maximum, of pieces by turns, and their sums
    float* m_s = (float*)(small + S::EXCHANGE_AT) + row;
    float* l_s = m_s + 2 * LA_ROWS;
    uint32_t tiles = 0, pieces = 0;
    bool ok = true;
    while (ok) {
      int n, n_shared;  // tiles of the piece, and those of them that are the prefix's
      // keys that there are, from the piece's first tile on: of the prefix, of the line, of these that this row sees
      int shared_end, own_end, own_sees;
      bool any;  // whether this warp has rows
      {
        LaWalk w = *walk_s;
        __syncwarp();
        LaUnit unit;
        if (!w.next(*plan_s, unit)) break;
        if (lane == 0) *walk_s = w;
        __syncwarp();
        n = w.n;
        n_shared = unit.lead - w.j0;
        shared_end = plan_s->prefix - w.j0 * LA_KEYS;
        own_end = unit.own_end - (w.j0 - unit.lead) * LA_KEYS;
        own_sees = unit.sees + tok - (w.j0 - unit.lead) * LA_KEYS;
        any = 32 * quarter < unit.rows;
      }
      float* m_row = m_s + (pieces & 1) * LA_ROWS;
      // this thread's sum, and the maximum that it refers to
      float m = -INFINITY, l = 0.0f;
      auto refer = [&](float to) {
        if (to != m) {
          l *= m == -INFINITY ? 0.0f : la_exp2(m - to);
          m = to;
        }
      };
      for (int i = (tiles ^ group) & 1; i < n; i += 2) {
        const uint32_t tile = tiles + i, buf = tile % S::S_BUFS;
        if (!(ok = la_warp_wait(s_full + buf, (tile / S::S_BUFS) & 1))) break;
        tc_fence_after();
        const int valid = (i < n_shared ? shared_end : own_end) - i * LA_KEYS;  // keys of this tile, if not all
        if (valid < LA_KEYS) {
          // V's rows past the end, in the stages of this tile's V. A wait for a phase passes, too, while the phase before
          // it is not complete: where the last tile's V may still be coming into one of these stages, its product first.
          if (S::SLICES > 1 && !(ok = la_warp_wait(o_full + (tile - 1) % 4, ((tile - 1) / 4) & 1))) break;
          const uint32_t vs = S::SLICES * tile;
          for (int sl = 0; ok && sl < S::SLICES; ++sl) {
            const uint32_t st = (vs + sl) % S::V_STAGES;
            if (!(ok = la_warp_wait(v_full + st, ((vs + sl) / S::V_STAGES) & 1))) break;
            for (int r = valid + 4 * quarter + (lane >> 3); r < LA_KEYS; r += 2 * LA_ROW_WARPS)
#pragma unroll
              for (int y = 0; y < S::PER_STAGE; ++y)
                *(uint4*)(ring + (S::K_STAGES + st) * S::STAGE + y * LA_SLICE + r * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
          if (!ok) break;
          fence_async_smem();
          __syncwarp();
        }
        if (any) {
          const uint32_t s_at = tmem_s + lanes + 128 * buf;
          // of the tile's keys, those that there are and that this row sees
          const int lim = i < n_shared ? valid : own_sees - i * LA_KEYS;
          // Two forms of the same steps, with and without a limit inside the tile, chosen by the whole warp: with the
          // comparisons in the one form every tile paid for them.
          const bool cut_tile = __any_sync(0xffffffffu, lim < LA_KEYS);
          uint32_t s[64];
          auto load = [&](int key, auto limited) {
            tmem_ld64(s_at + key, s);
            if constexpr (decltype(limited)::value) {  // -inf past the limit
#pragma unroll
              for (int x = 0; x < 64; ++x)
                if (key + x >= lim) s[x] = 0xff800000u;
            }
          };
          auto maximum = [&](auto limited) {
            float t[4];  // four chains
            load(0, limited);
#pragma unroll
            for (int x = 0; x < 4; ++x) t[x] = fmaxf(__uint_as_float(s[x]), __uint_as_float(s[x + 4]));
#pragma unroll
            for (int x = 8; x < 64; x += 8)
#pragma unroll
              for (int y = 0; y < 4; ++y)
                t[y] = la_max3(t[y], __uint_as_float(s[x + y]), __uint_as_float(s[x + y + 4]));
            load(64, limited);
#pragma unroll
            for (int x = 0; x < 64; x += 8)
#pragma unroll
              for (int y = 0; y < 4; ++y)
                t[y] = la_max3(t[y], __uint_as_float(s[x + y]), __uint_as_float(s[x + y + 4]));
            return fmaf(fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])), a.scale_log2, F16 ? -LA_F16_SHIFT : 0.0f);
          };
          float top = cut_tile ? maximum(LaLimited{}) : maximum(LaWhole{});
          float before = -INFINITY;
          if (i > 0) {
            if (!(ok = la_warp_wait(m_full + 4 * (1 - group) + quarter, ((tile - 1) >> 1) & 1))) break;
            before = *m_row;
            if (!(top > before + LA_RESCALE || (before == -INFINITY && top > before))) top = before;
          }
          *m_row = top;
          __syncwarp();
          if (lane == 0) mbar_arrive(m_full + 4 * group + quarter);
          refer(top);
          if (i > 0 && __any_sync(0xffffffffu, top != before)) {
            const float f = top == before ? 1.0f : before == -INFINITY ? 0.0f : la_exp2(before - top);
            if (!(ok = la_warp_wait(o_full + (tile - 1) % 4, ((tile - 1) / 4) & 1))) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              uint32_t o[32];
              const uint32_t at = tmem_o + lanes + c;
              tmem_ld32(at, o);
#pragma unroll
              for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
              tmem_st32(at, o);
            }
            tmem_wait_st();
          }
          const float base = m == -INFINITY ? 0.0f : m;
          const uint64_t scale2 = f2_make(a.scale_log2, a.scale_log2), base2 = f2_make(-base, -base);
          uint64_t sums[2] = {0, 0};
          auto weigh = [&](int key, int c) {  // s[c] is key `key`
            uint32_t p[16];
#pragma unroll
            for (int x = 0; x < 32; x += 2) {
              const uint64_t y =
                  f2_fma(f2_make(__uint_as_float(s[c + x]), __uint_as_float(s[c + x + 1])), scale2, base2);
              float p0, p1;
              f2_split(y, p0, p1);
              p0 = la_exp2(p0);
              p1 = la_exp2(p1);
              sums[x / 2 & 1] = f2_add(sums[x / 2 & 1], f2_make(p0, p1));
              p[x / 2] = la_pack<F16>(p0, p1);
            }
            tmem_st16(s_at + key, p);
          };
          auto weights = [&](auto limited) {
#pragma unroll 1
            for (int part = 0; part < 2; ++part) {  // keys 64 .. 127, still in registers, then the others
              if (part == 1) load(0, limited);
              weigh(64 * (1 - part), 0);
              weigh(64 * (1 - part) + 32, 32);
              tmem_wait_st();
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(p_full + 2 * buf + part);
            }
          };
          if (cut_tile)
            weights(LaLimited{});
          else
            weights(LaWhole{});
          float s0, s1;
          f2_split(f2_add(sums[0], sums[1]), s0, s1);
          l += s0 + s1;
        } else if (lane == 0) {
          mbar_arrive(m_full + 4 * group + quarter);
          mbar_arrive(p_full + 2 * buf);
          mbar_arrive(p_full + 2 * buf + 1);
        }
      }
      if (!ok) break;
      tiles += n;
      const uint32_t end = tiles - 1;
      if (!(ok = la_warp_wait(o_full + end % 4, (end / 4) & 1))) break;
      tc_fence_after();
      if (!(ok = la_warp_wait(m_full + 4 * (end & 1) + quarter, (end >> 1) & 1))) break;
      // the row's sum: both threads', the same order in both
      if (any) refer(*m_row);
      l_s[group * LA_ROWS] = l;
      __syncwarp();
      if (lane == 0) mbar_arrive(l_full + quarter);
      if (!(ok = la_warp_wait(l_full + quarter, pieces & 1))) break;
      l = l_s[0] + l_s[LA_ROWS];
      ++pieces;
      // results: a whole unit's rows are done; a part's go to the workspace
      const LaPlan plan = *plan_s;
      LaWalk w = *walk_s;
      const LaUnit unit = plan.unit(w.u);
      const bool live = row < unit.rows;
      const bool first = w.j0 == 0, last = w.j0 + w.n == unit.tiles;
      const bool whole = first && last && plan.together;
      long long part = row;
      if (!first)
        part += la_part_rest(run);
      else if (!plan.together)
        part += la_part_apart(a, unit.line >= 0, w.h) + (long long)unit.token0 * a.G;
      else
        part += la_part_open(a, run);
      if (!first && plan.together && tid == 32 * LA_ROW_WARP) {
        // a unit's first cut: it is joined under this run's number
        const int from = w.head0 + unit.at;
        if (from / plan.per == run - 1)
          a.joints[run] = make_int4(unit.token0, unit.rows, w.h, (from + unit.tiles - 1) / plan.per);
      }
      if (any) {
        const int t = unit.token0 + tok, head = w.h * a.G + g, half = group;  // a thread takes half of the columns
        const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
#pragma unroll 1
        for (int c = half * (D / 2); c < (half + 1) * (D / 2); c += 32) {
          uint32_t o[32];
          tmem_ld32(tmem_o + lanes + c, o);
          if (live && whole) {
            uint4* dst = (uint4*)((uint16_t*)a.out + ((long long)t * a.Hq + head) * D + c);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              uint32_t v[4];
#pragma unroll
              for (int y = 0; y < 4; ++y)
                v[y] = la_pack<F16>(__uint_as_float(o[8 * x + 2 * y]) * inv, __uint_as_float(o[8 * x + 2 * y + 1]) * inv);
              dst[x] = make_uint4(v[0], v[1], v[2], v[3]);
            }
          } else if (live) {
            uint4* dst = (uint4*)a.part_o + la_part_at<D>(part, c / 4);
#pragma unroll
            for (int x = 0; x < 8; ++x)
              dst[32 * x] = make_uint4(o[4 * x], o[4 * x + 1], o[4 * x + 2], o[4 * x + 3]);
          }
        }
        if (live && group == 0) {
          if (!whole)
            a.part_ml[part] = make_float2(m, l);
          else if (a.lse)
            a.lse[(long long)t * a.Hq + head] = (m + log2f(l)) * 0.69314718055994531f;
        }
      }
      tc_fence_before();
      w.step(plan);
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(o_empty);
        *walk_s = w;
      }
      __syncwarp();
    }
    // tokens of no line, or of a plan that does not fit the call: nothing to see
    const int tokens = plan.fits ? plan.tokens : 0;
    const long long total = (long long)(a.T - tokens) * a.Hq;
    for (long long x = (long long)run * LA_ROW_WARPS + warp - LA_ROW_WARP; x < total;
         x += (long long)a.runs * LA_ROW_WARPS) {
      const long long r = (long long)tokens * a.Hq + x;
      for (int c = lane; c < D / 8; c += 32)
        *(uint4*)((uint16_t*)a.out + r * D + 8 * c) = make_uint4(0, 0, 0, 0);
      if (a.lse && lane == 0) a.lse[r] = -INFINITY;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, S::TMEM_COLS);
  }
}

// The joining: with M the largest of a row's parts' maxima, out = sum 2^(m_i - M) O_i / sum 2^(m_i - M) l_i, the parts
// taken in order. A lane is a row (of 32 neighbouring ones of a KV head), a warp takes groups of four columns. Bound
// by latency: N x AHEAD loads are in flight at a time; 2 to 3 us of a decode step's attention. (A counter per cut unit would
// let the last CTA to arrive join its parts, in the same order, without this launch; not built.)
// The parts of a row: `first`, then those that the runs r0 + 1 .. r1 left at `rest` rows into theirs.
struct LaParts {
  long long first;
  int rest, r0, r1;
};

// Columns 4c .. 4c + 4N - 1 of a row whose parts are p's, then q's.
template <int D, bool F16, int N, int AHEAD>
D3_DEV void la_join_row(const LaArgs& a, int c, bool live, const LaParts& p, const LaParts& q, int t, int head) {
  const int np = live ? p.r1 - p.r0 + 1 : 0, n = live ? np + q.r1 - q.r0 + 1 : 0;
  const int longest = __reduce_max_sync(0xffffffffu, n);
  float M = -INFINITY, L = 0.0f;
  float4 o[N];
#pragma unroll
  for (int k = 0; k < N; ++k) o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
  for (int i0 = 0; i0 < longest; i0 += AHEAD) {
    float2 ml[AHEAD];
    float4 v[AHEAD][N];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int i = i0 + j;
      ml[j] = make_float2(-INFINITY, 0.0f);
      if (i < n) {
        const long long r = i < np ? (i == 0 ? p.first : la_part_rest(p.r0 + i) + p.rest)
                                   : (i == np ? q.first : la_part_rest(q.r0 + i - np) + q.rest);
        ml[j] = a.part_ml[r];
#pragma unroll
        for (int k = 0; k < N; ++k) v[j][k] = a.part_o[la_part_at<D>(r, c + k)];
      }
    }
    float top = M;
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) top = fmaxf(top, ml[j].x);
    const float base = top == -INFINITY ? 0.0f : top;
    const float f = la_exp2(M - base);  // 0 at first
    L *= f;
#pragma unroll
    for (int k = 0; k < N; ++k) o[k].x *= f, o[k].y *= f, o[k].z *= f, o[k].w *= f;
    M = top;
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      if (ml[j].y == 0.0f) continue;  // nothing there (a NaN stays one)
      const float g = la_exp2(ml[j].x - base);
      L = fmaf(g, ml[j].y, L);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        o[k].x = fmaf(g, v[j][k].x, o[k].x);
        o[k].y = fmaf(g, v[j][k].y, o[k].y);
        o[k].z = fmaf(g, v[j][k].z, o[k].z);
        o[k].w = fmaf(g, v[j][k].w, o[k].w);
      }
    }
  }
  if (live) {
    const float inv = L > 0.0f ? 1.0f / L : L == 0.0f ? 0.0f : L;
    const long long r = (long long)t * a.Hq + head;
#pragma unroll
    for (int k = 0; k < N; ++k)
      ((uint2*)a.out)[r * (D / 4) + c + k] =
          make_uint2(la_pack<F16>(o[k].x * inv, o[k].y * inv), la_pack<F16>(o[k].z * inv, o[k].w * inv));
    if (a.lse && c == 0) a.lse[r] = (M + log2f(L)) * 0.69314718055994531f;
  }
}

constexpr int LJ_WARPS = 8;

template <int D, bool F16>
__global__ void __launch_bounds__(LJ_WARPS * 32) lines_join_kernel(LaArgs a) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int groups = (int)(la_apart_rows(a.T, a.G) / 32), tasks = groups * a.Hkv * (D / 4);
  // task x, prefix and own units apart: 32 rows of a KV head x 4 columns
  auto row_of = [&](int x, int& h, int& packed) {
    const int y = x / (D / 4);
    h = y / groups;
    packed = (y - h * groups) * 32 + lane;
    return packed / a.G;
  };
  int x = blockIdx.x * LJ_WARPS + warp, h, packed;
  grid_dependency_wait();
  allow_dependents();
  // the first task's own unit on its way with the header
  int t = row_of(min(x, tasks - 1), h, packed), own_unit = t < a.T ? __ldg(a.work + LW_HEADER + t) : -1;
  int probe;
  const LaPlan plan(a, probe);
  if (!plan.fits) return;
  if (plan.together) {
    // the unit that is first cut at a run's start, 32 rows x 16 columns a warp at a time (two or three parts, as a rule),
    // by as many blocks as there are
    const int split = max(1, (int)gridDim.x / max(1, plan.runs));
    for (int y = blockIdx.x; y < plan.runs * split; y += gridDim.x) {
      const int run = y / split;
      const int4 joint = a.joints[run];
      const int count = (joint.y + 31) / 32 * (D / 16);
      for (int z = (y - run * split) * LJ_WARPS + warp; z < count; z += split * LJ_WARPS) {
        const int row = z / (D / 16) * 32 + lane, tok = row / a.G;
        la_join_row<D, F16, 4, 4>(a, z % (D / 16) * 4, row < joint.y,
                                  LaParts{la_part_open(a, run - 1) + row, row, run - 1, joint.w}, LaParts{0, 0, 0, -1},
                                  joint.x + tok, joint.z * a.G + row - tok * a.G);
      }
    }
    return;
  }
  for (; x < tasks; x += gridDim.x * LJ_WARPS, t = row_of(min(x, tasks - 1), h, packed),
                    own_unit = t < a.T ? __ldg(a.work + LW_HEADER + t) : -1) {
    const bool live = t < plan.tokens;
    LaParts p[2] = {};
    if (live) {
      const int units[2] = {t / la_tile_tokens(a.G), own_unit};  // its prefix unit, its own
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const LaUnit u = plan.unit(units[i]);
        const int from = h * plan.cost + u.at;
        p[i] = LaParts{la_part_apart(a, i == 1, h) + packed, packed - u.token0 * a.G, from / plan.per,
                       (from + u.tiles - 1) / plan.per};
      }
    }
    la_join_row<D, F16, 1, 8>(a, x % (D / 4), live, p[0], p[1], t, h * a.G + packed - t * a.G);
  }
}

}  // namespace d3
