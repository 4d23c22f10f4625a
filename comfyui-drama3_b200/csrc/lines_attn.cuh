// Attention of lines decoded together over a paged key/value cache: every line's tokens see all keys of a prefix that
// the lines share and the line's own keys up to their own.
//   out[t, h] = sum_j p_j V_j / sum_j p_j,   p_j = exp(scale (q_t,h . K_j - max)),   j over prefix, then own keys
// as one pass over the keys with a running maximum and sum per row, all in 32 bits; the products are 16-bit operands
// with 32-bit accumulators on the tensor cores, and p is rounded to the values' type for the second product (its sum
// is taken before the rounding).
//
// A unit (lines_plan.cuh) is a tile of up to 128 rows (a token x one query head of a KV head) and its key tiles of 64.
// The key tiles of all units of all KV heads, laid end to end, are cut into equal runs, one per CTA: every CTA streams
// the same number of keys whatever the lengths are. A run crosses units; a unit cut by a run's end leaves parts, which
// lines_combine_kernel joins. With few lines the rows of all of them share the prefix's tiles, so a prefix key is
// read from memory once for all lines.
//
// Per CTA (192 threads; two CTAs per SM for heads of 64 and 128, so that one's products run under the other's
// exponentials; one for 256):
//   warp 0     loads: lane l issues one TMA box (a page's keys x 64 columns, 128-byte swizzle) of the stage's K or V
//              tile into a ring; a page outside the cache reads as zeros (the tensor map's fill)
//   warp 1     issues the MMAs (one elected thread) and owns the tensor memory: S = Q K^T (128 x 64, two buffers),
//              O += P V (128 x D, A = P from tensor memory, B = V as it lies in the cache: keys are its rows, so
//              it is the MN-major operand). S of the next tile is issued before O of this one.
//   warps 2-5  a thread owns a row: S from tensor memory, mask, maximum, exponentials, P back over S, the row's
//              sum. O is rescaled only when the maximum has grown by more than 2^8 since the last time (p <= 256 in
//              between, the same value after the division). They also stage Q and write the results.
// Keys of a tile past the end of the prefix or of the line are masked in S, and their V rows are cleared in shared
// memory before the product, since the cache may hold anything there (0 x NaN is NaN).
// Every wait is bounded (2 s) and records FAULT_WAIT_TIMEOUT instead of hanging.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "lines_plan.cuh"
#include "tcgen05.cuh"

namespace d3 {

constexpr int LA_THREADS = 192;
constexpr int LA_ROW_WARP = 2;        // first of the four row warps
constexpr int LA_MIN_TILES = 2;       // shortest run of key tiles worth a CTA
constexpr float LA_RESCALE = 8.0f;    // growth of the maximum, in powers of two, that rescales O

template <int D>
struct LaShape {
  static constexpr int SLICES = D / 64;                 // 128-byte column slices of a row
  static constexpr int Q_BYTES = LA_ROWS * D * 2;
  static constexpr int STAGE = LA_KEYS * D * 2;         // a K or V tile
  static constexpr int PER_SM = D == 256 ? 1 : 2;
  static constexpr int STAGES = D == 256 ? 4 : D == 128 ? 5 : 8;
  static constexpr int TMEM_COLS = D == 256 ? 512 : 256;  // O: D columns, S: 2 x 64
  static constexpr int SMEM = Q_BYTES + STAGES * STAGE + 1024;
};

struct LaArgs {
  const void* q;
  long long q_token, q_head;  // strides in elements
  int T, Hq, Hkv, G;
  int pages, page, page_box;  // page_box: keys of a TMA box, min(page, 64)
  const int* table;
  int W;
  const int* prefix_table;
  int PW;
  const int* line;
  const int* cu;
  const int* work;
  int B;
  float scale_log2;  // scale * log2(e)
  void* out;         // [T, Hq, D]
  float* lse;        // [T, Hq] or null
  float* part_o;     // partial rows [.., D], not divided
  float2* part_ml;   // their (maximum * scale_log2, sum)
  int runs;          // CTAs of the attention kernel
};

// Partial rows: LA_ROWS for the part that a run starts in the middle of a unit, LA_ROWS for the part that it leaves
// unfinished, then (prefix and own units apart) the first part of every row's prefix unit and of its own unit.
D3_DEV long long la_part_rest(int run) { return (long long)run * LA_ROWS; }
D3_DEV long long la_part_open(const LaArgs& a, int run) { return (long long)(a.runs + run) * LA_ROWS; }
D3_DEV long long la_part_apart(const LaArgs& a, bool own, int h, int row) {
  return (long long)2 * a.runs * LA_ROWS + ((long long)(own ? a.Hkv : 0) + h) * a.T * a.G + row;
}
__host__ __device__ inline long long la_part_rows(int runs, int T, int G, int Hkv) {
  return (long long)2 * runs * LA_ROWS + ((long long)T * G <= LA_APART_ROWS ? 2ll * Hkv * T * G : 0);
}

// Key tiles of a run.
D3_DEV long long la_run_tiles(const LaArgs& a) {
  const long long total = (long long)a.work[LW_TILES] * a.Hkv;
  const long long even = (total + a.runs - 1) / a.runs;
  return even > LA_MIN_TILES ? even : LA_MIN_TILES;
}

D3_DEV bool la_plan_fits(const LaArgs& a) {
  return a.work[LW_GROUP] == a.G && a.work[LW_LINES] == a.B && a.work[LW_T] == a.T;
}

D3_DEV LaUnit la_unit(const LaUnit* units, int u) {
  const int4 v = __ldg((const int4*)(units + u));
  return LaUnit{v.x, v.y, v.z, v.w};
}

// The last unit with start <= tile, by the whole warp: 32 probes a round.
D3_DEV int la_find_unit(const LaUnit* units, int count, int tile) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = count;  // the answer is in [lo, lo + n)
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int at = lo + lane * step;
    const bool below = lane * step < n && __ldg(&units[at].start) <= tile;
    const int hit = __popc(__ballot_sync(0xffffffffu, below)) - 1;
    n = min(step, n - hit * step);
    lo += hit * step;
  }
  return lo;
}

// A CTA's run, piece by piece (a piece: consecutive key tiles of one unit). Every warp walks it by itself.
struct LaWalk {
  long long pos, end;
  int h, rem, u, W1, units_n;
  const LaUnit* units;
  LaUnit unit;
  int j0, n;  // the piece: tiles [j0, j0 + n) of the unit

  D3_DEV void start(const LaArgs& a, int run) {
    const long long per = la_run_tiles(a), total = (long long)a.work[LW_TILES] * a.Hkv;
    pos = per * run;
    end = pos + per < total ? pos + per : total;
    W1 = a.work[LW_TILES];
    units_n = a.work[LW_UNITS];
    units = (const LaUnit*)(a.work + la_unit_offset(a.B));
    if (pos < end) {
      h = (int)(pos / W1);
      rem = (int)(pos - (long long)h * W1);
      u = la_find_unit(units, units_n, rem);
    }
  }
  D3_DEV bool next() {
    if (pos >= end) return false;
    unit = la_unit(units, u);
    j0 = rem - unit.start;
    n = (int)min((long long)(unit.tiles - j0), end - pos);
    return true;
  }
  D3_DEV void step() {
    pos += n;
    rem += n;
    if (++u == units_n) {
      u = 0;
      rem = 0;
      ++h;
    }
  }
};

// What a unit's rows and key tiles are.
struct LaSpan {
  int rows;       // rows of the unit
  int lead;       // key tiles of the prefix at its front
  int prefix;     // keys of the prefix
  int own_end;    // own keys that its last row sees (0 for a prefix unit)
  int kept, token0;
  D3_DEV LaSpan(const LaArgs& a, const LaUnit& u) {
    prefix = a.work[LW_PREFIX];
    if (u.line < 0) {
      rows = min(LA_ROWS, a.work[LW_TOKENS] * a.G - u.row0);
      lead = u.tiles;
      own_end = kept = token0 = 0;
    } else {
      token0 = a.cu[u.line];
      const int all = (a.cu[u.line + 1] - token0) * a.G;
      rows = min(LA_ROWS, all - u.row0);
      lead = a.work[LW_TOGETHER] ? a.work[LW_PREFIX_TILES] : 0;
      kept = a.work[LW_HEADER + u.line];
      own_end = kept + (u.row0 + rows - 1) / a.G + 1;
    }
  }
  // first key of tile j (of the prefix when own is false) and how many of its LA_KEYS there are
  D3_DEV int tile(int j, bool& own, int& valid) const {
    own = j >= lead;
    const int key0 = (own ? j - lead : j) * LA_KEYS;
    valid = min(LA_KEYS, (own ? own_end : prefix) - key0);
    return key0;
  }
};

// Shared-memory descriptor of V as the MMA's B: MN-major (columns contiguous), 128-byte swizzle; 8 keys x 64 columns
// atoms of 1024 bytes, SBO between groups of 8 keys, LBO between 64-column slices.
D3_DEV uint64_t la_v_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)((LA_KEYS * 128) >> 4) << 16) |
         ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// D += A B with A in tensor memory (16-bit values, two to a column).
D3_DEV void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
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
D3_DEV bool la_warp_wait(uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity)); }

D3_DEV float la_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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

template <int D, bool F16>
__global__ void __launch_bounds__(LA_THREADS, LaShape<D>::PER_SM)
    lines_attn_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, LaArgs a) {
  using S = LaShape<D>;
  extern __shared__ __align__(1024) uint8_t la_smem[];
  uint8_t* q_s = la_smem;
  uint8_t* ring = la_smem + S::Q_BYTES;
  uint64_t* bars = (uint64_t*)(la_smem + S::Q_BYTES + S::STAGES * S::STAGE);
  uint64_t* kv_full = bars;                    // [STAGES]
  uint64_t* kv_empty = kv_full + S::STAGES;    // [STAGES]
  uint64_t* q_full = kv_empty + S::STAGES;
  uint64_t* s_full = q_full + 1;               // [2]
  uint64_t* p_full = s_full + 2;               // [2]
  uint64_t* o_full = p_full + 2;               // [2], by tile parity: a waiter may be up to two products behind
  uint32_t* tmem_slot = (uint32_t*)(o_full + 2);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, run = blockIdx.x;
  const bool aligned = (smem_u32(la_smem) & 1023u) == 0;  // the swizzle's atoms
  if (tid == 0) {
    for (int i = 0; i < S::STAGES; ++i) {
      mbar_init(kv_full + i, 1);
      mbar_init(kv_empty + i, 1);
    }
    mbar_init(q_full, 4);
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + i, 1);
      mbar_init(p_full + i, 4);
      mbar_init(o_full + i, 1);
    }
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
  const uint32_t tmem_o = tmem, tmem_s = tmem + D;  // S / P buffer b: columns D + 64 b
  const bool fits = la_plan_fits(a) && aligned;
  if (!fits && tid == 0) record_fault(FAULT_PLAN);
  LaWalk w;
  w.pos = w.end = 0;
  if (fits && a.work[LW_TILES] > 0) w.start(a, run);

  if (warp == 0) {
    // ---- loads: K0, K1, V0, K2, V1, ... of each piece
    uint32_t seq = 0;
    bool ok = true;
    int win_first = 0, win_page = -1;  // a window of 32 page ids, one per lane
    const int* win_table = nullptr;
    const int slice = lane % S::SLICES, box = lane / S::SLICES;
    auto fetch = [&](const CUtensorMap* map, int h, int boxes, int page_id, int in_page) {
      const uint32_t st = seq % S::STAGES, ph = (seq / S::STAGES) & 1;
      ++seq;
      ok = la_warp_wait(kv_empty + st, ph ^ 1);
      if (!ok) return;
      if (lane == 0) mbar_arrive_expect_tx(kv_full + st, boxes * a.page_box * S::SLICES * 128);
      __syncwarp();
      if (box < boxes)
        tma_load_4d(smem_u32(ring) + st * S::STAGE + slice * (LA_KEYS * 128) + box * a.page_box * 128, map, slice * 64,
                    in_page, h, page_id, kv_full + st);
    };
    for (; ok && w.next(); w.step()) {
      const LaSpan sp(a, w.unit);
      int before_boxes = 0, before_page = 0, before_in = 0;
      for (int i = 0; ok && i < w.n; ++i) {
        bool own;
        int valid;
        const int key0 = sp.tile(w.j0 + i, own, valid);
        const int boxes = (valid + a.page_box - 1) / a.page_box;
        const int first = key0 / a.page, in_page = key0 - first * a.page;
        const int* table = own ? a.table + (size_t)w.unit.line * a.W : a.prefix_table;
        const int width = own ? a.W : a.PW;
        if (table != win_table || first < win_first || first + boxes > win_first + 32) {
          win_table = table;
          win_first = first;
          win_page = first + lane < width ? table[first + lane] : -1;
        }
        int page_id = __shfl_sync(0xffffffffu, win_page, (first - win_first + box) & 31);
        if (box < boxes && (page_id < 0 || page_id >= a.pages)) {
          record_fault(FAULT_PAGES);
          page_id = -1;  // outside the map: zeros
        }
        fetch(&kmap, w.h, boxes, page_id, in_page);
        if (ok && i > 0) fetch(&vmap, w.h, before_boxes, before_page, before_in);
        before_boxes = boxes;
        before_page = page_id;
        before_in = in_page;
      }
      if (ok) fetch(&vmap, w.h, before_boxes, before_page, before_in);
    }
    // nothing may land after the CTA is gone: a stage's last load has arrived once its phase is complete
    for (uint32_t i = seq < (uint32_t)S::STAGES ? 0 : seq - S::STAGES; i < seq; ++i)
      mbar_wait(kv_full + i % S::STAGES, (i / S::STAGES) & 1);
  } else if (warp == 1) {
    // ---- MMAs
    if (lane == 0) {
      const uint32_t type = F16 ? 0u : (1u << 7) | (1u << 10);
      const uint32_t idesc_s = (1u << 4) | type | ((LA_KEYS >> 3) << 17) | ((LA_ROWS >> 4) << 24);
      const uint32_t idesc_o = (1u << 4) | type | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((LA_ROWS >> 4) << 24);
      uint32_t seq = 0, tiles = 0, pieces = 0;
      bool ok = true;
      const uint32_t q_base = smem_u32(q_s), ring_base = smem_u32(ring);
      auto scores = [&](uint32_t tile) {
        const uint32_t st = seq % S::STAGES, ph = (seq / S::STAGES) & 1;
        ++seq;
        if (!(ok = mbar_wait(kv_full + st, ph))) return;
        tc_fence_after();
        const uint32_t kb = ring_base + st * S::STAGE;
#pragma unroll
        for (int c = 0; c < D / 16; ++c)
          umma_f16(tmem_s + 64 * (tile & 1), umma_desc_sw128(q_base + (c >> 2) * (LA_ROWS * 128) + (c & 3) * 32),
                   umma_desc_sw128(kb + (c >> 2) * (LA_KEYS * 128) + (c & 3) * 32), idesc_s, c > 0);
        umma_commit(kv_empty + st);
        umma_commit(s_full + (tile & 1));
      };
      for (; ok && w.next(); w.step()) {
        if (!(ok = mbar_wait(q_full, pieces & 1))) break;
        ++pieces;
        tc_fence_after();
        scores(tiles);
        for (int i = 0; ok && i < w.n; ++i, ++tiles) {
          if (i + 1 < w.n) {
            // S of tile + 1 goes where P of tile - 1 is, once that product has read it
            if (i > 0 && !(ok = mbar_wait(o_full + ((tiles - 1) & 1), ((tiles - 1) >> 1) & 1))) break;
            scores(tiles + 1);
          }
          if (!ok || !(ok = mbar_wait(p_full + (tiles & 1), (tiles >> 1) & 1))) break;
          const uint32_t st = seq % S::STAGES, ph = (seq / S::STAGES) & 1;
          ++seq;
          if (!(ok = mbar_wait(kv_full + st, ph))) break;
          tc_fence_after();
          const uint32_t vb = ring_base + st * S::STAGE;
#pragma unroll
          for (int c = 0; c < LA_KEYS / 16; ++c)
            umma_f16_ts(tmem_o, tmem_s + 64 * (tiles & 1) + 8 * c, la_v_desc(vb + c * 2048), idesc_o, i > 0 || c > 0);
          umma_commit(kv_empty + st);
          umma_commit(o_full + (tiles & 1));
        }
      }
    }
    __syncwarp();
  } else {
    // ---- rows
    const int quarter = warp & 3;
    const uint32_t lanes = (uint32_t)(32 * quarter) << 16;
    const int row = 32 * quarter + lane;
    uint32_t seq = 0, tiles = 0;
    bool ok = true;
    for (; ok && w.next(); w.step()) {
      const LaSpan sp(a, w.unit);
      const int R = w.unit.row0 + row;
      const bool live = row < sp.rows, any = 32 * quarter < sp.rows;
      const int tok = R / a.G;
      const int t = w.unit.line < 0 ? tok : sp.token0 + tok, head = w.h * a.G + R - tok * a.G;
      const int own_keys = sp.kept + tok + 1;  // own keys that this row sees
      // stage Q: this warp's 32 rows, 16 bytes a lane; rows past the unit's are zeros
      if (any) {
        constexpr int CH = D / 8;  // 16-byte chunks of a row
        const long long off = live ? (long long)t * a.q_token + (long long)head * a.q_head : -1;
#pragma unroll 8
        for (int i = 0; i < CH; ++i) {
          const int x = i * 32 + lane, r = x / CH, c = x % CH;
          const long long o = __shfl_sync(0xffffffffu, off, r);
          uint4 v = make_uint4(0, 0, 0, 0);
          if (o >= 0) v = *(const uint4*)((const uint16_t*)a.q + o + 8 * c);
          *(uint4*)(q_s + (c >> 3) * (LA_ROWS * 128) + sw128_offset(32 * quarter + r, c & 7)) = v;
        }
        fence_async_smem();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
      float m = -INFINITY, l = 0.0f;
      for (int i = 0; i < w.n; ++i, ++tiles) {
        const uint32_t buf = tiles & 1;
        if (!(ok = la_warp_wait(s_full + buf, (tiles >> 1) & 1))) break;
        tc_fence_after();
        bool own;
        int valid;
        const int key0 = sp.tile(w.j0 + i, own, valid);
        if (any) {
          uint32_t s[64];
          tmem_ld64(tmem_s + lanes + 64 * buf, s);
          const int lim = own ? min(valid, own_keys - key0) : valid;
          if (lim < LA_KEYS) {
#pragma unroll
            for (int x = 0; x < 64; ++x)
              if (x >= lim) s[x] = 0xff800000u;  // -inf
          }
          float mx = __uint_as_float(s[0]);
#pragma unroll
          for (int x = 1; x < 64; ++x) mx = fmaxf(mx, __uint_as_float(s[x]));
          mx *= a.scale_log2;
          if (i == 0) {
            m = mx;
          } else if (__any_sync(0xffffffffu, mx > m + LA_RESCALE || (m == -INFINITY && mx > m))) {
            const float top = fmaxf(m, mx);
            const float f = m == -INFINITY ? 0.0f : la_exp2(m - top);
            m = top;
            l *= f;
            if (!(ok = la_warp_wait(o_full + ((tiles - 1) & 1), ((tiles - 1) >> 1) & 1))) break;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < D; c += 32) {
              uint32_t o[32];
              tmem_ld32(tmem_o + lanes + c, o);
#pragma unroll
              for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
              tmem_st32(tmem_o + lanes + c, o);
            }
          }
          const float base = m == -INFINITY ? 0.0f : m;
          uint32_t p[32];
          float sum = 0.0f;
#pragma unroll
          for (int x = 0; x < 64; x += 2) {
            const float p0 = la_exp2(fmaf(__uint_as_float(s[x]), a.scale_log2, -base));
            const float p1 = la_exp2(fmaf(__uint_as_float(s[x + 1]), a.scale_log2, -base));
            sum += p0 + p1;
            p[x / 2] = la_pack<F16>(p0, p1);
          }
          l += sum;
          tmem_st32(tmem_s + lanes + 64 * buf, p);
          tmem_wait_st();
        }
        if (valid < LA_KEYS) {
          // V's rows past the end: V of tile i is the (i + 1 < n ? 2 i + 2 : 2 n - 1)-th load of the piece
          const uint32_t vs = seq + (i + 1 < w.n ? 2 * i + 2 : 2 * w.n - 1);
          if (!(ok = la_warp_wait(kv_full + vs % S::STAGES, (vs / S::STAGES) & 1))) break;
          uint8_t* v = ring + (vs % S::STAGES) * S::STAGE;
          for (int x = tid - 32 * LA_ROW_WARP; x < (LA_KEYS - valid) * 8 * S::SLICES; x += 128) {
            const int c = x & 7, r = (x >> 3) % (LA_KEYS - valid), sl = (x >> 3) / (LA_KEYS - valid);
            *(uint4*)(v + sl * (LA_KEYS * 128) + (valid + r) * 128 + c * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_async_smem();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + buf);
      }
      seq += 2 * w.n;
      if (!ok) break;
      if (!(ok = la_warp_wait(o_full + ((tiles - 1) & 1), ((tiles - 1) >> 1) & 1))) break;
      tc_fence_after();
      // results: a whole unit's rows are done; a part's go to the workspace
      const bool first = w.j0 == 0, last = w.j0 + w.n == w.unit.tiles;
      const bool apart = !a.work[LW_TOGETHER];
      const bool whole = first && last && !apart;
      long long part = 0;
      if (!first)
        part = la_part_rest(run) + row;
      else if (apart)
        part = la_part_apart(a, w.unit.line >= 0, w.h, w.unit.line < 0 ? R : sp.token0 * a.G + R);
      else
        part = la_part_open(a, run) + row;
      if (any) {
        const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
#pragma unroll
        for (int c = 0; c < D; c += 32) {
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
            uint4* dst = (uint4*)(a.part_o + part * D + c);
#pragma unroll
            for (int x = 0; x < 8; ++x) dst[x] = make_uint4(o[4 * x], o[4 * x + 1], o[4 * x + 2], o[4 * x + 3]);
          }
        }
        if (live) {
          if (!whole)
            a.part_ml[part] = make_float2(m, l);
          else if (a.lse)
            a.lse[(long long)t * a.Hq + head] = (m + log2f(l)) * 0.69314718055994531f;
        }
      }
      tc_fence_before();
    }
    // tokens of no line: nothing to see
    if (fits) {
      const int tokens = a.work[LW_TOKENS];
      const long long total = (long long)(a.T - tokens) * a.Hq;
      for (long long x = (long long)run * 4 + warp - LA_ROW_WARP; x < total; x += (long long)a.runs * 4) {
        const long long r = (long long)tokens * a.Hq + x;
        for (int c = lane; c < D / 8; c += 32)
          *(uint4*)((uint16_t*)a.out + r * D + 8 * c) = make_uint4(0, 0, 0, 0);
        if (a.lse && lane == 0) a.lse[r] = -INFINITY;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, S::TMEM_COLS);
  }
}

// Joins the parts of a row: with M the largest of their maxima, out = sum 2^(m_i - M) O_i / sum 2^(m_i - M) l_i. A
// block of four warps per row, part i to warp i mod 4, then the four through shared memory.
constexpr int LC_WARPS = 4;

template <int D, bool F16>
__global__ void __launch_bounds__(LC_WARPS * 32) lines_combine_kernel(LaArgs a) {
  constexpr int PER = D / 32;  // columns a lane holds: lane, lane + 32, ...
  __shared__ float s_o[LC_WARPS][D];
  __shared__ float2 s_ml[LC_WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_dependency_wait();
  allow_dependents();
  if (!la_plan_fits(a) || a.work[LW_TILES] <= 0) return;
  const LaUnit* units = (const LaUnit*)(a.work + la_unit_offset(a.B));
  const bool apart = !a.work[LW_TOGETHER];
  const long long per = la_run_tiles(a);
  const int W1 = a.work[LW_TILES], tokens = a.work[LW_TOKENS];

  float m, l, o[PER];
  auto add = [&](long long part) {
    const float2 ml = a.part_ml[part];
    float v[PER];
#pragma unroll
    for (int c = 0; c < PER; ++c) v[c] = a.part_o[part * D + 32 * c + lane];
    if (ml.x == -INFINITY) return;
    const float top = fmaxf(m, ml.x);
    const float f = m == -INFINITY ? 0.0f : la_exp2(m - top), g = la_exp2(ml.x - top);
    m = top;
    l = l * f + ml.y * g;
#pragma unroll
    for (int c = 0; c < PER; ++c) o[c] = o[c] * f + v[c] * g;
  };
  // parts of unit u's row: the first one at `first_part`, the others by the runs that start inside the unit
  int turn = 0;
  auto add_unit = [&](const LaUnit& u, int h, long long first_part, int row) {
    const long long s0 = (long long)h * W1 + u.start, s1 = s0 + u.tiles - 1;
    const int r0 = (int)(s0 / per), r1 = (int)(s1 / per);
    for (int r = r0; r <= r1; ++r, ++turn)
      if (turn % LC_WARPS == warp) add(r == r0 ? first_part : la_part_rest(r) + row);
  };
  auto begin = [&]() {
    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int c = 0; c < PER; ++c) o[c] = 0.0f;
    turn = 0;
  };
  auto finish = [&](int t, int head) {
    if (lane == 0) s_ml[warp] = make_float2(m, l);
#pragma unroll
    for (int c = 0; c < PER; ++c) s_o[warp][32 * c + lane] = o[c];
    __syncthreads();
    float M = -INFINITY, L = 0.0f;
#pragma unroll
    for (int i = 0; i < LC_WARPS; ++i) M = fmaxf(M, s_ml[i].x);
    float f[LC_WARPS];
#pragma unroll
    for (int i = 0; i < LC_WARPS; ++i) {
      f[i] = s_ml[i].x == -INFINITY ? 0.0f : la_exp2(s_ml[i].x - M);
      L += s_ml[i].y * f[i];
    }
    const float inv = L > 0.0f ? 1.0f / L : L == 0.0f ? 0.0f : L;
    const long long r = (long long)t * a.Hq + head;
    for (int c = threadIdx.x; c < D / 2; c += LC_WARPS * 32) {
      float x = 0.0f, y = 0.0f;
#pragma unroll
      for (int i = 0; i < LC_WARPS; ++i) {
        x += s_o[i][2 * c] * f[i];
        y += s_o[i][2 * c + 1] * f[i];
      }
      ((uint32_t*)a.out)[(r * D) / 2 + c] = la_pack<F16>(x * inv, y * inv);
    }
    if (a.lse && threadIdx.x == 0) a.lse[r] = (M + log2f(L)) * 0.69314718055994531f;
    __syncthreads();
  };

  if (apart) {
    const long long rows = (long long)tokens * a.Hq;
    for (long long x = blockIdx.x; x < rows; x += gridDim.x) {
      const int t = (int)(x / a.Hq), head = (int)(x - (long long)t * a.Hq), h = head / a.G, g = head - h * a.G;
      const int packed = t * a.G + g;
      begin();
      add_unit(la_unit(units, packed / LA_ROWS), h, la_part_apart(a, false, h, packed), packed % LA_ROWS);
      const int b = a.line[t];
      const int R = (t - a.cu[b]) * a.G + g;
      add_unit(la_unit(units, a.work[LW_HEADER + a.B + b] + R / LA_ROWS), h, la_part_apart(a, true, h, packed),
               R % LA_ROWS);
      finish(t, head);
    }
    return;
  }
  // together: only the units that a run's end cuts; the first such run start inside a unit takes it
  const long long total = (long long)W1 * a.Hkv;
  for (long long x = blockIdx.x; x < (long long)(a.runs - 1) * LA_ROWS; x += gridDim.x) {
    const int run = 1 + (int)(x / LA_ROWS), row = (int)(x % LA_ROWS);
    const long long pos = per * run;
    if (pos >= total) continue;
    const int h = (int)(pos / W1), rem = (int)(pos - (long long)h * W1);
    const LaUnit u = la_unit(units, la_find_unit(units, a.work[LW_UNITS], rem));
    const long long s0 = (long long)h * W1 + u.start;
    if (s0 == pos || s0 / per != run - 1) continue;
    const LaSpan sp(a, u);
    if (row >= sp.rows) continue;
    const int R = u.row0 + row, tok = R / a.G;
    begin();
    add_unit(u, h, la_part_open(a, run - 1) + row, row);
    finish(sp.token0 + tok, h * a.G + R - tok * a.G);
  }
}

}  // namespace d3
