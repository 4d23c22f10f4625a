// Linear attention (lines_delta.cuh has the formulas) over many tokens of a line: in chunks of 64 tokens, with the products on
// the tensor cores. With G_i the sum of the log decays from the chunk's first token on, gamma_i = exp(G_i), and the rows of a
// chunk's Q, K, V, the corrections U solve a triangular system:
//   U = T R,  R = V - diag(gamma) K S^T,  T = (I + A)^-1 diag(beta),  A_ij = beta_i exp(G_i - G_j) k_i . k_j  (j < i)
//   O = scale (diag(gamma) Q S^T + P U),  P_ij = exp(G_i - G_j) q_i . k_j  (j <= i)
//   S <- gamma_last S + U^T D K,          D = diag(exp(G_last - G_j))
// What depends on the tokens alone is formed for all chunks at once (the preparation): not T itself, but P T and K~ = T^T D K, with
// which U is never needed:
//   O = scale (diag(gamma) Q S^T + P T R),  S <- gamma_last S + R^T K~
// So the chain from chunk to chunk (the scan) has two products, S -> R -> S. Without the delta rule R = V, T = I.
// Exponents are differences that are never above 0, of sums in 64 bits.
//
// Chunks are cut from the packed tokens, whatever lines they belong to: entries of two lines are zeros, sums and exponents
// start again with each line. A line's scan masks the tokens of others.
//
// Values. k and q become fp16 rows times powers of two, exactly (values below 2^-14 of the row's largest lose what is below
// 2^-25 of it), and their norms are numbers that results are multiplied by. What is not exact in 16 bits, S, R, T, P T and K~, is
// the sum of two fp16 or tf32 terms, 22 bits, rows of fp16 scaled by a power of two of their own; products are summed in 32 bits, and
// of the four of two such factors the smallest, low times low, is left out (2^-22). S and T are formed in 32 bits. Where the chunk
// overwrites the state an output is the difference of two terms as large as the state, so that all of its factors have two terms too; the
// second one of P T has eight bits (2^-15 of it): an output's own rounding is 2^-11 of it at least.
// Where a row's values lie far apart fp16 ends: S and R towards the state keep 2^-38 of the row's largest, R towards the outputs, whose
// second terms are held 2^11 times, 2^-49, P T 2^-41.
// Corrections with beta |k|^2 above 2 overshoot, and T grows with them; where that leaves 32 bits, the line's other tokens of the chunk may
// be lost with it.
//
// A value that is not finite reaches its line's state and tokens from its own token on, one in v those of its column, one in q its own
// token only.
#pragma once

#include "lines_delta.cuh"
#include "tcgen05.cuh"

namespace d3 {

constexpr int LD_C = 64;  // tokens of a chunk

// What the preparation leaves of a chunk for a key head: fp16 rows [64][Dk], 16-byte pieces in the order of ld_at.
template <int DK> struct alignas(128) LdRows {
  uint16_t k[LD_C * DK];
};
// ... and for a value head: rows likewise, and factors of the tokens' columns.
template <int DK> struct alignas(128) LdHead {
  uint16_t kt_hi[LD_C * DK], kt_lo[LD_C * DK];  // K~ [64][Dk], row j times 1 / kt_scale[j]
  uint16_t q[LD_C * DK];                        // Q [64][Dk], row i times 1 / q_scale[i] (gamma_i among it)
  uint16_t p[LD_C * LD_C];                      // P T [64][64], row i times 1 / p_scale[i]: blocks of 16 x 16 up to the diagonal, second
                                                // terms where the others would be (ld_rest)
  float kt_scale[LD_C], q_scale[LD_C], p_scale[LD_C];
  float r_in[LD_C];  // gamma_i |k| factor: of K S^T
  float gamma[LD_C];
};

// Element offset of 16-byte piece c of row r in rows of `pieces` of them (a multiple of 8): eight rows' pieces of one column lie
// in different banks.
template <int PIECES> D3_DEV int ld_at(int r, int c) { return (r * PIECES + (c ^ (r & 7))) * 8; }

// Element offset of a lane's eight second terms of block (i, j) of P T, j <= i, each 2^11 times the term and rounded to e5m2, in the order
// of ld_matrix4's registers: in the 16-byte pieces of the blocks above the diagonal.
D3_DEV int ld_rest(int i, int j, int lane) {  // rows 0 to 15 hold those of i 0 to 2, the next ones those of i 3
  const int row = (i == 3 ? 16 : 0) + (lane >> 1), piece = i == 3 ? 4 + j : i * (i + 1) / 2 + 2 + j;
  return ld_at<8>(row, piece) + (lane & 1) * 4;
}

D3_DEV void ld_matrix4(uint32_t (&r)[4], const uint16_t* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(smem_u32(p)));
}
D3_DEV void ld_matrix4_trans(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(smem_u32(p)));
}
D3_DEV void st_matrix4_trans(void* p, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(smem_u32(p)), "r"(a), "r"(b), "r"(c),
               "r"(d)
               : "memory");
}
D3_DEV void ld_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm (
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
D3_DEV uint32_t ld_half2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// x, y as e5m2 bytes.
D3_DEV uint32_t ld_bytes(float x, float y) {
  uint16_t r;
  asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(r) : "f"(y), "f"(x));
  return r;
}
// x, y as two fp16 terms each.
D3_DEV void ld_split(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = ld_half2(x, y);
  lo = ld_half2(x - h_lo(hi), y - h_hi(hi));
}

struct LdChunkArgs {
  LdArgs a;
  int block0, blocks;  // of the pass's blocks of 64 tokens, those of this launch
  void* rows;          // [blocks][Hk] LdRows
  void* heads;         // [blocks][Hv] LdHead
};

// ---- The preparation. A CTA per chunk and value head; the first of a key head's leaves the rows. K K^T and Q K^T are mma.sync
// products. T: the 16 x 16 blocks on the diagonal of I + A are inverted by columns, a thread each, then blocks of 32 and of 64 by
// [T1, 0; X, T2], X = -T2 A21 T1, in tf32 terms. (By columns of all 64 at once the same numbers took 2000 unrolled steps and the time
// went into fetching instructions.) P T in tf32 terms too, whose range of exponents needs no scales; K~ in fp16 terms.
// Bound by instructions, their latency and their fetch, 0.48 of the issue slots with four CTAs an SM: 32 chunks of 32 value heads 57 us
// (B200). Loops that need not be unrolled are not: an earlier form took a fifth longer with them unrolled.
constexpr int LD_PREP_THREADS = 128;
constexpr int LD_PITCH = 68;  // floats of a row of A and T in shared memory
constexpr float LD_MAX = 3.4028234e38f;

template <int DK> struct LdPrepShape {
  static constexpr int K = LD_C * DK * 2;          // the rows of k, K~'s low terms; the rows of q
  static constexpr int A = LD_C * LD_PITCH * 4;  // A and T, A21 T1 above them; T^T D, two terms; K~'s high terms
  static constexpr int SMEM = 2 * K + A;
  static_assert(A >= K && A >= 2 * LD_C * LD_C * 2, "");
};

D3_DEV void ld_mma_tf32(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
// x as two tf32 terms, 22 bits and the whole range of exponents.
D3_DEV void ld_split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(x));
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(x - __uint_as_float(hi)));
}

// acc += X Y by a warp: X [16][8 STEPS] at x, Y [8 STEPS][8 TILES] at y, 32-bit rows of pitch px and py.
template <int STEPS, int TILES>
D3_DEV void ld_product(float (&acc)[TILES][4], const float* x, int px, const float* y, int py, int lane) {
  const int g = lane >> 2, cc = lane & 3;
#pragma unroll 1
  for (int k = 0; k < STEPS; ++k) {
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) ld_split_tf32(x[(g + (e & 1) * 8) * px + k * 8 + cc + (e >> 1) * 4], hi[e], lo[e]);
#pragma unroll
    for (int n = 0; n < TILES; ++n) {
      uint32_t b_hi[2], b_lo[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) ld_split_tf32(y[(k * 8 + cc + e * 4) * py + n * 8 + g], b_hi[e], b_lo[e]);
      ld_mma_tf32(acc[n], lo, b_hi);
      ld_mma_tf32(acc[n], hi, b_lo);
      ld_mma_tf32(acc[n], hi, b_hi);
    }
  }
}

// X = -T2 (A21 T1) for the blocks of N x N at rows r0 + N.., columns r0.. of A, of which a warp has 16 rows from `row` on and 8
// TILES columns from `col` on; all four warps go through it together.
template <int N, int TILES> D3_DEV void ld_join(float* A, float* Y, unsigned long long starts, int r0, int row, int col, int lane) {
  const int g = lane >> 2, cc = lane & 3;
  {
    float acc[TILES][4] = {};
    ld_product<N / 8, TILES>(acc, A + (r0 + N + row) * LD_PITCH + r0, LD_PITCH, A + r0 * LD_PITCH + r0 + col, LD_PITCH, lane);
#pragma unroll
    for (int n = 0; n < TILES; ++n)
#pragma unroll
      for (int r = 0; r < 2; ++r)
        *(float2*)(Y + (row + g + r * 8) * LD_PITCH + col + n * 8 + cc * 2) = make_float2(acc[n][2 * r], acc[n][2 * r + 1]);
  }
  __syncthreads();
  float acc[TILES][4] = {};
  ld_product<N / 8, TILES>(acc, A + (r0 + N + row) * LD_PITCH + r0 + N, LD_PITCH, Y + col, LD_PITCH, lane);
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int i = r0 + N + row + g + r * 8;
    const unsigned long long until = starts & (~0ull >> (63 - i));
#pragma unroll
    for (int n = 0; n < TILES; ++n) {
      const int j = r0 + col + n * 8 + cc * 2;  // entries of two lines (one starts in between) are zeros whatever the sums met
      *(float2*)(A + i * LD_PITCH + j) =
          make_float2(until >> (j + 1) ? 0.0f : -acc[n][2 * r], until >> (j + 2) ? 0.0f : -acc[n][2 * r + 1]);
    }
  }
  __syncthreads();
}

// A shared-memory area into global memory by the copy engine: `bytes` a multiple of 16, both 16-byte aligned. One thread issues
// it after every writer's fence_async_smem and a barrier, and waits for it (ld_bulk_read) before the area is used again.
D3_DEV void ld_bulk_out(void* dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(smem_u32(src)), "r"(bytes) : "memory");
}
D3_DEV void ld_bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// The areas have been read; with ld_bulk_done what was written is there too.
D3_DEV void ld_bulk_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
D3_DEV void ld_bulk_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }

// e^x for x <= 0, off by about (2 + |x|) 2^-22 of itself: an exponent of which the argument is rounded to 32 bits is no nearer.
D3_DEV float ld_exp(float x) {
  float r;
  asm("ex2.approx.f32 %0, %1;" : "=f"(r) : "f"(x * 1.4426950408889634f));
  return r;
}

template <int TYPE, int DK, bool DELTA>
__global__ void __launch_bounds__(LD_PREP_THREADS, 4) lines_delta_prep_kernel(LdChunkArgs c) {
  using TT = QrType<TYPE>;
  using E = typename TT::T;
  using Shape = LdPrepShape<DK>;
  constexpr int PIECES = DK / 8;
  extern __shared__ __align__(128) uint8_t ld_smem[];
  uint16_t* const ks = (uint16_t*)ld_smem;
  uint16_t* const qs = (uint16_t*)(ld_smem + Shape::K);
  float* const A = (float*)(ld_smem + 2 * Shape::K);  // A, then T
  float* const Y = A + LD_C / 2;                      // A21 T1, in the upper right quarter, of which T has nothing
  uint16_t* const td = (uint16_t*)A;                  // T^T D, two terms, when T has been read
  __shared__ __align__(8) uint64_t arrived;
  __shared__ int line_s[LD_C];
  __shared__ uint32_t starts_s[2], odd_s[2];  // a bit a token: a line's first one; something of it is not finite
  __shared__ __align__(16) float d_s[LD_C], r_in_s[LD_C], k_factor[LD_C], q_factor[LD_C], beta_s[LD_C], kt_scale[LD_C], q_scale_s[LD_C];
  __shared__ double sum_s;
  __shared__ float2 G_s[LD_C];  // as the sum of two
  __shared__ int bad_s[LD_C];   // by a line's first token in the chunk: its state will not be finite
  const LdArgs& a = c.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, cc = lane & 3;
  const int block = blockIdx.x, h = blockIdx.y, many = a.Hv / a.Hk, hk = h / many;
  const long long t0 = (long long)(c.block0 + block) * LD_C;
  LdHead<DK>* const out = (LdHead<DK>*)c.heads + (size_t)block * a.Hv + h;
  if (tid == 0) {
    mbar_init(&arrived, 1);
    fence_mbar_init();
  }
  grid_dependency_wait();
  allow_dependents();
  __syncthreads();
  // the rows of k and q come together, a copy each; where the pass has ended, zeros
  {
    const bool is_q = tid >= LD_C;
    const int row = tid & (LD_C - 1), live = (int)min((long long)LD_C, a.T - t0);
    uint16_t* const to = (is_q ? qs : ks) + row * DK;
    if (tid == 0) mbar_arrive_expect_tx(&arrived, 2 * live * DK * 2);
    if (row < live) {
      const QrTensor& x = is_q ? a.q : a.k;
      bulk_g2s(to, (const E*)x.p + (t0 + row) * x.token + hk * x.head, DK * 2, &arrived, policy_evict_last());
    } else {
      for (int i = 0; i < PIECES; ++i) ((uint4*)to)[i] = make_uint4(0, 0, 0, 0);
    }
  }
  float decay = 0.0f, beta = 0.0f;
  int my_line = -1;
  if (tid < LD_C) {
    const int l = t0 + tid < a.T ? a.line[t0 + tid] : -1;
    my_line = l >= 0 && l < a.B ? l : -1;
    line_s[tid] = my_line;
    bad_s[tid] = 0;
    if (my_line >= 0) {
      decay = ld_log_decay<TYPE>(a, t0 + tid, h);
      if (DELTA) beta = ld_beta<TYPE>(a, t0 + tid, h);
    }
  }
  __syncthreads();  // the zeros
  if (!__syncthreads_and(mbar_wait(&arrived, 0))) {  // copies in flight land before the block ends
    mbar_wait(&arrived, 0);
    return;
  }
  // rows to fp16, each by the power of two that brings its largest value into [1, 2): four lanes a row, in place
#pragma unroll 1
  for (int i0 = 0; i0 < 4; ++i0) {
    const bool is_q = i0 >= 2;
    const int row = warp * 16 + (i0 & 1) * 8 + g;
    uint16_t* const at = (is_q ? qs : ks) + row * DK;
    constexpr int MINE = PIECES / 4;
    uint4 raw[MINE];
    float most = 0.0f, sum = 0.0f, up, down;
#pragma unroll
    for (int i = 0; i < MINE; ++i) raw[i] = *(const uint4*)(at + ((cc + 4 * i + 4 * (row & 1)) & (PIECES - 1)) * 8);
    float v[MINE][8];
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      qr_unpack<TYPE, 8>(&raw[i].x, v[i]);
#pragma unroll
      for (int e = 0; e < 8; e += 2) most = fmaxf(most, fmaxf(fabsf(v[i][e]), fabsf(v[i][e + 1])));
    }
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
    ld_scale(most, up, down);
    up *= 0x1p-13f, down *= 0x1p13f;
#pragma unroll
    for (int i = 0; i < MINE; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[i][e] *= up;
        sum = fmaf(v[i][e], v[i][e], sum);
      }
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    float f = ld_unit(sum, a.eps, up, down);
    if (most == 0.0f) f = 0.0f;  // a row of zeros: its factor must not set the scale of what it is summed with
    const bool finite = sum <= LD_MAX;
    if (!finite) f = __uint_as_float(0x7fc00000u);
    __syncwarp();  // the row has been read
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      uint4 w = make_uint4(ld_half2(v[i][0], v[i][1]), ld_half2(v[i][2], v[i][3]), ld_half2(v[i][4], v[i][5]), ld_half2(v[i][6], v[i][7]));
      if (!finite) w = make_uint4(0, 0, 0, 0);
      *(uint4*)((is_q ? qs : ks) + ld_at<PIECES>(row, (cc + 4 * i + 4 * (row & 1)) & (PIECES - 1))) = w;
    }
    if (cc == 0) (is_q ? q_factor : k_factor)[row] = is_q ? f * a.scale : f;
  }
  fence_async_smem();
  __syncthreads();
  if (h == hk * many && tid == 0) {  // the rows, as every value head's scan reads them
    LdRows<DK>* rows = (LdRows<DK>*)c.rows + (size_t)block * a.Hk + hk;
    ld_bulk_out(rows->k, ks, sizeof(rows->k));
    ld_bulk_commit();
  }
  if (warp < 2) {
    const uint32_t starts = __ballot_sync(0xffffffffu, tid == 0 || line_s[tid - 1] != my_line);
    const bool finite = k_factor[tid] == k_factor[tid] && decay == decay && fabsf(beta) <= LD_MAX;
    const uint32_t odd = __ballot_sync(0xffffffffu, my_line >= 0 && !finite);
    if (lane == 0) starts_s[warp] = starts, odd_s[warp] = odd;
  }
  __syncthreads();
  const unsigned long long starts = starts_s[0] | (unsigned long long)starts_s[1] << 32;
  auto first_of = [&](int i) { return 63 - __clzll(starts & (~0ull >> (63 - i))); };
  // From a line's first token on whose key, decay or strength is not finite, its tokens count as not there, and get NaN in the end: what
  // comes before stays clear of it.
  int first = 0, last = 0;
  bool lost = false;
  if (tid < LD_C) {
    first = first_of(tid);
    const unsigned long long later = tid == 63 ? 0 : starts >> (tid + 1), odd = odd_s[0] | (unsigned long long)odd_s[1] << 32;
    last = later ? tid + __ffsll((long long)later) - 1 : 63;
    lost = (odd & (~0ull >> (63 - tid))) >> first;
    if (lost) decay = beta = k_factor[tid] = 0.0f, bad_s[first] = 1;
  }
  // sums of the log decays that start again with each line
  double G = decay < -104.0f ? -104.0f : decay;  // exp of it is 0 already; keeps infinities out of the sums
  if (warp < 2) {
    const int from = max(first - warp * 32, 0);  // in this warp
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double before = __shfl_up_sync(0xffffffffu, G, o);
      if (lane - o >= from) G += before;
    }
    if (tid == 31) sum_s = G;
  }
  __syncthreads();
  if (tid < LD_C) {
    if (tid >= 32 && first < 32) G += sum_s;
    const float G_hi = (float)G;
    G_s[tid] = make_float2(G_hi, (float)(G - G_hi));
    beta_s[tid] = beta;
  }
  // K K^T and Q K^T: rows 16 warp + g, + 8, columns 8 n + 2 cc, + 1 up to the diagonal
  float p[8][4] = {}, kk[8][4] = {};
#pragma unroll 2
  for (int kt = 0; kt < DK / 16; ++kt) {
    uint32_t ak[4], aq[4];
    const int ar = warp * 16 + (lane & 15), ap = kt * 2 + (lane >> 4);
    if (DELTA) ld_matrix4(ak, ks + ld_at<PIECES>(ar, ap));
    ld_matrix4(aq, qs + ld_at<PIECES>(ar, ap));
#pragma unroll
    for (int n = 0; n < 8; n += 2)
      if (n <= 2 * warp) {
        uint32_t b[4];
        ld_matrix4(b, ks + ld_at<PIECES>(n * 8 + (lane & 7) + (lane >> 4) * 8, kt * 2 + ((lane >> 3) & 1)));
        if (DELTA) ld_mma(kk[n], ak, b[0], b[1]), ld_mma(kk[n + 1], ak, b[2], b[3]);
        ld_mma(p[n], aq, b[0], b[1]), ld_mma(p[n + 1], aq, b[2], b[3]);
      }
  }
  __syncthreads();
  if (tid < LD_C) {
    const float2 Gl = G_s[last], Gi = G_s[tid];
    d_s[tid] = my_line >= 0 ? ld_exp((Gl.x - Gi.x) + (Gl.y - Gi.y)) * k_factor[tid] : 0.0f;
    r_in_s[tid] = my_line >= 0 ? ld_exp(Gi.x + Gi.y) * k_factor[tid] : 0.0f;
  }
  int from[2];  // the first token of the row's line
  {
    float qf[2], kf[2];
    float2 Gi[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int i = warp * 16 + g + r * 8;
      qf[r] = q_factor[i], kf[r] = k_factor[i] * beta_s[i], Gi[r] = G_s[i];
      from[r] = line_s[i] >= 0 ? first_of(i) : LD_C;  // the row's first entry
    }
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int j = n * 8 + cc * 2 + x;
        float av[2] = {0.0f, 0.0f}, pv[2] = {0.0f, 0.0f};
        if (n <= 2 * warp + 1) {
          const float kfj = k_factor[j];
          const float2 Gj = G_s[j];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int i = warp * 16 + g + r * 8, e = r * 2 + x;
            const float ratio = ld_exp((Gi[r].x - Gj.x) + (Gi[r].y - Gj.y)) * kfj;
            const bool in = j >= from[r] && j <= i;
            pv[r] = in ? ratio * qf[r] * p[n][e] : 0.0f;
            if (DELTA) av[r] = in && j < i ? ratio * kf[r] * kk[n][e] : 0.0f;
          }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          p[n][r * 2 + x] = pv[r];
          if (DELTA) A[(warp * 16 + g + r * 8) * LD_PITCH + j] = av[r];
        }
      }
  }
  __syncthreads();
  float most[2] = {0.0f, 0.0f};
  bool good[2] = {true, true};
  if constexpr (DELTA) {
    if (tid < LD_C) {  // the blocks on the diagonal
      const int d = tid & ~15, j = tid & 15;
      float x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        x[i] = i == j ? 1.0f : 0.0f;
#pragma unroll
        for (int m = 0; m < 16; m += 4)
          if (m < i) {
            const float4 v = *(const float4*)(A + (d + i) * LD_PITCH + d + m);
            x[i] = fmaf(-v.x, x[m], x[i]);
            if (m + 1 < i) x[i] = fmaf(-v.y, x[m + 1], x[i]);
            if (m + 2 < i) x[i] = fmaf(-v.z, x[m + 2], x[i]);
            if (m + 3 < i) x[i] = fmaf(-v.w, x[m + 3], x[i]);
          }
        if (i < j) x[i] = 0.0f;  // whatever stands in the rows of an earlier line
      }
      __syncwarp();
      const int from = first_of(d + j);
#pragma unroll
      for (int i = 0; i < 16; ++i) A[(d + i) * LD_PITCH + d + j] = first_of(d + i) == from ? x[i] : 0.0f;
    }
    __syncthreads();
    ld_join<16, 1>(A, Y + (warp >> 1) * 16 * LD_PITCH, starts, (warp >> 1) * 32, 0, (warp & 1) * 8, lane);
    ld_join<32, 2>(A, Y, starts, 0, (warp >> 1) * 16, (warp & 1) * 16, lane);
    // P T: a warp has 16 rows, in steps of 8 columns of P; two neighbouring columns of an accumulator are columns cc and cc + 4 of a
    // tf32 operand, with T's rows taken in that order
    float tp[8][4] = {};
#pragma unroll
    for (int m = 0; m < 8; ++m)
      if (m <= 2 * warp + 1) {
        uint32_t hi[4], lo[4];
        ld_split_tf32(p[m][0], hi[0], lo[0]), ld_split_tf32(p[m][2], hi[1], lo[1]);
        ld_split_tf32(p[m][1], hi[2], lo[2]), ld_split_tf32(p[m][3], hi[3], lo[3]);
#pragma unroll
        for (int n = 0; n <= m; ++n) {
          uint32_t b_hi[2], b_lo[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) ld_split_tf32(A[(m * 8 + cc * 2 + e) * LD_PITCH + n * 8 + g], b_hi[e], b_lo[e]);
          ld_mma_tf32(tp[n], lo, b_hi);
          ld_mma_tf32(tp[n], hi, b_lo);
          ld_mma_tf32(tp[n], hi, b_hi);
        }
      }
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = n * 8 + cc * 2 + (e & 1), i = warp * 16 + g + (e >> 1) * 8;  // zeros for other lines whatever the sums met
        p[n][e] = j >= from[e >> 1] && j <= i ? tp[n][e] * beta_s[j] : 0.0f;
      }
  }
  // the rows of P T (of P) out, both terms
#pragma unroll
  for (int n = 0; n < 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (!(fabsf(p[n][e]) <= LD_MAX)) good[e >> 1] = false, p[n][e] = 0.0f;
      most[e >> 1] = fmaxf(most[e >> 1], fabsf(p[n][e]));
    }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int i = warp * 16 + g + r * 8;
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) most[r] = fmaxf(most[r], __shfl_xor_sync(0xffffffffu, most[r], o));
    const uint32_t row = 0xfu << (lane & ~3);
    const bool all_good = (__ballot_sync(0xffffffffu, good[r]) & row) == row;
    float up, down;
    ld_scale(most[r], up, down);
    if (cc == 0) {
      out->p_scale[i] = all_good ? down : __uint_as_float(0x7fc00000u);
      q_scale_s[i] = ld_exp(G_s[i].x + G_s[i].y) * q_factor[i];
    }
#pragma unroll
    for (int n = 0; n < 8; ++n)
      if (n <= 2 * warp + 1) {
        float& x = p[n][r * 2];
        float& y = p[n][r * 2 + 1];
        x *= up, y *= up;
        const uint32_t hi = ld_half2(x, y);
        *(uint32_t*)(out->p + ld_at<8>(i, n) + cc * 2) = hi;
        x = (x - h_lo(hi)) * 0x1p11f, y = (y - h_hi(hi)) * 0x1p11f;
      }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j <= warp)
      *(uint2*)(out->p + ld_rest(warp, j, lane)) =
          make_uint2(ld_bytes(p[2 * j][0], p[2 * j][1]) | ld_bytes(p[2 * j + 1][0], p[2 * j + 1][1]) << 16,
                     ld_bytes(p[2 * j][2], p[2 * j][3]) | ld_bytes(p[2 * j + 1][2], p[2 * j + 1][3]) << 16);
  if constexpr (DELTA) {
    {  // columns of T become rows of T^T D: two threads each, four rows by turns
      const int j = tid >> 1, half = tid & 1;
      const float b = beta_s[j];
      float d[32], m_d = 0.0f, sum = 0.0f;
#pragma unroll
      for (int e = 0; e < 32; e += 4) {
        const int i = e * 2 + half * 4;
        const float4 d4 = *(const float4*)(d_s + i);
        const float ds[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float v = i + x >= j ? A[(i + x) * LD_PITCH + j] * b : 0.0f;
          d[e + x] = v != 0.0f ? v * ds[x] : 0.0f;  // nothing of another line, where that is not finite
          sum += fabsf(d[e + x]);                   // finite where all are
        }
        m_d = fmaxf(m_d, fmaxf(fmaxf(fabsf(d[e]), fabsf(d[e + 1])), fmaxf(fabsf(d[e + 2]), fabsf(d[e + 3]))));
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      m_d = fmaxf(m_d, __shfl_xor_sync(0xffffffffu, m_d, 1));
      if (!(sum <= LD_MAX)) {
        bad_s[first_of(j)] = 1;
        m_d = 0.0f;
#pragma unroll
        for (int e = 0; e < 32; ++e) d[e] = 0.0f;
      }
      float up_d, down_d;
      ld_scale(m_d, up_d, down_d);
      if (half == 0) kt_scale[j] = m_d > 0.0f ? down_d * 0x1p6f : 0.0f;  // a row of zeros must not set a scale
      __syncthreads();                                                    // T has been read
#pragma unroll
      for (int e = 0; e < 32; e += 4) {
        uint2 h2, l2;
        const int at = ld_at<8>(j, e >> 2) + half * 4;
        ld_split(d[e] * up_d, d[e + 1] * up_d, h2.x, l2.x), ld_split(d[e + 2] * up_d, d[e + 3] * up_d, h2.y, l2.y);
        *(uint2*)(td + at) = h2, *(uint2*)(td + LD_C * LD_C + at) = l2;
      }
    }
  }
  if (tid == 0) ld_bulk_read();  // the rows of k are on their way
  __syncthreads();
  uint16_t* const kt_hi = (uint16_t*)A;
  uint16_t* const kt_lo = ks;
  if constexpr (DELTA) {
    // K~ = T^T D K: a warp has Dk / 4 columns
    constexpr int N = DK / 32;
    float kt[4][N][4] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // 16 tokens i of the sum
      uint32_t b[N][2];
#pragma unroll
      for (int n = 0; n < N; n += 2) {
        uint32_t b4[4];
        ld_matrix4_trans(b4, ks + ld_at<PIECES>(i * 16 + (lane & 15), warp * N + n + (lane >> 4)));
        b[n][0] = b4[0], b[n][1] = b4[1], b[n + 1][0] = b4[2], b[n + 1][1] = b4[3];
      }
#pragma unroll
      for (int j = 0; j <= i; ++j) {
        uint32_t hi[4], lo[4];
        const int at = ld_at<8>(j * 16 + (lane & 15), i * 2 + (lane >> 4));
        ld_matrix4(lo, td + LD_C * LD_C + at);
        ld_matrix4(hi, td + at);
#pragma unroll
        for (int n = 0; n < N; ++n) ld_mma(kt[j][n], lo, b[n][0], b[n][1]);
#pragma unroll
        for (int n = 0; n < N; ++n) ld_mma(kt[j][n], hi, b[n][0], b[n][1]);
      }
    }
    __syncthreads();  // T^T D and the rows of k have been read
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r) {  // at most 64 x 2^14 x 2: 2^-6 of it is an fp16 number
          uint32_t hi, lo;
          ld_split(kt[j][n][2 * r] * 0x1p-6f, kt[j][n][2 * r + 1] * 0x1p-6f, hi, lo);
          const int at = ld_at<PIECES>(j * 16 + g + r * 8, warp * N + n) + cc * 2;
          *(uint32_t*)(kt_hi + at) = hi, *(uint32_t*)(kt_lo + at) = lo;
        }
  } else {
    // K~ = D K
    for (int i = tid; i < LD_C * PIECES; i += LD_PREP_THREADS) {
      const int j = i / PIECES;
      const uint4 raw = *(const uint4*)(ks + i * 8);  // the piece's place in its row does not matter: row j's are together
      const bool finite = fabsf(d_s[j]) <= LD_MAX;
      float up, down;
      ld_scale(finite ? fabsf(d_s[j]) : 1.0f, up, down);
      const float f = finite ? d_s[j] * up * 0x1p-7f : 0.0f;
      uint4 hi, lo;  // the low ones in the piece's own place
      ld_split(h_lo(raw.x) * f, h_hi(raw.x) * f, hi.x, lo.x), ld_split(h_lo(raw.y) * f, h_hi(raw.y) * f, hi.y, lo.y);
      ld_split(h_lo(raw.z) * f, h_hi(raw.z) * f, hi.z, lo.z), ld_split(h_lo(raw.w) * f, h_hi(raw.w) * f, hi.w, lo.w);
      ((uint4*)kt_hi)[i] = hi, ((uint4*)kt_lo)[i] = lo;
    }
    if (tid < LD_C) {
      const bool finite = fabsf(d_s[tid]) <= LD_MAX;
      float up, down;
      ld_scale(finite ? fabsf(d_s[tid]) : 1.0f, up, down);
      kt_scale[tid] = d_s[tid] != 0.0f ? down * 0x1p7f : 0.0f;
      if (!finite) bad_s[first] = 1;
    }
  }
  fence_async_smem();
  __syncthreads();
  if (tid == 0) {
    ld_bulk_out(out->kt_hi, kt_hi, sizeof(out->kt_hi));
    ld_bulk_out(out->kt_lo, kt_lo, sizeof(out->kt_lo));
    ld_bulk_out(out->q, qs, sizeof(out->q));
    ld_bulk_commit();
  }
  if (tid < LD_C) {
    const float nan = __uint_as_float(0x7fc00000u);
    const bool bad = bad_s[first] != 0, live = my_line >= 0;
    out->gamma[tid] = ld_exp(G_s[tid].x + G_s[tid].y);
    out->kt_scale[tid] = !live ? 0.0f : bad ? nan : kt_scale[tid];
    out->r_in[tid] = r_in_s[tid];
    out->q_scale[tid] = !live ? 0.0f : lost ? nan : q_scale_s[tid];
  }
  if (tid == 0) ld_bulk_done();
}

// ---- The scan. A CTA has 16 x WARPS rows of a head's state of one line and goes along the line's chunks. 16 rows are a team of
// warps: one, or PARTS = 2 that have half of the state's columns and half of the chunk's tokens each, carry the state, S -> R -> S;
// as many others make the outputs from what those leave in shared memory (S's terms, and R as it is), a step behind, so that their
// products and conversions fill what the first ones leave of the tensor core and of the issue slots. They take P T into registers and
// let the chunk's stage go before R comes: the next chunk but one is asked for by then. S stays in registers, as the accumulator of
// products [rows of S, tokens or columns of K]; an accumulator of mma.sync is laid out as the next product's A operand is, so that a
// single warp's chain has no exchange in it. Two warps give one another their terms of S and of R, and each begins with its own while
// the other's come. K, Q, K~ and P T, as B operands, come from shared memory, where the first output warp keeps chunks coming (bulk
// copies; the rows of v by TMA). (tcgen05 would want S as a 16-bit operand in shared or tensor memory, and R brought there and back
// between the products: with 16 rows a warp the chain is shorter in registers.)
//
// Bound by the chain's latency: 8192 tokens are 128 chunks one after another, and a head's rows are all that can be spread. Measured
// (B200, 16 / 32 heads of 128, one line): 2.4 us a chunk, of which the 160 products of a warp that carries the state take 1330 of its
// tensor core's clocks and the 94 of the output warp beside it 780; the rest are conversions (500 for R, 320 for its terms), barriers
// and the latency of what they wait for. One warp a team with four teams a CTA (which share the operands' loads) takes 3.9 us a chunk
// and half the SMs: the better where lines and heads fill the GPU.
template <int DK, int WARPS, int PARTS> struct LdScanShape {
  static constexpr int HEAD = sizeof(LdRows<DK>), V = HEAD + sizeof(LdHead<DK>), STAGE = V + WARPS * LD_C * 32;
  // a team's place: S's terms as A fragments, with its rows' scales of each part; R times K~'s factors likewise, for the other part; R
  // itself, for the outputs; those; and each part's first tokens that are not finite, where there are such
  static constexpr int S_SCALES = DK * 64, RK = S_SCALES + 128, RK_SCALES = RK + (PARTS > 1 ? LD_C * 64 : 0);
  static constexpr int R = RK_SCALES + 128, OUT = R + LD_C * 64, CLEAN = OUT + LD_C * 32, TEAM = CLEAN + 128;
  static constexpr int ROOM = 227 * 1024 - 2048 - WARPS * TEAM, STAGES = ROOM / STAGE < 4 ? ROOM / STAGE : 4;
  static constexpr int SMEM = STAGES * STAGE + WARPS * TEAM + 1024;
  static constexpr int OUTS = PARTS;  // warps for the outputs, each of a share of the tokens: as many on every quarter of an SM
  static constexpr int THREADS = WARPS * (PARTS + OUTS) * 32;
  static_assert(STAGES >= 2, "a chunk is loaded while the one before it is worked on");
};

// 1 / x of a power of two.
D3_DEV float ld_inverse(float x) { return __uint_as_float(0x7f000000u - __float_as_uint(x)); }

// Largest of the values of a row held by the four lanes of a group.
D3_DEV float ld_row_most(float m) {
  m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
  return fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
}

// The larger one; NaN where one is.
D3_DEV float ld_most(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// mbar_wait by a whole warp, the same answer in all lanes.
D3_DEV bool ld_wait(uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity)); }
// What this warp has written or read is done with: one arrival.
D3_DEV void ld_arrive(uint64_t* bar, int lane) {
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
}

template <int TYPE, int DK, bool DELTA, int WARPS, int PARTS>
__global__ void __launch_bounds__(LdScanShape<DK, WARPS, PARTS>::THREADS, 1)
    lines_delta_scan_kernel(const __grid_constant__ CUtensorMap vmap, LdChunkArgs c) {
  using TT = QrType<TYPE>;
  using Shape = LdScanShape<DK, WARPS, PARTS>;
  constexpr int PIECES = DK / 8, NK = DK / 8 / PARTS, KT = DK / 16 / PARTS, NT = LD_C / 8, STAGES = Shape::STAGES;
  constexpr int G = NK < 8 ? NK : 8;  // sums of S that take turns
  constexpr int OUTS = Shape::OUTS, NO = NT / OUTS;
  extern __shared__ uint8_t ld_raw[];
  __shared__ __align__(8) uint64_t full[STAGES], empty[STAGES];  // the chunks' stages
  // a team's S and R: written (R times K~'s factors too), and both read by the outputs. A part writes the next S when the outputs have
  // read this one, and has the other part's when that has written it, so that none is ever two phases ahead.
  __shared__ __align__(8) uint64_t s_full[WARPS], rk_full[WARPS], r_full[WARPS], read[WARPS];
  __shared__ int odd_s[WARPS][PARTS];  // 1 + the last chunk with values that are not finite
  const LdArgs& a = c.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, cc = lane & 3;
  const int h = blockIdx.y, b = blockIdx.z;
  const bool outputs = warp >= WARPS * PARTS;
  const int team = (outputs ? warp - WARPS * PARTS : warp) / PARTS, part = warp % PARTS;  // OUTS is PARTS
  uint8_t* const ring = (uint8_t*)(((uintptr_t)ld_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* const place = ring + STAGES * Shape::STAGE + team * Shape::TEAM;
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], (PARTS + OUTS) * WARPS);
    for (int i = 0; i < WARPS; ++i) {
      mbar_init(&s_full[i], PARTS), mbar_init(&rk_full[i], PARTS), mbar_init(&r_full[i], PARTS);
      mbar_init(&read[i], OUTS);
      for (int y = 0; y < PARTS; ++y) odd_s[i][y] = 0;
    }
    fence_mbar_init();
  }
  __syncthreads();
  grid_dependency_wait();
  allow_dependents();
  const long long first_token = (long long)c.block0 * LD_C, end_token = min((long long)a.T, first_token + (long long)c.blocks * LD_C);
  const int row0 = (blockIdx.x * WARPS + team) * 16;  // this team's rows of the state
  const bool there = row0 < a.Dv;
  if (b == a.B) {  // the places past the lines' last token
    const long long from = max((long long)min(max(a.cu[b], 0), a.T), first_token);
    if (outputs && part == 0 && there)
      for (long long t = from + (lane >> 1); t < end_token; t += 16)
        *(uint4*)((uint16_t*)a.out + (t * a.Hv + h) * a.Dv + row0 + (lane & 1) * 8) = make_uint4(0, 0, 0, 0);
    return;
  }
  const long long s = max((long long)min(max(a.cu[b], 0), a.T), first_token), e = min((long long)a.cu[b + 1], end_token);
  if (e <= s) return;
  const int block_a = (int)((s - first_token) / LD_C), chunks = (int)((e - 1 - first_token) / LD_C) - block_a + 1;
  bool ok = true;
  if (outputs) {
    constexpr uint32_t row_bytes = DELTA ? sizeof(LdRows<DK>) : 0;  // for K S^T
    // 16 tokens at a time, of two warps' two times those that have as many blocks of P T before them
    auto tokens = [&](int x) { return (PARTS == 1 ? x : x == 0 ? part : 3 - part) * 16; };
    auto blocks_of = [](int x) constexpr { return PARTS == 1 ? x + 1 : x == 0 ? 2 : 4; };  // at most
    const int v_boxes = min(WARPS, (a.Dv - (int)blockIdx.x * WARPS * 16) / 16);
    const uint64_t keep = policy_evict_last();
    const LdRows<DK>* rows_at = (const LdRows<DK>*)c.rows + (size_t)block_a * a.Hk + h / (a.Hv / a.Hk);
    const LdHead<DK>* head_at = (const LdHead<DK>*)c.heads + (size_t)block_a * a.Hv + h;
    int token_at = (int)(first_token + (long long)block_a * LD_C), loads = 0;
    auto load = [&] {  // the next chunk; by one lane, whose stage is free
      uint8_t* const to = ring + loads % STAGES * Shape::STAGE;
      uint64_t* const bar = &full[loads % STAGES];
      mbar_arrive_expect_tx(bar, row_bytes + (uint32_t)sizeof(LdHead<DK>) + v_boxes * LD_C * 32);
      if (DELTA) bulk_g2s(to, rows_at, row_bytes, bar, keep);
      bulk_g2s(to + Shape::HEAD, head_at, sizeof(LdHead<DK>), bar, keep);
      for (int w = 0; w < v_boxes; ++w)
        tma_load_3d(smem_u32(to + Shape::V + w * LD_C * 32), &vmap, (blockIdx.x * WARPS + w) * 16, h, token_at, bar);
      rows_at += a.Hk, head_at += a.Hv, token_at += LD_C;
      ++loads;
    };
    if (warp == WARPS * PARTS && lane == 0)
      for (int i = 0; i < STAGES && i < chunks; ++i) load();
    const uint32_t out_token = (uint32_t)a.Hv * a.Dv;  // at most 2^24
    uint16_t* out_at = (uint16_t*)a.out + ((first_token + (long long)block_a * LD_C) * a.Hv + h) * a.Dv + row0 + (lane & 1) * 8;
#pragma unroll 1
    for (int i = 0; i < chunks && ok; ++i) {
      const int st = i % STAGES;
      ok = ld_wait(&full[st], (i / STAGES) & 1) && ld_wait(&s_full[team], i & 1);
      if (!ok) break;
      bool released = true;
      if (warp == WARPS * PARTS && lane == 0 && i > 0 && loads < chunks) {  // the stage of the chunk before this one
        released = mbar_wait(&empty[(i - 1) % STAGES], ((i - 1) / STAGES) & 1);
        if (released) load();
      }
      ok = __all_sync(0xffffffffu, released);  // where it ran out, the warp goes through this chunk and leaves the loop together
      const uint8_t* const stage = ring + st * Shape::STAGE;
      const LdHead<DK>& head = *(const LdHead<DK>*)(stage + Shape::HEAD);
      const long long t0 = first_token + (long long)(block_a + i) * LD_C;
      const int lo = (int)max(0ll, s - t0), hi = (int)min((long long)LD_C, e - t0);
      float O[PARTS][NO][4] = {};
#pragma unroll
      for (int kt = 0; kt < DK / 16; ++kt) {
        const uint4* const from = (const uint4*)place + kt * 32 + lane;
        const uint4 h = from[0], l = from[DK * 2];
        const uint32_t h4[4] = {h.x, h.y, h.z, h.w}, l4[4] = {l.x, l.y, l.z, l.w};
        uint32_t q4[NO / 2][4];
#pragma unroll
        for (int x = 0; x < NO / 2; ++x)
          ld_matrix4(q4[x], head.q + ld_at<PIECES>(tokens(x) + (lane & 7) + (lane >> 4) * 8, kt * 2 + ((lane >> 3) & 1)));
#pragma unroll
        for (int x = 0; x < NO; ++x) ld_mma(O[kt / KT][x], l4, q4[x / 2][x % 2 * 2], q4[x / 2][x % 2 * 2 + 1]);
#pragma unroll
        for (int x = 0; x < NO; ++x) ld_mma(O[kt / KT][x], h4, q4[x / 2][x % 2 * 2], q4[x / 2][x % 2 * 2 + 1]);
      }
      // P T and the factors of the columns, so that the stage is free before R comes
      uint32_t p_hi[NO / 2][LD_C / 16][4];
      uint2 p_rest[NO / 2][LD_C / 16];
      float2 fp[NO];
#pragma unroll
      for (int x = 0; x < NO / 2; ++x)
#pragma unroll
        for (int kt = 0; kt < blocks_of(x); ++kt)
          if (kt * 16 <= tokens(x)) {
            ld_matrix4(p_hi[x][kt], head.p + ld_at<8>(tokens(x) + (lane & 7) + (lane >> 4) * 8, kt * 2 + ((lane >> 3) & 1)));
            p_rest[x][kt] = *(const uint2*)(head.p + ld_rest(tokens(x) / 16, kt, lane));
          }
      const float* const s_scales = (const float*)(place + Shape::S_SCALES);
#pragma unroll
      for (int n = 0; n < NO; ++n) {
        const int j = tokens(n / 2) + n % 2 * 8 + cc * 2;
        const float2 fq = *(const float2*)(head.q_scale + j);
        fp[n] = *(const float2*)(head.p_scale + j);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          float o = O[0][n][x] * s_scales[g + (x >> 1) * 8];
#pragma unroll
          for (int y = 1; y < PARTS; ++y) o = fmaf(O[y][n][x], s_scales[y * 16 + g + (x >> 1) * 8], o);
          O[0][n][x] = o * (x & 1 ? fq.y : fq.x);
        }
      }
      ld_arrive(&empty[st], lane);
      ok = ld_wait(&r_full[team], i & 1);
      if (!ok) break;
      // R as A fragments of two terms, rows by a power of two; low ones times 2^11, as P T's: what is small beside the row's largest
      // keeps its bits. (Without the delta rule R is V, and values of fp16 are one term as they are.)
      constexpr bool ONE_TERM = !DELTA && TYPE == QR_F16;
      uint32_t r_hi[LD_C / 16][4], r_lo[LD_C / 16][4];
      float r_down[2];
      int until = LD_C;  // of column lane % 16
      {
        float4 v[NT];
        float most[2] = {0.0f, 0.0f}, up[2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          v[n] = ((const float4*)(place + Shape::R))[n * 32 + lane];
          most[0] = fmaxf(most[0], fmaxf(fabsf(v[n].x), fabsf(v[n].y)));
          most[1] = fmaxf(most[1], fmaxf(fabsf(v[n].z), fabsf(v[n].w)));
        }
#pragma unroll
        for (int y = 0; y < PARTS; ++y)  // a value that is not finite: its column's outputs from there on
          if (odd_s[team][y] == i + 1) until = min(until, ((const int*)(place + Shape::CLEAN))[y * 16 + lane % 16]);
        ld_arrive(&read[team], lane);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          up[r] = r_down[r] = 1.0f;
          if (!ONE_TERM) ld_scale(ld_row_most(most[r]), up[r], r_down[r]);
        }
#pragma unroll
        for (int kt = 0; kt < LD_C / 16; ++kt)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float4& from = v[2 * kt + (x >> 1)];
            const float v0 = (x & 1 ? from.z : from.x) * up[x & 1], v1 = (x & 1 ? from.w : from.y) * up[x & 1];
            r_hi[kt][x] = ld_half2(v0, v1);
            if (!ONE_TERM) r_lo[kt][x] = ld_half2((v0 - h_lo(r_hi[kt][x])) * 0x1p11f, (v1 - h_hi(r_hi[kt][x])) * 0x1p11f);
          }
      }
      uint8_t* const out_s = place + Shape::OUT;
#pragma unroll
      for (int m = 0; m < NO; m += 2) {
        float high[2][4] = {}, low[2][4] = {};  // the latter times 2^11
#pragma unroll
        for (int kt = 0; kt < blocks_of(m / 2); ++kt)
          if (kt * 16 <= tokens(m / 2)) {
            const auto& p = p_hi[m / 2][kt];
            const uint2 rest = p_rest[m / 2][kt];
            // a byte of e5m2 is the upper one of an fp16 number
            const uint32_t p_lo[4] = {__byte_perm(rest.x, 0, 0x1404), __byte_perm(rest.x, 0, 0x3424), __byte_perm(rest.y, 0, 0x1404),
                                      __byte_perm(rest.y, 0, 0x3424)};
            if (!ONE_TERM) ld_mma(low[0], r_lo[kt], p[0], p[1]), ld_mma(low[1], r_lo[kt], p[2], p[3]);
            ld_mma(high[0], r_hi[kt], p[0], p[1]), ld_mma(high[1], r_hi[kt], p[2], p[3]);
            ld_mma(low[0], r_hi[kt], p_lo[0], p_lo[1]), ld_mma(low[1], r_hi[kt], p_lo[2], p_lo[3]);
          }
        uint32_t o4[4];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float o[4];
#pragma unroll
          for (int y = 0; y < 4; ++y)
            o[y] = fmaf(fmaf(low[x][y], 0x1p-11f, high[x][y]) * (y & 1 ? fp[m + x].y : fp[m + x].x), r_down[y >> 1], O[0][m + x][y]);
          o4[2 * x] = TT::put2(o[0], o[1]), o4[2 * x + 1] = TT::put2(o[2], o[3]);
        }
        const int token = tokens(m / 2) + (lane & 7) + (lane >> 4) * 8, piece = ((lane >> 3) & 1) ^ ((token >> 2) & 1);
        st_matrix4_trans(out_s + token * 32 + piece * 16, o4[0], o4[1], o4[2], o4[3]);
      }
      __syncwarp();
      if (__any_sync(0xffffffffu, until < LD_C)) {
#pragma unroll 1
        for (int x = 0; x < NO / 2; ++x)
#pragma unroll 1
          for (int token = max(tokens(x) + lane / 16 * 8, until); token < tokens(x) + lane / 16 * 8 + 8; ++token)
            *(uint16_t*)(out_s + token * 32 + ((lane / 8 & 1) ^ ((token >> 2) & 1)) * 16 + lane % 8 * 2) = 0x7fff;  // NaN in both types
        __syncwarp();
      }
      if (there)
#pragma unroll
        for (int x = 0; x < LD_C / 16 / OUTS; ++x) {
          const int token = tokens(x) + (lane >> 1), piece = (lane & 1) ^ ((token >> 2) & 1);
          if (token >= lo && token < hi)
            *(uint4*)(out_at + (size_t)token * out_token) = *(const uint4*)(out_s + token * 32 + piece * 16);
        }
      out_at += (size_t)LD_C * out_token;
      __syncwarp();  // its outputs have been read
    }
    // copies in flight land before the block ends (where a wait ran out: those of the other chunks have been waited for)
    if (warp == WARPS * PARTS && lane == 0 && !ok)
      for (int i = loads - 1; i >= 0 && i >= loads - STAGES; --i) mbar_wait(&full[i % STAGES], (i / STAGES) & 1);
    return;
  }
  // ---- the state
  float* const state = a.state + (((size_t)b * a.Hv + h) * a.Dv + row0) * DK + part * (DK / PARTS);
  const uint32_t quad = 0xfu << (lane & ~3);  // the lanes of this one's rows
  float S[NK][4] = {};                        // times down[] it is the state
  float down[2] = {1.0f, 1.0f};
  if (there)
#pragma unroll
    for (int n = 0; n < NK; ++n) {
      const float2 x = *(const float2*)(state + g * DK + n * 8 + cc * 2), y = *(const float2*)(state + (g + 8) * DK + n * 8 + cc * 2);
      S[n][0] = x.x, S[n][1] = x.y, S[n][2] = y.x, S[n][3] = y.y;
    }
  ok = ld_wait(&full[0], 0);
#pragma unroll 1
  for (int i = 0; i < chunks && ok; ++i) {
    const int st = i % STAGES;
    const uint8_t* const stage = ring + st * Shape::STAGE;
    const LdRows<DK>& rows = *(const LdRows<DK>*)stage;
    const LdHead<DK>& head = *(const LdHead<DK>*)(stage + Shape::HEAD);
    const uint8_t* const v_s = stage + Shape::V + team * LD_C * 32;
    const long long t0 = first_token + (long long)(block_a + i) * LD_C;
    const int lo = (int)max(0ll, s - t0), hi = (int)min((long long)LD_C, e - t0);
    const bool partial = lo > 0 || hi < LD_C;
    // operands are asked for before what they are multiplied by is known
    uint32_t k4[2][NO / 2][4];
    auto get_k = [&](int step, int at, int x) {  // 16 columns `at` of 16 of this part's tokens
      ld_matrix4(k4[step & 1][x], rows.k + ld_at<PIECES>((part * NO + x * 2) * 8 + (lane & 7) + (lane >> 4) * 8, at * 2 + ((lane >> 3) & 1)));
    };
    if (DELTA)
#pragma unroll
      for (int x = 0; x < NO / 2; ++x) get_k(0, part * KT, x);
    // S's rows between 2^9 and 2^15 at their largest, which is nearly always so already: votes tell, without the largest itself
    {
      float m[2] = {0.0f, 0.0f};
#pragma unroll
      for (int n = 0; n < NK; ++n) {
        m[0] = fmaxf(m[0], fmaxf(fabsf(S[n][0]), fabsf(S[n][1])));
        m[1] = fmaxf(m[1], fmaxf(fabsf(S[n][2]), fabsf(S[n][3])));
      }
      const uint32_t some[2] = {__ballot_sync(0xffffffffu, m[0] >= 0x1p9f), __ballot_sync(0xffffffffu, m[1] >= 0x1p9f)};
      const bool off = fmaxf(m[0], m[1]) >= 0x1p15f || !(some[0] & quad) || !(some[1] & quad);
      if (__any_sync(0xffffffffu, off)) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float up, dn;
          ld_scale(ld_row_most(m[r]) * down[r], up, dn);
          up *= down[r];
          down[r] = dn;
#pragma unroll
          for (int n = 0; n < NK; ++n) S[n][2 * r] *= up, S[n][2 * r + 1] *= up;
        }
      }
    }
    // S K^T for this part's tokens, high and low terms of S apart so that the sums take turns. S's terms go to the outputs and to the
    // other part, whose columns' products come second, when its terms are there. Conversions and loads of the next step stand between the
    // products of this one: a warp's instructions issue in order, and a product holds its pipe for 8 clocks.
    float high[PARTS][NO][4] = {}, low[PARTS][NO][4] = {};
    auto s_term = [&](int kt, int x, uint32_t& h, uint32_t& l) {
      ld_split(S[2 * kt + (x >> 1)][(x & 1) * 2], S[2 * kt + (x >> 1)][(x & 1) * 2 + 1], h, l);
    };
    auto products = [&](int who, int step, const uint32_t (&h)[4], const uint32_t (&l)[4], auto&& between) {
      const auto& k = k4[step & 1];
#pragma unroll
      for (int x = 0; x < 2 * NO; ++x) {
        const int n = x % NO;
        if (DELTA) {
          if (x < NO)
            ld_mma(high[who][n], h, k[n / 2][n % 2 * 2], k[n / 2][n % 2 * 2 + 1]);
          else
            ld_mma(low[who][n], l, k[n / 2][n % 2 * 2], k[n / 2][n % 2 * 2 + 1]);
        }
        between(x);
      }
    };
    float other_down[2] = {0.0f, 0.0f};
    auto publish_scales = [&] {
      if (cc == 0) {
        float* const s_scales = (float*)(place + Shape::S_SCALES) + part * 16;
        s_scales[g] = down[0], s_scales[g + 8] = down[1];
      }
      ld_arrive(&s_full[team], lane);
    };
    if constexpr (PARTS == 1) {
      uint32_t h4[2][4], l4[2][4];
#pragma unroll
      for (int x = 0; x < 4; ++x) s_term(0, x, h4[0][x], l4[0][x]);
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        uint4* const to = (uint4*)place + kt * 32 + lane;
        to[0] = make_uint4(h4[kt & 1][0], h4[kt & 1][1], h4[kt & 1][2], h4[kt & 1][3]);
        to[DK * 2] = make_uint4(l4[kt & 1][0], l4[kt & 1][1], l4[kt & 1][2], l4[kt & 1][3]);
        products(0, kt, h4[kt & 1], l4[kt & 1], [&](int x) {
          if (kt + 1 < KT) {
            if (x % 4 == 1) s_term(kt + 1, x / 4, h4[(kt + 1) & 1][x / 4], l4[(kt + 1) & 1][x / 4]);
            if (DELTA && x % 4 == 3) get_k(kt + 1, kt + 1, x / 4);
          }
        });
      }
      publish_scales();
    } else {
      uint32_t h4[KT][4], l4[KT][4];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
        for (int x = 0; x < 4; ++x) s_term(kt, x, h4[kt][x], l4[kt][x]);
        uint4* const to = (uint4*)place + (part * KT + kt) * 32 + lane;
        to[0] = make_uint4(h4[kt][0], h4[kt][1], h4[kt][2], h4[kt][3]);
        to[DK * 2] = make_uint4(l4[kt][0], l4[kt][1], l4[kt][2], l4[kt][3]);
      }
      publish_scales();
      const int other = (1 - part) * KT;
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
        products(0, kt, h4[kt], l4[kt], [&](int x) {
          if (DELTA && x % 4 == 3) get_k(kt + 1, kt + 1 < KT ? part * KT + kt + 1 : other, x / 4);
        });
      ok = ld_wait(&s_full[team], i & 1);
      if (!ok) break;
      if (DELTA) {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          const uint4* const from = (const uint4*)place + (other + kt) * 32 + lane;
          const uint4 h = from[0], l = from[DK * 2];
          h4[kt][0] = h.x, h4[kt][1] = h.y, h4[kt][2] = h.z, h4[kt][3] = h.w;
          l4[kt][0] = l.x, l4[kt][1] = l.y, l4[kt][2] = l.z, l4[kt][3] = l.w;
        }
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
          products(PARTS - 1, KT + kt, h4[kt], l4[kt], [&](int x) {
            if (kt + 1 < KT && x % 4 == 3) get_k(KT + kt + 1, other + kt + 1, x / 4);
          });
        const float* const s_scales = (const float*)(place + Shape::S_SCALES) + (1 - part) * 16;
        other_down[0] = s_scales[g], other_down[1] = s_scales[g + 8];
      }
    }
    // K~'s first columns; R = V - gamma K S^T of this part's tokens, zeros for those of other lines; R times K~'s factors
    uint32_t b_hi[2][G / 2][4], b_lo[2][G / 2][4];
    constexpr int KR = LD_C / 16 / PARTS, STEPS = LD_C / 16 * (NK / G);
    auto get_b = [&](int at, int x) {  // step `at`: G columns of this part, 16 tokens, its own first
      const int group = at / (LD_C / 16), kt = (at % (LD_C / 16) + part * KR) % (LD_C / 16);
      const int where = ld_at<PIECES>(kt * 16 + (lane & 15), part * NK + group * G + x / 2 * 2 + (lane >> 4));
      if (x % 2) ld_matrix4_trans(b_hi[at & 1][x / 2], head.kt_hi + where);
      else ld_matrix4_trans(b_lo[at & 1][x / 2], head.kt_lo + where);
    };
    float RK[NO][4], m[2] = {0.0f, 0.0f};
    {
      uint32_t v4[NO / 2][4];
#pragma unroll
      for (int n = 0; n < NO; n += 2) {
        const int token = (part * NO + n) * 8 + (lane & 7) + (lane >> 4) * 8, piece = ((lane >> 3) & 1) ^ ((token >> 2) & 1);
        ld_matrix4_trans(v4[n / 2], v_s + token * 32 + piece * 16);
      }
#pragma unroll
      for (int n = 0; n < NO; ++n) {
        const int j = (part * NO + n) * 8 + cc * 2;
        float v[4];
        float2 f = *(const float2*)(head.kt_scale + j);
        TT::get2(v4[n / 2][n % 2 * 2], v[0], v[1]);
        TT::get2(v4[n / 2][n % 2 * 2 + 1], v[2], v[3]);
        if (DELTA) {
          const float2 in = *(const float2*)(head.r_in + j);
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            float ks = (high[0][n][y] + low[0][n][y]) * down[y >> 1];
            if (PARTS > 1) ks = fmaf(high[PARTS - 1][n][y] + low[PARTS - 1][n][y], other_down[y >> 1], ks);
            v[y] = fmaf(-ks, y & 1 ? in.y : in.x, v[y]);
          }
        }
        if (partial) {
          if (j < lo || j >= hi) v[0] = v[2] = f.x = 0.0f;
          if (j + 1 < lo || j + 1 >= hi) v[1] = v[3] = f.y = 0.0f;
        }
        ((float4*)(place + Shape::R))[(part * NO + n) * 32 + lane] = make_float4(v[0], v[1], v[2], v[3]);
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          RK[n][y] = v[y] * (y & 1 ? f.y : f.x);
          m[y >> 1] = ld_most(m[y >> 1], fabsf(RK[n][y]));
        }
        if (n < G) get_b(0, n);
      }
      if (NO < G)
#pragma unroll
        for (int n = NO; n < G; ++n) get_b(0, n);
    }
    if (__any_sync(0xffffffffu, !(ld_most(m[0], m[1]) <= LD_MAX))) {  // outputs before a value that is not finite stay clear of it
      int clean[2] = {LD_C, LD_C};
#pragma unroll 1
      for (int n = NO - 1; n >= 0; --n) {
        float* const v = (float*)(place + Shape::R) + ((part * NO + n) * 32 + lane) * 4;
#pragma unroll
        for (int y = 3; y >= 0; --y)
          if (!(fabsf(v[y]) <= LD_MAX)) v[y] = 0.0f, clean[y >> 1] = (part * NO + n) * 8 + cc * 2 + (y & 1);
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) clean[r] = min(clean[r], __shfl_xor_sync(0xffffffffu, clean[r], o));
        if (cc == 0) ((int*)(place + Shape::CLEAN))[part * 16 + g + r * 8] = clean[r];
      }
      odd_s[team][part] = i + 1;
    }
    ld_arrive(&r_full[team], lane);
    // its two terms, for this part's columns and the other's. Each part's tokens have a scale.
    uint32_t h4[LD_C / 16][4], l4[LD_C / 16][4];
    float rk_down[PARTS][2];
    {
      float up[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) ld_scale(ld_row_most(m[r]), up[r], rk_down[0][r]);
#pragma unroll
      for (int kt = 0; kt < KR; ++kt) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int n = 2 * kt + (x >> 1), y = x & 1;
          ld_split(RK[n][2 * y] * up[y], RK[n][2 * y + 1] * up[y], h4[kt][x], l4[kt][x]);
        }
        if (PARTS > 1) {
          uint4* const to = (uint4*)(place + Shape::RK) + (part * KR + kt) * 64 + lane;
          to[0] = make_uint4(h4[kt][0], h4[kt][1], h4[kt][2], h4[kt][3]);
          to[32] = make_uint4(l4[kt][0], l4[kt][1], l4[kt][2], l4[kt][3]);
        }
      }
      if (PARTS > 1) {
        if (cc == 0) {
          float* const rk_scales = (float*)(place + Shape::RK_SCALES) + part * 16;
          rk_scales[g] = rk_down[0][0], rk_scales[g + 8] = rk_down[0][1];
        }
        ld_arrive(&rk_full[team], lane);
      }
    }
    // S = gamma_last S + R^T K~, G columns at a time, each part's tokens in a sum of their own
    const float gamma = head.gamma[hi - 1];
    bool next = true;
#pragma unroll
    for (int group = 0; group < NK / G; ++group) {
      float sum[PARTS][G][4] = {};
#pragma unroll
      for (int kt = 0; kt < LD_C / 16; ++kt) {
        const int at = group * (LD_C / 16) + kt, who = kt / KR;
        if (PARTS > 1 && kt == KR) {  // the other part's
          ok = ld_wait(&rk_full[team], i & 1);
#pragma unroll
          for (int y = 0; y < KR; ++y) {
            const uint4* const from = (const uint4*)(place + Shape::RK) + ((1 - part) * KR + y) * 64 + lane;
            const uint4 h = from[0], l = from[32];
            h4[(KR + y) % (LD_C / 16)][0] = h.x, h4[(KR + y) % (LD_C / 16)][1] = h.y;
            h4[(KR + y) % (LD_C / 16)][2] = h.z, h4[(KR + y) % (LD_C / 16)][3] = h.w;
            l4[(KR + y) % (LD_C / 16)][0] = l.x, l4[(KR + y) % (LD_C / 16)][1] = l.y;
            l4[(KR + y) % (LD_C / 16)][2] = l.z, l4[(KR + y) % (LD_C / 16)][3] = l.w;
          }
          const float* const rk_scales = (const float*)(place + Shape::RK_SCALES) + (1 - part) * 16;
          rk_down[PARTS - 1][0] = rk_scales[g], rk_down[PARTS - 1][1] = rk_scales[g + 8];
        }
        const auto& bh = b_hi[at & 1];
        const auto& bl = b_lo[at & 1];
#pragma unroll
        for (int x = 0; x < 3 * G; ++x) {
          const int y = x % G;
          if (x < G) ld_mma(sum[who][y], h4[kt], bl[y / 2][y % 2 * 2], bl[y / 2][y % 2 * 2 + 1]);
          else if (x < 2 * G) ld_mma(sum[who][y], l4[kt], bh[y / 2][y % 2 * 2], bh[y / 2][y % 2 * 2 + 1]);
          else ld_mma(sum[who][y], h4[kt], bh[y / 2][y % 2 * 2], bh[y / 2][y % 2 * 2 + 1]);
          if (x % 3 == 0 && at + 1 < STEPS) get_b(at + 1, x / 3);
          if (at == STEPS - 1 && x == 3 * G / 2 && i + 1 < chunks)
            next = mbar_wait(&full[(i + 1) % STAGES], ((i + 1) / STAGES) & 1) && mbar_wait(&read[team], i & 1);
        }
      }
      if (group == 0) {  // where S vanishes beside what is added, in the scale of that: all stays within 32 bits
        const float most[2] = {fmaxf(rk_down[0][0], rk_down[PARTS - 1][0]), fmaxf(rk_down[0][1], rk_down[PARTS - 1][1])};
        if (__any_sync(0xffffffffu, most[0] > down[0] * 0x1p50f || most[1] > down[1] * 0x1p50f))
#pragma unroll
          for (int r = 0; r < 2; ++r)
            if (most[r] > down[r] * 0x1p50f) {
              const float f = down[r] * ld_inverse(most[r]);
              down[r] = most[r];
#pragma unroll
              for (int n = 0; n < NK; ++n) S[n][2 * r] *= f, S[n][2 * r + 1] *= f;
            }
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float up = ld_inverse(down[r]);
        const float c0 = rk_down[0][r] * up, c1 = PARTS > 1 ? rk_down[PARTS - 1][r] * up : 0.0f;
#pragma unroll
        for (int n = 0; n < G; ++n)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            float& to = S[group * G + n][2 * r + y];
            to = fmaf(sum[0][n][2 * r + y], c0, to * gamma);
            if (PARTS > 1) to = fmaf(sum[PARTS - 1][n][2 * r + y], c1, to);
          }
      }
    }
    ld_arrive(&empty[st], lane);
    next = next && ok;
    ok = __all_sync(0xffffffffu, next);
  }
  if (there && ok)
#pragma unroll
    for (int n = 0; n < NK; ++n) {
      *(float2*)(state + g * DK + n * 8 + cc * 2) = make_float2(S[n][0] * down[0], S[n][1] * down[0]);
      *(float2*)(state + (g + 8) * DK + n * 8 + cc * 2) = make_float2(S[n][2] * down[1], S[n][3] * down[1]);
    }
}

}  // namespace d3
