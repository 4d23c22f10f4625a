// Linear attention (lines_delta.cuh has the formulas) over many tokens of a line: in chunks of 64 tokens, with the products on
// the tensor cores. With G_i the sum of the log decays from the chunk's first token on, gamma_i = exp(G_i), and the rows of a
// chunk's Q, K, V and of the corrections U:
//   (I + A) U = diag(beta) (V - diag(gamma) K S^T),   A_ij = beta_i exp(G_i - G_j) k_i . k_j  (j < i)
//   O = scale (diag(gamma) Q S^T + P U),              P_ij = exp(G_i - G_j) q_i . k_j  (j <= i)
//   S <- gamma_last S + (diag(exp(G_last - G_j)) U)^T K
// so that what depends on the tokens alone, (I + A)^-1 diag(beta) and P, is formed for all chunks at once (the preparation),
// and the chain from chunk to chunk (the scan) has four products left. Exponents are differences that are never above 0, of
// sums in 64 bits.
//
// Chunks are cut from the packed tokens, whatever lines they belong to: entries of two lines are zeros, sums and exponents
// start again with each line. A line's scan masks the tokens of others.
//
// Values. k and q become fp16 rows times powers of two, exactly (values below 2^-14 of the row's largest lose what is below
// 2^-25 of it), and their norms are numbers that the results are multiplied by. What is not exact in 16 bits, S, the right-hand
// sides, U and the inverse, is the sum of two fp16 terms, 22 bits, each row scaled by a power of two of its own; their products
// are summed in 32 bits and the smallest of four, low times low, left out (2^-22). S itself stays in 32 bits. For the outputs, which are
// rounded to 16 bits anyway, one term of S, P and U is enough: 2^-12 of each.
//
// A value that is not finite reaches the state and the tokens of its own line, in its chunk earlier ones too.
#pragma once

#include "lines_delta.cuh"
#include "tcgen05.cuh"

namespace d3 {

constexpr int LD_C = 64;  // tokens of a chunk

// What the preparation leaves of a chunk for a key head: fp16 rows [64][Dk], 16-byte pieces in the order of ld_at.
template <int DK> struct alignas(128) LdRows {
  uint16_t k[LD_C * DK], q[LD_C * DK];
};
// ... and for a value head: rows [64][64] likewise, and factors of the tokens' columns.
struct alignas(128) LdHead {
  uint16_t t_hi[LD_C * LD_C], t_lo[LD_C * LD_C];  // (I + A)^-1 diag(beta), row i times 1 / t_scale[i]
  uint16_t p[LD_C * LD_C];                        // P, row i times 1 / p_scale[i]
  float t_scale[LD_C], p_scale[LD_C];
  float r_in[LD_C];   // gamma_i |k| factor: of K S^T
  float q_in[LD_C];   // scale gamma_i |q| factor: of Q S^T
  float k_out[LD_C];  // exp(G_last - G_j) |k| factor: of U in the state
  float gamma[LD_C];
};

// Element offset of 16-byte piece c of row r in rows of `pieces` of them (a multiple of 8): eight rows' pieces of one column lie
// in different banks.
template <int PIECES> D3_DEV int ld_at(int r, int c) { return (r * PIECES + (c ^ (r & 7))) * 8; }

D3_DEV void ld_matrix4(uint32_t (&r)[4], const uint16_t* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(smem_u32(p))
               : "memory");
}
D3_DEV void ld_matrix4_trans(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(smem_u32(p))
               : "memory");
}
D3_DEV void st_matrix4_trans(void* p, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(smem_u32(p)), "r"(a), "r"(b), "r"(c),
               "r"(d)
               : "memory");
}
D3_DEV void ld_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
D3_DEV uint32_t ld_half2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// x, y as two fp16 terms each.
D3_DEV void ld_split(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = ld_half2(x, y);
  lo = ld_half2(x - h_lo(hi), y - h_hi(hi));
}

// The power of two that takes values of at most `most` below 2^14, and its inverse (exact, normal numbers both; 1 for a row
// of zeros).
D3_DEV void ld_scale(float most, float& up, float& down) {
  const int e = most > 0.0f ? max((int)(__float_as_uint(most) >> 23) - 127, -113) : 13;
  up = __uint_as_float((uint32_t)(127 + 13 - e) << 23);
  down = __uint_as_float((uint32_t)(127 - 13 + e) << 23);
}

struct LdChunkArgs {
  LdArgs a;
  int block0, blocks;  // of the pass's blocks of 64 tokens, those of this launch
  void* rows;          // [blocks][Hk] LdRows
  LdHead* heads;       // [blocks][Hv]
};

// ---- The preparation. A CTA per chunk and key head; its value heads two at a time. k and q come in as 16-bit rows and go out as
// fp16 ones; K K^T and Q K^T are mma.sync products whose results stay in registers for all value heads. The inverse of I + A is
// found by columns, a thread each: x_i = [i = j] - sum_{m < i} A_im x_m, with x in registers and A's entries broadcast from
// shared memory, updating all later rows as soon as x_m is known so that the additions do not wait for one another.
constexpr int LP2_THREADS = 128;
constexpr int LD_PITCH = 68;  // floats of a column of A (and of a row of the inverse) in shared memory

template <int DK> struct LdPrepShape {
  static constexpr int ROWS = 2 * LD_C * DK * 2, A = LD_C * LD_PITCH * 4;
  static constexpr int SMEM = ROWS + 2 * A;
};

template <int TYPE, int DK, bool DELTA>
__global__ void __launch_bounds__(LP2_THREADS, 3) lines_delta_prep_kernel(LdChunkArgs c) {
  using TT = QrType<TYPE>;
  using E = typename TT::T;
  constexpr int PIECES = DK / 8, LANES = PIECES, AT_ONCE = 32 / LANES;
  extern __shared__ __align__(128) uint8_t ld_smem[];
  uint16_t* const ks = (uint16_t*)ld_smem;
  uint16_t* const qs = ks + LD_C * DK;
  float* const As = (float*)(ld_smem + LdPrepShape<DK>::ROWS);  // [2][64 columns][LD_PITCH]
  __shared__ int line_s[LD_C];
  __shared__ int last_s[LD_C];  // the last token of token i's line in the chunk
  __shared__ float k_factor[LD_C], q_factor[LD_C];
  __shared__ double G_s[2][LD_C];
  __shared__ float beta_s[2][LD_C];
  __shared__ int bad_s[2][LD_C];  // row i of the inverse has a value that is not finite
  const LdArgs& a = c.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, cc = lane & 3;
  const int block = blockIdx.x, hk = blockIdx.y, many = a.Hv / a.Hk;
  const long long t0 = (long long)(c.block0 + block) * LD_C;
  grid_dependency_wait();
  allow_dependents();
  if (tid < LD_C) {
    const int l = t0 + tid < a.T ? a.line[t0 + tid] : -1;
    line_s[tid] = l >= 0 && l < a.B ? l : -1;
  }
  // rows to fp16, each by the power of two that brings its largest value into [1, 2)
  const int l = lane % LANES;
#pragma unroll 2
  for (int i = 0; i < 2 * LD_C / 4; i += AT_ONCE) {  // a warp: 16 rows of k, then 16 of q
    const int at = i + lane / LANES;
    const bool is_q = at >= LD_C / 4;
    const int row = warp * (LD_C / 4) + (is_q ? at - LD_C / 4 : at);
    const QrTensor& x = is_q ? a.q : a.k;
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (t0 + row < a.T) raw = *(const uint4*)((const E*)x.p + (t0 + row) * x.token + hk * x.head + l * 8);
    float v[8];
    qr_unpack<TYPE, 8>(&raw.x, v);
    float most = 0.0f;
    bool finite = true;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      most = fmaxf(most, fabsf(v[e]));
      finite = finite && fabsf(v[e]) <= 3.4028234e38f;
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    const uint32_t group = (LANES == 32 ? 0xffffffffu : ((1u << LANES) - 1u)) << (lane / LANES * LANES);
    finite = (__ballot_sync(0xffffffffu, finite) & group) == group;
    float up, down;
    ld_scale(most, up, down);
    up *= 0x1p-13f, down *= 0x1p13f;
    float sum = 0.0f;
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      w[e / 2] = finite ? ld_half2(v[e] * up, v[e + 1] * up) : 0u;
      sum = fmaf(v[e] * up, v[e] * up, fmaf(v[e + 1] * up, v[e + 1] * up, sum));
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    *(uint4*)((is_q ? qs : ks) + ld_at<PIECES>(row, l)) = make_uint4(w[0], w[1], w[2], w[3]);
    // x / sqrt(|x|^2 + eps) = (up x) / sqrt(|up x|^2 + up^2 eps)
    float f = a.eps >= 0.0f ? rsqrtf(sum + a.eps * up * up) : down;
    if (most == 0.0f) f = 0.0f;  // a row of zeros: its factor must not set the scale of what it is summed with
    if (!finite) f = __uint_as_float(0x7fc00000u);
    if (l == 0) (is_q ? q_factor : k_factor)[row] = is_q ? f * a.scale : f;
  }
  __syncthreads();
  if (tid < LD_C) {
    int last = tid;
    while (last + 1 < LD_C && line_s[last + 1] == line_s[tid]) ++last;
    last_s[tid] = last;
  }
  // K K^T and Q K^T: rows 16 warp + g, + 8, columns 8 n + 2 cc, + 1 up to the diagonal
  float kk[8][4] = {}, qk[8][4] = {};
#pragma unroll
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
        ld_mma(qk[n], aq, b[0], b[1]), ld_mma(qk[n + 1], aq, b[2], b[3]);
      }
  }
  // the rows, as every value head's scan reads them
  {
    LdRows<DK>* out = (LdRows<DK>*)c.rows + (size_t)block * a.Hk + hk;
    const uint4* from = (const uint4*)ks;
    for (int i = tid; i < (int)sizeof(LdRows<DK>) / 16; i += LP2_THREADS) ((uint4*)out)[i] = from[i];
  }
  for (int y0 = 0; y0 < many; y0 += 2) {
    const int n_heads = min(2, many - y0);
    __syncthreads();
    {  // gates: two threads of a token's two heads; sums of the log decays that start again with each line
      const int y = tid >> 6, i = tid & 63, h = hk * many + y0 + y;
      double G = 0.0;
      float beta = 0.0f;
      if (y < n_heads && line_s[i] >= 0) {
        const float decay = ld_log_decay<TYPE>(a, t0 + i, h);
        G = decay < -104.0f ? -104.0f : decay;  // exp of it is 0 already; keeps infinities out of the sums, and NaN in
        if (DELTA) beta = ld_beta<TYPE>(a, t0 + i, h);
      }
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double before = __shfl_up_sync(0xffffffffu, G, o);
        if (lane >= o && line_s[i - o] == line_s[i]) G += before;
      }
      G_s[y][i] = G;
      beta_s[y][i] = beta;
      bad_s[y][i] = 0;
      __syncthreads();
      if (i >= 32 && line_s[31] == line_s[i]) G_s[y][i] += G_s[y][31];
    }
    __syncthreads();
    for (int y = 0; y < n_heads; ++y) {
      LdHead* out = c.heads + (size_t)block * a.Hv + hk * many + y0 + y;
      float* A = As + y * LD_C * LD_PITCH;
      float most[2] = {0.0f, 0.0f};
      bool good[2] = {true, true};
      float pv[8][4];
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = warp * 16 + g + (e >> 1) * 8, j = n * 8 + cc * 2 + (e & 1);
          float p = 0.0f, x = 0.0f;
          if (n <= 2 * warp + 1 && j <= i && line_s[i] == line_s[j] && line_s[i] >= 0) {
            const float ratio = expf((float)(G_s[y][i] - G_s[y][j])) * k_factor[j];
            p = ratio * q_factor[i] * qk[n][e];
            if (DELTA && j < i) x = ratio * k_factor[i] * beta_s[y][i] * kk[n][e];
          }
          if (!(fabsf(p) <= 3.4028234e38f)) good[e >> 1] = false, p = 0.0f;
          if (DELTA && !(fabsf(x) <= 3.4028234e38f)) bad_s[y][i] = 1, x = 0.0f;
          most[e >> 1] = fmaxf(most[e >> 1], fabsf(p));
          pv[n][e] = p;
          if (DELTA) A[j * LD_PITCH + i] = x;
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
        if (cc == 0) out->p_scale[i] = all_good ? down : __uint_as_float(0x7fc00000u);
#pragma unroll
        for (int n = 0; n < 8; ++n)
          *(uint32_t*)(out->p + ld_at<8>(i, n) + cc * 2) = ld_half2(pv[n][r * 2] * up, pv[n][r * 2 + 1] * up);
      }
      if (tid < LD_C) {
        const int i = tid;
        const float gamma = expf((float)G_s[y][i]);
        const bool live = line_s[i] >= 0;
        out->gamma[i] = gamma;
        out->q_in[i] = live ? gamma * q_factor[i] : 0.0f;
        out->r_in[i] = live ? gamma * k_factor[i] : 0.0f;
        out->k_out[i] = live ? expf((float)(G_s[y][last_s[i]] - G_s[y][i])) * k_factor[i] : 0.0f;
      }
    }
    if constexpr (DELTA) {
      __syncthreads();
      const int y = tid >> 6, j = tid & 63;
      float x[LD_C];
      float* A = As + y * LD_C * LD_PITCH;
      if (y < n_heads) {
#pragma unroll
        for (int i = 0; i < LD_C; ++i) x[i] = i == j ? 1.0f : 0.0f;
#pragma unroll
        for (int m = 0; m < LD_C - 1; ++m) {
#pragma unroll
          for (int i = (m + 1) & ~3; i < LD_C; i += 4) {
            const float4 v = *(const float4*)(A + m * LD_PITCH + i);
            if (i > m) x[i] = fmaf(-v.x, x[m], x[i]);
            if (i + 1 > m) x[i + 1] = fmaf(-v.y, x[m], x[i + 1]);
            if (i + 2 > m) x[i + 2] = fmaf(-v.z, x[m], x[i + 2]);
            if (i + 3 > m) x[i + 3] = fmaf(-v.w, x[m], x[i + 3]);
          }
        }
      }
      __syncthreads();
      if (y < n_heads) {  // rows of the inverse, entries of two lines as zeros
        const float beta = beta_s[y][j];
#pragma unroll
        for (int i = 0; i < LD_C; ++i) A[i * LD_PITCH + j] = line_s[i] == line_s[j] && i >= j ? x[i] * beta : 0.0f;
      }
      __syncthreads();
      // a row's 64 values by two threads, 32 each
      for (int y2 = 0; y2 < n_heads; ++y2) {
        LdHead* out = c.heads + (size_t)block * a.Hv + hk * many + y0 + y2;
        const int i = tid >> 1, half = tid & 1;
        float* row = As + y2 * LD_C * LD_PITCH + i * LD_PITCH + half * 32;
        float most = 0.0f;
        bool good = bad_s[y2][i] == 0;
        for (int e = 0; e < 32; ++e) {
          if (!(fabsf(row[e]) <= 3.4028234e38f)) good = false, row[e] = 0.0f;
          most = fmaxf(most, fabsf(row[e]));
        }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        good = __shfl_xor_sync(0xffffffffu, good, 1) && good;
        float up, down;
        ld_scale(most, up, down);
        if (half == 0) out->t_scale[i] = good ? down : __uint_as_float(0x7fc00000u);
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          uint4 hi, lo;
          const float4 v0 = *(const float4*)(row + p * 8), v1 = *(const float4*)(row + p * 8 + 4);
          ld_split(v0.x * up, v0.y * up, hi.x, lo.x), ld_split(v0.z * up, v0.w * up, hi.y, lo.y);
          ld_split(v1.x * up, v1.y * up, hi.z, lo.z), ld_split(v1.z * up, v1.w * up, hi.w, lo.w);
          *(uint4*)(out->t_hi + ld_at<8>(i, half * 4 + p)) = hi;
          *(uint4*)(out->t_lo + ld_at<8>(i, half * 4 + p)) = lo;
        }
      }
    }
  }
}

// ---- The scan. A CTA has 16 x WARPS rows of a head's state of one line and goes along the line's chunks; a warp has 16 rows
// by itself, S in its registers as the accumulator of S^T-shaped products [rows of S, tokens or columns of K]. An accumulator of
// mma.sync is laid out as the next product's A operand is, so S -> R -> U -> S needs no exchange between warps: K, Q, the
// inverse and P, as B operands, come from shared memory, where a producer warp keeps LdScanShape::STAGES chunks coming (bulk
// copies; the rows of v by TMA). (tcgen05 would want S as a 16-bit operand in shared or tensor memory and R and U brought
// there and back between the products: with 16 rows a warp the chain is shorter in registers.)
template <int DK, int WARPS, bool DELTA> struct LdScanShape {
  static constexpr int V = WARPS * LD_C * 32, STAGE = (int)(sizeof(LdRows<DK>) + sizeof(LdHead)) + V;
  static constexpr int STAGES = (227 * 1024 - 2048) / STAGE < 4 ? (227 * 1024 - 2048) / STAGE : 4;
  static constexpr int SMEM = STAGES * STAGE + 1024;
};

// Largest of the values of a row held by the four lanes of a group.
D3_DEV float ld_row_most(float m) {
  m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
  return fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
}

template <int TYPE, int DK, bool DELTA, int WARPS>
__global__ void __launch_bounds__((WARPS + 1) * 32, 1)
    lines_delta_scan_kernel(const __grid_constant__ CUtensorMap vmap, LdChunkArgs c) {
  using TT = QrType<TYPE>;
  using S_ = LdScanShape<DK, WARPS, DELTA>;
  constexpr int PIECES = DK / 8, NK = DK / 8, NT = LD_C / 8, STAGES = S_::STAGES;
  extern __shared__ uint8_t ld_raw[];
  __shared__ __align__(8) uint64_t full[STAGES], empty[STAGES];
  const LdArgs& a = c.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, cc = lane & 3;
  const int h = blockIdx.y, b = blockIdx.z;
  uint8_t* const ring = (uint8_t*)(((uintptr_t)ld_raw + 1023) & ~(uintptr_t)1023);
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], WARPS);
    fence_mbar_init();
  }
  __syncthreads();
  grid_dependency_wait();
  allow_dependents();
  const long long first_token = (long long)c.block0 * LD_C, end_token = min((long long)a.T, first_token + (long long)c.blocks * LD_C);
  const int row0 = (blockIdx.x * WARPS + warp) * 16;  // this warp's rows of the state
  if (b == a.B) {  // the places past the lines' last token
    const long long from = max((long long)min(max(a.cu[b], 0), a.T), first_token);
    if (warp < WARPS && row0 < a.Dv)
      for (long long t = from + (lane >> 1); t < end_token; t += 16)
        *(uint4*)((uint16_t*)a.out + (t * a.Hv + h) * a.Dv + row0 + (lane & 1) * 8) = make_uint4(0, 0, 0, 0);
    return;
  }
  const long long s = max((long long)min(max(a.cu[b], 0), a.T), first_token), e = min((long long)a.cu[b + 1], end_token);
  if (e <= s) return;
  const int block_a = (int)((s - first_token) / LD_C), chunks = (int)((e - 1 - first_token) / LD_C) - block_a + 1;
  if (warp == WARPS) {  // the producer
    if (lane == 0) {
      bool ok = true;
      int i = 0;
      for (; i < chunks && ok; ++i) {
        const int st = i % STAGES;
        if (i >= STAGES) ok = mbar_wait(&empty[st], (i / STAGES - 1) & 1);
        if (!ok) break;
        uint8_t* to = ring + st * S_::STAGE;
        const size_t block = block_a + i;
        const int v_boxes = min(WARPS, (a.Dv - (int)blockIdx.x * WARPS * 16) / 16);
        const uint32_t head_bytes = DELTA ? sizeof(LdHead) : sizeof(LdHead) - offsetof(LdHead, p);
        mbar_arrive_expect_tx(&full[st], (uint32_t)sizeof(LdRows<DK>) + head_bytes + v_boxes * LD_C * 32);
        const uint64_t keep = policy_evict_last();
        bulk_g2s(to, (const LdRows<DK>*)c.rows + block * a.Hk + h / (a.Hv / a.Hk), sizeof(LdRows<DK>), &full[st], keep);
        const uint8_t* head = (const uint8_t*)(c.heads + block * a.Hv + h);
        bulk_g2s(to + sizeof(LdRows<DK>) + sizeof(LdHead) - head_bytes, head + sizeof(LdHead) - head_bytes, head_bytes, &full[st], keep);
        for (int w = 0; w < v_boxes; ++w)
          tma_load_3d(smem_u32(to + sizeof(LdRows<DK>) + sizeof(LdHead) + w * LD_C * 32), &vmap,
                      (blockIdx.x * WARPS + w) * 16, h, (int)(first_token + (long long)block * LD_C), &full[st]);
      }
      if (!ok)  // the copies in flight land before the block ends
        for (int st = 0; st < STAGES && st < i; ++st) mbar_wait(&full[st], ((i - 1 - st) / STAGES) & 1);
    }
    return;
  }
  float* const state = a.state + (((size_t)b * a.Hv + h) * a.Dv + row0) * DK;
  const bool there = row0 < a.Dv;
  float S[NK][4] = {};
  if (there)
#pragma unroll
    for (int n = 0; n < NK; ++n) {
      const float2 x = *(const float2*)(state + g * DK + n * 8 + cc * 2), y = *(const float2*)(state + (g + 8) * DK + n * 8 + cc * 2);
      S[n][0] = x.x, S[n][1] = x.y, S[n][2] = y.x, S[n][3] = y.y;
    }
  bool ok = true;
#pragma unroll 1
  for (int i = 0; i < chunks; ++i) {
    const int st = i % STAGES;
    ok = mbar_wait(&full[st], (i / STAGES) & 1);
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) break;
    const uint8_t* stage = ring + st * S_::STAGE;
    const LdRows<DK>& rows = *(const LdRows<DK>*)stage;
    const LdHead& head = *(const LdHead*)(stage + sizeof(LdRows<DK>));
    uint8_t* v_s = ring + st * S_::STAGE + sizeof(LdRows<DK>) + sizeof(LdHead) + warp * LD_C * 32;  // and, later, its outputs
    const long long t0 = first_token + (long long)(block_a + i) * LD_C;
    const int lo = (int)max(0ll, s - t0), hi = (int)min((long long)LD_C, e - t0);
    const bool partial = lo > 0 || hi < LD_C;
    float up[2], down[2], m_s[2] = {0.0f, 0.0f};
    {
      float (&m)[2] = m_s;
#pragma unroll
      for (int n = 0; n < NK; ++n) {
        m[0] = fmaxf(m[0], fmaxf(fabsf(S[n][0]), fabsf(S[n][1])));
        m[1] = fmaxf(m[1], fmaxf(fabsf(S[n][2]), fabsf(S[n][3])));
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        m[r] = ld_row_most(m[r]);
        ld_scale(m[r], up[r], down[r]);
      }
    }
    // S K^T and S Q^T
    float R[NT][4] = {}, O[NT][4] = {};
#pragma unroll
    for (int kt = 0; kt < DK / 16; ++kt) {
      uint32_t hi4[4], lo4[4];
      ld_split(S[2 * kt][0] * up[0], S[2 * kt][1] * up[0], hi4[0], lo4[0]);
      ld_split(S[2 * kt][2] * up[1], S[2 * kt][3] * up[1], hi4[1], lo4[1]);
      ld_split(S[2 * kt + 1][0] * up[0], S[2 * kt + 1][1] * up[0], hi4[2], lo4[2]);
      ld_split(S[2 * kt + 1][2] * up[1], S[2 * kt + 1][3] * up[1], hi4[3], lo4[3]);
#pragma unroll
      for (int n = 0; n < NT; n += 2) {
        uint32_t bk[4];
        const int at = ld_at<PIECES>(n * 8 + (lane & 7) + (lane >> 4) * 8, kt * 2 + ((lane >> 3) & 1));
        if (DELTA) {
          ld_matrix4(bk, rows.k + at);
          ld_mma(R[n], lo4, bk[0], bk[1]), ld_mma(R[n + 1], lo4, bk[2], bk[3]);
          ld_mma(R[n], hi4, bk[0], bk[1]), ld_mma(R[n + 1], hi4, bk[2], bk[3]);
        }
        ld_matrix4(bk, rows.q + at);
        ld_mma(O[n], hi4, bk[0], bk[1]), ld_mma(O[n + 1], hi4, bk[2], bk[3]);
      }
    }
    // R = V - gamma K S^T (without the delta rule V is U), zeros for the tokens of other lines
#pragma unroll
    for (int n = 0; n < NT; n += 2) {
      uint32_t v4[4];
      const int token = n * 8 + (lane & 7) + (lane >> 4) * 8, piece = ((lane >> 3) & 1) ^ ((token >> 2) & 1);
      ld_matrix4_trans(v4, v_s + token * 32 + piece * 16);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float v[4];
        TT::get2(v4[2 * x], v[0], v[1]);
        TT::get2(v4[2 * x + 1], v[2], v[3]);
        const int j = (n + x) * 8 + cc * 2;
        if (DELTA) {
          const float2 f = *(const float2*)(head.r_in + j);
          v[0] = fmaf(-R[n + x][0] * down[0], f.x, v[0]), v[1] = fmaf(-R[n + x][1] * down[0], f.y, v[1]);
          v[2] = fmaf(-R[n + x][2] * down[1], f.x, v[2]), v[3] = fmaf(-R[n + x][3] * down[1], f.y, v[3]);
        }
        if (partial) {
          if (j < lo || j >= hi) v[0] = v[2] = 0.0f;
          if (j + 1 < lo || j + 1 >= hi) v[1] = v[3] = 0.0f;
        }
#pragma unroll
        for (int y = 0; y < 4; ++y) R[n + x][y] = v[y];
      }
    }
    float U[NT][4];
    if (DELTA) {  // U = inverse R
      float m[2] = {0.0f, 0.0f}, ru[2], rd[2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        m[0] = fmaxf(m[0], fmaxf(fabsf(R[n][0]), fabsf(R[n][1])));
        m[1] = fmaxf(m[1], fmaxf(fabsf(R[n][2]), fabsf(R[n][3])));
      }
      ld_scale(ld_row_most(m[0]), ru[0], rd[0]);
      ld_scale(ld_row_most(m[1]), ru[1], rd[1]);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int y = 0; y < 4; ++y) U[n][y] = 0.0f;
#pragma unroll
      for (int kt = 0; kt < LD_C / 16; ++kt) {
        uint32_t hi4[4], lo4[4];
        ld_split(R[2 * kt][0] * ru[0], R[2 * kt][1] * ru[0], hi4[0], lo4[0]);
        ld_split(R[2 * kt][2] * ru[1], R[2 * kt][3] * ru[1], hi4[1], lo4[1]);
        ld_split(R[2 * kt + 1][0] * ru[0], R[2 * kt + 1][1] * ru[0], hi4[2], lo4[2]);
        ld_split(R[2 * kt + 1][2] * ru[1], R[2 * kt + 1][3] * ru[1], hi4[3], lo4[3]);
#pragma unroll
        for (int n = 2 * kt; n < NT; n += 2) {
          uint32_t t4[4];
          const int at = ld_at<8>(n * 8 + (lane & 7) + (lane >> 4) * 8, kt * 2 + ((lane >> 3) & 1));
          ld_matrix4(t4, head.t_lo + at);
          ld_mma(U[n], hi4, t4[0], t4[1]), ld_mma(U[n + 1], hi4, t4[2], t4[3]);
          ld_matrix4(t4, head.t_hi + at);
          ld_mma(U[n], lo4, t4[0], t4[1]), ld_mma(U[n + 1], lo4, t4[2], t4[3]);
          ld_mma(U[n], hi4, t4[0], t4[1]), ld_mma(U[n + 1], hi4, t4[2], t4[3]);
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int j = n * 8 + cc * 2;
        const float2 f = *(const float2*)(head.t_scale + j);
        U[n][0] *= f.x * rd[0], U[n][1] *= f.y * rd[0], U[n][2] *= f.x * rd[1], U[n][3] *= f.y * rd[1];
        if (partial) {
          if (j < lo || j >= hi) U[n][0] = U[n][2] = 0.0f;
          if (j + 1 < lo || j + 1 >= hi) U[n][1] = U[n][3] = 0.0f;
        }
      }
    } else {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int y = 0; y < 4; ++y) U[n][y] = R[n][y];
    }
    // O = gamma Q S^T + P U
    {
      float m[2] = {0.0f, 0.0f}, uu[2], ud[2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        m[0] = fmaxf(m[0], fmaxf(fabsf(U[n][0]), fabsf(U[n][1])));
        m[1] = fmaxf(m[1], fmaxf(fabsf(U[n][2]), fabsf(U[n][3])));
      }
      ld_scale(ld_row_most(m[0]), uu[0], ud[0]);
      ld_scale(ld_row_most(m[1]), uu[1], ud[1]);
      uint32_t u4[LD_C / 16][4];
#pragma unroll
      for (int kt = 0; kt < LD_C / 16; ++kt) {
        u4[kt][0] = ld_half2(U[2 * kt][0] * uu[0], U[2 * kt][1] * uu[0]);
        u4[kt][1] = ld_half2(U[2 * kt][2] * uu[1], U[2 * kt][3] * uu[1]);
        u4[kt][2] = ld_half2(U[2 * kt + 1][0] * uu[0], U[2 * kt + 1][1] * uu[0]);
        u4[kt][3] = ld_half2(U[2 * kt + 1][2] * uu[1], U[2 * kt + 1][3] * uu[1]);
      }
      __syncwarp();  // v has been read by all lanes
#pragma unroll
      for (int n = 0; n < NT; n += 2) {
        float pu[2][4] = {};
#pragma unroll
        for (int kt = 0; kt <= n / 2; ++kt) {
          uint32_t p4[4];
          ld_matrix4(p4, head.p + ld_at<8>(n * 8 + (lane & 7) + (lane >> 4) * 8, kt * 2 + ((lane >> 3) & 1)));
          ld_mma(pu[0], u4[kt], p4[0], p4[1]), ld_mma(pu[1], u4[kt], p4[2], p4[3]);
        }
        uint32_t o4[4];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int j = (n + x) * 8 + cc * 2;
          const float2 fq = *(const float2*)(head.q_in + j), fp = *(const float2*)(head.p_scale + j);
          float o[4];
          o[0] = fmaf(O[n + x][0] * down[0], fq.x, pu[x][0] * ud[0] * fp.x), o[1] = fmaf(O[n + x][1] * down[0], fq.y, pu[x][1] * ud[0] * fp.y);
          o[2] = fmaf(O[n + x][2] * down[1], fq.x, pu[x][2] * ud[1] * fp.x), o[3] = fmaf(O[n + x][3] * down[1], fq.y, pu[x][3] * ud[1] * fp.y);
          o4[2 * x] = TT::put2(o[0], o[1]), o4[2 * x + 1] = TT::put2(o[2], o[3]);
        }
        const int token = n * 8 + (lane & 7) + (lane >> 4) * 8, piece = ((lane >> 3) & 1) ^ ((token >> 2) & 1);
        st_matrix4_trans(v_s + token * 32 + piece * 16, o4[0], o4[1], o4[2], o4[3]);
      }
      __syncwarp();
      if (there)
#pragma unroll
        for (int x = 0; x < LD_C / 16; ++x) {
          const int token = x * 16 + (lane >> 1), piece = (lane & 1) ^ ((token >> 2) & 1);
          if (token >= lo && token < hi)
            *(uint4*)((uint16_t*)a.out + ((t0 + token) * a.Hv + h) * a.Dv + row0 + (lane & 1) * 8) =
                *(const uint4*)(v_s + token * 32 + piece * 16);
        }
    }
    // S = gamma_last S + (k_out U)^T K, the sum in the scale of U's row
    {
      float m[2] = {0.0f, 0.0f}, wu[2], wd[2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int j = n * 8 + cc * 2;
        float2 f = *(const float2*)(head.k_out + j);
        if (partial) {
          if (j < lo || j >= hi) f.x = 0.0f;
          if (j + 1 < lo || j + 1 >= hi) f.y = 0.0f;
        }
        U[n][0] *= f.x, U[n][1] *= f.y, U[n][2] *= f.x, U[n][3] *= f.y;
        m[0] = fmaxf(m[0], fmaxf(fabsf(U[n][0]), fabsf(U[n][1])));
        m[1] = fmaxf(m[1], fmaxf(fabsf(U[n][2]), fabsf(U[n][3])));
      }
      const float gamma = head.gamma[hi - 1];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        // no less than 2^-40 of the state's size: what is smaller does not change it, and the state stays within 32 bits
        ld_scale(fmaxf(ld_row_most(m[r]), m_s[r] * 0x1p-40f), wu[r], wd[r]);
      }
#pragma unroll
      for (int n = 0; n < NK; ++n) {
        S[n][0] *= gamma * wu[0], S[n][1] *= gamma * wu[0], S[n][2] *= gamma * wu[1], S[n][3] *= gamma * wu[1];
      }
#pragma unroll
      for (int kt = 0; kt < LD_C / 16; ++kt) {
        uint32_t hi4[4], lo4[4];
        ld_split(U[2 * kt][0] * wu[0], U[2 * kt][1] * wu[0], hi4[0], lo4[0]);
        ld_split(U[2 * kt][2] * wu[1], U[2 * kt][3] * wu[1], hi4[1], lo4[1]);
        ld_split(U[2 * kt + 1][0] * wu[0], U[2 * kt + 1][1] * wu[0], hi4[2], lo4[2]);
        ld_split(U[2 * kt + 1][2] * wu[1], U[2 * kt + 1][3] * wu[1], hi4[3], lo4[3]);
#pragma unroll
        for (int n = 0; n < NK; n += 2) {
          uint32_t b4[4];
          ld_matrix4_trans(b4, rows.k + ld_at<PIECES>(kt * 16 + (lane & 15), n + (lane >> 4)));
          ld_mma(S[n], lo4, b4[0], b4[1]), ld_mma(S[n + 1], lo4, b4[2], b4[3]);
          ld_mma(S[n], hi4, b4[0], b4[1]), ld_mma(S[n + 1], hi4, b4[2], b4[3]);
        }
      }
#pragma unroll
      for (int n = 0; n < NK; ++n) S[n][0] *= wd[0], S[n][1] *= wd[0], S[n][2] *= wd[1], S[n][3] *= wd[1];
    }
    fence_async_smem();  // the outputs' place is the next TMA load's
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[st]);
  }
  if (there && ok)
#pragma unroll
    for (int n = 0; n < NK; ++n) {
      *(float2*)(state + g * DK + n * 8 + cc * 2) = make_float2(S[n][0], S[n][1]);
      *(float2*)(state + (g + 8) * DK + n * 8 + cc * 2) = make_float2(S[n][2], S[n][3]);
    }
}

}  // namespace d3
