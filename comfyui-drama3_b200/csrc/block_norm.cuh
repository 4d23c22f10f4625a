// The norms of a decoder block's rows with what stands next to them, one pass each.
//   gated:  out = x * rsqrt(mean(x^2) + eps) * w * act(gate)        per (token, head), x [D]; act: SiLU or the sigmoid
//   join:   b = x, or x * rsqrt(mean(x^2) + eps) * w_post           the norm after the block, where it has one
//           r = residual + scale * gate * b                         gate: one value a row, one a channel, one each, or none
//           normed = r * rsqrt(mean(r^2) + eps) * w                 the norm before the next block, of r before it is rounded
// All in 32 bits, rounded once when stored.
//
// Bound by memory: each row is read once and written once, in 16-byte vectors that stay in registers between the sum of
// squares and the product. Gated rows are short (a head): a group of lanes each, four rows of a group at a time so that enough
// loads are in flight (two 35.6, eight 43.9 us in the case below), and no block-wide step. Joined rows are long: a warp each where
// they are many (a row's loads are in flight together), a block each, whose threads hold one or two vectors, where they are few.
// Measured (B200, bf16): gated, 8192 tokens of 32 heads of 128 34 us, 5.9 TB/s; joined, 16384 rows of 2048 with a norm after the block
// and a gate a row 52 us, 5.2 TB/s (a block a row: 73), without them 43 where the calls follow one another; 16 tokens 1.6 and 1.9 us, latency.
// fp32 63 and 92 us. Rows that are no whole vectors are read in single values, twice and three times: heads of 129 107 us, 1001 columns 69 to 104.
#pragma once

#include "rows.cuh"

namespace d3 {

constexpr int BN_WARPS = 4;        // a block of the gated rows
constexpr int BN_MAX_THREADS = 1024;

struct GnArgs {
  QrTensor x, gate;  // rows [T, H, D]
  int T, H, D;
  const void* w;
  int w_f32;
  float w_add, eps;
  int act;    // 0 SiLU, 1 sigmoid
  void* out;  // [T, H, D]
};

// LANES lanes a row, NV vectors a lane, AHEAD rows of each group of lanes at a time.
template <int TYPE, int LANES, int NV, int AHEAD>
__global__ void __launch_bounds__(BN_WARPS * 32) gated_norm_kernel(GnArgs a) {
  using E = typename QrType<TYPE>::T;
  constexpr int VEC = 16 / (int)sizeof(E), GROUPS = 32 / LANES;
  const int lane = threadIdx.x & 31, l = lane % LANES, vectors = a.D / VEC;
  const unsigned rows = (unsigned)a.T * (unsigned)a.H;  // at most 2^31
  const unsigned row0 = (blockIdx.x * BN_WARPS + (threadIdx.x >> 5)) * (GROUPS * AHEAD) + lane / LANES;
  grid_dependency_wait();
  allow_dependents();
  uint4 x[AHEAD][NV] = {}, z[AHEAD][NV] = {};
#pragma unroll
  for (int r = 0; r < AHEAD; ++r) {
    const unsigned row = row0 + r * GROUPS;
    if (row < rows) {
      const unsigned t = row / (unsigned)a.H, h = row - t * (unsigned)a.H;
      const E* xr = (const E*)a.x.p + t * a.x.token + h * a.x.head;
      const E* zr = (const E*)a.gate.p + t * a.gate.token + h * a.gate.head;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (l + i * LANES < vectors) {
          x[r][i] = *(const uint4*)(xr + (l + i * LANES) * VEC);
          z[r][i] = *(const uint4*)(zr + (l + i * LANES) * VEC);
        }
    }
  }
  float w[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (l + i * LANES < vectors) qr_weights<TYPE, VEC>(a.w, a.w_f32, a.w_add, (l + i * LANES) * VEC, w[i]);
#pragma unroll
  for (int r = 0; r < AHEAD; ++r) {
    const unsigned row = row0 + r * GROUPS;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float v[VEC];
      qr_unpack<TYPE, VEC>(&x[r][i].x, v);
#pragma unroll
      for (int e = 0; e < VEC; ++e) sum = fmaf(v[e], v[e], sum);
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float scale = rsqrtf(sum / a.D + a.eps);
    if (row >= rows) continue;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (l + i * LANES < vectors) {
        float v[VEC], g[VEC];
        qr_unpack<TYPE, VEC>(&x[r][i].x, v);
        qr_unpack<TYPE, VEC>(&z[r][i].x, g);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float s = row_sigmoid<TYPE>(g[e]);
          v[e] = v[e] * scale * w[i][e] * (a.act ? s : g[e] * s);
        }
        uint4 out;
        qr_pack<TYPE, VEC>(v, &out.x);
        *(uint4*)((E*)a.out + (size_t)row * a.D + (l + i * LANES) * VEC) = out;
      }
  }
}

// Rows of any size and alignment: a warp each, read twice.
template <int TYPE>
__global__ void __launch_bounds__(BN_WARPS * 32) gated_norm_any_kernel(GnArgs a) {
  using TT = QrType<TYPE>;
  using E = typename TT::T;
  const int lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * BN_WARPS + (threadIdx.x >> 5);
  grid_dependency_wait();
  allow_dependents();
  if (row >= (long long)a.T * a.H) return;
  const long long t = row / a.H;
  const int h = (int)(row - t * a.H);
  const E* xr = (const E*)a.x.p + t * a.x.token + h * a.x.head;
  const E* zr = (const E*)a.gate.p + t * a.gate.token + h * a.gate.head;
  float sum = 0.0f;
  for (int d = lane; d < a.D; d += 32) {
    const float v = TT::get(xr[d]);
    sum = fmaf(v, v, sum);
  }
  const float scale = rsqrtf(warp_sum(sum) / a.D + a.eps);
  for (int d = lane; d < a.D; d += 32) {
    const float g = TT::get(zr[d]), s = row_sigmoid<TYPE>(g);
    ((E*)a.out)[row * a.D + d] =
        TT::put(TT::get(xr[d]) * scale * qr_weight<TYPE>(a.w, a.w_f32, a.w_add, d) * (a.act ? s : g * s));
  }
}

enum { AN_NONE = 0, AN_ROW = 1, AN_EACH = 2 };  // the gate: none, one value a row, one for each (or each channel: token stride 0)

struct AnArgs {
  const void* x;
  const void* residual;
  long long x_token, r_token;  // strides in elements
  int T, W;
  const void* w;
  const void* post;  // may be null: no norm after the block
  int w_f32;
  float w_add, eps, scale;
  const void* gate;
  long long gate_token;
  int gate_kind;
  void* sum_out;   // [T, W]
  void* norm_out;  // [T, W]
};

// The sum of v over the block's threads, in every one of them. `part`: a float for each warp, another one each time.
D3_DEV float bn_block_sum(float v, float* part) {
  const int warps = blockDim.x >> 5;
  v = warp_sum(v);
  if (warps == 1) return v;
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = (threadIdx.x & 31) < warps ? part[threadIdx.x & 31] : 0.0f;
  return warp_sum(v);
}

// What a thread does with its vectors of one row: NV of them, `step` apart from the first one on. SUM(v) adds v up over the row's threads.
template <int TYPE, int NV, class SUM>
D3_DEV void an_row(const AnArgs& a, long long t, int first, int step, SUM&& row_sum) {
  using TT = QrType<TYPE>;
  using E = typename TT::T;
  constexpr int VEC = 16 / (int)sizeof(E);
  const int vectors = a.W / VEC;
  uint4 x[NV] = {}, r[NV] = {};
  float row_gate = 1.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = first + i * step;
    if (v < vectors) {
      x[i] = *(const uint4*)((const E*)a.x + t * a.x_token + v * VEC);
      r[i] = *(const uint4*)((const E*)a.residual + t * a.r_token + v * VEC);
    }
  }
  if (a.gate_kind == AN_ROW) row_gate = TT::get(((const E*)a.gate)[t * a.gate_token]);
  float factor = a.scale * row_gate;
  if (a.post) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float v[VEC];
      qr_unpack<TYPE, VEC>(&x[i].x, v);
#pragma unroll
      for (int e = 0; e < VEC; ++e) sum = fmaf(v[e], v[e], sum);
    }
    factor *= rsqrtf(row_sum(sum) / a.W + a.eps);
  }
  float sum = 0.0f;
  float total[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = first + i * step;
    if (v < vectors) {
      float b[VEC], m[VEC];
      qr_unpack<TYPE, VEC>(&x[i].x, b);
      qr_unpack<TYPE, VEC>(&r[i].x, total[i]);
      if (a.post) {
        qr_weights<TYPE, VEC>(a.post, a.w_f32, a.w_add, v * VEC, m);
#pragma unroll
        for (int e = 0; e < VEC; ++e) b[e] *= m[e];
      }
      if (a.gate_kind == AN_EACH) {
        const uint4 g = *(const uint4*)((const E*)a.gate + t * a.gate_token + v * VEC);
        qr_unpack<TYPE, VEC>(&g.x, m);
#pragma unroll
        for (int e = 0; e < VEC; ++e) b[e] *= m[e];
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        total[i][e] = fmaf(factor, b[e], total[i][e]);
        sum = fmaf(total[i][e], total[i][e], sum);
      }
      uint4 out;
      qr_pack<TYPE, VEC>(total[i], &out.x);
      *(uint4*)((E*)a.sum_out + t * a.W + v * VEC) = out;
    }
  }
  const float scale = rsqrtf(row_sum(sum) / a.W + a.eps);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = first + i * step;
    if (v < vectors) {
      float w[VEC];
      qr_weights<TYPE, VEC>(a.w, a.w_f32, a.w_add, v * VEC, w);
#pragma unroll
      for (int e = 0; e < VEC; ++e) w[e] *= total[i][e] * scale;
      uint4 out;
      qr_pack<TYPE, VEC>(w, &out.x);
      *(uint4*)((E*)a.norm_out + t * a.W + v * VEC) = out;
    }
  }
}

// A block a row.
template <int TYPE, int NV>
__global__ void __launch_bounds__(BN_MAX_THREADS) add_norm_kernel(AnArgs a) {
  __shared__ float part[2][32];
  int which = 0;
  grid_dependency_wait();
  allow_dependents();
  an_row<TYPE, NV>(a, blockIdx.x, threadIdx.x, blockDim.x, [&](float v) { return bn_block_sum(v, part[which++]); });
}

// A warp a row: no step of the block, and a row's loads are all in flight together.
template <int TYPE, int NV>
__global__ void __launch_bounds__(BN_WARPS * 32) add_norm_warp_kernel(AnArgs a) {
  const long long t = (long long)blockIdx.x * BN_WARPS + (threadIdx.x >> 5);
  grid_dependency_wait();
  allow_dependents();
  if (t < a.T) an_row<TYPE, NV>(a, t, threadIdx.x & 31, 32, [](float v) { return warp_sum(v); });
}

// Rows of any size and alignment: a block each; x and the residual are read again for each sum, from the caches.
template <int TYPE>
__global__ void __launch_bounds__(256) add_norm_any_kernel(AnArgs a) {
  using TT = QrType<TYPE>;
  using E = typename TT::T;
  __shared__ float part[2][32];
  const long long t = blockIdx.x;
  grid_dependency_wait();
  allow_dependents();
  const E* x = (const E*)a.x + t * a.x_token;
  const E* r = (const E*)a.residual + t * a.r_token;
  const E* g = (const E*)a.gate + t * a.gate_token;
  float factor = a.scale;
  if (a.gate_kind == AN_ROW) factor *= TT::get(g[0]);
  if (a.post) {
    float sum = 0.0f;
    for (int d = threadIdx.x; d < a.W; d += blockDim.x) {
      const float v = TT::get(x[d]);
      sum = fmaf(v, v, sum);
    }
    factor *= rsqrtf(bn_block_sum(sum, part[0]) / a.W + a.eps);
  }
  auto total = [&](int d) {
    float b = TT::get(x[d]);
    if (a.post) b *= qr_weight<TYPE>(a.post, a.w_f32, a.w_add, d);
    if (a.gate_kind == AN_EACH) b *= TT::get(g[d]);
    return fmaf(factor, b, TT::get(r[d]));
  };
  float sum = 0.0f;
  for (int d = threadIdx.x; d < a.W; d += blockDim.x) {
    const float v = total(d);
    sum = fmaf(v, v, sum);
  }
  const float scale = rsqrtf(bn_block_sum(sum, part[1]) / a.W + a.eps);
  for (int d = threadIdx.x; d < a.W; d += blockDim.x) {
    const float v = total(d);
    ((E*)a.sum_out)[t * a.W + d] = TT::put(v);
    ((E*)a.norm_out)[t * a.W + d] = TT::put(v * scale * qr_weight<TYPE>(a.w, a.w_f32, a.w_add, d));
  }
}

}  // namespace d3
