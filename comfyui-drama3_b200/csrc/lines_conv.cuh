// The short causal convolution in front of linear attention, over each line's own tokens:
//   y_t[c] = bias[c] + sum_j w[c][j] x_{t - (W - 1) + j}[c],  out = y * sigmoid(y) (or y)      W taps, one filter a channel
// Inputs before the line's first new token are its state [W - 1, C], which becomes the line's last W - 1 inputs. Sums in
// 32 bits, rounded once.
//
// Bound by memory: x is read once and out written once (each tile of tokens reads W - 1 rows of the one before it too). A
// thread has a 16-byte vector of channels and goes along the tokens, the last W - 1 inputs and the weights in registers, a
// few loads ahead. The packed tokens are cut into tiles whatever lines they belong to; a line's first W - 1 tokens, which
// read its state, and the state's change are one block's (for each block of channels), so nothing reads a state that
// another block writes: a decode step has only such blocks' work.
// Measured (B200, bf16, 8192 channels, 4 taps): 8192 tokens 55 us, 4.9 TB/s (tiles of 32 tokens 59, of 128 61), 2000 tokens 21, 64 to 500
// 17, a tile's latency; 16 lines of a token 2.3 us, latency. fp32 8192 tokens 104. Five to eight taps and channels that are no whole vectors take
// a thread a channel: 8 taps 570 us, 777 channels 80.
#pragma once

#include "f32x2.cuh"
#include "rows.cuh"

namespace d3 {

constexpr int LC_THREADS = 128;
constexpr int LC_TILE = 64;  // tokens
constexpr int LC_AHEAD = 4;  // of them loaded together, while as many before them are summed
constexpr int LC_MAX_TAPS = 8;

struct LcArgs {
  const void* x;
  long long x_token;  // stride in elements
  int T, C, W, B;
  const void* w;     // [C, W]
  const void* bias;  // [C] or null
  int w_f32;
  void* state;  // [B, W - 1, C]
  const int* cu;
  const int* line;
  int silu;
  void* out;  // [T, C]
  int tiles;  // blocks of tokens; the lines' blocks come behind them
};

// What a tile does with token t: compute it (2), zeros (1, no line's token), or nothing (0, one of a line's first W - 1).
D3_DEV int lc_role(const LcArgs& a, long long t) {
  if (t >= a.T) return 0;
  const int b = a.line[t];
  if (b < 0 || b >= a.B) return 1;
  return t - a.cu[b] >= a.W - 1 ? 2 : 0;
}

// The tokens [s, s + n) of line b, within the pass.
D3_DEV void lc_line(const LcArgs& a, int b, long long& s, long long& n) {
  s = min(max(a.cu[b], 0), a.T);
  n = min(max((long long)a.cu[b + 1], s), (long long)a.T) - s;
}

template <int TYPE, int W>
__global__ void __launch_bounds__(LC_THREADS) lines_conv_kernel(LcArgs a) {
  using TT = QrType<TYPE>;
  using E = typename TT::T;
  constexpr int VEC = 16 / (int)sizeof(E);
  __shared__ int roles[LC_TILE];
  const int c = (blockIdx.y * LC_THREADS + threadIdx.x) * VEC;
  const bool there = c < a.C;
  const E* x = (const E*)a.x + c;
  E* out = (E*)a.out + c;
  float w[W][VEC], bias[VEC];
  auto weights = [&] {  // the filters of neighbouring channels lie next to one another
    float all[W * VEC];
#pragma unroll
    for (int i = 0; i < W; ++i) qr_weights<TYPE, VEC>(a.w, a.w_f32, 0.0f, c * W + i * VEC, all + i * VEC);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
#pragma unroll
      for (int j = 0; j < W; ++j) w[j][e] = all[e * W + j];
      bias[e] = a.bias ? qr_weight<TYPE>(a.bias, a.w_f32, 0.0f, c + e) : 0.0f;
    }
  };
  auto finish = [&](const float (&y)[VEC], long long t) {
    float v[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = a.silu ? y[e] * row_sigmoid<TYPE>(y[e]) : y[e];
    uint4 q;
    qr_pack<TYPE, VEC>(v, &q.x);
    *(uint4*)(out + t * a.C) = q;
  };
  auto row = [&](long long t) { return *(const uint4*)(x + t * a.x_token); };
  grid_dependency_wait();
  allow_dependents();
  if ((int)blockIdx.x >= a.tiles) {  // a line: its first tokens and its state
    long long s, n;
    const int b = blockIdx.x - a.tiles;
    lc_line(a, b, s, n);
    if (n == 0 || !there) return;
    E* state = (E*)a.state + (size_t)b * (W - 1) * a.C + c;
    uint4 in[2 * (W - 1)] = {}, last[W - 1];
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
      in[j] = *(const uint4*)(state + (size_t)j * a.C);
      if (j < n) in[W - 1 + j] = row(s + j);
    }
#pragma unroll
    for (int j = 0; j < W - 1; ++j)
      if (n - (W - 1) + j >= 0) last[j] = row(s + n - (W - 1) + j);
    weights();
#pragma unroll
    for (int i = 0; i < W - 1; ++i)
      if (i < n) {
        float y[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) y[e] = bias[e];
#pragma unroll
        for (int j = 0; j < W; ++j) {
          float v[VEC];
          qr_unpack<TYPE, VEC>(&in[i + j].x, v);
#pragma unroll
          for (int e = 0; e < VEC; ++e) y[e] = fmaf(w[j][e], v[e], y[e]);
        }
        finish(y, s + i);
      }
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
      uint4 v = last[j];
#pragma unroll
      for (int k = 1; k < W - 1; ++k)  // fewer new inputs than the state holds: the old ones move up
        if (j + k < W - 1 && n == k) v = in[j + k];
      *(uint4*)(state + (size_t)j * a.C) = v;
    }
    return;
  }
  const long long t0 = (long long)blockIdx.x * LC_TILE;
  if (threadIdx.x < LC_TILE) roles[threadIdx.x] = lc_role(a, t0 + threadIdx.x);
  const bool plain = __syncthreads_and(threadIdx.x >= LC_TILE || roles[threadIdx.x] == 2);  // nearly always, of a long text
  if (!__syncthreads_or(threadIdx.x < LC_TILE && roles[threadIdx.x]) || !there) return;
  weights();
  float in[W][VEC];  // in[(i + j) % W]: the input j of token i
#pragma unroll
  for (int j = 0; j < W - 1; ++j) {
    const long long t = t0 - (W - 1) + j;
    uint4 q = make_uint4(0, 0, 0, 0);
    if (t >= 0) q = row(t);
    qr_unpack<TYPE, VEC>(&q.x, in[j]);
  }
  uint4 next[LC_AHEAD];
  auto fetch = [&](int i0) {
#pragma unroll
    for (int i = 0; i < LC_AHEAD; ++i) {
      next[i] = make_uint4(0, 0, 0, 0);
      if (i0 + i < LC_TILE && t0 + i0 + i < a.T) next[i] = row(t0 + i0 + i);
    }
  };
  fetch(0);
#pragma unroll 1
  for (int i0 = 0; i0 < LC_TILE; i0 += LC_AHEAD) {
    uint4 q[LC_AHEAD];
#pragma unroll
    for (int i = 0; i < LC_AHEAD; ++i) q[i] = next[i];
    fetch(i0 + LC_AHEAD);
#pragma unroll
    for (int i = 0; i < LC_AHEAD; ++i) {
      float y[VEC];
      qr_unpack<TYPE, VEC>(&q[i].x, in[W - 1]);
#pragma unroll
      for (int e = 0; e < VEC; e += 2) {
        uint64_t two = f2_make(bias[e], bias[e + 1]);
#pragma unroll
        for (int j = 0; j < W; ++j) two = f2_fma(f2_make(w[j][e], w[j][e + 1]), f2_make(in[j][e], in[j][e + 1]), two);
        f2_split(two, y[e], y[e + 1]);
#pragma unroll
        for (int j = 0; j < W - 1; ++j) in[j][e] = in[j + 1][e], in[j][e + 1] = in[j + 1][e + 1];
      }
      const int role = plain ? 2 : roles[i0 + i];
      if (role == 2) finish(y, t0 + i0 + i);
      if (role == 1) *(uint4*)(out + (t0 + i0 + i) * a.C) = make_uint4(0, 0, 0, 0);
    }
  }
}

// Channels, strides and addresses of any kind, any number of taps: a thread has a channel.
template <int TYPE>
__global__ void __launch_bounds__(LC_THREADS) lines_conv_any_kernel(LcArgs a) {
  using TT = QrType<TYPE>;
  using E = typename TT::T;
  const int c = blockIdx.y * LC_THREADS + threadIdx.x, W = a.W;
  grid_dependency_wait();
  allow_dependents();
  if (c >= a.C) return;
  const E* x = (const E*)a.x + c;
  E* out = (E*)a.out + c;
  float w[LC_MAX_TAPS], in[LC_MAX_TAPS];
#pragma unroll
  for (int j = 0; j < LC_MAX_TAPS; ++j) {
    w[j] = j < W ? qr_weight<TYPE>(a.w, a.w_f32, 0.0f, c * W + j) : 0.0f;
    in[j] = 0.0f;
  }
  const float bias = a.bias ? qr_weight<TYPE>(a.bias, a.w_f32, 0.0f, c) : 0.0f;
  // in[k]: the input k tokens ago
  auto push = [&](float v) {
#pragma unroll
    for (int j = LC_MAX_TAPS - 1; j > 0; --j) in[j] = in[j - 1];
    in[0] = v;
  };
  auto put = [&](long long t) {
    float y = bias;
#pragma unroll
    for (int j = LC_MAX_TAPS - 1; j >= 0; --j) {
      float tap = 0.0f;  // the weight of the input j tokens ago
#pragma unroll
      for (int k = 0; k < LC_MAX_TAPS; ++k)
        if (k == W - 1 - j) tap = w[k];
      if (j < W) y = fmaf(tap, in[j], y);
    }
    out[t * a.C] = TT::put(a.silu ? y * row_sigmoid<TYPE>(y) : y);
  };
  if ((int)blockIdx.x >= a.tiles) {
    long long s, n;
    const int b = blockIdx.x - a.tiles;
    lc_line(a, b, s, n);
    if (n == 0) return;
    E* state = (E*)a.state + (size_t)b * (W - 1) * a.C + c;
    for (int j = 0; j < W - 1; ++j) push(TT::get(state[(size_t)j * a.C]));
    for (int i = 0; i < W - 1 && i < n; ++i) {
      push(TT::get(x[(s + i) * a.x_token]));
      put(s + i);
    }
    for (int j = 0; j < W - 1; ++j) {  // in order: row j + n is still the old one
      const long long at = n - (W - 1) + j;
      state[(size_t)j * a.C] = at >= 0 ? x[(s + at) * a.x_token] : state[(size_t)(j + n) * a.C];
    }
    return;
  }
  const long long t0 = (long long)blockIdx.x * LC_TILE;
  for (int j = W - 1; j > 0; --j) push(t0 >= j ? TT::get(x[(t0 - j) * a.x_token]) : 0.0f);
  for (long long t = t0; t < t0 + LC_TILE && t < a.T; ++t) {
    push(TT::get(x[t * a.x_token]));
    const int role = lc_role(a, t);
    if (role == 2) put(t);
    if (role == 1) out[t * a.C] = TT::put(0.0f);
  }
}

}  // namespace d3
