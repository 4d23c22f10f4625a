// Linear attention with a decay for each head, over a state of each line (drama3/config.py:59-60: three of four layers of the
// reference's decoder; its own code leaves them to its host application). For each head, S [Dv, Dk]:
//   S <- exp(g_t) S
//   u = beta_t (v_t - S k_t)      with the delta rule;  u = v_t without (beta null)
//   S <- S + u k_t^T
//   o_t = scale S q_t
// g = -exp(a_log) softplus(decay + dt_bias) and beta = sigmoid(beta) where a_log is given (the projections' raw outputs),
// else decay is the logarithm itself (above 0 counts as 0) and beta is taken as it is. With eps >= 0, q and k are divided by
// sqrt(sum of squares + eps) first. Value head h reads key head h / (Hv / Hk).
#pragma once

#include "rows.cuh"

namespace d3 {

struct LdArgs {
  QrTensor q, k, v;  // rows [T, heads, D]
  int T, B, Hk, Hv, Dk, Dv;
  const void* decay;  // [T, Hv]
  const void* beta;   // [T, Hv] or null
  long long decay_token, beta_token;  // strides in elements
  int gates_f32;                      // decay and beta are fp32 rather than of the rows' type
  const float* a_log;    // [Hv] or null
  const float* dt_bias;  // [Hv] or null (0)
  float eps, scale;      // eps < 0: rows as they are
  float* state;          // [B, Hv, Dv, Dk]
  const int* cu;
  const int* line;
  void* out;  // [T, Hv, Dv]
};

template <int TYPE> D3_DEV float ld_gate(const void* p, bool f32, long long at) {
  return f32 ? ((const float*)p)[at] : QrType<TYPE>::get(((const typename QrType<TYPE>::T*)p)[at]);
}

// The logarithm of the decay of token t's head h, at most 0 (a NaN stays one).
template <int TYPE> D3_DEV float ld_log_decay(const LdArgs& a, long long t, int h) {
  float g = ld_gate<TYPE>(a.decay, a.gates_f32, t * a.decay_token + h);
  if (a.a_log) {
    if (a.dt_bias) g += a.dt_bias[h];
    // log(1 + e^g) without overflow
    g = -expf(a.a_log[h]) * (fmaxf(g, 0.0f) + log1pf(expf(-fabsf(g))));
  }
  return g > 0.0f ? 0.0f : g;
}

// How strongly token t's head h corrects the state.
template <int TYPE> D3_DEV float ld_beta(const LdArgs& a, long long t, int h) {
  const float b = ld_gate<TYPE>(a.beta, a.gates_f32, t * a.beta_token + h);
  return a.a_log ? 1.0f / (1.0f + expf(-b)) : b;
}

// The power of two that takes values of at most `most` below 2^14, and its inverse (exact, normal numbers both; 1 for a row
// of zeros).
D3_DEV void ld_scale(float most, float& up, float& down) {
  const int e = most > 0.0f ? max((int)(__float_as_uint(most) >> 23) - 127, -113) : 13;
  up = __uint_as_float((uint32_t)(127 + 13 - e) << 23);
  down = __uint_as_float((uint32_t)(127 - 13 + e) << 23);
}

// What takes a row up x, with squares that add up to `sum`, to x / sqrt(|x|^2 + eps), or with eps < 0 to x: up a power of two, down its
// inverse. (Where eps is past 32 bits in the row's scale, nothing of the row counts beside it.)
D3_DEV float ld_unit(float sum, float eps, float up, float down) {
  if (eps < 0.0f) return down;
  const float e = eps * up * up;
  return e <= 3.4028234e38f ? rsqrtf(sum + e) : rsqrtf(eps) * down;
}

// ---- Token by token. A warp holds LS_ROWS x (32 / lanes) rows of a head's state in registers, 16 bytes of a row a lane,
// and takes the line's tokens in turn. S k and S q are summed in one go, on the state before the token: o = scale (e^g S q +
// u (k . q)). Bound by memory where the tokens are few: a state is read once and written once, 8 Dk Dv bytes a head against 7
// Dk Dv operations a token, so that all of a warp's rows are asked for at once. Sums over a row's lanes halve the values as
// they halve the lanes: nine exchanges for eight rows where a butterfly for each would take forty.
// Measured (B200, bf16, 16 / 32 heads of 128): 256 lines of a token 126 us device time, 6.5 TB/s; 16 lines 13.4 us in a stream of calls, 9.3
// where the states stay in L2; one line 2.8 to 3.1 us, the latency of a launch and three loads that wait for one another.
constexpr int LS_WARPS = 4;
constexpr int LS_ROWS = 8;

// v[r] summed over groups of LANES lanes: the sum of v[ls_row(lane)] in each lane.
template <int LANES> D3_DEV float ls_sum(float (&v)[LS_ROWS], int lane) {
  int o = LANES / 2;
#pragma unroll
  for (int n = LS_ROWS / 2; n > 0; n >>= 1, o >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float give = up ? v[i] : v[i + n], keep = up ? v[i + n] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
    }
  }
  float s = v[0];
  for (; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}
// Which of the rows that is, and a lane of the group that has row r.
template <int LANES> D3_DEV int ls_row(int lane) { return (lane & (LANES - 1)) / (LANES / LS_ROWS); }
template <int LANES> D3_DEV int ls_lane(int r) { return r * (LANES / LS_ROWS); }

// Grid: (blocks of rows of a head, Hv, B + 1): the last one writes zeros for the places past the lines' last token.
template <int TYPE, int DK, bool DELTA>
__global__ void __launch_bounds__(LS_WARPS * 32) lines_delta_step_kernel(LdArgs a) {
  using TT = QrType<TYPE>;
  using E = typename TT::T;
  constexpr int LANES = DK / 4, GROUPS = 32 / LANES, ROWS = LS_ROWS * GROUPS;
  const int lane = threadIdx.x & 31, group = lane / LANES, l = lane % LANES;
  const int h = blockIdx.y, b = blockIdx.z, hk = h / (a.Hv / a.Hk);
  const int row0 = (blockIdx.x * LS_WARPS + (threadIdx.x >> 5)) * ROWS + group * LS_ROWS;  // LS_ROWS rows of this group
  const int mine = row0 + ls_row<LANES>(lane);
  const bool writes = l % (LANES / LS_ROWS) == 0 && mine < a.Dv;
  E* out = (E*)a.out + (size_t)h * a.Dv + mine;
  grid_dependency_wait();
  allow_dependents();
  const int s = min(max(a.cu[b], 0), a.T);
  if (b == a.B) {
    if (writes)
      for (long long t = s; t < a.T; ++t) out[t * a.Hv * a.Dv] = TT::put(0.0f);
    return;
  }
  const int e = min(a.cu[b + 1], a.T);
  if (e <= s) return;
  float* state = a.state + (((size_t)b * a.Hv + h) * a.Dv + row0) * DK + l * 4;
  float S[LS_ROWS][4] = {};
#pragma unroll
  for (int r = 0; r < LS_ROWS; ++r)
    if (row0 + r < a.Dv) {
      const float4 x = *(const float4*)(state + r * DK);
      S[r][0] = x.x, S[r][1] = x.y, S[r][2] = x.z, S[r][3] = x.w;
    }
  for (long long t = s; t < e; ++t) {
    float k[4], q[4];
    {
      const E* kp = (const E*)a.k.p + t * a.k.token + hk * a.k.head + l * 4;
      const E* qp = (const E*)a.q.p + t * a.q.token + hk * a.q.head + l * 4;
      const uint2 kw = *(const uint2*)kp, qw = *(const uint2*)qp;
      TT::get2(kw.x, k[0], k[1]), TT::get2(kw.y, k[2], k[3]);
      TT::get2(qw.x, q[0], q[1]), TT::get2(qw.y, q[2], q[3]);
    }
    const float v = mine < a.Dv ? TT::get(((const E*)a.v.p)[t * a.v.token + h * a.v.head + mine]) : 0.0f;
    const float alpha = expf(ld_log_decay<TYPE>(a, t, h));
    const float beta = DELTA ? ld_beta<TYPE>(a, t, h) : 1.0f;
    float kk, qq, kq, k_up = 1.0f, k_down = 1.0f, q_up = 1.0f, q_down = 1.0f;
    auto sums = [&] {
      kk = qq = kq = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) kk = fmaf(k[i], k[i], kk), qq = fmaf(q[i], q[i], qq), kq = fmaf(k[i], q[i], kq);
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) {
        kk += __shfl_xor_sync(0xffffffffu, kk, o);
        qq += __shfl_xor_sync(0xffffffffu, qq, o);
        kq += __shfl_xor_sync(0xffffffffu, kq, o);
      }
    };
    sums();
    // rows whose squares leave 32 bits, or come near to (or are zeros): by a power of two that brings the largest value into [1, 2)
    if (__any_sync(0xffffffffu, !(fminf(kk, qq) >= 0x1p-60f && fmaxf(kk, qq) <= 0x1p100f))) {
      float most[2] = {fmaxf(fmaxf(fabsf(k[0]), fabsf(k[1])), fmaxf(fabsf(k[2]), fabsf(k[3]))),
                       fmaxf(fmaxf(fabsf(q[0]), fabsf(q[1])), fmaxf(fabsf(q[2]), fabsf(q[3])))};
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < 2; ++i) most[i] = fmaxf(most[i], __shfl_xor_sync(0xffffffffu, most[i], o));
      ld_scale(most[0], k_up, k_down);
      ld_scale(most[1], q_up, q_down);
      k_up *= 0x1p-13f, k_down *= 0x1p13f, q_up *= 0x1p-13f, q_down *= 0x1p13f;
#pragma unroll
      for (int i = 0; i < 4; ++i) k[i] *= k_up, q[i] *= q_up;
      sums();
    }
    // a row of zeros stays one, with eps 0 too
    const float rk = kk == 0.0f ? 0.0f : ld_unit(kk, a.eps, k_up, k_down);
    const float rq = (qq == 0.0f ? 0.0f : ld_unit(qq, a.eps, q_up, q_down)) * a.scale;
    float sk[LS_ROWS], sq[LS_ROWS];
#pragma unroll
    for (int r = 0; r < LS_ROWS; ++r) {
      sk[r] = sq[r] = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (DELTA) sk[r] = fmaf(S[r][i], k[i], sk[r]);
        sq[r] = fmaf(S[r][i], q[i], sq[r]);
      }
    }
    const float Sq = ls_sum<LANES>(sq, lane);
    float u = v;
    if (DELTA) u = beta * (v - alpha * rk * ls_sum<LANES>(sk, lane));
    if (writes) out[t * a.Hv * a.Dv] = TT::put(rq * (alpha * Sq + u * rk * kq));
    u *= rk;
#pragma unroll
    for (int r = 0; r < LS_ROWS; ++r) {
      const float ur = __shfl_sync(0xffffffffu, u, group * LANES + ls_lane<LANES>(r));
#pragma unroll
      for (int i = 0; i < 4; ++i) S[r][i] = fmaf(ur, k[i], alpha * S[r][i]);
    }
  }
#pragma unroll
  for (int r = 0; r < LS_ROWS; ++r)
    if (row0 + r < a.Dv) *(float4*)(state + r * DK) = make_float4(S[r][0], S[r][1], S[r][2], S[r][3]);
}

}  // namespace d3
