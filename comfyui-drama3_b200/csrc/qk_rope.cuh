// Norms of queries and keys for each head with the position rotation in the same pass, and the cache write.
//   y = x * rsqrt(mean(x^2) + eps) * w          per (token, head), x [D]; w may be absent (no norm for that tensor)
//   pair f of the first `rot` columns, (a, b) = (y[f], y[f + rot/2]), or (y[2f], y[2f + 1]) with `pairs`:
//   (a, b) -> (a c - b s, b c + a s),  (c, s) = rotary[position[axis[f]]][f]
// The columns past `rot` keep their norm only. Sums, products and the rotation are in 32 bits; a value is rounded
// once, to the row's type, when it is stored. Positions have one axis (text) or several (time, height, width): axis[f]
// names the one that turns pair f.
// q goes to a fresh tensor; k to one too, or, with the rows of v, to their slots of a paged cache.
//
// Bound by memory: each row is read once and written once. A warp owns a token (or, where the tokens are too few to
// fill the GPU, a share of its heads) and walks its heads with the same cosines and sines in registers: a lane holds
// 16 bytes of a head (8 columns of 16 bits), a head of 128 takes 16 lanes, so a warp takes two heads at a time, and
// four such loads are in flight before the first is used.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace d3 {

enum { QR_BF16 = 0, QR_F16 = 1, QR_F32 = 2 };
constexpr int QR_WARPS = 8;
constexpr int QR_MAX_AXES = 4;
constexpr int QR_MAX_D = 1024;

struct QrTensor {  // rows [T, heads, D], the last dimension contiguous
  const void* p;
  long long token, head;  // strides in elements
};
struct QrCache {  // [pages, page, heads, D], the last dimension contiguous
  void* p;
  long long page, token, head;
};
struct QrArgs {
  QrTensor q, k, v;
  int T, Hq, Hkv, D;
  const void* qw;
  const void* kw;
  int w_f32;        // the weights are fp32 rather than of the rows' type
  float w_add;      // added to each weight (1 for weights stored around zero)
  float eps;
  const float2* rotary;  // [length, rot / 2] (cos, sin)
  int rot, length;
  const int64_t* pos;   // [axes, T]
  int axes;
  const uint8_t* axis;  // [rot / 2], null with one axis
  void* q_out;          // [T, Hq, D]
  void* k_out;          // [T, Hkv, D], or null: into the cache
  QrCache kc, vc;
  const int64_t* slots;  // [T]
  int page;
  long long slot_count;
  int share;  // warps per token
};

template <int TYPE> struct QrType;
template <> struct QrType<QR_BF16> {
  using T = uint16_t;
  static D3_DEV float get(uint16_t v) { return bf16_to_f32(v); }
  static D3_DEV uint16_t put(float v) { return __bfloat16_as_ushort(__float2bfloat16_rn(v)); }
};
template <> struct QrType<QR_F16> {
  using T = uint16_t;
  static D3_DEV float get(uint16_t v) { return __half2float(__ushort_as_half(v)); }
  static D3_DEV uint16_t put(float v) { return __half_as_ushort(__float2half_rn(v)); }
};
template <> struct QrType<QR_F32> {
  using T = float;
  static D3_DEV float get(float v) { return v; }
  static D3_DEV float put(float v) { return v; }
};

template <int TYPE> D3_DEV float qr_weight(const void* w, bool f32, float add, int d) {
  if (!w) return 1.0f;
  return (f32 ? ((const float*)w)[d] : QrType<TYPE>::get(((const typename QrType<TYPE>::T*)w)[d])) + add;
}

// (cos, sin) of pair f of token t; (1, 0) with the fault word set where the table has none.
D3_DEV float2 qr_turn(const QrArgs& a, int t, int f) {
  const int ax = a.axis ? a.axis[f] : 0;
  if (ax < a.axes) {
    const int64_t p = a.pos[(size_t)ax * a.T + t];
    if (p >= 0 && p < a.length) return __ldg(a.rotary + (size_t)p * (a.rot / 2) + f);
  }
  record_fault(FAULT_POSITION);
  return make_float2(1.0f, 0.0f);
}

// Destination of token t's row in a cache; null for a token without a slot, or (fault) one outside the cache.
template <class E>
D3_DEV E* qr_slot(const QrArgs& a, const QrCache& c, int64_t slot, int head) {
  if (slot < 0) return nullptr;
  if (slot >= a.slot_count) {
    record_fault(FAULT_BAD_SLOT);
    return nullptr;
  }
  const int64_t page = slot / a.page;
  return (E*)c.p + page * c.page + (slot - page * a.page) * c.token + head * c.head;
}

D3_DEV const void* qr_row(const QrArgs& a, int t, int h, int size) {
  const QrTensor* x = &a.q;
  if (h >= a.Hq) {
    h -= a.Hq;
    x = &a.k;
    if (h >= a.Hkv) {
      h -= a.Hkv;
      x = &a.v;
    }
  }
  return (const char*)x->p + (t * x->token + h * x->head) * size;
}

// Where row h (query heads, then key heads, then value heads) of token t goes; null: nowhere.
template <class E>
D3_DEV E* qr_target(const QrArgs& a, int t, int h, int64_t slot) {
  if (h < a.Hq) return (E*)a.q_out + ((size_t)t * a.Hq + h) * a.D;
  h -= a.Hq;
  if (a.k_out) return (E*)a.k_out + ((size_t)t * a.Hkv + h) * a.D;
  return h < a.Hkv ? qr_slot<E>(a, a.kc, slot, h) : qr_slot<E>(a, a.vc, slot, h - a.Hkv);
}

// ---- rows of whole 16-byte vectors, no pair's halves inside one vector (with `pairs`: no pair cut by one). LANES
// lanes (a power of two) per head, NV vectors a lane; vector i of lane l is number l + i * LANES of the head.
template <int TYPE, int LANES, int NV, bool PAIRS>
__global__ void __launch_bounds__(QR_WARPS * 32) qk_rope_kernel(QrArgs a) {
  using TT = QrType<TYPE>;
  using E = typename TT::T;
  constexpr int VEC = 16 / (int)sizeof(E);
  constexpr int HEADS = 32 / LANES;  // heads a warp takes at a time
  constexpr int AHEAD = 4;
  union Vec {
    uint4 q;
    E e[VEC];
  };
  const int lane = threadIdx.x & 31, sub = lane / LANES, l = lane % LANES;
  const int gw = blockIdx.x * QR_WARPS + (threadIdx.x >> 5);
  const int t = gw / a.share, part = gw - t * a.share;
  grid_dependency_wait();
  allow_dependents();
  if (t >= a.T) return;
  const int vectors = a.D / VEC, half = a.rot / 2, shift = half / VEC;
  const int heads = a.Hq + a.Hkv * (a.k_out ? 1 : 2);
  const int64_t slot = a.k_out ? -1 : a.slots[t];
  Vec raw[AHEAD][NV];
  auto load = [&](int h, Vec (&r)[NV]) {
    if (h >= heads) return;
    const uint4* p = (const uint4*)qr_row(a, t, h, sizeof(E));
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (l + i * LANES < vectors) r[i].q = p[l + i * LANES];
  };
  const int step = HEADS * a.share;
  const int h_first = HEADS * part + sub;
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) load(h_first + j * step, raw[j]);
  // this lane's cosines and sines: with halves, column d becomes y[d] * c + y[partner] * s (s of the first half
  // negative); with pairs, entries 2e and 2e + 1 of a vector share cs[e]
  float c[NV][VEC], s[NV][VEC], wq[NV][VEC], wk[NV][VEC];
  bool turned[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int vi = l + i * LANES, d0 = vi * VEC;
    turned[i] = d0 < a.rot;
    const bool second = !PAIRS && d0 >= half;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      c[i][e] = 1.0f;
      s[i][e] = 0.0f;
      if (turned[i] && (!PAIRS || e % 2 == 0)) {
        const float2 cs = qr_turn(a, t, PAIRS ? (d0 + e) / 2 : d0 + e - (second ? half : 0));
        c[i][e] = cs.x;
        s[i][e] = PAIRS || second ? cs.y : -cs.y;
      }
      wq[i][e] = vi < vectors ? qr_weight<TYPE>(a.qw, a.w_f32, a.w_add, d0 + e) : 0.0f;
      wk[i][e] = vi < vectors ? qr_weight<TYPE>(a.kw, a.w_f32, a.w_add, d0 + e) : 0.0f;
    }
  }
  const float inv_d = 1.0f / (float)a.D;
  for (int h0 = h_first; h0 - sub < heads; h0 += AHEAD * step) {
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int h = h0 + j * step;
      if (h - sub >= heads) break;  // the same for the whole warp
      const bool live = h < heads, is_q = h < a.Hq, is_v = h >= a.Hq + a.Hkv;
      float y[NV][VEC], sum = 0.0f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          y[i][e] = live && l + i * LANES < vectors ? TT::get(raw[j][i].e[e]) : 0.0f;
          sum = fmaf(y[i][e], y[i][e], sum);
        }
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      const float inv = (is_q ? a.qw : a.kw) ? rsqrtf(fmaf(sum, inv_d, a.eps)) : 1.0f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) y[i][e] *= inv * (is_q ? wq[i][e] : wk[i][e]);
      Vec out[NV];
      if (PAIRS) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int e = 0; e < VEC; e += 2) {
            out[i].e[e] = TT::put(fmaf(y[i][e], c[i][e], -y[i][e + 1] * s[i][e]));
            out[i].e[e + 1] = TT::put(fmaf(y[i][e + 1], c[i][e], y[i][e] * s[i][e]));
          }
      } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int vi = l + i * LANES;
          const int pv = vi < shift ? vi + shift : vi - shift;  // partner vector (unused where not turned)
          const int src = sub * LANES + (pv & (LANES - 1));
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            float other = 0.0f;
#pragma unroll
            for (int n = 0; n < NV; ++n) {
              const float o = __shfl_sync(0xffffffffu, y[n][e], src);
              if (NV == 1 || pv / LANES == n) other = o;
            }
            out[i].e[e] = TT::put(turned[i] ? fmaf(y[i][e], c[i][e], other * s[i][e]) : y[i][e]);
          }
        }
      }
      if (live) {
        E* p = qr_target<E>(a, t, h, slot);
        if (p) {
#pragma unroll
          for (int i = 0; i < NV; ++i)
            if (l + i * LANES < vectors) ((uint4*)p)[l + i * LANES] = is_v ? raw[j][i].q : out[i].q;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) load(h0 + (AHEAD + j) * step, raw[j]);
  }
}

// ---- any other row (odd sizes, strides or addresses): a warp per (token, head), two passes of single elements
template <int TYPE>
__global__ void __launch_bounds__(QR_WARPS * 32) qk_rope_any_kernel(QrArgs a, int pairs) {
  using TT = QrType<TYPE>;
  using E = typename TT::T;
  const int lane = threadIdx.x & 31;
  grid_dependency_wait();
  allow_dependents();
  const int heads = a.Hq + a.Hkv * (a.k_out ? 1 : 2);
  const long long gw = (long long)blockIdx.x * QR_WARPS + (threadIdx.x >> 5);
  const int t = (int)(gw / heads), h = (int)(gw - (long long)t * heads);
  if (t >= a.T) return;
  const E* x = (const E*)qr_row(a, t, h, sizeof(E));
  E* out = qr_target<E>(a, t, h, a.k_out ? -1 : a.slots[t]);
  if (!out) return;
  if (h >= a.Hq + a.Hkv) {
    for (int d = lane; d < a.D; d += 32) out[d] = x[d];
    return;
  }
  const void* w = h < a.Hq ? a.qw : a.kw;
  float inv = 1.0f;
  if (w) {
    float sum = 0.0f;
    for (int d = lane; d < a.D; d += 32) {
      const float v = TT::get(x[d]);
      sum = fmaf(v, v, sum);
    }
    inv = rsqrtf(fmaf(warp_sum(sum), 1.0f / (float)a.D, a.eps));
  }
  auto normed = [&](int d) { return TT::get(x[d]) * (inv * qr_weight<TYPE>(w, a.w_f32, a.w_add, d)); };
  const int half = a.rot / 2;
  for (int f = lane; f < half; f += 32) {
    const int da = pairs ? 2 * f : f, db = pairs ? 2 * f + 1 : f + half;
    const float2 cs = qr_turn(a, t, f);
    const float ya = normed(da), yb = normed(db);
    out[da] = TT::put(fmaf(ya, cs.x, -yb * cs.y));
    out[db] = TT::put(fmaf(yb, cs.x, ya * cs.y));
  }
  for (int d = a.rot + lane; d < a.D; d += 32) out[d] = TT::put(normed(d));
}

}  // namespace d3
