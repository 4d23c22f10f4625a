// Norms of queries and keys for each head with the position rotation in the same pass, and the cache write.
//   y = x * rsqrt(mean(x^2) + eps) * w          per (token, head), x [D]; w may be absent (no norm for that tensor)
//   pair f of the first `rot` columns, (a, b) = (y[f], y[f + rot/2]), or (y[2f], y[2f + 1]) with `pairs`:
//   (a, b) -> (a c - b s, b c + a s),  (c, s) = rotary[position[axis[f]]][f]
// The columns past `rot` keep their norm only. Sums, products and the rotation are in 32 bits; a value is rounded
// once, to the row's type, when it is stored. Positions have one axis (text) or several (time, height, width): axis[f]
// names the one that turns pair f.
// q goes to a fresh tensor; k to one too, or, with the rows of v, to their slots of a paged cache.
//
// Bound by memory: each row is read once and written once. A lane holds two 16-byte vectors of a head: the ones that turn
// with one another (columns 8i .. and rot/2 + 8i ..), so that the rotation stays within the lane; a head of 128 takes 8
// lanes and a warp four heads at a time, with QR_AHEAD such loads in flight. A warp owns a token, or, where the tokens are
// too few to fill the GPU, a share of its heads. The token's cosines and sines are looked up into shared memory (axis,
// position and table are three loads that wait for one another), then the warp takes its queries, keys and values in
// turn, with the weights in registers. 16 warps an SM of 128 registers; 24 of 80 spilled and took a quarter longer.
// Measured (B200, bf16, device time in graph replays): 16384 tokens of 32 + 4 heads of 128 79 us, 3.8 TB/s; 2048 tokens of
// 16 + 2 heads of 256 with the cache write 15 us, 2.8 TB/s; 16 tokens 3.3 us, the latency of a launch and four loads that
// wait for one another (a call from Python takes the host 15 us). Rows of the other form, 16384 tokens of 32 + 4 heads of
// 80 with 40 columns turned, 270 us; with all 80 turned, in this form, 75.
#pragma once

#include "f32x2.cuh"
#include "rows.cuh"

namespace d3 {

constexpr int QR_WARPS = 4;
constexpr int QR_AHEAD = 2;
constexpr int QR_MAX_AXES = 4;
constexpr int QR_MAX_D = 1024;

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
  const uint8_t* axis;  // [rot / 2], may be null with one axis
  void* q_out;          // [T, Hq, D]
  void* k_out;          // [T, Hkv, D], or null: into the cache
  QrCache kc, vc;
  const int64_t* slots;  // [T]
  int page;
  long long slot_count;
  int share;   // warps per token
  int tokens;  // tokens per block (1 where a token's warps fill more than one)
};

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

// ---- rows of whole 16-byte vectors in twos. A slot is two vectors of a head that one lane has: number i and i + rot / 2
// columns further on of the turned columns (with `pairs`, two neighbours), two neighbours of the others. LANES (a power
// of two) lanes per head, one per slot. Dynamic shared memory: float2 [tokens][rot / 2].
template <int TYPE, int LANES, bool PAIRS>
__global__ void __launch_bounds__(QR_WARPS * 32, 4) qk_rope_kernel(QrArgs a) {
  using TT = QrType<TYPE>;
  using E = typename TT::T;
  constexpr int VEC = 16 / (int)sizeof(E);
  constexpr int HEADS = 32 / LANES;  // heads a warp takes at a time, all queries, keys or values
  constexpr int AHEAD = QR_AHEAD;
  union Vec {
    uint4 q;
    uint32_t w[4];
  };
  extern __shared__ __align__(16) float2 qr_turns[];
  const int lane = threadIdx.x & 31, sub = lane / LANES, l = lane % LANES, warp = threadIdx.x >> 5;
  const int per = (a.share + QR_WARPS - 1) / QR_WARPS;  // blocks of a token, where there are more than one
  const int group = per > 1 ? 0 : warp / a.share;       // of the block's tokens
  const int t = per > 1 ? blockIdx.x / per : blockIdx.x * a.tokens + group;
  const int before = per > 1 ? (blockIdx.x - t * per) * QR_WARPS : 0;  // the token's warps in earlier blocks
  const int part = before + warp - group * a.share;
  const bool active = group < a.tokens && t < a.T && part < a.share;
  const int half = a.rot / 2;
  const bool there = l < a.D / (2 * VEC);
  const bool turned = l * 2 * VEC < a.rot;
  // the first columns of the lane's two vectors
  const int d0 = turned && !PAIRS ? l * VEC : l * 2 * VEC, d1 = turned && !PAIRS ? d0 + half : d0 + VEC;
  const int apart = (d1 - d0) * (int)sizeof(E);
  const int q_items = (a.Hq + HEADS - 1) / HEADS, k_items = (a.Hkv + HEADS - 1) / HEADS;
  float2* turns = qr_turns + group * half;
  grid_dependency_wait();
  allow_dependents();
  // An item is HEADS heads of the token's queries (0), keys (1) or values (2); of the items in that order a warp takes
  // part, part + share, ...
  Vec raw[AHEAD][2] = {};  // a lane without a slot keeps zeros
  const int first = part < q_items ? 0 : part < q_items + k_items ? 1 : 2;
  int n0 = 0, count = 0, heads = 0;  // this warp's first item of the kind, the kind's items and heads
  const char* from = nullptr;        // this lane's row of the next fetch
  long long from_step = 0;
  auto fetch = [&](int n, Vec (&r)[2]) {
    if (n < count && n * HEADS + sub < heads && there) {
      r[0].q = *(const uint4*)from;
      r[1].q = *(const uint4*)(from + apart);
    }
    from += from_step;
  };
  auto begin = [&](int kind) {
    const QrTensor& x = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
    const int earlier = kind == 0 ? 0 : kind == 1 ? q_items : q_items + k_items;
    n0 = part >= earlier ? part - earlier : (a.share - (earlier - part) % a.share) % a.share;
    count = kind == 0 ? q_items : k_items;
    heads = kind == 0 ? a.Hq : a.Hkv;
    const long long step = HEADS * x.head * (long long)sizeof(E);
    from = (const char*)x.p + (t * x.token + sub * x.head + d0) * (long long)sizeof(E) + n0 * step;
    from_step = a.share * step;
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) fetch(n0 + j * a.share, raw[j]);
  };
  if (active) {
    begin(first);
    const int warps = min(a.share - before, QR_WARPS);  // of the token, in this block
    for (int f = (part - before) * 32 + lane; f < half; f += warps * 32) turns[f] = qr_turn(a, t, f);
  }
  if (a.share > 1)
    __syncthreads();
  else
    __syncwarp();
  if (!active) return;
  // the turned columns' cosines and sines: with halves, column e of both vectors turns by the same ones
  uint64_t c2[VEC / 2], s2[VEC / 2];
  if (!PAIRS && turned) {
#pragma unroll
    for (int e = 0; e < VEC / 2; ++e) {
      const float4 x = *(const float4*)(turns + d0 + 2 * e);  // d0 is even
      c2[e] = f2_make(x.x, x.z);
      s2[e] = f2_make(x.y, x.w);
    }
  }
  const float inv_d = 1.0f / (float)a.D;
#pragma unroll 1
  for (int kind = first; kind < (a.k_out ? 2 : 3); ++kind) {
    if (kind != first) begin(kind);
    if (n0 >= count) continue;
    char* to;
    long long to_step;
    if (kind > 0 && !a.k_out) {
      const QrCache& cache = kind == 1 ? a.kc : a.vc;
      to = (char*)qr_slot<E>(a, cache, a.slots[t], sub);
      if (!to) continue;
      to_step = HEADS * cache.head * (long long)sizeof(E);
    } else {
      to = (char*)(kind == 0 ? a.q_out : a.k_out) + ((size_t)t * heads + sub) * a.D * sizeof(E);
      to_step = HEADS * (long long)a.D * (long long)sizeof(E);
    }
    to += d0 * (long long)sizeof(E) + n0 * to_step;
    to_step *= a.share;
    const void* w = kind == 0 ? a.qw : a.kw;
    uint64_t W[2][VEC / 2];  // two columns each
    if (kind < 2 && there) {
      float x[VEC];
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        qr_weights<TYPE, VEC>(w, a.w_f32, a.w_add, v ? d1 : d0, x);
#pragma unroll
        for (int e = 0; e < VEC / 2; ++e) W[v][e] = f2_make(x[2 * e], x[2 * e + 1]);
      }
    }
#pragma unroll 1
    for (int n = n0; n < count; n += AHEAD * a.share) {
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const int nj = n + j * a.share;
        if (nj >= count) break;  // the same for the whole warp
        Vec out[2];
        if (kind == 2) {
          out[0].q = raw[j][0].q;
          out[1].q = raw[j][1].q;
          fetch(nj + AHEAD * a.share, raw[j]);
        } else {
          uint64_t x2[2][VEC / 2], sums = 0;
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            float x[VEC];
            qr_unpack<TYPE, VEC>(raw[j][v].w, x);
#pragma unroll
            for (int e = 0; e < VEC / 2; ++e) {
              x2[v][e] = f2_make(x[2 * e], x[2 * e + 1]);
              sums = f2_fma(x2[v][e], x2[v][e], sums);
              x2[v][e] = f2_mul(x2[v][e], W[v][e]);
            }
          }
          fetch(nj + AHEAD * a.share, raw[j]);
          float inv = 1.0f;
          if (w) {
            float s0, s1;
            f2_split(sums, s0, s1);
            float sum = s0 + s1;
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            inv = rsqrtf(fmaf(sum, inv_d, a.eps));
          }
          const uint64_t inv2 = f2_make(inv, inv);
          float y[2][VEC];
          if (!turned) {
#pragma unroll
            for (int v = 0; v < 2; ++v)
#pragma unroll
              for (int e = 0; e < VEC / 2; ++e) f2_split(f2_mul(x2[v][e], inv2), y[v][2 * e], y[v][2 * e + 1]);
          } else if (!PAIRS) {
#pragma unroll
            for (int e = 0; e < VEC / 2; ++e) {
              const uint64_t c = f2_mul(c2[e], inv2), s = f2_mul(s2[e], inv2), minus = f2_mul(s, f2_make(-1.0f, -1.0f));
              f2_split(f2_fma(x2[1][e], minus, f2_mul(x2[0][e], c)), y[0][2 * e], y[0][2 * e + 1]);
              f2_split(f2_fma(x2[0][e], s, f2_mul(x2[1][e], c)), y[1][2 * e], y[1][2 * e + 1]);
            }
          } else {
#pragma unroll
            for (int v = 0; v < 2; ++v)
#pragma unroll
              for (int e = 0; e < VEC / 2; ++e) {
                const float2 cs = turns[(v ? d1 : d0) / 2 + e];
                const float c = cs.x * inv, s = cs.y * inv;
                float lo, hi;
                f2_split(x2[v][e], lo, hi);
                y[v][2 * e] = fmaf(hi, -s, lo * c);
                y[v][2 * e + 1] = fmaf(lo, s, hi * c);
              }
          }
          qr_pack<TYPE, VEC>(y[0], out[0].w);
          qr_pack<TYPE, VEC>(y[1], out[1].w);
        }
        if (nj * HEADS + sub < heads && there) {
          *(uint4*)to = out[0].q;
          *(uint4*)(to + apart) = out[1].q;
        }
        to += to_step;
      }
    }
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
  auto normed = [&](int d) { return TT::get(x[d]) * qr_weight<TYPE>(w, a.w_f32, a.w_add, d); };
  const int half = a.rot / 2;
  for (int f = lane; f < half; f += 32) {  // the same steps as in the other form
    const int da = pairs ? 2 * f : f, db = pairs ? 2 * f + 1 : f + half;
    const float2 cs = qr_turn(a, t, f);
    const float xa = normed(da), xb = normed(db), c = cs.x * inv, s = cs.y * inv;
    out[da] = TT::put(fmaf(xb, -s, xa * c));
    out[db] = TT::put(fmaf(xa, s, xb * c));
  }
  for (int d = a.rot + lane; d < a.D; d += 32) out[d] = TT::put(normed(d) * inv);
}

}  // namespace d3
