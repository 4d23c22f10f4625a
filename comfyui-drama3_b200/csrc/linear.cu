// C ABI of the linear half of a hybrid decoder (declared in include/drama3_b200.h): the short convolution of each line's
// tokens, linear attention with decays over a state of each line, the norm of its heads with their gate, and the join of a
// block to its residual with its norms. Same conventions as drama3_b200.cu: arguments are checked before anything is
// launched, nothing is allocated, nothing synchronizes.
#include "block_norm.cuh"
#include "host.cuh"
#include "lines_conv.cuh"
#include "lines_delta_chunk.cuh"

using namespace d3host;

// This translation unit's fault word (each has its own), read and cleared for d3_take_fault.
int d3_linear_take_fault(unsigned int* fault) {
  unsigned int v = 0, zero = 0;
  if (int st = cuda_status(cudaMemcpyFromSymbol(&v, d3::g_fault, sizeof(v)))) return st;
  *fault = v;
  return cuda_status(cudaMemcpyToSymbol(d3::g_fault, &zero, sizeof(zero)));
}

namespace {

constexpr int kMaxLines = 8192;

template <int TYPE, int LANES, int NV>
int gated_launch(const d3::GnArgs& a, const DeviceInfo& d, cudaStream_t s) {
  // four rows of a group of lanes at a time once that leaves every SM 16 warps
  constexpr int AHEAD = NV == 1 ? 4 : NV == 2 ? 2 : 1;
  const long long rows = (long long)a.T * a.H, per = 32 / LANES * d3::BN_WARPS;
  const dim3 threads(d3::BN_WARPS * 32);
  if (rows >= per * AHEAD * 4 * d.sms)
    return launch(d3::gated_norm_kernel<TYPE, LANES, NV, AHEAD>, dim3((unsigned)((rows + per * AHEAD - 1) / (per * AHEAD))),
                  threads, 0, s, true, a);
  return launch(d3::gated_norm_kernel<TYPE, LANES, NV, 1>, dim3((unsigned)((rows + per - 1) / per)), threads, 0, s, true, a);
}

template <int TYPE>
int gated_type(const d3::GnArgs& a, bool vectors, const DeviceInfo& d, cudaStream_t s) {
  constexpr int VEC = TYPE == d3::QR_F32 ? 4 : 8;
  const int n = a.D / VEC;
  if (!vectors || a.D % VEC || n > 128) {
    const long long rows = (long long)a.T * a.H;
    return launch(d3::gated_norm_any_kernel<TYPE>, dim3((unsigned)((rows + d3::BN_WARPS - 1) / d3::BN_WARPS)),
                  dim3(d3::BN_WARPS * 32), 0, s, true, a);
  }
  if (n <= 8) return gated_launch<TYPE, 8, 1>(a, d, s);
  if (n <= 16) return gated_launch<TYPE, 16, 1>(a, d, s);
  if (n <= 32) return gated_launch<TYPE, 32, 1>(a, d, s);
  if (n <= 64) return gated_launch<TYPE, 32, 2>(a, d, s);
  return gated_launch<TYPE, 32, 4>(a, d, s);
}

template <int TYPE>
int join_type(const d3::AnArgs& a, bool vectors, const DeviceInfo& d, cudaStream_t s) {
  constexpr int VEC = TYPE == d3::QR_F32 ? 4 : 8;
  const int n = a.W / VEC;
  if (!vectors || a.W % VEC || n > 2 * d3::BN_MAX_THREADS)
    return launch(d3::add_norm_any_kernel<TYPE>, dim3(a.T), dim3(256), 0, s, true, a);
  // a warp a row where that leaves every SM 16 warps
  if (n <= 256 && a.T >= 16 * d.sms) {
    const dim3 blocks((a.T + d3::BN_WARPS - 1) / d3::BN_WARPS), threads(d3::BN_WARPS * 32);
    if (n <= 64) return launch(d3::add_norm_warp_kernel<TYPE, 2>, blocks, threads, 0, s, true, a);
    if (n <= 128) return launch(d3::add_norm_warp_kernel<TYPE, 4>, blocks, threads, 0, s, true, a);
    return launch(d3::add_norm_warp_kernel<TYPE, 8>, blocks, threads, 0, s, true, a);
  }
  const int nv = n <= d3::BN_MAX_THREADS ? 1 : 2;
  const int threads = ((n + nv - 1) / nv + 31) / 32 * 32;
  const dim3 blocks(a.T);
  return nv == 1 ? launch(d3::add_norm_kernel<TYPE, 1>, blocks, dim3(threads), 0, s, true, a)
                 : launch(d3::add_norm_kernel<TYPE, 2>, blocks, dim3(threads), 0, s, true, a);
}

template <int TYPE>
int conv_type(const d3::LcArgs& a, bool vectors, cudaStream_t s) {
  constexpr int VEC = TYPE == d3::QR_F32 ? 4 : 8;
  const dim3 threads(d3::LC_THREADS);
  const int per = vectors && a.W <= 4 ? d3::LC_THREADS * VEC : d3::LC_THREADS;
  const dim3 blocks(a.tiles + a.B, (a.C + per - 1) / per);
  if (per == d3::LC_THREADS) return launch(d3::lines_conv_any_kernel<TYPE>, blocks, threads, 0, s, true, a);
  switch (a.W) {
    case 2: return launch(d3::lines_conv_kernel<TYPE, 2>, blocks, threads, 0, s, true, a);
    case 3: return launch(d3::lines_conv_kernel<TYPE, 3>, blocks, threads, 0, s, true, a);
    default: return launch(d3::lines_conv_kernel<TYPE, 4>, blocks, threads, 0, s, true, a);
  }
}

// Whether lines_delta goes token by token (or in chunks). Measured (B200, 16 / 32 heads of 128, us by tokens / in chunks): lines of 4
// tokens each, 1 line 5.7 / 27, 16 lines 21 / 68, 256 lines 303 / 753; of 8, 16 lines 37 / 69, 256 lines 537 / 778; of 16, 1 line 17 / 26,
// 16 lines 69 / 75, 256 lines 1017 / 835; one line of 32 31 / 26. So lines of equal length meet near 12 tokens, but how tokens are spread is
// known on the GPU alone, and the longest line sets the time by tokens: all but one line with a token, the last with the rest of 4 a
// line, 16 lines 58 / 68, 256 lines 1082 / 796; 1024 tokens of one line, the other 255 idle, 985 / 115.
bool delta_steps(int T, int B) { return T <= 4LL * B || T <= 16; }

size_t delta_block_bytes(int Hk, int Hv, int Dk) {
  return Dk == 64 ? Hk * sizeof(d3::LdRows<64>) + Hv * sizeof(d3::LdHead<64>)
                  : Hk * sizeof(d3::LdRows<128>) + Hv * sizeof(d3::LdHead<128>);
}

// Chunks prepared and scanned by a pair of launches: as many as 384 MB hold (eight at least), or equal parts below that. (B200, 8192 tokens of 16 / 32
// heads of 128, an earlier form of the scan: 438 us in one pair, 469 in parts of 37 chunks, whose 70 MB stay in L2, 714 in parts of 9:
// the scan starts anew in each.)
int delta_blocks(int T, int Hk, int Hv, int Dk) {
  const size_t all = ((size_t)T + d3::LD_C - 1) / d3::LD_C, most = (384u << 20) / delta_block_bytes(Hk, Hv, Dk);
  const size_t fit = most < 8 ? 8 : most, parts = (all + fit - 1) / fit;
  return (int)((all + parts - 1) / parts);
}

template <int TYPE, int DK, bool DELTA, int WARPS, int PARTS>
int scan_launch(const CUtensorMap& vmap, const d3::LdChunkArgs& c, cudaStream_t s) {
  constexpr int smem = d3::LdScanShape<DK, WARPS, PARTS>::SMEM;
  static std::atomic<uint64_t> done{0};
  if (int st = allow_smem_once(d3::lines_delta_scan_kernel<TYPE, DK, DELTA, WARPS, PARTS>, smem, done)) return st;
  const dim3 blocks((c.a.Dv / 16 + WARPS - 1) / WARPS, c.a.Hv, c.a.B + 1);
  return launch(d3::lines_delta_scan_kernel<TYPE, DK, DELTA, WARPS, PARTS>, blocks,
                dim3(d3::LdScanShape<DK, WARPS, PARTS>::THREADS), smem, s, true, vmap, c);
}

template <int TYPE, int DK, bool DELTA>
int chunk_launch(const d3::LdArgs& a, void* workspace, const DeviceInfo& d, cudaStream_t s) {
  constexpr int prep_smem = d3::LdPrepShape<DK>::SMEM;
  static std::atomic<uint64_t> done{0};
  if (int st = allow_smem_once(d3::lines_delta_prep_kernel<TYPE, DK, DELTA>, prep_smem, done)) return st;
  CUtensorMap vmap;
  cuuint64_t dims[3] = {(cuuint64_t)a.Dv, (cuuint64_t)a.Hv, (cuuint64_t)a.T};
  cuuint64_t strides[2] = {(cuuint64_t)a.v.head * 2, (cuuint64_t)a.v.token * 2};
  cuuint32_t box[3] = {16, 1, d3::LD_C};
  if (!encode_tiled(&vmap, TYPE == d3::QR_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, a.v.p,
                    dims, strides, box, CU_TENSOR_MAP_SWIZZLE_32B))
    return D3_ERR_ARG;
  const int all = (int)(((long long)a.T + d3::LD_C - 1) / d3::LD_C), most = delta_blocks(a.T, a.Hk, a.Hv, DK);
  d3::LdChunkArgs c = {a, 0, 0, workspace, nullptr};
  for (; c.block0 < all; c.block0 += most) {
    c.blocks = all - c.block0 < most ? all - c.block0 : most;
    c.heads = (char*)workspace + (size_t)c.blocks * a.Hk * sizeof(d3::LdRows<DK>);
    if (int st = launch(d3::lines_delta_prep_kernel<TYPE, DK, DELTA>, dim3(c.blocks, a.Hv), dim3(d3::LD_PREP_THREADS), prep_smem, s,
                        true, c))
      return st;
    // four teams of one warp a CTA where that gives every SM one, else two of two (B200, 16 / 32 heads of 128, us in a graph, the former / the
    // latter: 8192 tokens of one line 670 / 473, 16 texts of up to 192 tokens 132 / 151). Lines without tokens count: how many have some is
    // known on the GPU alone.
    const long long wide = (long long)a.B * a.Hv * ((a.Dv + 63) / 64);
    if (int st = wide >= d.sms ? scan_launch<TYPE, DK, DELTA, 4, 1>(vmap, c, s) : scan_launch<TYPE, DK, DELTA, 2, 2>(vmap, c, s))
      return st;
  }
  return D3_OK;
}

template <int TYPE, int DK>
int delta_launch(const d3::LdArgs& a, void* workspace, const DeviceInfo& d, cudaStream_t s) {
  if (!delta_steps(a.T, a.B))
    return a.beta ? chunk_launch<TYPE, DK, true>(a, workspace, d, s) : chunk_launch<TYPE, DK, false>(a, workspace, d, s);
  constexpr int rows = d3::LS_WARPS * d3::LS_ROWS * (128 / DK);
  const dim3 blocks((a.Dv + rows - 1) / rows, a.Hv, a.B + 1), threads(d3::LS_WARPS * 32);
  return a.beta ? launch(d3::lines_delta_step_kernel<TYPE, DK, true>, blocks, threads, 0, s, true, a)
                : launch(d3::lines_delta_step_kernel<TYPE, DK, false>, blocks, threads, 0, s, true, a);
}

bool multiple(const int64_t* st, int n, int64_t of) {
  for (int i = 0; i < n; ++i)
    if (st[i] % of) return false;
  return true;
}

bool row_type(int type) { return type >= d3::QR_BF16 && type <= d3::QR_F32; }

}  // namespace

extern "C" {

int d3_gated_norm(const void* x, const int64_t* x_strides, const void* gate, const int64_t* gate_strides, int type, int T,
                  int H, int D, const void* weight, int w_f32, float w_add, float eps, int act, void* out, void* stream) {
  if (!row_type(type) || T < 0 || H < 1 || D < 1 || (long long)T * H > (1ll << 31) || act < 0 || act > 1 || !(eps >= 0.0f))
    return D3_ERR_ARG;
  if (T == 0) return D3_OK;
  if (!x || !x_strides || !gate || !gate_strides || !weight || !out) return D3_ERR_ARG;
  const int size = type == d3::QR_F32 ? 4 : 2;
  if (!aligned(x, size) || !aligned(gate, size) || !aligned(out, size) || !aligned(weight, w_f32 ? 4 : size))
    return D3_ERR_ALIGN;
  DeviceInfo d;
  if (int st = device_info(&d)) return st;
  const d3::GnArgs a = {{x, x_strides[0], x_strides[1]}, {gate, gate_strides[0], gate_strides[1]}, T, H, D, weight, w_f32,
                        w_add, eps, act, out};
  const bool vectors = aligned(x, 16) && aligned(gate, 16) && aligned(out, 16) && aligned(weight, 16) &&
                       multiple(x_strides, 2, 16 / size) && multiple(gate_strides, 2, 16 / size);
  cudaStream_t s = (cudaStream_t)stream;
  switch (type) {
    case d3::QR_BF16: return gated_type<d3::QR_BF16>(a, vectors, d, s);
    case d3::QR_F16: return gated_type<d3::QR_F16>(a, vectors, d, s);
    default: return gated_type<d3::QR_F32>(a, vectors, d, s);
  }
}

int d3_add_norm(const void* x, int64_t x_token, const void* residual, int64_t r_token, int type, int T, int W,
                const void* weight, const void* post, int w_f32, float w_add, const void* gate, int64_t gate_token,
                int gate_kind, float scale, float eps, void* sum_out, void* norm_out, void* stream) {
  if (!row_type(type) || T < 0 || W < 1 || gate_kind < d3::AN_NONE || gate_kind > d3::AN_EACH || !(eps >= 0.0f))
    return D3_ERR_ARG;
  if (T == 0) return D3_OK;
  if (!x || !residual || !weight || (gate_kind && !gate) || !sum_out || !norm_out) return D3_ERR_ARG;
  const int size = type == d3::QR_F32 ? 4 : 2, wsize = w_f32 ? 4 : size;
  if (!aligned(x, size) || !aligned(residual, size) || !aligned(gate, size) || !aligned(sum_out, size) ||
      !aligned(norm_out, size) || !aligned(weight, wsize) || !aligned(post, wsize))
    return D3_ERR_ALIGN;
  DeviceInfo d;
  if (int st = device_info(&d)) return st;
  const d3::AnArgs a = {x, residual, x_token, r_token, T, W, weight, post, w_f32, w_add, eps, scale, gate, gate_token,
                        gate_kind, sum_out, norm_out};
  const int64_t strides[3] = {x_token, r_token, gate_kind == d3::AN_EACH ? gate_token : 0};
  const bool vectors = aligned(x, 16) && aligned(residual, 16) && (gate_kind != d3::AN_EACH || aligned(gate, 16)) &&
                       aligned(weight, 16) && aligned(post, 16) && aligned(sum_out, 16) && aligned(norm_out, 16) &&
                       multiple(strides, 3, 16 / size);
  cudaStream_t s = (cudaStream_t)stream;
  switch (type) {
    case d3::QR_BF16: return join_type<d3::QR_BF16>(a, vectors, d, s);
    case d3::QR_F16: return join_type<d3::QR_F16>(a, vectors, d, s);
    default: return join_type<d3::QR_F32>(a, vectors, d, s);
  }
}

int d3_lines_conv(const void* x, int64_t x_token, int type, int T, int C, const void* weight, const void* bias, int W,
                  int w_f32, void* state, const int* cu, const int* line, int B, int silu, void* out, void* stream) {
  if (!row_type(type) || T < 0 || C < 1 || W < 2 || W > d3::LC_MAX_TAPS || B < 1 || B > kMaxLines ||
      (long long)C * W > 0x7fffffffLL)
    return D3_ERR_ARG;
  if (T == 0) return D3_OK;
  if (!x || !weight || !state || !cu || !line || !out) return D3_ERR_ARG;
  const int size = type == d3::QR_F32 ? 4 : 2, wsize = w_f32 ? 4 : size;
  if (!aligned(x, size) || !aligned(state, size) || !aligned(out, size) || !aligned(weight, wsize) || !aligned(bias, wsize))
    return D3_ERR_ALIGN;
  DeviceInfo d;
  if (int st = device_info(&d)) return st;
  d3::LcArgs a = {x, x_token, T, C, W, B, weight, bias, w_f32, state, cu, line, silu, out, 0};
  a.tiles = (T + d3::LC_TILE - 1) / d3::LC_TILE;
  const int vec = 16 / size;
  const bool vectors = C % vec == 0 && x_token % vec == 0 && aligned(x, 16) && aligned(state, 16) && aligned(out, 16) &&
                       aligned(weight, 16);
  cudaStream_t s = (cudaStream_t)stream;
  switch (type) {
    case d3::QR_BF16: return conv_type<d3::QR_BF16>(a, vectors, s);
    case d3::QR_F16: return conv_type<d3::QR_F16>(a, vectors, s);
    default: return conv_type<d3::QR_F32>(a, vectors, s);
  }
}

size_t d3_lines_delta_workspace(int T, int B, int Hk, int Hv, int Dk) {
  if (T < 1 || Hk < 1 || Hv < 1 || delta_steps(T, B)) return 0;
  return delta_blocks(T, Hk, Hv, Dk) * delta_block_bytes(Hk, Hv, Dk);
}

int d3_lines_delta(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v,
                   const int64_t* v_strides, int type, int T, int Hk, int Hv, int Dk, int Dv, const void* decay,
                   int64_t decay_token, const void* beta, int64_t beta_token, int gates_f32, const float* a_log,
                   const float* dt_bias, float eps, float scale, float* state, const int* cu, const int* line, int B,
                   void* out, void* workspace, size_t workspace_bytes, void* stream) {
  if ((type != d3::QR_BF16 && type != d3::QR_F16) || T < 0 || Hk < 1 || Hv < Hk || Hv % Hk || Hv > 65535 ||
      (Dk != 64 && Dk != 128) || Dv < 16 || Dv > 256 || Dv % 16 || B < 1 || B > kMaxLines || !(scale > 0.0f) ||
      !(scale < 1e30f) || eps != eps)
    return D3_ERR_ARG;
  if (T == 0) return D3_OK;
  if (!q || !q_strides || !k || !k_strides || !v || !v_strides || !decay || !state || !cu || !line || !out) return D3_ERR_ARG;
  const int gsize = gates_f32 ? 4 : 2;
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 16) || !aligned(state, 16) ||
      !aligned(workspace, 128) || !aligned(decay, gsize) || !aligned(beta, gsize) || !aligned(a_log, 4) || !aligned(dt_bias, 4) ||
      !multiple(q_strides, 2, 8) || !multiple(k_strides, 2, 8) || !multiple(v_strides, 2, 8))
    return D3_ERR_ALIGN;
  const size_t need = d3_lines_delta_workspace(T, B, Hk, Hv, Dk);
  if (need && !workspace) return D3_ERR_ARG;
  if (workspace_bytes < need) return D3_ERR_WORKSPACE;
  for (int i = 0; i < 2; ++i)
    if (q_strides[i] < 0 || k_strides[i] < 0 || v_strides[i] < 1) return D3_ERR_ARG;
  DeviceInfo d;
  if (int st = device_info(&d)) return st;
  const d3::LdArgs a = {{q, q_strides[0], q_strides[1]}, {k, k_strides[0], k_strides[1]}, {v, v_strides[0], v_strides[1]},
                        T, B, Hk, Hv, Dk, Dv, decay, beta, decay_token, beta_token, gates_f32, a_log, dt_bias, eps, scale,
                        state, cu, line, out};
  cudaStream_t s = (cudaStream_t)stream;
  const bool f16 = type == d3::QR_F16;
  if (Dk == 64)
    return f16 ? delta_launch<d3::QR_F16, 64>(a, workspace, d, s) : delta_launch<d3::QR_BF16, 64>(a, workspace, d, s);
  return f16 ? delta_launch<d3::QR_F16, 128>(a, workspace, d, s) : delta_launch<d3::QR_BF16, 128>(a, workspace, d, s);
}

}  // extern "C"
