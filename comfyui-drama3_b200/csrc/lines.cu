// C ABI of the attention half of a decoder layer (declared in include/drama3_b200.h): the plan of a pass over a paged
// key/value cache, the norms and rotation of queries and keys with the cache write, and the attention of lines that
// share a prefix. Same conventions as drama3_b200.cu: arguments are checked before anything is launched, nothing is
// allocated, nothing synchronizes.
#include "host.cuh"
#include "lines_attn.cuh"
#include "lines_plan.cuh"
#include "qk_rope.cuh"

using namespace d3host;

// This translation unit's fault word (each has its own), read and cleared for d3_take_fault.
int d3_lines_take_fault(unsigned int* fault) {
  unsigned int v = 0, zero = 0;
  if (int st = cuda_status(cudaMemcpyFromSymbol(&v, d3::g_fault, sizeof(v)))) return st;
  *fault = v;
  return cuda_status(cudaMemcpyToSymbol(d3::g_fault, &zero, sizeof(zero)));
}

namespace {

// A cache [pages, page, heads, D] of 16-bit values as a 4-D map (column, key in page, head, page), read in boxes of 64
// columns x `box` keys of one head.
bool cache_map(CUtensorMap* map, bool f16, const void* base, int D, int heads, int page, int pages, const int64_t* st,
               int box) {
  cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)page, (cuuint64_t)heads, (cuuint64_t)pages};
  cuuint64_t strides[3] = {(cuuint64_t)st[1] * 2, (cuuint64_t)st[2] * 2, (cuuint64_t)st[0] * 2};
  cuuint32_t boxes[4] = {64, (cuuint32_t)box, 1, 1};
  return encode_tiled(map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, base, dims, strides,
                      boxes, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Queries [T, heads, D] as a 3-D map (column, head, token), read in boxes of 64 columns x the heads of a KV head x the
// tokens of a unit.
bool query_map(CUtensorMap* map, bool f16, const void* base, int D, int heads, int T, const int64_t* st, int group) {
  cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)T};
  cuuint64_t strides[2] = {(cuuint64_t)st[1] * 2, (cuuint64_t)st[0] * 2};
  cuuint32_t boxes[3] = {64, (cuuint32_t)group, (cuuint32_t)d3::la_tile_tokens(group)};
  return encode_tiled(map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, base, dims, strides,
                      boxes, CU_TENSOR_MAP_SWIZZLE_128B);
}

bool attn_shape(int T, int Hq, int Hkv, int D) {
  return T >= 0 && Hkv >= 1 && Hq >= Hkv && Hq % Hkv == 0 && Hq / Hkv <= d3::LA_ROWS &&
         (D == 64 || D == 128 || D == 256) && (long long)T * Hq <= 0x7fffffffLL - 1024;
}

template <int D, bool F16>
int attn_launch(const CUtensorMap& qm, const CUtensorMap& km, const CUtensorMap& vm, const d3::LaArgs& a, int join_blocks,
                cudaStream_t s) {
  constexpr int smem = d3::LaShape<D>::SMEM;
  static std::atomic<uint64_t> done{0};
  if (int st = allow_smem_once(d3::lines_attn_kernel<D, F16>, smem, done)) return st;
  if (int st = launch(d3::lines_attn_kernel<D, F16>, dim3(a.runs), dim3(d3::LA_THREADS), smem, s, true, qm, km, vm, a))
    return st;
  return launch(d3::lines_join_kernel<D, F16>, dim3(join_blocks), dim3(d3::LJ_WARPS * 32), 0, s, true, a);
}

template <int TYPE, int LANES>
int rope_launch(const d3::QrArgs& a, int pairs, int blocks, cudaStream_t s) {
  const dim3 threads(d3::QR_WARPS * 32);
  const size_t smem = (size_t)a.tokens * (a.rot / 2) * sizeof(float2);  // at most 4 x 256 x 8 bytes
  return pairs ? launch(d3::qk_rope_kernel<TYPE, LANES, true>, dim3(blocks), threads, smem, s, true, a)
               : launch(d3::qk_rope_kernel<TYPE, LANES, false>, dim3(blocks), threads, smem, s, true, a);
}

template <int TYPE>
int rope_type(d3::QrArgs a, int pairs, bool vectors, const DeviceInfo& d, cudaStream_t s) {
  constexpr int VEC = TYPE == d3::QR_F32 ? 4 : 8;
  const int slots = a.D / (2 * VEC);  // of two vectors: a lane each
  const int lanes = slots <= 4 ? 4 : slots <= 8 ? 8 : slots <= 16 ? 16 : 32;
  // vectors in twos need rows, strides and pointers of whole vectors, and turned columns and others in whole slots
  if (!vectors || a.D % (2 * VEC) || slots > 32 || a.rot % (2 * VEC)) {
    const long long warps = (long long)a.T * (a.Hq + a.Hkv * (a.k_out ? 1 : 2));
    return launch(d3::qk_rope_any_kernel<TYPE>, dim3((unsigned)((warps + d3::QR_WARPS - 1) / d3::QR_WARPS)),
                  dim3(d3::QR_WARPS * 32), 0, s, true, a, pairs);
  }
  // a warp per token where that fills the GPU (16 warps per SM), several with fewer tokens
  const int at_once = 32 / lanes, want = (16 * d.sms + a.T - 1) / a.T;
  const int most = (a.Hq + at_once - 1) / at_once + (a.Hkv + at_once - 1) / at_once * (a.k_out ? 1 : 2);
  a.share = want < most ? want : most;
  a.tokens = a.share < d3::QR_WARPS ? d3::QR_WARPS / a.share : 1;
  const int per = (a.share + d3::QR_WARPS - 1) / d3::QR_WARPS;
  const int blocks = per > 1 ? a.T * per : (a.T + a.tokens - 1) / a.tokens;
  switch (lanes) {
    case 4: return rope_launch<TYPE, 4>(a, pairs, blocks, s);
    case 8: return rope_launch<TYPE, 8>(a, pairs, blocks, s);
    case 16: return rope_launch<TYPE, 16>(a, pairs, blocks, s);
    default: return rope_launch<TYPE, 32>(a, pairs, blocks, s);
  }
}

bool multiple(const int64_t* st, int n, int64_t of) {
  for (int i = 0; i < n; ++i)
    if (st[i] % of) return false;
  return true;
}

}  // namespace

extern "C" {

size_t d3_lines_plan_ints(int B, int T, int group) {
  if (B < 1 || B > d3::LP_MAX_LINES || T < 0 || group < 1 || group > d3::LA_ROWS) return 0;
  return d3::la_unit_offset(T) + d3::LA_UNIT_INTS * (size_t)d3::la_max_units(B, T, group);
}

int d3_lines_plan(const int* kept, const int* counts, int B, int* table, int W, const int* free_pages, int F,
                  const int* used, const int* prefix, int page, int T, int group, int64_t* slots, int64_t* positions,
                  int* line, int* cu, int* lengths, int* used_out, int* work, size_t work_ints, void* stream) {
  if (B < 1 || B > d3::LP_MAX_LINES || W < 1 || F < 0 || page < 1 || T < 0 || group < 1 || group > d3::LA_ROWS ||
      (long long)T * group > d3::LP_MAX_TOKENS)
    return D3_ERR_ARG;
  if (!kept || !counts || !table || (F > 0 && !free_pages) || !used || !cu || !lengths || !used_out || !work ||
      (T > 0 && (!slots || !positions || !line)))
    return D3_ERR_ARG;
  if (!aligned(work, 16) || !aligned(slots, 8) || !aligned(positions, 8)) return D3_ERR_ALIGN;
  if (work_ints < d3_lines_plan_ints(B, T, group)) return D3_ERR_WORKSPACE;
  DeviceInfo d;
  if (int st = device_info(&d)) return st;
  const int smem = 4 * (B + 1) * 4;
  // asked for whatever B is: 48 KB hold the kernel's own static arrays too, so the limit is below 48 KB of these
  static std::atomic<uint64_t> done{0};
  if (int st = allow_smem_once(d3::lines_plan_kernel, 4 * (d3::LP_MAX_LINES + 1) * 4, done)) return st;
  const d3::LinesPlanArgs a = {kept, counts, B, table, W, free_pages, F, used, prefix, page, T, group, slots, positions,
                               line, cu, lengths, used_out, work};
  return launch(d3::lines_plan_kernel, dim3(1 + (T + d3::LP_TOKENS - 1) / d3::LP_TOKENS), dim3(d3::LP_THREADS), smem,
                (cudaStream_t)stream, true, a);
}

int d3_qk_norm_rope(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v,
                    const int64_t* v_strides, int type, int T, int Hq, int Hkv, int D, const void* q_weight,
                    const void* k_weight, int w_f32, float w_add, float eps, const float* rotary, int rot, int length,
                    const int64_t* positions, int axes, const uint8_t* axis, int pairs, void* q_out, void* k_out,
                    void* k_cache, const int64_t* kc_strides, void* v_cache, const int64_t* vc_strides, int pages,
                    int page, const int64_t* slots, void* stream) {
  if (type < 0 || type > 2 || T < 0 || Hq < 1 || Hkv < 1 || D < 1 || D > d3::QR_MAX_D || rot < 0 || rot > D || rot % 2 ||
      axes < 1 || axes > d3::QR_MAX_AXES || length < 0 || !(eps >= 0.0f))
    return D3_ERR_ARG;
  if ((long long)T * (Hq + 2 * (long long)Hkv) > (1ll << 31)) return D3_ERR_ARG;
  if (T == 0) return D3_OK;
  if (!q || !q_strides || !k || !k_strides || !q_out || (rot > 0 && (!rotary || !positions)) || (axes > 1 && !axis))
    return D3_ERR_ARG;
  const bool cache = k_out == nullptr;
  if (cache && (!v || !v_strides || !k_cache || !kc_strides || !v_cache || !vc_strides || !slots || pages < 1 || page < 1))
    return D3_ERR_ARG;
  const int size = type == d3::QR_F32 ? 4 : 2;
  if (!aligned(q, size) || !aligned(k, size) || !aligned(q_out, size) || !aligned(rotary, 8) || !aligned(positions, 8) ||
      (cache ? !aligned(v, size) || !aligned(k_cache, size) || !aligned(v_cache, size) : !aligned(k_out, size)))
    return D3_ERR_ALIGN;
  DeviceInfo d;
  if (int st = device_info(&d)) return st;
  d3::QrArgs a = {};
  a.q = {q, q_strides[0], q_strides[1]};
  a.k = {k, k_strides[0], k_strides[1]};
  a.T = T, a.Hq = Hq, a.Hkv = Hkv, a.D = D;
  a.qw = q_weight, a.kw = k_weight, a.w_f32 = w_f32, a.w_add = w_add, a.eps = eps;
  a.rotary = (const float2*)rotary, a.rot = rot, a.length = length, a.pos = positions, a.axes = axes;
  a.axis = axis;
  a.q_out = q_out, a.k_out = k_out, a.share = 1;
  const int64_t vec = 16 / size;
  bool vectors = aligned(q, 16) && aligned(k, 16) && aligned(q_out, 16) && aligned(q_weight, 16) &&
                 aligned(k_weight, 16) && multiple(q_strides, 2, vec) &&
                 multiple(k_strides, 2, vec);
  if (cache) {
    a.v = {v, v_strides[0], v_strides[1]};
    a.kc = {k_cache, kc_strides[0], kc_strides[1], kc_strides[2]};
    a.vc = {v_cache, vc_strides[0], vc_strides[1], vc_strides[2]};
    a.slots = slots, a.page = page, a.slot_count = (long long)pages * page;
    vectors = vectors && aligned(v, 16) && aligned(k_cache, 16) && aligned(v_cache, 16) && multiple(v_strides, 2, vec) &&
              multiple(kc_strides, 3, vec) && multiple(vc_strides, 3, vec);
  } else {
    vectors = vectors && aligned(k_out, 16);
  }
  cudaStream_t s = (cudaStream_t)stream;
  switch (type) {
    case d3::QR_BF16: return rope_type<d3::QR_BF16>(a, pairs, vectors, d, s);
    case d3::QR_F16: return rope_type<d3::QR_F16>(a, pairs, vectors, d, s);
    default: return rope_type<d3::QR_F32>(a, pairs, vectors, d, s);
  }
}

size_t d3_lines_attention_workspace(int T, int Hq, int Hkv, int D) {
  DeviceInfo d;
  if (!attn_shape(T, Hq, Hkv, D) || device_info(&d)) return 0;
  const long long rows = d3::la_part_rows(d.sms, T, Hq / Hkv, Hkv);
  return (size_t)rows * (D + 2) * 4 + (size_t)d.sms * 16;
}

int d3_lines_attention(const void* q, const int64_t* q_strides, int type, int T, int Hq, int Hkv, int D,
                       const void* k_cache, const int64_t* kc_strides, const void* v_cache, const int64_t* vc_strides,
                       int pages, int page, const int* table, int W, const int* prefix_table, int PW, const int* work,
                       int B, float scale, void* out, float* lse, void* workspace,
                       size_t workspace_bytes, void* stream) {
  if ((type != d3::QR_BF16 && type != d3::QR_F16) || !attn_shape(T, Hq, Hkv, D) || pages < 1 ||
      !(page == 16 || page == 32 || (page >= 64 && page % 64 == 0)) || (long long)pages * page > 0x7fffffffLL || W < 1 ||
      PW < 0 || B < 1 || B > d3::LP_MAX_LINES || !(scale > 0.0f) || !(scale < 1e30f))
    return D3_ERR_ARG;
  if (T == 0) return D3_OK;
  if (!q || !q_strides || !k_cache || !kc_strides || !v_cache || !vc_strides || !table || (PW > 0 && !prefix_table) ||
      !work || !out || !workspace)
    return D3_ERR_ARG;
  for (int i = 0; i < 3; ++i)
    if (kc_strides[i] < 1 || vc_strides[i] < 1 || (i < 2 && q_strides[i] < 1)) return D3_ERR_ARG;
  if (!aligned(q, 16) || !aligned(k_cache, 16) || !aligned(v_cache, 16) || !aligned(out, 16) || !aligned(workspace, 16) ||
      !aligned(work, 16) || !multiple(q_strides, 2, 8) || !multiple(kc_strides, 3, 8) || !multiple(vc_strides, 3, 8))
    return D3_ERR_ALIGN;
  DeviceInfo d;
  if (int st = device_info(&d)) return st;
  if (workspace_bytes < d3_lines_attention_workspace(T, Hq, Hkv, D)) return D3_ERR_WORKSPACE;
  const bool f16 = type == d3::QR_F16;
  // a box is as many keys of a page as a tile can hold
  const int box = page % d3::LA_KEYS == 0 ? d3::LA_KEYS : page < 64 ? page : 64;
  CUtensorMap qm, km, vm;
  if (!query_map(&qm, f16, q, D, Hq, T, q_strides, Hq / Hkv) ||
      !cache_map(&km, f16, k_cache, D, Hkv, page, pages, kc_strides, box) ||
      !cache_map(&vm, f16, v_cache, D, Hkv, page, pages, vc_strides, box))
    return D3_ERR_ARG;
  d3::LaArgs a = {};
  a.T = T, a.Hq = Hq, a.Hkv = Hkv, a.G = Hq / Hkv;
  a.pages = pages, a.page = page, a.page_box = box;
  a.table = table, a.W = W, a.prefix_table = prefix_table, a.PW = PW;
  a.work = work, a.B = B;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.out = out, a.lse = lse;
  a.runs = d.sms;
  const long long rows = d3::la_part_rows(a.runs, T, a.G, Hkv);
  a.part_o = (float4*)workspace;
  a.part_ml = (float2*)((float*)workspace + rows * D);
  a.joints = (int4*)(a.part_ml + rows);
  a.units_most = (int)d3::la_max_units(B, T, a.G);
  // the joining kernel: a block per run, or enough for a warp per 32 rows x 4 columns that may have parts
  const long long tasks = (long long)T * a.G <= d3::LA_APART_ROWS ? d3::la_apart_rows(T, a.G) / 32 * Hkv * (D / 4) : 0;
  const long long want = (tasks + d3::LJ_WARPS - 1) / d3::LJ_WARPS, most = 16ll * d.sms;
  const int blocks = (int)(want < a.runs ? a.runs : want < most ? want : most);
  cudaStream_t s = (cudaStream_t)stream;
  switch (D) {
    case 64: return f16 ? attn_launch<64, true>(qm, km, vm, a, blocks, s) : attn_launch<64, false>(qm, km, vm, a, blocks, s);
    case 128: return f16 ? attn_launch<128, true>(qm, km, vm, a, blocks, s) : attn_launch<128, false>(qm, km, vm, a, blocks, s);
    default: return f16 ? attn_launch<256, true>(qm, km, vm, a, blocks, s) : attn_launch<256, false>(qm, km, vm, a, blocks, s);
  }
}

}  // extern "C"
