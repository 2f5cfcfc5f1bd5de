// Attention over the paged KV pool under masks other than the causal one: a
// tree of drafted tokens, and a sliding window with sinks.
#include <algorithm>
#include <cfloat>
#include <initializer_list>

#include <cuda_bf16.h>

#include "npl_common.cuh"

namespace npl {
namespace {

struct MaArgs {
  const void* q;
  void* out;
  const void* k;
  const void* v;
  long long ld_q, ld_out;  // elements between tokens
  const int32_t* bt;
  long long bt_stride;
  const int32_t* ctx_lens;
  const int32_t* q_lens;     // null: one token of each sequence
  const int32_t* q_offsets;  // null with q_lens
  const uint8_t* mask;       // tree: [total_q, mask_cols]
  long long ld_mask;
  int mask_cols;
  int window, sinks;
  int B, H, Hkv, G, num_blocks, block_size, max_blocks, total_q, max_q_len;
  float scale;
  int* status;
};

__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_float(__half* p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void from_float(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// One warp for each (sequence, token, head): keys one after the other, the
// head dimension over the lanes.
template <typename T, int D, bool kTree>
__global__ void __launch_bounds__(128) masked_attn_simple(const MaArgs p) {
  const int b = blockIdx.y, h = blockIdx.z * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (h >= p.H) return;
  const int n = p.q_lens ? p.q_lens[b] : 1, start = p.q_offsets ? p.q_offsets[b] : b, ctx = p.ctx_lens[b];
  if (n <= 0) return;
  if (start < 0 || start > p.total_q - n || n > p.max_q_len) {
    atomicCAS(p.status, 0, NPL_DEV_BAD_INDEX);
    return;
  }
  const int prefix = ctx - n, kvh = h / p.G;
  for (int j = blockIdx.x; j < n; j += gridDim.x) {
    constexpr int E = D / 32;
    float q[E], acc[E], m = -INFINITY, l = 0.f;
    const T* qp = static_cast<const T*>(p.q) + (start + j) * p.ld_q + (long long)h * D + lane * E;
    for (int e = 0; e < E; ++e) q[e] = to_float(qp[e]) * p.scale, acc[e] = 0.f;
    const int pos = prefix + j, end = kTree ? ctx : min(ctx, pos + 1);
    if (prefix < 0 && ctx != 0) atomicCAS(p.status, 0, NPL_DEV_BAD_INDEX);
    for (int i = 0; i < (prefix < 0 ? 0 : end); ++i) {
      if (kTree) {
        const int c = i - prefix;
        if (c >= 0 && (c >= p.mask_cols || !p.mask[(start + j) * p.ld_mask + c])) continue;
      } else if (i <= pos - p.window && i >= p.sinks) {
        i = pos - p.window;
        continue;
      }
      const int page = i / p.block_size;
      const int blk = page < p.max_blocks ? p.bt[b * p.bt_stride + page] : -1;
      float s = 0.f, x[E];
      const bool ok = blk >= 0 && blk < p.num_blocks;
      const long long row = ok ? (((long long)blk * p.block_size + i % p.block_size) * p.Hkv + kvh) * D + lane * E : 0;
      if (!ok) atomicCAS(p.status, 0, NPL_DEV_BAD_INDEX);
      for (int e = 0; e < E; ++e) s += ok ? q[e] * to_float(static_cast<const T*>(p.k)[row + e]) : 0.f;
      for (int e = 0; e < E; ++e) x[e] = ok ? to_float(static_cast<const T*>(p.v)[row + e]) : 0.f;
      s = warp_sum(s);
      const float mn = fmaxf(m, s), base = mn == -INFINITY ? 0.f : mn;
      const float a = expf(m - base), w = expf(s - base);
      m = mn;
      l = l * a + w;
      for (int e = 0; e < E; ++e) acc[e] = acc[e] * a + w * x[e];
    }
    T* op = static_cast<T*>(p.out) + (start + j) * p.ld_out + (long long)h * D + lane * E;
    for (int e = 0; e < E; ++e) from_float(op + e, l == 0.f ? 0.f : acc[e] / l);
  }
}

template <typename T, int D, bool kTree>
int launch(const char* what, const MaArgs& p, cudaStream_t st) {
  masked_attn_simple<T, D, kTree><<<dim3(std::min(p.max_q_len, 65535), p.B, (p.H + 3) / 4), 128, 0, st>>>(p);
  return launch_status(what);
}

template <bool kTree>
int run(const char* what, const MaArgs& p, int dtype, int D, cudaStream_t st) {
  if (dtype == NPL_F16) return D == 128 ? launch<__half, 128, kTree>(what, p, st) : launch<__half, 64, kTree>(what, p, st);
  return D == 128 ? launch<__nv_bfloat16, 128, kTree>(what, p, st) : launch<__nv_bfloat16, 64, kTree>(what, p, st);
}

int check(const char* what, const MaArgs& p, int dtype, int D) {
  if (dtype != NPL_F16 && dtype != NPL_BF16)
    return fail(NPL_ERR_ARG, "%s: element type %d (NPL_F16 or NPL_BF16)", what, dtype);
  if (!p.q || !p.k || !p.v || !p.bt || !p.ctx_lens || !p.out) return fail(NPL_ERR_ARG, "%s: null pointer", what);
  if (!p.q_lens != !p.q_offsets) return fail(NPL_ERR_ARG, "%s: q_lens and q_offsets go together", what);
  if (p.total_q < 0 || p.B < 0 || p.max_q_len < 0 || p.H <= 0 || p.Hkv <= 0 || p.H % p.Hkv || p.num_blocks <= 0 ||
      p.block_size <= 0 || p.max_blocks <= 0 || p.bt_stride < p.max_blocks)
    return fail(NPL_ERR_ARG, "%s: bad shape", what);
  if (!p.q_lens && p.B != p.total_q)
    return fail(NPL_ERR_ARG, "%s: without q_lens every sequence has one token (%d sequences, %d tokens)", what, p.B,
                p.total_q);
  if (D != 128 && D != 64) return fail(NPL_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128)", what, D);
  if (p.ld_q < (long long)p.H * D || p.ld_out < (long long)p.H * D || p.ld_q % 8 || p.ld_out % 8)
    return fail(NPL_ERR_ARG, "%s: token strides must be multiples of 8 and hold all heads", what);
  if (!(p.scale > 0.f) || !(p.scale < 3.0e38f))
    return fail(NPL_ERR_ARG, "%s: scale must be positive and finite", what);
  if (p.block_size % 8) return fail(NPL_ERR_UNSUPPORTED, "%s: block_size %d (a multiple of 8)", what, p.block_size);
  if (p.G > 128) return fail(NPL_ERR_UNSUPPORTED, "%s: %d query heads for each kv head (at most 128)", what, p.G);
  if (p.B > 65535) return fail(NPL_ERR_UNSUPPORTED, "%s: %d sequences (at most 65535)", what, p.B);
  if ((long long)p.num_blocks * p.block_size >= (1ll << 31) - 256 ||
      (long long)p.max_blocks * p.block_size >= (1ll << 31) - 256 || p.total_q >= (1 << 30))
    return fail(NPL_ERR_UNSUPPORTED, "%s: pool, table or batch too large for 32-bit rows", what);
  for (const void* x : std::initializer_list<const void*>{p.q, p.k, p.v, p.out})
    if (!aligned16(x)) return fail(NPL_ERR_ARG, "%s: pointers must be 16-byte aligned", what);
  return NPL_OK;
}

}  // namespace
}  // namespace npl

using namespace npl;

extern "C" int npl_paged_tree_attention(const void* q, int dtype, int64_t ld_q, int total_q, int H, int Hkv, int D,
                                        const void* k_cache, const void* v_cache, int num_blocks, int block_size,
                                        const int32_t* block_tables, int64_t bt_stride, int max_blocks,
                                        const int32_t* context_lens, const int32_t* q_lens, const int32_t* q_offsets,
                                        int B, int max_q_len, const uint8_t* tree_mask, int64_t ld_mask,
                                        int mask_cols, float scale, void* out, int64_t ld_out, void* stream) {
  const char* what = "npl_paged_tree_attention";
  MaArgs p{};
  p.q = q, p.out = out, p.k = k_cache, p.v = v_cache, p.ld_q = ld_q, p.ld_out = ld_out, p.bt = block_tables;
  p.bt_stride = bt_stride, p.ctx_lens = context_lens, p.q_lens = q_lens, p.q_offsets = q_offsets;
  p.mask = tree_mask, p.ld_mask = ld_mask, p.mask_cols = mask_cols;
  p.B = B, p.H = H, p.Hkv = Hkv, p.G = Hkv > 0 ? H / Hkv : 0, p.num_blocks = num_blocks, p.block_size = block_size;
  p.max_blocks = max_blocks, p.total_q = total_q, p.max_q_len = max_q_len, p.scale = scale;
  if (int rc = check(what, p, dtype, D)) return rc;
  if (!tree_mask || !q_lens) return fail(NPL_ERR_ARG, "%s: null pointer", what);
  if (mask_cols < max_q_len || ld_mask < mask_cols)
    return fail(NPL_ERR_ARG, "%s: the mask has %d columns (stride %lld) for up to %d drafts", what, mask_cols,
                (long long)ld_mask, max_q_len);
  if (int rc = check_device()) return rc;
  if (B == 0 || total_q == 0 || max_q_len == 0) return NPL_OK;
  p.status = device_status_ptr();
  return run<true>(what, p, dtype, D, static_cast<cudaStream_t>(stream));
}

extern "C" int npl_paged_window_attention(const void* q, int dtype, int64_t ld_q, int total_q, int H, int Hkv, int D,
                                          const void* k_cache, const void* v_cache, int num_blocks, int block_size,
                                          const int32_t* block_tables, int64_t bt_stride, int max_blocks,
                                          const int32_t* context_lens, const int32_t* q_lens,
                                          const int32_t* q_offsets, int B, int max_q_len, int window, int sinks,
                                          float scale, void* out, int64_t ld_out, void* stream) {
  const char* what = "npl_paged_window_attention";
  MaArgs p{};
  p.q = q, p.out = out, p.k = k_cache, p.v = v_cache, p.ld_q = ld_q, p.ld_out = ld_out, p.bt = block_tables;
  p.bt_stride = bt_stride, p.ctx_lens = context_lens, p.q_lens = q_lens, p.q_offsets = q_offsets;
  p.window = window, p.sinks = sinks;
  p.B = B, p.H = H, p.Hkv = Hkv, p.G = Hkv > 0 ? H / Hkv : 0, p.num_blocks = num_blocks, p.block_size = block_size;
  p.max_blocks = max_blocks, p.total_q = total_q, p.max_q_len = q_lens ? max_q_len : 1, p.scale = scale;
  if (int rc = check(what, p, dtype, D)) return rc;
  if (window < 1 || sinks < 0)
    return fail(NPL_ERR_ARG, "%s: window %d (at least 1), sinks %d (at least 0)", what, window, sinks);
  if (int rc = check_device()) return rc;
  if (B == 0 || total_q == 0 || p.max_q_len == 0) return NPL_OK;
  p.status = device_status_ptr();
  return run<false>(what, p, dtype, D, static_cast<cudaStream_t>(stream));
}
