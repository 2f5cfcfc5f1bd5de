// Block-scaled e4m3 quantisers of the fp8 layer path: plain rows, fused
// (residual add +) RMSNorm, SiLU * up, and 128 x 128 weight blocks.
//
// One fp32 scale per block: 128 consecutive columns of a token, or a 128 x
// 128 tile of a weight (the last ones may be partial). With a = max |v| over
// the block's values v,
//   s = max(a / 448, 2^-126)         (448 = the largest finite e4m3 value;
//                                     2^-126 = the smallest normal fp32)
//   q = e4m3(v * (1 / s))            (fp32 steps, one rounding each; q s ~ v)
// The values v are kept in fp32 from the inputs to the codes (RMSNorm and
// SiLU * up included): the only rounding to fewer bits is the code itself. v / s
// differs from v * (1 / s) by at most 1.5 fp32 ulps, 2^-19 of a code step, and
// |v| (1 / s) <= 448 (1 + 2^-22), which rounds to 448, so nothing saturates
// that should not. The max propagates NaN: a block that holds a NaN or an
// infinity gets a non-finite scale, and all its values read back as NaN.
//
// Every kernel is one pass over its input: the block stays in registers
// between the maximum and the codes, 8 columns a thread, 16 threads a block.
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <algorithm>

#include "npl_common.cuh"

namespace npl {
namespace {

constexpr int kBlock = 128;       // columns (and weight rows) per scale
constexpr int kVecCols = 8;       // columns per thread
constexpr int kGroup = kBlock / kVecCols;  // threads per block of a row
constexpr float kE4m3Max = 448.0f;
constexpr float kScaleMin = 0x1p-126f;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// 8 consecutive elements as they lie in memory.
template <typename T>
struct alignas(16) Raw8 {
  T e[8];
};

// The first n of 8 consecutive elements at p (zeros after them). kVec: p is
// 16-byte aligned, and 8 elements are loaded at once.
template <bool kVec, typename T>
__device__ __forceinline__ Raw8<T> load8(const T* p, int n) {
  Raw8<T> r;
  if (kVec && n >= 8) {
    const uint4* s = reinterpret_cast<const uint4*>(p);
    uint4* d = reinterpret_cast<uint4*>(&r);
#pragma unroll
    for (int i = 0; i < (int)sizeof(Raw8<T>) / 16; ++i) d[i] = s[i];
    return r;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) r.e[i] = i < n ? p[i] : T(0.0f);
  return r;
}

template <typename T>
__device__ __forceinline__ void widen8(const Raw8<T>& r, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = to_f32(r.e[i]);
}

// max that returns NaN when either operand is NaN (fmaxf drops it)
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float absmax8(const float (&v)[8]) {
  float a = fabsf(v[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) a = max_nan(a, fabsf(v[i]));
  return a;
}

// Over the 16 lanes that share a block; every lane receives the result.
__device__ __forceinline__ float group_max(float a) {
#pragma unroll
  for (int o = kGroup / 2; o > 0; o >>= 1) a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, o));
  return a;
}

__device__ __forceinline__ float block_scale(float absmax) {
  return max_nan(__fdiv_rn(absmax, kE4m3Max), kScaleMin);
}

__device__ __forceinline__ uint2 codes8(const float (&v)[8], float inv) {
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const __nv_fp8x2_storage_t lo = __nv_cvt_float2_to_fp8x2(
        make_float2(__fmul_rn(v[4 * h], inv), __fmul_rn(v[4 * h + 1], inv)), __NV_SATFINITE, __NV_E4M3);
    const __nv_fp8x2_storage_t hi = __nv_cvt_float2_to_fp8x2(
        make_float2(__fmul_rn(v[4 * h + 2], inv), __fmul_rn(v[4 * h + 3], inv)), __NV_SATFINITE, __NV_E4M3);
    w[h] = (uint32_t)lo | ((uint32_t)hi << 16);
  }
  return make_uint2(w[0], w[1]);
}

// Stores the first n of 8 codes; kVecQ: dst is 8-byte aligned.
template <bool kVecQ>
__device__ __forceinline__ void store_codes(uint8_t* dst, uint2 q, int n) {
  if (kVecQ && n >= 8) {
    *reinterpret_cast<uint2*>(dst) = q;
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) dst[i] = (uint8_t)((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
}

// Where the quantised values come from.
template <typename T, bool kVec>
struct RowSource {  // the row itself
  using Raw = Raw8<T>;
  const T* x;
  long long ldx;
  __device__ __forceinline__ Raw load(int row, int col, int n) const { return load8<kVec>(x + row * ldx + col, n); }
  __device__ __forceinline__ static void values(const Raw& r, float (&v)[8]) { widen8(r, v); }
};

template <typename T, bool kVec>
struct SiluSource {  // silu(gate) * up = gate / (1 + e^-gate) * up, fp32
  struct Raw {
    Raw8<T> g, u;
  };
  const T* gate;
  const T* up;
  long long ld_gate, ld_up;
  __device__ __forceinline__ Raw load(int row, int col, int n) const {
    return {load8<kVec>(gate + row * ld_gate + col, n), load8<kVec>(up + row * ld_up + col, n)};
  }
  __device__ __forceinline__ static void values(const Raw& r, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float g = to_f32(r.g.e[i]);
      v[i] = __fmul_rn(__fdiv_rn(g, __fadd_rn(1.0f, expf(-g))), to_f32(r.u.e[i]));
    }
  }
};

struct CodeSink {
  uint8_t* q;
  long long ldq;
  float* scale;
  long long ld_scale;
};

constexpr int kQuantThreads = 256;
constexpr int kUnroll = 4;  // blocks per 16-thread group
constexpr int kNormThreads = 512;

// Blocks are numbered row by row; a CTA takes 16 * kUnroll consecutive ones.
template <typename Source, bool kVecQ>
__global__ void __launch_bounds__(kQuantThreads) fp8_quant_kernel(const Source src, const CodeSink out, int rows,
                                                                  int cols, int k_blocks) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x % kGroup, group = threadIdx.x / kGroup;
  constexpr int kGroups = kQuantThreads / kGroup;
  const unsigned total = (unsigned)rows * (unsigned)k_blocks;
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const unsigned item = (blockIdx.x * kUnroll + u) * kGroups + group;
    const bool in = item < total;
    const int row = in ? (int)(item / (unsigned)k_blocks) : 0;
    const int kb = (int)(item - (unsigned)row * (unsigned)k_blocks);
    const int col = kb * kBlock + lane * kVecCols;
    const int n = in ? min(8, max(0, cols - col)) : 0;
    const typename Source::Raw raw = src.load(row, n > 0 ? col : 0, n);
    float v[8];
    Source::values(raw, v);
    const float s = block_scale(group_max(absmax8(v)));
    const uint2 q = codes8(v, __frcp_rn(s));
    if (n > 0) store_codes<kVecQ>(out.q + row * out.ldq + col, q, n);
    if (in && lane == 0) out.scale[row * out.ld_scale + kb] = s;
  }
}

// (x + residual) -> RMSNorm -> codes; one CTA per row. kChunks > 0: the row
// stays in registers, kChunks * 8 columns a thread; 0: any length, the row is
// read again for the second half.
template <typename T, int kChunks, bool kVec, bool kVecQ>
__global__ void __launch_bounds__(kNormThreads)
    fp8_rmsnorm_kernel(const T* x, long long ldx, const T* res, long long ld_res, const T* __restrict__ w, float eps,
                       int cols, T* sum_out, long long ld_sum, const CodeSink out) {  // sum_out may be x or res
  __shared__ float red[32];
  pdl_wait();
  pdl_trigger();
  const long long row = blockIdx.x;
  const int step = (int)blockDim.x * kVecCols;
  const int chunks = kChunks > 0 ? kChunks : (cols + step - 1) / step;
  constexpr int kKeep = kChunks > 0 ? kChunks : 1;
  float keep[kKeep][8];
  float ss = 0.f;
  auto one = [&](int c, float(&v)[8]) {
    const int col = c * step + (int)threadIdx.x * kVecCols;
    const int n = min(8, max(0, cols - col));
    const int at = n > 0 ? col : 0;
    widen8(load8<kVec>(x + row * ldx + at, n), v);
    if (res) {
      float r[8];
      widen8(load8<kVec>(res + row * ld_res + at, n), r);
      Raw8<T> t;
#pragma unroll
      for (int i = 0; i < 8; ++i) {  // rounded as it is stored: the norm is that of the stored sum
        t.e[i] = from_f32<T>(__fadd_rn(v[i], r[i]));
        v[i] = to_f32(t.e[i]);
      }
      if (kVec && n >= 8) {
        *reinterpret_cast<uint4*>(sum_out + row * ld_sum + col) = *reinterpret_cast<const uint4*>(&t);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < n) sum_out[row * ld_sum + col + i] = t.e[i];
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = __fmaf_rn(v[i], v[i], ss);
  };
  if constexpr (kChunks > 0) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) one(c, keep[c]);
  } else {
    for (int c = 0; c < chunks; ++c) one(c, keep[0]);
  }
  ss = block_sum(ss, red);
  const float r = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(ss, (float)cols), eps)));
  // The second reading takes the stored sum where there is one: it may have
  // replaced x or the residual.
  const T* again = res ? sum_out + row * ld_sum : x + row * ldx;
#pragma unroll
  for (int c = 0; c < chunks; ++c) {
    const int col = c * step + (int)threadIdx.x * kVecCols;
    const int n = min(8, max(0, cols - col));
    const int at = n > 0 ? col : 0;
    float v[8], wv[8];
    widen8(load8<kVec>(w + at, n), wv);
    if constexpr (kChunks > 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = keep[c][i];
    } else {
      widen8(load8<kVec>(again + at, n), v);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(__fmul_rn(v[i], r), wv[i]);
    const float s = block_scale(group_max(absmax8(v)));
    const uint2 q = codes8(v, __frcp_rn(s));
    if (n > 0) {
      store_codes<kVecQ>(out.q + row * out.ldq + col, q, n);
      if (threadIdx.x % kGroup == 0) out.scale[row * out.ld_scale + col / kBlock] = s;
    }
  }
}

// One 128 x 128 weight block per CTA: 16 threads across, 16 rows at a time,
// the block held in registers between its maximum and its codes.
constexpr int kWeightRows = kQuantThreads / kGroup;

template <typename T, bool kVec, bool kVecQ>
__global__ void __launch_bounds__(kQuantThreads) fp8_quant_weight_kernel(const T* __restrict__ w, long long ldw,
                                                                         int rows, int cols, const CodeSink out) {
  __shared__ float red[32];
  pdl_wait();
  constexpr int kSteps = kBlock / kWeightRows;
  const int nb = blockIdx.x, kb = blockIdx.y;
  const int col = kb * kBlock + (int)(threadIdx.x % kGroup) * kVecCols;
  const int n = min(8, max(0, cols - col));
  const int row0 = nb * kBlock + (int)threadIdx.x / kGroup;
  Raw8<T> raw[kSteps];
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int row = row0 + i * kWeightRows;
    const bool in = row < rows && n > 0;
    raw[i] = load8<kVec>(w + (in ? (long long)row * ldw + col : 0), in ? n : 0);
  }
  float a = 0.f;
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    float v[8];
    widen8(raw[i], v);
    a = max_nan(a, absmax8(v));
  }
  a = group_max(a);
  a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, 16));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = a;
  __syncthreads();
  a = red[0];
#pragma unroll
  for (int i = 1; i < kQuantThreads / 32; ++i) a = max_nan(a, red[i]);
  const float s = block_scale(a);
  const float inv = __frcp_rn(s);
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int row = row0 + i * kWeightRows;
    float v[8];
    widen8(raw[i], v);
    if (row < rows && n > 0) store_codes<kVecQ>(out.q + (long long)row * out.ldq + col, codes8(v, inv), n);
  }
  if (threadIdx.x == 0) out.scale[(long long)nb * out.ld_scale + kb] = s;
  pdl_trigger_after_writes();
}

// ------------------------------------------------------------------ host
constexpr long long kMaxInt = 2147483647ll;

int elem_size(int dtype) { return dtype == NPL_F32 ? 4 : 2; }

// Whether all rows, `ld` elements apart from `p` on, start on 16-byte boundaries.
bool vec_rows(const void* p, long long rows, long long ld, int dtype) {
  return aligned16(p) && (rows == 1 || (ld * elem_size(dtype)) % 16 == 0);
}

int check_codes(const char* what, long long rows, long long cols, const void* q, long long ldq, const void* scale,
                long long ld_scale) {
  if (rows < 0 || cols <= 0 || rows > kMaxInt - kBlock || cols > kMaxInt - kBlock)
    return fail(NPL_ERR_ARG, "%s: bad shape rows=%lld cols=%lld", what, rows, cols);
  const long long kb = (cols + kBlock - 1) / kBlock;
  if (ldq < cols || ld_scale < kb)
    return fail(NPL_ERR_ARG, "%s: ldq=%lld (>= %lld) or ld_scale=%lld (>= %lld) too small", what, ldq, cols, ld_scale,
                kb);
  if (rows > 0 && (!q || !scale)) return fail(NPL_ERR_ARG, "%s: null pointer", what);
  if (reinterpret_cast<uintptr_t>(scale) & 3u) return fail(NPL_ERR_ARG, "%s: scale must be 4-byte aligned", what);
  return NPL_OK;
}

int check_input(const char* what, const char* name, const void* p, int dtype, bool f32_ok, long long rows,
                long long cols, long long ld) {
  if (dtype != NPL_F16 && dtype != NPL_BF16 && !(f32_ok && dtype == NPL_F32))
    return fail(NPL_ERR_ARG, "%s: element type %d (NPL_F16%s or NPL_BF16)", what, dtype, f32_ok ? ", NPL_F32" : "");
  if (rows > 0 && !p) return fail(NPL_ERR_ARG, "%s: null pointer (%s)", what, name);
  if (rows > 1 && ld < cols) return fail(NPL_ERR_ARG, "%s: row stride of %s %lld < %lld columns", what, name, ld, cols);
  if (reinterpret_cast<uintptr_t>(p) % elem_size(dtype))
    return fail(NPL_ERR_ARG, "%s: %s is not aligned to its elements", what, name);
  return NPL_OK;
}

template <typename Fn>
int by_type(int dtype, Fn&& fn) {
  if (dtype == NPL_F32) return fn(float());
  if (dtype == NPL_F16) return fn(__half());
  return fn(__nv_bfloat16());
}

bool vec_codes(const CodeSink& o) {
  return (reinterpret_cast<uintptr_t>(o.q) & 7u) == 0 && o.ldq % 8 == 0;
}

template <typename Source>
int launch_quant(const char* what, const Source& src, const CodeSink& out, int rows, int cols, cudaStream_t st) {
  const long long kb = (cols + kBlock - 1) / kBlock;
  const long long total = rows * kb;
  if (total > kMaxInt) return fail(NPL_ERR_UNSUPPORTED, "%s: %lld blocks (at most 2^31 - 1)", what, total);
  constexpr int per_cta = kQuantThreads / kGroup * kUnroll;
  const dim3 grid((unsigned)((total + per_cta - 1) / per_cta));
  return launch_pdl(what, vec_codes(out) ? fp8_quant_kernel<Source, true> : fp8_quant_kernel<Source, false>, grid,
                    dim3(kQuantThreads), 0, st, src, out, rows, cols, (int)kb);
}

template <typename T, bool kVec, bool kVecQ>
int launch_rmsnorm(const T* x, long long ldx, const T* res, long long ld_res, const T* w, float eps, int rows,
                   int cols, T* sum_out, long long ld_sum, const CodeSink& out, cudaStream_t st) {
  const int lanes = (cols + kVecCols - 1) / kVecCols;
  const int threads = std::min(kNormThreads, (lanes + 31) / 32 * 32);
  const int chunks = (lanes + threads - 1) / threads;
  auto kern = chunks <= 1   ? fp8_rmsnorm_kernel<T, 1, kVec, kVecQ>
              : chunks <= 2 ? fp8_rmsnorm_kernel<T, 2, kVec, kVecQ>
              : chunks <= 4 ? fp8_rmsnorm_kernel<T, 4, kVec, kVecQ>
                            : fp8_rmsnorm_kernel<T, 0, kVec, kVecQ>;
  return launch_pdl("npl_fp8_rmsnorm_quant", kern, dim3((unsigned)rows), dim3((unsigned)threads), 0, st, x, ldx, res,
                    ld_res, w, eps, cols, sum_out, ld_sum, out);
}

}  // namespace
}  // namespace npl

using namespace npl;

extern "C" int npl_fp8_quant_rows(const void* x, int x_dtype, int64_t rows, int64_t cols, int64_t ldx, uint8_t* q,
                                  int64_t ldq, float* scale, int64_t ld_scale, void* stream) {
  const char* what = "npl_fp8_quant_rows";
  if (int rc = check_codes(what, rows, cols, q, ldq, scale, ld_scale)) return rc;
  if (int rc = check_input(what, "x", x, x_dtype, true, rows, cols, ldx)) return rc;
  if (rows == 0) return NPL_OK;
  if (int rc = check_device()) return rc;
  const CodeSink out{q, ldq, scale, ld_scale};
  return by_type(x_dtype, [&](auto t) {
    using T = decltype(t);
    const T* p = static_cast<const T*>(x);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (vec_rows(x, rows, ldx, x_dtype))
      return launch_quant(what, RowSource<T, true>{p, ldx}, out, (int)rows, (int)cols, st);
    return launch_quant(what, RowSource<T, false>{p, ldx}, out, (int)rows, (int)cols, st);
  });
}

extern "C" int npl_fp8_silu_mul_quant(const void* gate, int64_t ld_gate, const void* up, int64_t ld_up, int dtype,
                                      int64_t rows, int64_t cols, uint8_t* q, int64_t ldq, float* scale,
                                      int64_t ld_scale, void* stream) {
  const char* what = "npl_fp8_silu_mul_quant";
  if (int rc = check_codes(what, rows, cols, q, ldq, scale, ld_scale)) return rc;
  if (int rc = check_input(what, "gate", gate, dtype, false, rows, cols, ld_gate)) return rc;
  if (int rc = check_input(what, "up", up, dtype, false, rows, cols, ld_up)) return rc;
  if (rows == 0) return NPL_OK;
  if (int rc = check_device()) return rc;
  const CodeSink out{q, ldq, scale, ld_scale};
  auto go = [&](auto t) {
    using T = decltype(t);
    const T* g = static_cast<const T*>(gate);
    const T* u = static_cast<const T*>(up);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (vec_rows(gate, rows, ld_gate, dtype) && vec_rows(up, rows, ld_up, dtype))
      return launch_quant(what, SiluSource<T, true>{g, u, ld_gate, ld_up}, out, (int)rows, (int)cols, st);
    return launch_quant(what, SiluSource<T, false>{g, u, ld_gate, ld_up}, out, (int)rows, (int)cols, st);
  };
  return dtype == NPL_F16 ? go(__half()) : go(__nv_bfloat16());
}

extern "C" int npl_fp8_rmsnorm_quant(const void* x, int64_t ldx, const void* residual, int64_t ld_res,
                                     const void* weight, int dtype, float eps, int64_t rows, int64_t cols,
                                     void* sum_out, int64_t ld_sum, uint8_t* q, int64_t ldq, float* scale,
                                     int64_t ld_scale, void* stream) {
  const char* what = "npl_fp8_rmsnorm_quant";
  if (int rc = check_codes(what, rows, cols, q, ldq, scale, ld_scale)) return rc;
  if (int rc = check_input(what, "x", x, dtype, false, rows, cols, ldx)) return rc;
  if (int rc = check_input(what, "weight", weight, dtype, false, 1, cols, cols)) return rc;
  if (!residual != !sum_out) return fail(NPL_ERR_ARG, "%s: residual and sum_out go together", what);
  if (residual) {
    if (int rc = check_input(what, "residual", residual, dtype, false, rows, cols, ld_res)) return rc;
    if (int rc = check_input(what, "sum_out", sum_out, dtype, false, rows, cols, ld_sum)) return rc;
  }
  if (rows == 0) return NPL_OK;
  if (int rc = check_device()) return rc;
  const CodeSink out{q, ldq, scale, ld_scale};
  const bool vec = vec_rows(x, rows, ldx, dtype) && aligned16(weight) &&
                   (!residual || (vec_rows(residual, rows, ld_res, dtype) && vec_rows(sum_out, rows, ld_sum, dtype)));
  const bool vecq = vec_codes(out);
  auto go = [&](auto t) {
    using T = decltype(t);
    auto* fn = vec ? (vecq ? launch_rmsnorm<T, true, true> : launch_rmsnorm<T, true, false>)
                   : (vecq ? launch_rmsnorm<T, false, true> : launch_rmsnorm<T, false, false>);
    return fn(static_cast<const T*>(x), ldx, static_cast<const T*>(residual), ld_res, static_cast<const T*>(weight),
              eps, (int)rows, (int)cols, static_cast<T*>(sum_out), ld_sum, out, static_cast<cudaStream_t>(stream));
  };
  return dtype == NPL_F16 ? go(__half()) : go(__nv_bfloat16());
}

extern "C" int npl_fp8_quant_weight(const void* w, int w_dtype, int64_t rows, int64_t cols, int64_t ldw, uint8_t* q,
                                    int64_t ldq, float* scale, int64_t ld_scale, void* stream) {
  const char* what = "npl_fp8_quant_weight";
  if (int rc = check_codes(what, rows, cols, q, ldq, scale, ld_scale)) return rc;
  if (int rc = check_input(what, "w", w, w_dtype, true, rows, cols, ldw)) return rc;
  if (rows == 0) return NPL_OK;
  if (int rc = check_device()) return rc;
  const long long nb = (rows + kBlock - 1) / kBlock, kb = (cols + kBlock - 1) / kBlock;
  if (kb > 65535) return fail(NPL_ERR_UNSUPPORTED, "%s: %lld columns (at most 65535 blocks)", what, (long long)cols);
  const CodeSink out{q, ldq, scale, ld_scale};
  const bool vec = vec_rows(w, rows, ldw, w_dtype), vecq = vec_codes(out);
  return by_type(w_dtype, [&](auto t) {
    using T = decltype(t);
    auto kern = vec ? (vecq ? fp8_quant_weight_kernel<T, true, true> : fp8_quant_weight_kernel<T, true, false>)
                    : (vecq ? fp8_quant_weight_kernel<T, false, true> : fp8_quant_weight_kernel<T, false, false>);
    return launch_pdl(what, kern, dim3((unsigned)nb, (unsigned)kb), dim3(kQuantThreads), 0,
                      static_cast<cudaStream_t>(stream), static_cast<const T*>(w), ldw, (int)rows, (int)cols, out);
  });
}
