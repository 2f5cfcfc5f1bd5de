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

// max |v| is taken on the bit patterns without their sign: they order like the
// magnitudes, an infinity above every number and a NaN above infinity, so a
// NaN is never lost. A key is such a pattern, of fp32 or of a 16-bit type.
template <typename T>
__device__ __forceinline__ float key_value(uint32_t key);
template <>
__device__ __forceinline__ float key_value<float>(uint32_t key) { return __uint_as_float(key); }
template <>
__device__ __forceinline__ float key_value<__half>(uint32_t key) {
  return __half2float(__ushort_as_half((unsigned short)key));
}
template <>
__device__ __forceinline__ float key_value<__nv_bfloat16>(uint32_t key) { return __uint_as_float(key << 16); }

__device__ __forceinline__ uint32_t key8(const float (&v)[8]) {
  uint32_t a = __float_as_uint(v[0]) & 0x7fffffffu;
#pragma unroll
  for (int i = 1; i < 8; ++i) a = max(a, __float_as_uint(v[i]) & 0x7fffffffu);
  return a;
}

template <typename T>
__device__ __forceinline__ uint32_t key8(const Raw8<T>& r) {
  if constexpr (sizeof(T) == 4) {
    return key8(r.e);
  } else {  // two 16-bit patterns at a time
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
    const uint32_t m = __vmaxu2(__vmaxu2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu),
                                __vmaxu2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu));
    return max(m & 0xffffu, m >> 16);
  }
}

__device__ __forceinline__ uint32_t max_xor(uint32_t own, uint32_t sent, int o) {
  return max(own, __shfl_xor_sync(0xffffffffu, sent, o));
}

// The largest key of U blocks (1, 2 or 4) over the 16 lanes that share them.
// Halving the blocks with each exchange costs 4, 4 or 5 shuffles instead of
// 4 U, and leaves lane l with block own_block<U>(l), whose scale it then works
// out for the other lanes too.
template <int U>
__device__ __forceinline__ int own_block(int lane) { return U == 4 ? (lane >> 2) & 3 : U == 2 ? (lane >> 3) & 1 : 0; }

template <int U>
__device__ __forceinline__ uint32_t block_key(const uint32_t (&k)[U], int lane) {
  uint32_t m;
  if constexpr (U == 4) {
    const bool hi = lane & 8, mid = lane & 4;
    const uint32_t a = max_xor(hi ? k[2] : k[0], hi ? k[0] : k[2], 8);
    const uint32_t b = max_xor(hi ? k[3] : k[1], hi ? k[1] : k[3], 8);
    m = max_xor(mid ? b : a, mid ? a : b, 4);
  } else if constexpr (U == 2) {
    const bool hi = lane & 8;
    m = max_xor(hi ? k[1] : k[0], hi ? k[0] : k[1], 8);
    m = max_xor(m, m, 4);
  } else {
    m = max_xor(k[0], k[0], 8);
    m = max_xor(m, m, 4);
  }
  m = max_xor(m, m, 2);
  return max_xor(m, m, 1);
}

// Block u's value of `v`, held by the lanes whose own_block is u.
template <int U>
__device__ __forceinline__ float from_block(float v, int u) {
  return U == 1 ? v : __shfl_sync(0xffffffffu, v, (int)(threadIdx.x & 16) + u * (kGroup / U));
}

__device__ __forceinline__ float block_scale(float absmax) {
  // absmax >= 0 or NaN: the comparison keeps a NaN
  const float s = __fdiv_rn(absmax, kE4m3Max);
  return s < kScaleMin ? kScaleMin : s;
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

// Where the quantised values come from: what a thread loads for its 8 columns,
// what it keeps of them, their key and the fp32 values.
template <typename T, bool kVec>
struct RowSource {  // the row itself
  using Elem = T;
  using Raw = Raw8<T>;
  using Kept = Raw8<T>;
  const T* x;
  long long ldx;
  __device__ __forceinline__ Raw load(int row, int col, int n) const { return load8<kVec>(x + row * ldx + col, n); }
  __device__ __forceinline__ static Kept keep(const Raw& r) { return r; }
  __device__ __forceinline__ static uint32_t key(const Kept& k) { return key8(k); }
  __device__ __forceinline__ static void values(const Kept& k, float (&v)[8]) { widen8(k, v); }
};

// silu(g) up = g / (1 + e^-g) up in fp32. With t = e^-|g| <= 1 it is
// (g < 0 ? g t : g) / (1 + t): nothing overflows, and 1 + t in [1, 2] has a
// fast reciprocal (1 ulp) without special cases.
template <typename T, bool kVec>
struct SiluSource {
  using Elem = float;
  struct Raw {
    Raw8<T> g, u;
  };
  struct Kept {
    float v[8];
  };
  const T* gate;
  const T* up;
  long long ld_gate, ld_up;
  __device__ __forceinline__ Raw load(int row, int col, int n) const {
    return {load8<kVec>(gate + row * ld_gate + col, n), load8<kVec>(up + row * ld_up + col, n)};
  }
  __device__ __forceinline__ static Kept keep(const Raw& r) {
    Kept k;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float g = to_f32(r.g.e[i]);
      const float t = expf(-fabsf(g));
      float inv;
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(__fadd_rn(1.0f, t)));
      const float num = g >= 0.f ? g : __fmul_rn(g, t);
      k.v[i] = __fmul_rn(__fmul_rn(num, inv), to_f32(r.u.e[i]));
    }
    return k;
  }
  __device__ __forceinline__ static uint32_t key(const Kept& k) { return key8(k.v); }
  __device__ __forceinline__ static void values(const Kept& k, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k.v[i];
  }
};

struct CodeSink {
  uint8_t* q;
  long long ldq;
  float* scale;
  long long ld_scale;
};

constexpr int kQuantThreads = 256;
constexpr int kNormThreads = 1024;

// A warp takes 2 U consecutive blocks of a row, each of its two 16-lane groups
// every other one, all loads before the first store, which the compiler would
// not move them across. The bound on registers keeps 24 to 40 warps, and 80 KB
// of loads or more, in flight on an SM.
template <typename Source, int U, bool kVecQ>
__global__ void __launch_bounds__(kQuantThreads, sizeof(typename Source::Raw) > 16 ? 3 : 5)
    fp8_quant_kernel(const Source src, const CodeSink out, int rows, int cols, unsigned spans) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x % kGroup;
  const unsigned item = blockIdx.x * (kQuantThreads / 32) + (threadIdx.x >> 5);  // (row, span of 2 U blocks)
  const int row = (int)(item / spans);
  if (row >= rows) return;  // whole warps
  const int kb0 = (int)(item - (unsigned)row * spans) * (2 * U) + (int)(threadIdx.x & 31) / kGroup;
  const int col0 = kb0 * kBlock + lane * kVecCols;
  typename Source::Raw raw[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int col = col0 + u * (2 * kBlock);
    raw[u] = src.load(row, col < cols ? col : 0, cols - col);
  }
  typename Source::Kept kept[U];
  uint32_t key[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    kept[u] = Source::keep(raw[u]);
    key[u] = Source::key(kept[u]);
  }
  const float s = block_scale(key_value<typename Source::Elem>(block_key<U>(key, lane)));
  const float inv = __frcp_rn(s);
  {
    const int kb = kb0 + 2 * own_block<U>(lane);
    if (lane % (kGroup / U) == 0 && kb * kBlock < cols) out.scale[row * out.ld_scale + kb] = s;
  }
  uint8_t* q = out.q + row * out.ldq;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const float inv_u = from_block<U>(inv, u);
    const int col = col0 + u * (2 * kBlock);
    float v[8];
    Source::values(kept[u], v);
    if (col < cols) store_codes<kVecQ>(q + col, codes8(v, inv_u), cols - col);
  }
}

// (x + residual) -> RMSNorm -> codes; one CTA per row. kChunks > 0: the row
// stays in registers as T, kChunks * 8 columns a thread; 0: any length, the
// row is read again for the second half.
template <typename T, int kChunks, bool kVec, bool kVecQ>
__global__ void __launch_bounds__(kNormThreads)
    fp8_rmsnorm_kernel(const T* x, long long ldx, const T* res, long long ld_res, const T* __restrict__ w, float eps,
                       int cols, T* sum_out, long long ld_sum, const CodeSink out) {  // sum_out may be x or res
  __shared__ float red[32];
  pdl_wait();
  pdl_trigger();
  const long long row = blockIdx.x;
  const int lane = threadIdx.x % kGroup;
  const int step = (int)blockDim.x * kVecCols;
  constexpr int kKeep = kChunks > 0 ? kChunks : 1;
  Raw8<T> keep[kKeep], other[kKeep];
  float ss = 0.f;
  // the sum as it is stored, and its squares: the norm is that of the stored sum
  auto add = [&](int col, Raw8<T>& t, const Raw8<T>& r) {
    const int n = cols - col;
    float v[8];
    widen8(t, v);
    if (res) {
      float rv[8];
      widen8(r, rv);
#pragma unroll
      for (int i = 0; i < 8; ++i) t.e[i] = from_f32<T>(__fadd_rn(v[i], rv[i]));
      widen8(t, v);
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
  auto fetch = [&](const T* p, long long ld, int col) {
    return load8<kVec>(p + row * ld + (col < cols ? col : 0), cols - col);
  };
  const int col0 = (int)threadIdx.x * kVecCols;
  if constexpr (kChunks > 0) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      keep[c] = fetch(x, ldx, col0 + c * step);
      if (res) other[c] = fetch(res, ld_res, col0 + c * step);
    }
#pragma unroll
    for (int c = 0; c < kChunks; ++c) add(col0 + c * step, keep[c], other[c]);
  } else {
    for (int col = col0; col < cols; col += step) {
      keep[0] = fetch(x, ldx, col);
      if (res) other[0] = fetch(res, ld_res, col);
      add(col, keep[0], other[0]);
    }
  }
  if constexpr (kChunks > 0) {  // the norm's weights, on their way while the sums are joined
#pragma unroll
    for (int c = 0; c < kChunks; ++c) other[c] = fetch(w, 0, col0 + c * step);
  }
  ss = warp_sum(ss);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = ss;
  __syncthreads();
  ss = warp_sum((threadIdx.x & 31) < (blockDim.x >> 5) ? red[threadIdx.x & 31] : 0.f);
  const float r = rsqrtf(__fadd_rn(__fdividef(ss, (float)cols), eps));  // both within 2 ulps
  // kChunks blocks at a time; the second reading takes the stored sum where
  // there is one: it may have replaced x or the residual
  for (int base = 0; base < cols; base += kKeep * step) {
    float v[kKeep][8];
    uint32_t key[kKeep];
#pragma unroll
    for (int c = 0; c < kKeep; ++c) {
      if constexpr (kChunks == 0) {
        keep[0] = res ? fetch(sum_out, ld_sum, base + col0) : fetch(x, ldx, base + col0);
        other[0] = fetch(w, 0, base + col0);
      }
      float wv[8];
      widen8(keep[c], v[c]);
      widen8(other[c], wv);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[c][i] = __fmul_rn(__fmul_rn(v[c][i], r), wv[i]);
      key[c] = key8(v[c]);
    }
    const float s = block_scale(__uint_as_float(block_key<kKeep>(key, lane)));
    const float inv = __frcp_rn(s);
#pragma unroll
    for (int c = 0; c < kKeep; ++c) {
      const float inv_c = from_block<kKeep>(inv, c);
      const int col = base + col0 + c * step;
      if (col < cols) store_codes<kVecQ>(out.q + row * out.ldq + col, codes8(v[c], inv_c), cols - col);
      if (lane == c * (kGroup / kKeep) && col - lane * kVecCols < cols)
        out.scale[row * out.ld_scale + col / kBlock] = s;
    }
  }
}

// One 128 x 128 weight block per CTA: 16 threads across, 32 rows at a time,
// the block held in registers between its maximum and its codes.
constexpr int kWeightThreads = 512;
constexpr int kWeightRows = kWeightThreads / kGroup;

template <typename T, bool kVec, bool kVecQ>
__global__ void __launch_bounds__(kWeightThreads) fp8_quant_weight_kernel(const T* __restrict__ w, long long ldw,
                                                                         int rows, int cols, const CodeSink out) {
  __shared__ uint32_t red[kWeightThreads / 32];
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
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < kSteps; ++i) a = max(a, key8(raw[i]));
  a = __reduce_max_sync(0xffffffffu, a);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = a;
  __syncthreads();
  a = __reduce_max_sync(0xffffffffu, red[threadIdx.x & (kWeightThreads / 32 - 1)]);
  const float s = block_scale(key_value<T>(a));
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

template <typename Source, int U>
int launch_quant_spans(const char* what, const Source& src, const CodeSink& out, int rows, int cols, cudaStream_t st) {
  const long long spans = (cols + 2 * U * kBlock - 1) / (2 * U * kBlock);
  constexpr int per_cta = kQuantThreads / 32;
  const long long ctas = (rows * spans + per_cta - 1) / per_cta;
  if (ctas * per_cta > kMaxInt) return fail(NPL_ERR_UNSUPPORTED, "%s: rows=%d cols=%d is too large", what, rows, cols);
  return launch_pdl(what, vec_codes(out) ? fp8_quant_kernel<Source, U, true> : fp8_quant_kernel<Source, U, false>,
                    dim3((unsigned)ctas), dim3(kQuantThreads), 0, st, src, out, rows, cols, (unsigned)spans);
}

// Four blocks a thread, except where the rows are short (half of the warps'
// lanes or more would idle) or so few that one block a thread fits on the SMs
// at once (8 x 4096: X us against Y with four).
template <typename Source>
int launch_quant(const char* what, const Source& src, const CodeSink& out, int rows, int cols, cudaStream_t st) {
  const long long blocks = (long long)rows * ((cols + kBlock - 1) / kBlock);
  if (cols <= 4 * kBlock || blocks <= 64ll * num_sms()) return launch_quant_spans<Source, 1>(what, src, out, rows, cols, st);
  return launch_quant_spans<Source, 4>(what, src, out, rows, cols, st);
}

template <typename T, bool kVec, bool kVecQ>
int launch_rmsnorm(const T* x, long long ldx, const T* res, long long ld_res, const T* w, float eps, int rows,
                   int cols, T* sum_out, long long ld_sum, const CodeSink& out, cudaStream_t st) {
  // Few rows: one chunk a thread, the shortest way through a row. More rows
  // than run at once: two, which halves the share of the two barriers and of
  // the scales (16000 x 4096: X us against Y).
  const int lanes = (cols + kVecCols - 1) / kVecCols;
  const int want = lanes <= kNormThreads && rows <= 2 * num_sms() ? 1 : 2;
  const int threads = std::min(kNormThreads, (lanes + 32 * want - 1) / (32 * want) * 32);
  const int chunks = (lanes + threads - 1) / threads;
  auto kern = chunks <= 1   ? fp8_rmsnorm_kernel<T, 1, kVec, kVecQ>
              : chunks <= 2 ? fp8_rmsnorm_kernel<T, 2, kVec, kVecQ>
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
    return launch_pdl(what, kern, dim3((unsigned)nb, (unsigned)kb), dim3(kWeightThreads), 0,
                      static_cast<cudaStream_t>(stream), static_cast<const T*>(w), ldw, (int)rows, (int)cols, out);
  });
}
