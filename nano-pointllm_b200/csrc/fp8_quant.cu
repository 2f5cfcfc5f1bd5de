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
// between the maximum and the codes, 16 columns a thread, 8 threads a block.
// No input is __restrict__: a load that may take memory for constant could be
// moved ahead of the wait for the kernel that writes it.
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <type_traits>

#include "npl_common.cuh"

namespace npl {
namespace {

constexpr int kBlock = 128;       // columns (and weight rows) per scale
constexpr int kCols = 16;         // columns per thread
constexpr int kGroup = kBlock / kCols;  // threads per block of a row
constexpr float kE4m3Max = 448.0f;
constexpr float kScaleMin = 0x1p-126f;

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// 16 consecutive elements as they lie in memory.
template <typename T>
struct alignas(16) Raw {
  T e[kCols];
  static constexpr int kWords = kCols * (int)sizeof(T) / 4;
};

// How rows can be accessed: their alignment in bytes (32, 16, or that of an element).
enum Access { kElements = 0, kBy16 = 1, kBy32 = 2 };

__device__ __forceinline__ void ld32(const void* p, uint32_t* r) {  // one 256-bit load
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "l"(p));
}

// 16 consecutive elements at any p: the aligned 16-byte words around them,
// shifted into place. [lo, hi) bounds what may be read; false where the words
// do not lie in it. (Tokens 1000 x 5003 fp16: 4.5 us; element by element 7.7.)
template <typename T>
__device__ __forceinline__ bool load_shifted(const T* p, const T* lo, const T* hi, Raw<T>& r) {
  constexpr int W = Raw<T>::kWords;
  const uintptr_t at = reinterpret_cast<uintptr_t>(p);
  const uint32_t off = (uint32_t)at & 15u;
  const uint4* from = reinterpret_cast<const uint4*>(at - off);
  if (from < reinterpret_cast<const uint4*>(lo) || from + (W / 4 + 1) > reinterpret_cast<const uint4*>(hi)) return false;
  uint32_t w[W + 4];
#pragma unroll
  for (int i = 0; i < W / 4 + 1; ++i) {
    const uint4 x = from[i];
    w[4 * i] = x.x;
    w[4 * i + 1] = x.y;
    w[4 * i + 2] = x.z;
    w[4 * i + 3] = x.w;
  }
#pragma unroll
  for (int i = 0; i < W + 3; ++i) w[i] = off & 4 ? w[i + 1] : w[i];
#pragma unroll
  for (int i = 0; i < W + 1; ++i) w[i] = off & 8 ? w[i + 2] : w[i];
  uint32_t* out = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
  for (int i = 0; i < W; ++i) out[i] = sizeof(T) == 2 ? __funnelshift_r(w[i], w[i + 1], (off & 2) * 8) : w[i];
  return true;
}

// The first n of 16 consecutive elements at p (zeros after them) of a tensor
// that lies in [lo, hi).
template <int kAccess, typename T>
__device__ __forceinline__ Raw<T> load16(const T* p, int n, const T* lo, const T* hi) {
  Raw<T> r;
  if (kAccess != kElements && n >= kCols) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&r);
    if constexpr (kAccess == kBy32) {
#pragma unroll
      for (int i = 0; i < Raw<T>::kWords; i += 8) ld32(reinterpret_cast<const uint32_t*>(p) + i, w + i);
    } else {
#pragma unroll
      for (int i = 0; i < Raw<T>::kWords; i += 4)
        *reinterpret_cast<uint4*>(w + i) = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(p) + i);
    }
    return r;
  }
  if (kAccess == kElements && n >= kCols && load_shifted(p, lo, hi, r)) return r;
#pragma unroll
  for (int i = 0; i < kCols; ++i) r.e[i] = i < n ? p[i] : T(0.0f);
  return r;
}

// The first n of 16 elements; by16: p is 16-byte aligned.
template <typename T>
__device__ __forceinline__ void store16(T* p, const Raw<T>& r, int n, bool by16) {
  if (by16 && n >= kCols) {
    const uint4* w = reinterpret_cast<const uint4*>(&r);
#pragma unroll
    for (int i = 0; i < Raw<T>::kWords / 4; ++i) reinterpret_cast<uint4*>(p)[i] = w[i];
    return;
  }
#pragma unroll
  for (int i = 0; i < kCols; ++i)
    if (i < n) p[i] = r.e[i];
}

__device__ __forceinline__ void widen(const Raw<float>& r, float (&v)[kCols]) {
#pragma unroll
  for (int i = 0; i < kCols; ++i) v[i] = r.e[i];
}
__device__ __forceinline__ void widen(const Raw<__half>& r, float (&v)[kCols]) {
  const __half2* h = reinterpret_cast<const __half2*>(&r);
#pragma unroll
  for (int i = 0; i < kCols / 2; ++i) {
    const float2 f = __half22float2(h[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void widen(const Raw<__nv_bfloat16>& r, float (&v)[kCols]) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
#pragma unroll
  for (int i = 0; i < kCols / 2; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

// A key is max |v| as a bit pattern, of fp32 or of a 16-bit type. Patterns
// without a sign order like the magnitudes, an infinity above every number
// and a NaN above infinity; with the NaN-propagating max of a thread's own
// values a NaN is never lost.
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

__device__ __forceinline__ float max_abs(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)));
  return r;
}
__device__ __forceinline__ __half2 max_abs(__half2 a, __half2 b) { return __hmax2_nan(__habs2(a), __habs2(b)); }
__device__ __forceinline__ __nv_bfloat162 max_abs(__nv_bfloat162 a, __nv_bfloat162 b) {
  return __hmax2_nan(__habs2(a), __habs2(b));
}

template <typename V, int N>
__device__ __forceinline__ V max_abs_all(const V* v) {
  if constexpr (N == 1)
    return v[0];
  else
    return max_abs(max_abs_all<V, N / 2>(v), max_abs_all<V, N / 2>(v + N / 2));
}

__device__ __forceinline__ uint32_t key_of(const float (&v)[kCols]) {
  return __float_as_uint(max_abs_all<float, kCols>(v));
}

template <typename T>
__device__ __forceinline__ uint32_t key_of(const Raw<T>& r) {
  if constexpr (sizeof(T) == 4) {
    return key_of(r.e);
  } else {
    using Pair = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
    const Pair m = max_abs_all<Pair, kCols / 2>(reinterpret_cast<const Pair*>(&r));
    const uint32_t bits = *reinterpret_cast<const uint32_t*>(&m);
    return max(bits & 0xffffu, bits >> 16);
  }
}

__device__ __forceinline__ uint32_t max_xor(uint32_t own, uint32_t sent, int o) {
  return max(own, __shfl_xor_sync(0xffffffffu, sent, o));
}

// The largest key of U blocks (1 or 2) over the 8 lanes that share them. With
// two, half of the lanes go on with each after the first exchange: 3 shuffles
// instead of 6, and lane l is left with block own_block<U>(l), whose scale it
// works out for the other lanes too.
template <int U>
__device__ __forceinline__ int own_block(int lane) { return U == 2 ? (lane >> 2) & 1 : 0; }

template <int U>
__device__ __forceinline__ uint32_t block_key(const uint32_t (&k)[U], int lane) {
  uint32_t m;
  if constexpr (U == 2)
    m = max_xor(lane & 4 ? k[1] : k[0], lane & 4 ? k[0] : k[1], 4);
  else
    m = max_xor(k[0], k[0], 4);
  m = max_xor(m, m, 2);
  return max_xor(m, m, 1);
}

// Block u's value of `v`, held by the lanes whose own_block is u.
template <int U>
__device__ __forceinline__ float from_block(float v, int u) {
  return U == 1 ? v : __shfl_sync(0xffffffffu, v, (int)(threadIdx.x & 24) + u * (kGroup / U));
}

__device__ __forceinline__ float block_scale(float absmax) {
  // absmax >= 0 or NaN: the comparison keeps a NaN
  const float s = __fdiv_rn(absmax, kE4m3Max);
  return s < kScaleMin ? kScaleMin : s;
}

__device__ __forceinline__ uint4 codes16(const float (&v)[kCols], float inv) {
  uint32_t w[4];
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    const __nv_fp8x2_storage_t lo = __nv_cvt_float2_to_fp8x2(
        make_float2(__fmul_rn(v[4 * h], inv), __fmul_rn(v[4 * h + 1], inv)), __NV_SATFINITE, __NV_E4M3);
    const __nv_fp8x2_storage_t hi = __nv_cvt_float2_to_fp8x2(
        make_float2(__fmul_rn(v[4 * h + 2], inv), __fmul_rn(v[4 * h + 3], inv)), __NV_SATFINITE, __NV_E4M3);
    w[h] = (uint32_t)lo | ((uint32_t)hi << 16);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Stores the first n of 16 codes; kVecQ: dst is 16-byte aligned.
template <bool kVecQ>
__device__ __forceinline__ void store_codes(uint8_t* dst, uint4 q, int n) {
  if (kVecQ && n >= kCols) {
    *reinterpret_cast<uint4*>(dst) = q;
    return;
  }
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < kCols; ++i)
    if (i < n) dst[i] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
}

// Where the quantised values come from: what a thread loads for its columns,
// what it keeps of them, their key and the fp32 values. rework() works them out
// anew from the same columns, loaded again, for a warp that holds rare values;
// whether it did so is the same in all lanes.
template <typename T, int kAccess>
struct RowSource {  // the row itself
  using Elem = T;
  using Loaded = Raw<T>;
  using Kept = Raw<T>;
  const T* x;
  long long ldx;
  const T* end;
  __device__ __forceinline__ Loaded load(int row, int col, int n) const {
    return load16<kAccess>(x + row * ldx + col, n, x, end);
  }
  __device__ __forceinline__ static Kept keep(const Loaded& r) { return r; }
  __device__ __forceinline__ bool rework(int, int, int, Kept&) const { return false; }
  __device__ __forceinline__ static uint32_t key(const Kept& k) { return key_of(k); }
  __device__ __forceinline__ static void values(const Kept& k, float (&v)[kCols]) { widen(k, v); }
};

// silu(g) up = g / (1 + e^-g) up in fp32, within a few ulps. Below -87.3 the
// approximate reciprocal flushes to 0, and from -88.7 on e^-g overflows, although
// a large up makes such a product any size. For these far gates, where 1 + e^g is
// 1 in fp32, it is (g p) (p up) with p = e^(g / 2). Below -174 p is subnormal, off
// by 2^-150 at most, and the product by 2^-149 |g| p up: at scales of 2^-126 or
// more under 2^-13 in units of a code, whose smallest is 2^-9. A warp that holds
// one loads its columns again for it: 16000 x 11008 takes 205 us (bf16 210), 201
// without the question, 229 (239) with this formula for all gates, which needs
// no question, and 217 (232) with the columns kept until it is answered.
constexpr float kFarGate = -86.0f;

template <typename T, int kAccess>
struct SiluSource {
  using Elem = float;
  struct Loaded {
    Raw<T> g, u;
  };
  struct Kept {
    float v[kCols];
    bool far;
  };
  // Two of kFarGate. Patterns above it are those of numbers below it, and of NaNs with a sign.
  static constexpr uint32_t kFarBits = std::is_same_v<T, __half> ? 0xd560d560u : 0xc2acc2acu;
  const T* gate;
  const T* up;
  long long ld_gate, ld_up;
  const T *gate_end, *up_end;
  __device__ __forceinline__ Loaded load(int row, int col, int n) const {
    return {load16<kAccess>(gate + row * ld_gate + col, n, gate, gate_end),
            load16<kAccess>(up + row * ld_up + col, n, up, up_end)};
  }
  __device__ __forceinline__ static Kept keep(const Loaded& r) {
    Kept k;
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&r.g);
    uint32_t top = __vimax3_u16x2(w[0], w[1], w[2]);
    top = __vimax3_u16x2(top, w[3], w[4]);
    top = __vimax3_u16x2(top, w[5], w[6]);
    k.far = __vimax3_u16x2(top, w[7], kFarBits) != kFarBits;
    float up[kCols];
    widen(r.g, k.v);
    widen(r.u, up);
#pragma unroll
    for (int i = 0; i < kCols; ++i) {
      float sig;
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(sig) : "f"(__fadd_rn(1.0f, expf(-k.v[i]))));
      k.v[i] = __fmul_rn(__fmul_rn(k.v[i], sig), up[i]);
    }
    return k;
  }
  __device__ __forceinline__ bool rework(int row, int col, int n, Kept& k) const {
    if (!__any_sync(0xffffffffu, k.far)) return false;
    const Loaded r = load(row, col, n);
#pragma unroll
    for (int i = 0; i < kCols; ++i) {
      const float g = (float)r.g.e[i];
      if (g < kFarGate) {
        const float p = expf(__fmul_rn(0.5f, g));
        k.v[i] = __fmul_rn(__fmul_rn(g, p), __fmul_rn(p, (float)r.u.e[i]));
      }
    }
    return true;
  }
  __device__ __forceinline__ static uint32_t key(const Kept& k) { return key_of(k.v); }
  __device__ __forceinline__ static void values(const Kept& k, float (&v)[kCols]) {
#pragma unroll
    for (int i = 0; i < kCols; ++i) v[i] = k.v[i];
  }
};

struct CodeSink {
  uint8_t* q;
  long long ldq;
  float* scale;
  long long ld_scale;
};

constexpr int kQuantThreads = 256;
constexpr int kNormThreads = 512;

// A warp takes 4 U consecutive blocks of a row, each of its four 8-lane groups
// every fourth, all loads before the first store, which the compiler would not
// move them across. Bound by instructions and memory alike: 16000 x 4096 fp16
// takes 37.8 us (5.3 TB/s), SiLU * up of 16000 x 11008 205 us (4.3 TB/s). With 8
// columns a thread, which doubles the work per block, they took 48 and 281
// (when SiLU took 197); warps that stay and load their next span first, 53 and 281.
template <typename Source, int U, bool kVecQ>
__global__ void __launch_bounds__(kQuantThreads, sizeof(typename Source::Loaded) > 32 ? 4 : 5)
    fp8_quant_kernel(const Source src, const CodeSink out, int rows, int cols, unsigned spans) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x % kGroup;
  const unsigned item = blockIdx.x * (kQuantThreads / 32) + (threadIdx.x >> 5);  // (row, span of 4 U blocks)
  const int row = (int)(item / spans);
  if (row >= rows) return;  // whole warps
  const int kb0 = (int)(item - (unsigned)row * spans) * (4 * U) + (int)(threadIdx.x & 31) / kGroup;
  const int col0 = kb0 * kBlock + lane * kCols;
  typename Source::Loaded raw[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int col = col0 + u * (4 * kBlock);
    raw[u] = src.load(row, col < cols ? col : 0, cols - col);
  }
  typename Source::Kept kept[U];
  uint32_t key[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    kept[u] = Source::keep(raw[u]);
    key[u] = Source::key(kept[u]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int col = col0 + u * (4 * kBlock);
    if (src.rework(row, col < cols ? col : 0, cols - col, kept[u])) key[u] = Source::key(kept[u]);
  }
  const float s = block_scale(key_value<typename Source::Elem>(block_key<U>(key, lane)));
  const float inv = __frcp_rn(s);
  const int kb = kb0 + 4 * own_block<U>(lane);
  if (lane % (kGroup / U) == 0 && kb * kBlock < cols) out.scale[row * out.ld_scale + kb] = s;
  uint8_t* q = out.q + row * out.ldq + col0;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const float inv_u = from_block<U>(inv, u);
    float v[kCols];
    Source::values(kept[u], v);
    const int n = cols - col0 - u * (4 * kBlock);
    if (n > 0) store_codes<kVecQ>(q + u * (4 * kBlock), codes16(v, inv_u), n);
  }
}

// (x + residual) -> RMSNorm -> codes; one CTA per row. kMaxThreads > 0: the row
// stays in registers, 16 columns a thread, with as many registers as the longest
// row's threads leave (up to 704 threads two CTAs share an SM: 16000 x 11008
// with residual takes 273 us, one CTA an SM 358); 0: the row, of any length, is
// read again for the second half.
template <typename T, int kMaxThreads, int kAccess, bool kVecQ>
__global__ void __launch_bounds__(kMaxThreads ? kMaxThreads : kNormThreads, kMaxThreads == 704 ? 2 : 1)
    fp8_rmsnorm_kernel(const T* x, long long ldx, const T* res, long long ld_res, const T* w, float eps,
                       int cols, T* sum_out, long long ld_sum, bool sum_by16, const CodeSink out) {  // sum_out may be x or res
  constexpr bool kInRegs = kMaxThreads > 0;
  __shared__ float red[32];
  pdl_wait();
  pdl_trigger();
  const long long row = blockIdx.x;
  const int lane = threadIdx.x % kGroup;
  const int step = (int)blockDim.x * kCols;
  const int col0 = (int)threadIdx.x * kCols;
  // the rows of p end with the last CTA's; w, with ld 0, is one row
  auto fetch = [&](const T* p, long long ld, int col) {
    return load16<kAccess>(p + row * ld + (col < cols ? col : 0), cols - col, p, p + (gridDim.x - 1) * ld + cols);
  };
  Raw<T> kept, other;
  float ss = 0.f;
  for (int col = col0; kInRegs || col < cols; col += step) {
    kept = fetch(x, ldx, col);
    if (res) other = fetch(res, ld_res, col);
    float v[kCols];
    widen(kept, v);
    if (res) {  // rounded as it is stored: the norm is that of the stored sum
      float r[kCols];
      widen(other, r);
#pragma unroll
      for (int i = 0; i < kCols; ++i) kept.e[i] = from_f32<T>(__fadd_rn(v[i], r[i]));
      widen(kept, v);
      store16(sum_out + row * ld_sum + (col < cols ? col : 0), kept, cols - col, sum_by16);
    }
#pragma unroll
    for (int i = 0; i < kCols; ++i) ss = __fmaf_rn(v[i], v[i], ss);
    if (kInRegs) break;
  }
  if (kInRegs) other = fetch(w, 0, col0);  // on its way while the sums are joined
  ss = warp_sum(ss);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = ss;
  __syncthreads();
  ss = warp_sum((threadIdx.x & 31) < (blockDim.x >> 5) ? red[threadIdx.x & 31] : 0.f);
  // Both within 2 ulps of the IEEE steps, which every thread of the row would
  // pay; the tests count them. cols < 2^31 is far below 2^126, from where on
  // __fdividef gives 0. (A row whose squares overflow fp32 has r = 0.)
  const float r = rsqrtf(__fadd_rn(__fdividef(ss, (float)cols), eps));
  for (int base = 0; base < cols; base += step) {
    const int col = base + col0;
    if (!kInRegs) {  // the stored sum, where there is one: it may have replaced x or the residual
      kept = res ? fetch(sum_out, ld_sum, col) : fetch(x, ldx, col);
      other = fetch(w, 0, col);
    }
    float v[kCols], wv[kCols];
    widen(kept, v);
    widen(other, wv);
#pragma unroll
    for (int i = 0; i < kCols; ++i) v[i] = __fmul_rn(__fmul_rn(v[i], r), wv[i]);
    const uint32_t key[1] = {key_of(v)};
    const float s = block_scale(__uint_as_float(block_key<1>(key, lane)));
    if (col < cols) {
      store_codes<kVecQ>(out.q + row * out.ldq + col, codes16(v, __frcp_rn(s)), cols - col);
      if (lane == 0) out.scale[row * out.ld_scale + col / kBlock] = s;
    }
  }
}

// 128 x 128 weight blocks, one after the other in each of kWeightCtas CTAs an
// SM: 8 threads across, 32 rows at a time, the block held in registers between
// its maximum and its codes. Bound by the way of a block through a CTA (load,
// join, store): 32003 x 4096 fp16 takes 88.7 us, 4.4 TB/s; fp32, twice the
// bytes, 105. A CTA for every block, each with the fence at its end, took 102
// us; loading the next block first, for which half of the warps' registers
// go, 86 at best and 118 in fp32.
constexpr int kWeightThreads = 256;
constexpr int kWeightCtas = 3;
constexpr int kWeightRows = kWeightThreads / kGroup;

template <typename T, int kAccess, bool kVecQ>
__global__ void __launch_bounds__(kWeightThreads, kWeightCtas)
    fp8_quant_weight_kernel(const T* w, long long ldw, int rows, int cols, int k_blocks, unsigned blocks,
                            const CodeSink out) {
  __shared__ uint32_t red[2][kWeightThreads / 32];
  pdl_wait();
  pdl_trigger();
  constexpr int kSteps = kBlock / kWeightRows;
  const T* end = w + (long long)(rows - 1) * ldw + cols;
  int turn = 0;
  for (unsigned block = blockIdx.x; block < blocks; block += gridDim.x, turn ^= 1) {
    const int nb = (int)(block / (unsigned)k_blocks), kb = (int)(block - (unsigned)nb * (unsigned)k_blocks);
    const int col = kb * kBlock + (int)(threadIdx.x % kGroup) * kCols;
    const int row0 = nb * kBlock + (int)threadIdx.x / kGroup;
    Raw<T> raw[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int row = row0 + i * kWeightRows;
      const bool in = row < rows && col < cols;
      raw[i] = load16<kAccess>(w + (in ? (long long)row * ldw + col : 0), in ? cols - col : 0, w, end);
    }
    uint32_t a = 0;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) a = max(a, key_of(raw[i]));
    a = __reduce_max_sync(0xffffffffu, a);
    if ((threadIdx.x & 31) == 0) red[turn][threadIdx.x >> 5] = a;
    __syncthreads();  // the other turn's maxima have been read, too
    a = __reduce_max_sync(0xffffffffu, red[turn][threadIdx.x & (kWeightThreads / 32 - 1)]);
    const float s = block_scale(key_value<T>(a));
    const float inv = __frcp_rn(s);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int row = row0 + i * kWeightRows;
      float v[kCols];
      widen(raw[i], v);
      if (row < rows && col < cols)
        store_codes<kVecQ>(out.q + (long long)row * out.ldq + col, codes16(v, inv), cols - col);
    }
    if (threadIdx.x == 0) out.scale[(long long)nb * out.ld_scale + kb] = s;
  }
}

// ------------------------------------------------------------------ host
constexpr long long kMaxInt = 2147483647ll;
constexpr long long kMaxCols = kMaxInt - kNormThreads * kCols;  // a step past the last column is an int, too

int elem_size(int dtype) { return dtype == NPL_F32 ? 4 : 2; }

// How all rows, `ld` elements apart from `p` on, can be accessed.
int row_access(const void* p, long long rows, long long ld, int dtype) {
  const uintptr_t bits = reinterpret_cast<uintptr_t>(p) | (rows == 1 ? 0 : (uintptr_t)(ld * elem_size(dtype)));
  return bits % 32 == 0 ? kBy32 : bits % 16 == 0 ? kBy16 : kElements;
}

// fn(std::integral_constant<int, access>())
template <typename Fn>
int by_access(int access, Fn&& fn) {
  if (access == kBy32) return fn(std::integral_constant<int, kBy32>());
  if (access == kBy16) return fn(std::integral_constant<int, kBy16>());
  return fn(std::integral_constant<int, kElements>());
}

int check_codes(const char* what, long long rows, long long cols, const void* q, long long ldq, const void* scale,
                long long ld_scale) {
  if (rows < 0 || cols <= 0 || rows > kMaxInt - kBlock || cols > kMaxCols)
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
  return aligned16(o.q) && o.ldq % 16 == 0;
}

template <typename Source, int U>
int launch_quant_spans(const char* what, const Source& src, const CodeSink& out, int rows, int cols, cudaStream_t st) {
  const long long spans = (cols + 4 * U * kBlock - 1) / (4 * U * kBlock);
  constexpr int per_cta = kQuantThreads / 32;
  const long long ctas = (rows * spans + per_cta - 1) / per_cta;
  if (ctas * per_cta > kMaxInt) return fail(NPL_ERR_UNSUPPORTED, "%s: rows=%d cols=%d is too large", what, rows, cols);
  return launch_pdl(what, vec_codes(out) ? fp8_quant_kernel<Source, U, true> : fp8_quant_kernel<Source, U, false>,
                    dim3((unsigned)ctas), dim3(kQuantThreads), 0, st, src, out, rows, cols, (unsigned)spans);
}

// Two blocks a thread where a thread's loads are 32 bytes, except where the
// rows are short (half of the warps' lanes or more would idle) or so few that
// one block a thread fits on the SMs at once. For SiLU, whose values take 16
// registers a block, one (16000 x 4096: 71 us when this was chosen, with two 114).
template <typename Source>
int launch_quant(const char* what, const Source& src, const CodeSink& out, int rows, int cols, cudaStream_t st) {
  constexpr int U = sizeof(typename Source::Loaded) > 32 ? 1 : 2;
  const long long blocks = (long long)rows * ((cols + kBlock - 1) / kBlock);
  if (cols <= 4 * kBlock || blocks <= 128ll * num_sms())
    return launch_quant_spans<Source, 1>(what, src, out, rows, cols, st);
  return launch_quant_spans<Source, U>(what, src, out, rows, cols, st);
}

template <typename T, int kAccess, bool kVecQ>
int launch_rmsnorm(const T* x, long long ldx, const T* res, long long ld_res, const T* w, float eps, int rows,
                   int cols, T* sum_out, long long ld_sum, bool sum_by16, const CodeSink& out, cudaStream_t st) {
  const int lanes = (cols + kCols - 1) / kCols;
  const int threads = lanes <= 1024 ? (lanes + 31) / 32 * 32 : kNormThreads;
  // The instance of 704 threads has 40 registers a thread, so that an SM holds three
  // rows of 8192 columns; that of 512 (48 for bf16, 56 for fp16) two. bf16 takes it
  // for long rows (1000 x 6144 with residual 10.2 us with 48, 9.1 with 40; 4000 x 8192
  // 50.0 and 42.6) and for more rows than the SMs hold at once, 1280 threads each
  // (16000 x 4096 83.3 and 80.6, 4000 x 3584 21.2 and 19.8, 1200 x 2560 5.9 and 5.4;
  // 4000 x 1024 6.8 and 7.1), not where they hold all (560 x 4096 4.4 and 4.9). fp16
  // spills 60 bytes at 40: 4000 x 8192 31.5 us and 27.5, 1000 x 5120 5.9 and 5.6, but
  // with a residual 1000 x 8192 13.5 and 14.7.
  const bool fills = (long long)rows * threads > 1280ll * num_sms();
  const int few = !std::is_same<T, __half>::value ? (fills ? 0 : 320) : res ? 512 : 416;
  auto kern = lanes <= few    ? fp8_rmsnorm_kernel<T, 512, kAccess, kVecQ>
              : lanes <= 704  ? fp8_rmsnorm_kernel<T, 704, kAccess, kVecQ>
              : lanes <= 1024 ? fp8_rmsnorm_kernel<T, 1024, kAccess, kVecQ>
                              : fp8_rmsnorm_kernel<T, 0, kAccess, kVecQ>;
  return launch_pdl("npl_fp8_rmsnorm_quant", kern, dim3((unsigned)rows), dim3((unsigned)threads), 0, st, x, ldx, res,
                    ld_res, w, eps, cols, sum_out, ld_sum, sum_by16, out);
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
    return by_access(row_access(x, rows, ldx, x_dtype), [&](auto a) {
      return launch_quant(what, RowSource<T, a.value>{p, ldx, p + (rows - 1) * ldx + cols}, out, (int)rows, (int)cols, st);
    });
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
    const int access = std::min(row_access(gate, rows, ld_gate, dtype), row_access(up, rows, ld_up, dtype));
    return by_access(access, [&](auto a) {
      const SiluSource<T, a.value> src{g, u, ld_gate, ld_up, g + (rows - 1) * ld_gate + cols, u + (rows - 1) * ld_up + cols};
      return launch_quant(what, src, out, (int)rows, (int)cols, st);
    });
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
  int access = std::min(row_access(x, rows, ldx, dtype), row_access(weight, 1, cols, dtype));
  // the row that is not kept in registers is read back from the sum
  if (residual) access = std::min(access, row_access(residual, rows, ld_res, dtype));
  const bool sum_by16 = residual && row_access(sum_out, rows, ld_sum, dtype) >= kBy16;
  if (residual && (cols + kCols - 1) / kCols > 1024)
    access = std::min(access, row_access(sum_out, rows, ld_sum, dtype));
  const bool vecq = vec_codes(out);
  auto go = [&](auto t) {
    using T = decltype(t);
    return by_access(access, [&](auto a) {
      auto* fn = vecq ? launch_rmsnorm<T, a.value, true> : launch_rmsnorm<T, a.value, false>;
      return fn(static_cast<const T*>(x), ldx, static_cast<const T*>(residual), ld_res, static_cast<const T*>(weight),
                eps, (int)rows, (int)cols, static_cast<T*>(sum_out), ld_sum, sum_by16, out,
                static_cast<cudaStream_t>(stream));
    });
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
  if (nb * kb > kMaxInt) return fail(NPL_ERR_UNSUPPORTED, "%s: %lld blocks (at most 2^31 - 1)", what, nb * kb);
  const CodeSink out{q, ldq, scale, ld_scale};
  const bool vecq = vec_codes(out);
  return by_type(w_dtype, [&](auto t) {
    using T = decltype(t);
    return by_access(row_access(w, rows, ldw, w_dtype), [&](auto a) {
      auto kern = vecq ? fp8_quant_weight_kernel<T, a.value, true> : fp8_quant_weight_kernel<T, a.value, false>;
      return launch_pdl(what, kern, dim3((unsigned)std::min(nb * kb, (long long)kWeightCtas * num_sms())),
                        dim3(kWeightThreads), 0, static_cast<cudaStream_t>(stream), static_cast<const T*>(w), ldw,
                        (int)rows, (int)cols, (int)kb, (unsigned)(nb * kb), out);
    });
  });
}
