// Log probabilities of given tokens, the entropy of their distributions and
// the top alternatives, from rows of logits.
//
// npl_token_logprobs (no counterpart in the reference). With x a row, M its
// maximum and d = x - M:
//   S = sum e^d,  T = sum d e^d,  ln p = d - ln S,  entropy = ln S - T / S
// in one read of the row: a thread keeps the maximum m of what it has read and
// s, t relative to it; when m moves by delta = m - m' < 0,
//   t' = e^delta (t + delta s),  s' = e^delta s
// and the threads' sums are joined the same way.
//
// Top k: of the threads' maxima, the k-th largest is no larger than the k-th
// largest logit, so only threads whose own maximum reaches it (k of them, and
// those that tie) have their words read once more, from L2, for the logits that
// reach it. Those few are ranked by counting: larger first, of equal ones the
// lowest index.
//
// One CTA of 128 threads takes a row, each with 8 words in flight and two sums an
// instruction (16000 x 32003 fp16, top 5: 180 us,
// 5.7 TB/s); few rows are split over a cluster of CTAs each, whose sums and best
// logits its first CTA joins (64 x 32003 fp32, top 20: 11.5 us).
#include <algorithm>

#include <cuda_bf16.h>

#include "npl_common.cuh"

namespace npl {
namespace {

constexpr int kLpMaxTop = 32;
constexpr int kLpThreads = 128;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpUnroll = 8;      // 16-byte words that a thread has in flight
constexpr int kLpCandidates = 512;  // at least kLpMaxTop * (kLpMaxSplit + 1)
constexpr int kLpRounds = 10;       // top tokens from which on every thread ranks its maximum
constexpr int kLpStep = 2048;     // logits that a CTA looks through at a time for equal ones
constexpr int kLpMaxSplit = 8;    // CTAs of a cluster at most
constexpr float kLpFar = -200.f;  // e^-200 is 0 in fp32: distances are cut here, so that 0 * infinity cannot arise
constexpr float kLog2e = 1.4426950408889634f;

// Whole numbers in the order of the values: equal ones for +0 and -0, the
// largest for every NaN; 0 is left for "no value".
__device__ __forceinline__ unsigned lp_key(float x) {
  if (x != x) return 0xffffffffu;
  const int b = __float_as_int(x);
  return (unsigned)(b < 0 ? -(b & 0x7fffffff) : b) ^ 0x80000000u;
}

__device__ __forceinline__ float lp_max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float lp_exp(float d) {  // e^d for d <= 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(d * kLog2e));
  return y;
}

// 16 bytes of logits as floats, and their maximum (NaN if there is one).
template <typename T>
struct LpWord;
template <>
struct LpWord<float> {
  static constexpr int kN = 4;
  static constexpr uint32_t kNone = 0xff800000u;  // minus infinity
  __device__ static float top(const uint4& w) {
    return lp_max_nan(lp_max_nan(__uint_as_float(w.x), __uint_as_float(w.y)),
                      lp_max_nan(__uint_as_float(w.z), __uint_as_float(w.w)));
  }
  __device__ static void get(const uint4& w, float (&x)[4]) {
    x[0] = __uint_as_float(w.x), x[1] = __uint_as_float(w.y);
    x[2] = __uint_as_float(w.z), x[3] = __uint_as_float(w.w);
  }
  __device__ static float one(float x) { return x; }
  // logits below kFloor taken as kFloor: where the maximum is above kSlow, e^(x - m) is 0 either way
  static constexpr float kSlow = -1e29f;
  __device__ static void cut(uint4& w) {
    w.x = __float_as_uint(fmaxf(__uint_as_float(w.x), -1e30f)), w.y = __float_as_uint(fmaxf(__uint_as_float(w.y), -1e30f));
    w.z = __float_as_uint(fmaxf(__uint_as_float(w.z), -1e30f)), w.w = __float_as_uint(fmaxf(__uint_as_float(w.w), -1e30f));
  }
};
template <typename H2>
__device__ __forceinline__ H2 lp_as(uint32_t w) {
  return *reinterpret_cast<const H2*>(&w);
}
template <typename H2>
__device__ __forceinline__ uint32_t lp_bits(H2 h) {
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
struct LpWord<__half> {
  static constexpr int kN = 8;
  static constexpr uint32_t kNone = 0xfc00fc00u;
  __device__ static float top(const uint4& w) {
    const __half2 m = __hmax2_nan(__hmax2_nan(lp_as<__half2>(w.x), lp_as<__half2>(w.y)),
                                  __hmax2_nan(lp_as<__half2>(w.z), lp_as<__half2>(w.w)));
    return __half2float(__hmax_nan(__low2half(m), __high2half(m)));
  }
  __device__ static void get(const uint4& w, float (&x)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(lp_as<__half2>(u[i]));
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
  }
  __device__ static float one(__half x) { return __half2float(x); }
  static constexpr float kSlow = -65000.f;
  __device__ static void cut(uint4& w) {
    const __half2 least = __half2half2(__ushort_as_half(0xfbff));  // -65504
    w.x = lp_bits(__hmax2(lp_as<__half2>(w.x), least)), w.y = lp_bits(__hmax2(lp_as<__half2>(w.y), least));
    w.z = lp_bits(__hmax2(lp_as<__half2>(w.z), least)), w.w = lp_bits(__hmax2(lp_as<__half2>(w.w), least));
  }
};
template <>
struct LpWord<__nv_bfloat16> {
  static constexpr int kN = 8;
  static constexpr uint32_t kNone = 0xff80ff80u;
  __device__ static float top(const uint4& w) {
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(lp_as<__nv_bfloat162>(w.x), lp_as<__nv_bfloat162>(w.y)),
                                         __hmax2_nan(lp_as<__nv_bfloat162>(w.z), lp_as<__nv_bfloat162>(w.w)));
    return __bfloat162float(__hmax_nan(__low2bfloat16(m), __high2bfloat16(m)));
  }
  __device__ static void get(const uint4& w, float (&x)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      x[2 * i] = __uint_as_float(u[i] << 16), x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
  }
  __device__ static float one(__nv_bfloat16 x) { return __bfloat162float(x); }
  static constexpr float kSlow = -1e29f;
  __device__ static void cut(uint4& w) {
    const __nv_bfloat162 least = __float2bfloat162_rn(-1e30f);
    w.x = lp_bits(__hmax2(lp_as<__nv_bfloat162>(w.x), least)), w.y = lp_bits(__hmax2(lp_as<__nv_bfloat162>(w.y), least));
    w.z = lp_bits(__hmax2(lp_as<__nv_bfloat162>(w.z), least)), w.w = lp_bits(__hmax2(lp_as<__nv_bfloat162>(w.w), least));
  }
};

struct LpSum {  // of values seen so far: maximum, sum e^(x - m), sum (x - m) e^(x - m)
  float m, s, t;
};

__device__ __forceinline__ void lp_move(LpSum& a, float m) {  // to a maximum m >= a.m (or NaN)
  const float delta = fmaxf(a.m - m, kLpFar);  // a.m == m: 0; minus infinities and NaN: far, with s = t = 0 or no result
  const float f = a.m == m ? 1.f : lp_exp(delta);
  a.t = a.m == m ? a.t : f * fmaf(delta, a.s, a.t);
  a.s *= f;
  a.m = m;
}

__device__ __forceinline__ void lp_add(LpSum& a, float x) {  // x <= a.m
  const float d = fmaxf(x - a.m, kLpFar), e = a.m == -INFINITY ? 0.f : lp_exp(d);
  a.s += e;
  a.t = fmaf(d, e, a.t);
}

// Two sums at a time (one instruction for two fp32 numbers).
__device__ __forceinline__ uint64_t lp_pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 lp_unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t lp_add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t lp_mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t lp_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float lp_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct LpSmem {
  float red[3][kLpWarps];
  alignas(16) unsigned keys[kLpThreads];
  unsigned threshold;
  int n_candidates, n_list;
  int list[kLpThreads];  // threads whose maximum reaches the threshold
  unsigned long long candidate[kLpCandidates];  // key << 32 | ~index: larger is better
  unsigned long long best[kLpMaxTop];           // of this CTA, best first
  LpSum sum;                                    // of this CTA
  unsigned scan[kLpWarps];
  unsigned long long round[kLpWarps];
};

__device__ __forceinline__ unsigned long long lp_pack(unsigned key, int index) {
  return ((unsigned long long)key << 32) | (unsigned)~index;
}

template <typename T>
struct LpRow {  // this CTA's part of a row: words [w0, w1) of 16 bytes from `words`, and single logits around them
  const T* x;
  const uint4* words;
  int head, w0, w1;  // logits before the first word; this CTA's words
  int tail, n_tail;  // logits behind the last word, and how many of them are this CTA's
  bool first;        // the row's first part, to which the logits before the first word belong
  int end;           // one past this part's last logit
  __device__ int single(int thread) const {  // the single logit of a thread, -1: none
    if (first && thread < head) return thread;
    return thread >= 32 && thread - 32 < n_tail ? tail + thread - 32 : -1;
  }
};

template <typename T>
__device__ __forceinline__ float lp_at(const T* x, int i) {
  return LpWord<T>::one(x[i]);
}

template <typename T, typename F>
__device__ __forceinline__ void lp_each(const LpRow<T>& r, F&& f) {  // this thread's logits: f(value, index)
  constexpr int N = LpWord<T>::kN;
  const int single = r.single(threadIdx.x);
  if (single >= 0) f(lp_at(r.x, single), single);
  for (int w = r.w0 + (int)threadIdx.x; w < r.w1; w += kLpThreads) {
    float v[N];
    LpWord<T>::get(r.words[w], v);
#pragma unroll
    for (int e = 0; e < N; ++e) f(v[e], r.head + w * N + e);
  }
}

// The k best of this CTA's logits into s.best (empty places are 0).
template <typename T>
__device__ void lp_top(LpSmem& s, const LpRow<T>& r, float own_max, bool any, int k) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const unsigned own = any ? lp_key(own_max) : 0u;
  s.keys[tid] = own;
  if (tid == 0) s.n_candidates = s.n_list = 0;
  if (tid < kLpMaxTop) s.best[tid] = 0;
  __syncthreads();
  // The k-th largest of the maxima (1, below every logit's key, where fewer threads have any): few of them one below
  // the other by a warp, a round each; from kLpRounds on every thread counts those above its own, in one time for all
  // k. Rows of 32003, rounds / counting, us: 64 in fp32, top 5 9.0 / 10.3, top 8 9.3 / 10.4, top 20 11.2 / 11.6; 3000 in
  // fp32, 83.5 / 85.6, 89.2 / 89.6, 114.3 / 113.0; one, 6.7 / 7.0, 7.0 / 7.1, top 16 7.8 / 7.3. They meet at 9 to 16.
  if (k >= kLpRounds) {
    int above[4] = {0, 0, 0, 0}, from[4] = {0, 0, 0, 0};
#pragma unroll 8
    for (int i = 0; i < kLpThreads; i += 4) {
      const uint4 y = *reinterpret_cast<const uint4*>(&s.keys[i]);
      above[0] += y.x > own, above[1] += y.y > own, above[2] += y.z > own, above[3] += y.w > own;
      from[0] += y.x >= own, from[1] += y.y >= own, from[2] += y.z >= own, from[3] += y.w >= own;
    }
    if (above[0] + above[1] + above[2] + above[3] < k && from[0] + from[1] + from[2] + from[3] >= k) s.threshold = max(own, 1u);  // those that are equal write the same
  } else if (warp == 0) {
    unsigned key[kLpWarps], last = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < kLpWarps; ++i) key[i] = s.keys[lane + i * 32];
    for (int have = 0; have < k && last;) {
      unsigned c = 0;
#pragma unroll
      for (int i = 0; i < kLpWarps; ++i) c = max(c, key[i]);
      last = __reduce_max_sync(0xffffffffu, c);
      int equal = 0;
#pragma unroll
      for (int i = 0; i < kLpWarps; ++i) {
        equal += key[i] == last;
        if (key[i] == last) key[i] = 0;
      }
      have += __reduce_add_sync(0xffffffffu, equal);
    }
    if (lane == 0) s.threshold = max(last, 1u);
  }
  __syncthreads();
  const unsigned least = s.threshold;
  if (own >= least) s.list[atomicAdd(&s.n_list, 1)] = tid;
  __syncthreads();
  // a warp takes threads that reach it, a lane one of a thread's words (of few words: several threads at a time)
  int per_log = 5;
  while (per_log > 0 && (kLpThreads << (per_log - 1)) >= r.w1 - r.w0) --per_log;
  const int at_once = 32 >> per_log;
  for (int q = warp * at_once + (lane >> per_log); q < s.n_list; q += kLpWarps * at_once) {
    const int who = s.list[q], first = lane & ((1 << per_log) - 1);
    auto take = [&](float x, int i) {
      const unsigned key = lp_key(x);
      if (key < least) return;
      const int at = atomicAdd(&s.n_candidates, 1);
      if (at < kLpCandidates) s.candidate[at] = lp_pack(key, i);
    };
    if (first == 0 && r.single(who) >= 0) take(lp_at(r.x, r.single(who)), r.single(who));
    for (int w = r.w0 + who + first * kLpThreads; w < r.w1; w += kLpThreads << per_log) {
      const uint4 word = r.words[w];
      if (lp_key(LpWord<T>::top(word)) < least) continue;
      float v[LpWord<T>::kN];
      LpWord<T>::get(word, v);
#pragma unroll
      for (int e = 0; e < LpWord<T>::kN; ++e) take(v[e], r.head + w * LpWord<T>::kN + e);
    }
  }
  __syncthreads();
  int n = s.n_candidates;
  if (n > kLpCandidates) {
    // Many equal logits (the zeros of a padding row, say), or many large ones with one thread. A pass finds the best
    // logit after the last one taken; then those equal to it are taken in the order of their places, a few at a time.
    const int from = r.first ? 0 : r.head + r.w0 * LpWord<T>::kN;
    unsigned long long most = ~0ull;  // not taken yet: this (a NaN in the first place) and less
    for (int j = 0; j < k;) {
      unsigned long long c = 0;
      lp_each(r, [&](float x, int i) {
        const unsigned long long y = lp_pack(lp_key(x), i);
        if (y <= most && y > c) c = y;
      });
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) c = max(c, __shfl_xor_sync(0xffffffffu, c, o));
      if (lane == 0) s.round[warp] = c;
      __syncthreads();
      c = 0;
#pragma unroll
      for (int i = 0; i < kLpWarps; ++i) c = max(c, s.round[i]);
      if (c == 0) break;  // this part holds no more logits
      const unsigned key = (unsigned)(c >> 32);
      int place = (int)~(unsigned)c;
      if (tid == 0) s.best[j] = c;
      ++j;
      for (int base = from + (place - from) / kLpStep * kLpStep; j < k && base < r.end;) {
        unsigned next = 0x7fffffffu;
        for (int e = kLpStep / kLpThreads - 1; e >= 0; --e) {
          const int i = base + tid * (kLpStep / kLpThreads) + e;
          if (i > place && i < r.end && lp_key(lp_at(r.x, i)) == key) next = i;
        }
        next = __reduce_min_sync(0xffffffffu, next);
        __syncthreads();
        if (lane == 0) s.scan[warp] = next;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kLpWarps; ++i) next = min(next, s.scan[i]);
        if (next == 0x7fffffffu) {
          base += kLpStep;
        } else {
          place = (int)next;
          if (tid == 0) s.best[j] = lp_pack(key, place);
          ++j;
        }
      }
      most = ((unsigned long long)key << 32) - 1;  // where places are left, all that are equal have been taken; key > 0
      __syncthreads();
    }
    __syncthreads();
    return;
  }
  for (int i = tid; i < n; i += kLpThreads) {
    const unsigned long long mine = s.candidate[i];
    int better = 0;
    #pragma unroll 4
    for (int j = 0; j < n; ++j) better += s.candidate[j] > mine;
    if (better < k) s.best[better] = mine;
  }
  __syncthreads();
}

__device__ __forceinline__ LpSum lp_ld_sum(const LpSum* p, int rank) {
  const uint32_t a = cluster_map(p, rank);
  LpSum r;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(r.m) : "r"(a) : "memory");
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(r.s) : "r"(a + 4) : "memory");
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(r.t) : "r"(a + 8) : "memory");
  return r;
}

struct LpArgs {
  const void* logits;
  long long ld;
  int vocab, top_k, split, split_log;
  const int64_t* ids;
  float* lp;
  float* entropy;
  int64_t* top_ids;
  float* top_lp;
  int* status;
};

template <typename T>
__global__ void __launch_bounds__(kLpThreads) logprobs_kernel(const LpArgs p) {
  __shared__ LpSmem s;
  constexpr int N = LpWord<T>::kN;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = blockIdx.x & (p.split - 1);
  const long long row = blockIdx.x >> p.split_log;
  pdl_wait();
  pdl_trigger();
  LpRow<T> r;
  r.x = static_cast<const T*>(p.logits) + row * p.ld;
  r.head = min(p.vocab, (int)((16 - (reinterpret_cast<uintptr_t>(r.x) & 15)) & 15) / (int)sizeof(T));
  r.words = reinterpret_cast<const uint4*>(r.x + r.head);
  const int words = (p.vocab - r.head) / N;
  r.w0 = (int)(((long long)words * rank) >> p.split_log);
  r.w1 = (int)(((long long)words * (rank + 1)) >> p.split_log);
  r.first = rank == 0;
  r.tail = r.head + words * N;
  r.n_tail = rank == p.split - 1 ? p.vocab - r.tail : 0;
  r.end = rank == p.split - 1 ? p.vocab : r.head + r.w1 * N;
  const int single = r.single(tid);

  LpSum a = {-INFINITY, 0.f, 0.f};
  if (single >= 0) a = {lp_at(r.x, single), 1.f, 0.f};
  if (a.m == -INFINITY) a.s = 0.f;
  for (int w = r.w0 + tid; w < r.w1; w += kLpThreads * kLpUnroll) {
    uint4 v[kLpUnroll];
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u)
      v[u] = w + u * kLpThreads < r.w1 ? r.words[w + u * kLpThreads]
                                       : make_uint4(LpWord<T>::kNone, LpWord<T>::kNone, LpWord<T>::kNone,
                                                    LpWord<T>::kNone);
    float m = a.m;
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u) m = lp_max_nan(m, LpWord<T>::top(v[u]));
    lp_move(a, m);
    if (m > LpWord<T>::kSlow) {
      const uint64_t from = lp_pair(-m, -m), scale = lp_pair(kLog2e, kLog2e);
      uint64_t s2 = lp_pair(0.f, 0.f), t2 = s2;
#pragma unroll
      for (int u = 0; u < kLpUnroll; ++u) {
        float x[N];
        LpWord<T>::cut(v[u]);
        LpWord<T>::get(v[u], x);
#pragma unroll
        for (int e = 0; e < N; e += 2) {
          const uint64_t d = lp_add2(lp_pair(x[e], x[e + 1]), from);
          const float2 y = lp_unpair(lp_mul2(d, scale));
          const uint64_t ex = lp_pair(lp_exp2(y.x), lp_exp2(y.y));
          s2 = lp_add2(s2, ex);
          t2 = lp_fma2(d, ex, t2);
        }
      }
      const float2 s1 = lp_unpair(s2), t1 = lp_unpair(t2);
      a.s += s1.x + s1.y;
      a.t += t1.x + t1.y;
    } else if (m != -INFINITY) {  // nothing but logits near the type's lowest value so far (or a NaN)
#pragma unroll 1
      for (int u = 0; u < kLpUnroll; ++u) {
        if (w + u * kLpThreads >= r.w1) break;
        float x[N];
        LpWord<T>::get(r.words[w + u * kLpThreads], x);
#pragma unroll
        for (int e = 0; e < N; ++e) lp_add(a, x[e]);
      }
    }
  }

  // the CTA's maximum and sums
  const float own_max = a.m;
  float m = a.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = lp_max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) s.red[0][warp] = m;
  __syncthreads();
  m = s.red[0][0];
#pragma unroll
  for (int i = 1; i < kLpWarps; ++i) m = lp_max_nan(m, s.red[0][i]);
  lp_move(a, m);
  a.s = warp_sum(a.s);
  a.t = warp_sum(a.t);
  if (lane == 0) s.red[1][warp] = a.s, s.red[2][warp] = a.t;
  __syncthreads();
  a.s = a.t = 0.f;
#pragma unroll
  for (int i = 0; i < kLpWarps; ++i) a.s += s.red[1][i], a.t += s.red[2][i];

  if (p.top_k) lp_top(s, r, own_max, single >= 0 || r.w0 + tid < r.w1, p.top_k);

  if (p.split > 1) {
    if (tid == 0) s.sum = a;
    cluster_arrive_release();
    cluster_wait_acquire();
    if (rank == 0) {
      LpSum part[kLpMaxSplit];
      m = -INFINITY;
#pragma unroll
      for (int j = 0; j < kLpMaxSplit; ++j) {  // where there are fewer, the first ones again
        part[j] = lp_ld_sum(&s.sum, j & (p.split - 1));
        m = lp_max_nan(m, part[j].m);
      }
      a = {m, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < kLpMaxSplit; ++j) {
        lp_move(part[j], m);
        if (j < p.split) a.s += part[j].s, a.t += part[j].t;
      }
      const int n = p.top_k ? p.split * kLpMaxTop : 0;
      for (int i = tid; i < n; i += kLpThreads) {
        const uint32_t at = cluster_map(&s.best[i & (kLpMaxTop - 1)], i / kLpMaxTop);
        unsigned long long y;
        asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(y) : "r"(at) : "memory");
        s.candidate[i] = y;
      }
      __syncthreads();
      for (int i = tid; i < n; i += kLpThreads) {
        const unsigned long long mine = s.candidate[i];
        if (mine == 0) continue;
        // those above it, in each CTA's list (best first, empty places 0) by halving
        int better = 0;
#pragma unroll
        for (int j = 0; j < kLpMaxSplit; ++j) {
          const unsigned long long* list = s.candidate + (j & (p.split - 1)) * kLpMaxTop;
          int above = 0;
#pragma unroll
          for (int step = kLpMaxTop / 2; step > 0; step /= 2) above += list[above + step - 1] > mine ? step : 0;
          above += list[above] > mine;
          better += j < p.split ? above : 0;
        }
        if (better < p.top_k) s.candidate[n + better] = mine;
      }
      __syncthreads();
      if (tid < p.top_k) s.best[tid] = s.candidate[n + tid];
    }
    cluster_arrive_release();  // no CTA leaves while the first reads its shared memory
    cluster_wait_acquire();
    if (rank != 0) return;
  }

  const bool bad = !(fabsf(a.m) < INFINITY);  // NaN, plus infinity, or nothing but minus infinity
  const float ls = bad ? NAN : logf(a.s);
  if (tid < p.top_k) {
    const int i = (int)~(unsigned)s.best[tid];
    p.top_ids[row * p.top_k + tid] = i;
    p.top_lp[row * p.top_k + tid] = lp_at(r.x, i) - a.m - ls;
  }
  if (tid == kLpThreads - 1) {
    const long long id = p.ids[row];
    const bool in = id >= 0 && id < p.vocab;
    if (!in && id != -1) atomicCAS(p.status, 0, NPL_DEV_BAD_INDEX);
    p.lp[row] = in ? lp_at(r.x, (int)id) - a.m - ls : id == -1 ? 0.f : NAN;
    p.entropy[row] = ls - a.t / a.s;
  }
}

template <typename T>
int launch(const char* what, LpArgs p, long long rows, cudaStream_t st) {
  const int sms = num_sms() > 0 ? num_sms() : 148;
  p.split_log = 0;
  while ((1 << p.split_log) < kLpMaxSplit && (rows << p.split_log) * 2 <= 4ll * sms &&
         p.vocab >> p.split_log >= 2 * kLpThreads * LpWord<T>::kN)
    ++p.split_log;
  p.split = 1 << p.split_log;
  return launch_pdl_cluster(what, logprobs_kernel<T>, dim3((unsigned)(rows * p.split)), dim3(kLpThreads), 0, st,
                            (unsigned)p.split, p);
}

}  // namespace
}  // namespace npl

using namespace npl;

extern "C" int npl_token_logprobs(const void* logits, int dtype, int64_t ld, int64_t rows, int64_t vocab,
                                  const int64_t* token_ids, int top_k, float* logprobs, float* entropy,
                                  int64_t* top_ids, float* top_logprobs, void* stream) {
  const char* what = "npl_token_logprobs";
  if (dtype != NPL_F16 && dtype != NPL_BF16 && dtype != NPL_F32)
    return fail(NPL_ERR_ARG, "%s: element type %d (NPL_F32, NPL_F16 or NPL_BF16)", what, dtype);
  if (rows < 0 || vocab < 1 || vocab >= (1ll << 31) - 65536 || rows >= (1ll << 31) || (rows > 1 && ld < vocab))
    return fail(NPL_ERR_ARG, "%s: bad shape rows=%lld vocab=%lld stride=%lld", what, (long long)rows,
                (long long)vocab, (long long)ld);
  if (top_k < 0 || top_k > kLpMaxTop || top_k > vocab)
    return fail(NPL_ERR_ARG, "%s: top_k %d (0 to %d, and no more than the vocabulary)", what, top_k, kLpMaxTop);
  if (rows > 0 && (!logits || !token_ids || !logprobs || !entropy || (top_k && (!top_ids || !top_logprobs))))
    return fail(NPL_ERR_ARG, "%s: null pointer", what);
  const uintptr_t esz = dtype == NPL_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) % esz)
    return fail(NPL_ERR_ARG, "%s: logits are not aligned to their elements", what);
  if ((reinterpret_cast<uintptr_t>(token_ids) | reinterpret_cast<uintptr_t>(top_ids)) & 7u ||
      (reinterpret_cast<uintptr_t>(logprobs) | reinterpret_cast<uintptr_t>(entropy) |
       reinterpret_cast<uintptr_t>(top_logprobs)) & 3u)
    return fail(NPL_ERR_ARG, "%s: ids or outputs are not aligned to their elements", what);
  if (int rc = check_device()) return rc;
  if (rows == 0) return NPL_OK;
  LpArgs p{};
  p.logits = logits, p.ld = ld, p.vocab = (int)vocab, p.top_k = top_k, p.ids = token_ids;
  p.lp = logprobs, p.entropy = entropy, p.top_ids = top_ids, p.top_lp = top_logprobs;
  p.status = device_status_ptr();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == NPL_F32) return launch<float>(what, p, rows, st);
  return dtype == NPL_F16 ? launch<__half>(what, p, rows, st) : launch<__nv_bfloat16>(what, p, rows, st);
}
