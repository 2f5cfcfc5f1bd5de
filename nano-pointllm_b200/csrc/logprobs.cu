// Log probabilities of given tokens, the entropy of their distributions and
// the top alternatives, from rows of logits.
#include <cuda_bf16.h>

#include "npl_common.cuh"

namespace npl {
namespace {

constexpr int kLpMaxTop = 32;
constexpr int kLpThreads = 256;

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// Whole numbers in the order of the values: equal ones for +0 and -0, the
// largest for every NaN.
__device__ __forceinline__ int order_key(float x) {
  if (x != x) return 0x7fffffff;
  const int b = __float_as_int(x);
  return b < 0 ? -(b & 0x7fffffff) : b;
}

template <typename T>
__global__ void __launch_bounds__(kLpThreads)
    logprobs_simple(const T* logits, long long ld, int V, const int64_t* ids, int top_k, float* lp, float* ent,
                    int64_t* top_ids, float* top_lp, int* status) {
  __shared__ float red[32];
  __shared__ long long best[32];
  const long long r = blockIdx.x;
  const T* x = logits + r * ld;
  float m = -INFINITY;
  for (int i = threadIdx.x; i < V; i += blockDim.x) m = fmaxf(m, to_float(x[i]));
  m = block_max(m, red);
  __syncthreads();
  float s = 0.f, t = 0.f;
  for (int i = threadIdx.x; i < V; i += blockDim.x) {
    const float d = to_float(x[i]) - m, e = expf(d);
    s += e;
    t += d == -INFINITY ? 0.f : d * e;
  }
  s = block_sum(s, red);
  __syncthreads();
  t = block_sum(t, red);
  const float ls = logf(s);
  if (threadIdx.x == 0) {
    const long long id = ids[r];
    if (id < -1 || id >= V) atomicCAS(status, 0, NPL_DEV_BAD_INDEX);
    lp[r] = id == -1 ? 0.f : id < 0 || id >= V ? NAN : to_float(x[id]) - m - ls;
    ent[r] = ls - t / s;
  }
  long long prev = 0x7fffffffffffffffll;  // (key, places from the end) of the last one taken
  for (int k = 0; k < top_k; ++k) {
    long long c = -0x7fffffffffffffffll;
    for (int i = threadIdx.x; i < V; i += blockDim.x) {
      const long long y = ((long long)order_key(to_float(x[i])) << 32) | (unsigned)(0x7fffffff - i);
      if (y < prev && y > c) c = y;
    }
    __syncthreads();
    c = block_max(c, best);
    prev = c;
    if (threadIdx.x == 0) {
      const int id = 0x7fffffff - (int)(unsigned)c;
      top_ids[r * top_k + k] = id;
      top_lp[r * top_k + k] = to_float(x[id]) - m - ls;
    }
  }
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
  int* status = device_status_ptr();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == NPL_F32)
    logprobs_simple<<<(unsigned)rows, kLpThreads, 0, st>>>(static_cast<const float*>(logits), ld, (int)vocab,
                                                          token_ids, top_k, logprobs, entropy, top_ids,
                                                          top_logprobs, status);
  else if (dtype == NPL_F16)
    logprobs_simple<<<(unsigned)rows, kLpThreads, 0, st>>>(static_cast<const __half*>(logits), ld, (int)vocab,
                                                          token_ids, top_k, logprobs, entropy, top_ids,
                                                          top_logprobs, status);
  else
    logprobs_simple<<<(unsigned)rows, kLpThreads, 0, st>>>(static_cast<const __nv_bfloat16*>(logits), ld, (int)vocab,
                                                          token_ids, top_k, logprobs, entropy, top_ids,
                                                          top_logprobs, status);
  return launch_status(what);
}
