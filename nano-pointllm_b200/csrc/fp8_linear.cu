// Block-scaled e4m3 linear on the 5th-generation tensor cores (tcgen05,
// kind::f8f6f4):
//
//   out[m, n] = T(sum_b sa[m, b] sw[n / 128, b] P_b[m, n] + bias[n] + residual[m, n])
//   P_b[m, n] = sum over the 128 columns k of block b of qa[m, k] qw[n, k]
//
// The tensor cores sum one block P_b (fp32, in TMEM); its two scales cannot be
// applied inside the MMA, so every block starts a new accumulator and the
// epilogue warps add it, scaled, to fp32 sums in registers. The output is rounded
// to T once, after bias and residual.
//
// Decode tiles (M <= 64): the weight tile is the MMA's A operand and the tokens
// are its N dimension (D[n, m], 128 weight rows x NT tokens), so a decode
// batch fills an MMA with NT = 16..64. Prefill tiles: see below.
//
// Per decode CTA (192 threads):
//   warp 0     TMA producer: weight tile [128 x 128 B] and token tile
//              [NT x 128 B] per block, 128-byte swizzle, a ring of stages
//   warp 1     TMEM owner + MMA issuer: 4 MMAs of K = 32 per block into a ring
//              of 4 accumulators
//   warps 2-5  TMEM lane = weight row, column = token: acc += (sa sw) * D
//
// Split over K: the S CTAs of a thread-block cluster share a tile's blocks.
// Each leaves its fp32 sums in its own shared memory; after a cluster barrier
// CTA r adds those of ranks 0, 1, .. S - 1, in this order, for its share of
// the tokens. No workspace and no atomics: two calls in flight share nothing,
// and equal inputs give equal bits.
//
// All mbarrier waits are bounded (~1 s); on expiry the kernel records a code
// in the device status word, drains its in-flight copies and MMAs, meets its
// cluster, frees TMEM and returns.
#include <cuda_bf16.h>
#include <cudaTypedefs.h>

#include <algorithm>

#include "npl_common.cuh"

namespace npl {
namespace {

constexpr int kTileN = 128;   // weight rows per tile (MMA M) and per scale
constexpr int kBlockK = 128;  // columns per scale = bytes per stage row (one 128-byte swizzle atom)
constexpr int kThreads = 192;
constexpr int kMaxStages = 6;
constexpr int kAccBufs = 4;
constexpr int kMaxSplit = 8;

struct Fp8LinearArgs {
  int M, N;
  int k_blocks;
  int m_tiles;
  int n_tiles;
  int stages;    // decode tiles
  int split;     // decode tiles: CTAs per tile
  int raster_g;  // prefill tiles: token tiles per raster group
  int tma_out;   // prefill tiles: out's rows start on 16-byte boundaries
  int vec_res;   // the same of residual's
  const float* sa;
  long long ld_sa;
  const float* sw;
  long long ld_sw;
  const float* bias;
  const void* residual;
  long long ld_res;
  void* out;
  long long ld_out;
  int* status;
};

struct Fp8Ctl {
  uint64_t full[kMaxStages];
  uint64_t empty[kMaxStages];
  uint64_t tfull[kAccBufs];
  uint64_t tempty[kAccBufs];
  uint64_t teardown;
  uint32_t tmem_base;
};

// D[tmem] (+)= A[smem] * B[smem]^T, e4m3 x e4m3 -> fp32 (kind::f8f6f4).
__device__ __forceinline__ void mma_e4m3(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Instruction descriptor of kind::f8f6f4: fp32 accumulator (c_format [4,6) =
// 1), e4m3 A and B (formats 0 at [7,10) and [10,13)), both K-major, N >> 3 at
// [17,23), M >> 4 at [24,29).
__host__ __device__ constexpr uint32_t idesc_e4m3(int m, int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ float wide(__half v) { return __half2float(v); }
__device__ __forceinline__ float wide(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void narrow(float v, __half& o) { o = __float2half_rn(v); }
__device__ __forceinline__ void narrow(float v, __nv_bfloat16& o) { o = __float2bfloat16_rn(v); }

__host__ __device__ constexpr uint32_t tmem_cols_for(int nt) { return (uint32_t)(kAccBufs * nt); }

// T: element type of residual and out; NT: tokens per tile.
template <typename T, int NT>
__global__ void __launch_bounds__(kThreads)
    fp8_linear_decode_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
                             const Fp8LinearArgs p) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                                         ~uintptr_t(1023));
  __shared__ Fp8Ctl c;
  __shared__ __align__(16) float s_scale[4][2][NT];  // per epilogue warp, double buffered
  constexpr uint32_t kStageW = kTileN * kBlockK, kStageX = NT * kBlockK;
  unsigned char* ring_w = base;
  unsigned char* ring_x = base + (size_t)p.stages * kStageW;
  constexpr uint32_t kIdesc = idesc_e4m3(kTileN, NT);
  constexpr uint32_t kTmemCols = tmem_cols_for(NT);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)(blockIdx.x % (unsigned)p.split);
  const int tile = (int)(blockIdx.x / (unsigned)p.split);
  const int m_tile = tile / p.n_tiles, n_tile = tile - m_tile * p.n_tiles;
  const int kb0 = (int)((long long)rank * p.k_blocks / p.split);
  const int kb1 = (int)((long long)(rank + 1) * p.k_blocks / p.split);

  if (threadIdx.x == 0) {
    prefetch_tensormap(&tmap_w);
    prefetch_tensormap(&tmap_x);
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(&c.full[i], 1);
      mbar_init(&c.empty[i], 1);
    }
    for (int i = 0; i < kAccBufs; ++i) {
      mbar_init(&c.tfull[i], 1);
      mbar_init(&c.tempty[i], 4);
    }
    mbar_init(&c.teardown, 1);
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&c.tmem_base, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = c.tmem_base;
  pdl_wait();
  pdl_trigger();

  const int quarter = warp & 3;  // TMEM lanes this warp may access
  const int row = quarter * 32 + lane;
  float acc[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) acc[j] = 0.f;

  if (warp == 0) {
    if (lane == 0) {
      const uint64_t pol_w = policy_evict_first();
      const uint64_t pol_x = policy_evict_last();
      int stage = 0, loads = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&c.empty[stage], phase ^ 1, p.status, NPL_DEV_TIMEOUT_TMA)) break;
        mbar_arrive_expect_tx(&c.full[stage], kStageW + kStageX);
        tma_load_2d(ring_w + (size_t)stage * kStageW, &tmap_w, kb * kBlockK, n_tile * kTileN, &c.full[stage], pol_w);
        tma_load_2d(ring_x + (size_t)stage * kStageX, &tmap_x, kb * kBlockK, m_tile * NT, &c.full[stage], pol_x);
        ++loads;
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1;
        }
      }
      // every issued load lands before the ring is used again or released:
      // stage i was last loaded with the parity of that load
      for (int i = 0; i < min(loads, p.stages); ++i)
        mbar_wait(&c.full[i], i < stage ? phase : phase ^ 1, p.status, NPL_DEV_TIMEOUT_TEARDOWN);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        const int i = kb - kb0, buf = i % kAccBufs;
        if (!mbar_wait(&c.tempty[buf], ((i / kAccBufs) & 1) ^ 1, p.status, NPL_DEV_TIMEOUT_MMA)) break;
        if (!mbar_wait(&c.full[stage], phase, p.status, NPL_DEV_TIMEOUT_MMA)) break;
        tc_fence_after();
        const uint32_t a0 = smem_u32(ring_w + (size_t)stage * kStageW);
        const uint32_t b0 = smem_u32(ring_x + (size_t)stage * kStageX);
        const uint32_t d = tmem_base + (uint32_t)(buf * NT);
#pragma unroll
        for (int kk = 0; kk < kBlockK / 32; ++kk)
          mma_e4m3(d, sdesc_k_sw128(a0 + kk * 32), sdesc_k_sw128(b0 + kk * 32), kIdesc, kk > 0 ? 1u : 0u);
        tc_commit(&c.empty[stage]);
        tc_commit(&c.tfull[buf]);
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1;
        }
      }
      // all MMAs issued by this thread complete before the ring and TMEM are given up
      tc_commit(&c.teardown);
      mbar_wait(&c.teardown, 0, p.status, NPL_DEV_TIMEOUT_TEARDOWN);
    }
  } else {
    // Lanes hold the scales of tokens lane and lane + 32 of the next block.
    constexpr int kPer = (NT + 31) / 32;
    float next[kPer], next_sw;
    auto fetch = [&](int kb) {
      next_sw = p.sw[(long long)n_tile * p.ld_sw + kb];
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int m = m_tile * NT + lane + 32 * i;
        next[i] = (lane + 32 * i < NT && m < p.M) ? p.sa[(long long)m * p.ld_sa + kb] : 0.f;
      }
    };
    if (kb0 < kb1) fetch(kb0);
    for (int kb = kb0; kb < kb1; ++kb) {
      const int i = kb - kb0, buf = i % kAccBufs;
      float* sc = s_scale[quarter][i & 1];
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        if (lane + 32 * e < NT) sc[lane + 32 * e] = __fmul_rn(next[e], next_sw);
      __syncwarp();
      if (kb + 1 < kb1) fetch(kb + 1);
      if (!mbar_wait(&c.tfull[buf], (i / kAccBufs) & 1, p.status, NPL_DEV_TIMEOUT_EPILOGUE)) break;
      tc_fence_after();
      const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(buf * NT);
#pragma unroll
      for (int c0 = 0; c0 < NT; c0 += 16) {
        int32_t d[2][8];
        tmem_ld_x8(taddr + c0, d[0]);
        tmem_ld_x8(taddr + c0 + 8, d[1]);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 16; ++j)
          acc[c0 + j] = __fmaf_rn(__int_as_float(d[j / 8][j % 8]), sc[c0 + j], acc[c0 + j]);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&c.tempty[buf]);
    }
  }

  tc_fence_before();
  __syncthreads();  // every copy has landed and every MMA is done: the ring is free
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, kTmemCols);

  const int n = n_tile * kTileN + row;
  int j0 = 0, j1 = NT;
  float* part = reinterpret_cast<float*>(base);  // [NT][128] fp32 sums of this CTA
  if (p.split > 1) {
    if (warp >= 2) {
#pragma unroll
      for (int j = 0; j < NT; ++j) part[j * kTileN + row] = acc[j];
    }
    cluster_arrive_release();
    cluster_wait_acquire();
    j0 = rank * NT / p.split;
    j1 = (rank + 1) * NT / p.split;
  }
  if (warp >= 2 && n < p.N) {
    const T* res = static_cast<const T*>(p.residual);
    T* out = static_cast<T*>(p.out);
    const float b = p.bias ? p.bias[n] : 0.f;
    auto finish = [&](int j, float v) {
      const long long m = (long long)m_tile * NT + j;
      if (m >= p.M) return;
      if (p.bias) v = __fadd_rn(v, b);
      if (res) v = __fadd_rn(v, wide(res[m * p.ld_res + n]));
      narrow(v, out[m * p.ld_out + n]);
    };
    if (p.split > 1) {
      for (int j = j0; j < j1; ++j) {
        float v = 0.f;
        for (int r = 0; r < p.split; ++r) {
          const float x = ld_cluster_f32(cluster_map(part + j * kTileN + row, (uint32_t)r));
          v = r == 0 ? x : __fadd_rn(v, x);
        }
        finish(j, v);
      }
    } else {
#pragma unroll
      for (int j = 0; j < NT; ++j) finish(j, acc[j]);
    }
  }
  if (p.split > 1) {  // no CTA's shared memory is given up while another reads it
    cluster_arrive_release();
    cluster_wait_acquire();
  }
}

// ------------------------------------------------------------- prefill tiles
//
// Tokens are the MMA's A rows and weights its N columns here: a thread of the
// epilogue holds one token, so a block's scale is one value per thread and 128
// columns (one weight scale), and the update is one packed FMA for two sums.
// Per CTA (384 threads, one CTA per SM, persistent over 128 x 256 tiles): warp
// 0 TMA, warp 1 MMA, warps 4-7 and 8-11 the epilogue of 128 columns each, with
// all of its sums (128 a thread) in registers: the first warpgroup hands most
// of its registers to the other two. Two 256-column accumulators fill TMEM:
// the MMAs of a block run while the epilogue adds up the one before.
constexpr int kPM = 128;   // tokens per tile
constexpr int kPN = 256;   // weight rows per tile
constexpr int kPThreads = 384;
// 168 a thread at launch; 48 + 2 * 224 <= 3 * 168
constexpr int kPRegsFew = 48, kPRegsMany = 224;
constexpr int kPStages = 4;
constexpr uint32_t kPStageX = kPM * kBlockK, kPStageW = kPN * kBlockK;
constexpr uint32_t kPStage = kPStageX + kPStageW;
constexpr int kPOutCols = 64;                         // columns staged at a time by a warpgroup
constexpr uint32_t kPOut = kPM * kPOutCols * 2;       // 16 KB
constexpr int kPSmem = kPStages * (int)kPStage + 2 * (int)kPOut + 1024;

struct PrefillCtl {
  uint64_t full[kPStages];
  uint64_t empty[kPStages];
  uint64_t tfull[2];
  uint64_t tempty[2];
  uint64_t teardown;
  uint32_t tmem_base;
};

__device__ __forceinline__ void tmem_ld_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

// tcgen05.wait::ld that the loaded registers pass through, so that no use of
// them can be moved before it.
__device__ __forceinline__ void tmem_wait_regs(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                 "+r"(r[15])::"memory");
}

__device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(lo), "r"(hi));
  return v;
}

__device__ __forceinline__ float2 unpack2(uint64_t v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}

// Two fp32 FMAs in one instruction.
__device__ __forceinline__ void fma2(uint64_t& acc, uint64_t a, uint64_t b) {
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(a), "l"(b));
}

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* smem, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(c0), "r"(c1), "r"(smem_u32(smem))
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}

__device__ __forceinline__ void tma_store_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}

// Tile t -> (token tile, weight tile): groups of raster_g token tiles, the
// token tile running fastest, so that the tiles in flight at one time share
// raster_g token tiles and 148 / raster_g weight tiles in L2.
__device__ __forceinline__ void prefill_tile(const Fp8LinearArgs& p, int t, int& m_tile, int& n_tile) {
  const int span = p.raster_g * p.n_tiles;
  const int grp = t / span, r = t - grp * span;
  const int m0 = grp * p.raster_g;
  const int gs = min(p.raster_g, p.m_tiles - m0);
  m_tile = m0 + r % gs;
  n_tile = r / gs;
}

template <typename T>
__device__ __forceinline__ uint32_t narrow2(float a, float b) {
  T v[2];
  narrow(a, v[0]);
  narrow(b, v[1]);
  uint32_t u;
  memcpy(&u, v, 4);
  return u;
}

template <typename T>
__global__ void __launch_bounds__(kPThreads, 1)
    fp8_linear_prefill_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w,
                              const __grid_constant__ CUtensorMap tmap_out, const Fp8LinearArgs p) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                                         ~uintptr_t(1023));
  unsigned char* staging = ring + kPStages * kPStage;
  __shared__ PrefillCtl c;
  constexpr uint32_t kIdesc = idesc_e4m3(kPM, kPN);
  constexpr uint32_t kTmemCols = 2 * kPN;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles = p.m_tiles * p.n_tiles;

  if (threadIdx.x == 0) {
    prefetch_tensormap(&tmap_x);
    prefetch_tensormap(&tmap_w);
    prefetch_tensormap(&tmap_out);
    for (int i = 0; i < kPStages; ++i) {
      mbar_init(&c.full[i], 1);
      mbar_init(&c.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&c.tfull[i], 1);
      mbar_init(&c.tempty[i], 8);
    }
    mbar_init(&c.teardown, 1);
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&c.tmem_base, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = c.tmem_base;
  pdl_wait();
  pdl_trigger();

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPRegsFew));
    if (warp == 0 && lane == 0) {
      const uint64_t pol = policy_evict_normal();
      int stage = 0, loads = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
        int m_tile, n_tile;
        prefill_tile(p, t, m_tile, n_tile);
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          if (!mbar_wait(&c.empty[stage], phase ^ 1, p.status, NPL_DEV_TIMEOUT_TMA)) {
            ok = false;
            break;
          }
          unsigned char* at = ring + (size_t)stage * kPStage;
          mbar_arrive_expect_tx(&c.full[stage], kPStage);
          tma_load_2d(at, &tmap_x, kb * kBlockK, m_tile * kPM, &c.full[stage], pol);
          tma_load_2d(at + kPStageX, &tmap_w, kb * kBlockK, n_tile * kPN, &c.full[stage], pol);
          loads = min(loads + 1, kPStages);
          if (++stage == kPStages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      for (int i = 0; i < loads; ++i)  // every issued load lands before the ring is released
        mbar_wait(&c.full[i], i < stage ? phase : phase ^ 1, p.status, NPL_DEV_TIMEOUT_TEARDOWN);
    } else if (warp == 1 && lane == 0) {
      int stage = 0;
      uint32_t phase = 0, it = 0;
      bool ok = true;
      for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
        for (int kb = 0; kb < p.k_blocks; ++kb, ++it) {
          const uint32_t buf = it & 1;
          if (!mbar_wait(&c.tempty[buf], ((it >> 1) & 1) ^ 1, p.status, NPL_DEV_TIMEOUT_MMA) ||
              !mbar_wait(&c.full[stage], phase, p.status, NPL_DEV_TIMEOUT_MMA)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a0 = smem_u32(ring + (size_t)stage * kPStage), b0 = a0 + kPStageX;
#pragma unroll
          for (int kk = 0; kk < kBlockK / 32; ++kk)
            mma_e4m3(tmem_base + buf * kPN, sdesc_k_sw128(a0 + kk * 32), sdesc_k_sw128(b0 + kk * 32), kIdesc,
                     kk > 0 ? 1u : 0u);
          tc_commit(&c.empty[stage]);
          tc_commit(&c.tfull[buf]);
          if (++stage == kPStages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      tc_commit(&c.teardown);  // all MMAs complete before TMEM is freed
      mbar_wait(&c.teardown, 0, p.status, NPL_DEV_TIMEOUT_TEARDOWN);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPRegsMany));
    const int group = (warp - 4) >> 2;  // columns [128 group, 128 group + 128) of the tile
    const int row = (warp & 3) * 32 + lane;
    const bool elected = (int)threadIdx.x == 128 + 128 * group;
    unsigned char* stg = staging + group * kPOut;
    auto group_bar = [&] { asm volatile("bar.sync %0, 128;" ::"r"(1 + group) : "memory"); };
    const T* res = static_cast<const T*>(p.residual);
    T* out = static_cast<T*>(p.out);
    uint32_t it = 0;
    bool ok = true;
    for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
      int m_tile, n_tile;
      prefill_tile(p, t, m_tile, n_tile);
      const int m = m_tile * kPM + row;
      const int n0 = n_tile * kPN + group * 128;
      const bool live = m < p.M && n0 < p.N;
      const float* sa = p.sa + (live ? (long long)m * p.ld_sa : 0);
      const float* sw = p.sw + (live ? (long long)(n0 / kTileN) * p.ld_sw : 0);
      uint64_t acc[64];
#pragma unroll
      for (int j = 0; j < 64; ++j) acc[j] = 0;
      float s_next = live ? __fmul_rn(sa[0], sw[0]) : 0.f;
      for (int kb = 0; kb < p.k_blocks; ++kb, ++it) {
        const uint32_t buf = it & 1;
        const uint32_t sbits = __float_as_uint(s_next);
        const uint64_t s2 = pack2(sbits, sbits);
        if (live && kb + 1 < p.k_blocks) s_next = __fmul_rn(sa[kb + 1], sw[kb + 1]);
        if (!mbar_wait(&c.tfull[buf], (it >> 1) & 1, p.status, NPL_DEV_TIMEOUT_EPILOGUE)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t taddr = tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + buf * kPN + group * 128;
        uint32_t d[2][16];
        tmem_ld_x16(taddr, d[0]);
        tmem_wait_regs(d[0]);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          if (q < 7) tmem_ld_x16(taddr + (q + 1) * 16, d[(q + 1) & 1]);
#pragma unroll
          for (int j = 0; j < 8; ++j) fma2(acc[q * 8 + j], pack2(d[q & 1][2 * j], d[q & 1][2 * j + 1]), s2);
          if (q < 7) tmem_wait_regs(d[(q + 1) & 1]);
          if (q == 6) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&c.tempty[buf]);
          }
        }
      }
      if (!ok) break;
      // bias, residual, rounding; 64 columns at a time through shared memory
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int nh = n0 + h * kPOutCols;
        if (elected) tma_store_wait_read();
        group_bar();  // the staging buffer is free
#pragma unroll
        for (int ch = 0; ch < 8; ++ch) {
          float v[8];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = unpack2(acc[h * 32 + ch * 4 + j]);
            v[2 * j] = f.x;
            v[2 * j + 1] = f.y;
          }
          const int n = nh + ch * 8;
          if (p.bias) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (n + j < p.N) v[j] = __fadd_rn(v[j], p.bias[n + j]);
          }
          if (res && m < p.M) {
            const T* r = res + (long long)m * p.ld_res + n;
            if (p.vec_res && n + 8 <= p.N) {
              const uint4 raw = *reinterpret_cast<const uint4*>(r);
              T e[8];
              memcpy(e, &raw, 16);
#pragma unroll
              for (int j = 0; j < 8; ++j) v[j] = __fadd_rn(v[j], wide(e[j]));
            } else {
#pragma unroll
              for (int j = 0; j < 8; ++j)
                if (n + j < p.N) v[j] = __fadd_rn(v[j], wide(r[j]));
            }
          }
          uint4 o;
          o.x = narrow2<T>(v[0], v[1]);
          o.y = narrow2<T>(v[2], v[3]);
          o.z = narrow2<T>(v[4], v[5]);
          o.w = narrow2<T>(v[6], v[7]);
          // the 128-byte swizzle of the output's tensor map
          *reinterpret_cast<uint4*>(stg + row * 128 + ((ch ^ (row & 7)) << 4)) = o;
        }
        if (p.tma_out) {
          fence_proxy_async_smem();
          group_bar();
          if (elected && nh < p.N) tma_store_2d(&tmap_out, stg, nh, m_tile * kPM);
        } else {  // rows that TMA cannot store: element by element, 32 columns a warp
          group_bar();
          for (int r = (warp & 3); r < kPM; r += 4) {
            const long long mr = (long long)m_tile * kPM + r;
            if (mr >= p.M) break;
#pragma unroll
            for (int e = lane; e < kPOutCols; e += 32)
              if (nh + e < p.N)
                out[mr * p.ld_out + nh + e] =
                    *reinterpret_cast<const T*>(stg + r * 128 + (((e >> 3) ^ (r & 7)) << 4) + (e & 7) * 2);
          }
        }
      }
    }
    if (elected) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

// ------------------------------------------------------------------ host
PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    cudaDriverEntryPointQueryResult q;
    void* f = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  }();
  return fn;
}

// e4m3 row-major [rows, cols] with row stride ld bytes; box [box_rows, 128 B].
// Elements past the edges read as zero, which is the code of 0.
int code_map(CUtensorMap* map, const void* base, long long rows, long long cols, long long ld, int box_rows) {
  auto fn = tensor_map_encoder();
  if (!fn) return fail(NPL_ERR_LAUNCH, "npl_fp8_linear: cuTensorMapEncodeTiled unavailable");
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld};
  const cuuint32_t box[2] = {(cuuint32_t)kBlockK, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(NPL_ERR_ARG, "npl_fp8_linear: cuTensorMapEncodeTiled failed (%d)", (int)r);
  return NPL_OK;
}

struct Operands {
  const void *qa, *qw;
  long long lda, ldw, K;
  int out_dtype;
};

// Shared memory of a decode CTA. More than a third of an SM's, so that at
// most two CTAs share an SM: their TMEM (at most 2 x 256 columns) then always
// fits, and no CTA of a cluster waits for TMEM that a CTA of another cluster
// holds.
constexpr int kDecodeSmemMin = 78 * 1024;
constexpr int kDecodeSmemMax = 110 * 1024;

template <typename T, int NT>
int launch_decode(const Operands& o, Fp8LinearArgs& p, cudaStream_t st) {
  CUtensorMap tw, tx;
  if (int rc = code_map(&tw, o.qw, p.N, o.K, o.ldw, kTileN)) return rc;
  if (int rc = code_map(&tx, o.qa, p.M, o.K, o.lda, NT)) return rc;
  constexpr int stage = (kTileN + NT) * kBlockK;
  p.stages = std::min(kMaxStages, (kDecodeSmemMax - 1024) / stage);
  const int smem = std::max(p.stages * stage + 1024, kDecodeSmemMin);
  const long long m_tiles = (p.M + NT - 1) / NT;
  const long long tiles = m_tiles * p.n_tiles;
  p.split = 1;
  while (p.split < kMaxSplit && tiles * p.split * 2 <= 2ll * num_sms() && p.split * 2 <= p.k_blocks) p.split *= 2;
  if (tiles * p.split > 2147483647ll)
    return fail(NPL_ERR_UNSUPPORTED, "npl_fp8_linear: M=%d N=%d has too many tiles", p.M, p.N);
  auto kern = fp8_linear_decode_kernel<T, NT>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kDecodeSmemMax) != cudaSuccess)
    return launch_status("npl_fp8_linear: smem attribute");
  return launch_pdl_cluster("npl_fp8_linear", kern, dim3((unsigned)(tiles * p.split)), dim3(kThreads), (size_t)smem,
                            st, (unsigned)p.split, tw, tx, p);
}

// Row-major [rows, cols] of a 16-bit type with row stride ld, in boxes of 128 rows x 64 columns.
int out_map(CUtensorMap* map, void* base, int dtype, long long rows, long long cols, long long ld) {
  auto fn = tensor_map_encoder();
  if (!fn) return fail(NPL_ERR_LAUNCH, "npl_fp8_linear: cuTensorMapEncodeTiled unavailable");
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  const cuuint32_t box[2] = {(cuuint32_t)kPOutCols, (cuuint32_t)kPM};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = fn(map, dtype == NPL_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                        base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(NPL_ERR_ARG, "npl_fp8_linear: cuTensorMapEncodeTiled failed (%d)", (int)r);
  return NPL_OK;
}

template <typename T>
int launch_prefill(const Operands& o, Fp8LinearArgs& p, cudaStream_t st) {
  CUtensorMap tx, tw, to;
  if (int rc = code_map(&tx, o.qa, p.M, o.K, o.lda, kPM)) return rc;
  if (int rc = code_map(&tw, o.qw, p.N, o.K, o.ldw, kPN)) return rc;
  p.tma_out = aligned16(p.out) && p.ld_out % 8 == 0;
  p.vec_res = aligned16(p.residual) && p.ld_res % 8 == 0;
  to = tx;
  if (p.tma_out)
    if (int rc = out_map(&to, p.out, o.out_dtype, p.M, p.N, p.ld_out)) return rc;
  p.m_tiles = (p.M + kPM - 1) / kPM;
  p.n_tiles = (p.N + kPN - 1) / kPN;
  const long long tiles = (long long)p.m_tiles * p.n_tiles;
  if (tiles > 1ll << 30)
    return fail(NPL_ERR_UNSUPPORTED, "npl_fp8_linear: M=%d N=%d has too many tiles", p.M, p.N);
  p.raster_g = std::min(16, p.m_tiles);
  auto kern = fp8_linear_prefill_kernel<T>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kPSmem) != cudaSuccess)
    return launch_status("npl_fp8_linear: smem attribute");
  return launch_pdl("npl_fp8_linear", kern, dim3((unsigned)std::min<long long>(tiles, num_sms())), dim3(kPThreads),
                    (size_t)kPSmem, st, tx, tw, to, p);
}

template <typename T>
int launch(const Operands& o, Fp8LinearArgs& p, cudaStream_t st) {
  if (p.M > 64) return launch_prefill<T>(o, p, st);
  if (p.M <= 16) return launch_decode<T, 16>(o, p, st);
  if (p.M <= 32) return launch_decode<T, 32>(o, p, st);
  return launch_decode<T, 64>(o, p, st);
}

}  // namespace
}  // namespace npl

using namespace npl;

extern "C" int npl_fp8_linear(const uint8_t* qa, int64_t lda, const float* sa, int64_t ld_sa, const uint8_t* qw,
                              int64_t ldw, const float* sw, int64_t ld_sw, const float* bias, int64_t M, int64_t N,
                              int64_t K, const void* residual, int64_t ld_res, void* out, int64_t ld_out,
                              int out_dtype, void* stream) {
  constexpr int64_t kMax = 2147483647ll - 2 * kTileN;
  if (M < 0 || N <= 0 || K <= 0 || M > kMax || N > kMax || K > kMax)
    return fail(NPL_ERR_ARG, "npl_fp8_linear: bad shape M=%lld N=%lld K=%lld", (long long)M, (long long)N,
                (long long)K);
  const int64_t kb = (K + kBlockK - 1) / kBlockK;
  if (!qw || !sw || (M > 0 && (!qa || !sa || !out))) return fail(NPL_ERR_ARG, "npl_fp8_linear: null pointer");
  if (!aligned16(qa) || !aligned16(qw) || lda < K || ldw < K || lda % 16 || ldw % 16)
    return fail(NPL_ERR_ARG,
                "npl_fp8_linear: codes need 16-byte aligned rows (lda=%lld, ldw=%lld: multiples of 16, >= K)",
                (long long)lda, (long long)ldw);
  if (ld_sa < kb || ld_sw < kb)
    return fail(NPL_ERR_ARG, "npl_fp8_linear: scale rows need %lld values (ld_sa=%lld, ld_sw=%lld)", (long long)kb,
                (long long)ld_sa, (long long)ld_sw);
  if (out_dtype != NPL_F16 && out_dtype != NPL_BF16)
    return fail(NPL_ERR_ARG, "npl_fp8_linear: out_dtype must be NPL_F16 or NPL_BF16");
  if (ld_out < N || (residual && ld_res < N))
    return fail(NPL_ERR_ARG, "npl_fp8_linear: row strides of out and residual must be >= N");
  if ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(residual)) & 1u ||
      (reinterpret_cast<uintptr_t>(sa) | reinterpret_cast<uintptr_t>(sw) | reinterpret_cast<uintptr_t>(bias)) & 3u)
    return fail(NPL_ERR_ARG, "npl_fp8_linear: a pointer is not aligned to its elements");
  if (M == 0) return NPL_OK;
  if (int rc = check_device()) return rc;
  Fp8LinearArgs p{};
  p.M = (int)M;
  p.N = (int)N;
  p.k_blocks = (int)kb;
  p.n_tiles = (int)((N + kTileN - 1) / kTileN);
  p.sa = sa;
  p.ld_sa = ld_sa;
  p.sw = sw;
  p.ld_sw = ld_sw;
  p.bias = bias;
  p.residual = residual;
  p.ld_res = ld_res;
  p.out = out;
  p.ld_out = ld_out;
  p.status = device_status_ptr();
  const Operands o{qa, qw, lda, ldw, K, out_dtype};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return out_dtype == NPL_F16 ? launch<__half>(o, p, st) : launch<__nv_bfloat16>(o, p, st);
}
