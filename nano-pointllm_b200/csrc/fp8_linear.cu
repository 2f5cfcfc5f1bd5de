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
// Decode tiles (M <= 64, some M <= 128): the weight tile is the MMA's A operand and the tokens
// are its N dimension (D[n, m], 128 weight rows x NT tokens), so a decode
// batch fills an MMA with NT = 16..64. Prefill tiles: see below.
//
// Per decode CTA (192 threads):
//   warp 0     TMA producer: weight tile [128 x 128 B] and token tile
//              [NT x 128 B] per block, 128-byte swizzle, a ring of stages
//   warp 1     TMEM owner + MMA issuer: 4 MMAs of K = 32 per block, a ring of
//              4 units of 64 columns, which hold 64 / NT blocks each
//   warps 2-5  TMEM lane = weight row, column = token: acc += (sa sw) * D, a
//              unit at a time (waiting for every block of 16 tokens took longer
//              than adding it up)
//
// Split over K: the S CTAs of a thread-block cluster share a tile's blocks.
// Each leaves its fp32 sums in its own shared memory; after a cluster barrier
// CTA r adds those of ranks 0, 1, .. S - 1, in this order, for its share of
// the tokens. No workspace and no atomics: two calls in flight share nothing,
// and equal calls give equal bits.
//
// All mbarrier waits are bounded (~1 s); on expiry the kernel records a code
// in the device status word, drains its in-flight copies and MMAs, meets its
// cluster, frees TMEM and returns. Warps that meet at named barriers do so
// whether or not their waits ran out (fp8_epilogue.cuh).
#include <cuda_bf16.h>
#include <cudaTypedefs.h>

#include <algorithm>

#include "fp8_epilogue.cuh"
#include "npl_common.cuh"

namespace npl {
namespace {

constexpr int kTileN = 128;   // weight rows per tile (MMA M) and per scale
constexpr int kBlockK = 128;  // columns per scale = bytes per stage row (one 128-byte swizzle atom)
constexpr int kThreads = 192;
constexpr int kMaxStages = 6;
constexpr int kUnitCols = 64;  // TMEM columns handed over at a time: 64 / NT blocks
constexpr int kUnits = 4;     // TMEM ring: 256 columns
constexpr int kMaxSplit = 8;
constexpr int kScaleBlocks = 32;  // blocks whose scales a decode CTA holds at a time

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
  uint64_t tfull[kUnits];
  uint64_t tempty[kUnits];
  uint64_t teardown;
  uint32_t tmem_base;
};

// D[tmem] (+)= A[smem] * B[smem]^T, e4m3 x e4m3 -> fp32 (kind::f8f6f4).
template <bool kAccumulate>
__device__ __forceinline__ void mma_e4m3(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "n"((int)kAccumulate)
      : "memory");
}

// One lane of the warp, the same each time.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one != 0;
}

// mbar_wait of a whole warp, the same in all lanes. It looks at the clock only
// after many polls (of 20 ns or more): where every block waits, reading it
// takes longer than most waits. kVote: the lanes vote on every poll, which is
// faster in the decode kernel (32 x 12288 x 4096: 15.5 us, without 16.4) and slower
// in the prefill kernel (16000 x 22016 x 4096: 1568 us, without 1530).
template <bool kVote>
__device__ __forceinline__ bool poll_wait(uint64_t* bar, uint32_t parity, int* status, int code) {
  uint64_t t0 = 0;
  auto try_once = [&] { return mbar_try_wait(bar, parity); };
  auto late = [&] {
    const uint64_t t = globaltimer_ns();
    if (t0 == 0) t0 = t;
    return t - t0 > kWaitLimitNs;
  };
  bool done;
  if constexpr (kVote)
    done = wait_voting(1024, try_once, [](bool v) { return __all_sync(0xffffffffu, v) != 0; }, late);
  else
    done = wait_as_one(1024, try_once, [](bool v) { return __any_sync(__activemask(), v) != 0; }, late);
  if (!done && status) atomicExch(status, code);
  return done;
}

// Whether ok holds in all 128 threads of a warpgroup, which meet at barrier `id`.
__device__ __forceinline__ bool warpgroup_agrees(int id, bool ok) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %2, 0;\n\t"
      "barrier.cta.red.and.pred q, %1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"(id), "r"((uint32_t)ok)
      : "memory");
  return all != 0;
}

// Instruction descriptor of kind::f8f6f4: fp32 accumulator (c_format [4,6) =
// 1), e4m3 A and B (formats 0 at [7,10) and [10,13)), both K-major, N >> 3 at
// [17,23), M >> 4 at [24,29).
__host__ __device__ constexpr uint32_t idesc_e4m3(int m, int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// acc += d * s. Volatile, like tcgen05.ld and its wait: it stays behind the
// wait for d. (The packed fma.rn.f32x2 has the same rate on B200, 128 FMAs a
// cycle and SM, and its operand pairs cost moves: 1810 us against 1511 for
// 16000 x 22016 x 4096.)
__device__ __forceinline__ void fma_after_ld(float& acc, uint32_t d, float s) {
  asm volatile("fma.rn.f32 %0, %1, %2, %0;" : "+f"(acc) : "f"(__uint_as_float(d)), "f"(s));
}

__device__ __forceinline__ void tma_prefetch_l2(const CUtensorMap* map, int c0, int c1) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(c0), "r"(c1)
               : "memory");
}

__device__ __forceinline__ void lds128(const float* p, float* v) {
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3])
               : "r"(smem_u32(p))
               : "memory");
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

// T: element type of residual and out; NT: tokens per tile.
template <typename T, int NT>
__global__ void __launch_bounds__(kThreads, 2)
    fp8_linear_decode_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
                             const Fp8LinearArgs p) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                                         ~uintptr_t(1023));
  __shared__ Fp8Ctl c;
  __shared__ __align__(16) float s_scale[kScaleBlocks][NT + 4];  // the tokens' scales times the weight's, by block
  constexpr int U = kUnitCols / NT;  // blocks per unit
  constexpr uint32_t kStageW = kTileN * kBlockK, kStageX = NT * kBlockK;
  unsigned char* ring_w = base;
  unsigned char* ring_x = base + (size_t)p.stages * kStageW;
  constexpr uint32_t kIdesc = idesc_e4m3(kTileN, NT);
  constexpr uint32_t kTmemCols = kUnits * kUnitCols;

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
    for (int i = 0; i < kUnits; ++i) {
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
  pdl_trigger();

  const int quarter = warp & 3;  // TMEM lanes this warp may access
  const int row = quarter * 32 + lane;
  float acc[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) acc[j] = 0.f;

  if (warp == 0) {
    // As warp 1, all lanes run the loop and one issues: the copies' operands
    // stay in uniform registers.
    const bool issuer = elect_one();
    const uint64_t pol_w = policy_evict_first();
    const uint64_t pol_x = policy_evict_last();
    // Before the kernels ahead of this one on its stream are done nothing may
    // be read, not even weights, which one of them may have written. But their
    // first tiles may be brought into L2, where such a write would meet them.
    const int ahead = min(p.stages, kb1 - kb0);
    for (int i = 0; i < ahead; ++i)
      if (issuer) tma_prefetch_l2(&tmap_w, (kb0 + i) * kBlockK, n_tile * kTileN);
    pdl_wait();
    int stage = 0, loads = 0;
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!poll_wait<true>(&c.empty[stage], phase ^ 1, p.status, NPL_DEV_TIMEOUT_TMA)) break;
      if (issuer) {
        mbar_arrive_expect_tx(&c.full[stage], kStageW + kStageX);
        tma_load_2d(ring_w + (size_t)stage * kStageW, &tmap_w, kb * kBlockK, n_tile * kTileN, &c.full[stage], pol_w);
        tma_load_2d(ring_x + (size_t)stage * kStageX, &tmap_x, kb * kBlockK, m_tile * NT, &c.full[stage], pol_x);
      }
      loads = min(loads + 1, p.stages);
      if (++stage == p.stages) {
        stage = 0;
        phase ^= 1;
      }
    }
    // every issued load lands before the ring is used again or released: stage
    // i was last loaded with the parity of that load
    for (int i = 0; i < loads; ++i)
      poll_wait<true>(&c.full[i], i < stage ? phase : phase ^ 1, p.status, NPL_DEV_TIMEOUT_TEARDOWN);
    __syncwarp();
  } else if (warp == 1) {
    // The whole warp runs this loop and one lane issues, so that descriptors
    // stay in uniform registers (see the prefill kernel).
    const bool issuer = elect_one();
    const uint64_t desc_w = sdesc_k_sw128(smem_u32(ring_w)), desc_x = sdesc_k_sw128(smem_u32(ring_x));
    int stage = 0;
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      const int i = kb - kb0, unit = i / U, buf = unit % kUnits, u = i % U;
      if (!poll_wait<true>(&c.full[stage], phase, p.status, NPL_DEV_TIMEOUT_MMA)) break;
      if (u == 0 && !poll_wait<true>(&c.tempty[buf], ((unit / kUnits) & 1) ^ 1, p.status, NPL_DEV_TIMEOUT_MMA)) break;
      tc_fence_after();
      const uint64_t a = desc_w + (uint32_t)stage * (kStageW >> 4), b = desc_x + (uint32_t)stage * (kStageX >> 4);
      const uint32_t d = tmem_base + (uint32_t)(buf * kUnitCols + u * NT);
      if (issuer) {
        mma_e4m3<false>(d, a, b, kIdesc);
#pragma unroll
        for (int kk = 1; kk < kBlockK / 32; ++kk) mma_e4m3<true>(d, a + kk * 2, b + kk * 2, kIdesc);
        if (u == U - 1 || kb + 1 == kb1) tc_commit(&c.tfull[buf]);
        tc_commit(&c.empty[stage]);
      }
      __syncwarp();
      if (++stage == p.stages) {
        stage = 0;
        phase ^= 1;
      }
    }
    // all MMAs issued complete before the ring and TMEM are given up
    if (issuer) tc_commit(&c.teardown);
    poll_wait<true>(&c.teardown, 0, p.status, NPL_DEV_TIMEOUT_TEARDOWN);
    __syncwarp();
  } else {
    pdl_wait();
    // The scales of the next kScaleBlocks blocks: a warp reads a token's with
    // one load, all loads of a thread at once.
    auto scales = [&](int kc) {
      const int b = kc + lane;
      const float w = b < kb1 ? p.sw[(long long)n_tile * p.ld_sw + b] : 0.f;
      float a[NT / 4];
#pragma unroll
      for (int i = 0; i < NT / 4; ++i) {
        const int m = m_tile * NT + 4 * i + quarter;
        a[i] = b < kb1 && m < p.M ? p.sa[(long long)m * p.ld_sa + b] : 0.f;
      }
      if (kc > kb0) asm volatile("bar.sync 1, 128;" ::: "memory");  // the scales before are read
#pragma unroll
      for (int i = 0; i < NT / 4; ++i) s_scale[lane][4 * i + quarter] = __fmul_rn(a[i], w);
      asm volatile("bar.sync 1, 128;" ::: "memory");
    };
    auto add_unit = [&](int unit, int, int k, int kn) {
      const int buf = unit % kUnits;
      if (!poll_wait<true>(&c.tfull[buf], (unit / kUnits) & 1, p.status, NPL_DEV_TIMEOUT_EPILOGUE)) return false;
      tc_fence_after();
      const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(buf * kUnitCols);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float sc[32];  // loaded ahead of their uses
#pragma unroll
        for (int q = 0; q < 32; q += 4) {
          const int at = 32 * h + q;
          lds128(&s_scale[k + at / NT][at % NT], sc + q);
        }
        uint32_t d[32];
        tmem_ld_x32(taddr + 32 * h, d);
        tmem_wait_ld();
        if (h == 1) {  // the unit is read
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&c.tempty[buf]);
        }
#pragma unroll
        for (int q = 0; q < 32; ++q) {
          const int at = 32 * h + q;  // block at / NT, which a last unit may lack: what TMEM holds there is not used
          if (at % NT == 0 && k + at / NT >= kn) break;
          fma_after_ld(acc[at % NT], d[q], sc[q]);
        }
      }
      return true;
    };
    decode_epilogue(kb0, kb1, kScaleBlocks, U, scales, add_unit);
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
        float x[kMaxSplit];  // all ranks' loads at once
#pragma unroll
        for (int r = 0; r < kMaxSplit; ++r)
          if (r < p.split) x[r] = ld_cluster_f32(cluster_map(part + j * kTileN + row, (uint32_t)r));
        float v = x[0];
#pragma unroll
        for (int r = 1; r < kMaxSplit; ++r)
          if (r < p.split) v = __fadd_rn(v, x[r]);
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
// columns (one weight scale; two where they straddle blocks of a 192-row tile),
// and the update is one FMA a sum.
//
// Two CTAs of a cluster share a tile of 256 tokens x 256 weight rows
// (cta_group::2): each loads 128 rows of both, CTA 0 issues the MMAs for both,
// and each holds the accumulator of its 128 tokens. (Or x 192 weight rows; see
// launch_prefill.) An SM takes in about 58
// bytes a cycle from L2 (measured), and a block's MMAs run 512 cycles; a CTA
// of its own with a 128 x 256 tile needs 48 KB for a block and waits for them,
// one of a pair 32 KB.
//
// Per CTA (384 threads, one CTA per SM, persistent): warp 0 TMA, warp 1 MMA,
// warps 2-3 the scales, two warpgroups the epilogue of half the columns each, with
// all of its sums in registers (128 a thread, or 96; the first warpgroup hands most
// of its registers to the other two). Two 256-column accumulators fill TMEM:
// the MMAs of a block run while the epilogue adds up the one before, so the
// block's whole round (MMAs, hand-over, TMEM loads, hand-back) has to fit into
// the time of two blocks' MMAs. What counts there is instructions: four
// warpgroups of 64 columns spend as many on waiting and scales as on sums.
// The scales' products go through shared memory, 8 blocks at a time: read by
// the threads that use them, every load would touch 32 rows, and these loads
// alone took as long as the MMAs.
constexpr int kPM = 128;   // tokens per CTA
constexpr int kPGroups = 2;  // epilogue warpgroups
constexpr int kPThreads = 128 + 128 * kPGroups;
// 168 a thread at launch (65536 / 384); 56 + 2 * 224 = 3 * 168
constexpr int kPRegsFew = 56, kPRegsMany = 224;
constexpr uint32_t kPStageX = kPM * kBlockK;
constexpr uint32_t kPAccCols = 256;  // TMEM columns from one accumulator to the other
constexpr int kPScaleBlocks = 8;     // blocks of scales loaded at a time
constexpr int kPScaleLd = kPM + 4;   // a warp's 8 blocks x 4 tokens hit 32 banks

// What follows from a tile's weight rows, 256 or 192.
template <int kPN>
struct PrefillTile {
  static constexpr int kGroupCols = kPN / kPGroups;
  static constexpr int kStages = kPN == 256 ? 5 : 6;
  static constexpr uint32_t kStageW = kPN / 2 * kBlockK;
  static constexpr uint32_t kStage = kPStageX + kStageW;
  static constexpr int kOutCols = kPN == 256 ? 64 : 32;     // columns staged at a time by a warpgroup
  static constexpr uint32_t kOut = kPM * kOutCols * 2;
  static constexpr int kSmem = kStages * (int)kStage + kPGroups * (int)kOut + 1024;
};

template <int kPStages>
struct PrefillCtl {
  uint64_t full[kPStages];   // CTA 0's: both CTAs' loads of a stage
  uint64_t empty[kPStages];
  uint64_t tfull[2];
  uint64_t tempty[2];        // CTA 0's: both CTAs' epilogue warps
  uint64_t sfull[2];
  uint64_t sempty[2];
  uint64_t teardown;
  uint32_t tmem_base;
  __align__(16) float scale[2][2][kPScaleBlocks][kPScaleLd];  // with each of the tile's two weight scales
};

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

// TMA load into this CTA's shared memory, counted on a barrier of either CTA
// of the pair (a shared::cluster address).
__device__ __forceinline__ void tma_load_2d_pair(void* smem_dst, const CUtensorMap* map, int c0, int c1,
                                                 uint32_t bar_cluster, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2.L2::cache_hint"
      " [%0], [%1, {%2, %3}], [%4], %5;" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar_cluster), "l"(policy)
      : "memory");
}

// The pair's MMA: 256 x N, rows 0-127 in CTA 0's TMEM, the others in CTA 1's.
template <bool kAccumulate>
__device__ __forceinline__ void mma_e4m3_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "n"((int)kAccumulate)
      : "memory");
}

// Completion of the MMAs issued so far arrives on this barrier in both CTAs
// (`mask`: their ranks in the cluster, as bits).
__device__ __forceinline__ void tc_commit_pair(uint64_t* bar, uint16_t mask) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"(mask)
      : "memory");
}

// One arrival on a barrier of either CTA of the pair. It carries no ordinary
// memory from CTA to CTA (TMEM reads are ordered by the tcgen05 fences), so it
// and the waits need no cluster scope, which costs a fence each: with it a
// block took 1.4 us.
__device__ __forceinline__ void mbar_arrive_pair(uint32_t bar_cluster) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar_cluster) : "memory");
}

// Byte offset of 16-byte chunk `ch` of row `row` in a staged box of 128- or
// 64-byte rows: the swizzle of the output's tensor map.
template <int kOutCols>
__device__ __forceinline__ int staged(int row, int ch) {
  if constexpr (kOutCols == 64) return row * 128 + ((ch ^ (row & 7)) << 4);
  return row * 64 + ((ch ^ ((row >> 1) & 3)) << 4);
}

// Tile t -> (token tile, weight tile): groups of raster_g token tiles, the
// token tile running fastest, so that the tiles in flight at one time share
// raster_g token tiles and 74 / raster_g weight tiles in L2.
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

// kSplit: pairs per tile, which share its blocks (1 or 2). kPN: weight rows per tile.
template <typename T, int kSplit, int kPN>
__global__ void __launch_bounds__(kPThreads, 1)
    fp8_linear_prefill_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w,
                              const __grid_constant__ CUtensorMap tmap_out, const Fp8LinearArgs p) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                                         ~uintptr_t(1023));
  using Tile = PrefillTile<kPN>;
  constexpr int kPStages = Tile::kStages, kPGroupCols = Tile::kGroupCols, kPOutCols = Tile::kOutCols;
  constexpr uint32_t kPStage = Tile::kStage, kPOut = Tile::kOut;
  unsigned char* staging = ring + kPStages * kPStage;
  __shared__ PrefillCtl<kPStages> c;
  constexpr uint32_t kIdesc = idesc_e4m3(2 * kPM, kPN);
  constexpr uint32_t kTmemCols = 2 * kPAccCols;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles = p.m_tiles * p.n_tiles;
  constexpr int cluster_size = 2 * kSplit;
  const int cluster_rank = (int)(blockIdx.x % (unsigned)cluster_size);
  const int rank = cluster_rank & 1;                   // in the pair
  const uint32_t leader = kSplit == 1 ? 0 : (uint32_t)cluster_rank & ~1u;  // the pair's CTA 0
  const uint16_t both = (uint16_t)(3u << leader);
  const int part = kSplit == 1 ? 0 : cluster_rank >> 1;  // of the tile's blocks
  const int kb0 = (int)((long long)part * p.k_blocks / kSplit);
  const int kb1 = (int)((long long)(part + 1) * p.k_blocks / kSplit);
  const int cluster = (int)(blockIdx.x / (unsigned)cluster_size), clusters = (int)(gridDim.x / (unsigned)cluster_size);

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
      mbar_init(&c.tempty[i], 2 * 4 * kPGroups);
      mbar_init(&c.sfull[i], 64);
      mbar_init(&c.sempty[i], 4 * kPGroups);
    }
    mbar_init(&c.teardown, 1);
    fence_mbar_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&c.tmem_base)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_arrive_release();  // both CTAs' barriers and TMEM are ready
  cluster_wait_acquire();
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
      for (int t = cluster; ok && t < tiles; t += clusters) {
        int m_tile, n_tile;
        prefill_tile(p, t, m_tile, n_tile);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(&c.empty[stage], phase ^ 1, p.status, NPL_DEV_TIMEOUT_TMA)) {
            ok = false;
            break;
          }
          unsigned char* at = ring + (size_t)stage * kPStage;
          if (rank == 0) mbar_arrive_expect_tx(&c.full[stage], 2 * kPStage);
          const uint32_t bar = cluster_map(&c.full[stage], leader);
          tma_load_2d_pair(at, &tmap_x, kb * kBlockK, (2 * m_tile + rank) * kPM, bar, pol);
          tma_load_2d_pair(at + kPStageX, &tmap_w, kb * kBlockK, n_tile * kPN + rank * (kPN / 2), bar, pol);
          loads = min(loads + 1, kPStages);
          if (++stage == kPStages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      // every load is read by its MMAs (or, where those gave up, has landed)
      // before the ring is released
      for (int i = 0; i < loads; ++i) {
        const uint32_t last = i < stage ? phase : phase ^ 1;
        if (!mbar_wait(&c.empty[i], last, p.status, NPL_DEV_TIMEOUT_TEARDOWN) && rank == 0)
          mbar_wait(&c.full[i], last, p.status, NPL_DEV_TIMEOUT_TEARDOWN);
      }
    } else if (warp == 1) {
      // The whole warp runs this loop and one lane issues: addresses and
      // descriptors then stay in uniform registers, which tcgen05.mma reads.
      // From one lane's branch each is moved there first, and issuing a block
      // took 650 cycles.
      const bool issuer = elect_one();
      const uint64_t desc0 = sdesc_k_sw128(smem_u32(ring));
      int stage = 0;
      uint32_t phase = 0, it = 0;
      bool ok = rank == 0;
      for (int t = cluster; ok && t < tiles; t += clusters) {
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const uint32_t buf = it & 1;
          if (!poll_wait<false>(&c.full[stage], phase, p.status, NPL_DEV_TIMEOUT_MMA) ||
              !poll_wait<false>(&c.tempty[buf], ((it >> 1) & 1) ^ 1, p.status, NPL_DEV_TIMEOUT_MMA)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t a = desc0 + (uint32_t)stage * (kPStage >> 4), b = a + (kPStageX >> 4);
          const uint32_t d = tmem_base + buf * kPAccCols;
          if (issuer) {
            mma_e4m3_pair<false>(d, a, b, kIdesc);
#pragma unroll
            for (int kk = 1; kk < kBlockK / 32; ++kk) mma_e4m3_pair<true>(d, a + kk * 2, b + kk * 2, kIdesc);
            tc_commit_pair(&c.tfull[buf], both);
            tc_commit_pair(&c.empty[stage], both);
          }
          __syncwarp();
          if (++stage == kPStages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      // all MMAs complete, in both CTAs' view, before TMEM is freed
      if (rank == 0 && issuer) tc_commit_pair(&c.teardown, both);
      poll_wait<false>(&c.teardown, 0, p.status, NPL_DEV_TIMEOUT_TEARDOWN);
      __syncwarp();
    } else if (warp >= 2) {
      // A load of a warp reads kPScaleBlocks blocks of 32 / kPScaleBlocks tokens;
      // transposed into shared memory. Eight loads before the first store: the
      // compiler does not move them across.
      constexpr int kRows = 32 / kPScaleBlocks, kStep = 2 * kRows;
      const int kk = lane % kPScaleBlocks, r0 = (warp - 2) * kRows + lane / kPScaleBlocks;
      uint32_t chunk = 0;
      bool ok = true;
      for (int t = cluster; ok && t < tiles; t += clusters) {
        int m_tile, n_tile;
        prefill_tile(p, t, m_tile, n_tile);
        const int m0 = (2 * m_tile + rank) * kPM;
        const int nb = n_tile * kPN / kTileN;  // the tile's first block of weight rows
        const float* sw0 = p.sw + (long long)nb * p.ld_sw;
        const bool two = (nb + 1) * kTileN < p.N;  // it has a second one
        for (int kb = kb0 + kk; kb - kk < kb1; kb += kPScaleBlocks, ++chunk) {
          const uint32_t buf = chunk & 1;
          const bool in = kb < kb1;
          const float w0 = in ? sw0[kb] : 0.f, w1 = in && two ? sw0[p.ld_sw + kb] : 0.f;
          if (!mbar_wait(&c.sempty[buf], ((chunk >> 1) & 1) ^ 1, p.status, NPL_DEV_TIMEOUT_EPILOGUE)) {
            ok = false;
            break;
          }
          for (int r = r0; r < kPM; r += 8 * kStep) {
            float a[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int m = m0 + r + i * kStep;
              a[i] = in && m < p.M ? p.sa[(long long)m * p.ld_sa + kb] : 0.f;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              c.scale[buf][0][kk][r + i * kStep] = __fmul_rn(a[i], w0);
              c.scale[buf][1][kk][r + i * kStep] = __fmul_rn(a[i], w1);
            }
          }
          mbar_arrive(&c.sfull[buf]);
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPRegsMany));
    const int group = (warp - 4) >> 2;  // columns [kPGroupCols group, kPGroupCols (group + 1)) of the tile
    const int row = (warp & 3) * 32 + lane;
    const bool elected = (threadIdx.x & 127) == 0;
    unsigned char* stg = staging + group * kPOut;
    auto group_bar = [&] { asm volatile("bar.sync %0, 128;" ::"r"(1 + group) : "memory"); };
    const T* res = static_cast<const T*>(p.residual);
    T* out = static_cast<T*>(p.out);
    const uint32_t tempty0 = cluster_map(&c.tempty[0], leader), tempty1 = cluster_map(&c.tempty[1], leader);
    const uint32_t taddr0 = tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + group * kPGroupCols;
    uint32_t it = 0, chunk = 0;
    float acc[kPGroupCols];
    int m_base = 0, n_out = 0;  // the first token and column that this warpgroup writes, in `boxes` boxes
    constexpr int boxes = kSplit > 1 ? 1 : kPGroupCols / kPOutCols;
    auto sums_of = [&](int t) {
      int m_tile, n_tile;
      prefill_tile(p, t, m_tile, n_tile);
      m_base = (2 * m_tile + rank) * kPM;
      const int n0 = n_tile * kPN + group * kPGroupCols;
      const int second = (n_tile * kPN / kTileN + 1) * kTileN - n0;  // the group's first column of the second block
      bool ok = true;
      n_out = n0;
#pragma unroll
      for (int j = 0; j < kPGroupCols; ++j) acc[j] = 0.f;
      for (int kb = kb0; ok && kb < kb1; kb += kPScaleBlocks, ++chunk) {
        const uint32_t sbuf = chunk & 1;
        ok = poll_wait<false>(&c.sfull[sbuf], (chunk >> 1) & 1, p.status, NPL_DEV_TIMEOUT_EPILOGUE);
        const int kn = min(kPScaleBlocks, kb1 - kb);
        const float* scale = &c.scale[sbuf][kPN == 256 ? group : 0][0][row];
        for (int kk = 0; ok && kk < kn; ++kk, ++it, scale += kPScaleLd) {
          const uint32_t buf = it & 1;
          const float s = *scale;
          const float s2 = kPN == 256 ? s : scale[kPScaleBlocks * kPScaleLd];
          if (!poll_wait<false>(&c.tfull[buf], (it >> 1) & 1, p.status, NPL_DEV_TIMEOUT_EPILOGUE)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t taddr = taddr0 + buf * kPAccCols;
          constexpr int kRead = kPN == 256 ? 64 : 96;  // columns at a time
          uint32_t d[kRead / 32][32];
#pragma unroll
          for (int q = 0; q < kPGroupCols; q += kRead) {
#pragma unroll
            for (int i = 0; i < kRead / 32; ++i) tmem_ld_x32(taddr + q + 32 * i, d[i]);
            tmem_wait_ld();
            if (q + kRead == kPGroupCols) {  // the accumulator is read: its next MMAs may start
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive_pair(buf ? tempty1 : tempty0);
            }
#pragma unroll
            for (int j = 0; j < kRead; ++j)
              fma_after_ld(acc[q + j], d[j >> 5][j & 31], kPN == 256 || q + (j & ~31) < second ? s : s2);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&c.sempty[sbuf]);  // the chunk of scales is read
      }
      if constexpr (kSplit > 1) {
        // The sums of this CTA's blocks go to its ring, which its last MMAs are
        // done with, [column][token]; after the barrier the CTAs of one rank add
        // those of parts 0, 1 for 128 columns each, 64 a warpgroup.
        static_assert(kSplit * kPGroups * kPOutCols == kPN);
        float* sums = reinterpret_cast<float*>(ring);
        if (ok) {
#pragma unroll
          for (int j = 0; j < kPGroupCols; ++j) sums[(group * kPGroupCols + j) * kPM + row] = acc[j];
        }
        cluster_arrive_release();
        cluster_wait_acquire();
        const int col = (part * kPGroups + group) * kPOutCols;
        n_out = n_tile * kPN + col;
        if (ok) {
          uint32_t from[kSplit];
#pragma unroll
          for (int q = 0; q < kSplit; ++q) from[q] = cluster_map(sums + col * kPM + row, (uint32_t)(2 * q + rank));
#pragma unroll
          for (int j = 0; j < kPOutCols; ++j) {
            float v = ld_cluster_f32(from[0] + j * kPM * 4);
#pragma unroll
            for (int q = 1; q < kSplit; ++q) v = __fadd_rn(v, ld_cluster_f32(from[q] + j * kPM * 4));
            acc[j] = v;
          }
        }
      }
      return ok;
    };
    auto write = [&](int) {
      const int m = m_base + row;
      // bias, residual, rounding; kPOutCols columns at a time through shared memory
#pragma unroll
      for (int h = 0; h < boxes; ++h) {
        const int nh = n_out + h * kPOutCols;
        if (elected) tma_store_wait_read();
        group_bar();  // the staging buffer is free
#pragma unroll
        for (int ch = 0; ch < kPOutCols / 8; ++ch) {
          float v[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = acc[h * kPOutCols + ch * 8 + j];
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
          *reinterpret_cast<uint4*>(stg + staged<kPOutCols>(row, ch)) = o;
        }
        if (p.tma_out) {
          fence_proxy_async_smem();
          group_bar();
          if (elected && nh < p.N && m_base < p.M) tma_store_2d(&tmap_out, stg, nh, m_base);
        } else {  // rows that TMA cannot store: element by element, 32 columns a warp
          group_bar();
          constexpr int kAtOnce = 8;  // rows read before the first store (8000 x 513 x 1024: 22.6 us, one by one 28.3)
          for (int r0 = (warp & 3); r0 < kPM && m_base + r0 < p.M; r0 += 4 * kAtOnce) {
#pragma unroll
            for (int e = lane; e < kPOutCols; e += 32) {
              T v[kAtOnce];
#pragma unroll
              for (int i = 0; i < kAtOnce; ++i)
                v[i] = *reinterpret_cast<const T*>(stg + staged<kPOutCols>(r0 + 4 * i, e >> 3) + (e & 7) * 2);
#pragma unroll
              for (int i = 0; i < kAtOnce; ++i) {
                const long long mr = (long long)m_base + r0 + 4 * i;
                if (mr < p.M && nh + e < p.N) out[mr * p.ld_out + nh + e] = v[i];
              }
            }
          }
        }
      }
    };
    prefill_epilogue(cluster, clusters, tiles, sums_of, [&](bool ok) { return warpgroup_agrees(1 + group, ok); }, write);
    if (elected) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  if (kSplit > 1 && warp < 4) {  // the epilogue warps' barrier over the sums
    cluster_arrive_release();
    cluster_wait_acquire();
  }

  tc_fence_before();
  __syncthreads();
  cluster_arrive_release();  // no CTA's shared memory or TMEM is given up while another uses it
  cluster_wait_acquire();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols) : "memory");
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

// Shared memory of a decode CTA: more than a third of an SM's, so that at most
// two such CTAs share an SM. Their TMEM (2 x 256 columns) then always fits, and
// no CTA of a cluster waits for TMEM that a CTA of another cluster holds (a
// prefill CTA, with 512 columns, fills an SM's shared memory alone).
constexpr int kDecodeSmem = 110 * 1024;
constexpr int kThirdOfSm = 76 * 1024;

// CTAs that share a decode tile: as many as keep 1.75 CTAs an SM (beyond it not
// all clusters run at once: 96 tiles of 32 blocks take 12.6 us unsplit, 13.6
// two-way, 17.9 three-way; 76 tiles 12.6, 13.0, 10.7, 14.3 four-way) and two
// blocks a CTA. Where that gives two, from 87 to 129 tiles, joining costs more
// than two CTAs save (96 tiles above; 128 tiles 13.4 us unsplit, 15.0 two-way), so
// such tiles stay whole, and 96 of them leave 52 SMs without one.
int decode_split(long long tiles, int k_blocks) {
  const long long s = std::min({(long long)kMaxSplit, 7ll * num_sms() / (4 * tiles), (long long)k_blocks / 2});
  return s <= 2 ? 1 : (int)s;
}

template <typename T, int NT>
int launch_decode(const Operands& o, Fp8LinearArgs& p, cudaStream_t st) {
  CUtensorMap tw, tx;
  if (int rc = code_map(&tw, o.qw, p.N, o.K, o.ldw, kTileN)) return rc;
  if (int rc = code_map(&tx, o.qa, p.M, o.K, o.lda, NT)) return rc;
  constexpr int stage = (kTileN + NT) * kBlockK;
  constexpr int stages = std::min(kMaxStages, (kDecodeSmem - 1024) / stage);
  constexpr int smem = stages * stage + 1024;
  static_assert(smem > kThirdOfSm && PrefillTile<192>::kSmem + smem > 3 * kThirdOfSm);
  p.stages = stages;
  const long long m_tiles = (p.M + NT - 1) / NT;
  const long long tiles = m_tiles * p.n_tiles;
  p.split = decode_split(tiles, p.k_blocks);
  if (tiles * p.split > 2147483647ll)
    return fail(NPL_ERR_UNSUPPORTED, "npl_fp8_linear: M=%d N=%d has too many tiles", p.M, p.N);
  auto kern = fp8_linear_decode_kernel<T, NT>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return launch_status("npl_fp8_linear: smem attribute");
  return launch_pdl_cluster("npl_fp8_linear", kern, dim3((unsigned)(tiles * p.split)), dim3(kThreads), (size_t)smem,
                            st, (unsigned)p.split, tw, tx, p);
}

// Row-major [rows, cols] of a 16-bit type with row stride ld, in boxes of 128 rows x 64 or 32 columns.
int out_map(CUtensorMap* map, void* base, int dtype, long long rows, long long cols, long long ld, int box_cols) {
  auto fn = tensor_map_encoder();
  if (!fn) return fail(NPL_ERR_LAUNCH, "npl_fp8_linear: cuTensorMapEncodeTiled unavailable");
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)kPM};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = fn(map, dtype == NPL_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                        base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        box_cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                        CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(NPL_ERR_ARG, "npl_fp8_linear: cuTensorMapEncodeTiled failed (%d)", (int)r);
  return NPL_OK;
}

template <typename T, int kSplit, int kPN>
int launch_prefill_tiles(const Operands& o, Fp8LinearArgs& p, cudaStream_t st) {
  using Tile = PrefillTile<kPN>;
  CUtensorMap tx, tw, to;
  if (int rc = code_map(&tx, o.qa, p.M, o.K, o.lda, kPM)) return rc;
  if (int rc = code_map(&tw, o.qw, p.N, o.K, o.ldw, kPN / 2)) return rc;
  p.tma_out = aligned16(p.out) && p.ld_out % 8 == 0;
  p.vec_res = aligned16(p.residual) && p.ld_res % 8 == 0;
  to = tx;
  if (p.tma_out)
    if (int rc = out_map(&to, p.out, o.out_dtype, p.M, p.N, p.ld_out, Tile::kOutCols)) return rc;
  p.m_tiles = (p.M + 2 * kPM - 1) / (2 * kPM);
  p.n_tiles = (p.N + kPN - 1) / kPN;
  const long long tiles = (long long)p.m_tiles * p.n_tiles;
  if (tiles > 1ll << 30)
    return fail(NPL_ERR_UNSUPPORTED, "npl_fp8_linear: M=%d N=%d has too many tiles", p.M, p.N);
  p.raster_g = std::min(8, p.m_tiles);
  auto kern = fp8_linear_prefill_kernel<T, kSplit, kPN>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Tile::kSmem) != cudaSuccess)
    return launch_status("npl_fp8_linear: smem attribute");
  const unsigned clusters = (unsigned)std::min<long long>(tiles, num_sms() / 2);
  return launch_pdl_cluster("npl_fp8_linear", kern, dim3(clusters * 2 * kSplit), dim3(kPThreads), (size_t)Tile::kSmem, st,
                            2u * kSplit, tx, tw, to, p);
}

// Few tiles of 256 weight rows: two pairs share one where all clusters run at
// once (33 of them do; with 34 256 x 8704 x 4096 takes 32.3 us, unsplit 18.3) and
// have 12 blocks a pair or more (512 x 4096 x 11008: 27.2 us, unsplit 37.6; 256 x
// 4096 x 3584 14.4 and 15.6; 512 x 4096 x 2560 14.2 and 13.9). Four pairs, clusters
// of 8 CTAs with an SM each, take 29 us where two take 16 (256 x 4096 x 4096).
// Otherwise tiles of 192 weight rows, whose blocks take seven eighths of the time,
// where the pairs have them done in as many rounds as those of 256 (560 x 4096 x
// 11008, 66 tiles or 48: 40.1 us against 45.3; 1024 x 5120 x 5120, 108 or 80: 36.6
// against 40.7), but not for one round more (560 x 12288 x 4096, 192 or 144: 47.6
// against 37.9; 560 x 32003 x 4096, 501 or 378: 145 against 130).
template <typename T>
int launch_prefill(const Operands& o, Fp8LinearArgs& p, cudaStream_t st) {
  const long long pairs = num_sms() / 2, m_tiles = ((long long)p.M + 2 * kPM - 1) / (2 * kPM);
  const long long wide = m_tiles * ((p.N + 255ll) / 256), narrow = m_tiles * ((p.N + 191ll) / 192);
  if (2 * wide <= pairs && p.k_blocks >= 24) {
    auto* kern = fp8_linear_prefill_kernel<T, 2, 256>;
    constexpr int smem = PrefillTile<256>::kSmem;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
      return launch_status("npl_fp8_linear: smem attribute");
    if (wide <= max_active_clusters(reinterpret_cast<const void*>(kern), smem, 4, kPThreads))
      return launch_prefill_tiles<T, 2, 256>(o, p, st);
  }
  if ((narrow + pairs - 1) / pairs <= (wide + pairs - 1) / pairs) return launch_prefill_tiles<T, 1, 192>(o, p, st);
  return launch_prefill_tiles<T, 1, 256>(o, p, st);
}

// Decode tiles up to 64 tokens. Two rows of them, up to 128 tokens, as long as
// they still split three ways (100 x 4096 x 4096: 12.6 us against 15.1 with
// prefill tiles; 100 x 5504 x 4096 15.0 and 16.3; 100 x 6144 x 4096, which does not
// split, 20.1 and 16.4) and the rows are not short (128 x 4096 x 1024: 9.5 and 7.5;
// x 2048 10.6 and 10.2). Four rows: 200 x 4096 x 4096 20.0 and 15.5.
template <typename T>
int launch(const Operands& o, Fp8LinearArgs& p, cudaStream_t st) {
  if (p.M <= 16) return launch_decode<T, 16>(o, p, st);
  if (p.M <= 32) return launch_decode<T, 32>(o, p, st);
  const bool two_rows = p.M <= 128 && p.k_blocks >= 20 && decode_split(2ll * p.n_tiles, p.k_blocks) >= 3;
  if (p.M <= 64 || two_rows) return launch_decode<T, 64>(o, p, st);
  return launch_prefill<T>(o, p, st);
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
