// Attention over the paged KV pool under masks other than the causal one: a
// tree of drafted tokens, and a sliding window with sinks.
//
// npl_paged_tree_attention, npl_paged_window_attention (no counterpart in the
// reference, whose kernels are causal).
//
// For a query row with the keys S that it sees:
//   s_i = scale * q . k_i,  out = sum_{i in S} e^(s_i - m) v_i / sum_{i in S} e^(s_i - m)
// in one pass over the keys. m is a running reference of the row, not its
// maximum: it moves only when a tile's maximum is more than 2^8 above it (in
// the exponentials), so that the sums in tensor memory are rarely rescaled.
// p = 2^(s log2(e) + 6 - m): at most 2^14, and an fp16 p keeps 2^-30 of the
// largest. The normaliser sums the unrounded p. For P.V, whose operands have
// the type of the caches, up to 32 rows of a kv head have p as two numbers of it,
// p rounded and the rest (below 2^-22 of p in fp16, 2^-16 in bf16: single
// tokens keep what a product in fp32 keeps); more rows have p rounded once, as
// in causal prompts: the rest has no room beside S and O in tensor memory.
//
// On the tensor cores (tcgen05 kind::f16, fp32 sums in TMEM). A CTA works on two
// streams, each with its own rows, its own warpgroup and its own TMEM, so that
// one stream's softmax runs while the tensor core works for the other:
//   shared (more rows than one tile of 128): two neighbouring row tiles of one
//     kv head read the same K and V tiles;
//   not shared (single tokens, trees): the same rows of two kv heads.
// Rows are (token, query head of one kv head): grouped heads share their keys.
// Two kernels: masked_attn_kernel has rows as M and one thread a row; P goes over
// S in TMEM, where the P.V product reads it. few_rows_kernel (at most 32 rows) has
// them as N. 384 threads: warps 0-3 and 4-7 softmax of the streams, warp 8 loads,
// warp 9 products, warps 10 and 11 clean V or load it. The order S0, S1, then
// O0 S0 O1 S1 ... makes every S of a stream arrive after the O before it, so no
// further barrier guards a rescale.
//
// Keys come in pieces of gcd(block_size, 32): the visible ones of a CTA's rows
// only (the sinks' pieces, then the window's). Whole pieces that lie together in
// the pool, up to 128 rows, come in one load with both halves of the head; loads
// of 32 rows and one half made the load warp the bottleneck (32 x 25 drafts in
// pages of 16: 270 us, now 140). A long axis with few rows is split over a cluster of
// CTAs, whose partial sums are joined through distributed shared memory.
//
// What a masked slot holds must not reach a row that does not see it, and
// 0 * infinity would: in tiles that some row sees in part, the V rows that no
// row sees are zeroed, and V elements that are not finite are replaced by 0 and
// added at the end to the rows that do see them.
//
// Bound by memory where there are few rows (64 tokens, 32 heads, 1028 keys each:
// 166 us, 6.0 TB/s); for long prompts by a stream's chain of product, scores out of
// TMEM (twice: held in registers they spill), exponentials (a quarter of them by
// a polynomial: 375 us for 16000 tokens of 32/8 heads under a window of 1024, none
// 409, half 415; 325 with tiles packed, 310 with 32-byte stores, 314 with NaN kept)
// and P back. For many prompts of few row tiles by uneven shares: the row tile is
// the fastest index of the items and a CTA takes every 148th, so that with 4 row
// tiles (20 x 800 tokens) a CTA meets one of them only, of 2, 4, 5 or 3 key tiles,
// and has 34 to 90 key tiles to do, 61 in the mean (312 us).
#include <algorithm>
#include <initializer_list>

#include <cuda_bf16.h>
#include <cudaTypedefs.h>

#include "npl_common.cuh"

namespace npl {
namespace {

constexpr int kMaThreads = 384;
constexpr int kMaTile = 128;
constexpr int kMaFixed = 10;            // what a round of clusters costs beside its tiles, in tiles
constexpr int kMaBad = 12;             // keys with V elements that are not finite, remembered for an item
constexpr int kMaPieceLog = 5;         // 32 keys of a piece at most
constexpr int kMaBoxLog = 7;           // 128 keys of a load at most
constexpr int kMaMaxSplit = 8;          // CTAs of a cluster at most
constexpr int kMaPoly = 4;              // of as many pairs of exponentials one by a polynomial
constexpr float kMaShift = 6.f;        // p = 2^(x - m + 6)
constexpr float kMaSlack = 8.f;        // m moves when a score is more than this above it

// Division of 0 <= n < 2^31 by a number known at the launch: with s = ceil(log2 d) and mul = ceil(2^(31 + s) / d),
// floor(n / d) = floor(n mul / 2^(31 + s)), since n (mul d - 2^(31 + s)) < 2^31 2^s. One number needs one of these
// instead of 30 instructions, which a CTA that runs them once has to fetch.
struct MaDiv {
  uint32_t mul;
  int shift;  // s - 1, -1 for d = 1
  static MaDiv of(int d) {
    int s = 0;
    while ((1ll << s) < d) ++s;
    return {(uint32_t)(((1ull << (31 + s)) + d - 1) / d), s - 1};
  }
  __device__ __forceinline__ int operator()(int n) const { return shift < 0 ? n : (int)(__umulhi(n, mul) >> shift); }
};

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
  bool out32;    // rows of out start on 32-byte boundaries
  int tokens;    // of a row tile: 128 / G
  int capacity;  // keys that a row of the table has room for
  int piece, piece_log;  // keys of a piece, a power of two
  int box_log;           // pieces of a large load, a power of two
  int levels;   // items of a sequence and kv head (or pair of them)
  int n_items;  // levels * B * (kv heads, or pairs of them)
  MaDiv by_levels, by_units, by_group, by_page;
  int split, split_log;  // CTAs of a cluster, which share an item's keys, a power of two
  float c2;     // scale * log2(e)
  int* status;
};

// Lists of keys whose V rows held elements that are not finite, of the last kLists items of one stream and of the last
// kLists of two. A list is written again when the first V tile of an item of its kind has come. That tile's stage, one
// of kStages, has been free, and an item takes two stages or more, so every product of the item kStages / 2 + 1 before
// it has been issued, for which every stream that has rows in it has left the items before. The two kinds are counted
// apart because the second stream takes no part in items of one: it may still read its last list while the first goes
// through any number of those.
template <int kLists>
struct MaBarriers {
  static_assert((kLists & (kLists - 1)) == 0, "a power of two");
  static constexpr int kListMask = (kLists - 1) * 0x10001;  // the count of items of one stream, and of two above it
  __device__ static int list(int count, bool second) { return second ? kLists + (count >> 16) : count & 0xffff; }
  __device__ static int next(int count, bool second) { return (count + (second ? 0x10000 : 1)) & kListMask; }
  uint64_t q_full[2], q_empty[2], s_full[2], p_full[2], o_full[2], mma_done;
  uint32_t tmem_base;
  int abort;
  int n_bad[2 * kLists][2][2];  // [list][stream whose V it is][warp 10 or 11]
  int bad[2 * kLists][2][2][kMaBad];
};

template <int D>
struct MaSmem : MaBarriers<D == 128 ? 4 : 8> {
  static constexpr bool kFew = false;
  static constexpr int kRows = kMaTile;
  static constexpr uint32_t kQHalf = kMaTile * 128;  // Q: 128 rows x 64 elements (one swizzle span), twice for D = 128
  static constexpr uint32_t kGroup = 8 * D * 2;      // K, V: 8 rows x 64 elements, twice for D = 128, then 8 more rows
  static constexpr uint32_t kTileBytes = kMaTile * D * 2;
  static constexpr int kStages = D == 128 ? 5 : 8;
  static constexpr uint32_t kScoreCols = 128, kOutCols = 128, kTmemCols = 512;  // S of the streams (P over it), then O
  uint64_t full[kStages], empty[kStages], raw[kStages];
  static constexpr int kQBufs = 1;
  alignas(1024) uint8_t q[1][2][kTileBytes];
  alignas(1024) uint8_t kv[kStages][kTileBytes];  // K and V tiles in the order of their use; partial sums at the end
};

// Few rows, as the N side of the products.
template <int D, int kN>
struct MaFewSmem : MaBarriers<D == 128 ? 4 : 8> {
  static constexpr bool kFew = true;
  static constexpr int kRows = kN;
  static constexpr uint32_t kQHalf = kN * 128;
  static constexpr uint32_t kGroup = 8 * D * 2;
  static constexpr uint32_t kTileBytes = kMaTile * D * 2;
  static constexpr int kStages = D == 64 ? 10 : 5;
  static constexpr uint32_t kScoreCols = kN, kOutCols = 2 * kN, kTmemCols = 8 * kN;  // S of the streams, then O
  uint64_t full[kStages], empty[kStages], raw[kStages];
  alignas(16) float add[2][kN];  // of a row: 6 - m
  float alpha[2][kN];            // what its sums are scaled with
  float top[2][4][kN];           // a warp's maxima, at the end its sums
  float2 ml[2][kN];              // m and the normaliser at the end
  float inv[2][kN];              // and what a row of sums is multiplied with
  static constexpr int kQBufs = kN == 16 ? 2 : 1;  // Q of this item, and of the next one where there is room
  alignas(1024) uint8_t q[kQBufs][2][kN * D * 2];
  alignas(1024) uint8_t p[2][kMaTile * 128];  // P^T: a key's rows, then what their roundings left, in one 128-byte line
  alignas(1024) uint8_t kv[kStages][kTileBytes];
};

constexpr size_t kMaMaxSmem = 232448 - 1024;  // of a CTA, without the room to align
static_assert(sizeof(MaSmem<128>) <= kMaMaxSmem && sizeof(MaSmem<64>) <= kMaMaxSmem, "shared memory");
static_assert(sizeof(MaFewSmem<128, 16>) <= kMaMaxSmem && sizeof(MaFewSmem<64, 16>) <= kMaMaxSmem, "shared memory");
static_assert(std::max(MaSmem<128>::kStages, MaFewSmem<128, 16>::kStages) / 2 + 2 <= 4, "lists");
static_assert(std::max(MaSmem<64>::kStages, MaFewSmem<64, 16>::kStages) / 2 + 2 <= 8, "lists");
static_assert(sizeof(MaFewSmem<128, 32>) <= kMaMaxSmem && sizeof(MaFewSmem<64, 32>) <= kMaMaxSmem, "shared memory");

template <typename T>
struct MaType;
template <>
struct MaType<__half> {
  static constexpr uint32_t kIdesc = 0;  // a_format, b_format: F16
  static constexpr uint32_t kExp = 0x7c007c00u, kOne = 0x04000400u;
  static constexpr CUtensorMapDataType kMap = CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  __device__ static float2 unpack(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
  __device__ static uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  __device__ static float get(const void* p, size_t i) { return __half2float(static_cast<const __half*>(p)[i]); }
  __device__ static uint32_t times0(uint32_t v, uint32_t sum) {
    const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&v), __half2half2(__ushort_as_half(0)),
                              *reinterpret_cast<const __half2*>(&sum));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  __device__ static void put(__half* p, float x) { *p = __float2half_rn(x); }
  __device__ static void add(__half* p, float x) { *p = __float2half_rn(__half2float(*p) + x); }
};
template <>
struct MaType<__nv_bfloat16> {
  static constexpr uint32_t kIdesc = (1u << 7) | (1u << 10);
  static constexpr uint32_t kExp = 0x7f807f80u, kOne = 0x00800080u;
  static constexpr CUtensorMapDataType kMap = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  __device__ static float2 unpack(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
  __device__ static uint32_t pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  __device__ static float get(const void* p, size_t i) {
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  }
  __device__ static uint32_t times0(uint32_t v, uint32_t sum) {
    const __nv_bfloat162 r = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&v), __float2bfloat162_rn(0.f),
                                     *reinterpret_cast<const __nv_bfloat162*>(&sum));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  __device__ static void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }
  __device__ static void add(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(__bfloat162float(*p) + x); }
};

// 2^x (ex2.approx.ftz: a result below 2^-126 is 0, which adds less than that to sums of 2^6 and more).
__device__ __forceinline__ float ma_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Bounded wait that also gives up once another role of the CTA gave up. (Its
// loop is a call: a CTA of few tiles runs most of its code once, and fetching
// that code is what it waits for.)
__device__ __noinline__ bool ma_wait_long(uint64_t* bar, uint32_t parity, int* abort, int* status, int code) {
  const uint64_t t0 = globaltimer_ns();
  while (true) {
    for (int i = 0; i < 32; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    if (*reinterpret_cast<volatile int*>(abort)) return false;
    if (globaltimer_ns() - t0 > kWaitLimitNs) {
      *reinterpret_cast<volatile int*>(abort) = 1;
      if (status) atomicCAS(status, 0, code);
      return false;
    }
  }
}
__device__ __forceinline__ bool ma_wait(uint64_t* bar, uint32_t parity, int* abort, int* status, int code) {
  return mbar_try_wait(bar, parity) || ma_wait_long(bar, parity, abort, status, code);
}

// The same for a warp: its lanes go on, or give up, together.
__device__ __forceinline__ bool ma_wait_warp(uint64_t* bar, uint32_t parity, int* abort, int* status, int code) {
  return __all_sync(0xffffffffu, ma_wait(bar, parity, abort, status, code));
}

__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one != 0;
}

// D[tmem] (+)= A[tmem] * B[smem], 16-bit floats, fp32 sums (kind::f16); A packed two K elements a column.
__device__ __forceinline__ void ma_mma_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 32 lanes x 16 columns from registers (thread i of the warp: lane i).
__device__ __forceinline__ void ma_tmem_st_x16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// Loads from TMEM have arrived; the registers go through it, so that no use of them moves ahead of it.
__device__ __forceinline__ void ma_tmem_wait_ld(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]));
  asm volatile("" : "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]));
}
__device__ __forceinline__ void ma_tmem_st_x32(uint32_t taddr, const uint32_t (&r)[32]) {
  ma_tmem_st_x16(taddr, r);
  ma_tmem_st_x16(taddr + 16, r + 16);
}
__device__ __forceinline__ void ma_tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float4 ma_ld_cluster(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ float2 ma_ld_cluster2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ void ma_st_32b(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// Scores of columns that are not seen become minus infinity. False: every row of the warp sees all of them.
__device__ __forceinline__ bool ma_hide(uint32_t (&v)[32], uint32_t seen) {
  if (__all_sync(0xffffffffu, seen == 0xffffffffu)) return false;
#pragma unroll
  for (int c = 0; c < 32; ++c)
    if (!(seen & (1u << c))) v[c] = 0xff800000u;
  return true;
}

__device__ __forceinline__ void ma_max32(const uint32_t (&v)[32], float (&mx)[4]) {
#pragma unroll
  for (int c = 0; c < 32; c += 2)
    mx[c >> 1 & 3] = fmaxf(mx[c >> 1 & 3], fmaxf(__uint_as_float(v[c]), __uint_as_float(v[c + 1])));
}

// Two fp32 numbers in one operation.
__device__ __forceinline__ uint64_t ma_pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 ma_unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t ma_add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t ma_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

__device__ __forceinline__ uint64_t ma_mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// 2^x for two x <= 127 without the special function unit, which is what the
// softmax of many rows waits for: x = n + f with the whole number n next to x (by
// adding 1.5 * 2^23), 2^f by the polynomial of degree 5 with the least relative
// error on [-1/2, 1/2] (Remez; 7.5e-8), times 2^n, whose bits come from those of
// n. x below -126.5 (n = -127) gives 0. NaN gives NaN: 2^f is NaN, and a product
// keeps it (n added to its exponent would make a number of it).
__device__ __forceinline__ float2 ma_exp2_poly(uint64_t x2) {
  const float2 u = ma_unpair(x2);
  float x0, x1;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(x0) : "f"(u.x), "f"(-127.f));
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(x1) : "f"(u.y), "f"(-127.f));
  const uint64_t x = ma_pair(x0, x1);
  const uint64_t t = ma_add2(x, ma_pair(12582912.f, 12582912.f));
  const uint64_t n = ma_add2(t, ma_pair(-12582912.f, -12582912.f));
  const uint64_t f = ma_fma2(n, ma_pair(-1.f, -1.f), x);
  uint64_t y = ma_pair(1.3276472454890609e-03f, 1.3276472454890609e-03f);
  y = ma_fma2(y, f, ma_pair(9.675540961325169e-03f, 9.675540961325169e-03f));
  y = ma_fma2(y, f, ma_pair(5.550713092088699e-02f, 5.550713092088699e-02f));
  y = ma_fma2(y, f, ma_pair(2.4022120237350464e-01f, 2.4022120237350464e-01f));
  y = ma_fma2(y, f, ma_pair(6.931469440460205e-01f, 6.931469440460205e-01f));
  y = ma_fma2(y, f, ma_pair(1.0000001192092896f, 1.0000001192092896f));
  const float2 tt = ma_unpair(t);
  const uint64_t power = ma_pair(__int_as_float((__float_as_int(tt.x) << 23) + 0x3f800000),
                                 __int_as_float((__float_as_int(tt.y) << 23) + 0x3f800000));
  const float2 r = ma_unpair(ma_mul2(y, power));
  return make_float2(r.x, r.y);
}

// p = 2^(score c2 + add) of 32 columns, packed; their sums go to ls. One pair of
// kPoly takes the polynomial (0: none).
template <typename T, int kPoly>
__device__ __forceinline__ void ma_exp_pack(const uint32_t (&v)[32], float c2, float add, uint64_t (&ls)[2],
                                            uint32_t (&pk)[16]) {
  const uint64_t c22 = ma_pair(c2, c2), add2 = ma_pair(add, add);
#pragma unroll
  for (int c = 0; c < 16; ++c) {
    const uint64_t x = ma_fma2(ma_pair(__uint_as_float(v[2 * c]), __uint_as_float(v[2 * c + 1])), c22, add2);
    float2 e;
    if (kPoly && c % kPoly == kPoly - 1) {
      e = ma_exp2_poly(x);
    } else {
      const float2 u = ma_unpair(x);
      e = make_float2(ma_exp2(u.x), ma_exp2(u.y));
    }
    ls[c & 1] = ma_add2(ls[c & 1], ma_pair(e.x, e.y));
    pk[c] = MaType<T>::pack(e.x, e.y);
  }
}

// One item: 128 rows (or twice 128, shared) of one sequence and kv head (or
// the same rows of two). Every role decodes the same items from the same
// read-only metadata. Tiles are numbered through x: key(x) = x below sink_x
// (the sinks' pieces), x + shift from hole_x on (the window's), and nothing is
// loaded between. This CTA takes the tiles x0 <= x < x1.
struct MaItem {
  int b, kvh, tok0, n, ctx, start, prefix;
  int lo, hi;  // keys that some row of the item sees: lo <= key < hi, and the sinks
  int sink_x, hole_x, shift, x0, x1, nt;
  int full0, full1;  // full0 <= x < full1: every row of the item sees the key
  bool skip, second;  // no such rows; the second stream has rows
};

template <bool kTree, bool kShared>
__device__ __forceinline__ MaItem ma_item(const MaArgs& p, int i, int rank) {
  MaItem it;
  const int units = kShared ? p.Hkv : (p.Hkv + 1) / 2;
  const int rem = p.by_levels(i), level = i - rem * p.levels;
  it.b = p.by_units(rem);
  it.kvh = (rem - it.b * units) * (kShared ? 1 : 2);
  it.tok0 = level * p.tokens * (kShared ? 2 : 1);
  it.n = p.q_lens ? p.q_lens[it.b] : 1;
  it.start = p.q_offsets ? p.q_offsets[it.b] : it.b;
  it.ctx = p.ctx_lens[it.b];
  it.prefix = it.ctx - it.n;
  it.skip = it.tok0 >= it.n || it.n > p.max_q_len || it.start < 0 || it.start > p.total_q - it.n || it.ctx < 0 ||
            it.ctx > p.capacity;
  it.second = kShared ? it.tok0 + p.tokens < it.n : it.kvh + 1 < p.Hkv;
  const int last = min(it.n, it.tok0 + p.tokens * (kShared ? 2 : 1));  // one past the item's last token
  int end = 0;
  it.lo = it.sink_x = it.hole_x = it.shift = 0;
  it.hi = kTree ? it.ctx : it.prefix + last;
  if (it.prefix < 0) it.hi = 0;
  if (it.hi > 0) {
    end = (((it.hi - 1) >> p.piece_log) + 1) << p.piece_log;
    if (!kTree) {
      it.lo = max(0, it.prefix + it.tok0 - p.window + 1);
      const int sp = (min(p.sinks, it.lo) + p.piece - 1) >> p.piece_log << p.piece_log;
      const int lp = it.lo >> p.piece_log << p.piece_log;
      if (sp < lp) {
        // the first x from sp on with lp's place in a tile, so that tiles lie in pages; sp itself if that saves a tile
        const int hole = (lp - sp) & (kMaTile - 1), used = (sp + end - lp - 1) & (kMaTile - 1);
        it.sink_x = sp;
        it.hole_x = used + hole >= kMaTile ? sp : sp + hole;
        it.shift = lp - it.hole_x;
        end -= it.shift;
      }
    }
  }
  const int tiles = (end + kMaTile - 1) / kMaTile;
  const int t0 = (int)(((long long)tiles * rank) >> p.split_log);
  it.nt = (int)(((long long)tiles * (rank + 1)) >> p.split_log) - t0;
  it.x0 = t0 * kMaTile;
  it.x1 = min(end, it.x0 + it.nt * kMaTile);
  if (it.skip) it.nt = 0;
  it.full0 = 0;
  it.full1 = min(it.prefix, it.x1);
  if (!kTree) {
    // what the item's first row and its last row both see
    const int from = max(0, it.prefix + last - p.window);
    it.full0 = from <= p.sinks && !it.shift ? 0 : from - it.shift;
    it.full1 = min(it.prefix + it.tok0 + 1 - it.shift, it.x1);
  }
  return it;
}

// The n lowest bits of word w of a 128-bit mask of columns.
__device__ __forceinline__ uint32_t ma_low(int n, int w) {
  uint32_t above;  // shl takes more than 31 places too
  asm("shl.b32 %0, %1, %2;" : "=r"(above) : "r"(0xffffffffu), "r"(max(n - w * 32, 0)));
  return ~above;
}

// Whether some row of a CTA's item does not see some of the tile's columns from xt on.
__device__ __forceinline__ bool ma_part(const MaItem& it, int xt) { return xt < it.full0 || xt + kMaTile > it.full1; }

// Whether the row of a token sees a key: the bits of a tile, for one key.
template <bool kTree>
__device__ __forceinline__ bool ma_sees(const MaArgs& p, const MaItem& it, int token, int key) {
  if (kTree) return key < it.prefix || p.mask[(it.start + token) * p.ld_mask + (key - it.prefix)] != 0;
  const int pos = it.prefix + token;
  return key <= pos && (key > pos - p.window || key < p.sinks);
}

// V row of a tile (in shared memory) made safe to multiply by 0. Returns
// whether it held elements that are not finite, which are now 0.
template <typename T, int D>
__device__ __forceinline__ bool ma_clean_row(uint8_t* tile, int row, bool seen) {
  uint32_t any[4] = {0, 0, 0, 0};  // sums of 0 * v: NaN where v is not finite
#pragma unroll 1
  for (int hf = 0; hf < D / 64; ++hf) {
    uint4* line = reinterpret_cast<uint4*>(tile + (row >> 3) * (8 * D * 2) + hf * 1024 + (row & 7) * 128);
    if (!seen) {
#pragma unroll
      for (int c = 0; c < 8; ++c) line[c] = make_uint4(0, 0, 0, 0);
    } else {
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const uint4 x = line[c ^ (row & 7)];  // 8 rows use all banks
        any[0] = MaType<T>::times0(x.x, any[0]), any[1] = MaType<T>::times0(x.y, any[1]);
        any[2] = MaType<T>::times0(x.z, any[2]), any[3] = MaType<T>::times0(x.w, any[3]);
      }
    }
  }
  if (!((any[0] | any[1] | any[2] | any[3]) & 0x7fff7fffu)) return false;
#pragma unroll 1
  for (int c = 0; c < D / 2; ++c) {
    uint32_t* w = reinterpret_cast<uint32_t*>(tile + (row >> 3) * (8 * D * 2) + (c >> 5) * 1024 + (row & 7) * 128) + (c & 31);
    const uint32_t t = ((*w & MaType<T>::kExp) + MaType<T>::kOne) & 0x80008000u;
    *w &= ~((t >> 15) * 0xffffu);
  }
  return true;
}

// Keys whose V rows ma_clean_row took elements out of, for a row that sees them
// (a rare path). ma_bad_count says how many are to be looked at: those that were
// remembered, or, where there were more, all in the CTA's tiles that are seen in
// part. ma_bad_key gives one of them, -1 for none, and where its V row begins.
template <bool kTree, bool kShared>
__device__ __noinline__ int ma_bad_count(const MaArgs* args, const int* counts, int item, int rank) {
  if (max(counts[0], counts[1]) <= kMaBad) return counts[0] + counts[1];
  const MaItem it = ma_item<kTree, kShared>(*args, item, rank);
  const int ahead = min(max(it.full0 - it.x0, 0), it.x1 - it.x0);
  return ahead + max(it.x1 - max(it.full1, it.x0 + ahead), 0);
}
template <int D, bool kTree, bool kShared>
__device__ __noinline__ int ma_bad_key(const MaArgs* args, const int* counts, const int (*lists)[kMaBad], int item,
                                       int rank, int kvh, int j, size_t* at) {
  const MaArgs& p = *args;
  const MaItem it = ma_item<kTree, kShared>(p, item, rank);
  int key;
  if (max(counts[0], counts[1]) <= kMaBad) {
    key = j < counts[0] ? lists[0][j] : lists[1][j - counts[0]];
  } else {
    const int ahead = min(max(it.full0 - it.x0, 0), it.x1 - it.x0);
    const int x = j < ahead ? it.x0 + j : max(it.full1, it.x0 + ahead) + j - ahead;
    if (x >= it.sink_x && x < it.hole_x) return -1;
    key = x < it.sink_x ? x : x + it.shift;
  }
  if (key >= it.hi) return -1;
  const int page = p.by_page(key);
  const int blk = page < p.max_blocks ? p.bt[it.b * p.bt_stride + page] : -1;
  if (blk < 0 || blk >= p.num_blocks) return -1;
  *at = (((size_t)blk * p.block_size + (key - page * p.block_size)) * p.Hkv + kvh) * D;
  return key;
}

// Barriers among the 128 threads of a stream.
__device__ __forceinline__ void ma_stream_sync(int st) {
  if (st == 0)
    asm volatile("bar.sync 1, 128;" ::: "memory");
  else
    asm volatile("bar.sync 2, 128;" ::: "memory");
}
__device__ __forceinline__ bool ma_stream_any(int st, bool x) {
  int r;
  if (st == 0)
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.s32 p, %1, 0;\n\tbar.red.or.pred q, 1, 128, p;\n\t"
                 "selp.s32 %0, 1, 0, q;\n\t}" : "=r"(r) : "r"((int)x) : "memory");
  else
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.s32 p, %1, 0;\n\tbar.red.or.pred q, 2, 128, p;\n\t"
                 "selp.s32 %0, 1, 0, q;\n\t}" : "=r"(r) : "r"((int)x) : "memory");
  return r != 0;
}

// Reduces 16 values a lane over a warp: lane i is left with the result of value i % 16.
template <typename Op>
__device__ __forceinline__ void ma_warp_reduce(float (&v)[16], int lane, Op&& op) {
#pragma unroll
  for (int n = 8; n > 0; n /= 2) {
#pragma unroll
    for (int e = 0; e < n; ++e) {
      const bool up = lane & n;
      const float give = up ? v[e] : v[e + n], keep = up ? v[e + n] : v[e];
      v[e] = op(keep, __shfl_xor_sync(0xffffffffu, give, n));
    }
  }
  v[0] = op(v[0], __shfl_xor_sync(0xffffffffu, v[0], 16));
}

// Twice 4, or 16 columns of this lane from TMEM.
__device__ __forceinline__ void ma_tmem_ld_2x4(uint32_t at0, uint32_t at1, uint32_t (&r)[4], uint32_t (&q)[4]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%8];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x4.b32 {%4, %5, %6, %7}, [%9];\n\ttcgen05.wait::ld.sync.aligned;"
      : "=&r"(r[0]), "=&r"(r[1]), "=&r"(r[2]), "=&r"(r[3]), "=&r"(q[0]), "=&r"(q[1]), "=&r"(q[2]), "=&r"(q[3])
      : "r"(at0), "r"(at1)
      : "memory");
}
__device__ __forceinline__ void ma_tmem_ld_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];\n\ttcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// Shared-memory descriptors of a K or V tile (128-byte swizzle, 8 rows of 64
// elements in 1024 bytes, the rows' second halves in the next 1024): with the
// head dimension as K (groups of 8 rows `group` bytes apart), and as M or N
// (64-element halves `half` bytes apart).
__device__ __forceinline__ uint64_t ma_desc_k(uint32_t addr, uint32_t group) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | (1ull << 16) | ((uint64_t)(group >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ uint64_t ma_desc_mn(uint32_t addr, uint32_t half, uint32_t group) {
  return sdesc_mn_sw128(addr, half, group);
}

// Rows of one kv head of the pool, 8 * row8 and following, by one load.
__device__ __forceinline__ void ma_load_rows(void* dst, const CUtensorMap* map, int row8, int kvh, uint64_t* bar,
                                             uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%2, %2, %2, %3, %4}], [%5], %6;" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(row8), "r"(kvh), "r"(smem_u32(bar)), "l"(policy)
      : "memory");
}

// Warp 10, and warp 11 where row tiles share their keys: in tiles that some row
// sees in part, V rows are made safe to multiply by 0 before the P.V product
// reads them. Such a tile's load arrives at a barrier of its own, the tiles of
// the kind one after the other, and these warps arrive at the stage's in its
// place.
template <typename S, typename T, int D, bool kTree, bool kShared>
__device__ __forceinline__ void ma_clean_role(S& s, const MaArgs& p, int first, int stride, int rank) {
  constexpr int kStages = S::kStages;
  constexpr int kWarps = kShared ? 2 : 1;
  const int lane = threadIdx.x & 31, which = (threadIdx.x >> 5) - 10;
  int ring = 0, n_raw = 0, item_no = 0;
  bool ok = true;
  for (int i = first; ok && i < p.n_items; i += stride) {
    const MaItem it = ma_item<kTree, kShared>(p, i, rank);
    if (it.nt == 0) continue;
    const int streams = !kShared && it.second ? 2 : 1, list = S::list(item_no, it.second);
    const int pa = it.prefix + it.tok0, pb = it.prefix + min(it.n, it.tok0 + p.tokens * (kShared ? 2 : 1)) - 1;
    bool fresh = true;
#pragma unroll 1
    for (int t = 0; ok && t < it.nt; ++t) {
      const int xt = it.x0 + t * kMaTile;
      if (!ma_part(it, xt)) continue;
#pragma unroll 1
      for (int st = 0; ok && st < streams; ++st) {
        // V's place in the order of the loads
        const int r = ring + (streams == 1 ? 1 + 2 * t : (st == 0 ? 2 : t + 1 < it.nt ? 4 : 3) + 4 * t);
        ok = ma_wait_warp(&s.raw[n_raw % kStages], (n_raw / kStages) & 1, &s.abort, p.status,
                          NPL_DEV_TIMEOUT_EPILOGUE);
        if (!ok) break;
        ++n_raw;
        if (fresh) {  // not before a tile of the item has come: till then this warp may be any number of items ahead
          if (lane < 2) s.n_bad[list][lane][which] = 0;
          if (kWarps == 1 && lane < 2) s.n_bad[list][lane][1] = 0;
          __syncwarp();
          fresh = false;
        }
#pragma unroll 1
        for (int row = which * 32 + lane; row < kMaTile; row += 32 * kWarps) {
          const int x = xt + row, key = x < it.sink_x ? x : x + it.shift;
          const bool some = x < it.x1 && key < it.hi && (kTree || key >= it.lo || key < p.sinks);
          // a row that every row of the item sees is left as it is
          if (some && (kTree ? key < it.prefix : key <= pa && (key > pb - p.window || key < p.sinks))) continue;
          if (ma_clean_row<T, D>(s.kv[r % kStages], row, some)) {
            const int at = atomicAdd(&s.n_bad[list][st][which], 1);
            if (at < kMaBad) s.bad[list][st][which][at] = key;
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.full[r % kStages]);
      }
    }
    ring += 2 * it.nt * streams;
    item_no = S::next(item_no, it.second);
  }
}

// Loads by TMA: warp 8 of Q and K and, where row tiles share their keys, of V;
// else warp 11 of V: in pages of 16 slots a tile takes 8 loads, which one warp
// does not issue as fast as memory delivers them (32 x 25 drafts over 500 to 8000
// keys in such pages: 173 us with one warp, 137 with two). Lane i looks up and
// loads piece i of a tile. Both warps count all tiles in their order.
template <typename S, int D, bool kTree, bool kShared, bool kV>
__device__ __forceinline__ void ma_load_role(S& s, const MaArgs& p, const CUtensorMap& tmap_q, const CUtensorMap& tmap_k,
                                             const CUtensorMap& tmap_kb, const CUtensorMap& tmap_v,
                                             const CUtensorMap& tmap_vb, int first, int stride, int rank) {
  constexpr int kStages = S::kStages;
  const int lane = threadIdx.x & 31;
  if (lane == 0) {
    if (!kV) prefetch_tensormap(&tmap_q);
    prefetch_tensormap(kV ? &tmap_v : &tmap_k);
    prefetch_tensormap(kV ? &tmap_vb : &tmap_kb);
  }
  const uint64_t pol_q = policy_evict_first();
  const uint64_t pol_kv = policy_evict_normal();
  const int oob = p.num_blocks * p.block_size;
  const int per_tile = kMaTile >> p.piece_log;
  int nq = 0, ring = 0, n_raw = 0;  // Q loads, K and V tiles, and V tiles to be cleaned issued
  bool ok = true;
  for (int i = first; ok && i < p.n_items; i += stride) {
    const MaItem it = ma_item<kTree, kShared>(p, i, rank);
    if (it.skip) {
      if (!kV && lane == 0 && it.tok0 < it.n) atomicCAS(p.status, 0, NPL_DEV_BAD_INDEX);
      continue;
    }
    if (!kV && lane == 0 && it.prefix < 0 && it.ctx != 0)
      atomicCAS(p.status, 0, NPL_DEV_BAD_INDEX);
    if (it.nt == 0) continue;
    const int32_t* table = p.bt + it.b * p.bt_stride;
    // the pool row of this lane's piece of tile t (zeros where its page is none of the pool), -1: not loaded
    auto lookup = [&](int t) -> int {
      const int x = it.x0 + t * kMaTile + (lane << p.piece_log);
      if (lane >= per_tile || x >= it.x1 || (x >= it.sink_x && x < it.hole_x)) return -1;
      const int key = x < it.sink_x ? x : x + it.shift;
      const int page = p.by_page(key);
      const int blk = page < p.max_blocks ? table[page] : -1;
      if (blk < 0 || blk >= p.num_blocks) {
        atomicCAS(p.status, 0, NPL_DEV_BAD_INDEX);
        return oob;
      }
      return blk * p.block_size + (key - page * p.block_size);
    };
    auto load = [&](bool k, bool part, int t, int row, int kvh) -> bool {
      const int st = ring % kStages;
      if (!kShared && k == kV) {  // the other warp's
        ++ring;
        return true;
      }
      const uint32_t loaded = __ballot_sync(0xffffffffu, row >= 0);
      bool go = true;
      if (lane == 0) {
        go = ma_wait(&s.empty[st], ((ring / kStages) & 1) ^ 1, &s.abort, p.status, NPL_DEV_TIMEOUT_TMA);
        if (go) {
          if (kShared && !part) mbar_arrive(&s.full[st]);  // in the place of the second warp that cleans
          mbar_arrive_expect_tx(part ? &s.raw[n_raw % kStages] : &s.full[st], (__popc(loaded) << p.piece_log) * D * 2);
        }
      }
      go = __shfl_sync(0xffffffffu, (int)go, 0);
      if (!go) return false;
      // pieces that lie together in the pool by one load, the ragged ends of a context or a window one by one
      const int lead = lane >> p.box_log << p.box_log, lead_x = it.x0 + t * kMaTile + (lead << p.piece_log);
      const uint32_t group = (1u << (1 << p.box_log)) - 1;  // at most 16 pieces of 8 keys
      const int row0 = __shfl_sync(0xffffffffu, row, lead), row1 = __shfl_sync(0xffffffffu, row, lead + (1 << p.box_log) - 1);
      const bool big = ((loaded >> lead) & group) == group && row1 - row0 == (p.piece << p.box_log) - p.piece &&
                       (lead_x >= it.hole_x || lead_x + (p.piece << p.box_log) <= it.sink_x);
      if (row >= 0 && (!big || lane == lead))
        ma_load_rows(s.kv[st] + (lane << p.piece_log) * D * 2, k ? (big ? &tmap_kb : &tmap_k) : (big ? &tmap_vb : &tmap_v),
                     row >> 3, kvh, part ? &s.raw[n_raw % kStages] : &s.full[st], pol_kv);
      ++ring;
      n_raw += part;
      return true;
    };
    // K of the first tile, then V of tile t and K of the next one, for each stream of its own tiles
    int row = -1, next = lookup(0);
    const int streams = !kShared && it.second ? 2 : 1;
#pragma unroll 1
    for (int t = -1; ok && t < it.nt; ++t) {
      const bool part = t >= 0 && ma_part(it, it.x0 + t * kMaTile);
      const int after = t + 2 < it.nt ? lookup(t + 2) : -1;  // ahead of the wait for a free stage
#pragma unroll 1
      for (int n = t < 0 ? 1 : 0; ok && n < 2 * streams; ++n) {
        const bool k = n & 1;
        if (t < 0 && !k) continue;
        if (!k || t + 1 < it.nt) ok = load(k, !k && part, k ? t + 1 : t, k ? next : row, it.kvh + (n >> 1));
      }
      if (!kV && t == (kShared ? 0 : -1) && ok) {  // three or two tiles ahead: less than the ring holds
        // Q after the first tiles: those need not wait until the Q before has been read
        if (lane == 0) {
          const int buf = nq % S::kQBufs;
          ok = ma_wait(&s.q_empty[buf], (nq / S::kQBufs & 1) ^ 1, &s.abort, p.status, NPL_DEV_TIMEOUT_TMA);
          if (ok) {
            mbar_arrive_expect_tx(&s.q_full[buf], (it.second ? 2 : 1) * p.tokens * p.G * D * 2);
#pragma unroll 1
            for (int q = 0; q < (it.second ? 2 : 1); ++q)
#pragma unroll
              for (int hf = 0; hf < D / 64; ++hf)
                tma_load_3d(s.q[buf][q] + hf * S::kQHalf, &tmap_q, hf * 64, (it.kvh + (kShared ? 0 : q)) * p.G,
                            it.start + it.tok0 + (kShared ? q * p.tokens : 0), &s.q_full[buf], pol_q);
          }
        }
        ok = __shfl_sync(0xffffffffu, (int)ok, 0);
        if (ok) ++nq;
      }
      row = next;
      next = after;
    }
  }
  // Every load issued here has landed before the CTA may exit.
  if (lane == 0) {
    for (int j = max(0, nq - S::kQBufs); j < nq; ++j)
      mbar_wait(&s.q_full[j % S::kQBufs], (j / S::kQBufs) & 1, p.status, NPL_DEV_TIMEOUT_TEARDOWN);
    for (int j = max(0, ring - kStages); j < ring; ++j)
      mbar_wait(&s.full[j % kStages], (j / kStages) & 1, p.status, NPL_DEV_TIMEOUT_TEARDOWN);
  }
  __syncwarp();
}

// Warp 9: matrix products. All lanes go through it, one issues: addresses and
// descriptors then stay in uniform registers, which tcgen05.mma reads, and the
// votes tell the compiler that the branches are uniform too.
template <typename S, typename T, int D, bool kTree, bool kShared>
__device__ __forceinline__ void ma_mma_role(S& s, const MaArgs& p, uint32_t tmem, int first, int stride, int rank) {
  constexpr int kStages = S::kStages;
  constexpr uint32_t kTile = S::kTileBytes >> 4;  // in units of a descriptor's address
  // rows as M: S = Q K^T, O = P V with P in TMEM; rows as N: S^T = K Q^T, O^T = V^T P^T with P^T in shared memory (for
  // D = 64 the rows of O^T come twice, the second time to lanes that nobody reads)
  constexpr uint32_t kIdQK = idesc_f16(kMaTile, S::kFew ? S::kRows : kMaTile, false) | MaType<T>::kIdesc;
  constexpr uint32_t kIdPV =
      idesc_f16(kMaTile, S::kFew ? 2 * S::kRows : D, true) | (S::kFew ? 1u << 15 : 0u) | MaType<T>::kIdesc;
  const bool issuer = elect_one();
  const uint64_t q_desc = sdesc_k_sw128(smem_u32(s.q)), k_desc = ma_desc_k(smem_u32(s.kv), S::kGroup);
  const uint64_t v_desc = ma_desc_mn(smem_u32(s.kv), S::kFew && D == 64 ? 0 : 1024, S::kGroup);
  int stage = 0, nq = 0;
  uint32_t phase = 0, p_phase[2] = {0, 0};
  auto next = [&](int& st, uint32_t& ph) {
    if (++st == kStages) st = 0, ph ^= 1;
  };
  auto wait = [&](uint64_t* bar, uint32_t ph) -> bool {
    const bool ok = ma_wait_warp(bar, ph, &s.abort, p.status, NPL_DEV_TIMEOUT_MMA);
    tc_fence_after();
    return ok;
  };
  auto issue_s = [&](int st, int at, int qb) {  // S of stream st from the K tile in stage `at`
    const uint64_t qd = q_desc + (uint32_t)(qb * 2 + st) * (sizeof(s.q[0][0]) >> 4), kd = k_desc + (uint32_t)at * kTile;
    if (issuer) {
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const uint64_t qk = qd + (((kk >> 2) * S::kQHalf + (kk & 3) * 32) >> 4), kk2 = kd + (((kk >> 2) * 1024 + (kk & 3) * 32) >> 4);
        mma_f16(tmem + st * S::kScoreCols, S::kFew ? kk2 : qk, S::kFew ? qk : kk2, kIdQK, kk > 0 ? 1u : 0u);
      }
      tc_commit(&s.s_full[st]);
    }
  };
  auto issue_o = [&](int st, int at, uint32_t add) {  // O of stream st (+)= P V
    const uint64_t vd = v_desc + (uint32_t)at * kTile;
    const uint32_t o = tmem + 2 * S::kScoreCols + st * S::kOutCols;
    if (issuer) {
#pragma unroll
      for (int kk = 0; kk < kMaTile / 16; ++kk) {
        const uint64_t vk = vd + (kk * 2 * S::kGroup >> 4);
        if constexpr (S::kFew)
          mma_f16(o, vk, sdesc_mn_sw128(smem_u32(s.p[st]), 0, 1024) + (kk * 16 * 128 >> 4), kIdPV, kk > 0 ? 1u : add);
        else
          ma_mma_ts(o, tmem + st * S::kScoreCols + kk * 8, vk, kIdPV, kk > 0 ? 1u : add);
      }
    }
  };
  bool ok = true;
  for (int i = first; ok && i < p.n_items; i += stride) {
    const MaItem it = ma_item<kTree, kShared>(p, i, rank);
    if (__all_sync(0xffffffffu, it.nt == 0)) continue;
    const int qb = nq % S::kQBufs;
    ok = wait(&s.q_full[qb], (nq / S::kQBufs) & 1);
    ++nq;
    const bool two = __any_sync(0xffffffffu, it.second);
    // S of the first tile, then O of tile t and S of the next one, for each stream
#pragma unroll 1
    for (int t = -1; __all_sync(0xffffffffu, ok && t < it.nt); ++t) {
      const bool more = __any_sync(0xffffffffu, t + 1 < it.nt), old = t >= 0;
      int sv = stage, sk = stage;  // stages of the V and the K tile
      uint32_t pv = phase, pk = phase;
      if (old) next(sk, pk);
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        if (st == 1 && !two) break;
        const bool last = !kShared || st == 1 || !two;  // of those that read these tiles
        if (old) {
          ok = wait(&s.p_full[st], p_phase[st]) && wait(&s.full[sv], pv);
          if (!ok) break;
          p_phase[st] ^= 1;
          issue_o(st, sv, t > 0 ? 1u : 0u);
          if (issuer && last) tc_commit(&s.empty[sv]);
          if (issuer && !more) tc_commit(&s.o_full[st]);
        }
        if (more) {
          ok = wait(&s.full[sk], pk);
          if (!ok) break;
          issue_s(st, sk, qb);
          if (issuer && last) tc_commit(&s.empty[sk]);
        }
        if (last) {
          if (old) next(stage, phase);
          if (more) next(stage, phase);
          if (!kShared) {
            sv = sk = stage;
            pv = pk = phase;
            if (old) next(sk, pk);
          }
        }
      }
      if (issuer && ok && t + 2 == it.nt) tc_commit(&s.q_empty[qb]);  // the last S of the item has been issued
    }
  }
  if (issuer) tc_commit(&s.mma_done);  // arrives once every MMA issued above has completed
  mbar_wait(&s.mma_done, 0, p.status, NPL_DEV_TIMEOUT_TEARDOWN);
  __syncwarp();
}

// Barriers and tensor memory of a CTA.
template <typename S, bool kShared>
__device__ __forceinline__ void ma_start(S& s) {
  constexpr int kStages = S::kStages;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&s.full[i], kShared ? 2 : 1);
      mbar_init(&s.empty[i], 1);
      mbar_init(&s.raw[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.q_full[i], 1);
      mbar_init(&s.q_empty[i], 1);
      mbar_init(&s.s_full[i], 1);
      mbar_init(&s.p_full[i], 4);  // one arrival a warp
      mbar_init(&s.o_full[i], 1);
    }
    mbar_init(&s.mma_done, 1);
    s.abort = 0;
    fence_mbar_init();
  }
  if (threadIdx.x >> 5 == 9) {
    tmem_alloc(&s.tmem_base, S::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
}

// Joins the partial sums of a cluster's CTAs. A warp takes a row of the item:
// out = sum_j 2^(m_j - M) O_j / sum_j 2^(m_j - M) l_j. where(stream, row, chunk
// of 4 columns) says where a CTA keeps its m and l, and its O.
struct MaPart {
  const float2* ml;
  const float* o;
};
template <typename T, int D, typename Where, typename Head, typename Token>
__device__ __forceinline__ void ma_join(const MaArgs& p, const MaItem& it, int rank, int r0, int r1, Where&& where,
                                        Head&& head_of, Token&& token_of) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kLanes = D / 4;  // lanes of a row: 4 columns each
  const int sub = lane / kLanes, col = lane % kLanes;
#pragma unroll 1
  for (int w = (rank * (kMaThreads / 32) + warp) * (32 / kLanes); w < r0 + r1;
       w += p.split * (kMaThreads / 32) * (32 / kLanes)) {
    const int idx = w + sub;
    const bool on = idx < r0 + r1;
    const int st = on && idx >= r0 ? 1 : 0, r = on ? idx - (st ? r0 : 0) : 0;
    const MaPart at = where(st, r, col);
    float2 part[kMaMaxSplit];
    float4 v[kMaMaxSplit];
#pragma unroll
    for (int j = 0; j < kMaMaxSplit; ++j) {  // all on their way at once; the first ones again where there are fewer
      part[j] = ma_ld_cluster2(cluster_map(at.ml, j & (p.split - 1)));
      v[j] = ma_ld_cluster(cluster_map(at.o, j & (p.split - 1)));
    }
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < kMaMaxSplit; ++j) top = part[j].x > top || part[j].x != part[j].x ? part[j].x : top;
    if (top == -INFINITY) top = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
#pragma unroll
    for (int j = 0; j < kMaMaxSplit; ++j) {
      if (j >= p.split || part[j].y == 0.f) continue;  // y 0: no key of this part is seen
      const float f = ma_exp2(part[j].x - top);
      l = fmaf(part[j].y, f, l);
      acc.x = fmaf(v[j].x, f, acc.x);
      acc.y = fmaf(v[j].y, f, acc.y);
      acc.z = fmaf(v[j].z, f, acc.z);
      acc.w = fmaf(v[j].w, f, acc.w);
    }
    const float inv = l == 0.f ? 0.f : __frcp_rn(l);
    if (on) {
      const int tok = p.by_group(r);
      T* const dst = static_cast<T*>(p.out) + (it.start + it.tok0 + token_of(st) + tok) * p.ld_out +
                     (long long)((it.kvh + head_of(st)) * p.G + r - tok * p.G) * D;
      reinterpret_cast<uint2*>(dst)[col] =
          make_uint2(MaType<T>::pack(acc.x * inv, acc.y * inv), MaType<T>::pack(acc.z * inv, acc.w * inv));
    }
  }
}

template <typename T, int D, bool kTree, bool kShared>
__global__ void __launch_bounds__(kMaThreads, 1)
    masked_attn_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                       const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ CUtensorMap tmap_kb,
                    const __grid_constant__ CUtensorMap tmap_vb, const __grid_constant__ MaArgs p) {
  using S = MaSmem<D>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  S& s = *reinterpret_cast<S*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // a cluster of `split` CTAs works on one item; without a split a CTA takes items with the grid's stride
  const int rank = blockIdx.x & (p.split - 1);
  const int first = blockIdx.x >> p.split_log;
  const int stride = p.split > 1 ? p.n_items : gridDim.x;

  ma_start<S, kShared>(s);
  const uint32_t tmem = s.tmem_base;
  pdl_wait();  // q, the pool and the metadata come from earlier work on the stream
  pdl_trigger();

  if (warp == 8) {
    ma_load_role<S, D, kTree, kShared, false>(s, p, tmap_q, tmap_k, tmap_kb, tmap_v, tmap_vb, first, stride, rank);
  } else if (warp == 9) {
    ma_mma_role<S, T, D, kTree, kShared>(s, p, tmem, first, stride, rank);
  } else if (!kShared && warp == 11) {
    ma_load_role<S, D, kTree, kShared, true>(s, p, tmap_q, tmap_k, tmap_kb, tmap_v, tmap_vb, first, stride, rank);
  } else if (warp >= 10) {
    ma_clean_role<S, T, D, kTree, kShared>(s, p, first, stride, rank);
  } else {
    // -------------------------------------------------------- softmax
    const int st = warp >> 2;            // stream
    const int r = threadIdx.x & 127;     // row of the tile = TMEM lane
    const int row_tok = p.by_group(r), row_head = r - row_tok * p.G;
    const uint32_t lane_tm = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t s_tm = lane_tm + st * 128, o_tm = lane_tm + 256 + st * 128;
    const int owner = kShared ? 0 : st;  // the stream whose V tiles this one reads
    uint32_t s_phase = 0, o_phase = 0;
    int item_no = 0;
    bool ok = true;
    MaItem ahead = ma_item<kTree, kShared>(p, min(first, p.n_items - 1), rank);
    for (int i = first; ok && i < p.n_items; i += stride) {
      const MaItem it = ahead;
      if (it.skip || (st == 1 && !it.second)) {
        ahead = ma_item<kTree, kShared>(p, min(i + stride, p.n_items - 1), rank);
        continue;
      }
      const int kvh = it.kvh + (kShared ? 0 : st);
      const int tok0 = it.tok0 + (kShared ? st * p.tokens : 0);
      const int n_rows = min(p.tokens, it.n - tok0) * p.G;
      const bool row_ok = r < n_rows;
      const bool warp_on = (warp & 3) * 32 < n_rows;
      const int token = tok0 + row_tok, pos = it.prefix + token;
      const int list = S::list(item_no, it.second);
      bool any_part = false;
      float m = -INFINITY, l = 0.f;  // m in units of log2
      // this row sees x < row_a and row_b <= x < row_e (window)
      const int row_a = row_ok ? min(it.sink_x ? p.sinks : min(p.sinks, pos + 1), it.x1) : 0;
      const int row_b = max(0, pos - p.window + 1) - it.shift, row_e = row_ok ? min(pos + 1 - it.shift, it.x1) : 0;
      for (int t = 0; ok && t < it.nt; ++t) {
        const int xt = it.x0 + t * kMaTile;
        // which of the tile's columns this row sees
        uint32_t seen[4];
        const bool part = ma_part(it, xt);
        any_part |= part;
        if (kTree) {
#pragma unroll
          for (int w = 0; w < 4; ++w) seen[w] = !part ? 0xffffffffu : row_ok ? ma_low(min(it.prefix, it.x1) - xt, w) : 0u;
          if (part && row_ok) {
            const uint8_t* mask = p.mask + (it.start + token) * p.ld_mask;
            const int j1 = min(it.n, it.x1 - it.prefix);
#pragma unroll 1
            for (int w = 0; w < 4; ++w) {
              const int j0 = xt - it.prefix + w * 32;
              if (j0 + 32 <= 0 || j0 >= j1) continue;
              uint32_t bits = 0;
#pragma unroll
              for (int c = 0; c < 32; ++c)
                if (j0 + c >= 0 && j0 + c < j1 && mask[j0 + c]) bits |= 1u << c;
              seen[0] |= w == 0 ? bits : 0u;
              seen[1] |= w == 1 ? bits : 0u;
              seen[2] |= w == 2 ? bits : 0u;
              seen[3] |= w == 3 ? bits : 0u;
            }
          }
        } else {
#pragma unroll
          for (int w = 0; w < 4; ++w) seen[w] = 0xffffffffu;
          if (part) {
#pragma unroll
            for (int w = 0; w < 4; ++w)
              seen[w] = ma_low(row_a - xt, w) | (ma_low(row_e - xt, w) & ~ma_low(row_b - xt, w));
          }
        }
        if (!ma_wait_warp(&s.s_full[st], s_phase, &s.abort, p.status, NPL_DEV_TIMEOUT_EPILOGUE)) {
          ok = false;
          break;
        }
        s_phase ^= 1;
        tc_fence_after();
        if (warp_on) {
          const bool masked = __any_sync(0xffffffffu, (seen[0] & seen[1] & seen[2] & seen[3]) != 0xffffffffu);
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          uint64_t ls[2] = {ma_pair(0.f, 0.f), ma_pair(0.f, 0.f)};
          // m moves to the tile's maximum where that is far above it, and the sums with it
          auto settle = [&]() -> float {
            const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.c2;
            const bool move = t == 0 || top > m + kMaSlack;
            const float m_new = move ? top : m;
            if (t > 0 && __any_sync(0xffffffffu, move)) {
              const float alpha = !move ? 1.f : m == -INFINITY ? 0.f : ma_exp2(m - m_new);
              l *= alpha;
#pragma unroll 1
              for (int c = 0; c < D / 32; ++c) {
                uint32_t o[32];
                tmem_ld_x32(o_tm + c * 32, o);
                ma_tmem_wait_ld(o);
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                ma_tmem_st_x16(o_tm + c * 32, o);
                ma_tmem_st_x16(o_tm + c * 32 + 16, o + 16);
              }
            }
            m = m_new;
            const float add = m == -INFINITY ? 0.f : kMaShift - m;
            return add;
          };
          // The row is read twice, 32 columns at a time and the next ones ahead: its maximum, then the exponentials.
          // (Held in registers, its 128 scores spilled.) Masked scores are written back in between.
          uint32_t v[2][32];
          tmem_ld_x32(s_tm, v[0]);
          if (!masked) {
#pragma unroll
            for (int h = 0; h < 4; ++h) {
              ma_tmem_wait_ld(v[h & 1]);
              tmem_ld_x32(s_tm + (h < 3 ? h + 1 : 0) * 32, v[(h + 1) & 1]);
              ma_max32(v[h & 1], mx);
            }
          } else {
#pragma unroll 1
            for (int h = 0; h < 4; h += 2) {
              ma_tmem_wait_ld(v[0]);
              tmem_ld_x32(s_tm + (h + 1) * 32, v[1]);
              if (ma_hide(v[0], h ? seen[2] : seen[0])) ma_tmem_st_x32(s_tm + h * 32, v[0]);
              ma_max32(v[0], mx);
              ma_tmem_wait_ld(v[1]);
              if (h == 0) tmem_ld_x32(s_tm + 64, v[0]);
              if (ma_hide(v[1], h ? seen[3] : seen[1])) ma_tmem_st_x32(s_tm + h * 32 + 32, v[1]);
              ma_max32(v[1], mx);
            }
            ma_tmem_wait_st();
            tmem_ld_x32(s_tm, v[0]);
          }
          ma_tmem_wait_ld(v[0]);
          const float add = settle();
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            uint32_t pk[16];
            if (h > 0) ma_tmem_wait_ld(v[h & 1]);
            if (h < 3) tmem_ld_x32(s_tm + (h + 1) * 32, v[(h + 1) & 1]);
            ma_exp_pack<T, kMaPoly>(v[h & 1], p.c2, add, ls, pk);
            ma_tmem_st_x16(s_tm + h * 16, pk);  // over columns that have been read
          }
          const float2 l0 = ma_unpair(ls[0]), l1 = ma_unpair(ls[1]);
          l += (l0.x + l0.y) + (l1.x + l1.y);
          ma_tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.p_full[st]);
      }
      ahead = ma_item<kTree, kShared>(p, min(i + stride, p.n_items - 1), rank);  // while the last products run
      // every MMA of the item has completed; before the partial sums go over the ring, those of the other stream too
      if (ok && it.nt > 0) {
        ok = ma_wait_warp(&s.o_full[st], o_phase, &s.abort, p.status, NPL_DEV_TIMEOUT_EPILOGUE);
        if (ok && p.split > 1 && it.second)
          ok = ma_wait_warp(&s.o_full[st ^ 1], o_phase, &s.abort, p.status, NPL_DEV_TIMEOUT_EPILOGUE);
        o_phase ^= 1;
        tc_fence_after();
      }
      if (!ok) break;
      if (warp_on) {
        const int* const n_bad = s.n_bad[list][owner];
        const bool bad = any_part && n_bad[0] + n_bad[1] > 0;  // written before the P.V products of such tiles
        const float inv = p.split > 1 ? 1.f : l == 0.f ? 0.f : __frcp_rn(l);
        float* const stage = reinterpret_cast<float*>(s.kv) + (size_t)(st * kMaTile + r) * D;
        T* const dst = static_cast<T*>(p.out) + (it.start + token) * p.ld_out +
                       (long long)(kvh * p.G + row_head) * D;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          if (it.nt > 0) {
            tmem_ld_x32(o_tm + c * 32, o);
            ma_tmem_wait_ld(o);
          }
          if (!row_ok) continue;
          if (l == 0.f) {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0;
          }
          if (p.split > 1) {
#pragma unroll
            for (int e = 0; e < 8; ++e)  // 16-byte chunks exchanged within 8, so that 8 rows use all banks
              *reinterpret_cast<uint4*>(stage + (((c * 8 + e) ^ (r & 7)) << 2)) =
                  make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
          } else {
            uint32_t w[16];
#pragma unroll
            for (int e = 0; e < 16; ++e)
              w[e] = MaType<T>::pack(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv);
            if (p.out32) {
#pragma unroll
              for (int e = 0; e < 2; ++e) ma_st_32b(dst + c * 32 + e * 16, w + e * 8);
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                reinterpret_cast<uint4*>(dst)[c * 4 + e] = make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
            }
          }
        }
        if (bad && row_ok && l != 0.f) {
          const int n = ma_bad_count<kTree, kShared>(&p, n_bad, i, rank);
#pragma unroll 1
          for (int j = 0; j < n; ++j) {
            size_t at;
            const int key = ma_bad_key<D, kTree, kShared>(&p, n_bad, s.bad[list][owner], i, rank, kvh, j, &at);
            if (key < 0 || !ma_sees<kTree>(p, it, token, key)) continue;
#pragma unroll 1
            for (int d = 0; d < D; ++d) {
              const float x = MaType<T>::get(p.v, at + d);
              if (isfinite(x)) continue;
              if (p.split > 1)
                stage[(((d >> 2) ^ (r & 7)) << 2) + (d & 3)] += x;
              else
                MaType<T>::add(dst + d, x);
            }
          }
        }
        if (p.split > 1 && row_ok)
          reinterpret_cast<float2*>(reinterpret_cast<float*>(s.kv) + 2 * kMaTile * D)[st * kMaTile + r] =
              make_float2(m, l);
      }
      if (it.nt > 0) item_no = S::next(item_no, it.second);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, S::kTmemCols);
  }
  if (p.split > 1) {
    cluster_arrive_release();
    cluster_wait_acquire();
    const MaItem it = ma_item<kTree, kShared>(p, first, rank);
    if (!it.skip) {
      const int r0 = min(p.tokens, it.n - it.tok0) * p.G;
      const int r1 = !it.second ? 0 : kShared ? min(p.tokens, it.n - it.tok0 - p.tokens) * p.G : r0;
      const float* base = reinterpret_cast<const float*>(s.kv);
      ma_join<T, D>(p, it, rank, r0, r1, [&](int st, int r, int chunk) {
        return MaPart{reinterpret_cast<const float2*>(base + 2 * kMaTile * D) + st * kMaTile + r,
                      base + (st * kMaTile + r) * D + ((chunk ^ (r & 7)) << 2)};
      }, [&](int st) { return kShared ? 0 : st; }, [&](int st) { return kShared ? st * p.tokens : 0; });
    }
    cluster_arrive_release();  // no CTA leaves while another reads its shared memory
    cluster_wait_acquire();
  }
}

// Few rows (at most kN of a kv head: single tokens, small trees) as the N side
// (8 x 16 drafts over 560 to 2000 keys of 32 heads 40.1 us, as rows of a tile 45.3;
// 8 x 32 44.4 and 47.7; from 33 rows on the other kernel is as fast):
// S^T = K Q^T has a key a TMEM lane and a row a column, so that a thread takes
// kN exponentials a tile and none is spent on rows that do not exist. O^T =
// V^T P^T has a column of the head a lane. P^T has twice kN columns, p rounded and
// what the rounding left, in one product whose two halves are added at the end
// (1 token 14.1 -> 14.2 us, 64 tokens 165.1 -> 166.2). The rows' references m are kept in
// shared memory and moved, by all threads of the stream together, in the rare
// tile that exceeds one by more than 2^8. Columns are taken 16 at a time.
template <typename T, int D, bool kTree, int kN>
__global__ void __launch_bounds__(kMaThreads, 1)
    few_rows_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                    const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ CUtensorMap tmap_kb,
                    const __grid_constant__ CUtensorMap tmap_vb, const __grid_constant__ MaArgs p) {
  using S = MaFewSmem<D, kN>;
  constexpr float kNone = 3e38f;  // 6 - m of a row that has seen no key yet
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  S& s = *reinterpret_cast<S*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x & (p.split - 1);
  const int first = blockIdx.x >> p.split_log;
  const int stride = p.split > 1 ? p.n_items : gridDim.x;
  ma_start<S, false>(s);
  const uint32_t tmem = s.tmem_base;
  pdl_wait();  // q, the pool and the metadata come from earlier work on the stream
  pdl_trigger();

  if (warp == 8) {
    ma_load_role<S, D, kTree, false, false>(s, p, tmap_q, tmap_k, tmap_kb, tmap_v, tmap_vb, first, stride, rank);
  } else if (warp == 9) {
    ma_mma_role<S, T, D, kTree, false>(s, p, tmem, first, stride, rank);
  } else if (warp == 11) {
    ma_load_role<S, D, kTree, false, true>(s, p, tmap_q, tmap_k, tmap_kb, tmap_v, tmap_vb, first, stride, rank);
  } else if (warp == 10) {
    ma_clean_role<S, T, D, kTree, false>(s, p, first, stride, rank);
  } else {
    // -------------------------------------------------------- softmax
    const int st = warp >> 2;         // stream
    const int r = threadIdx.x & 127;  // key of the tile, and column of the output: TMEM lane
    const uint32_t lane_tm = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t s_tm = lane_tm + st * kN, o_tm = lane_tm + 2 * kN + st * 2 * kN;
    uint32_t s_phase = 0, o_phase = 0;
    int item_no = 0;
    bool ok = true;  // the same for all threads of the stream at the top of a loop
    for (int i = first; ok && i < p.n_items; i += stride) {
      const MaItem it = ma_item<kTree, false>(p, i, rank);
      if (it.skip) continue;
      if (st == 1 && !it.second) continue;
      const int kvh = it.kvh + st;
      const int n_rows = min(p.tokens, it.n - it.tok0) * p.G;
      const int list = S::list(item_no, it.second);
      bool any_part = false;
      float m = -INFINITY;  // of row r, units of log2 (threads r < kN)
      if (r < kN) s.add[st][r] = r < n_rows ? kNone : -INFINITY;  // p = 0 in rows that do not exist
      ma_stream_sync(st);
      float l[kN];  // of this thread's keys
#pragma unroll
      for (int n = 0; n < kN; ++n) l[n] = 0.f;
#pragma unroll 1
      for (int t = 0; ok && t < it.nt; ++t) {
        const int xt = it.x0 + t * kMaTile, x = xt + r, key = x < it.sink_x ? x : x + it.shift;
        // which rows see this thread's key, and whether all rows see all of the tile's keys
        const bool part = ma_part(it, xt);
        any_part |= part;
        uint32_t seen[(kN + 31) / 32];
        const bool some = x < it.x1 && key < it.hi && (kTree || key >= it.lo || key < p.sinks);
        if (part) {
          int from = 0, to = some ? kN : 0;  // rows
          if (!kTree && some) {
            from = max(0, key - it.prefix - it.tok0) * p.G;
            if (key >= p.sinks) to = (int)min((long long)kN, ((long long)key + p.window - it.prefix - it.tok0) * p.G);
          }
          if (kTree && some && key >= it.prefix) to = 0;
#pragma unroll
          for (int w = 0; w < (kN + 31) / 32; ++w) seen[w] = ma_low(to, w) & ~ma_low(from, w);
          if (kTree && some && key >= it.prefix) {
            const uint8_t* mask = p.mask + (long long)it.start * p.ld_mask + (key - it.prefix);
#pragma unroll 4
            for (int tok = 0; tok < it.n; ++tok) {
              if (!mask[tok * p.ld_mask]) continue;
#pragma unroll
              for (int w = 0; w < (kN + 31) / 32; ++w)
                seen[w] |= ma_low((tok + 1) * p.G, w) & ~ma_low(tok * p.G, w);
            }
          }
        }
        bool fine = ma_wait(&s.s_full[st], s_phase, &s.abort, p.status, NPL_DEV_TIMEOUT_EPILOGUE);
        s_phase ^= 1;
        fine = __all_sync(0xffffffffu, fine);
        tc_fence_after();
        auto hide = [&](uint32_t(&v)[16], int n) {  // scores of rows n .. n + 15 that do not see this key
          const uint32_t bits = (n >> 5 ? seen[(kN - 1) >> 5] : seen[0]) >> (n & 31);
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (!(bits & (1u << e))) v[e] = 0xff800000u;
        };
        uint32_t v[16];
        bool above = false;
        if (fine) {
#pragma unroll 1
          for (int n = 0; n < kN; n += 16) {
            ma_tmem_ld_x16(s_tm + n, v);
            if (part) hide(v, n);
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
              const float4 add = *reinterpret_cast<const float4*>(&s.add[st][n + e]);
              above |= fmaxf(fmaxf(fmaf(__uint_as_float(v[e]), p.c2, add.x), fmaf(__uint_as_float(v[e + 1]), p.c2, add.y)),
                             fmaxf(fmaf(__uint_as_float(v[e + 2]), p.c2, add.z),
                                   fmaf(__uint_as_float(v[e + 3]), p.c2, add.w))) > kMaShift + kMaSlack;
            }
          }
        }
        if (ma_stream_any(st, above || !fine)) {
          if (ma_stream_any(st, !fine)) {
            ok = false;
            break;
          }
          // some row's reference moves to its maximum so far
#pragma unroll 1
          for (int n = 0; n < kN; n += 16) {
            if (kN > 16) {
              ma_tmem_ld_x16(s_tm + n, v);
              if (part) hide(v, n);
            }
            float top[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) top[e] = __uint_as_float(v[e]);
            ma_warp_reduce(top, lane, [](float a, float b) { return fmaxf(a, b); });
            if (lane < 16) s.top[st][warp & 3][n + lane] = top[0];
          }
          ma_stream_sync(st);
          if (r < kN) {
            const float top = fmaxf(fmaxf(s.top[st][0][r], s.top[st][1][r]),
                                    fmaxf(s.top[st][2][r], s.top[st][3][r])) * p.c2;
            const bool move = r < n_rows && (m == -INFINITY || top > m + kMaSlack);
            const float m_new = move ? top : m;
            s.alpha[st][r] = !move ? 1.f : m == -INFINITY ? 0.f : ma_exp2(m - m_new);
            m = m_new;
            if (r < n_rows) s.add[st][r] = m == -INFINITY ? kNone : kMaShift - m;
          }
          ma_stream_sync(st);
#pragma unroll
          for (int n = 0; n < kN; ++n) l[n] *= s.alpha[st][n];
          if (t > 0) {
#pragma unroll 1
            for (int n = 0; n < 2 * kN; n += 16) {
              uint32_t o[16];
              ma_tmem_ld_x16(o_tm + n, o);
#pragma unroll
              for (int e = 0; e < 16; ++e)
                o[e] = __float_as_uint(__uint_as_float(o[e]) * s.alpha[st][(n & (kN - 1)) + e]);
              ma_tmem_st_x16(o_tm + n, o);
            }
            ma_tmem_wait_st();
          }
        }
        // P^T of this key: 16-byte chunks exchanged with the key's place in its 8 (128-byte swizzle)
        uint8_t* const line = s.p[st] + (r >> 3) * 1024 + (r & 7) * 128;
#pragma unroll
        for (int n = 0; n < kN; n += 16) {
          if (kN > 16) {
            ma_tmem_ld_x16(s_tm + n, v);
            if (part) hide(v, n);
          }
          uint32_t w[8], rest[8];  // p, and p less what w holds of it
#pragma unroll
          for (int e = 0; e < 16; e += 4) {
            const float4 add = *reinterpret_cast<const float4*>(&s.add[st][n + e]);
            const float p0 = ma_exp2(fmaf(__uint_as_float(v[e]), p.c2, add.x));
            const float p1 = ma_exp2(fmaf(__uint_as_float(v[e + 1]), p.c2, add.y));
            const float p2 = ma_exp2(fmaf(__uint_as_float(v[e + 2]), p.c2, add.z));
            const float p3 = ma_exp2(fmaf(__uint_as_float(v[e + 3]), p.c2, add.w));
            l[n + e] += p0;
            l[n + e + 1] += p1;
            l[n + e + 2] += p2;
            l[n + e + 3] += p3;
            w[e / 2] = MaType<T>::pack(p0, p1);
            w[e / 2 + 1] = MaType<T>::pack(p2, p3);
            const float2 a = MaType<T>::unpack(w[e / 2]), b = MaType<T>::unpack(w[e / 2 + 1]);
            rest[e / 2] = MaType<T>::pack(p0 - a.x, p1 - a.y);
            rest[e / 2 + 1] = MaType<T>::pack(p2 - b.x, p3 - b.y);
          }
          *reinterpret_cast<uint4*>(line + (((n >> 3) ^ (r & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
          *reinterpret_cast<uint4*>(line + (((n >> 3) + 1 ^ (r & 7)) << 4)) = make_uint4(w[4], w[5], w[6], w[7]);
          *reinterpret_cast<uint4*>(line + (((kN + n) >> 3 ^ (r & 7)) << 4)) = make_uint4(rest[0], rest[1], rest[2], rest[3]);
          *reinterpret_cast<uint4*>(line + (((kN + n) >> 3) + 1 ^ (r & 7)) * 16) = make_uint4(rest[4], rest[5], rest[6], rest[7]);
        }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.p_full[st]);
      }
      // every MMA of the item has completed; before the partial sums go over the ring, those of the other stream too
      if (it.nt > 0) {
        bool fine = ok && ma_wait(&s.o_full[st], o_phase, &s.abort, p.status, NPL_DEV_TIMEOUT_EPILOGUE);
        if (fine && p.split > 1 && it.second)
          fine = ma_wait(&s.o_full[st ^ 1], o_phase, &s.abort, p.status, NPL_DEV_TIMEOUT_EPILOGUE);
        o_phase ^= 1;
        ok = !ma_stream_any(st, !fine);
        tc_fence_after();
      }
      // the rows' normalisers: sums over the stream's keys
#pragma unroll
      for (int n = 0; n < kN; n += 16) {
        float sum[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) sum[e] = l[n + e];
        ma_warp_reduce(sum, lane, [](float a, float b) { return a + b; });
        if (lane < 16) s.top[st][warp & 3][n + lane] = sum[0];
      }
      ma_stream_sync(st);
      if (r < kN) {
        const float sum = (s.top[st][0][r] + s.top[st][1][r]) + (s.top[st][2][r] + s.top[st][3][r]);
        s.ml[st][r] = make_float2(m, sum);
        s.inv[st][r] = sum == 0.f ? 0.f : p.split > 1 ? 1.f : __frcp_rn(sum);
      }
      ma_stream_sync(st);
      if (ok) {
        float* const stage = reinterpret_cast<float*>(s.kv) + (size_t)st * kN * D + r;
        T* const dst = static_cast<T*>(p.out) + (it.start + it.tok0) * p.ld_out + (long long)kvh * p.G * D + r;
        T* at = dst;
        int head = 0;
#pragma unroll 1
        for (int n = 0; n < n_rows; n += 4) {
          uint32_t o[4], rest[4];
          if (it.nt > 0) ma_tmem_ld_2x4(o_tm + n, o_tm + kN + n, o, rest);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float inv = s.inv[st][n + e];
            const float y = inv == 0.f ? 0.f : (__uint_as_float(o[e]) + __uint_as_float(rest[e])) * inv;
            if (n + e < n_rows && r < D) {
              if (p.split > 1)
                stage[(n + e) * D] = y;
              else
                MaType<T>::put(at, y);
            }
            at += D;
            if (++head == p.G) head = 0, at += p.ld_out - p.G * D;
          }
        }
        const int* const n_bad = s.n_bad[list][st];
        if (any_part && n_bad[0] + n_bad[1] > 0) {  // written before the P.V products of such tiles
          ma_stream_sync(st);
          const int n_keys = ma_bad_count<kTree, false>(&p, n_bad, i, rank);
#pragma unroll 1
          for (int j = 0; r < D && j < n_keys; ++j) {
            size_t from;
            const int key = ma_bad_key<D, kTree, false>(&p, n_bad, s.bad[list][st], i, rank, kvh, j, &from);
            if (key < 0) continue;
            const float x = MaType<T>::get(p.v, from + r);
            if (isfinite(x)) continue;
#pragma unroll 1
            for (int n = 0; n < n_rows; ++n) {
              const int of = p.by_group(n);
              if (s.ml[st][n].y == 0.f || !ma_sees<kTree>(p, it, it.tok0 + of, key)) continue;
              if (p.split > 1)
                stage[n * D] += x;
              else
                MaType<T>::add(dst + of * p.ld_out + (n - of * p.G) * D, x);
            }
          }
        }
      }
      if (it.nt > 0) item_no = S::next(item_no, it.second);
      tc_fence_before();  // O has been read before this thread's next arrival, which the next O waits for
      ma_stream_sync(st);  // and the normalisers, before the next item's
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, S::kTmemCols);
  }
  if (p.split > 1) {
    cluster_arrive_release();
    cluster_wait_acquire();
    const MaItem it = ma_item<kTree, false>(p, first, rank);
    if (!it.skip) {
      const int rows = min(p.tokens, it.n - it.tok0) * p.G;
      const float* base = reinterpret_cast<const float*>(s.kv);
      ma_join<T, D>(p, it, rank, rows, it.second ? rows : 0, [&](int st, int r, int chunk) {
        return MaPart{&s.ml[st][r], base + (st * kN + r) * D + chunk * 4};
      }, [&](int st) { return st; }, [&](int) { return 0; });
    }
    cluster_arrive_release();  // no CTA leaves while another reads its shared memory
    cluster_wait_acquire();
  }
}

PFN_cuTensorMapEncodeTiled_v12000 ma_encode_fn() {
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

// K or V rows of the pool [rows][Hkv][D] as a 5-D tensor map whose box holds
// `box` rows of one head: 8 rows of 64 elements (128-byte swizzle), their second
// halves, the next 8 rows.
int ma_pool_map(const char* what, CUtensorMap* map, CUtensorMapDataType type, const void* base, long long rows, int Hkv,
                int D, int box) {
  const PFN_cuTensorMapEncodeTiled_v12000 fn = ma_encode_fn();
  if (!fn) return fail(NPL_ERR_LAUNCH, "%s: cuTensorMapEncodeTiled unavailable", what);
  const cuuint64_t ld = (cuuint64_t)Hkv * D * 2;
  const cuuint64_t dims[5] = {64, 8, (cuuint64_t)D / 64, (cuuint64_t)rows / 8, (cuuint64_t)Hkv};
  const cuuint64_t strides[4] = {ld, 128, 8 * ld, (cuuint64_t)D * 2};
  const cuuint32_t size[5] = {64, 8, (cuuint32_t)D / 64, (cuuint32_t)box / 8, 1};
  const cuuint32_t one[5] = {1, 1, 1, 1, 1};
  const CUresult r = fn(map, type, 5, const_cast<void*>(base), dims, strides, size, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(NPL_ERR_ARG, "%s: cuTensorMapEncodeTiled failed (%d)", what, (int)r);
  return NPL_OK;
}

// [rows][heads][D] (rows ld elements apart, heads contiguous) as a 3-D tensor
// map with a (64, box_heads, box_rows) box and the 128-byte swizzle.
int ma_map(const char* what, CUtensorMap* map, CUtensorMapDataType type, const void* base, long long rows, int heads,
           int D, long long ld, int box_heads, int box_rows) {
  const PFN_cuTensorMapEncodeTiled_v12000 fn = ma_encode_fn();
  if (!fn) return fail(NPL_ERR_LAUNCH, "%s: cuTensorMapEncodeTiled unavailable", what);
  const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)rows};
  const cuuint64_t strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)ld * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_rows};
  const cuuint32_t one[3] = {1, 1, 1};
  const CUresult r = fn(map, type, 3, const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(NPL_ERR_ARG, "%s: cuTensorMapEncodeTiled failed (%d)", what, (int)r);
  return NPL_OK;
}

// kRows: 0 for row tiles that share their keys, 128 for one row tile of two kv heads, else few rows.
template <typename T, int D, bool kTree, int kRows>
int launch(const char* what, MaArgs p, cudaStream_t st) {
  constexpr bool kShared = kRows == 0, kFew = kRows > 0 && kRows < kMaTile;
  p.tokens = (kFew ? kRows : kMaTile) / p.G;
  p.levels = kShared ? (p.max_q_len + 2 * p.tokens - 1) / (2 * p.tokens) : 1;
  const long long items = (long long)p.levels * p.B * (kShared ? p.Hkv : (p.Hkv + 1) / 2);
  if (items >= (1ll << 27)) return fail(NPL_ERR_UNSUPPORTED, "%s: too many row tiles", what);
  p.n_items = (int)items;
  p.by_levels = MaDiv::of(p.levels);
  p.by_units = MaDiv::of(kShared ? p.Hkv : (p.Hkv + 1) / 2);
  p.by_group = MaDiv::of(p.G);
  p.by_page = MaDiv::of(p.block_size);
  CUtensorMap tq, tk, tv, tkb, tvb;
  const long long slots = (long long)p.num_blocks * p.block_size;
  const int box = p.piece << p.box_log;
  if (int rc = ma_map(what, &tq, MaType<T>::kMap, p.q, p.total_q, p.H, D, p.ld_q, p.G, p.tokens)) return rc;
  if (int rc = ma_pool_map(what, &tk, MaType<T>::kMap, p.k, slots, p.Hkv, D, p.piece)) return rc;
  if (int rc = ma_pool_map(what, &tv, MaType<T>::kMap, p.v, slots, p.Hkv, D, p.piece)) return rc;
  if (int rc = ma_pool_map(what, &tkb, MaType<T>::kMap, p.k, slots, p.Hkv, D, box)) return rc;
  if (int rc = ma_pool_map(what, &tvb, MaType<T>::kMap, p.v, slots, p.Hkv, D, box)) return rc;
  void (*kernel)(CUtensorMap, CUtensorMap, CUtensorMap, CUtensorMap, CUtensorMap, MaArgs);
  int smem;
  if constexpr (kFew) {
    kernel = few_rows_kernel<T, D, kTree, kRows>;
    smem = (int)sizeof(MaFewSmem<D, kRows>) + 1024;
  } else {
    kernel = masked_attn_kernel<T, D, kTree, kShared>;
    smem = (int)sizeof(MaSmem<D>) + 1024;
  }
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return launch_status(what);
  // The cluster size with the least time in tiles of 128 keys: the longest item, or all rounds of clusters, each with
  // kMaFixed for the start of its CTAs and the join. Contexts may have any length up to the table's: three quarters of
  // it are taken as usual. Windows are mostly full. Split 1, 2, 4 and 8 ways, us (* is taken): 16 drafts over 1040 keys
  // of 32 heads 22.0, 19.9, 16.7*, 29.8; 8 x 64 drafts over 2000 keys 56.2*, 79.5, 110, 191; 61 drafts over 4000 keys of
  // 28/4 heads of 64 62.9, 42.1, 28.0, 21.3*; windows of 4096 of 16 tokens, 32/8 heads 71.3, 49.2*, 57.8, 89.4. Of 54
  // such (1 to 64 sequences, 1 to 2000 rows, heads of 64 and 128, even and uneven contexts, all kernels) the least time
  // is taken in 53, and one 6% above it, by any kMaFixed from 8 to 14; 6 loses up to 23%, and so does taking half the
  // table as usual. A table four times as wide as the contexts need costs up to 41%.
  long long keys = (long long)p.max_blocks * p.block_size;  // the most that an item's rows may see
  if (!kTree) keys = std::min(keys, (long long)p.window + p.sinks + 2 * p.tokens);
  const int sms = num_sms() > 0 ? num_sms() : 148;
  p.split_log = 0;
  double least = 0.0;
  for (int lg = 0; (1 << lg) <= kMaMaxSplit && (lg == 0 || p.n_items << (lg - 1) < 2 * sms); ++lg) {
    const int fit = lg == 0 ? sms : max_active_clusters(reinterpret_cast<const void*>(kernel), smem, 1 << lg, kMaThreads);
    if (fit <= 0) break;
    const double most = (double)((keys >> lg) + kMaTile - 1) / kMaTile, usual = kTree ? 0.75 * most : most;
    const int rounds = (p.n_items + fit - 1) / fit;  // without a split the CTAs stay
    const double all = lg == 0 ? rounds * usual + kMaFixed : rounds * (usual + kMaFixed);
    const double cost = std::max(most + kMaFixed, all);
    if (lg == 0 || cost < least) least = cost, p.split_log = lg;
  }
  p.split = 1 << p.split_log;
  const int grid = p.split > 1 ? p.n_items * p.split : std::min(p.n_items, sms);
  return launch_pdl_cluster(what, kernel, dim3(grid), dim3(kMaThreads), (size_t)smem, st, (unsigned)p.split, tq, tk,
                            tv, tkb, tvb, p);
}

template <typename T, int D, bool kTree>
int run_type(const char* what, const MaArgs& p, cudaStream_t st) {
  const long long rows = (long long)p.max_q_len * p.G;
  if (rows <= 16) return launch<T, D, kTree, 16>(what, p, st);
  if (rows <= 32) return launch<T, D, kTree, 32>(what, p, st);
  if (p.max_q_len <= kMaTile / p.G) return launch<T, D, kTree, 128>(what, p, st);
  return launch<T, D, kTree, 0>(what, p, st);
}

template <bool kTree>
int run(const char* what, MaArgs p, int dtype, int D, float scale, cudaStream_t st) {
  p.c2 = scale * 1.4426950408889634f;
  p.capacity = p.max_blocks * p.block_size;
  p.out32 = ((reinterpret_cast<uintptr_t>(p.out) | (uintptr_t)(p.ld_out * 2)) & 31u) == 0;
  p.piece_log = kMaPieceLog;
  while (p.block_size & ((1 << p.piece_log) - 1)) --p.piece_log;
  p.piece = 1 << p.piece_log;
  p.box_log = kMaBoxLog - p.piece_log;
  while (p.block_size & ((p.piece << p.box_log) - 1)) --p.box_log;
  if (dtype == NPL_F16)
    return D == 128 ? run_type<__half, 128, kTree>(what, p, st) : run_type<__half, 64, kTree>(what, p, st);
  return D == 128 ? run_type<__nv_bfloat16, 128, kTree>(what, p, st)
                  : run_type<__nv_bfloat16, 64, kTree>(what, p, st);
}

int check(const char* what, const MaArgs& p, int dtype, int D, float scale) {
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
  if (!(scale > 0.f) || !(scale < 2.0e38f))
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
  p.max_blocks = max_blocks, p.total_q = total_q, p.max_q_len = max_q_len;
  if (int rc = check(what, p, dtype, D, scale)) return rc;
  if (!tree_mask || !q_lens) return fail(NPL_ERR_ARG, "%s: null pointer", what);
  if (mask_cols < max_q_len || ld_mask < mask_cols)
    return fail(NPL_ERR_ARG, "%s: the mask has %d columns (stride %lld) for up to %d drafts", what, mask_cols,
                (long long)ld_mask, max_q_len);
  if (int rc = check_device()) return rc;
  if (B == 0 || total_q == 0 || max_q_len == 0) return NPL_OK;
  // No count of tiles overflows. A bound far above the lengths still costs: row tiles that do not exist are looked at
  // and passed over, and the kernel and the cluster size, and with them a row's last bits, go by the bound.
  p.max_q_len = std::min(max_q_len, total_q);
  p.status = device_status_ptr();
  return run<true>(what, p, dtype, D, scale, static_cast<cudaStream_t>(stream));
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
  p.max_blocks = max_blocks, p.total_q = total_q, p.max_q_len = q_lens ? max_q_len : 1;
  if (int rc = check(what, p, dtype, D, scale)) return rc;
  if (window < 1 || sinks < 0)
    return fail(NPL_ERR_ARG, "%s: window %d (at least 1), sinks %d (at least 0)", what, window, sinks);
  if (int rc = check_device()) return rc;
  if (B == 0 || total_q == 0 || p.max_q_len == 0) return NPL_OK;
  p.max_q_len = std::min(p.max_q_len, total_q);
  p.status = device_status_ptr();
  return run<false>(what, p, dtype, D, scale, static_cast<cudaStream_t>(stream));
}
