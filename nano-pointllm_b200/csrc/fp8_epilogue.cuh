// The order in which the threads of the e4m3 linear's epilogue meet, apart
// from what they do in between: a host program can run it too, with waits that
// run out where it wants them to.
//
// A wait is bounded, so a warp may give up where another warp of its warpgroup
// does not (the last arrival comes between their deadlines), but a named
// barrier (bar.sync) waits for all of them without a limit. So whether a
// barrier is met never goes by one warp's own waits.
#pragma once

#ifdef __CUDACC__
#define NPL_DEVICE __device__ __forceinline__
#else
#define NPL_DEVICE inline
#endif

namespace npl {

// Bounded waits of a converged warp: all lanes return the same, so none leaves
// the others alone in front of a warp-wide instruction. try_once(): whether the
// phase is complete. late(): whether this lane's deadline has passed, looked at
// after `polls` tries and then every 64 (reading the clock takes longer than
// most waits).
//
// With a vote in every try; all(v): whether v holds in all lanes.
template <typename Try, typename All, typename Late>
NPL_DEVICE bool wait_voting(int polls, Try&& try_once, All&& all, Late&& late) {
#pragma unroll 1
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < polls; ++i)
      if (all(try_once())) return true;
    if (!all(!late())) return false;
    polls = 64;
  }
}

// With a vote at the deadline only; any(v): whether v holds in one of the lanes
// still here. Lanes may see a completion in two tries that follow each other.
// Once one has left, every later try succeeds; so those that are late give up
// only after a try that succeeds in none of them.
template <typename Try, typename Any, typename Late>
NPL_DEVICE bool wait_as_one(int polls, Try&& try_once, Any&& any, Late&& late) {
#pragma unroll 1
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < polls; ++i)
      if (try_once()) return true;
    if (any(late()) && !any(try_once())) return false;
    polls = 64;
  }
}

// Decode tiles: blocks [kb0, kb1), `chunk` at a time. scales(kc) shares the
// scales of a chunk (the warps meet in it); unit(i, kc, k, kn) waits for blocks k,
// k + 1, .. of the chunk's kn (`per_unit` of them) and adds them up; false: the
// wait ran out, after which a warp still meets the others in every chunk.
template <typename Scales, typename Unit>
NPL_DEVICE void decode_epilogue(int kb0, int kb1, int chunk, int per_unit, Scales&& scales, Unit&& unit) {
  bool ok = true;
  int i = 0;
  for (int kc = kb0; kc < kb1; kc += chunk) {
    scales(kc);
    const int kn = kb1 - kc < chunk ? kb1 - kc : chunk;
    for (int k = 0; ok && k < kn; k += per_unit, ++i) ok = unit(i, kc, k, kn);
  }
}

// Prefill tiles first, first + step, ..: sums(t) adds a tile up; false: a wait
// ran out. agree(ok): the warpgroup's warps meet, whether all of them have
// their sums; only then they go on to write(t), in which they meet, too.
template <typename Sums, typename Agree, typename Write>
NPL_DEVICE void prefill_epilogue(int first, int step, int tiles, Sums&& sums, Agree&& agree, Write&& write) {
  for (int t = first; t < tiles; t += step) {
    if (!agree(sums(t))) return;
    write(t);
  }
}

}  // namespace npl
