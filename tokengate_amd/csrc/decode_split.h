// What the decode attentions that cut every sequence's keys into chunks on the device share: lane exchanges without
// the LDS crossbar, agent-scope accesses, and the rule that cuts.
#pragma once

#include "tg_common.h"

namespace tg {
namespace {

template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, CTRL, 0xf, 0xf, true);
}
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return u32_as_f32(dpp<CTRL>(__builtin_bit_cast(uint32_t, x)));
}

template <typename T>
__device__ __forceinline__ void st_agent(T *p, T v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <typename T>
__device__ __forceinline__ T ld_agent(const T *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// 0 * x = 0, whatever x is.  (The builtin: an asm statement right behind the exponential that feeds it would read the
// register too early, as the compiler keeps the wait that such a pair needs from its own instructions only.)
extern "C" __device__ float tg_fmul_legacy(float, float) __asm("llvm.amdgcn.fmul.legacy");
__device__ __forceinline__ float mul_zero(float a, float b) { return tg_fmul_legacy(a, b); }
__device__ __forceinline__ float wave_max(float x) {
  x = fmaxf(x, dpp<0xB1>(x));    // quad_perm 1 0 3 2
  x = fmaxf(x, dpp<0x4E>(x));    // quad_perm 2 3 0 1
  x = fmaxf(x, dpp<0x141>(x));   // row_half_mirror
  x = fmaxf(x, dpp<0x140>(x));   // row_mirror
  return quad_swap_max(x);
}
__device__ __forceinline__ float add_row_pair(float x) {   // x of lanes l and l ^ 16
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t a0 = a[0], a1 = a[1];
  return u32_as_f32(a0) + u32_as_f32(a1);
}
__device__ __forceinline__ float add_rows(float x) {       // x of lanes l, l ^ 16, l ^ 32, l ^ 48
  const uint32_t v = __builtin_bit_cast(uint32_t, add_row_pair(x));
  const auto c = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  const uint32_t c0 = c[0], c1 = c[1];
  return u32_as_f32(c0) + u32_as_f32(c1);
}
__device__ __forceinline__ float wave_add(float x) {
  x += dpp<0xB1>(x);
  x += dpp<0x4E>(x);
  x += dpp<0x141>(x);
  x += dpp<0x140>(x);
  return add_rows(x);
}

// The chunk that a workgroup takes: the q-th of all sequences' chunks in turn.  A sequence of n tiles is cut into
// ceil(n / T) chunks of even length, with one T for all, from their tiles, which only the device knows: the least that
// makes no more workgroups than are resident at once (a workgroup's fixed costs, 5 us, and a second round's uneven
// end cost more than idle places), or, where the sequences' remainders alone would fill most of these, two
// rounds.
// Quantised caches, 16 / 8 heads, T for one round as far as it goes / two rounds / as here, us: 64 sequences of 512 ..
// 4099 at 8 bits 76 / 78 / 76; 64 alike of 300 18.3 / 25.5 / 18.0; 8 of 16k .. 128k at 4 bits 162 / 178 / 161; 16 of 4k
// .. 30k 82 / 91 / 82; 64 alike of 4096 69 / 78 / 69; 300 of 300 .. 3000 168 / 154 / 154; 120 of 50 .. 20000 323 / 298 / 297.
constexpr int kRounds = 2;
struct SplitRule {
  int nseq, sets;                // sequences; kv heads times head sets
  int slots, least;              // workgroups that are resident at once; fewest tiles per chunk
  float per_root = 0.f;          // if positive: least times as many as this times the root of the longest's tiles, and at
};                               // least 3 times, where that takes all of it
struct Chunk {
  int seq, chunk, chunks, tiles, sk;
  int64_t start;
};
struct Keys {                    // of a sequence: where they begin, and how many with the new one
  int64_t start;
  int sk;
};
template <int CTRL, int ROWS>
__device__ __forceinline__ int scan_step(int x) { return x + __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false); }
__device__ __forceinline__ int wave_scan(int x) {   // sum over the lanes up to this one
  x = scan_step<0x111, 0xf>(x);   // row_shr 1, 2, 4, 8
  x = scan_step<0x112, 0xf>(x);
  x = scan_step<0x114, 0xf>(x);
  x = scan_step<0x118, 0xf>(x);
  x = scan_step<0x142, 0xa>(x);   // row_bcast 15: the first row's sum to the second, the third's to the fourth
  return scan_step<0x143, 0xc>(x);   // row_bcast 31: the first half's to the second
}
__device__ __forceinline__ int wave_max_int(int x) {   // of all lanes, in every lane (whole numbers below 2^24)
  return (int)wave_max((float)x);
}
// ceil(n / T), n and T below 2^22: the quotient's float is off by less than 1 / T
__device__ __forceinline__ int ceil_div(int n, float inv) { return (int)(((float)n - 0.5f) * inv) + 1; }
// keys_of(s): the Keys of sequence s < nseq.  Tiles are of TILE keys, the new one apart.
template <int TILE, typename KeysOf>
__device__ __forceinline__ Chunk find_chunk(const SplitRule &a, int q, int lane, KeysOf keys_of) {
  int sk = 0, start = 0, tiles = 0;
  auto read = [&](int s) {                       // of sequence s, this lane's
    const Keys k = s < a.nseq ? keys_of(s) : Keys{0, 0};
    start = (int)k.start;
    sk = k.sk;
    tiles = (max(0, sk - 1) + TILE - 1) / TILE;
  };
  auto count = [&](int T, bool all) {            // chunks of all sequences, or their tiles
    int n = 0;
    const float inv = 1.f / (float)T;
    for (int s0 = 0; s0 < a.nseq; s0 += 64) {
      if (s0 > 0 || all) read(s0 + lane);
      n += wave_sum_int(all ? tiles : s0 + lane < a.nseq ? max(1, ceil_div(tiles, inv)) : 0);
    }
    if (a.nseq > 64) read(lane);
    return __builtin_amdgcn_readfirstlane(n);
  };
  const float work = (float)count(1, true) * (float)a.sets, slots = (float)a.slots;
  float target = slots;
  int least = a.least;
  if (a.per_root > 0.f) {
    int longest = 0;
    for (int s0 = 0; s0 < a.nseq; s0 += 64) {
      if (a.nseq > 64) read(s0 + lane);
      longest = max(longest, wave_max_int(tiles));
    }
    if (a.nseq > 64) read(lane);
    least = longest <= 3 * least ? max(least, longest) : least * max(1, (int)(a.per_root * __builtin_amdgcn_sqrtf((float)longest)));
  }
  int T = max(least, (int)(work / target) + 1);
  // (where not even an even cut of every sequence would fill one round, nothing is counted)
  for (int i = 0; i < 3 && work / (float)T + (float)a.nseq * (float)a.sets > slots; ++i) {
    const float over = (float)count(T, false) * (float)a.sets - slots;
    if (over <= 0.f) break;
    if (over > 0.75f * slots) {
      T = max(least, (int)(work / (kRounds * slots)) + 1);
      break;
    }
    target = fmaxf(target - over, 0.25f * slots);
    T = max(T + 1, (int)(work / target) + 1);
  }
  const float inv = 1.f / (float)T;
  int before = 0;
  for (int s0 = 0; s0 < a.nseq; s0 += 64) {
    if (s0 > 0) read(s0 + lane);
    const int n = s0 + lane < a.nseq ? max(1, ceil_div(tiles, inv)) : 0;
    const int up_to = wave_scan(n) + before;
    const uint64_t in = __builtin_amdgcn_ballot_w64(up_to > q);
    if (in) {
      const int l = (int)__builtin_ctzll(in);
      const int chunks = __builtin_amdgcn_readlane(n, l);
      return Chunk{s0 + l, q - (__builtin_amdgcn_readlane(up_to, l) - chunks), chunks, __builtin_amdgcn_readlane(tiles, l),
                   __builtin_amdgcn_readlane(sk, l), __builtin_amdgcn_readlane(start, l)};
    }
    before = __builtin_amdgcn_readlane(up_to, 63);
  }
  return Chunk{-1, 0, 0, 0, 0, 0};
}

}  // namespace
}  // namespace tg
