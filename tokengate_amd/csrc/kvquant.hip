// KV caches of 4 and 8 bits: the rows are quantised as they are written, read back as bf16, and read by the
// attention of a decode step.
//
// A row of one head (128 values) is four groups of 32 consecutive values, each with its least value m and a
// step s, both bf16; a value is held as the whole number c in 0 .. L nearest to (x - m) / s and stands for
// s c + m (L = 15 or 255, s = bf16((max - m) / L)).  Why this form: at 4 bits the least value costs 16 bits a
// group and takes the mean squared error of normal data from 0.0105 (symmetric steps of max |x| / 7) to 0.0063;
// whole numbers up to 255 are bf16 numbers, so the matrix cores take them as they are, and s and m, constant
// over the 32 values that one matrix instruction sums, are applied to its sums.
//
// Layout (head-major, so that the rows that one workgroup reads are contiguous): codes (heads, rows, 16 words of
// 4 bits x 8 or pairs of words of 8 bits x 8), element 16 e + w in nibble (byte) e of word (pair) w, so that a
// lane's word holds values of all four groups; meta (heads, rows, 4) x (s, m).
#include <algorithm>
#include <type_traits>

#include "tg_common.h"
#include "../../include/tokengate_hip.h"

namespace tg {
namespace {

constexpr int kGroups = 4;                       // of 32 values
template <int BITS> constexpr int row_words() { return 4 * BITS; }
template <int BITS> constexpr float top_code() { return BITS == 4 ? 15.f : 255.f; }
constexpr float kLeastStep = 0x1p-100f;          // smaller steps are held as 0: quotients below stay normal numbers

struct QuantCache {
  uint32_t *k, *v;               // codes
  uint32_t *km, *vm;             // (s, m) bf16 pairs
  int64_t rows, head_rows;       // rows of a head, and from one head to the next
};

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("v_maximum3_f32 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c));
  return d;
}
__device__ __forceinline__ float min3_nan(float a, float b, float c) {
  float d;
  asm("v_minimum3_f32 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c));
  return d;
}

// x of lane l ^ M, of 16 lanes, without the LDS crossbar
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, CTRL, 0xf, 0xf, true);
}
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return u32_as_f32(dpp<CTRL>(__builtin_bit_cast(uint32_t, x)));
}
template <int M>
__device__ __forceinline__ uint32_t lane_xor(uint32_t x) {
  static_assert(M == 1 || M == 2 || M == 4 || M == 8, "a row of 16 lanes");
  if constexpr (M == 1) return dpp<0xB1>(x);                 // quad_perm 1 0 3 2
  else if constexpr (M == 2) return dpp<0x4E>(x);            // quad_perm 2 3 0 1
  else if constexpr (M == 4) return dpp<0x1B>(dpp<0x141>(x));   // row_half_mirror (l ^ 7), quad_perm 3 2 1 0 (l ^ 3)
  else return dpp<0x128>(x);                                 // row_ror 8
}
template <int M>
__device__ __forceinline__ float lane_xor(float x) {
  return u32_as_f32(lane_xor<M>(__builtin_bit_cast(uint32_t, x)));
}

// Lanes j = 2 e + p of 16 lanes hold element i of an 8 x 8 table (e, i) in byte i of the pair w (4 bits: nibble i of
// w): transposed among the eight lanes of the same p, part by part: a lane whose bit of e is 0 keeps its parts of
// that bit 0 and takes its partner's, the partner those of bit 1.
__device__ __forceinline__ uint32_t swap_bytes(uint32_t x, uint32_t y, bool up) {    // of 16
  return __builtin_amdgcn_perm(y, x, up ? 0x03070105u : 0x06020400u);
}
__device__ __forceinline__ uint32_t swap_halves(uint32_t x, uint32_t y, bool up) {   // of 32
  return __builtin_amdgcn_perm(y, x, up ? 0x03020706u : 0x05040100u);
}
__device__ __forceinline__ uint32_t swap_nibbles(uint32_t x, uint32_t y, bool up) {  // of 8
  const uint32_t keep = up ? 0xF0F0F0F0u : 0x0F0F0F0Fu, moved = up ? y >> 4 : y << 4;
  return (x & keep) | (moved & ~keep);
}
template <int BITS>
__device__ __forceinline__ void transpose8(uint32_t (&w)[BITS / 4], int j) {
  if constexpr (BITS == 4) {
    w[0] = swap_halves(w[0], lane_xor<8>(w[0]), j & 8);
    w[0] = swap_bytes(w[0], lane_xor<4>(w[0]), j & 4);
    w[0] = swap_nibbles(w[0], lane_xor<2>(w[0]), j & 2);
  } else {
    const uint32_t got = lane_xor<8>(j & 8 ? w[0] : w[1]);
    w[0] = j & 8 ? got : w[0];
    w[1] = j & 8 ? w[1] : got;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      w[i] = swap_halves(w[i], lane_xor<4>(w[i]), j & 4);
      w[i] = swap_bytes(w[i], lane_xor<2>(w[i]), j & 2);
    }
  }
}
// The word (pair) that lane j of a row holds after transpose8
__device__ __forceinline__ int word_of(int j) { return 8 * (j & 1) + (j >> 1); }

// Quantises a row held by 16 lanes, lane j its elements 8 j .. 8 j + 7: word (pair) word_of(j) of its codes, and the
// (s, m) pair of its group j / 4.  Quotients are fp32 division's: q = d r with r about 1 / s, and one correction by the
// remainder, which is off by 2^-45 of q before its rounding.  d has 24 significant bits at most (values may differ by many
// binary orders) and s has 8, so d / s is no nearer than 2^-33 of itself to a number half way between two floats, and never
// one: that would have 25 bits, and s times it as many.  So too span / L.  held: the values that the codes stand for.
template <int BITS>
__device__ __forceinline__ void quant_row(const float (&x)[8], int j, uint32_t (&w)[BITS / 4], uint32_t &meta,
                                          float (&held)[8]) {
  constexpr float L = top_code<BITS>(), kInvL = 1.f / L;
  float mn = min3_nan(min3_nan(x[0], x[1], x[2]), min3_nan(x[3], x[4], x[5]), min3_nan(x[6], x[7], x[7]));
  float mx = max3_nan(max3_nan(x[0], x[1], x[2]), max3_nan(x[3], x[4], x[5]), max3_nan(x[6], x[7], x[7]));
  float a = lane_xor<1>(mn), b = lane_xor<1>(mx);
  mn = min3_nan(mn, a, a);
  mx = max3_nan(mx, b, b);
  a = lane_xor<2>(mn), b = lane_xor<2>(mx);
  mn = min3_nan(mn, a, a);
  mx = max3_nan(mx, b, b);
  const float span = mx - mn;
  const bool fine = span < INFINITY;             // neither NaN nor infinite
  float s = span * kInvL;
  s = (float)(__bf16)fmaf(fmaf(-s, L, span), kInvL, s);
  s = s < kLeastStep ? 0.f : s;
  const float inv = fine && s > 0.f ? __builtin_amdgcn_rcpf(s) : 0.f;
  uint32_t c[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float d = x[i] - mn;
    float q = d * inv;
    q = fmaf(fmaf(-q, s, d), inv, q);
    // (the step's rounding takes q to 15 (1 + 2^-8) at most, which rounds to 15, and to 256)
    if constexpr (BITS == 8) q = fminf(q, L);
    const float r = q + 0x1p23f;                 // rounded to a whole number, in its low bits
    c[i] = __builtin_bit_cast(uint32_t, r);
    held[i] = fine ? fmaf(r - 0x1p23f, s, mn) : NAN;
  }
  auto bytes = [](uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {   // their low bytes
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(a3, a2, 0x0c0c0400u), __builtin_amdgcn_perm(a1, a0, 0x0c0c0400u),
                                 0x05040100u);
  };
  if constexpr (BITS == 4) {
    w[0] = bytes(c[0], c[2], c[4], c[6]) | (bytes(c[1], c[3], c[5], c[7]) << 4);
  } else {
    w[0] = bytes(c[0], c[1], c[2], c[3]);
    w[1] = bytes(c[4], c[5], c[6], c[7]);
  }
#pragma unroll
  for (int k = 0; k < BITS / 4; ++k) w[k] = fine ? w[k] : 0u;
  transpose8<BITS>(w, j);
  meta = fine ? pack_bf16x2(s, mn) : 0x7FC07FC0u;
}

// Elements 8 j .. 8 j + 7 of a row whose word (pair) word_of(j) lane j holds; meta: its group j / 4's.
template <int BITS>
__device__ __forceinline__ void read_row(uint32_t (&w)[BITS / 4], uint32_t meta, int j, float (&x)[8]) {
  transpose8<BITS>(w, j);
  const float s = u32_as_f32(meta << 16), m = u32_as_f32(meta & 0xffff0000u);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t c = (w[i * BITS / 32] >> (BITS * i % 32)) & ((1u << BITS) - 1u);
    x[i] = fmaf((float)c, s, m);
  }
}

// ---- rows into the cache, and back ------------------------------------------------------------------
struct RowSource {
  const bf16_t *k, *v;
  int64_t k_rs, k_hs, v_rs, v_hs;
  int64_t rows;
  const int32_t *src_rows, *dst_rows;
};
// A wave takes one head of K or V of 16 rows (kRows = 4 at a time: 4 rows of 16 lanes, 16 bytes each, all four
// requested at once; their codes are stored as 256 contiguous bytes).  Blocks go by head first, so that the rows that
// are read at one time are whole.  Bound by the bytes: 98765 rows of 8 heads at 4 bits (K and V, 531 MB) 108 to 126 us,
// 4.9 to 4.2 TB/s, and read back 109 to 120, by the card; 4096 rows at 8 bits (26 MB) 7.3 and 6.6; one launch, 3 us, for a few.
constexpr int kRows = 4;
template <int BITS>
__global__ __launch_bounds__(256) void kv_quantize_kernel(RowSource a, QuantCache c, int64_t n, int heads) {
  const int x = blockIdx.x % (2 * heads), head = x >> 1, j = threadIdx.x & 15;
  const bool is_v = x & 1;
  const int64_t t0 = ((int64_t)(blockIdx.x / (2 * heads)) * 4 + (threadIdx.x >> 6)) * (4 * kRows) + ((threadIdx.x >> 4) & 3);
  int64_t dst[kRows];
  u32x4 raw[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {              // alike in the 16 lanes
    const int64_t t = t0 + 4 * r;
    const bool in = t < n;
    const int64_t src = in && a.src_rows ? a.src_rows[t] : t;
    dst[r] = in && a.dst_rows ? a.dst_rows[t] : t;
    const bool ok = in && src >= 0 && src < a.rows && dst[r] >= 0 && dst[r] < c.rows;
    raw[r] = gload16((is_v ? a.v + src * a.v_rs + head * a.v_hs : a.k + src * a.k_rs + head * a.k_hs) + 8 * j, ok);
    dst[r] = ok ? dst[r] : -1;
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    float x[8], held[8];
    unpack8(raw[r], x);
    uint32_t w[BITS / 4], meta;
    quant_row<BITS>(x, j, w, meta, held);
    if (dst[r] < 0) continue;
    const int64_t row = head * c.head_rows + dst[r];
    uint32_t *out = (is_v ? c.v : c.k) + row * row_words<BITS>() + word_of(j) * (BITS / 4);
    if constexpr (BITS == 4) *out = w[0];
    else *reinterpret_cast<u32x2 *>(out) = u32x2{w[0], w[1]};
    if ((j & 3) == 0) (is_v ? c.vm : c.km)[row * kGroups + (j >> 2)] = meta;
  }
}

struct RowTarget {
  bf16_t *k, *v;
  int64_t k_rs, k_hs, v_rs, v_hs;
  const int32_t *rows;
};
template <int BITS>
__global__ __launch_bounds__(256) void kv_dequantize_kernel(QuantCache c, RowTarget a, int64_t n, int heads) {
  const int x = blockIdx.x % (2 * heads), head = x >> 1, j = threadIdx.x & 15;
  const bool is_v = x & 1;
  const int64_t t0 = ((int64_t)(blockIdx.x / (2 * heads)) * 4 + (threadIdx.x >> 6)) * (4 * kRows) + ((threadIdx.x >> 4) & 3);
  uint32_t w[kRows][BITS / 4], meta[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t t = t0 + 4 * r, src = t < n && a.rows ? a.rows[t] : t;
    const bool ok = t < n && src >= 0 && src < c.rows;
    const int64_t row = head * c.head_rows + (ok ? src : 0);
#pragma unroll
    for (int i = 0; i < BITS / 4; ++i) w[r][i] = 0;
    meta[r] = 0;
    if (ok) {
      const uint32_t *in = (is_v ? c.v : c.k) + row * row_words<BITS>() + word_of(j) * (BITS / 4);
#pragma unroll
      for (int i = 0; i < BITS / 4; ++i) w[r][i] = in[i];
      meta[r] = (is_v ? c.vm : c.km)[row * kGroups + (j >> 2)];
    }
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t t = t0 + 4 * r;
    float x[8];
    read_row<BITS>(w[r], meta[r], j, x);
    if (t < n) st16((is_v ? a.v + t * a.v_rs + head * a.v_hs : a.k + t * a.k_rs + head * a.k_hs) + 8 * j, pack8(x));
  }
}

// ---- attention of a decode step ---------------------------------------------------------------------
// z_j = scale (q . k_j + bias_j), out = sum_j p_j v_j / sum_j p_j, p_j = exp(z_j - max z), with k_j = s c + m by groups
// of 32 (g): q . k_j = sum_g s_jg (q . c_j)_g + m_jg Q_g,  Q_g the sum of q over the group, and
// out = sum_g (p_j s_jg) c'_j + sum_j p_j m'_jg with c' = c - C, m' = m + C s, C the middle code (8 or 128): values of
// either sign have codes around the middle, so the sums over the keys are as small as the values', where those of p s c
// and p m would grow with every key and cancel at the end.  Bound by the bytes of the cache (80 or 144 per key and kv
// head, K and V each), so a workgroup takes one kv head of one sequence, up to four query heads of its group at once,
// and a stretch of keys: chunks of chunk_tiles tiles of 64 keys, its four waves a tile each in turn.  Nothing is staged
// through LDS: a wave's matrix instructions take the codes from the registers that the loads fill.
//   * S = Q C^T on v_mfma_f32_16x16x32_bf16, one instruction per 16 keys and group.  A: row 4 r + i holds query head i
//     (each head four times), so that every lane group gets all heads' sums and lane l keeps those of key l: the
//     softmax's work is one key per lane and head, and a lane applies its own key's s and m.  B: lane (n, G) holds the
//     words 4 G .. 4 G + 3 of key n.
//   * At 4 bits codes become bf16 by their bits: 0x4180 | c << 3 is 16 + c (two per and-or).  At 8 bits they are
//     converted.  S starts from -16 Q_g (C operand).  O gets -24 P or -128 P, P times a constant B, ahead of every 32 keys, so
//     that its sums are of c' and no more than the 32 keys' offset is rounded with them.  (At 128 + c, the 128 taken off at
//     the end, bf16 outputs over 131072 keys were 1e-3 from the fp32 form's, relative L2; so they are 4e-5 to 1.7e-4, most of
//     it the fp32 form's own distance from float64.)
//   * O += P C with P = p s per group, from LDS in A's layout, as three bf16 numbers, 24 bits together as fp32's:
//     rounded to one, the weights of keys that cancel left errors of 0.4 % of the output, to two of 2^-18 L steps.  The
//     others take rows of A that would repeat the heads, so no more instructions.  The middles' part is summed in fp32.
//     B: lane (n, G) holds word n of keys 4 j + G, whose nibble (byte) e is element 16 e + n: eight keys of one element,
//     and the element's group depends on e alone.
//   * The new key is not in the tiles: it is a part of its own beside the waves', from registers.
//   * The running maximum moves only when a logit passes it by 2^8.  Values near the largest float would
//     pass fp32's range in these sums: a wave whose sums come near it takes its tiles once more, with weights 2^-64 of these.
//     Waves merge in LDS, chunks through the workspace in the workgroup that arrives last.
// Measured, 16 / 8 heads: 4 bits, one sequence of 1, 300, 2320, 32769, 131072 keys 6.5, 10.4, 11.3, 23, 47 us (over a bf16
// cache by tg_decode_attention 2320 13, 32769 36); 64 x 4096 76 (4.4 TB/s; bf16 191), 8 x 80000 157 (5.2 TB/s); 8 bits
// 6.4, 11.4, 12.4, 28, 66; 116 (5.2), 257 (5.7).  (With weights of 16 bits, 128 + c and sums that may pass fp32's range
// 6.0, 9.7, 10.5, 22, 44; 71, 152 and 6.0, 10.6, 11.8, 27, 64; 113, 251.)  A short sequence is bound by its chain of
// latencies: launch, lengths and norms 4.9 us, the waves' merge 2, arrival 1.8, the chunks' merge 2.7, beside the tiles.
struct QuantAttnArgs {
  const bf16_t *qkv;
  int64_t qkv_rs;
  const float *rope;
  int h, hkv, group;
  const bf16_t *qw, *kw;
  float eps;
  const float *q_head_scale, *q_row_scale;
  QuantCache c;
  const int32_t *kv_start, *kv_used;
  int max_k;
  const float *bias;
  int64_t bias_bs, bias_hs;
  float scale_log2;
  bf16_t *out;
  int64_t out_rs;
  int nseq, sets;                // kv heads times head sets
  int slots, least;              // workgroups that are resident at once; fewest tiles per chunk
  uint32_t *counters;            // per unit: chunks arrived; zero between launches
  uint64_t *ml;                  // [workgroup][head]: running max (log2 units) and sum
  uint64_t *po;                  // [workgroup][head][64]: O, pairs of fp32
};

constexpr int kWaves = 4;
constexpr int kRounds = 2;
constexpr int kTile = 64;        // keys of a wave's step
// Tiles that a wave holds or has on their way, and workgroups per CU, by the registers.  16 / 8 heads (two at once), 4
// bits, two tiles and 2 workgroups / one and 3: 32769 keys 23.5 / 24.5 us, 64 x 4096 79 / 77, with bias 73.4 / 72.6, 64 x
// 300 15.3 / 14.9; 8 bits, where two tiles spill: 34 / 28, 134 / 118, 148 / 113, 22.5 / 18.1.  Four heads at once, one
// tile, 2 / 3 workgroups (spills): 4 x 8192 keys of 16 / 2 heads 21.5 / 26.8 at 4 bits, 22.5 / 36.6 at 8.
constexpr int depth(int bits, int hp) { return bits == 4 && hp <= 2 ? 2 : 1; }
__host__ __device__ constexpr int per_cu(int bits, int hp) { return depth(bits, hp) == 2 || hp == 4 ? 2 : 3; }
constexpr float kRescaleTau = 8.f;
// A wave whose sums pass kLargeSum takes its tiles once more with weights 2^-kLift of these: 2^8 p s (c + 24) over 2^24 keys
// stays below it up to steps of 2^60, and then up to the largest.
constexpr float kLargeSum = 0x1p100f, kLift = 64.f;
constexpr int kParts = 3;        // bf16 numbers of a weight

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

// bf16 pairs of eight codes from four words (4 bits) or pairs of words (8) of as many rows, nibbles (bytes) e of each:
// low half a, high half b of code pairs (a, b).
constexpr uint32_t kNibbles = 0x00780078u, kBf16 = 0x41804180u;   // (a nibble three bits up, 16)
template <int BITS> constexpr float mid_code() { return BITS == 4 ? 8.f : 128.f; }
template <int BITS> constexpr uint32_t kMinusOffset = BITS == 4 ? 0xC1C0C1C0u : 0xC300C300u;   // -24, -128: c' less the pairs

// (a's code e, b's code e) as a bf16 pair; at 4 bits from the halves' merger y = lo/hi16(a) | lo/hi16(b) << 16
__device__ __forceinline__ uint32_t merge_half(uint32_t a, uint32_t b, int hi) {
  return __builtin_amdgcn_perm(b, a, hi ? 0x07060302u : 0x05040100u);
}
// (mask and bias in registers: as literals they cost an instruction each)
__device__ __forceinline__ uint32_t nibble_pair(uint32_t y, int e, uint32_t nibbles, uint32_t bf16) {
  return (((e & 3) == 0 ? y << 3 : y >> (4 * (e & 3) - 3)) & nibbles) | bf16;
}
__device__ __forceinline__ uint32_t byte_pair(uint32_t a, uint32_t b, int byte) {
  const float fa = (float)((a >> (8 * byte)) & 255u), fb = (float)((b >> (8 * byte)) & 255u);
  return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, fb), __builtin_bit_cast(uint32_t, fa), 0x07060302u);
}

// The chunk that a workgroup takes: the q-th of all sequences' chunks in turn.  A sequence of n tiles is cut into
// ceil(n / T) chunks of even length, with one T for all, from their tiles, which only the device knows: the least that
// makes no more workgroups than are resident at once (a workgroup's fixed costs, 5 us, and a second round's uneven
// end cost more than idle places), or, where the sequences' remainders alone would fill most of these, two
// rounds.
// 16 / 8 heads, T for one round as far as it goes / two rounds / as here, us: 64 sequences of 512 .. 4099 at 8 bits 76 / 78
// / 76; 64 alike of 300 18.3 / 25.5 / 18.0; 8 of 16k .. 128k at 4 bits 162 / 178 / 161; 16 of 4k .. 30k 82 / 91 / 82; 64
// alike of 4096 69 / 78 / 69; 300 of 300 .. 3000 168 / 154 / 154; 120 of 50 .. 20000 323 / 298 / 297.
struct Chunk {
  int seq, chunk, chunks, tiles, sk;
  int64_t start;
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
// ceil(n / T), n and T below 2^22: the quotient's float is off by less than 1 / T
__device__ __forceinline__ int ceil_div(int n, float inv) { return (int)(((float)n - 0.5f) * inv) + 1; }
__device__ __forceinline__ Chunk find_chunk(const QuantAttnArgs &a, int q, int lane) {
  int sk = 0, start = 0, tiles = 0;
  auto read = [&](int s) {                       // of sequence s, this lane's
    start = s < a.nseq ? a.kv_start[s] : 0;
    sk = s < a.nseq ? max(0, min(a.kv_used[s], a.max_k)) : 0;
    if (start < 0 || (int64_t)start + sk > a.c.rows) sk = 0;
    tiles = (max(0, sk - 1) + kTile - 1) / kTile;
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
  int T = max(a.least, (int)(work / target) + 1);
  // (where not even an even cut of every sequence would fill one round, nothing is counted)
  for (int i = 0; i < 3 && work / (float)T + (float)a.nseq * (float)a.sets > slots; ++i) {
    const float over = (float)count(T, false) * (float)a.sets - slots;
    if (over <= 0.f) break;
    if (over > 0.75f * slots) {
      T = max(a.least, (int)(work / (kRounds * slots)) + 1);
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

template <int BITS, int HP, bool HAS_BIAS>
__global__ __launch_bounds__(64 * kWaves, per_cu(BITS, HP)) void decode_attn_quant_kernel(QuantAttnArgs a) {
  constexpr int kRow = 16 * BITS;                 // bytes of a row's codes
  constexpr int KW = BITS;                        // words of a row that one lane takes for S: 16 B or 32 B
  constexpr int VW = BITS / 4;                    // and for O
  constexpr int kDepth = depth(BITS, HP);         // tiles in registers
  const int tid = threadIdx.x, wave = wave_id(), lane = tid & 63, n16 = lane & 15, G = lane >> 4;
  const int set = blockIdx.x % a.sets, kh = set % a.hkv, hg = set / a.hkv;
  const int h0 = kh * a.group + hg * HP, nh = min(HP, a.group - hg * HP);   // heads h0 .. h0 + nh - 1

  __shared__ __attribute__((aligned(16))) bf16_t qs[HP][kHeadDim];
  __shared__ __attribute__((aligned(16))) float new_x[2][kHeadDim];   // the new key and value as they are held
  __shared__ __attribute__((aligned(16))) bf16_t ps[kWaves][kGroups][kParts * HP][kTile];
  __shared__ __attribute__((aligned(16))) float part_o[kWaves + 1][HP][kHeadDim], part_ml[kWaves + 1][HP][2];

  const Chunk ck = find_chunk(a, blockIdx.x / a.sets, lane);
  if (ck.seq < 0) return;                        // workgroup-uniform: past the last chunk
  const int b = ck.seq, nk = max(0, ck.sk - 1);  // keys in the cache; the new one is apart
  const int64_t start = ck.start;
  const int n_tiles = ck.tiles, n_parts = ck.chunks, chunk = ck.chunk;
  const int t_lo = (int)((int64_t)n_tiles * chunk / n_parts), t_hi = (int)((int64_t)n_tiles * (chunk + 1) / n_parts);
  const bool has_new = chunk == n_parts - 1 && ck.sk > 0;

  // ---- loads of a tile: rows past nk read as zero (codes, s and m) ----
  const int64_t row0 = kh * a.c.head_rows + start;
  const brsrc_t krs = make_rsrc(a.c.k + row0 * row_words<BITS>(), (uint32_t)nk * kRow);
  const brsrc_t vrs = make_rsrc(a.c.v + row0 * row_words<BITS>(), (uint32_t)nk * kRow);
  const brsrc_t kmrs = make_rsrc(a.c.km + row0 * kGroups, (uint32_t)nk * 16);
  const brsrc_t vmrs = make_rsrc(a.c.vm + row0 * kGroups, (uint32_t)nk * 16);
  struct Tile {
    uint32_t kx[4][KW], vx[2][8][VW];
    u32x4 kmeta, vmeta;
    float bias[HP];
  } tiles[kDepth];
  // (past the chunk's end a tile past the rows: zeros, and no access)
  auto load_k = [&](Tile &l, int tile) {
    const int t = tile < t_hi ? tile : n_tiles;
    const uint32_t at = (uint32_t)t * (kTile * kRow) + n16 * kRow + G * (kRow / 4);
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
#pragma unroll
      for (int i = 0; i < KW / 4; ++i) {
        const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(krs, at + kb * 16 * kRow + 16 * i, 0, 0);
#pragma unroll
        for (int e = 0; e < 4; ++e) l.kx[kb][4 * i + e] = v[e];
      }
    const uint32_t key = (uint32_t)t * kTile + lane;
    l.kmeta = __builtin_amdgcn_raw_buffer_load_b128(kmrs, key * 16, 0, 0);
    if constexpr (HAS_BIAS) {
#pragma unroll
      for (int i = 0; i < HP; ++i) {
        const float *p = a.bias + (int64_t)b * a.bias_bs + (int64_t)(h0 + min(i, nh - 1)) * a.bias_hs;
        l.bias[i] = u32_as_f32(__builtin_amdgcn_raw_buffer_load_b32(make_rsrc(p, (uint32_t)nk * 4), key * 4, 0, 0));
      }
    }
  };
  auto load_v = [&](Tile &l, int tile) {
    const int t = tile < t_hi ? tile : n_tiles;
    const uint32_t at = (uint32_t)t * (kTile * kRow) + G * kRow + n16 * (4 * VW);
#pragma unroll
    for (int st = 0; st < 2; ++st)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t p = at + (32 * st + 4 * j) * kRow;
        if constexpr (BITS == 4) {
          l.vx[st][j][0] = __builtin_amdgcn_raw_buffer_load_b32(vrs, p, 0, 0);
        } else {
          const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(vrs, p, 0, 0);
          l.vx[st][j][0] = v[0];
          l.vx[st][j][1] = v[1];
        }
      }
    l.vmeta = __builtin_amdgcn_raw_buffer_load_b128(vmrs, ((uint32_t)t * kTile + lane) * 16, 0, 0);
  };
  // ---- the rows to form: 16 lanes a row; wave 0 the query heads, wave 1 the new key (lanes 0 .. 15) and value.  Their
  // loads come before the tiles': loads complete in issue order ----
  const bool forms = wave == 0 ? G < HP : wave == 1 && has_new && G < 2;
  const int head = wave == 0 ? h0 + min(G, nh - 1) : (G == 0 ? a.h : a.h + a.hkv) + kh;
  u32x4 raw = {0u, 0u, 0u, 0u}, norm_w = raw;
  f32x4 turn[4] = {};
  float q_scale = 1.f;
  if (forms) {
    raw = ld16(a.qkv + b * a.qkv_rs + (int64_t)head * kHeadDim + 8 * n16);
    norm_w = ld16((wave == 0 ? a.qw : a.kw) + 8 * n16);
    const f32x4 *rp = reinterpret_cast<const f32x4 *>(a.rope + b * kHeadDim + 16 * (n16 & 7));
#pragma unroll
    for (int i = 0; i < 4; ++i) turn[i] = rp[i];
    if (wave == 0)
      q_scale = (float)(__bf16)((a.q_head_scale ? a.q_head_scale[head] : 1.f) * (a.q_row_scale ? a.q_row_scale[b] : 1.f));
  }
  float new_bias = 0.f;
  if (HAS_BIAS && has_new && wave == kWaves - 1 && G < HP)
    new_bias = a.bias[(int64_t)b * a.bias_bs + (int64_t)(h0 + min(G, nh - 1)) * a.bias_hs + nk];
  int t = 0;
  auto first_loads = [&] {
    t = t_lo + wave;
    if (t >= t_hi) return;
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      load_k(tiles[d], t + d * kWaves);
      // (the loop's loads and these in one order: at its head the compiler waits for whatever either order has last)
      __builtin_amdgcn_sched_barrier(0);
      load_v(tiles[d], t + d * kWaves);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  first_loads();
  if (forms) {
    float x[8], wf[8], y[8], cs[8][2];
    unpack8(raw, x);
    unpack8(norm_w, wf);
#pragma unroll
    for (int i = 0; i < 16; ++i) cs[i >> 1][i & 1] = turn[i >> 2][i & 3];
    norm_rope8(x, wf, a.eps, cs, n16, q_scale, y);
    const u32x4 turned = pack8(y);
    if (wave == 0) {
      st16(&qs[G][8 * n16], turned);
    } else {
      unpack8(G == 0 ? turned : raw, x);
      uint32_t w[BITS / 4], meta;
      quant_row<BITS>(x, n16, w, meta, y);
#pragma unroll
      for (int i = 0; i < 8; ++i) new_x[G][8 * n16 + i] = y[i];
      if (hg == 0) {
        const int64_t row = row0 + nk;
        uint32_t *codes = G == 0 ? a.c.k : a.c.v, *metas = G == 0 ? a.c.km : a.c.vm;
#pragma unroll
        for (int i = 0; i < BITS / 4; ++i) codes[row * row_words<BITS>() + word_of(n16) * (BITS / 4) + i] = w[i];
        if ((n16 & 3) == 0) metas[row * kGroups + (n16 >> 2)] = meta;
      }
    }
  }
  __syncthreads();
  // ---- the new key: a part of its own, 16 lanes a head ----
  if (has_new && wave == kWaves - 1 && G < HP) {
    float q[8], z = 0.f;
    unpack8(*reinterpret_cast<const u32x4 *>(&qs[G][8 * n16]), q);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      z = fmaf(q[i], new_x[0][8 * n16 + i], z);
      part_o[kWaves][G][8 * n16 + i] = new_x[1][8 * n16 + i];
    }
    z += dpp<0xB1>(z);
    z += dpp<0x4E>(z);
    z += dpp<0x141>(z);
    z += dpp<0x140>(z);
    const bool hidden = new_bias == -INFINITY;
    if (n16 == 0) {
      part_ml[kWaves][G][0] = hidden ? -INFINITY : (z + new_bias) * a.scale_log2;
      part_ml[kWaves][G][1] = hidden ? 0.f : 1.f;
    }
  }

  // ---- Q in A's layout, and its sums by group ----
  bf16x8 qf[kGroups];
  float qsum[kGroups][HP];
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    const bf16_t *p = &qs[n16 & (HP - 1)][32 * g + 4 * G];
    const u32x2 lo = *reinterpret_cast<const u32x2 *>(p), hi = *reinterpret_cast<const u32x2 *>(p + 16);
    const u32x4 q = {lo[0], lo[1], hi[0], hi[1]};
    qf[g] = __builtin_bit_cast(bf16x8, q);
    float f[8], s = 0.f;
    unpack8(q, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) s += f[i];
    s = quad_sum(s);
#pragma unroll
    for (int i = 0; i < HP; ++i) qsum[g][i] = u32_as_f32(__builtin_amdgcn_readlane(__builtin_bit_cast(uint32_t, s), i));
  }

  f32x4 oacc[8];
  float mrun[HP], lsum[HP], rest[HP][kGroups];   // rest: sums of p m', by lane
  float lift = 0.f;                              // the running maximum is so far above the logits' (alike in the wave)
  // row of the weights that this lane holds in A: heads' first parts, second, third and as many rows of these again, which
  // no sum is taken of
  const int a_row = (n16 & (4 * HP - 1)) < kParts * HP ? n16 & (4 * HP - 1) : (n16 & (4 * HP - 1)) - HP;
  // position of this lane's key in A's order of keys: lane (m, G) takes keys 4 j + G, j = 0 .. 7, of 32
  bf16_t *const pw = &ps[wave][0][0][32 * (lane >> 5) + 8 * (lane & 3) + ((lane & 31) >> 2)];

  uint32_t nibbles = kNibbles, bf16 = kBf16;
  asm("" : "+v"(nibbles), "+v"(bf16));
  constexpr uint32_t kOff = kMinusOffset<BITS>;
  const bf16x8 minus_offset = __builtin_bit_cast(bf16x8, u32x4{kOff, kOff, kOff, kOff});
  auto step = [&](Tile &l) {
    // ---- logits of key `lane` ----
    float z[HP];
#pragma unroll
    for (int i = 0; i < HP; ++i) z[i] = HAS_BIAS ? l.bias[i] : 0.f;
    uint32_t ky[4][4];                           // 4 bits: merged halves (words 0 1 lo, 0 1 hi, 2 3 lo, 2 3 hi)
    if constexpr (BITS == 4) {
#pragma unroll
      for (int kb = 0; kb < 4; ++kb)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          ky[kb][2 * p] = merge_half(l.kx[kb][2 * p], l.kx[kb][2 * p + 1], 0);
          ky[kb][2 * p + 1] = merge_half(l.kx[kb][2 * p], l.kx[kb][2 * p + 1], 1);
        }
    }
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      f32x4 init = {0.f, 0.f, 0.f, 0.f};
      if constexpr (BITS == 4) {
#pragma unroll
        for (int i = 0; i < HP; ++i) init[i] = -16.f * qsum[g][i];
      }
      f32x4 s[4];
#pragma unroll
      for (int kb = 0; kb < 4; ++kb) {
        u32x4 c;
#pragma unroll
        for (int w = 0; w < 4; ++w) {            // codes e = 2 g (w < 2) and 2 g + 1 of words 0 1 or 2 3
          const int e = 2 * g + (w >> 1), p = w & 1;
          if constexpr (BITS == 4)
            c[w] = nibble_pair(ky[kb][2 * p + (e >> 2)], e, nibbles, bf16);
          else
            c[w] = byte_pair(l.kx[kb][4 * p + (e >> 2)], l.kx[kb][4 * p + 2 + (e >> 2)], e & 3);
        }
        s[kb] = mfma16(qf[g], __builtin_bit_cast(bf16x8, c), init);
      }
      const float step = u32_as_f32(l.kmeta[g] << 16), least = u32_as_f32(l.kmeta[g] & 0xffff0000u);
#pragma unroll
      for (int i = 0; i < HP; ++i) {
        const float s01 = G & 1 ? s[1][i] : s[0][i], s23 = G & 1 ? s[3][i] : s[2][i];
        z[i] = fmaf(G & 2 ? s23 : s01, step, fmaf(qsum[g][i], least, z[i]));
      }
    }
    bool up = false;
#pragma unroll
    for (int i = 0; i < HP; ++i) {
      z[i] *= a.scale_log2;
      asm("" : "+v"(z[i]));   // rounded: contracted into z - m below, a bias near the lowest float leaves the rounding's rest
      if (t * kTile + lane >= nk) z[i] = -INFINITY;
      if constexpr (HAS_BIAS) z[i] = l.bias[i] == -INFINITY ? -INFINITY : z[i];   // hidden, whatever the row holds
      up |= z[i] > mrun[i] + (kRescaleTau - lift);
    }
    load_k(l, t + kDepth * kWaves);
    __builtin_amdgcn_sched_barrier(0);
    if (__builtin_amdgcn_ballot_w64(up)) {
#pragma unroll
      for (int i = 0; i < HP; ++i) {
        const float m = fmaxf(mrun[i], wave_max(z[i]) + lift), f = mrun[i] == -INFINITY ? 0.f : fast_exp2(mrun[i] - m);
        mrun[i] = m;
        lsum[i] *= f;
#pragma unroll
        for (int g = 0; g < kGroups; ++g) rest[i][g] *= f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
#pragma unroll
          for (int r = i; r < 4; r += HP) oacc[e][r] *= f;   // the head's parts
        }
      }
    }
#pragma unroll
    for (int i = 0; i < HP; ++i) {
      const float p = fast_exp2(z[i] - (mrun[i] == -INFINITY ? 0.f : mrun[i]));
      lsum[i] += p;
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        const float step = u32_as_f32(l.vmeta[g] << 16), mid = fmaf(mid_code<BITS>(), step, u32_as_f32(l.vmeta[g] & 0xffff0000u));
        const float w = mul_zero(p, step);       // (a weight of 0 is 0, whatever the row holds)
        const __bf16 w0 = (__bf16)w, w1 = (__bf16)(w - (float)w0), w2 = (__bf16)(w - (float)w0 - (float)w1);
        pw[(kParts * HP * g + i) * kTile] = __builtin_bit_cast(uint16_t, w0);
        pw[(kParts * HP * g + HP + i) * kTile] = __builtin_bit_cast(uint16_t, w1);
        pw[(kParts * HP * g + 2 * HP + i) * kTile] = __builtin_bit_cast(uint16_t, w2);
        rest[i][g] += mul_zero(p, mid);
      }
    }
    // ---- O += P C ----
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      uint32_t vy[4][2];
      if constexpr (BITS == 4) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          vy[w][0] = merge_half(l.vx[st][2 * w][0], l.vx[st][2 * w + 1][0], 0);
          vy[w][1] = merge_half(l.vx[st][2 * w][0], l.vx[st][2 * w + 1][0], 1);
        }
      }
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        const bf16x8 pf = *reinterpret_cast<const bf16x8 *>(&ps[wave][g][a_row][32 * st + 8 * G]);
#pragma unroll
        for (int e = 2 * g; e < 2 * g + 2; ++e) oacc[e] = mfma16(pf, minus_offset, oacc[e]);
#pragma unroll
        for (int e = 2 * g; e < 2 * g + 2; ++e) {
          u32x4 c;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            if constexpr (BITS == 4)
              c[w] = nibble_pair(vy[w][e >> 2], e, nibbles, bf16);
            else
              c[w] = byte_pair(l.vx[st][2 * w][e >> 2], l.vx[st][2 * w + 1][e >> 2], e & 3);
          }
          oacc[e] = mfma16(pf, __builtin_bit_cast(bf16x8, c), oacc[e]);
        }
      }
    }
    load_v(l, t + kDepth * kWaves);
    __builtin_amdgcn_sched_barrier(0);
    t += kWaves;
  };
  for (;;) {
#pragma unroll
    for (int e = 0; e < 8; ++e) oacc[e] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < HP; ++i) {
      mrun[i] = -INFINITY;
      lsum[i] = 0.f;
#pragma unroll
      for (int g = 0; g < kGroups; ++g) rest[i][g] = 0.f;
    }
    if constexpr (kDepth == 2) {
      // (an exit between the two steps would leave the compiler a path on which the second tile's loads are the older)
      while (t + kWaves < t_hi) {
        step(tiles[0]);
        step(tiles[1]);
      }
      if (t < t_hi) step(tiles[0]);
    } else {
      while (t < t_hi) step(tiles[0]);
    }

    // ---- the waves' results meet in LDS ----
    bool fine = true;
#pragma unroll
    for (int i = 0; i < HP; ++i) {
      const float l = wave_add(lsum[i]);
      if (lane == 0) {
        part_ml[wave][i][0] = mrun[i];
        part_ml[wave][i][1] = l;
      }
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        const float r = wave_add(rest[i][g]);
        auto sum_parts = [&](const f32x4 &o) {     // (lane group G holds A's rows 4 G .. 4 G + 3)
          if constexpr (HP == 1) return o[0] + (o[1] + o[2]);
          else if constexpr (HP == 2) return add_row_pair(G & 1 ? o[i] : o[i] + o[i + 2]);
          else return add_rows(G < kParts ? o[i] : 0.f);
        };
        const float o0 = sum_parts(oacc[2 * g]), o1 = sum_parts(oacc[2 * g + 1]);
        if (G == g) {                              // lane group g writes group g's elements
          part_o[wave][i][32 * g + n16] = o0 + r;
          part_o[wave][i][32 * g + 16 + n16] = o1 + r;
          fine &= fabsf(o0 + r) < kLargeSum && fabsf(o1 + r) < kLargeSum;
        }
      }
    }
    // (a NaN that a key holds comes again)
    if (lift != 0.f || !__builtin_amdgcn_ballot_w64(!fine)) break;
    lift = kLift;
    first_loads();
  }
  __syncthreads();
  constexpr int kOuts = HP * kHeadDim / 2;       // pairs of output elements
  bf16_t *const orow = a.out + b * a.out_rs + (int64_t)h0 * kHeadDim;
  auto put = [&](int item, float o0, float o1, float l) {   // a row that saw no key: 0
    const float f = l == 0.f ? 0.f : 1.f / l;
    if (item / 64 < nh)
      *reinterpret_cast<uint32_t *>(orow + 2 * item) = l == 0.f ? 0u : pack_bf16x2(o0 * f, o1 * f);
  };
  for (int item = tid; item < kOuts; item += 64 * kWaves) {
    const int i = item / 64, d = 2 * (item % 64);
    float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves + 1; ++w)
      if (w < kWaves || has_new) m = fmaxf(m, part_ml[w][i][0]);
#pragma unroll
    for (int w = 0; w < kWaves + 1; ++w) {
      if (w == kWaves && !has_new) break;
      const float mw = part_ml[w][i][0], f = mw == -INFINITY ? (part_ml[w][i][1] == 0.f ? 0.f : 1.f) : fast_exp2(mw - m);
      l += f * part_ml[w][i][1];
      o0 += mul_zero(f, part_o[w][i][d]);
      o1 += mul_zero(f, part_o[w][i][d + 1]);
    }
    if (n_parts == 1) {
      put(item, o0, o1, l);
    } else {
      // (agent-scope accesses write through and read past the XCD's L2, where a release would write all of it back)
      const int64_t at = (int64_t)blockIdx.x * HP + i;
      const float2 o = {o0, o1}, mlv = {m, l};
      st_agent(a.po + at * 64 + item % 64, __builtin_bit_cast(uint64_t, o));
      if (d == 0) st_agent(a.ml + at, __builtin_bit_cast(uint64_t, mlv));
    }
  }
  if (n_parts == 1) return;
  __shared__ int last_s;
  uint32_t *const counter = a.counters + (int64_t)b * a.sets + set;
  wait_all_mem();                                // this wave's stores are done
  __syncthreads();
  if (tid == 0)
    last_s = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)n_parts - 1u;
  __syncthreads();
  if (!last_s) return;
  if (tid == 0) st_agent(counter, 0u);
  // ---- the last workgroup of the unit merges its chunks: four output elements per thread, every kSets-th chunk,
  // as many loads in flight as chunks; then the sets in turn ----
  constexpr int kItems = HP * 32, kSets = 64 * kWaves / kItems, kAhead = 8;
  const int item = tid % kItems, cs = tid / kItems, i = item / 32;
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  auto fold = [&](float mc, float lc, const float (&oc)[4]) {
    const float mn = fmaxf(m, mc), f0 = m == -INFINITY ? 0.f : fast_exp2(m - mn), f1 = mc == -INFINITY ? 1.f : fast_exp2(mc - mn);
    l = l * f0 + lc * f1;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = o[e] * f0 + oc[e] * f1;
    m = mn;
  };
  for (int c0 = cs; c0 < n_parts; c0 += kAhead * kSets) {
    uint64_t ml[kAhead], ow[kAhead][2];
#pragma unroll
    for (int r = 0; r < kAhead; ++r) {           // (every load is made, past the end the last's)
      const int64_t at = ((int64_t)blockIdx.x + (min(c0 + r * kSets, n_parts - 1) - chunk) * a.sets) * HP + i;
      ml[r] = ld_agent(a.ml + at);
      ow[r][0] = ld_agent(a.po + at * 64 + 2 * (item % 32));
      ow[r][1] = ld_agent(a.po + at * 64 + 2 * (item % 32) + 1);
    }
#pragma unroll
    for (int r = 0; r < kAhead; ++r) {
      const float2 mc = __builtin_bit_cast(float2, ml[r]), a0 = __builtin_bit_cast(float2, ow[r][0]), a1 = __builtin_bit_cast(float2, ow[r][1]);
      const float oc[4] = {a0.x, a0.y, a1.x, a1.y};
      if (c0 + r * kSets < n_parts && mc.y != 0.f) fold(mc.x, mc.y, oc);   // (0: saw no key)
    }
  }
  __shared__ float set_s[kSets > 1 ? kSets - 1 : 1][6][kItems];
  if (cs > 0) {
    set_s[cs - 1][0][item] = m;
    set_s[cs - 1][1][item] = l;
#pragma unroll
    for (int e = 0; e < 4; ++e) set_s[cs - 1][2 + e][item] = o[e];
  }
  __syncthreads();
  if (cs > 0) return;
#pragma unroll
  for (int s = 0; s < kSets - 1; ++s) {
    const float oc[4] = {set_s[s][2][item], set_s[s][3][item], set_s[s][4][item], set_s[s][5][item]};
    if (set_s[s][1][item] != 0.f) fold(set_s[s][0][item], set_s[s][1][item], oc);
  }
  put(2 * item, o[0], o[1], l);
  put(2 * item + 1, o[2], o[3], l);
}

// Workgroups of a launch: units of (sequence, kv head, head set), cut into chunks on the device.
struct QuantPlan {
  int hp, sets, slots, least;
  int64_t grid, bytes;
};
// The counters' region is the same for every launch, so that no launch writes partial results where another counts;
// launches of more units cut none.
constexpr int64_t kCounters = 1 << 14;
QuantPlan plan_quant(int bits, int64_t num_seqs, int num_heads, int num_heads_k, int max_k) {
  QuantPlan p;
  const int group = num_heads / num_heads_k;
  p.hp = group >= 3 ? 4 : group;
  p.sets = num_heads_k * ((group + p.hp - 1) / p.hp);
  p.slots = per_cu(bits, p.hp) * device_cus();
  const int64_t units = num_seqs * p.sets, tiles = std::max(1, (max_k + kTile - 1) / kTile);
  // (a wave's first tile: 2320 keys 10.5 us in chunks of four tiles at least, 13.1 of eight)
  p.least = units <= kCounters ? kWaves : 1 << 22;
  p.grid = std::min<int64_t>(units * ((tiles + p.least - 1) / p.least), units + kRounds * p.slots);
  // counters, (max, sum), O
  p.bytes = p.grid == units ? 0 : kCounters * 4 + (p.grid * p.hp * 8 + 255) / 256 * 256 + p.grid * p.hp * kHeadDim * 4;
  return p;
}

int check_cache(const char *what, int32_t num_heads_k, int32_t head_dim, int32_t bits, const void *k_codes,
                const void *k_meta, const void *v_codes, const void *v_meta, int64_t cache_rows, int64_t head_rows,
                QuantCache *c) {
  TG_CHECK(head_dim == kHeadDim, "%s: head_dim must be 128", what);
  TG_CHECK(bits == 4 || bits == 8, "%s: 4 or 8 bits (got %d)", what, bits);
  TG_CHECK(num_heads_k > 0 && num_heads_k <= 256, "%s: KV heads must be in 1..256", what);
  TG_CHECK(cache_rows >= 0 && head_rows >= cache_rows, "%s: head_rows must be at least cache_rows", what);
  TG_CHECK(cache_rows < (1ll << 31) && head_rows < (1ll << 40), "%s: too many cache rows", what);
  TG_CHECK(k_codes && k_meta && v_codes && v_meta, "%s: null cache pointer", what);
  TG_CHECK(aligned16(k_codes) && aligned16(k_meta) && aligned16(v_codes) && aligned16(v_meta),
           "%s: cache pointers must be 16-byte aligned", what);
  c->k = static_cast<uint32_t *>(const_cast<void *>(k_codes));
  c->v = static_cast<uint32_t *>(const_cast<void *>(v_codes));
  c->km = static_cast<uint32_t *>(const_cast<void *>(k_meta));
  c->vm = static_cast<uint32_t *>(const_cast<void *>(v_meta));
  c->rows = cache_rows;
  c->head_rows = head_rows;
  return 0;
}
// workgroups of the row kernels: 16 rows per wave
int64_t row_blocks(int64_t n_rows, int heads) { return (n_rows + 16 * kRows - 1) / (16 * kRows) * 2 * heads; }
int check_rows(const char *what, const void *k, int64_t k_rs, int64_t k_hs, const void *v, int64_t v_rs, int64_t v_hs,
               int64_t n_rows, int heads) {
  TG_CHECK(k && v, "%s: null row pointer", what);
  TG_CHECK(n_rows >= 0 && n_rows < (1ll << 31) && row_blocks(n_rows, heads) < (1ll << 31), "%s: bad row count", what);
  TG_CHECK(k_rs >= 0 && v_rs >= 0 && k_hs >= 0 && v_hs >= 0 && k_rs % 8 == 0 && v_rs % 8 == 0 && k_hs % 8 == 0 && v_hs % 8 == 0,
           "%s: strides must be multiples of 8 elements", what);
  TG_CHECK(aligned16(k) && aligned16(v), "%s: rows must be 16-byte aligned", what);
  return 0;
}

}  // namespace
}  // namespace tg

using namespace tg;

extern "C" int tg_kv_quantize(const void *k, int64_t k_row_stride, int64_t k_head_stride, const void *v,
                              int64_t v_row_stride, int64_t v_head_stride, int64_t source_rows,
                              const int32_t *src_rows, const int32_t *dst_rows, int64_t n_rows, int32_t num_heads_k,
                              int32_t head_dim, int32_t bits, void *k_codes, void *k_meta, void *v_codes, void *v_meta,
                              int64_t cache_rows, int64_t head_rows, hipStream_t stream) {
  clear_error();
  QuantCache c;
  if (int e = check_cache("kv_quantize", num_heads_k, head_dim, bits, k_codes, k_meta, v_codes, v_meta, cache_rows, head_rows, &c))
    return e;
  if (int e = check_rows("kv_quantize", k, k_row_stride, k_head_stride, v, v_row_stride, v_head_stride, n_rows, num_heads_k)) return e;
  TG_CHECK(source_rows >= 0 && (src_rows || n_rows <= source_rows), "kv_quantize: more rows than the source holds");
  TG_CHECK(dst_rows || n_rows <= cache_rows, "kv_quantize: more rows than the cache holds");
  if (n_rows == 0) return 0;
  const RowSource a{static_cast<const bf16_t *>(k), static_cast<const bf16_t *>(v), k_row_stride, k_head_stride,
                    v_row_stride, v_head_stride, source_rows, src_rows, dst_rows};
  const dim3 grid((unsigned)row_blocks(n_rows, num_heads_k)), block(256);
  if (bits == 4) hipLaunchKernelGGL(kv_quantize_kernel<4>, grid, block, 0, stream, a, c, n_rows, num_heads_k);
  else hipLaunchKernelGGL(kv_quantize_kernel<8>, grid, block, 0, stream, a, c, n_rows, num_heads_k);
  TG_HIP_CHECK(hipGetLastError());
  return 0;
}

extern "C" int tg_kv_dequantize(const void *k_codes, const void *k_meta, const void *v_codes, const void *v_meta,
                                int64_t cache_rows, int64_t head_rows, int32_t num_heads_k, int32_t head_dim,
                                int32_t bits, const int32_t *rows, int64_t n_rows, void *k_out, int64_t k_row_stride,
                                int64_t k_head_stride, void *v_out, int64_t v_row_stride, int64_t v_head_stride,
                                hipStream_t stream) {
  clear_error();
  QuantCache c;
  if (int e = check_cache("kv_dequantize", num_heads_k, head_dim, bits, k_codes, k_meta, v_codes, v_meta, cache_rows, head_rows, &c))
    return e;
  if (int e = check_rows("kv_dequantize", k_out, k_row_stride, k_head_stride, v_out, v_row_stride, v_head_stride, n_rows, num_heads_k))
    return e;
  TG_CHECK(rows || n_rows <= cache_rows, "kv_dequantize: more rows than the cache holds");
  TG_CHECK(k_head_stride >= kHeadDim && v_head_stride >= kHeadDim, "kv_dequantize: head strides of outputs must be at least 128");
  // no row of a head within 128 elements of another: of the same head, or of the one h heads on, whose nearest rows are the
  // two around h hs / rs
  auto apart = [&](int64_t rs, int64_t hs) {
    if (n_rows <= 1) return true;
    if (rs < kHeadDim) return false;
    for (int64_t h = 1; h < num_heads_k; ++h) {
      const int64_t d = std::min(h * hs / rs, n_rows - 1);
      if (h * hs - d * rs < kHeadDim || (d + 1 < n_rows && (d + 1) * rs - h * hs < kHeadDim)) return false;
    }
    return true;
  };
  TG_CHECK(apart(k_row_stride, k_head_stride) && apart(v_row_stride, v_head_stride), "kv_dequantize: rows of the outputs overlap");
  if (n_rows == 0) return 0;
  const RowTarget a{static_cast<bf16_t *>(k_out), static_cast<bf16_t *>(v_out), k_row_stride, k_head_stride, v_row_stride,
                    v_head_stride, rows};
  const dim3 grid((unsigned)row_blocks(n_rows, num_heads_k)), block(256);
  if (bits == 4) hipLaunchKernelGGL(kv_dequantize_kernel<4>, grid, block, 0, stream, c, a, n_rows, num_heads_k);
  else hipLaunchKernelGGL(kv_dequantize_kernel<8>, grid, block, 0, stream, c, a, n_rows, num_heads_k);
  TG_HIP_CHECK(hipGetLastError());
  return 0;
}

// (for the bits with more workgroups; enough for fewer sequences and keys too)
extern "C" int64_t tg_decode_attention_quant_workspace_size(int32_t num_seqs, int32_t num_heads, int32_t num_heads_k,
                                                            int32_t max_seqlen_k) {
  if (num_seqs <= 0 || num_heads <= 0 || num_heads_k <= 0 || num_heads % num_heads_k != 0 || max_seqlen_k <= 0) return 0;
  const int64_t fits = kCounters / plan_quant(8, 1, num_heads, num_heads_k, 1).sets;   // sequences that may be cut
  return plan_quant(8, std::min<int64_t>(num_seqs, fits), num_heads, num_heads_k, max_seqlen_k).bytes;
}

extern "C" int tg_decode_attention_quant(const void *qkv, int64_t qkv_row_stride, const float *rope, int32_t num_seqs,
                                         int32_t num_heads, int32_t num_heads_k, int32_t head_dim, int32_t bits,
                                         const void *q_norm_weight, const void *k_norm_weight, float eps,
                                         const float *q_head_scale, const float *q_row_scale, void *k_codes,
                                         void *k_meta, void *v_codes, void *v_meta, int64_t cache_rows,
                                         int64_t head_rows, const int32_t *kv_start, const int32_t *kv_used,
                                         int32_t max_seqlen_k, const float *bias_raw, int64_t bias_seq_stride,
                                         int64_t bias_head_stride, float softmax_scale, void *out,
                                         int64_t out_row_stride, void *workspace, int64_t workspace_bytes,
                                         hipStream_t stream) {
  clear_error();
  const char *what = "decode_attention_quant";
  QuantAttnArgs a{};
  if (int e = check_cache(what, num_heads_k, head_dim, bits, k_codes, k_meta, v_codes, v_meta, cache_rows, head_rows, &a.c))
    return e;
  TG_CHECK(qkv && rope && q_norm_weight && k_norm_weight && kv_start && kv_used && out, "%s: null pointer", what);
  TG_CHECK(num_heads > 0 && num_heads <= 256 && num_heads % num_heads_k == 0,
           "%s: heads must be in 1..256 and a multiple of the KV heads", what);
  TG_CHECK(num_seqs >= 0 && (int64_t)num_seqs * num_heads < (1 << 24) && max_seqlen_k >= 0,
           "%s: bad sequence count or length", what);
  TG_CHECK(qkv_row_stride % 8 == 0 && out_row_stride % 8 == 0 &&
               qkv_row_stride >= (int64_t)(num_heads + 2 * num_heads_k) * kHeadDim &&
               out_row_stride >= (int64_t)num_heads * kHeadDim,
           "%s: row strides must be multiples of 8 elements that hold every head", what);
  TG_CHECK(aligned16(qkv) && aligned16(q_norm_weight) && aligned16(k_norm_weight) && aligned16(rope) && aligned16(out) &&
               aligned16(workspace),
           "%s: pointers must be 16-byte aligned", what);
  TG_CHECK(softmax_scale > 0.f, "%s: softmax_scale must be positive", what);
  TG_CHECK(max_seqlen_k < (1 << 24), "%s: max_seqlen_k must be less than 2^24", what);   // spans of under 4 GiB
  TG_CHECK(!bias_raw || (bias_seq_stride >= 0 && bias_head_stride >= 0), "%s: negative bias stride", what);
  if (num_seqs == 0) return 0;
  const QuantPlan p = plan_quant(bits, num_seqs, num_heads, num_heads_k, max_seqlen_k);
  a.qkv = static_cast<const bf16_t *>(qkv);
  a.qkv_rs = qkv_row_stride;
  a.rope = rope;
  a.h = num_heads;
  a.hkv = num_heads_k;
  a.qw = static_cast<const bf16_t *>(q_norm_weight);
  a.kw = static_cast<const bf16_t *>(k_norm_weight);
  a.eps = eps;
  a.q_head_scale = q_head_scale;
  a.q_row_scale = q_row_scale;
  a.kv_start = kv_start;
  a.kv_used = kv_used;
  a.max_k = max_seqlen_k;
  a.bias = bias_raw;
  a.bias_bs = bias_seq_stride;
  a.bias_hs = bias_head_stride;
  a.scale_log2 = softmax_scale * 1.4426950408889634f;
  a.out = static_cast<bf16_t *>(out);
  a.out_rs = out_row_stride;
  a.group = num_heads / num_heads_k;
  a.nseq = num_seqs;
  a.sets = p.sets;
  a.slots = p.slots;
  a.least = p.least;
  if (p.bytes > 0) {
    TG_CHECK(workspace != nullptr && workspace_bytes >= p.bytes, "%s: needs a workspace of %lld bytes (got %lld)", what,
             (long long)p.bytes, (long long)workspace_bytes);
    char *ws = static_cast<char *>(workspace);
    a.counters = reinterpret_cast<uint32_t *>(ws);
    a.ml = reinterpret_cast<uint64_t *>(ws + kCounters * 4);
    a.po = reinterpret_cast<uint64_t *>(ws + p.bytes - p.grid * p.hp * kHeadDim * 4);
  }
  const dim3 grid((unsigned)p.grid), block(64 * kWaves);
  auto launch = [&](auto bits_c, auto hp_c) {
    constexpr int BITS = decltype(bits_c)::value, HP = decltype(hp_c)::value;
    if (bias_raw)
      hipLaunchKernelGGL((decode_attn_quant_kernel<BITS, HP, true>), grid, block, 0, stream, a);
    else
      hipLaunchKernelGGL((decode_attn_quant_kernel<BITS, HP, false>), grid, block, 0, stream, a);
  };
  auto with_heads = [&](auto bits_c) {
    if (p.hp == 1) launch(bits_c, std::integral_constant<int, 1>());
    else if (p.hp == 2) launch(bits_c, std::integral_constant<int, 2>());
    else launch(bits_c, std::integral_constant<int, 4>());
  };
  if (bits == 4) with_heads(std::integral_constant<int, 4>());
  else with_heads(std::integral_constant<int, 8>());
  TG_HIP_CHECK(hipGetLastError());
  return 0;
}
