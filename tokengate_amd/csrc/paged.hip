// KV caches in pages: rows appended on the way out of the projection, and the attention of a decode step over them.
#include <algorithm>
#include <type_traits>

#include "decode_split.h"
#include "paged.h"
#include "tg_common.h"
#include "../../include/tokengate_hip.h"

namespace tg {
namespace {

// ---- start of a step: the packed rows' slots and rotary table -----------------------------------------
// One wave a row.  The row's sequence is the last one that begins at or before it (a bisection over cu_seqlens, whose
// values the lanes read alike).  Angles as tg_decode_begin's and tg_qk_norm_rope's: position * inv_freq in fp32.  8 rows take the
// launch (2.3 us); 32768 rows 8.4 us, 2.8 of them for the bytes (17 MB, nearly all written), the rest sines and cosines.
struct BeginArgs {
  const int64_t *pos;
  int64_t n;
  const float *inv_freq;
  const int32_t *cu, *used;
  int nseq;
  const int32_t *table;
  int64_t table_rs;
  int cols, lg, n_pages;
  int32_t *slots;
  float2 *rope;
};
__global__ __launch_bounds__(256) void paged_begin_kernel(BeginArgs a) {
  const int64_t t = (int64_t)blockIdx.x * 4 + wave_id();
  if (t >= a.n) return;
  const int lane = threadIdx.x & 63;
  float s, c;
  sincosf((float)a.pos[t] * a.inv_freq[lane], &s, &c);
  a.rope[t * (kHeadDim / 2) + lane] = float2{c, s};
  if (lane != 0) return;
  int lo = 0, hi = a.nseq;                       // cu[lo] <= t < cu[hi], where the row has a sequence
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.cu[mid] <= t) lo = mid;
    else hi = mid;
  }
  const int64_t first = a.cu[lo], end = a.cu[lo + 1], key = a.used[lo] - end + t;
  int32_t slot = -1;
  if (t >= first && t < end && key >= 0 && key >> a.lg < a.cols) {
    const int32_t page = a.table[lo * a.table_rs + (key >> a.lg)];
    if ((uint32_t)page < (uint32_t)a.n_pages) slot = (page << a.lg) + (int32_t)(key & ((1 << a.lg) - 1));
  }
  a.slots[t] = slot;
}

// ---- append: q/k RMSNorm, rotary embedding, k and v rows into their slots ------------------------------------
// 16 lanes a row of one head, 8 elements a lane (the rotate-half partner sits in lane j ^ 8); a group of 16 lanes takes up
// to kRowsPer rows of one token, so that its (cos, sin) are read once for them and as many rows are in flight.
struct AppendArgs {
  const bf16_t *qkv;
  int64_t qkv_rs;
  const float *rope;
  int64_t n;
  int h, hkv;
  const bf16_t *qw, *kw;
  float eps;
  const float *q_head_scale, *q_row_scale;
  bf16_t *q;
  int64_t q_rs, q_hs;
  const int32_t *slots;
  PagePool c;
  int groups;                    // of 16 lanes per token
};
// Bound by bytes: q | k | v read and written once (32768 rows 101 .. 103 us, 5.4 TB/s), few rows by the launch (8: 3.1).
// Sixteen lanes take kRowsPer heads of a token, all loads ahead of the first product; with 1 / 2 / 4 heads 32768 rows take
// 112 / 104 / 116 us, and 110 with two whose stores go through the caches.
constexpr int kRowsPer = 2;

// (past the caches: the queries of a long prompt outgrow them, and a short one's stay in the last level)
__device__ __forceinline__ void st16_stream(bf16_t *p, u32x4 v) { __builtin_nontemporal_store(v, reinterpret_cast<u32x4 *>(p)); }
__global__ __launch_bounds__(256) void paged_append_kernel(AppendArgs a) {
  const int j = threadIdx.x & 15;
  const uint32_t id = blockIdx.x * 16 + (threadIdx.x >> 4);   // (below 2^32)
  const int64_t t = id / (uint32_t)a.groups;
  const int sub = (int)(id - (uint32_t)t * (uint32_t)a.groups), rows = a.h + 2 * a.hkv;
  if (t >= a.n) return;          // uniform over the 16 lanes
  const bf16_t *src = a.qkv + t * a.qkv_rs + 8 * j;
  u32x4 raw[kRowsPer];
#pragma unroll
  for (int i = 0; i < kRowsPer; ++i) {
    const int r = sub + i * a.groups;
    if (r < rows) raw[i] = ld16(src + (int64_t)r * kHeadDim);
  }
  const f32x4 *rp = reinterpret_cast<const f32x4 *>(a.rope + t * kHeadDim + 16 * (j & 7));
  float cs[8][2];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f32x4 x = rp[i];
    cs[2 * i][0] = x[0];
    cs[2 * i][1] = x[1];
    cs[2 * i + 1][0] = x[2];
    cs[2 * i + 1][1] = x[3];
  }
  const int32_t slot = a.slots[t];
  const bool keep = (uint32_t)slot < (uint32_t)a.c.n_pages << a.c.lg;
  const int64_t page = slot >> a.c.lg, off = slot & ((1 << a.c.lg) - 1);
#pragma unroll
  for (int i = 0; i < kRowsPer; ++i) {
    const int r = sub + i * a.groups;
    if (r >= rows) break;
    if (r >= a.h + a.hkv) {      // a value
      if (keep) st16_stream(a.c.v + page * a.c.v_ps + (r - a.h - a.hkv) * a.c.v_hs + off * a.c.v_rs + 8 * j, raw[i]);
      continue;
    }
    const bool is_q = r < a.h;
    float x[8], wf[8], y[8];
    unpack8(raw[i], x);
    unpack8(ld16((is_q ? a.qw : a.kw) + 8 * j), wf);
    const float hs = is_q ? (float)(__bf16)((a.q_head_scale ? a.q_head_scale[r] : 1.f) * (a.q_row_scale ? a.q_row_scale[t] : 1.f))
                          : 1.f;
    norm_rope8(x, wf, a.eps, cs, j, hs, y);
    if (is_q) st16_stream(a.q + t * a.q_rs + r * a.q_hs + 8 * j, pack8(y));
    else if (keep) st16_stream(a.c.k + page * a.c.k_ps + (r - a.h) * a.c.k_hs + off * a.c.k_rs + 8 * j, pack8(y));
  }
}

// ---- attention of a decode step ---------------------------------------------------------------------
//   z_j = scale (q . k_j + bias_j),   out = sum_j e^(z_j - m) v_j / sum_j e^(z_j - m)
// Units of (sequence, KV head, up to 16 of its query heads) are cut into chunks on the device, from the lengths themselves
// (find_chunk); the last workgroup of a unit to arrive merges its chunks.  A wave takes 32 keys at a time, straight from the
// pages to registers in the layouts that the matrix cores read, so nothing waits at a barrier.  Bound by the bytes of K and V
// where there are many keys (8 of up to 131072 keys 441 us: 5.8 TB/s; 64 of up to 4099 131: 4.8), by dependent latencies where
// there are few: lengths and pages, norms, one tile and the waves' merge take 5.8 us, 300 keys 8.0, 2320 10.4, 32769 31 (27 where
// they are in the last-level cache).
//   * S^T = K Q^T (v_mfma_f32_16x16x32_bf16): A holds keys, lane (n, G) (n = lane % 16, G = lane / 16) elements 32 i + 8 G
//     .. + 7 of key 8 (n / 4) + 4 t + n % 4 of instruction t (0, 1); B the query heads, head n % HP in column n.  So lane
//     (n, G) ends up with the logits of keys 8 G .. 8 G + 7 of its head: in the order that the weights have as O's A.
//   * O = P V: a lane reads 16 bytes (elements 8 n .. 8 n + 7) of keys 8 G .. 8 G + 7; instruction e takes element 8 n + e of
//     the eight, one byte permutation per two.
//   * A weight is two bf16 numbers, 16 bits together (relative error 2^-17; rounded to one it would be 2^-8, as much as
//     the output's own rounding): columns repeat the heads, and every other repetition holds the second numbers.  With 16
//     heads there is no repetition, and the second numbers are a second product.
//   * The new key is not in the tiles: it is a part of its own beside the waves', from registers.
//   * Keys past the sequence's last, or of no page (page 0's rows are read in their place), are of weight 0 and their values 0,
//     whatever the rows hold.  A key that a
//     bias of -inf hides from a head may hold anything too: a wave whose sums are not finite takes its tiles once more,
//     each head by itself with the rows it does not see left out, and with weights 2^-64 of these (values near the largest
//     float pass fp32's range in the first sums).
struct PagedAttnArgs {
  const bf16_t *qkv;
  int64_t qkv_rs;
  const float *rope;
  int h, hkv, group;
  const bf16_t *qw, *kw;
  float eps;
  const float *q_head_scale, *q_row_scale;
  PagePool c;
  const int32_t *table;
  int64_t table_rs;
  int cols;
  const int32_t *used;
  int max_k;
  const float *bias;
  int64_t bias_bs, bias_hs;
  float scale_log2;
  bf16_t *out;
  int64_t out_rs;
  int nseq, sets;                // kv heads times head sets
  int slots, least;              // workgroups that are resident at once; fewest tiles per chunk
  float per_root;                // and as many for the root of the longest's tiles
  uint32_t *counters;            // per unit: chunks arrived; zero between launches
  uint64_t *ml;                  // [workgroup][head]: running max (log2 units) and sum
  uint64_t *po;                  // [workgroup][head][64]: O, pairs of fp32
};

typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));
// Waves of a workgroup, and workgroups that a CU holds.  4 / 8 / 12 waves (3 / 1 / 1 workgroups), 16 / 8 heads: one sequence of
// 32 keys 5.8 / 7.0 / 7.2 us, 2320 10.2 / 12.8 / 13.3, 32769 31 / 32 / 33, 64 of 300 16.5 / 22.5 / 24.2, 64 x 4096 183 / 184 / 185.
constexpr int kWaves = 4, kPerCu = 3;
constexpr int kTile = 32;        // keys of a wave's step
constexpr float kRescaleTau = 8.f;               // the running maximum moves only when a logit passes it by 2^8
constexpr float kLargeSum = 0x1p100f, kLift = 64.f;

template <int HP, bool HAS_BIAS>
__global__ __launch_bounds__(64 * kWaves, kPerCu) void paged_decode_kernel(PagedAttnArgs a) {
  const int tid = threadIdx.x, wave = wave_id(), lane = tid & 63, n16 = lane & 15, G = lane >> 4;
  const int set = blockIdx.x % a.sets, kh = set % a.hkv, hg = set / a.hkv;
  const int h0 = kh * a.group + hg * HP, nh = min(HP, a.group - hg * HP);   // heads h0 .. h0 + nh - 1

  __shared__ __attribute__((aligned(16))) bf16_t qs[HP][kHeadDim];
  __shared__ __attribute__((aligned(16))) bf16_t new_x[2][kHeadDim];   // the new key and value
  __shared__ __attribute__((aligned(16))) float part_o[kWaves + 1][HP][kHeadDim], part_ml[kWaves + 1][HP][2];

  const Chunk ck = find_chunk<kTile>({a.nseq, a.sets, a.slots, a.least, a.per_root}, blockIdx.x / a.sets, lane,
                                     [&](int s) { return Keys{0, max(0, min(a.used[s], a.max_k))}; });
  if (ck.seq < 0) return;                        // workgroup-uniform: past the last chunk
  const int b = ck.seq, sk = ck.sk, nk = max(0, sk - 1);   // keys in the pages; the new one is apart
  const int n_parts = ck.chunks, chunk = ck.chunk;
  const int t_lo = (int)((int64_t)ck.tiles * chunk / n_parts), t_hi = (int)((int64_t)ck.tiles * (chunk + 1) / n_parts);
  const int32_t *const trow = a.table + b * a.table_rs;
  const int lg = a.c.lg, mask = (1 << lg) - 1;
  auto page_of = [&](int key) { return trow[min(key >> lg, a.cols - 1)]; };
  // ---- loads of the rows to form, 16 lanes a row: query heads, then the new key and the new value.  They come before the
  // tiles': loads complete in issue order, and the rows are formed while the tiles' are on their way ----
  const bool last_chunk = chunk == n_parts - 1 && sk > 0;
  struct Row {
    u32x4 raw, norm_w;
    f32x4 turn[4];
    float scale;
  };
  auto load_row = [&](int r) {
    Row x;
    const int head = r < HP ? h0 + min(r, nh - 1) : r == HP ? a.h + kh : a.h + a.hkv + kh;
    x.raw = ld16(a.qkv + b * a.qkv_rs + (int64_t)head * kHeadDim + 8 * n16);
    x.norm_w = ld16((r < HP ? a.qw : a.kw) + 8 * n16);
    const f32x4 *rp = reinterpret_cast<const f32x4 *>(a.rope + b * kHeadDim + 16 * (n16 & 7));
#pragma unroll
    for (int i = 0; i < 4; ++i) x.turn[i] = rp[i];
    x.scale = 1.f;
    if (r < HP) x.scale = (float)(__bf16)((a.q_head_scale ? a.q_head_scale[head] : 1.f) * (a.q_row_scale ? a.q_row_scale[b] : 1.f));
    return x;
  };
  const int rows = HP + (last_chunk ? 2 : 0), row0 = tid >> 4;
  Row row;
  if (row0 < rows) row = load_row(row0);
  const int32_t new_page = page_of(nk);

  struct Tile {
    u32x4 k[2][4], v[8];
    float bias[8];
    int valid;                   // of this lane's keys 8 G .. 8 G + 7, those that are there
  };
  const bf16_t *const kbase = a.c.k + kh * a.c.k_hs + 8 * G, *const vbase = a.c.v + kh * a.c.v_hs + 8 * n16;
  const float *const bias_row = HAS_BIAS ? a.bias + (int64_t)b * a.bias_bs + (int64_t)(h0 + min(n16 & (HP - 1), nh - 1)) * a.bias_hs : nullptr;
  // the page entries of the tile after the one whose loads are on their way
  int32_t kp = 0, vp = 0;
  auto load_entries = [&](int tile) {
    kp = page_of(tile * kTile + 8 * (n16 >> 2));
    vp = page_of(tile * kTile + 8 * G);
  };
  auto load_k = [&](Tile &l, int tile) {
    const int kk = tile * kTile + 8 * (n16 >> 2), vk = tile * kTile + 8 * G;
    const int64_t page = (uint32_t)kp < (uint32_t)a.c.n_pages ? kp : 0;   // (no page: any row will do)
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const bf16_t *p = kbase + page * a.c.k_ps + (int64_t)((kk & mask) + 4 * t + (n16 & 3)) * a.c.k_rs;
#pragma unroll
      for (int i = 0; i < 4; ++i) l.k[t][i] = ld16(p + 32 * i);
    }
    if constexpr (HAS_BIAS) {
      if (tile * kTile + kTile <= nk) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const f32x4_u x = *reinterpret_cast<const f32x4_u *>(bias_row + vk + 4 * i);
#pragma unroll
          for (int j = 0; j < 4; ++j) l.bias[4 * i + j] = x[j];
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) l.bias[j] = vk + j < nk ? bias_row[vk + j] : 0.f;
      }
    }
  };
  auto load_v = [&](Tile &l, int tile) {
    const int vk = tile * kTile + 8 * G;
    const bool there = (uint32_t)vp < (uint32_t)a.c.n_pages;
    const int64_t page = there ? vp : 0;
    l.valid = there ? max(0, min(8, nk - vk)) : 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) l.v[j] = ld16(vbase + page * a.c.v_ps + (int64_t)((vk & mask) + j) * a.c.v_rs);
  };

  Tile l;
  auto first_loads = [&](int t) {
    load_entries(t);
    load_k(l, t);
    load_v(l, t);
    load_entries(t + kWaves);
  };
  int t = t_lo + wave;
  if (t < t_hi) first_loads(t);

  const bool has_new = last_chunk && (uint32_t)new_page < (uint32_t)a.c.n_pages;
  for (int r = row0; r < rows; r += 4 * kWaves) {
    if (r != row0) row = load_row(r);
    u32x4 y8 = row.raw;
    if (r <= HP) {
      float x[8], wf[8], y[8], cs[8][2];
      unpack8(row.raw, x);
      unpack8(row.norm_w, wf);
#pragma unroll
      for (int i = 0; i < 16; ++i) cs[i >> 1][i & 1] = row.turn[i >> 2][i & 3];
      norm_rope8(x, wf, a.eps, cs, n16, row.scale, y);
      y8 = pack8(y);
    }
    if (r < HP) {
      st16(&qs[r][8 * n16], y8);
    } else {
      st16(&new_x[r - HP][8 * n16], y8);
      if (hg == 0 && has_new) {
        const int64_t page = new_page, off = nk & mask;
        st16((r == HP ? a.c.k + page * a.c.k_ps + kh * a.c.k_hs + off * a.c.k_rs
                      : a.c.v + page * a.c.v_ps + kh * a.c.v_hs + off * a.c.v_rs) + 8 * n16, y8);
      }
    }
  }
  __syncthreads();
  // ---- the new key: a part of its own, 16 lanes a head ----
  if (has_new && wave == kWaves - 1) {
    for (int i = G; i < HP; i += 4) {
      float q[8], k[8], v[8], z = 0.f;
      unpack8(*reinterpret_cast<const u32x4 *>(&qs[i][8 * n16]), q);
      unpack8(*reinterpret_cast<const u32x4 *>(&new_x[0][8 * n16]), k);
      unpack8(*reinterpret_cast<const u32x4 *>(&new_x[1][8 * n16]), v);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        z = fmaf(q[e], k[e], z);
        part_o[kWaves][i][8 * n16 + e] = v[e];
      }
      z += dpp<0xB1>(z);
      z += dpp<0x4E>(z);
      z += dpp<0x141>(z);
      z += dpp<0x140>(z);
      const float bias = HAS_BIAS ? a.bias[(int64_t)b * a.bias_bs + (int64_t)(h0 + min(i, nh - 1)) * a.bias_hs + nk] : 0.f;
      const bool hidden = bias == -INFINITY;
      if (n16 == 0) {
        part_ml[kWaves][i][0] = hidden ? -INFINITY : HAS_BIAS ? in_range((z + bias) * a.scale_log2) : z * a.scale_log2;
        part_ml[kWaves][i][1] = hidden ? 0.f : 1.f;
      }
    }
  }

  bf16x8 qf[4];                  // lane (n, G): elements 32 i + 8 G .. + 7 of head n % HP
#pragma unroll
  for (int i = 0; i < 4; ++i) qf[i] = *reinterpret_cast<const bf16x8 *>(&qs[n16 & (HP - 1)][32 * i + 8 * G]);
  const bool second = HP < 16 && (n16 & HP);     // this column holds the weights' second numbers

  f32x4 oacc[8];                 // lane (n, G): rows (columns of S^T) 4 G .. 4 G + 3, elements 8 n + e
  float mrun, lsum;
  // tile t; with NEXT the loads of the wave's next one are made as its registers fall free
  auto step = [&](Tile &l, int t, auto careful_c, auto next_c, float lift) {
    constexpr bool CAREFUL = decltype(careful_c)::value, NEXT = decltype(next_c)::value;
    f32x4 s[2] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int t = 0; t < 2; ++t) s[t] = mfma16(__builtin_bit_cast(bf16x8, l.k[t][i]), qf[i], s[t]);
    float z[8], most = -INFINITY;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      z[j] = (HAS_BIAS ? s[j >> 2][j & 3] + l.bias[j] : s[j >> 2][j & 3]) * a.scale_log2;
      asm("" : "+v"(z[j]));   // rounded: contracted into z - m below, a bias near the lowest float leaves the rounding's rest
      if constexpr (HAS_BIAS) z[j] = in_range(z[j]);
      if (j >= l.valid) z[j] = -INFINITY;
      if constexpr (HAS_BIAS) z[j] = l.bias[j] == -INFINITY ? -INFINITY : z[j];   // hidden, whatever the row holds
      most = fmaxf(most, z[j]);
    }
    if constexpr (NEXT) load_k(l, t + kWaves);
    __builtin_amdgcn_sched_barrier(0);
    if (__builtin_amdgcn_ballot_w64(most > mrun + (kRescaleTau - lift))) {
      const float m = fmaxf(mrun, quad_swap_max(most) + lift), f = mrun == -INFINITY ? 0.f : fast_exp2(mrun - m);
      mrun = m;
      lsum *= f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float fr = __shfl(f, 4 * G + i);   // of the row's head
#pragma unroll
        for (int e = 0; e < 8; ++e) oacc[e][i] *= fr;
      }
    }
    const float base = mrun == -INFINITY ? 0.f : mrun;
    u32x4 w0, w1;
    float p[8];
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      p[j] = fast_exp2(z[j] - base);
      p[j + 1] = fast_exp2(z[j + 1] - base);
      lsum += p[j] + p[j + 1];
      const uint32_t hi = pack_bf16x2(p[j], p[j + 1]);
      const uint32_t lo = pack_bf16x2(p[j] - u32_as_f32(hi << 16), p[j + 1] - u32_as_f32(hi & 0xffff0000u));
      w0[j >> 1] = second && !CAREFUL ? lo : hi;
      w1[j >> 1] = lo;
    }
    if (__builtin_amdgcn_ballot_w64(l.valid < 8)) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j >= l.valid) l.v[j] = u32x4{0u, 0u, 0u, 0u};
    }
    auto column = [&](auto word, int odd) {        // the low or high halves of word(j), j = 0 .. 7
      u32x4 c;
#pragma unroll
      for (int m = 0; m < 4; ++m) c[m] = __builtin_amdgcn_perm(word(2 * m + 1), word(2 * m), odd ? 0x07060302u : 0x05040100u);
      return __builtin_bit_cast(bf16x8, c);
    };
    const bf16x8 pa = __builtin_bit_cast(bf16x8, w0), pb = __builtin_bit_cast(bf16x8, w1);
    if constexpr (!CAREFUL) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bf16x8 v = column([&](int j) { return (uint32_t)l.v[j][e >> 1]; }, e & 1);   // element 8 n + e of keys 8 G .. 8 G + 7
        oacc[e] = mfma16(pa, v, oacc[e]);
        if constexpr (HP == 16) oacc[e] = mfma16(pb, v, oacc[e]);
      }
    } else {
      // (the second numbers times the finite values alone: such a number may be 0)
      auto finite = [](uint32_t x) {
        const uint32_t lo = (x & 0x7f80u) == 0x7f80u ? 0u : x & 0xffffu, hi = (x & 0x7f800000u) == 0x7f800000u ? 0u : x & 0xffff0000u;
        return lo | hi;
      };
#pragma unroll 1
      for (int hd = 0; hd < HP; ++hd) {
        bool sees[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) sees[j] = __shfl(p[j], 16 * G + hd) != 0.f;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          uint32_t v[8], u[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            v[j] = sees[j] ? l.v[j][x] : 0u;
            u[j] = finite(v[j]);
          }
#pragma unroll
          for (int odd = 0; odd < 2; ++odd) {
            const f32x4 first = mfma16(pa, column([&](int j) { return v[j]; }, odd), f32x4{0.f, 0.f, 0.f, 0.f});
            const f32x4 o = mfma16(pb, column([&](int j) { return u[j]; }, odd), first);
#pragma unroll
            for (int i = 0; i < 4; ++i) oacc[2 * x + odd][i] += 4 * G + i == hd ? o[i] : 0.f;
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
    if constexpr (NEXT) {
      load_v(l, t + kWaves);
      load_entries(t + 2 * kWaves);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  auto clear = [&] {
#pragma unroll
    for (int e = 0; e < 8; ++e) oacc[e] = f32x4{0.f, 0.f, 0.f, 0.f};
    mrun = -INFINITY;
    lsum = 0.f;
  };
  // elements 8 n .. 8 n + 7 of head i, i = 0 .. 3 of the lane group that holds the head's first rows, the numbers' sums
  auto sums = [&](int i, float (&o)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (HP == 1) o[e] = oacc[e][0] + oacc[e][1];
      else if constexpr (HP == 2) o[e] = oacc[e][i] + oacc[e][i + 2];
      else if constexpr (HP == 4) o[e] = add_row_pair(oacc[e][i]);
      else if constexpr (HP == 8) o[e] = pair_sum(oacc[e][i]);
      else o[e] = oacc[e][i];
    }
  };
  constexpr int kHere = HP < 4 ? HP : 4;         // heads of a lane group
  auto fine = [&] {
    bool ok = true;
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) ok &= fabsf(oacc[e][i]) < kLargeSum;
    return !__builtin_amdgcn_ballot_w64(!ok);
  };
  clear();
  if (t < t_hi) {
    for (; t + kWaves < t_hi; t += kWaves) step(l, t, std::false_type(), std::true_type(), 0.f);
    step(l, t, std::false_type(), std::false_type(), 0.f);
  }
  if (!fine()) {                                 // (a NaN that a visible key holds comes again)
    clear();
    for (t = t_lo + wave; t < t_hi; t += kWaves) {
      first_loads(t);
      step(l, t, std::true_type(), std::false_type(), kLift);
    }
  }

  // ---- the waves' results meet in LDS ----
  {
    const float l = add_rows(lsum);
    if (G == 0 && n16 < HP) {
      part_ml[wave][n16][0] = mrun;
      part_ml[wave][n16][1] = l;
    }
#pragma unroll
    for (int i = 0; i < kHere; ++i) {
      float o[8];
      sums(i, o);
      const int hd = 4 * G + i;
      if (hd < HP) {
#pragma unroll
        for (int e = 0; e < 8; ++e) part_o[wave][hd][8 * n16 + e] = o[e];
      }
    }
  }
  __syncthreads();
  bf16_t *const orow = a.out + b * a.out_rs + (int64_t)h0 * kHeadDim;
  auto put = [&](int item, float o0, float o1, float l) {   // a row that saw no key: 0
    const float f = l == 0.f ? 0.f : 1.f / l;
    if (item / 64 < nh)
      *reinterpret_cast<uint32_t *>(orow + 2 * item) = l == 0.f ? 0u : pack_bf16x2(o0 * f, o1 * f);
  };
  for (int item = tid; item < HP * kHeadDim / 2; item += 64 * kWaves) {
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
  constexpr int kThreads = 64 * kWaves, kAll = HP * 32, kItems = kAll < kThreads ? kAll : kThreads, kSets = kThreads / kItems, kAhead = 8;
  __shared__ float set_s[kSets > 1 ? kSets - 1 : 1][6][kItems];
  const int cs = tid / kItems;
#pragma unroll 1
  for (int item = tid % kItems; item < kAll; item += kItems) {
    const int i = item / 32;
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
    if constexpr (kSets > 1) {                     // (one item per thread)
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
    }
    put(2 * item, o[0], o[1], l);
    put(2 * item + 1, o[2], o[3], l);
  }
}

// Workgroups of a launch: units of (sequence, kv head, head set), cut into chunks on the device.
struct DecodePlan {
  int hp, sets, slots, least;    // query heads of a workgroup: a power of two that holds the KV head's, at most 16
  float per_root;                // see SplitRule
  int64_t grid, bytes;
};
// The counters' region is the same for every launch, so that no launch writes partial results where another counts;
// launches of more units cut none.
constexpr int64_t kCounters = 1 << 14;
DecodePlan plan_decode(int64_t num_seqs, int num_heads, int num_heads_k, int max_k) {
  DecodePlan p;
  const int group = num_heads / num_heads_k;
  for (p.hp = 1; p.hp < group && p.hp < 16;) p.hp *= 2;
  p.sets = num_heads_k * ((group + p.hp - 1) / p.hp);
  const int64_t units = num_seqs * p.sets;
  // Few units: a workgroup per CU, whose longer chunks make fewer to merge (one sequence of 8192 / 32769 / 131072 keys with
  // three per CU 17.7 / 34.3 / 100, with one 14.5 / 31.3 / 97 us; 2 of 8192 22.9 / 18.9); many, of uneven lengths, balance
  // better over more (64 of up to 4099 132, over one per CU 131, two 150; 40 of up to 6000 108, 131, 109).
  p.slots = (units < 128 ? 1 : kPerCu) * device_cus();
  // Chunks of some of the four waves' steps, more for longer sequences, as the merge takes 0.1 us a chunk, with 8 and 16 heads 0.3:
  // one of 8192 keys in 64 chunks 16.8, in 22 13.5, in 8 18; 8 of 8192 with 16 / 2 heads 31.5, 22.2, 19.5.  Up to 12 tiles
  // are not cut (300 keys 8.9 in three chunks, 8.1 in one).
  p.per_root = p.hp >= 8 ? 0.26f : 0.22f;
  const int64_t tiles = std::max(1, (max_k + kTile - 1) / kTile);
  p.least = units <= kCounters ? kWaves : 1 << 22;
  p.grid = std::min<int64_t>(units * ((tiles + p.least - 1) / p.least), units + kRounds * p.slots);
  // counters, (max, sum), O
  p.bytes = p.grid == units ? 0 : kCounters * 4 + (p.grid * p.hp * 8 + 255) / 256 * 256 + p.grid * p.hp * kHeadDim * 4;
  return p;
}

}  // namespace
}  // namespace tg

using namespace tg;

extern "C" int tg_paged_begin(const int64_t *positions, int64_t n_rows, const float *inv_freq, const int32_t *cu_seqlens,
                              const int32_t *kv_used, int32_t num_seqs, const int32_t *page_table, int64_t table_stride,
                              int32_t table_cols, int32_t num_pages, int32_t page_rows, int32_t *slots, float *rope,
                              hipStream_t stream) {
  clear_error();
  const char *what = "paged_begin";
  TG_CHECK(positions && inv_freq && cu_seqlens && kv_used && slots && rope, "%s: null pointer", what);
  TG_CHECK(n_rows >= 0 && n_rows < (1ll << 31) && num_seqs > 0, "%s: bad row or sequence count", what);
  TG_CHECK(num_pages >= 0 && page_rows >= 16 && page_rows <= 65536 && (page_rows & (page_rows - 1)) == 0 &&
               (int64_t)num_pages * page_rows < (1ll << 31),
           "%s: page rows must be a power of two from 16 to 65536, of less than 2^31 rows in all", what);
  if (int e = check_table(what, page_table, table_stride, table_cols, num_seqs)) return e;
  if (n_rows == 0) return 0;
  const BeginArgs a{positions, n_rows, inv_freq, cu_seqlens, kv_used, num_seqs, page_table, table_stride, table_cols,
                    __builtin_ctz((unsigned)page_rows), num_pages, slots, reinterpret_cast<float2 *>(rope)};
  hipLaunchKernelGGL(paged_begin_kernel, dim3((unsigned)((n_rows + 3) / 4)), dim3(256), 0, stream, a);
  TG_HIP_CHECK(hipGetLastError());
  return 0;
}

extern "C" int tg_paged_append(const void *qkv, int64_t qkv_row_stride, const float *rope, int64_t n_tokens,
                               int32_t num_heads, int32_t num_heads_k, int32_t head_dim, const void *q_norm_weight,
                               const void *k_norm_weight, float eps, const float *q_head_scale, const float *q_row_scale,
                               void *q_out, int64_t q_row_stride, int64_t q_head_stride, const int32_t *slots,
                               void *k_pages, int64_t k_page_stride, int64_t k_head_stride, int64_t k_row_stride,
                               void *v_pages, int64_t v_page_stride, int64_t v_head_stride, int64_t v_row_stride,
                               int32_t num_pages, int32_t page_rows, hipStream_t stream) {
  clear_error();
  const char *what = "paged_append";
  AppendArgs a{};
  if (int e = check_pool(what, k_pages, v_pages, {k_page_stride, k_head_stride, k_row_stride},
                         {v_page_stride, v_head_stride, v_row_stride}, num_pages, page_rows, num_heads_k, head_dim, &a.c))
    return e;
  TG_CHECK(qkv && rope && q_norm_weight && k_norm_weight && q_out && slots, "%s: null pointer", what);
  TG_CHECK(num_heads > 0 && num_heads <= 256, "%s: heads must be in 1..256", what);
  TG_CHECK(n_tokens >= 0 && n_tokens < (1ll << 31), "%s: bad token count", what);
  TG_CHECK(qkv_row_stride % 8 == 0 && qkv_row_stride >= (int64_t)(num_heads + 2 * num_heads_k) * kHeadDim,
           "%s: qkv rows must hold q, k and v of every head, strides be multiples of 8 elements", what);
  TG_CHECK(q_row_stride % 8 == 0 && q_head_stride % 8 == 0 && q_head_stride >= kHeadDim && q_row_stride >= 0,
           "%s: q strides must be multiples of 8 elements, heads apart", what);
  TG_CHECK(aligned16(qkv) && aligned16(q_norm_weight) && aligned16(k_norm_weight) && aligned16(rope) && aligned16(q_out),
           "%s: pointers must be 16-byte aligned", what);
  if (n_tokens == 0) return 0;
  a.qkv = static_cast<const bf16_t *>(qkv);
  a.qkv_rs = qkv_row_stride;
  a.rope = rope;
  a.n = n_tokens;
  a.h = num_heads;
  a.hkv = num_heads_k;
  a.qw = static_cast<const bf16_t *>(q_norm_weight);
  a.kw = static_cast<const bf16_t *>(k_norm_weight);
  a.eps = eps;
  a.q_head_scale = q_head_scale;
  a.q_row_scale = q_row_scale;
  a.q = static_cast<bf16_t *>(q_out);
  a.q_rs = q_row_stride;
  a.q_hs = q_head_stride;
  a.slots = slots;
  a.groups = (num_heads + 2 * num_heads_k + kRowsPer - 1) / kRowsPer;
  const int64_t blocks = (n_tokens * a.groups + 15) / 16;
  TG_CHECK(blocks < (1ll << 28), "%s: too many tokens", what);
  hipLaunchKernelGGL(paged_append_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, a);
  TG_HIP_CHECK(hipGetLastError());
  return 0;
}

extern "C" int64_t tg_paged_decode_attention_workspace_size(int32_t num_seqs, int32_t num_heads, int32_t num_heads_k,
                                                            int32_t max_seqlen_k) {
  if (num_seqs <= 0 || num_heads <= 0 || num_heads_k <= 0 || num_heads % num_heads_k != 0 || max_seqlen_k <= 0) return 0;
  const int64_t fits = kCounters / plan_decode(1, num_heads, num_heads_k, 1).sets;   // sequences that may be cut
  return plan_decode(std::min<int64_t>(num_seqs, fits), num_heads, num_heads_k, max_seqlen_k).bytes;
}

extern "C" int tg_paged_decode_attention(const void *qkv, int64_t qkv_row_stride, const float *rope, int32_t num_seqs,
                                         int32_t num_heads, int32_t num_heads_k, int32_t head_dim,
                                         const void *q_norm_weight, const void *k_norm_weight, float eps,
                                         const float *q_head_scale, const float *q_row_scale, void *k_pages,
                                         int64_t k_page_stride, int64_t k_head_stride, int64_t k_row_stride,
                                         void *v_pages, int64_t v_page_stride, int64_t v_head_stride,
                                         int64_t v_row_stride, int32_t num_pages, int32_t page_rows,
                                         const int32_t *page_table, int64_t table_stride, int32_t table_cols,
                                         const int32_t *kv_used, int32_t max_seqlen_k, const float *bias_raw,
                                         int64_t bias_seq_stride, int64_t bias_head_stride, float softmax_scale,
                                         void *out, int64_t out_row_stride, void *workspace, int64_t workspace_bytes,
                                         hipStream_t stream) {
  clear_error();
  const char *what = "paged_decode_attention";
  PagedAttnArgs a{};
  if (int e = check_pool(what, k_pages, v_pages, {k_page_stride, k_head_stride, k_row_stride},
                         {v_page_stride, v_head_stride, v_row_stride}, num_pages, page_rows, num_heads_k, head_dim, &a.c))
    return e;
  if (int e = check_table(what, page_table, table_stride, table_cols, num_seqs)) return e;
  TG_CHECK(qkv && rope && q_norm_weight && k_norm_weight && kv_used && out, "%s: null pointer", what);
  TG_CHECK(num_heads > 0 && num_heads <= 256 && num_heads % num_heads_k == 0,
           "%s: heads must be in 1..256 and a multiple of the KV heads", what);
  TG_CHECK(num_seqs >= 0 && (int64_t)num_seqs * num_heads < (1 << 24), "%s: bad sequence count", what);
  TG_CHECK(max_seqlen_k >= 0 && max_seqlen_k < (1 << 24), "%s: max_seqlen_k must be in 0..2^24 - 1", what);
  TG_CHECK(max_seqlen_k <= (int64_t)table_cols * page_rows, "%s: max_seqlen_k is more than the page table's columns hold", what);
  TG_CHECK(qkv_row_stride % 8 == 0 && out_row_stride % 8 == 0 &&
               qkv_row_stride >= (int64_t)(num_heads + 2 * num_heads_k) * kHeadDim &&
               out_row_stride >= (int64_t)num_heads * kHeadDim,
           "%s: row strides must be multiples of 8 elements that hold every head", what);
  TG_CHECK(aligned16(qkv) && aligned16(q_norm_weight) && aligned16(k_norm_weight) && aligned16(rope) && aligned16(out) &&
               aligned16(workspace),
           "%s: pointers must be 16-byte aligned", what);
  TG_CHECK(softmax_scale > 0.f, "%s: softmax_scale must be positive", what);
  TG_CHECK(!bias_raw || (bias_seq_stride >= 0 && bias_head_stride >= 0), "%s: negative bias stride", what);
  if (num_seqs == 0) return 0;
  a.qkv = static_cast<const bf16_t *>(qkv);
  a.qkv_rs = qkv_row_stride;
  a.rope = rope;
  a.h = num_heads;
  a.hkv = num_heads_k;
  a.group = num_heads / num_heads_k;
  a.qw = static_cast<const bf16_t *>(q_norm_weight);
  a.kw = static_cast<const bf16_t *>(k_norm_weight);
  a.eps = eps;
  a.q_head_scale = q_head_scale;
  a.q_row_scale = q_row_scale;
  a.table = page_table;
  a.table_rs = table_stride;
  a.cols = table_cols;
  a.used = kv_used;
  a.max_k = max_seqlen_k;
  a.bias = bias_raw;
  a.bias_bs = bias_seq_stride;
  a.bias_hs = bias_head_stride;
  a.scale_log2 = softmax_scale * 1.4426950408889634f;
  a.out = static_cast<bf16_t *>(out);
  a.out_rs = out_row_stride;
  a.nseq = num_seqs;
  const DecodePlan p = plan_decode(num_seqs, num_heads, num_heads_k, max_seqlen_k);
  const int hp = p.hp;
  a.sets = p.sets;
  a.slots = p.slots;
  a.least = p.least;
  a.per_root = p.per_root;
  if (p.bytes > 0) {
    TG_CHECK(workspace != nullptr && workspace_bytes >= p.bytes, "%s: needs a workspace of %lld bytes (got %lld)", what,
             (long long)p.bytes, (long long)workspace_bytes);
    char *ws = static_cast<char *>(workspace);
    a.counters = reinterpret_cast<uint32_t *>(ws);
    a.ml = reinterpret_cast<uint64_t *>(ws + kCounters * 4);
    a.po = reinterpret_cast<uint64_t *>(ws + p.bytes - p.grid * p.hp * kHeadDim * 4);
  }
  const dim3 grid((unsigned)p.grid), block(64 * kWaves);
  auto launch = [&](auto hp_c) {
    constexpr int HP = decltype(hp_c)::value;
    if (bias_raw) hipLaunchKernelGGL((paged_decode_kernel<HP, true>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((paged_decode_kernel<HP, false>), grid, block, 0, stream, a);
  };
  if (hp == 1) launch(std::integral_constant<int, 1>());
  else if (hp == 2) launch(std::integral_constant<int, 2>());
  else if (hp == 4) launch(std::integral_constant<int, 4>());
  else if (hp == 8) launch(std::integral_constant<int, 8>());
  else launch(std::integral_constant<int, 16>());
  TG_HIP_CHECK(hipGetLastError());
  return 0;
}
