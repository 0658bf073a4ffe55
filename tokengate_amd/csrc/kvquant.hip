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

// Lanes j = 2 e + p of 16 lanes hold element i of an 8 x 8 table (e, i) in nibble (byte) i of w: transposed among
// the eight lanes of the same p.  Its own inverse.
__device__ __forceinline__ uint32_t swap_parts(uint32_t x, uint32_t mask, int shift, int lanes, bool up) {
  const uint32_t y = __shfl_xor(x, lanes);
  return up ? (x & ~mask) | ((y >> shift) & mask) : (x & mask) | ((y & mask) << shift);
}
template <int BITS>
__device__ __forceinline__ void transpose8(uint32_t (&w)[BITS / 4], int j) {
  if constexpr (BITS == 4) {
    w[0] = swap_parts(w[0], 0x0F0F0F0Fu, 4, 2, j & 2);
    w[0] = swap_parts(w[0], 0x00FF00FFu, 8, 4, j & 4);
    w[0] = swap_parts(w[0], 0x0000FFFFu, 16, 8, j & 8);
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      w[i] = swap_parts(w[i], 0x00FF00FFu, 8, 2, j & 2);
      w[i] = swap_parts(w[i], 0x0000FFFFu, 16, 4, j & 4);
    }
    const uint32_t give = j & 8 ? w[0] : w[1], got = __shfl_xor(give, 8);
    w[0] = j & 8 ? got : w[0];
    w[1] = j & 8 ? w[1] : got;
  }
}
// The word (pair) that lane j of a row holds after transpose8
__device__ __forceinline__ int word_of(int j) { return 8 * (j & 1) + (j >> 1); }

// Quantises a row held by 16 lanes, lane j its elements 8 j .. 8 j + 7: word (pair) word_of(j) of its codes, and the
// (s, m) pair of its group j / 4.  The quotient is the correctly rounded one of a division: q = d (1/s) and one
// correction by its remainder.
template <int BITS>
__device__ __forceinline__ void quant_row(const float (&x)[8], int j, uint32_t (&w)[BITS / 4], uint32_t &meta) {
  float mn = min3_nan(min3_nan(x[0], x[1], x[2]), min3_nan(x[3], x[4], x[5]), min3_nan(x[6], x[7], x[7]));
  float mx = max3_nan(max3_nan(x[0], x[1], x[2]), max3_nan(x[3], x[4], x[5]), max3_nan(x[6], x[7], x[7]));
#pragma unroll
  for (int o = 1; o <= 2; o <<= 1) {
    const float a = __shfl_xor(mn, o), b = __shfl_xor(mx, o);
    mn = min3_nan(mn, a, a);
    mx = max3_nan(mx, b, b);
  }
  const float span = mx - mn;
  const bool fine = span < INFINITY;             // neither NaN nor infinite
  float s = (float)(__bf16)(span / top_code<BITS>());
  s = s < kLeastStep ? 0.f : s;
  const float inv = fine && s > 0.f ? 1.f / s : 0.f;
  uint32_t c[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float d = x[i] - mn;
    float q = d * inv;
    q = fmaf(fmaf(-q, s, d), inv, q);
    q = fminf(fmaxf(rintf(q), 0.f), top_code<BITS>());   // (a NaN gives 0)
    c[i] = (uint32_t)q;
  }
#pragma unroll
  for (int k = 0; k < BITS / 4; ++k) {
    w[k] = 0;
#pragma unroll
    for (int i = 0; i < 32 / BITS; ++i) w[k] |= c[k * (32 / BITS) + i] << (BITS * i);
  }
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
// One (row, head, K or V) per 16 lanes.
template <int BITS>
__global__ __launch_bounds__(256) void kv_quantize_kernel(RowSource a, QuantCache c, int64_t n) {
  const int64_t t = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  const int j = threadIdx.x & 15, head = blockIdx.y;
  const bool is_v = blockIdx.z;
  if (t >= n) return;
  const int64_t src = a.src_rows ? a.src_rows[t] : t, dst = a.dst_rows ? a.dst_rows[t] : t;
  if (src < 0 || src >= a.rows || dst < 0 || dst >= c.rows) return;   // alike in the 16 lanes
  const bf16_t *p = is_v ? a.v + src * a.v_rs + head * a.v_hs : a.k + src * a.k_rs + head * a.k_hs;
  float x[8];
  unpack8(ld16(p + 8 * j), x);
  uint32_t w[BITS / 4], meta;
  quant_row<BITS>(x, j, w, meta);
  const int64_t row = head * c.head_rows + dst;
  uint32_t *out = (is_v ? c.v : c.k) + row * row_words<BITS>() + word_of(j) * (BITS / 4);
#pragma unroll
  for (int i = 0; i < BITS / 4; ++i) out[i] = w[i];
  if ((j & 3) == 0) (is_v ? c.vm : c.km)[row * kGroups + (j >> 2)] = meta;
}

struct RowTarget {
  bf16_t *k, *v;
  int64_t k_rs, k_hs, v_rs, v_hs;
  const int32_t *rows;
};
template <int BITS>
__global__ __launch_bounds__(256) void kv_dequantize_kernel(QuantCache c, RowTarget a, int64_t n) {
  const int64_t t = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  const int j = threadIdx.x & 15, head = blockIdx.y;
  const bool is_v = blockIdx.z;
  if (t >= n) return;
  const int64_t src = a.rows ? a.rows[t] : t;
  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (src >= 0 && src < c.rows) {
    const int64_t row = head * c.head_rows + src;
    const uint32_t *in = (is_v ? c.v : c.k) + row * row_words<BITS>() + word_of(j) * (BITS / 4);
    uint32_t w[BITS / 4];
#pragma unroll
    for (int i = 0; i < BITS / 4; ++i) w[i] = in[i];
    read_row<BITS>(w, (is_v ? c.vm : c.km)[row * kGroups + (j >> 2)], j, x);
  }
  st16((is_v ? a.v + t * a.v_rs + head * a.v_hs : a.k + t * a.k_rs + head * a.k_hs) + 8 * j, pack8(x));
}

// ---- attention of a decode step ---------------------------------------------------------------------
struct QuantAttnArgs {
  const bf16_t *qkv;
  int64_t qkv_rs;
  const float *rope;
  int h, hkv;
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
};

// One workgroup per (query head, sequence); 16 lanes take a key at a time, every 16th of the sequence, each with a
// running maximum and sum of its own; the 16 results meet in LDS.
template <int BITS>
__global__ __launch_bounds__(256) void decode_attn_quant_kernel(QuantAttnArgs a) {
  const int h = blockIdx.x, b = blockIdx.y, kh = h / (a.h / a.hkv);
  const int grp = threadIdx.x >> 4, j = threadIdx.x & 15;
  __shared__ float qs[kHeadDim];
  __shared__ uint32_t new_w[2][row_words<BITS>()], new_m[2][kGroups];
  __shared__ float part[16][kHeadDim], pm[16], pl[16];
  const int64_t start = a.kv_start[b];
  int sk = min(a.kv_used[b], a.max_k);
  if (start < 0 || start + sk > a.c.rows) sk = 0;
  if (grp < 3) {          // this head's query, and the new key and value
    const int head = grp == 0 ? h : grp == 1 ? a.h + kh : a.h + a.hkv + kh;
    float x[8], y[8], wf[8];
    unpack8(ld16(a.qkv + b * a.qkv_rs + (int64_t)head * kHeadDim + 8 * j), x);
    if (grp < 2) {
      unpack8(ld16((grp == 0 ? a.qw : a.kw) + 8 * j), wf);
      const float hs = grp == 0 ? (float)(__bf16)((a.q_head_scale ? a.q_head_scale[h] : 1.f) *
                                                  (a.q_row_scale ? a.q_row_scale[b] : 1.f))
                                : 1.f;
      norm_rope8(x, wf, a.eps, reinterpret_cast<const float(*)[2]>(a.rope) + b * (kHeadDim / 2) + 8 * (j & 7), j, hs, y);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = (float)(__bf16)y[i];
    }
    if (grp == 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) qs[8 * j + i] = x[i];
    } else {
      uint32_t w[BITS / 4], meta;
      quant_row<BITS>(x, j, w, meta);
      const int64_t row = kh * a.c.head_rows + start + sk - 1;
      const bool write = sk > 0 && h % (a.h / a.hkv) == 0;
      uint32_t *codes = grp == 1 ? a.c.k : a.c.v, *metas = grp == 1 ? a.c.km : a.c.vm;
#pragma unroll
      for (int i = 0; i < BITS / 4; ++i) {
        const int at = word_of(j) * (BITS / 4) + i;
        new_w[grp - 1][at] = w[i];
        if (write) codes[row * row_words<BITS>() + at] = w[i];
      }
      if ((j & 3) == 0) {
        new_m[grp - 1][j >> 2] = meta;
        if (write) metas[row * kGroups + (j >> 2)] = meta;
      }
    }
  }
  __syncthreads();
  float q[8], acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) q[e] = qs[16 * e + j];
  auto load = [&](const uint32_t *w, const uint32_t *meta, float (&x)[8]) {   // elements 16 e + j of a row
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t c = (w[j * (BITS / 4) + e * BITS / 32] >> (BITS * e % 32)) & ((1u << BITS) - 1u);
      x[e] = fmaf((float)c, u32_as_f32(meta[e >> 1] << 16), u32_as_f32(meta[e >> 1] & 0xffff0000u));
    }
  };
  for (int k = grp; k < sk; k += 16) {
    const int64_t row = kh * a.c.head_rows + start + k;
    const bool is_new = k == sk - 1;
    float x[8], z = 0.f;
    load(is_new ? new_w[0] : a.c.k + row * row_words<BITS>(), is_new ? new_m[0] : a.c.km + row * kGroups, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) z = fmaf(q[e], x[e], z);
    z += __shfl_xor(z, 1);
    z += __shfl_xor(z, 2);
    z += __shfl_xor(z, 4);
    z += __shfl_xor(z, 8);
    const float bias = a.bias ? a.bias[b * a.bias_bs + h * a.bias_hs + k] : 0.f;
    if (bias == -INFINITY) continue;             // hidden, whatever the row holds
    z = (z + bias) * a.scale_log2;
    asm("" : "+v"(z));   // rounded: contracted into z - m below, a bias near the lowest float leaves the rounding's rest
    load(is_new ? new_w[1] : a.c.v + row * row_words<BITS>(), is_new ? new_m[1] : a.c.vm + row * kGroups, x);
    const float mn = fmaxf(m, z), keep = m == -INFINITY ? 0.f : fast_exp2(m - mn);
    const float p = z == -INFINITY ? 0.f : fast_exp2(z - mn);   // (NaN where z is)
    l = l * keep + p;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = acc[e] * keep + (p == 0.f ? 0.f : p * x[e]);
    m = mn;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) part[grp][16 * e + j] = acc[e];
  if (j == 0) {
    pm[grp] = m;
    pl[grp] = l;
  }
  __syncthreads();
  if (threadIdx.x < kHeadDim) {
    float mm = -INFINITY, sum = 0.f, o = 0.f;
    for (int g = 0; g < 16; ++g) mm = fmaxf(mm, pm[g]);
    for (int g = 0; g < 16; ++g) {
      const float w = pm[g] == -INFINITY ? 0.f : fast_exp2(pm[g] - mm);
      sum += w * pl[g];
      o += w == 0.f ? 0.f : w * part[g][threadIdx.x];
    }
    // (a row whose scores are NaN: pl is NaN, and so is the output)
    const float y = sum == 0.f ? 0.f : o / sum;
    a.out[b * a.out_rs + (int64_t)h * kHeadDim + threadIdx.x] = __builtin_bit_cast(uint16_t, (__bf16)y);
  }
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
int check_rows(const char *what, const void *k, int64_t k_rs, int64_t k_hs, const void *v, int64_t v_rs, int64_t v_hs,
               int64_t n_rows) {
  TG_CHECK(k && v, "%s: null row pointer", what);
  TG_CHECK(n_rows >= 0 && (n_rows + 15) / 16 < (1ll << 31), "%s: bad row count", what);
  TG_CHECK(k_rs >= 0 && v_rs >= 0 && k_hs >= kHeadDim && v_hs >= kHeadDim && k_rs % 8 == 0 && v_rs % 8 == 0 &&
               k_hs % 8 == 0 && v_hs % 8 == 0,
           "%s: strides must be multiples of 8 elements, head strides at least 128", what);
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
  if (int e = check_rows("kv_quantize", k, k_row_stride, k_head_stride, v, v_row_stride, v_head_stride, n_rows)) return e;
  TG_CHECK(source_rows >= 0 && (src_rows || n_rows <= source_rows), "kv_quantize: more rows than the source holds");
  TG_CHECK(dst_rows || n_rows <= cache_rows, "kv_quantize: more rows than the cache holds");
  if (n_rows == 0) return 0;
  const RowSource a{static_cast<const bf16_t *>(k), static_cast<const bf16_t *>(v), k_row_stride, k_head_stride,
                    v_row_stride, v_head_stride, source_rows, src_rows, dst_rows};
  const dim3 grid((unsigned)((n_rows + 15) / 16), (unsigned)num_heads_k, 2), block(256);
  if (bits == 4) hipLaunchKernelGGL(kv_quantize_kernel<4>, grid, block, 0, stream, a, c, n_rows);
  else hipLaunchKernelGGL(kv_quantize_kernel<8>, grid, block, 0, stream, a, c, n_rows);
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
  if (int e = check_rows("kv_dequantize", k_out, k_row_stride, k_head_stride, v_out, v_row_stride, v_head_stride, n_rows))
    return e;
  TG_CHECK(rows || n_rows <= cache_rows, "kv_dequantize: more rows than the cache holds");
  if (n_rows == 0) return 0;
  const RowTarget a{static_cast<bf16_t *>(k_out), static_cast<bf16_t *>(v_out), k_row_stride, k_head_stride, v_row_stride,
                    v_head_stride, rows};
  const dim3 grid((unsigned)((n_rows + 15) / 16), (unsigned)num_heads_k, 2), block(256);
  if (bits == 4) hipLaunchKernelGGL(kv_dequantize_kernel<4>, grid, block, 0, stream, c, a, n_rows);
  else hipLaunchKernelGGL(kv_dequantize_kernel<8>, grid, block, 0, stream, c, a, n_rows);
  TG_HIP_CHECK(hipGetLastError());
  return 0;
}

extern "C" int64_t tg_decode_attention_quant_workspace_size(int32_t num_seqs, int32_t num_heads, int32_t num_heads_k,
                                                            int32_t max_seqlen_k) {
  return 0;
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
  TG_CHECK(num_seqs >= 0 && num_seqs < 65536 && max_seqlen_k >= 0, "%s: bad sequence count or length", what);
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
  const dim3 grid((unsigned)num_heads, (unsigned)num_seqs), block(256);
  if (bits == 4) hipLaunchKernelGGL(decode_attn_quant_kernel<4>, grid, block, 0, stream, a);
  else hipLaunchKernelGGL(decode_attn_quant_kernel<8>, grid, block, 0, stream, a);
  TG_HIP_CHECK(hipGetLastError());
  return 0;
}
