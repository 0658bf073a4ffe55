// The next token of rows of logits: temperature, top-k, top-p, min-p and one given random number per row.
//
// With w_i = exp((x_i - max x) / T) and the order "larger logits first, equal ones by index": S1 = the first k;
// S2 = the shortest beginning of S1 whose mass (sum of w) is at least top_p times S1's, one at least; S3 = those
// of S2 with w >= min_p, one at least; the token is the first of S3 whose cumulated mass exceeds u times S3's, and
// its log probability is ln(w / mass(S3)).  Every set is a beginning of the same order, so the row is not sorted:
//   * sample_hist_kernel, several workgroups per row: logits in units of y = cc x (cc = 8 log2 e, or 4 log2 e / T for
//     T < 0.5, times 2^fine where they lie close together) fall into bins of width one, 512 from the part's largest down.
//     A bin's count and the sum of its elements' e^t, t = (the fraction of y - 1/2) T-scaled, need no common maximum,
//     and as whole numbers (one 64-bit LDS addition per logit) no order of additions.  (How wide the bins are depends on what
//     a part holds: cut into other parts, a row's sums differ within their roundings.)  The workgroup that arrives last
//     merges the row's bins and finds those in which the ends of S1, S2, S3 and the token must lie;
//   * sample_pick_kernel collects the elements of these bins (up to 16384), and the last workgroup finds each end in its
//     bin: by 512 parts of the bin's interval of keys (value and index), again in the part that decides, and from 64
//     elements down by comparing them with one another.
// Rows of up to 2048 logits take one workgroup and one launch, which sorts them all.  Where the bins that decide hold
// more than 16384 (thousands of equal logits), or lie below the bins' reach, one workgroup finds the places digit by
// digit over the whole row.
// Double throughout: a row has so many borders between tokens that sums good to 2^-24 would move one row in a hundred
// across one; here a logit's part of its bin is rounded to 2^-34, those of the bins that decide to 2^-45.
// Measured, 151936 columns, both launches: 1 row 30 us, 4 rows 36, 8 rows of top_p 47, 64 rows 59 (their bytes once:
// 0.1, 0.4, 0.8 and 6.3).  Bound by latency for few rows (7 us until the last part has arrived, 8 to merge 4 KB per part
// and find the bins; then 6 to collect, and 3 to 11 for every end), and for many by the double arithmetic of the
// second pass over a part (30 instructions a logit: 12 of 64 rows' 30 us; a copy of the logits in LDS or of the
// bins for every fourth lane changed nothing).  Rows whose logits are all alike: 0.4 to 0.8 ms.
#include <algorithm>

#include "tg_common.h"
#include "../../include/tokengate_hip.h"

namespace tg {
namespace {

constexpr double kLog2e = 1.4426950408889634, kLn2 = 0.6931471805599453;
constexpr int kThreads = 1024;
constexpr int kBins = 512;
// Columns that one workgroup sorts: 1500 take 24 us (64 rows 26) and in two launches 22 (25) and the gap between them;
// 4000 take 41, and 25.
constexpr int kSort = 2048;
constexpr int kList = 16384;                     // elements that are collected
constexpr int kTiny = 64;                        // elements that are compared with one another
constexpr int kRowsPerLaunch = 256;

struct SampleArgs {
  const float *x;
  int64_t rs;
  int n;
  const float *u, *temperature, *top_p, *min_p;
  const int32_t *top_k;
  int64_t *token;
  float *logprob;
};

// One workgroup's bins: [f, f + 1) of y for f in top - 511 .. top, at f mod 512
struct Part {
  double top;
  double tail;                                   // mass below the bins, in units of 2^(top / q)
  uint32_t best, least;                          // order bits of the largest logit, and of the smallest within reach
  uint32_t fine, pad;                            // Row's
  uint64_t hist[kBins];                          // count << 48 | sum of (e^t - 0.9) 2^33
};
// What the first launch leaves for the second, per row; bin j: y in [top - j, top - j + 1)
struct State {
  double top, mass;                              // mass of the whole row, in units of 2^(top / q), as all
  uint64_t mask[kBins / 64];                     // bins to collect
  uint32_t best, slow, m_lo, m_hi;               // bins that may hold min_p's end
  uint32_t fine, pad;                            // Row's
  double upto_mass[kBins];                       // up to and with bin j
  uint32_t upto_count[kBins];
};
enum : uint32_t { kUsual, kSlow, kDone };        // State::slow
struct Counters {
  uint32_t hist, pick, listed, pad;              // zero between launches
};

template <typename T>
__device__ __forceinline__ void st_agent(T *p, T v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <typename T>
__device__ __forceinline__ T ld_agent(const T *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ uint64_t bits_of(double x) { return __builtin_bit_cast(uint64_t, x); }
__device__ __forceinline__ double double_of(uint64_t x) { return __builtin_bit_cast(double, x); }

// Order-preserving bits of a float: larger floats, larger numbers; NaN is -inf, -0 is 0.
__device__ __forceinline__ uint32_t order_bits(float x) {
  x = x != x ? -INFINITY : x + 0.f;
  const uint32_t b = __builtin_bit_cast(uint32_t, x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float order_float(uint32_t o) { return u32_as_f32(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
constexpr uint32_t kNone = 0x007FFFFFu, kMost = 0xFF800000u;   // order bits of -inf, of +inf

// 2^z, to 2^-46, for z of up to some hundreds (the exponential's series over half an octave either way)
__device__ __forceinline__ double exp2_of(double z) {
  z = fmax(z, -1100.0);
  const double n = rint(z), t = (z - n) * kLn2;
  double p = 1.0 / 39916800;
  p = fma(p, t, 1.0 / 3628800);
  p = fma(p, t, 1.0 / 362880);
  p = fma(p, t, 1.0 / 40320);
  p = fma(p, t, 1.0 / 5040);
  p = fma(p, t, 1.0 / 720);
  p = fma(p, t, 1.0 / 120);
  p = fma(p, t, 1.0 / 24);
  p = fma(p, t, 1.0 / 6);
  p = fma(p, t, 0.5);
  p = fma(p, t, 1.0);
  p = fma(p, t, 1.0);
  return ldexp(p, (int)n);
}

// A row's settings.  Bins per octave of w: q; y = cc x.  Both are 2^fine times what lets the bins reach 64 octaves (at
// T <= 1) down: with 2^fine as large as the spread of the logits allows, a bin of a flat row holds no more than one of a
// steep row.
constexpr int kFinest = 12;
struct Row {
  double q, per_q, cc, per_cc;
  bool greedy;
  __device__ Row(const SampleArgs &a, int b) {
    const float t = a.temperature ? a.temperature[b] : 1.f;
    greedy = !(t > 0.f);
    const double temp = greedy ? 1.0 : (double)t;
    q = fmax(4.0, 8.0 * temp);
    per_q = 1.0 / q;
    cc = temp >= 0.5 ? 8.0 * kLog2e : 4.0 * kLog2e / temp;
    per_cc = temp >= 0.5 ? 0.125 * kLn2 : 0.25 * kLn2 * temp;
  }
  // the bins' reach, in logits; the finest bins (of a row of fine 0) that reach from most down to least
  __device__ float reach() const { return (float)(kBins * per_cc); }
  __device__ int finest(float most, float least) const {
    const double span = ((double)most - (double)least) * cc;
    if (!(span >= 0.0)) return 0;                // (nothing is within reach, or both are infinite)
    static_assert(kBins == 512, "9 bits");
    const int bits = span > 0.0 ? __builtin_amdgcn_frexp_exp(span) : -64;   // span < 2^bits
    return max(0, min(kFinest, 9 - bits - (ldexp(span, 9 - bits) < kBins - 2 ? 0 : 1)));
  }
  __device__ Row(const Row &coarse, int fine) : Row(coarse) {
    q = ldexp(q, fine);
    per_q = ldexp(per_q, -fine);
    cc = ldexp(cc, fine);
    per_cc = ldexp(per_cc, -fine);
  }
  // (+inf: so far above every finite one that those weigh nothing)
  __device__ double y(float x) const { return x == INFINITY ? 0x1p1000 : (double)x * cc; }
  __device__ double weight(double y, double top) const { return exp2_of((y - top) * per_q); }
  __device__ double weight_of(float x, double top) const { return x == -INFINITY ? 0.0 : weight(y(x), top); }
  // order bits of the first value, from below, of a bin not under low (above: not of low either)
  __device__ uint32_t first(double low, bool above) const {
    auto in = [&](uint32_t o) { return above ? floor(y(order_float(o))) > low : y(order_float(o)) >= low; };
    uint32_t o = order_bits((float)((above ? low + 1.0 : low) * per_cc));   // (off by its roundings)
    while (o > kNone && in(o - 1)) --o;
    while (o <= kMost && !in(o)) ++o;
    return o;
  }
  // whether x has less than least times the largest logit's weight
  __device__ bool under(float x, float best, float least) const {
    return x != best && (x == -INFINITY || weight(y(x), y(best)) < fmin((double)least, 1.0));
  }
};
// The other settings: top_k as 0 where it leaves everything, 1 where the row is greedy
struct Settings {
  int k;
  float tp, mp;
  double u;
  __device__ Settings(const SampleArgs &a, int b, bool greedy) {
    const int top_k = a.top_k ? a.top_k[b] : 0;
    const float top_p = a.top_p ? a.top_p[b] : 1.f, min_p = a.min_p ? a.min_p[b] : 0.f, u0 = a.u[b];
    k = greedy ? 1 : top_k > 0 && top_k < a.n ? top_k : 0;
    tp = greedy ? 1.f : top_p;
    mp = greedy ? 0.f : min_p;
    u = fmin(fmax((double)u0, 0.0), 1.0 - 0x1p-30);
  }
};
// u[b]; a one, which a rounded number may be, takes the last element of a mass of more than 2^-30
__device__ __forceinline__ double draw(const SampleArgs &a, int b) { return fmin(fmax((double)a.u[b], 0.0), 1.0 - 0x1p-30); }

// What an element adds to its bin: 1 << 48 | (e^t - 0.9) 2^33 for |t| <= 0.087, e^t to 2^-43.  The sum's whole number
// comes out of the fraction bits of 2^52 + it.
constexpr double kHistBase = 0.9, kHistUnit = 0x1p33;
constexpr int kMostChunk = 0xffff;               // elements whose sums and counts the fields hold
__device__ __forceinline__ double exp_small(double t) {
  double p = 1.0 / 5040;
  p = fma(p, t, 1.0 / 720);
  p = fma(p, t, 1.0 / 120);
  p = fma(p, t, 1.0 / 24);
  p = fma(p, t, 1.0 / 6);
  p = fma(p, t, 0.5);
  p = fma(p, t, 1.0);
  return fma(p, t, 1.0);
}
__device__ __forceinline__ uint64_t hist_add(double t) {
  return bits_of(fma(exp_small(t), kHistUnit, 0x1p52 - kHistBase * kHistUnit)) - (bits_of(0x1p52) - (1ull << 48));
}

// Mass of a bin, in units of 2^(its middle / q)
__device__ __forceinline__ double hist_mass(uint64_t h) {
  return kHistBase * (double)(uint32_t)(h >> 48) + (double)(h & 0xffffffffffffull) * (1.0 / kHistUnit);
}

template <int CTRL>
__device__ __forceinline__ uint64_t dpp(uint64_t x) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp((int)(uint32_t)x, (int)(uint32_t)x, CTRL, 0xf, 0xf, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp((int)(uint32_t)(x >> 32), (int)(uint32_t)(x >> 32), CTRL, 0xf, 0xf, true);
  return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
  auto step = [](uint64_t x, uint64_t y) { return x > y ? x : y; };
  v = step(v, dpp<0xB1>(v));     // quad_perm 1 0 3 2
  v = step(v, dpp<0x4E>(v));     // quad_perm 2 3 0 1
  v = step(v, dpp<0x141>(v));    // row_half_mirror
  v = step(v, dpp<0x140>(v));    // row_mirror
  auto p = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
  auto q = __builtin_amdgcn_permlane16_swap((uint32_t)(v >> 32), (uint32_t)(v >> 32), false, false);
  v = step((uint64_t)q[0] << 32 | p[0], (uint64_t)q[1] << 32 | p[1]);
  p = __builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false);
  q = __builtin_amdgcn_permlane32_swap((uint32_t)(v >> 32), (uint32_t)(v >> 32), false, false);
  return step((uint64_t)q[0] << 32 | p[0], (uint64_t)q[1] << 32 | p[1]);
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  auto step = [](uint32_t x, uint32_t y) { return x > y ? x : y; };
  v = step(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0xB1, 0xf, 0xf, true));    // quad_perm 1 0 3 2
  v = step(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x4E, 0xf, 0xf, true));    // quad_perm 2 3 0 1
  v = step(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x141, 0xf, 0xf, true));   // row_half_mirror
  v = step(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x140, 0xf, 0xf, true));   // row_mirror
  const auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = step(p[0], p[1]);
  const auto q = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return step(q[0], q[1]);
}
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t *tmp) {   // tmp: 16 words
  const int tid = threadIdx.x;
  v = wave_max(v);
  __syncthreads();
  if ((tid & 63) == 0) tmp[tid >> 6] = v;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) v = v > tmp[i] ? v : tmp[i];
  return v;
}
// Sums over the lanes up to this one, without the LDS crossbar
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t scan_step(uint32_t x) {
  return x + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double scan_step(double x) {
  const uint64_t u = bits_of(x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xf, false);
  return x + double_of((uint64_t)hi << 32 | lo);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t scan_step(uint64_t u) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xf, false);
  return u + ((uint64_t)hi << 32 | lo);
}
template <typename T>
__device__ __forceinline__ T wave_scan(T x) {
  x = scan_step<0x111, 0xf>(x);   // row_shr 1, 2, 4, 8
  x = scan_step<0x112, 0xf>(x);
  x = scan_step<0x114, 0xf>(x);
  x = scan_step<0x118, 0xf>(x);
  x = scan_step<0x142, 0xa>(x);   // row_bcast 15: the first row's sum to the second, the third's to the fourth
  return scan_step<0x143, 0xc>(x);   // row_bcast 31: the first half's to the second
}
template <typename T>
__device__ __forceinline__ T row_scan(T x) {     // of 16 lanes
  x = scan_step<0x111, 0xf>(x);
  x = scan_step<0x112, 0xf>(x);
  x = scan_step<0x114, 0xf>(x);
  return scan_step<0x118, 0xf>(x);
}
__device__ __forceinline__ uint32_t read_lane(uint32_t x, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)x, lane); }
__device__ __forceinline__ uint64_t read_lane(uint64_t x, int lane) {
  return (uint64_t)read_lane((uint32_t)(x >> 32), lane) << 32 | read_lane((uint32_t)x, lane);
}
__device__ __forceinline__ double read_lane(double x, int lane) { return double_of(read_lane(bits_of(x), lane)); }
// Sums over the threads up to this one; total: over all.  tmp: 16 of T.  Whole numbers: every wave adds the waves' sums
// up for itself, one per lane.
template <typename T>
__device__ __forceinline__ T block_scan(T v, T *tmp, T &total) {
  const int lane = threadIdx.x & 63, wave = wave_id();
  v = wave_scan(v);
  __syncthreads();
  if (lane == 63) tmp[wave] = v;
  __syncthreads();
  const T s = row_scan(tmp[lane & 15]);
  total = read_lane(s, 15);
  return v + (wave ? read_lane(s, wave - 1) : T(0));
}
// Three at once: of u and v the sums up to this thread, of w the sum of all; total: u's of all.
__device__ __forceinline__ void block_scan3(uint64_t &u, uint32_t &v, double &w, uint64_t *tmp_u, uint32_t *tmp_v, double *tmp_w,
                                            uint64_t &total) {
  const int lane = threadIdx.x & 63, wave = wave_id();
  u = wave_scan(u);
  v = wave_scan(v);
  w = wave_scan(w);
  __syncthreads();
  if (lane == 63) {
    tmp_u[wave] = u;
    tmp_v[wave] = v;
    tmp_w[wave] = w;
  }
  __syncthreads();
  const uint64_t su = row_scan(tmp_u[lane & 15]);
  const double sw = row_scan(tmp_w[lane & 15]);
  const uint32_t sv = row_scan(tmp_v[lane & 15]);
  total = read_lane(su, 15);
  w = read_lane(sw, 15);
  if (wave) {
    u += read_lane(su, wave - 1);
    v += read_lane(sv, wave - 1);
  }
}
// Doubles, for rows that are sorted
__device__ __forceinline__ double block_scan(double v, double *tmp, double &total) {
  const int lane = threadIdx.x & 63, wave = wave_id();
  v = wave_scan(v);
  __syncthreads();
  if (lane == 63) tmp[wave] = v;
  __syncthreads();
  double before = 0.0;
  total = 0.0;
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) {
    const double s = tmp[i];
    before += i < wave ? s : 0.0;
    total += s;
  }
  return v + before;
}

// ---- the elements of one list, in order ----------------------------------------------------------------
// list: n <= kSort entries (~order bits) << 32 | index; ascending is the row's order.
__device__ __forceinline__ int sort_list(uint64_t *list, int n) {
  const int tid = threadIdx.x;
  int size = 64;
  while (size < n) size *= 2;
  for (int i = n + tid; i < size; i += kThreads) list[i] = ~0ull;
  for (int k = 2; k <= size; k *= 2)
    for (int j = k / 2; j >= 1; j /= 2) {
      __syncthreads();
      for (int i = tid; i < size / 2; i += kThreads) {
        const int lo = 2 * i - (i & (j - 1)), hi = lo + j;
        const uint64_t a = list[lo], b = list[hi];
        if ((a > b) == ((lo & k) == 0)) {
          list[lo] = b;
          list[hi] = a;
        }
      }
    }
  __syncthreads();
  return size;
}

__device__ __forceinline__ float list_value(uint64_t entry) { return order_float(~(uint32_t)(entry >> 32)); }

// ---- rows of up to kSort logits --------------------------------------------------------------------------
__global__ __launch_bounds__(kThreads) void sample_small_kernel(SampleArgs a) {
  constexpr int kPer = kSort / kThreads;
  __shared__ uint64_t list[kSort];
  __shared__ uint32_t place_s[3];                // ends of S2 and of min_p, the token
  __shared__ double scan[16], mass_s[2];
  const int b = blockIdx.x, tid = threadIdx.x, n = a.n;
  const float *x = a.x + b * a.rs;
  const Row row(a, b);
  for (int i = tid; i < n; i += kThreads) list[i] = (uint64_t)~order_bits(x[i]) << 32 | (uint32_t)i;
  const int per = (sort_list(list, n) + kThreads - 1) / kThreads;   // elements of a thread, in order
  const float best = list_value(list[0]);
  if (row.greedy || best == -INFINITY) {
    if (tid == 0) {
      a.token[b] = (uint32_t)list[0];
      if (a.logprob) a.logprob[b] = 0.f;
    }
    return;
  }
  const double top = row.y(best);
  const int k = a.top_k && a.top_k[b] > 0 ? min(a.top_k[b], n) : n;
  double wt[kPer], cum[kPer], sum = 0.0, total;
#pragma unroll
  for (int r = 0; r < kPer; ++r) {
    const int i = tid * per + r;
    wt[r] = 0.0;
    if (r < per && i < k) wt[r] = row.weight_of(list_value(list[i]), top);   // S1
    sum += wt[r];
  }
  double before = block_scan(sum, scan, total) - sum;
#pragma unroll
  for (int r = 0; r < kPer; ++r) cum[r] = before += wt[r];
  auto each = [&](auto f) {
#pragma unroll
    for (int r = 0; r < kPer; ++r)
      if (r < per && tid * per + r < k) f(tid * per + r, r);
  };
  if (tid < 3) place_s[tid] = k - 1;
  if (tid < 2) mass_s[tid] = total;
  __syncthreads();
  const float tp = a.top_p ? a.top_p[b] : 1.f, mp = a.min_p ? a.min_p[b] : 0.f;
  each([&](int i, int r) {
    if (tp < 1.f && cum[r] >= (double)fmaxf(tp, 0.f) * total) atomicMin(&place_s[0], (uint32_t)i);
    if (mp > 0.f && i + 1 < k && row.under(list_value(list[i + 1]), best, mp)) atomicMin(&place_s[1], (uint32_t)i);
  });
  __syncthreads();
  const uint32_t end = min(place_s[0], place_s[1]);   // S3's last
  each([&](int i, int r) {
    if ((uint32_t)i == end) mass_s[0] = cum[r];
  });
  __syncthreads();
  const double s3 = mass_s[0], target = draw(a, b) * s3;
  each([&](int i, int r) {
    if (cum[r] > target && wt[r] > 0.0) atomicMin(&place_s[2], (uint32_t)i);
  });
  __syncthreads();
  const uint32_t at = min(place_s[2], end);
  each([&](int i, int r) {
    if ((uint32_t)i == at) {
      a.token[b] = (uint32_t)list[i];
      if (a.logprob) a.logprob[b] = (float)log(wt[r] / s3);
    }
  });
}

// ---- longer rows -------------------------------------------------------------------------------------------
struct SampleWork {
  Counters *counters;                            // per row
  State *states;
  uint64_t *lists;                               // kList per row
  Part *parts;                                   // gridDim.x per row
};

__device__ __forceinline__ int slot_of(double f) { return (int)(f - kBins * floor(f / kBins)); }

// A workgroup's logits: x[first], x[first + kThreads] and so on, while below end
struct Share {
  int first, end;
  __device__ Share(int n) {
    const int chunk = (n + gridDim.x - 1) / gridDim.x;
    first = blockIdx.x * chunk + threadIdx.x;
    end = min(n, (int)(blockIdx.x + 1) * chunk);
  }
  // f(value, its number), four loads at a time
  template <typename F>
  __device__ __forceinline__ void each(const float *x, F f) const {
    int i = first, k = 0;
    for (; i + 3 * kThreads < end; i += 4 * kThreads, k += 4) {
      float v[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = x[i + r * kThreads];
#pragma unroll
      for (int r = 0; r < 4; ++r) f(v[r], k + r);
    }
    for (; i < end; i += kThreads, ++k) f(x[i], k);
  }
};

__global__ __launch_bounds__(kThreads, 4) void sample_hist_kernel(SampleArgs a, SampleWork ws) {
  const int b = blockIdx.y, g = blockIdx.x, parts = gridDim.x, tid = threadIdx.x;
  const float *x = a.x + b * a.rs;
  __shared__ uint64_t hist[kBins];
  __shared__ uint32_t tmp[16];
  __shared__ double tail_s[16];
  __shared__ uint32_t last_s;
  const Share share(a.n);
  float most = -INFINITY, least = INFINITY;      // (maxima of pairs drop NaN; -inf has no weight)
  const Row coarse(a, b);
  const Settings set(a, b, coarse.greedy);       // (for the last workgroup: here their loads take no time of their own)
  const float reach = coarse.reach();
  share.each(x, [&](float v, int) {
    most = fmaxf(most, v);
    least = v > -INFINITY ? fminf(least, v) : least;
  });
  if (tid < kBins) hist[tid] = 0;
  uint32_t best = block_max(order_bits(most), tmp);   // (its barriers cover the bins)
  uint32_t low_bits = ~block_max(~order_bits(least), tmp);
  const float end = order_float(best) - reach;
  // the least of what lies within reach of the largest: what lies below, as a finite mask does, may not count, and takes
  // another pass (which logits are within reach is known only when the largest is)
  if (!(order_float(low_bits) > end)) {
    least = INFINITY;
    bool any = false;
    share.each(x, [&](float v, int) {
      const bool near = v > end;
      least = near ? fminf(least, v) : least;
      any |= near;
    });
    low_bits = ~block_max(any ? ~order_bits(least) : 0u, tmp);
  }
  const int fine = low_bits == ~0u ? 0 : coarse.finest(order_float(best), order_float(low_bits));
  const Row row(coarse, fine);
  const double top = best == kNone ? 0.0 : floor(row.y(order_float(best)));
  double tail_mine = 0.0;                        // (a double: weights of any size, in an order that the launch gives)
  const double scale = kLn2 * row.per_q;
  const int top_slot = slot_of(top);
  share.each(x, [&](float v, int) {
    if (!(v > -INFINITY)) return;
    const double y = row.y(v), f = floor(y), j = top - f;
    if (j < kBins) {
      atomicAdd((unsigned long long *)&hist[(top_slot - (int)j) & (kBins - 1)], (unsigned long long)hist_add((y - f - 0.5) * scale));
    } else {
      const double w = row.weight(y, top);
      if (w > 0x1p-72) tail_mine += w;           // (2^18 of less: 2^-54)
    }
  });
  tail_mine = wave_scan(tail_mine);
  if ((tid & 63) == 63) tail_s[wave_id()] = tail_mine;
  __syncthreads();
  Part *const part = ws.parts + (int64_t)b * parts;
  if (tid < kBins) st_agent(&part[g].hist[tid], hist[tid]);
  const double tail_part = read_lane(row_scan(tail_s[tid & 15]), 15);
  if (tid == 0) {
    st_agent((uint64_t *)&part[g].top, bits_of(top));
    st_agent((uint64_t *)&part[g].tail, bits_of(tail_part));
    st_agent((uint64_t *)&part[g].best, (uint64_t)low_bits << 32 | best);
    st_agent(&part[g].fine, (uint32_t)fine);
  }
  wait_all_mem();
  __syncthreads();
  if (tid == 0)
    last_s = __hip_atomic_fetch_add(&ws.counters[b].hist, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)parts - 1u;
  __syncthreads();
  if (!last_s) return;

  // ---- the row's bins ----
  __shared__ double mass_s[kBins];
  __shared__ uint64_t scan_m[16];
  __shared__ double scan_t[16];
  __shared__ uint64_t sums[2][kBins];
  __shared__ uint32_t counts[2][kBins], count_s[kBins], scan_u[16];
  __shared__ int first_s[4];
  // thread: one slot of every other part, requested before what they are merged by is formed
  constexpr int kAhead = 10;
  const int slot = tid & (kBins - 1), half = wave_id() / (kBins / 64);
  uint64_t h[kAhead];
  auto request = [&](int i0) {
#pragma unroll
    for (int r = 0; r < kAhead; ++r) h[r] = ld_agent(&part[min(i0 + 2 * r, parts - 1)].hist[slot]);
  };
  // every wave: a part per lane (at most 64)
  const int lane = tid & 63;
  double part_top = 0.0;
  uint32_t part_best = kNone, part_least = ~0u, part_fine = kFinest;
  if (lane < parts) {
    part_top = double_of(ld_agent((const uint64_t *)&part[lane].top));
    const uint64_t ends = ld_agent((const uint64_t *)&part[lane].best);
    part_best = (uint32_t)ends;
    part_least = (uint32_t)(ends >> 32);
    part_fine = ld_agent(&part[lane].fine);
  }
  request(half);
  (&sums[0][0])[tid] = 0;
  (&counts[0][0])[tid] = 0;
  best = wave_max(part_best);
  State *const st = ws.states + b;
  if (best == kNone) {                           // nothing but -inf
    if (tid == 0) {
      a.token[b] = 0;
      if (a.logprob) a.logprob[b] = 0.f;
      st->slow = kDone;
      st_agent(&ws.counters[b].hist, 0u);
    }
    return;
  }
  // the finest bins that the row's span and every part's allow
  const bool near_top = part_best != kNone && order_float(part_least) > order_float(best) - reach;
  const uint32_t least_row = ~wave_max(near_top ? ~part_least : 0u);
  int fine_row = kFinest - (int)wave_max(part_best == kNone ? 0u : kFinest - part_fine);
  fine_row = least_row == ~0u ? 0 : min(fine_row, coarse.finest(order_float(best), order_float(least_row)));
  const Row whole(coarse, fine_row);
  const double gtop = floor(whole.y(order_float(best))), scale_row = kLn2 * whole.per_q;
  const int part_finer = part_best == kNone ? 0 : (int)part_fine - fine_row, part_slot = slot_of(part_top);
  // its first bin lies so many of its bins below the row's first; past 2^29 in two numbers, part_beyond of the row's bins and
  // the rest (at high temperatures no distance is so large that it weighs nothing by itself)
  const double depth = ldexp(gtop, part_finer) - part_top;
  const double part_beyond = depth > 0x1p29 ? floor(ldexp(depth - 0x1p29, -part_finer)) : 0.0;
  const int part_depth = depth > 0x1p29 ? (int)fmin(fmax(depth - ldexp(part_beyond, part_finer), 0x1p28), 0x1p30) : (int)depth;
  __syncthreads();                               // (the sums are cleared)
  uint64_t sum = 0;
  uint32_t count = 0;
  double tail = 0.0;
  for (int i0 = half; i0 < parts; i0 += 2 * kAhead) {
    if (i0 > half) request(i0);
#pragma unroll
    for (int r = 0; r < kAhead; ++r) {
      const int i = i0 + 2 * r;
      if (i >= parts) continue;
      const int finer = __builtin_amdgcn_readlane(part_finer, i),   // (by all lanes, ahead of what only some do)
                d = __builtin_amdgcn_readlane(part_depth, i) + ((__builtin_amdgcn_readlane(part_slot, i) - slot) & (kBins - 1)),
                below = (d + (1 << finer) - 1) >> finer;
      const double beyond = read_lane(part_beyond, i);
      if (h[r] == 0) continue;
      const uint32_t c = (uint32_t)(h[r] >> 48);
      uint64_t s = h[r] & 0xffffffffffffull;
      if (finer) {                               // 2^finer of the part's bins are one of the row's: from one middle to another's
        const double off = ldexp((double)((below << finer) - d) + 0.5, -finer) - 0.5;
        s = (uint64_t)((hist_mass(h[r]) * exp_small(off * scale_row) - kHistBase * (double)c) * kHistUnit + 0.5);
      }
      if (below >= kBins) {
        tail += exp2_of((0.5 - below - beyond) * whole.per_q) * hist_mass((uint64_t)c << 48 | s);
      } else if (finer) {
        atomicAdd((unsigned long long *)&sums[half][below], (unsigned long long)s);
        atomicAdd(&counts[half][below], c);
      } else {
        count += c;
        sum += s;
      }
    }
  }
  if (tid < parts && part_best != kNone)
    tail += exp2_of((ldexp(part_top, -part_finer) - gtop) * whole.per_q) * double_of(ld_agent((const uint64_t *)&part[tid].tail));
  __syncthreads();
  {
    const int j = (slot_of(gtop) - slot) & (kBins - 1);
    sums[half][j] += sum;
    counts[half][j] += count;
  }
  __syncthreads();
  const int j = slot;                            // from here on a bin
  double m = 0.0;
  count = 0;
  if (half == 0) {
    count = counts[0][j] + counts[1][j];
    m = exp2_of((0.5 - j) * whole.per_q) * (kHistBase * (double)count + (double)(sums[0][j] + sums[1][j]) * (1.0 / kHistUnit));
  }
  // (as whole numbers: no bin's sum is less than the one's before it, as roundings could make it)
  uint32_t upto_count = count;
  uint64_t upto_u = (uint64_t)(m * 0x1p44 + 0.5), in_bins_u;
  double tail_all = tail;
  block_scan3(upto_u, upto_count, tail_all, scan_m, scan_u, scan_t, in_bins_u);
  const double upto = (double)upto_u * 0x1p-44;
  const double in_bins = (double)in_bins_u * 0x1p-44, mass = in_bins + tail_all;
  const bool tail_counts = tail_all > 0x1p-42 * mass;
  if (half == 0) {
    mass_s[j] = upto;
    count_s[j] = upto_count;
  }
  if (tid < 4) first_s[tid] = kBins;
  __syncthreads();
  auto first_mass = [&](int slot, double target) {   // the first bin up to which the mass reaches target
    if (half == 0 && upto >= target && (j == 0 || mass_s[j - 1] < target)) first_s[slot] = j;
  };
  constexpr double kEps = 0x1p-34;
  const uint32_t k = (uint32_t)set.k;
  const float tp = set.tp, mp = set.mp;
  bool slow = false;
  if (half == 0 && k && upto_count >= k && (j == 0 || count_s[j - 1] < k)) first_s[0] = j;
  __syncthreads();
  const int k_bin = k ? first_s[0] : kBins;
  double lo = mass, hi = mass;                   // bounds of S1's mass, then of S3's
  if (k && k_bin < kBins) {
    lo = k_bin ? mass_s[k_bin - 1] : 0.0;
    hi = mass_s[k_bin];
  } else if (k) {
    lo = in_bins;
    slow |= tail_counts;
  }
  const double p = fmax((double)tp, 0.0);
  if (tp < 1.f) {
    first_mass(1, p * lo * (1.0 - kEps));
    first_mass(2, p * hi * (1.0 + kEps));
  }
  __syncthreads();
  int p_lo = kBins, p_hi = kBins, m_lo = kBins, m_hi = kBins;
  if (tp < 1.f) {
    p_lo = min(first_s[1], kBins - 1);
    p_hi = min(first_s[2], kBins - 1);
    slow |= tail_counts && first_s[2] == kBins;
    lo = fmin(lo, p_lo ? mass_s[p_lo - 1] : 0.0);
    hi = fmin(hi, mass_s[p_hi]);
  }
  if (mp > 0.f) {
    const double thr = whole.y(order_float(best)) + whole.q * log2(fmin((double)mp, 1.0)), d0 = gtop - floor(thr + 1e-6),
                 d1 = gtop - floor(thr - 1e-6);
    m_lo = d0 < 0.0 ? 0 : d0 < kBins ? (int)d0 : kBins;
    m_hi = d1 < 0.0 ? 0 : d1 < kBins ? (int)d1 : kBins;
    slow |= tail_counts && m_hi == kBins;
    if (m_lo < kBins) lo = fmin(lo, m_lo ? mass_s[m_lo - 1] : 0.0);
    if (m_hi < kBins) hi = fmin(hi, mass_s[m_hi]);
  }
  const double u = set.u;
  __syncthreads();
  if (tid < 4) first_s[tid] = kBins;
  __syncthreads();
  first_mass(0, u * lo * (1.0 - kEps));
  first_mass(1, u * hi * (1.0 + kEps));
  __syncthreads();
  int t_lo = min(first_s[0], kBins - 1), t_hi = min(first_s[1], kBins - 1);
  slow |= tail_counts && first_s[1] == kBins;
  if (row.greedy) t_lo = t_hi = 0;
  auto in = [&](int lo_, int hi_) { return j >= lo_ && j <= hi_; };
  const bool wanted = half == 0 && (j == k_bin || (tp < 1.f && in(p_lo, p_hi)) || (mp > 0.f && in(m_lo, min(m_hi, kBins - 1))) || in(t_lo, t_hi));
  uint32_t listed;
  block_scan(wanted ? count : 0u, scan_u, listed);
  slow |= listed > kList;
  const uint64_t bits = __builtin_amdgcn_ballot_w64(wanted && !slow);
  if (half == 0) {
    st->upto_count[j] = upto_count;
    st->upto_mass[j] = upto;
    if ((tid & 63) == 0) st->mask[j >> 6] = bits;
  }
  if (tid == 0) {
    st->top = gtop;
    st->mass = mass;
    st->best = best;
    st->slow = slow ? kSlow : kUsual;
    st->m_lo = (uint32_t)m_lo;
    st->m_hi = (uint32_t)m_hi;
    st->fine = (uint32_t)fine_row;
    st_agent(&ws.counters[b].hist, 0u);
  }
}

// ---- a flat row: the places found digit by digit ----------------------------------------------------------
// A place in the order: the elements above `key`, and the first `ties` of those equal to it.
struct Place {
  uint32_t key;
  uint32_t ties;
  uint64_t above;   // count or mass of the elements above key
};
// Masses as whole numbers, `unit` the largest weight's: as large as the row's mass, at most row_mass of that weight,
// allows (2^18 roundings of 2^-62 of the whole).
__device__ void slow_row(const SampleArgs &a, int b, double row_mass) {
  const double unit = ldexp(1.0, 61 - __builtin_amdgcn_frexp_exp(row_mass));
  const int tid = threadIdx.x;
  const float *x = a.x + b * a.rs;
  __shared__ uint64_t hist[256], red[16];
  __shared__ uint32_t found;
  __shared__ uint64_t above_s;
  auto reduce_max = [&](uint32_t v) {
    for (int o = 32; o; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o));
    if ((tid & 63) == 0) red[tid >> 6] = v;
    __syncthreads();
    for (int i = 0; i < 16; ++i) v = max(v, (uint32_t)red[i]);
    __syncthreads();
    return v;
  };
  auto each = [&](auto f) {                      // f(order bits), eight loads at a time
    for (int i0 = tid; i0 < a.n; i0 += 8 * kThreads) {
      float v[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) v[r] = x[min(i0 + r * kThreads, a.n - 1)];
#pragma unroll 1
      for (int r = 0; r < 8; ++r) {
        float w = v[0];                          // (shifted down: no indexed registers)
#pragma unroll
        for (int q = 0; q < 7; ++q) v[q] = v[q + 1];
        if (i0 + r * kThreads < a.n) f(order_bits(w));
      }
    }
  };
  uint32_t best = 0;
  each([&](uint32_t key) { best = max(best, key); });
  best = reduce_max(best);
  const float top = order_float(best);
  const float temp = a.temperature ? a.temperature[b] : 1.f;
  const bool greedy = !(temp > 0.f) || top == -INFINITY;
  const double scale = greedy ? 1.0 : kLog2e / temp;
  auto weight = [&](float x) { return x == top ? 1.0 : exp2_of(((double)x - (double)top) * scale); };   // (both may be infinite)
  auto mass = [&](uint32_t key) { return (uint64_t)(weight(order_float(key)) * unit + 0.5); };
  // The first place at which the sum of value(key) over the elements up to it reaches target (> 0).
  auto find = [&](uint64_t target, bool by_mass) {
    uint32_t prefix = 0;
    uint64_t above = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      each([&](uint32_t key) {
        if (shift != 24 && (key >> (shift + 8)) != (prefix >> (shift + 8))) return;
        uint64_t m = by_mass ? mass(key) : 1;
        const uint32_t first = (uint32_t)__builtin_amdgcn_readfirstlane((int)key);
        const uint64_t here = __ballot(1), same = __ballot(key == first);
        if (here == same) {                      // (many equal ones make such a row: one addition for all of a wave's)
          m *= (uint64_t)__popcll(here);
          if ((tid & 63) != __builtin_ctzll(here)) return;
        }
        atomicAdd((unsigned long long *)&hist[(key >> shift) & 255], (unsigned long long)m);
      });
      __syncthreads();
      if (tid == 0) {
        uint64_t c = above;
        int d = 255;
        for (; d > 0 && c + hist[d] < target; --d) c += hist[d];
        found = prefix | ((uint32_t)d << shift);
        above_s = c;
      }
      __syncthreads();
      prefix = found;
      above = above_s;
      __syncthreads();
    }
    const uint64_t one = by_mass ? mass(prefix) : 1;
    const uint64_t need = target > above ? target - above : 1;
    return Place{prefix, (uint32_t)(one ? (need + one - 1) / one : 1), above};
  };
  auto sum_mass = [&](Place p) {                 // of the elements of a place's beginning
    uint64_t s = 0;
    each([&](uint32_t key) {
      if (key > p.key) s += mass(key);
    });
    for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
    if ((tid & 63) == 0) red[tid >> 6] = s;
    __syncthreads();
    s = 0;
    for (int i = 0; i < 16; ++i) s += red[i];
    __syncthreads();
    return s + p.ties * mass(p.key);
  };
  auto index_of = [&](Place p) {                 // the ties-th element equal to key, by index
    uint32_t seen = 0;
    for (int i0 = 0; i0 < a.n; i0 += kThreads) {
      const int i = i0 + tid;
      const bool eq = i < a.n && order_bits(x[i]) == p.key;
      const uint64_t m = __ballot(eq);
      if ((tid & 63) == 0) red[tid >> 6] = __popcll(m);
      __syncthreads();
      uint32_t before = seen, total = seen;
      for (int w = 0; w < 16; ++w) {
        if (w < (tid >> 6)) before += red[w];
        total += red[w];
      }
      const uint32_t rank = before + __popcll(m & ((1ull << (tid & 63)) - 1));
      if (eq && rank == p.ties - 1) found = i;
      __syncthreads();
      if (total >= p.ties) return found;
      seen = total;
    }
    return 0u;
  };
  if (greedy) {
    const uint32_t i = index_of(Place{best, 1, 0});
    if (tid == 0) {
      a.token[b] = i;
      if (a.logprob) a.logprob[b] = 0.f;
    }
    return;
  }
  Place last{0, (uint32_t)a.n, 0};               // the end of the set: at first every element
  uint64_t total;
  const int k = a.top_k ? a.top_k[b] : 0;
  if (k > 0 && k < a.n) last = find((uint64_t)k, false);
  total = sum_mass(last);
  const float tp = a.top_p ? a.top_p[b] : 1.f;
  if (tp < 1.f) {
    const double t = (double)fmaxf(tp, 0.f) * (double)total;
    const Place p = find(max((uint64_t)1, (uint64_t)ceil(t)), true);
    if (p.key > last.key || (p.key == last.key && p.ties < last.ties)) {
      last = p;
      total = last.above + last.ties * mass(last.key);
    }
  }
  const float mp = a.min_p ? a.min_p[b] : 0.f;
  if (mp > 0.f) {
    const double least = fmin((double)mp, 1.0);
    uint32_t end = 0xffffffffu;                  // the least that reaches min_p (a beginning as well)
    each([&](uint32_t key) {
      if (key < end && weight(order_float(key)) >= least) end = key;
    });
    end = ~reduce_max(~end);
    if (end > last.key) {
      last = Place{end - 1, 0, 0};
      total = sum_mass(last);
    }
  }
  const double t = draw(a, b) * (double)total;
  const uint64_t target = min((uint64_t)t + 1, total);
  const Place p = find(target, true);
  const uint32_t i = index_of(p);
  if (tid == 0) {
    a.token[b] = i;
    const float v = order_float(p.key);
    const double d = v == top ? 0.0 : ((double)v - (double)top) / (double)temp;
    if (a.logprob) a.logprob[b] = (float)(d - log((double)total / unit));
  }
}

// What the collected elements of a row are searched with
struct PickShared {
  uint64_t hist[kBins];                          // of 512 parts of an interval of keys, as Part's
  uint64_t key[kTiny], weight[kTiny];            // elements that are compared with one another
  uint64_t got_key, low[16], high[16];
  uint64_t scan[16];
  double above, got_cum, got_weight, bin_mass, bin_upto, bin_over, unit, mid;
  uint64_t ends[2];
  uint32_t scan_u[16], n, bin, above_n, in, place;
};

__global__ __launch_bounds__(kThreads, 4) void sample_pick_kernel(SampleArgs a, SampleWork ws) {
  const int b = blockIdx.y, g = blockIdx.x, parts = gridDim.x, tid = threadIdx.x, lane = tid & 63;
  const State *const st = ws.states + b;
  const float *x = a.x + b * a.rs;
  const uint32_t slow = st->slow;
  const double top = st->top;
  const uint64_t mask_bits = st->mask[tid & (kBins / 64 - 1)];
  const Row row(Row(a, b), (int)st->fine);
  const Settings set(a, b, row.greedy);
  if (slow != kUsual) {
    if (g == 0 && slow == kSlow) slow_row(a, b, st->mass);
    return;
  }
  __shared__ PickShared sh;
  __shared__ uint64_t mask[kBins / 64];
  __shared__ uint32_t base_s, last_s;
  if (tid < kBins / 64) mask[tid] = mask_bits;
  __syncthreads();
  const Share share(a.n);
  uint64_t wanted = 0;                           // (at most 64 of a thread)
  share.each(x, [&](float v, int i) {
    const double j = v > -INFINITY ? top - floor(row.y(v)) : (double)kBins;
    if (j < kBins && (mask[(int)j >> 6] >> ((int)j & 63) & 1)) wanted |= (uint64_t)1 << i;
  });
  uint64_t *const all = ws.lists + (int64_t)b * kList;
  Counters *const c = ws.counters + b;
  // places in the row's list: of the thread in the workgroup, of the workgroup in the row
  const uint32_t mine = (uint32_t)__builtin_popcountll(wanted);
  uint32_t n_mine, at = 0;
  if (__syncthreads_or(wanted != 0)) {
    at = block_scan(mine, sh.scan_u, n_mine) - mine;
    if (tid == 0) base_s = __hip_atomic_fetch_add(&c->listed, n_mine, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    at += base_s;
    for (; wanted; wanted &= wanted - 1, ++at) {
      const int i = share.first + __builtin_ctzll(wanted) * kThreads;
      // (all collected bins together hold at most kList)
      if (at < kList) st_agent(all + at, (uint64_t)~order_bits(x[i]) << 32 | (uint32_t)i);
    }
  }
  // up to and with bin tid, and above it (for the last workgroup: here their loads take no time of their own)
  double upto = 0.0, over = 0.0;
  uint32_t upto_n = 0, over_n = 0;
  if (tid < kBins) {
    upto = st->upto_mass[tid];
    upto_n = st->upto_count[tid];
    if (tid > 0) {
      over = st->upto_mass[tid - 1];
      over_n = st->upto_count[tid - 1];
    }
  }
  const uint32_t in_bins = st->upto_count[kBins - 1];
  const int m_lo = (int)st->m_lo, m_hi = (int)st->m_hi;
  const float best = order_float(st->best);
  wait_all_mem();
  __syncthreads();
  if (tid == 0)
    last_s = __hip_atomic_fetch_add(&c->pick, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)parts - 1u;
  __syncthreads();
  if (!last_s) return;
  // ---- the row's elements, in any order ----
  // (loops over LDS: unrolled over registers, their doubles' code was fetched for longer than it ran)
  __shared__ uint64_t list[kList];
  const uint64_t first_entry = ld_agent(all + tid);
  const int n = (int)min(ld_agent(&c->listed), (uint32_t)kList), wave = wave_id();
  if (tid < n) list[tid] = first_entry;
  for (int i = tid + kThreads; i < n; i += kThreads) list[i] = ld_agent(all + i);
  auto each = [&](auto f) {                      // (a thread's own)
#pragma unroll 1
    for (int i = tid; i < n; i += kThreads) f(list[i]);
  };
  double s3 = st->mass;                          // of S1, of S2, of S3: bins 0 .. from_hist - 1 as the first launch has them
  uint32_t from_hist = kBins;
  uint64_t end_key = ~0ull;                      // its last element
  __syncthreads();
  if (tid == 0) {
    st_agent(&c->listed, 0u);
    st_agent(&c->pick, 0u);
  }
  const double scale = kLn2 * row.per_q;
  const float tp = set.tp, mp = set.mp;
  const int k = set.k;
  // S1's end, S2's end, the token: each the first element up to which a count, or the mass, reaches a target (the
  // token's: passes it).  Its bin first; then, as long as an interval of keys holds more than kTiny elements, 512 parts
  // of what its least and largest key span (a few values, each of many elements, where logits are bf16: then the parts
  // are of indices); then element by element.
#pragma unroll 1
  for (int stage = 0; stage < 3; ++stage) {
    if (stage == 0 && !(k && (uint32_t)k <= in_bins)) continue;
    if (stage == 1 && !(tp < 1.f)) continue;
    if (stage == 2 && mp > 0.f && m_lo < kBins) {   // S3: also what reaches min_p, the bins above m_lo and elements of m_lo .. m_hi
      uint64_t sum = 0, all_sum, end_m = 0;
      each([&](uint64_t e) {
        const float v = list_value(e);
        const double y = row.y(v), j = top - floor(y);
        if (j >= (double)m_lo && j <= (double)m_hi && !row.under(v, best, mp)) {
          sum += (uint64_t)(row.weight(y, top - (double)m_lo) * 0x1p44 + 0.5);
          end_m = e > end_m ? e : end_m;
        }
      });
      end_m = wave_max(end_m);
      if (lane == 0) sh.high[wave] = end_m;      // (the scan's barriers stand before and behind its reads)
      block_scan(sum, sh.scan, all_sum);
      const double above = m_lo ? st->upto_mass[m_lo - 1] : 0.0;
      const double sum_m = above + (double)all_sum * (exp2_of(-(double)m_lo * row.per_q) * 0x1p-44);
      end_m = wave_max(sh.high[lane & 15]);      // 0: what reaches min_p ends above m_lo
      const uint64_t first_m = (uint64_t)~(row.first(top - (double)m_lo, true) - 1u) << 32;   // the least key of m_lo
      if ((end_m ? end_m : first_m - 1) < end_key) {
        s3 = sum_m;
        from_hist = (uint32_t)m_lo;
      }
    }
    const bool by_mass = stage > 0;
    const double target = stage == 0 ? (double)k : stage == 1 ? (double)fmaxf(tp, 0.f) * s3 : set.u * s3;
    auto reaches = [&](double x) { return stage == 2 ? x > target : x >= target; };
    // the first bin that reaches it (where rounding leaves none, the last), from its thread
    __syncthreads();
    if (tid < kBins) {
      const bool here = reaches(by_mass ? upto : (double)upto_n), before = tid > 0 && reaches(by_mass ? over : (double)over_n);
      if (tid == kBins - 1 ? !before : here && !before) {
        sh.bin = tid;
        sh.above = over;
        sh.above_n = over_n;
        sh.in = upto_n - over_n;
        sh.bin_upto = upto;
        sh.bin_over = over;
      }
    }
    if (tid == 0) {
      sh.place = ~0u;
      sh.n = 0;
    }
    __syncthreads();
    const uint32_t bin = sh.bin, first_in = sh.in;
    const double low = top - (double)bin;        // the bin's lower end
    // what all threads need of the bin, each from one wave (of one SIMD each)
    if (wave == 0) {
      const uint32_t o = row.first(low, true);
      if (lane == 0) sh.ends[0] = (uint64_t)~(o - 1u) << 32;
    } else if (wave == 1) {
      const uint32_t o = row.first(low, false);
      if (lane == 0) sh.ends[1] = (uint64_t)~o << 32 | 0xffffffffu;
    } else if (wave == 2) {
      const double w = exp2_of(-(double)bin * row.per_q);
      if (lane == 0) sh.unit = w * 0x1p-44;
    } else if (wave == 3) {
      const double w = exp2_of((0.5 - (double)bin) * row.per_q);
      if (lane == 0) sh.mid = w;
    }
    __syncthreads();
    double above = sh.above;
    uint32_t above_n = sh.above_n, in = first_in;
    const double unit = sh.unit, mid = sh.mid;
    // the interval: elements with lo <= key <= hi, at first those of the bin
    uint64_t lo = sh.ends[0], hi = sh.ends[1];
    auto mine = [&](uint64_t e) { return e >= lo && e <= hi; };
#pragma unroll 1
    for (int round = 0; round < 8 && in > kTiny; ++round) {   // (64 bits of keys, 9 and more a round)
      if (tid < kBins) sh.hist[tid] = 0;
      if (round > 0) {                           // what the elements span
        uint64_t l = ~0ull, r = 0;
        each([&](uint64_t e) {
          if (!mine(e)) return;
          l = e < l ? e : l;
          r = e > r ? e : r;
        });
        l = ~wave_max(~l);
        r = wave_max(r);
        if (lane == 0) {
          sh.low[wave] = l;
          sh.high[wave] = r;
        }
        __syncthreads();
        lo = ~wave_max(~sh.low[lane & 15]);
        hi = wave_max(sh.high[lane & 15]);
      } else {
        __syncthreads();
      }
      if (lo >= hi) break;                       // (not with more than one element)
      const int bits = 64 - __builtin_clzll(hi - lo), shift = bits > 9 ? bits - 9 : 0;
      each([&](uint64_t e) {
        if (!mine(e)) return;
        atomicAdd((unsigned long long *)&sh.hist[(e - lo) >> shift],
                  (unsigned long long)hist_add((row.y(list_value(e)) - low - 0.5) * scale));
      });
      __syncthreads();
      const uint64_t h = tid < kBins ? sh.hist[tid] : 0;
      const uint32_t cnt = (uint32_t)(h >> 48);
      const double m = hist_mass(h);
      uint32_t all_n;
      uint64_t all_m;
      const uint32_t c_upto = above_n + block_scan(cnt, sh.scan_u, all_n);
      const double m_upto = above + (double)block_scan((uint64_t)(m * 0x1p44), sh.scan, all_m) * (mid * 0x1p-44);
      // (the last where rounding leaves none)
      if (cnt > 0 && (reaches(by_mass ? m_upto : (double)c_upto) || c_upto == above_n + all_n)) atomicMin(&sh.place, (uint32_t)tid);
      __syncthreads();
      const uint32_t part = sh.place;
      if ((uint32_t)tid == part) {
        sh.above = m_upto - m * mid;
        sh.above_n = c_upto - cnt;
        sh.in = cnt;
      }
      __syncthreads();
      if (tid == 0) sh.place = ~0u;
      above = sh.above;
      above_n = sh.above_n;
      in = sh.in;
      lo += (uint64_t)part << shift;
      const uint64_t end = lo + (((uint64_t)1 << shift) - 1);
      hi = end < hi ? end : hi;
    }
    each([&](uint64_t e) {
      if (!mine(e)) return;
      const uint32_t at = atomicAdd(&sh.n, 1u);
      if (at < kTiny) sh.key[at] = e;
    });
    __syncthreads();
    if (wave == 0) {                             // one element per lane
      const uint32_t m = min(sh.n, (uint32_t)kTiny);
      const uint64_t own = (uint32_t)lane < m ? sh.key[lane] : ~0ull;
      const uint64_t weight = (uint32_t)lane < m ? (uint64_t)(row.weight(row.y(list_value(own)), low) * 0x1p44 + 0.5) : 0;
      sh.weight[lane] = weight;
      sh.key[lane] = own;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      uint64_t cum = 0;
      uint32_t rank = 0;
#pragma unroll 4
      for (uint32_t i = 0; i < m; ++i) {
        const bool upto_me = sh.key[i] <= own;
        rank += upto_me;
        cum += upto_me ? sh.weight[i] : 0;
      }
      const double mass = above + (double)cum * unit;
      const bool ok = (uint32_t)lane < m && (reaches(by_mass ? mass : (double)(above_n + rank)) || rank == m);
      const uint32_t place = ~wave_max(ok ? ~rank : 0u);
      if ((uint32_t)lane < m) {
        if (rank == place) {
          sh.got_key = own;
          sh.got_cum = mass;
          sh.got_weight = (double)weight * unit;
        }
        if (rank == m) sh.bin_mass = (double)cum * unit;
      }
    }
    __syncthreads();
    if (row.greedy) break;
    if (stage < 2) {
      if (sh.got_key <= end_key) {               // (a rounding could put S2's behind S1's)
        s3 = sh.got_cum;
        from_hist = bin;
        end_key = sh.got_key;
      }
    } else if (first_in <= kTiny && bin < from_hist) {
      // the whole bin is S3's: its sum from its elements' 2^-44 instead of 2^-34, so that the logarithm of a token with
      // nearly all of the mass, which may be alone, has few wrong digits
      s3 += sh.bin_mass - (sh.bin_upto - sh.bin_over);
    }
  }
  if (tid == 0) {
    a.token[b] = (uint32_t)sh.got_key;
    if (a.logprob) a.logprob[b] = row.greedy ? 0.f : (float)log(fmin(1.0, sh.got_weight / s3));
  }
}

struct SamplePlan {
  int parts;
  int64_t states, lists, parts_at, bytes;        // byte offsets; the counters come first, for any launch
};
// rows: of one launch.  Parts of 8192 logits, fewer and larger ones where that would make more than one workgroup per CU,
// but for what a bin's fields hold.  (Parts of 4096, 8192, 12288 and 16384, both launches: 4 rows of 151936 44, 41, 41 and
// 43 us, 1 row of them 36, 37, 39 and 40: a part costs its logits' time twice over, and 4 KB of the merge.)
constexpr int64_t kPart = 8 * kThreads;
int sample_parts(int64_t rows, int64_t n) {
  const int64_t least = (n + kMostChunk - 1) / kMostChunk, most = (n + kPart - 1) / kPart;
  return (int)std::max(least, std::min(most, device_cus() / rows));
}
SamplePlan plan_sample(int64_t rows, int64_t n) {
  SamplePlan p;
  p.parts = sample_parts(rows, n);
  p.states = kRowsPerLaunch * sizeof(Counters);
  p.lists = p.states + rows * (int64_t)sizeof(State);
  p.parts_at = p.lists + rows * kList * 8;
  p.bytes = p.parts_at + rows * p.parts * (int64_t)sizeof(Part);
  return p;
}

}  // namespace
}  // namespace tg

using namespace tg;

// (enough for fewer rows and columns: those may be cut into more parts, but then into no more than one per CU in all)
extern "C" int64_t tg_sample_rows_workspace_size(int32_t n_rows, int64_t n_cols) {
  if (n_rows <= 0 || n_cols <= kSort || n_cols > (1 << 18)) return 0;
  const int64_t rows = std::min<int32_t>(n_rows, kRowsPerLaunch);
  const int64_t parts = std::max(std::min<int64_t>(rows * sample_parts(1, n_cols), device_cus()), rows * sample_parts(rows, n_cols));
  return plan_sample(rows, n_cols).parts_at + parts * (int64_t)sizeof(Part);
}

extern "C" int tg_sample_rows(const float *x, int64_t x_row_stride, int32_t n_rows, int64_t n_cols, const float *u,
                              const float *temperature, const int32_t *top_k, const float *top_p, const float *min_p,
                              int64_t *token, float *logprob, void *workspace, int64_t workspace_bytes,
                              hipStream_t stream) {
  clear_error();
  TG_CHECK(x && u && token, "sample_rows: null pointer");
  TG_CHECK(n_rows >= 0 && n_rows < 65536 && n_cols > 0 && n_cols <= (1 << 18), "sample_rows: 0..65535 rows of 1..262144 columns");
  TG_CHECK(x_row_stride >= n_cols, "sample_rows: row stride must be >= n_cols");
  if (n_rows == 0) return 0;
  if (n_cols <= kSort) {
    const SampleArgs a{x, x_row_stride, (int)n_cols, u, temperature, top_p, min_p, top_k, token, logprob};
    hipLaunchKernelGGL(sample_small_kernel, dim3((unsigned)n_rows), dim3(kThreads), 0, stream, a);
    TG_HIP_CHECK(hipGetLastError());
    return 0;
  }
  const int64_t need = plan_sample(std::min<int32_t>(n_rows, kRowsPerLaunch), n_cols).bytes;
  TG_CHECK(workspace != nullptr && aligned16(workspace) && workspace_bytes >= need,
           "sample_rows: needs a 16-byte aligned workspace of %lld bytes (got %lld)", (long long)need, (long long)workspace_bytes);
  for (int32_t r0 = 0; r0 < n_rows; r0 += kRowsPerLaunch) {
    const int32_t rows = std::min<int32_t>(n_rows - r0, kRowsPerLaunch);
    auto at = [r0](auto *p) { return p ? p + r0 : p; };
    const SampleArgs a{x + r0 * x_row_stride, x_row_stride, (int)n_cols, u + r0, at(temperature), at(top_p), at(min_p),
                       at(top_k), token + r0, at(logprob)};
    const SamplePlan p = plan_sample(rows, n_cols);
    char *ws = static_cast<char *>(workspace);
    const SampleWork w{reinterpret_cast<Counters *>(ws), reinterpret_cast<State *>(ws + p.states),
                       reinterpret_cast<uint64_t *>(ws + p.lists), reinterpret_cast<Part *>(ws + p.parts_at)};
    const dim3 grid((unsigned)p.parts, (unsigned)rows), block(kThreads);
    hipLaunchKernelGGL(sample_hist_kernel, grid, block, 0, stream, a, w);
    hipLaunchKernelGGL(sample_pick_kernel, grid, block, 0, stream, a, w);
    TG_HIP_CHECK(hipGetLastError());
  }
  return 0;
}
