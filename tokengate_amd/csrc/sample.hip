// The next token of rows of logits: temperature, top-k, top-p, min-p and one given random number per row.
//
// With w_i = exp((x_i - max x) / T) and the order "larger logits first, equal ones by index": S1 = the first k;
// S2 = the shortest beginning of S1 whose mass (sum of w) is at least top_p times S1's, one at least; S3 = those
// of S2 with w >= min_p, one at least; the token is the first of S3 whose cumulated mass exceeds u times S3's, and
// its log probability is ln(w / mass(S3)).  Every set is a beginning of the same order, so the row is not sorted:
//   * sample_hist_kernel, several workgroups per row: logits in units of y = cc x (cc = 8 log2 e, or 4 log2 e / T for
//     T < 0.5) fall into bins of width one, 512 from the chunk's largest down.  A bin's count and the sum of its
//     elements' e^t, t = (the fraction of y - 1/2) T-scaled, need no common maximum, and as whole numbers (one 64-bit
//     LDS addition per logit) no order of additions.  The workgroup that arrives last merges the row's bins and finds
//     those in which the ends of S1, S2, S3 and the token must lie;
//   * sample_pick_kernel collects the elements of these bins (up to 16384), and the last workgroup finds each end in its
//     bin: by 512 bins of 1/512 of the bin, and in one of these by comparing its elements with one another.
// Rows of up to 2048 logits take one workgroup and one launch, which sorts them all.  Where the bins that decide hold
// more than that (rows that are nearly flat), one workgroup finds the places digit by digit over the whole row.
// Double throughout: a row has so many borders between tokens that sums good to 2^-24 would move one row in a hundred
// across one; here they are good to 2^-36.
// Bound by latency (two launches, two merges) for few rows and by the exponentials and LDS additions for many.
#include <algorithm>

#include "tg_common.h"
#include "../../include/tokengate_hip.h"

namespace tg {
namespace {

constexpr double kLog2e = 1.4426950408889634, kLn2 = 0.6931471805599453;
constexpr int kThreads = 1024;
constexpr int kBins = 512;
constexpr int kSort = 2048;                      // elements that one workgroup sorts
constexpr int kList = 16384;                     // elements that are collected
constexpr int kTiny = 1024;                      // elements that are compared with one another
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
  uint64_t tail;                                 // mass below the bins, in units of 2^-44 of 2^(top / q)
  uint32_t best, pad;                            // order bits of the largest logit
  uint64_t hist[kBins];                          // count << 48 | sum of (e^t - 0.9) 2^36
};
// What the first launch leaves for the second, per row; bin j: y in [top - j, top - j + 1)
struct State {
  double top, mass;                              // mass of the whole row, in units of 2^(top / q), as all
  uint64_t mask[kBins / 64];                     // bins to collect
  uint32_t best, slow, m_lo, m_hi;               // bins that may hold min_p's end
  double upto_mass[kBins];                       // up to and with bin j
  uint32_t upto_count[kBins];
};
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
constexpr uint32_t kNone = 0x007FFFFFu;          // order bits of -inf

// A row's settings.  Bins per octave of w: q; y = cc x.
struct Row {
  double q, cc;
  float temp;
  bool greedy;
  __device__ Row(const SampleArgs &a, int b) {
    const float t = a.temperature ? a.temperature[b] : 1.f;
    greedy = !(t > 0.f);
    temp = greedy ? 1.f : t;
    q = fmax(4.0, 8.0 * (double)temp);
    cc = q * kLog2e / (double)temp;
  }
  // (+inf: so far above every finite one that those weigh nothing)
  __device__ double y(float x) const { return x == INFINITY ? 0x1p1000 : (double)x * cc; }
  __device__ double weight(double y, double top) const { return exp2((y - top) / q); }
  __device__ double weight_of(float x, double top) const { return x == -INFINITY ? 0.0 : weight(y(x), top); }
  // whether x has less than least times the largest logit's weight
  __device__ bool under(float x, float best, float least) const {
    return x != best && (x == -INFINITY || weight(y(x), y(best)) < fmin((double)least, 1.0));
  }
};
// u[b]; a one, which a rounded number may be, takes the last element of a mass of more than 2^-30
__device__ __forceinline__ double draw(const SampleArgs &a, int b) { return fmin(fmax((double)a.u[b], 0.0), 1.0 - 0x1p-30); }

// e^t for |t| <= 0.087, to 2^-49
__device__ __forceinline__ double exp_small(double t) {
  double p = 1.0 / 40320;
  p = fma(p, t, 1.0 / 5040);
  p = fma(p, t, 1.0 / 720);
  p = fma(p, t, 1.0 / 120);
  p = fma(p, t, 1.0 / 24);
  p = fma(p, t, 1.0 / 6);
  p = fma(p, t, 0.5);
  p = fma(p, t, 1.0);
  return fma(p, t, 1.0);
}
constexpr double kHistBase = 0.9, kHistUnit = 0x1p36;

__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t *tmp) {   // tmp: 16 words
  const int tid = threadIdx.x;
#pragma unroll
  for (int o = 32; o; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o));
  __syncthreads();
  if ((tid & 63) == 0) tmp[tid >> 6] = v;
  __syncthreads();
  v = tmp[tid & 15];
#pragma unroll
  for (int o = 8; o; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o));
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
// Sums over the threads up to this one; total: over all.  tmp: 16 of T.
template <typename T>
__device__ __forceinline__ T block_scan(T v, T *tmp, T &total) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  v = wave_scan(v);
  __syncthreads();
  if (lane == 63) tmp[wave] = v;
  __syncthreads();
  T before = T(0);
  total = T(0);
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) {
    const T s = tmp[i];
    before += i < wave ? s : T(0);
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

template <int E>
__global__ __launch_bounds__(kThreads, E == 4 ? 4 : 8) void sample_hist_kernel(SampleArgs a, SampleWork ws) {
  const int b = blockIdx.y, g = blockIdx.x, parts = gridDim.x, tid = threadIdx.x;
  const float *x = a.x + b * a.rs;
  __shared__ uint64_t hist[kBins];
  __shared__ uint32_t tmp[16];
  __shared__ unsigned long long tail_s;
  __shared__ uint32_t last_s;
  float v[E];
  uint32_t best = kNone;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int i = (g * E + e) * kThreads + tid;
    v[e] = i < a.n ? x[i] : -INFINITY;
    best = max(best, order_bits(v[e]));
  }
  const Row row(a, b);
  if (tid < kBins) hist[tid] = 0;
  if (tid == 0) tail_s = 0;
  best = block_max(best, tmp);                   // (its barriers cover the bins)
  const double top = best == kNone ? 0.0 : floor(row.y(order_float(best)));
  const double scale = kLn2 / row.q;
  const int top_slot = slot_of(top);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (!(v[e] > -INFINITY)) continue;
    const double y = row.y(v[e]), f = floor(y), j = top - f;
    if (j < kBins) {
      const double t = (y - f - 0.5) * scale;
      atomicAdd((unsigned long long *)&hist[(top_slot - (int)j) & (kBins - 1)], (1ull << 48) + (unsigned long long)((exp_small(t) - kHistBase) * kHistUnit + 0.5));
    } else {
      const double w = row.weight(y, top);
      if (w > 0x1p-46) atomicAdd(&tail_s, (unsigned long long)(w * 0x1p44 + 0.5));
    }
  }
  __syncthreads();
  Part *const part = ws.parts + (int64_t)b * parts;
  if (tid < kBins) st_agent(&part[g].hist[tid], hist[tid]);
  if (tid == 0) {
    st_agent((uint64_t *)&part[g].top, bits_of(top));
    st_agent(&part[g].tail, (uint64_t)tail_s);
    st_agent(&part[g].best, best);
  }
  wait_all_mem();
  __syncthreads();
  if (tid == 0)
    last_s = __hip_atomic_fetch_add(&ws.counters[b].hist, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)parts - 1u;
  __syncthreads();
  if (!last_s) return;

  // ---- the row's bins ----
  __shared__ double tops[64], mass_s[kBins], scan_d[16];
  __shared__ uint64_t sums[2][kBins];
  __shared__ uint32_t counts[2][kBins], count_s[kBins], scan_u[16], bests[64];
  __shared__ int first_s[4], slots[64];
  if (tid < parts) {
    tops[tid] = double_of(ld_agent((const uint64_t *)&part[tid].top));
    slots[tid] = slot_of(tops[tid]);
    bests[tid] = ld_agent(&part[tid].best);
  }
  __syncthreads();
  best = kNone;
  for (int i = 0; i < parts; ++i) best = max(best, bests[i]);
  State *const st = ws.states + b;
  if (best == kNone) {                           // nothing but -inf: token 0, by the slow way
    if (tid == 0) {
      st->slow = 1;
      for (int i = 0; i < kBins / 64; ++i) st->mask[i] = 0;
      st_agent(&ws.counters[b].hist, 0u);
    }
    return;
  }
  const double gtop = floor(row.y(order_float(best)));
  // thread: one slot of every other part
  const int slot = tid & (kBins - 1), half = tid / kBins;
  uint64_t sum = 0;
  uint32_t count = 0;
  double tail = 0.0;
  constexpr int kAhead = E == 4 ? 20 : 8;
  for (int i0 = half; i0 < parts; i0 += 2 * kAhead) {
    uint64_t h[kAhead];
#pragma unroll
    for (int r = 0; r < kAhead; ++r) h[r] = ld_agent(&part[min(i0 + 2 * r, parts - 1)].hist[slot]);
#pragma unroll
    for (int r = 0; r < kAhead; ++r) {
      const int i = i0 + 2 * r;
      if (i >= parts || h[r] == 0) continue;
      const double below = gtop - tops[i] + ((slots[i] - slot) & (kBins - 1));   // the row's bin, if less than kBins
      if (below < kBins) {
        count += (uint32_t)(h[r] >> 48);
        sum += h[r] & 0xffffffffffffull;
      } else {
        tail += exp2((0.5 - below) / row.q) * (kHistBase * (double)(h[r] >> 48) + (double)(h[r] & 0xffffffffffffull) / kHistUnit);
      }
    }
  }
  if (tid < parts && bests[tid] != kNone) tail += exp2((tops[tid] - gtop) / row.q) * ((double)ld_agent(&part[tid].tail) * 0x1p-44);
  {
    const int j = (slot_of(gtop) - slot) & (kBins - 1);
    sums[half][j] = sum;
    counts[half][j] = count;
  }
  __syncthreads();
  const int j = slot;                            // from here on a bin
  double m = 0.0;
  count = 0;
  if (half == 0) {
    count = counts[0][j] + counts[1][j];
    m = exp2((0.5 - j) / row.q) * (kHistBase * (double)count + (double)(sums[0][j] + sums[1][j]) / kHistUnit);
  }
  double in_bins, tail_all;
  uint32_t n_bins;
  const double upto = block_scan(m, scan_d, in_bins);
  const uint32_t upto_count = block_scan(count, scan_u, n_bins);
  block_scan(tail, scan_d, tail_all);
  const double mass = in_bins + tail_all;
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
  const uint32_t k = row.greedy ? 1u : a.top_k && a.top_k[b] > 0 && a.top_k[b] < a.n ? (uint32_t)a.top_k[b] : 0u;
  const float tp = a.top_p && !row.greedy ? a.top_p[b] : 1.f, mp = a.min_p && !row.greedy ? a.min_p[b] : 0.f;
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
    const double thr = row.y(order_float(best)) + row.q * log2(fmin((double)mp, 1.0)), d0 = gtop - floor(thr + 1e-6),
                 d1 = gtop - floor(thr - 1e-6);
    m_lo = d0 < 0.0 ? 0 : d0 < kBins ? (int)d0 : kBins;
    m_hi = d1 < 0.0 ? 0 : d1 < kBins ? (int)d1 : kBins;
    slow |= tail_counts && m_hi == kBins;
    if (m_lo < kBins) lo = fmin(lo, m_lo ? mass_s[m_lo - 1] : 0.0);
    if (m_hi < kBins) hi = fmin(hi, mass_s[m_hi]);
  }
  const double u = fmin(fmax((double)a.u[b], 0.0), 1.0);
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
    st->slow = slow;
    st->m_lo = (uint32_t)m_lo;
    st->m_hi = (uint32_t)m_hi;
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
// Masses as whole numbers, in units of 2^-44 of the largest weight.
__device__ void slow_row(const SampleArgs &a, int b) {
  constexpr double kMassUnit = 0x1p44;
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
  uint32_t best = 0;
  for (int i = tid; i < a.n; i += kThreads) best = max(best, order_bits(x[i]));
  best = reduce_max(best);
  const float top = order_float(best);
  const float temp = a.temperature ? a.temperature[b] : 1.f;
  const bool greedy = !(temp > 0.f) || top == -INFINITY;
  const double scale = greedy ? 1.0 : kLog2e / temp;
  auto weight = [&](float x) { return x == top ? 1.0 : exp2(((double)x - (double)top) * scale); };   // (both may be infinite)
  auto mass = [&](uint32_t key) { return (uint64_t)(weight(order_float(key)) * kMassUnit + 0.5); };
  // The first place at which the sum of value(key) over the elements up to it reaches target (> 0).
  auto find = [&](uint64_t target, bool by_mass) {
    uint32_t prefix = 0;
    uint64_t above = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int i = tid; i < a.n; i += kThreads) {
        const uint32_t key = order_bits(x[i]);
        if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8)))
          atomicAdd((unsigned long long *)&hist[(key >> shift) & 255], (unsigned long long)(by_mass ? mass(key) : 1));
      }
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
    for (int i = tid; i < a.n; i += kThreads) {
      const uint32_t key = order_bits(x[i]);
      if (key > p.key) s += mass(key);
    }
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
    uint64_t s = 0;                              // mass of what reaches min_p (a beginning as well)
    const double least = fmin((double)mp, 1.0);
    uint32_t end = 0xffffffffu;
    for (int i = tid; i < a.n; i += kThreads) {
      const uint32_t key = order_bits(x[i]);
      if (weight(order_float(key)) >= least) end = min(end, key);
    }
    end = ~reduce_max(~end);
    if (end > last.key) {
      last = Place{end - 1, 0, 0};
      total = sum_mass(last);
    }
  }
  const double t = (double)a.u[b] * (double)total;
  const uint64_t target = min((uint64_t)t + 1, total);
  const Place p = find(target, true);
  const uint32_t i = index_of(p);
  if (tid == 0) {
    a.token[b] = i;
    const float v = order_float(p.key);
    const double d = v == top ? 0.0 : ((double)v - (double)top) / (double)temp;
    if (a.logprob) a.logprob[b] = (float)(d - log((double)total / kMassUnit));
  }
}

// The collected elements of a row, in any order: kList / kThreads per thread, and what they are searched with.
struct PickShared {
  uint64_t mass[kBins];                          // of a bin's 512 parts, in units of 2^-44 of the bin's lower end
  uint32_t count[kBins];
  uint64_t key[kTiny], weight[kTiny];            // elements that are compared with one another
  uint64_t got_key;
  double scan[16], got_cum, got_weight, above;
  uint32_t scan_u[16], n, bin, part, above_n, place;
};
struct Picked {
  uint64_t key;
  double cum, weight;                            // mass up to and with it, and its own
  bool ok;
};
template <int R>
struct Collected {
  const Row &row;
  const State *st;
  PickShared &sh;
  uint64_t key[R];
  int n;
  double top, upto;                              // upto: mass up to and with bin tid
  uint32_t upto_n;

  template <typename F>
  __device__ __forceinline__ void each(F f) const {
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (r * kThreads + (int)threadIdx.x < n) f(key[r]);
  }
  // The first element up to which the count, or the mass, reaches target (strictly: passes it).
  __device__ Picked find(bool by_mass, double target, bool strictly) {
    const int tid = threadIdx.x;
    auto reaches = [&](double c) { return strictly ? c > target : c >= target; };
    __syncthreads();
    if (tid == 0) {
      sh.bin = kBins;
      sh.n = 0;
      sh.place = ~0u;
    }
    __syncthreads();
    if (tid < kBins) {
      const double c = by_mass ? upto : (double)upto_n, p = tid == 0 ? -1.0 : by_mass ? st->upto_mass[tid - 1] : (double)st->upto_count[tid - 1];
      if (reaches(c) && (tid == 0 || !reaches(p))) {
        sh.bin = tid;
        sh.above = tid ? st->upto_mass[tid - 1] : 0.0;
        sh.above_n = tid ? st->upto_count[tid - 1] : 0;
        sh.part = upto_n - sh.above_n;           // elements of the bin
      }
    }
    __syncthreads();
    const uint32_t bin = sh.bin, in_bin = sh.part;
    if (bin == kBins) return Picked{0, 0.0, 0.0, false};
    const double low = top - (double)bin;        // the bin's lower end
    const double unit = exp2(-(double)bin / row.q) * 0x1p-44;
    auto mine = [&](uint64_t e) { return floor(row.y(list_value(e))) == low; };
    auto part_of = [&](uint64_t e) { return min(kBins - 1, (int)((low + 1.0 - row.y(list_value(e))) * kBins)); };
    auto units = [&](uint64_t e) { return (uint64_t)(row.weight(row.y(list_value(e)), low) * 0x1p44 + 0.5); };
    double above = sh.above;
    uint32_t above_n = sh.above_n, part = kBins;   // kBins: the whole bin
    if (in_bin > kTiny / 2) {                    // its 512 parts
      if (tid < kBins) {
        sh.mass[tid] = 0;
        sh.count[tid] = 0;
      }
      __syncthreads();
      each([&](uint64_t e) {
        if (!mine(e)) return;
        const int p = part_of(e);
        atomicAdd((unsigned long long *)&sh.mass[p], (unsigned long long)units(e));
        atomicAdd(&sh.count[p], 1u);
      });
      __syncthreads();
      const uint32_t c = tid < kBins ? sh.count[tid] : 0;
      const double m = tid < kBins ? (double)sh.mass[tid] * unit : 0.0;
      uint32_t all_n;
      double all;
      const uint32_t c_upto = above_n + block_scan(c, sh.scan_u, all_n);
      const double m_upto = above + block_scan(m, sh.scan, all);
      const bool here = c > 0 && reaches(by_mass ? m_upto : (double)c_upto);
      // (the last of the bin where rounding leaves none)
      if (here || (c > 0 && c_upto == above_n + all_n)) atomicMin(&sh.place, (uint32_t)tid);
      __syncthreads();
      part = sh.place;
      __syncthreads();
      if ((uint32_t)tid == part) {
        sh.above = m_upto - m;
        sh.above_n = c_upto - c;
      }
      if (tid == 0) sh.place = ~0u;
      __syncthreads();
      above = sh.above;
      above_n = sh.above_n;
    }
    each([&](uint64_t e) {
      if (!mine(e) || (part < kBins && part_of(e) != (int)part)) return;
      const uint32_t at = atomicAdd(&sh.n, 1u);
      if (at < kTiny) {
        sh.key[at] = e;
        sh.weight[at] = units(e);
      }
    });
    __syncthreads();
    const uint32_t m = sh.n;
    if (m == 0 || m > kTiny) return Picked{0, 0.0, 0.0, false};
    uint64_t own = 0, cum = 0;
    uint32_t rank = 0;
    if ((uint32_t)tid < m) {
      own = sh.key[tid];
      for (uint32_t i = 0; i < m; ++i) {
        const bool upto_me = sh.key[i] <= own;
        rank += upto_me;
        cum += upto_me ? sh.weight[i] : 0;
      }
      const double c = by_mass ? above + (double)cum * unit : (double)(above_n + rank);
      if (reaches(c) || rank == m) atomicMin(&sh.place, rank);
    }
    __syncthreads();
    if ((uint32_t)tid < m && rank == sh.place) {
      sh.got_key = own;
      sh.got_cum = above + (double)cum * unit;
      sh.got_weight = row.weight_of(list_value(own), top);
    }
    __syncthreads();
    return Picked{sh.got_key, sh.got_cum, sh.got_weight, true};
  }
};

template <int E>
__global__ __launch_bounds__(kThreads, 4) void sample_pick_kernel(SampleArgs a, SampleWork ws) {
  const int b = blockIdx.y, g = blockIdx.x, parts = gridDim.x, tid = threadIdx.x, lane = tid & 63;
  const State *const st = ws.states + b;
  const float *x = a.x + b * a.rs;
  float v[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int i = (g * E + e) * kThreads + tid;
    v[e] = i < a.n ? x[i] : -INFINITY;
  }
  if (st->slow) {
    if (g == 0) slow_row(a, b);
    return;
  }
  __shared__ PickShared sh;
  __shared__ uint64_t mask[kBins / 64];
  __shared__ uint32_t n_s, base_s, last_s;
  const Row row(a, b);
  if (tid < kBins / 64) mask[tid] = st->mask[tid];
  const double top = st->top;
  if (tid == 0) n_s = 0;
  __syncthreads();
  uint32_t wanted = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const double j = v[e] > -INFINITY ? top - floor(row.y(v[e])) : (double)kBins;
    if (j < kBins && (mask[(int)j >> 6] >> ((int)j & 63) & 1)) wanted |= 1u << e;
  }
  uint64_t *const all = ws.lists + (int64_t)b * kList;
  Counters *const c = ws.counters + b;
  // places in the row's list: of the thread in the workgroup, of the workgroup in the row
  const uint32_t mine = (uint32_t)__builtin_popcount(wanted);
  uint32_t n_mine, at = 0;
  if (__syncthreads_or(wanted != 0)) {
    at = block_scan(mine, sh.scan_u, n_mine) - mine;
    if (tid == 0) base_s = __hip_atomic_fetch_add(&c->listed, n_mine, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    at += base_s;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (wanted >> e & 1) {
        // (all collected bins together hold at most kList)
        if (at < kList) st_agent(all + at, (uint64_t)~order_bits(v[e]) << 32 | (uint32_t)((g * E + e) * kThreads + tid));
        ++at;
      }
  }
  wait_all_mem();
  __syncthreads();
  if (tid == 0)
    last_s = __hip_atomic_fetch_add(&c->pick, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)parts - 1u;
  __syncthreads();
  if (!last_s) return;
  constexpr int R = kList / kThreads;
  Collected<R> col{row, st, sh};
  col.n = (int)min(ld_agent(&c->listed), (uint32_t)kList);
  col.top = top;
  col.upto = tid < kBins ? st->upto_mass[tid] : 0.0;
  col.upto_n = tid < kBins ? st->upto_count[tid] : 0;
#pragma unroll
  for (int r = 0; r < R; ++r) col.key[r] = r * kThreads < col.n ? ld_agent(all + min(r * kThreads + tid, kList - 1)) : 0;
  __syncthreads();
  if (tid == 0) {
    st_agent(&c->listed, 0u);
    st_agent(&c->pick, 0u);
  }
  const double mass = st->mass;
  const float tp = a.top_p ? a.top_p[b] : 1.f, mp = a.min_p ? a.min_p[b] : 0.f;
  const int k = row.greedy ? 1 : a.top_k && a.top_k[b] > 0 && a.top_k[b] < a.n ? a.top_k[b] : 0;
  bool ok = true;
  double s3 = mass;                              // of S1, then of S3
  Picked p{0, 0.0, 0.0, true};
  if (k && (uint32_t)k <= st->upto_count[kBins - 1]) {
    p = col.find(false, (double)k, false);
    ok &= p.ok;
    s3 = p.cum;
  }
  if (!row.greedy) {
    double end = s3;
    if (tp < 1.f) {
      p = col.find(true, (double)fmaxf(tp, 0.f) * s3, false);
      ok &= p.ok;
      end = fmin(end, p.cum);
    }
    if (mp > 0.f && (int)st->m_lo < kBins) {     // what reaches min_p: the bins above m_lo and elements of m_lo .. m_hi
      const float best = order_float(st->best);
      const double lo = (double)st->m_lo, hi = (double)st->m_hi;
      uint64_t sum = 0;
      const double unit = exp2(-lo / row.q) * 0x1p-44;
      col.each([&](uint64_t e) {
        const float y = list_value(e);
        const double j = top - floor(row.y(y));
        if (j >= lo && j <= hi && !row.under(y, best, mp)) sum += (uint64_t)(row.weight(row.y(y), top - lo) * 0x1p44 + 0.5);
      });
      uint64_t all_sum;
      block_scan(sum, reinterpret_cast<uint64_t *>(sh.scan), all_sum);
      end = fmin(end, (st->m_lo ? st->upto_mass[st->m_lo - 1] : 0.0) + (double)all_sum * unit);
    }
    s3 = end;
    p = col.find(true, draw(a, b) * s3, true);
    ok &= p.ok;
  }
  if (!ok) return slow_row(a, b);                // more than kTiny elements in 1/512 of a bin
  if (tid == 0) {
    a.token[b] = (uint32_t)p.key;
    if (a.logprob) a.logprob[b] = row.greedy ? 0.f : (float)log(fmin(1.0, p.weight / s3));
  }
}

struct SamplePlan {
  int parts, e;
  int64_t states, lists, parts_at, bytes;        // byte offsets; the counters come first, for any launch
};
int sample_parts(int64_t n, int e) { return (int)((n + e * kThreads - 1) / (e * kThreads)); }
// rows: of one launch.  4 logits per thread while that makes at most two workgroups per CU, else 16.
SamplePlan plan_sample(int64_t rows, int64_t n) {
  SamplePlan p;
  p.e = rows * sample_parts(n, 4) <= 2 * device_cus() ? 4 : 16;
  p.parts = sample_parts(n, p.e);
  p.states = kRowsPerLaunch * sizeof(Counters);
  p.lists = p.states + rows * (int64_t)sizeof(State);
  p.parts_at = p.lists + rows * kList * 8;
  p.bytes = p.parts_at + rows * p.parts * (int64_t)sizeof(Part);
  return p;
}

}  // namespace
}  // namespace tg

using namespace tg;

// (enough for fewer rows and columns: those may take 4 logits per thread, but then no more parts than two per CU)
extern "C" int64_t tg_sample_rows_workspace_size(int32_t n_rows, int64_t n_cols) {
  if (n_rows <= 0 || n_cols <= kSort || n_cols > (1 << 18)) return 0;
  const int64_t rows = std::min<int32_t>(n_rows, kRowsPerLaunch);
  const int64_t parts = std::max(std::min<int64_t>(rows * sample_parts(n_cols, 4), 2 * device_cus()), rows * sample_parts(n_cols, 16));
  const SamplePlan p = plan_sample(rows, n_cols);
  return p.parts_at + parts * (int64_t)sizeof(Part);
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
    if (p.e == 4) {
      hipLaunchKernelGGL(sample_hist_kernel<4>, grid, block, 0, stream, a, w);
      hipLaunchKernelGGL(sample_pick_kernel<4>, grid, block, 0, stream, a, w);
    } else {
      hipLaunchKernelGGL(sample_hist_kernel<16>, grid, block, 0, stream, a, w);
      hipLaunchKernelGGL(sample_pick_kernel<16>, grid, block, 0, stream, a, w);
    }
    TG_HIP_CHECK(hipGetLastError());
  }
  return 0;
}
