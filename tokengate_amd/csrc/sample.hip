// The next token of rows of logits: temperature, top-k, top-p, min-p and one given random number per row.
//
// With w_i = exp((x_i - max x) / T) and the order "larger logits first, equal ones by index": S1 = the first k;
// S2 = the shortest beginning of S1 whose mass (sum of w) is at least top_p times S1's, one at least; S3 = those
// of S2 with w >= min_p, one at least; the token is the first of S3 whose cumulated mass exceeds u times S3's, and
// its log probability is ln(w / mass(S3)).  Every set is a beginning of the same order, so nothing is sorted: the
// element at which a count or a mass is reached is found by its bits, most significant digit first.  Masses are
// whole numbers (units of 2^-44): their sums are exact and the same in any order.
#include "tg_common.h"
#include "../../include/tokengate_hip.h"

namespace tg {
namespace {

constexpr double kMassUnit = 0x1p44;
constexpr double kLog2e = 1.4426950408889634;

struct SampleArgs {
  const float *x;
  int64_t rs;
  int n;
  const float *u, *temperature, *top_p, *min_p;
  const int32_t *top_k;
  int64_t *token;
  float *logprob;
};

// Order-preserving bits of a float: larger floats, larger numbers; NaN is -inf, -0 is 0.
__device__ __forceinline__ uint32_t order_bits(float x) {
  x = x != x ? -INFINITY : x + 0.f;
  const uint32_t b = __builtin_bit_cast(uint32_t, x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float order_float(uint32_t o) {
  return u32_as_f32(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
// exp((x - top) / T) for x <= top, scale = log2(e) / T; in units of 2^-44.  Double: a row has so many borders
// between tokens that sums good to 2^-24 would move one row in a hundred across one.
__device__ __forceinline__ double weight_of(float x, float top, double scale) {
  return x == top ? 1.0 : exp2(((double)x - (double)top) * scale);   // (both may be infinite)
}
__device__ __forceinline__ uint64_t mass_of(float x, float top, double scale) {
  return (uint64_t)(weight_of(x, top, scale) * kMassUnit + 0.5);
}

// A place in the order: the elements above `key`, and the first `ties` of those equal to it.
struct Place {
  uint32_t key;
  uint32_t ties;
  uint64_t above;   // count or mass of the elements above key
};

__global__ __launch_bounds__(1024) void sample_rows_kernel(SampleArgs a) {
  const int b = blockIdx.x, tid = threadIdx.x;
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
  for (int i = tid; i < a.n; i += 1024) best = max(best, order_bits(x[i]));
  best = reduce_max(best);
  const float top = order_float(best);
  const float temp = a.temperature ? a.temperature[b] : 1.f;
  const bool greedy = !(temp > 0.f) || top == -INFINITY;
  const double scale = greedy ? 1.0 : kLog2e / temp;
  auto mass = [&](uint32_t key) { return mass_of(order_float(key), top, scale); };
  // The first place at which the sum of value(key) over the elements up to it reaches target (> 0).
  auto find = [&](uint64_t target, bool by_mass) {
    uint32_t prefix = 0;
    uint64_t above = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int i = tid; i < a.n; i += 1024) {
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
    for (int i = tid; i < a.n; i += 1024) {
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
    for (int i0 = 0; i0 < a.n; i0 += 1024) {
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
    for (int i = tid; i < a.n; i += 1024) {
      const uint32_t key = order_bits(x[i]);
      if (weight_of(x[i], top, scale) >= least) end = min(end, key);
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

}  // namespace
}  // namespace tg

using namespace tg;

extern "C" int64_t tg_sample_rows_workspace_size(int32_t n_rows, int64_t n_cols) { return 0; }

extern "C" int tg_sample_rows(const float *x, int64_t x_row_stride, int32_t n_rows, int64_t n_cols, const float *u,
                              const float *temperature, const int32_t *top_k, const float *top_p, const float *min_p,
                              int64_t *token, float *logprob, void *workspace, int64_t workspace_bytes,
                              hipStream_t stream) {
  clear_error();
  TG_CHECK(x && u && token, "sample_rows: null pointer");
  TG_CHECK(n_rows >= 0 && n_rows < 65536 && n_cols > 0 && n_cols <= (1 << 18), "sample_rows: 0..65535 rows of 1..262144 columns");
  TG_CHECK(x_row_stride >= n_cols, "sample_rows: row stride must be >= n_cols");
  if (n_rows == 0) return 0;
  const SampleArgs a{x, x_row_stride, (int)n_cols, u, temperature, top_p, min_p, top_k, token, logprob};
  hipLaunchKernelGGL(sample_rows_kernel, dim3((unsigned)n_rows), dim3(1024), 0, stream, a);
  TG_HIP_CHECK(hipGetLastError());
  return 0;
}
