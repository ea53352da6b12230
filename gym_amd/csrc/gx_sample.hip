// Actions from a policy's logits: temperature, top-k, top-p, min-p and a draw by a given random number (gx_sample).
//
// The kept set is a beginning of the order "logit descending, equal logits by index", so it is described by one logit t
// and a count j: everything above t, and the first j (by index) of those equal to t.  What has to be found is t, and
// that is a search over the ordered bits of binary32, never a sort of the row.  Weights exp((x - m) / T) and their sums
// are binary64 throughout: which action u falls on is a border in a sum of up to 2^24 terms, and a sum in binary32
// would move it past one action in a thousand.
#include "gx_launch.h"
#include "gx_policy.h"

namespace gx {

namespace {

// ordered bits: a < b as numbers <=> key(a) < key(b); -0 and +0 are one, NaN is -inf
__device__ __forceinline__ float clean(float x) { return x != x ? -__builtin_inff() : x + 0.0f; }
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float(k ^ ((k & 0x80000000u) ? 0x80000000u : 0xFFFFFFFFu));
}
constexpr uint32_t kKeyNegInf = 0x007FFFFFu;

// A row's parameters, read as the interface says.
struct RowParams {
  double inv_t;  // 1 / T
  double p, q;   // p >= 1: no cut
  int32_t k;     // 1 .. n
  double u;
};

__device__ __forceinline__ RowParams row_params(const SampleArgs& a, uint64_t r) {
  RowParams s;
  const float t = a.temperature ? a.temperature[r] : a.temperature_all;
  int32_t k = a.top_k ? a.top_k[r] : a.top_k_all;
  const float p = a.top_p ? a.top_p[r] : a.top_p_all;
  const float q = a.min_p ? a.min_p[r] : a.min_p_all;
  if (k <= 0 || k > a.n) k = a.n;
  const bool greedy = !(t > 0.0f);  // T = 0, and what reads as it
  s.inv_t = greedy ? 1.0 : 1.0 / (double)t;
  s.k = greedy ? 1 : k;
  s.p = p < 1.0f ? (p > 0.0f ? (double)p : 0.0) : 1.0;  // NaN: no cut
  s.q = q > 0.0f ? (q < 1.0f ? (double)q : 1.0) : 0.0;
  if (a.u) {
    const float u = a.u[r];
    s.u = u > 0.0f ? (u < 1.0f ? (double)u : 1.0 - 0x1.0p-53) : 0.0;
  } else {
    s.u = word_uniform(policy_word(policy_block(a.seed_lo, a.seed_hi, a.tick, a.env_index_base + r), a.tick));
  }
  return s;
}

// exp(z), z <= 0, to 2^-50 relative: z = k ln 2 + f, |f| <= ln 2 / 2, the series to f^13 / 13!
__device__ __forceinline__ double exp_neg(double z) {
  z = fmax(z, -746.0);  // exp is 0 there
  const double k = rint(z * 1.4426950408889634);
  double f = __builtin_fma(k, -6.93147180369123816490e-01, z);
  f = __builtin_fma(k, -1.90821492927058770002e-10, f);
  double e = 1.0 / 6227020800.0;
  e = __builtin_fma(e, f, 1.0 / 479001600.0);
  e = __builtin_fma(e, f, 1.0 / 39916800.0);
  e = __builtin_fma(e, f, 1.0 / 3628800.0);
  e = __builtin_fma(e, f, 1.0 / 362880.0);
  e = __builtin_fma(e, f, 1.0 / 40320.0);
  e = __builtin_fma(e, f, 1.0 / 5040.0);
  e = __builtin_fma(e, f, 1.0 / 720.0);
  e = __builtin_fma(e, f, 1.0 / 120.0);
  e = __builtin_fma(e, f, 1.0 / 24.0);
  e = __builtin_fma(e, f, 1.0 / 6.0);
  e = __builtin_fma(e, f, 0.5);
  e = __builtin_fma(e, f, 1.0);
  e = __builtin_fma(e, f, 1.0);
  return ldexp(e, (int)k);
}

// the weight of a logit: 1 at the largest, 0 at -inf and beside +inf
__device__ __forceinline__ double weight(float x, float m, double inv_t) {
  if (x == m) return 1.0;
  if (x == -__builtin_inff() || m == __builtin_inff()) return 0.0;
  return exp_neg(((double)x - (double)m) * inv_t);
}

constexpr int kWavesPerGroup = 4;

// One wave a row; every pass reads the row again (from a cache, after the first).
template <class T>
__global__ void __launch_bounds__(64 * kWavesPerGroup) sample_kernel(SampleArgs a) {
  const int lane = threadIdx.x & 63;
  for (uint64_t r = (uint64_t)blockIdx.x * kWavesPerGroup + (threadIdx.x >> 6); r < a.rows; r += (uint64_t)gridDim.x * kWavesPerGroup) {
    const T* row = static_cast<const T*>(a.logits) + (int64_t)r * a.row_stride;
    auto at = [&](int i) { return clean(to_f32(row[(int64_t)i * a.col_stride])); };
    const RowParams s = row_params(a, r);
    float m = -__builtin_inff();
    for (int i = lane; i < a.n; i += 64) m = fmaxf(m, at(i));
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
    if (m == -__builtin_inff()) {
      if (lane == 0) {
        a.actions[r] = -1;
        if (a.logprob) a.logprob[r] = -__builtin_inff();
      }
      continue;
    }
    auto count_from = [&](uint32_t key) {
      int c = 0;
      for (int i = lane; i < a.n; i += 64) c += key_of(at(i)) >= key ? 1 : 0;
      return wave_sum(c);
    };
    auto mass_from = [&](uint32_t key) {
      double c = 0.0;
      for (int i = lane; i < a.n; i += 64) {
        const float x = at(i);
        if (key_of(x) >= key) c += weight(x, m, s.inv_t);
      }
      return wave_sum(c);
    };
    // top-k: the largest key that at least k logits reach (-inf, of weight 0, is never kept)
    uint32_t t = kKeyNegInf + 1;
    int ties = a.n;
    if (s.k < a.n) {
      uint32_t lo = t, hi = key_of(m) + 1;  // count_from(lo) >= k (or t stays the lowest key), count_from(hi) < k
      while (hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (count_from(mid) >= s.k) lo = mid; else hi = mid;
      }
      t = lo;
      ties = s.k - count_from(t + 1);
    }
    if (s.p < 1.0) {
      const double wt = weight(value_of(t), m, s.inv_t);
      const double above = mass_from(t + 1);
      const int here = count_from(t) - count_from(t + 1);
      const double target = s.p * (above + (double)(here < ties ? here : ties) * wt);
      if (above > 0.0 && above >= target) {
        uint32_t lo = t + 1, hi = key_of(m) + 1;  // mass_from(lo) >= target; hi: beyond the largest
        while (hi - lo > 1) {
          const uint32_t mid = lo + (hi - lo) / 2;
          if (mass_from(mid) >= target) lo = mid; else hi = mid;
        }
        t = lo;
        ties = a.n;
      }
      // the j-th of those equal to t is in while what lies ahead of it, (j - 1) of them and all above, is below the target
      const double need = (target - mass_from(t + 1)) / weight(value_of(t), m, s.inv_t);
      const double j = ceil(need);
      const int first = j >= (double)a.n ? a.n : (j > 1.0 ? (int)j : 1);
      ties = first < ties ? first : ties;
    }
    // what is kept, in index order; ties before index i are counted along
    auto walk = [&](double stop, double* total) {
      double sum = 0.0;
      int seen = 0;
      int last = -1;
      for (int base = 0; base < a.n; base += 64) {
        const int i = base + lane;
        const float x = i < a.n ? at(i) : -__builtin_inff();
        const uint32_t key = key_of(x);
        const unsigned long long equal = __ballot(key == t && i < a.n);
        const int rank = seen + __popcll(equal & ((1ull << lane) - 1));
        seen += __popcll(equal);
        double w = 0.0;
        if (key > t || (key == t && rank < ties)) {
          w = weight(x, m, s.inv_t);
          if (w < s.q) w = 0.0;
        }
        double c = w;  // inclusive sums over the lanes
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
          const double v = __hiloint2double(__shfl_up(__double2hiint(c), d, 64), __shfl_up(__double2loint(c), d, 64));
          if (lane >= d) c += v;
        }
        c += sum;
        const unsigned long long kept = __ballot(w > 0.0);
        const unsigned long long past = __ballot(w > 0.0 && c > stop);
        if (past) return base + __ffsll(past) - 1;
        if (kept) last = base + 63 - __clzll(kept);
        sum = __hiloint2double(__shfl(__double2hiint(c), 63, 64), __shfl(__double2loint(c), 63, 64));
      }
      *total = sum;
      return last;
    };
    double total = 0.0, unused = 0.0;
    walk(__builtin_inf(), &total);
    const int action = walk(s.u * total, &unused);
    if (lane == 0) {
      a.actions[r] = action;
      if (a.logprob) {
        const float x = at(action);
        a.logprob[r] = (float)((x == m ? 0.0 : ((double)x - (double)m) * s.inv_t) - log(total));
      }
    }
  }
}

}  // namespace

size_t sample_workspace(const SampleArgs&, int) { return 0; }

hipError_t launch_sample_logits(const SampleArgs& a, int dtype, void*, int num_cus, hipStream_t stream) {
  const uint64_t groups = (a.rows + kWavesPerGroup - 1) / kWavesPerGroup;
  const dim3 grid((unsigned)(groups < (uint64_t)num_cus * 64 ? groups : (uint64_t)num_cus * 64));
  if (dtype == GX_F32) hipLaunchKernelGGL(sample_kernel<float>, grid, dim3(64 * kWavesPerGroup), 0, stream, a);
  else if (dtype == GX_F16) hipLaunchKernelGGL(sample_kernel<f16>, grid, dim3(64 * kWavesPerGroup), 0, stream, a);
  else hipLaunchKernelGGL(sample_kernel<bf16>, grid, dim3(64 * kWavesPerGroup), 0, stream, a);
  return hipGetLastError();
}

}  // namespace gx
