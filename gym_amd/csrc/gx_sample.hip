// Actions from a policy's logits: temperature, top-k, top-p, min-p and a draw by a given random number (gx_sample).
//
// The kept set is a beginning of the order "logit descending, equal logits by index", so it is described by one logit t
// and a count j: everything above t, and the first j (by index) of those equal to t.  Weights exp((x - m) / T) and their
// sums are binary64 (or integers of 62 bits) throughout: which action u falls on is a border in a sum of up to 2^24 terms,
// and a sum in binary32 would move it past one action in a thousand.  The vector units do as many binary64 operations a
// cycle as binary32 ones, so this costs registers, not time.
//
// Three forms, by the number of actions:
//   up to 8      a lane a row, every pair of actions compared (row_kernel)
//   up to 256    16 or 64 lanes a row, the row sorted in registers where top-k or top-p ask for it (group_kernel)
//   more         a workgroup a row; the border of the kept set is found by histograms, never by a sort (wide_kernel)
#include "gx_launch.h"
#include "gx_policy.h"

namespace gx {

namespace {

constexpr float kInf = __builtin_inff();

// ordered bits: a < b as numbers <=> key(a) < key(b); -0 and +0 are one, NaN is -inf
__device__ __forceinline__ float clean(float x) { return x != x ? -kInf : x + 0.0f; }
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float(k ^ ((k & 0x80000000u) ? 0x80000000u : 0xFFFFFFFFu));
}

template <class T, int N> struct Elements { T v[N]; };
// N consecutive logits, at whatever address: gfx950 loads vectors at any alignment
template <class T, int N> __device__ __forceinline__ void load_logits(const T* p, float* x) {
  Elements<T, N> e;
  __builtin_memcpy(&e, p, sizeof e);
#pragma unroll
  for (int j = 0; j < N; j++) x[j] = clean(to_f32(e.v[j]));
}

// A row's parameters, read as the interface says.
struct RowParams {
  double inv_t;  // 1 / T
  double p, q;   // p = 1: no cut
  int32_t k;     // 1 .. n
  double u;
};

// CUT: top-k, top-p or min-p may leave something out
template <bool CUT> __device__ __forceinline__ RowParams row_params(const SampleArgs& a, uint64_t r) {
  RowParams s;
  bool greedy = a.greedy_all;
  s.inv_t = a.inv_t_all;
  if (a.temperature) {
    const float t = a.temperature[r];
    greedy = !(t > 0.0f);  // T = 0, and what reads as it
    s.inv_t = greedy ? 1.0 : 1.0 / (double)t;
  }
  s.k = a.n;
  s.p = 1.0;
  s.q = 0.0;
  if (CUT) {
    const int32_t k = a.top_k ? a.top_k[r] : a.top_k_all;
    const float p = a.top_p ? a.top_p[r] : a.top_p_all;
    const float q = a.min_p ? a.min_p[r] : a.min_p_all;
    if (k > 0 && k < a.n) s.k = k;
    if (greedy) s.k = 1;
    s.p = p < 1.0f ? (p > 0.0f ? (double)p : 0.0) : 1.0;  // NaN: no cut
    s.q = q > 0.0f ? (q < 1.0f ? (double)q : 1.0) : 0.0;
  }
  if (a.u) {
    const float u = a.u[r];
    s.u = u > 0.0f ? (u < 1.0f ? (double)u : 1.0 - 0x1.0p-53) : 0.0;
  } else {
    s.u = word_uniform(policy_word(policy_block(a.seed_lo, a.seed_hi, a.tick, a.env_index_base + r), a.tick));
  }
  return s;
}

// exp(z), z <= 0, to 1e-14 relative: z = k ln 2 + f, |f| <= ln 2 / 2, the series to f^11 / 11!
__device__ __forceinline__ double exp_neg(double z) {
  z = fmax(z, -746.0);  // exp is 0 there
  const double k = rint(z * 1.4426950408889634);
  double f = __builtin_fma(k, -0x1.62e42fefa39efp-1, z);  // k < 2^11: the product's error stays below 2^-43, of z's 2^-44
  double e = 1.0 / 39916800.0;
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
  return __builtin_ldexp(e, (int)k);
}

// log(c), c >= 1, to 1e-13: c = 2^k g, g in [sqrt(1/2), sqrt(2)), log g = 2 atanh((g - 1) / (g + 1))
__device__ __forceinline__ double log_from_one(double c) {
  int k;
  double g = __builtin_frexp(c, &k);
  if (g < 0.70710678118654752) {
    g += g;
    k -= 1;
  }
  const double d = g + 1.0;
  double r = __builtin_amdgcn_rcp(d);  // 2^-14 or better, doubled twice
  r = __builtin_fma(r, __builtin_fma(-d, r, 1.0), r);
  r = __builtin_fma(r, __builtin_fma(-d, r, 1.0), r);
  const double s = (g - 1.0) * r, s2 = s * s;
  double e = 1.0 / 17.0;
  e = __builtin_fma(e, s2, 1.0 / 15.0);
  e = __builtin_fma(e, s2, 1.0 / 13.0);
  e = __builtin_fma(e, s2, 1.0 / 11.0);
  e = __builtin_fma(e, s2, 1.0 / 9.0);
  e = __builtin_fma(e, s2, 1.0 / 7.0);
  e = __builtin_fma(e, s2, 1.0 / 5.0);
  e = __builtin_fma(e, s2, 1.0 / 3.0);
  e = __builtin_fma(e, s2, 1.0);
  return __builtin_fma((double)k, 0.69314718055994531, 2.0 * s * e);
}

// the weight of a logit: 1 at the largest, 0 at -inf and beside +inf
__device__ __forceinline__ double weight(float x, float m, double inv_t) {
  const double w = exp_neg(((double)x - (double)m) * inv_t);
  return x == m ? 1.0 : (x == -kInf || m == kInf ? 0.0 : w);
}

__device__ __forceinline__ void write_result(const SampleArgs& a, uint64_t r, int action, float x, float m, double inv_t, double total) {
  a.actions[r] = action;
  if (a.logprob) a.logprob[r] = action < 0 ? -kInf : (float)((x == m ? 0.0 : ((double)x - (double)m) * inv_t) - log_from_one(total));
}

// ------------------------------------------------------- up to 8 actions ---
// A lane a row.  Bound by the arithmetic about as much as by memory: N exponentials, and with a cut every pair of
// actions: the rank of an action and the mass ahead of it, which are all that the definition asks for.
template <class T, int N, bool CUT, bool PACKED>
__global__ void __launch_bounds__(kBlock) row_kernel(SampleArgs a) {
  for (uint64_t r = (uint64_t)blockIdx.x * kBlock + threadIdx.x; r < a.rows; r += (uint64_t)gridDim.x * kBlock) {
    const T* row = static_cast<const T*>(a.logits) + (int64_t)r * a.row_stride;
    float x[N];
    if (PACKED) load_logits<T, N>(row, x);
    else
#pragma unroll
      for (int i = 0; i < N; i++) x[i] = clean(to_f32(row[(int64_t)i * a.col_stride]));
    const RowParams s = row_params<CUT>(a, r);
    float m = x[0];
#pragma unroll
    for (int i = 1; i < N; i++) m = fmaxf(m, x[i]);
    double w[N];
#pragma unroll
    for (int i = 0; i < N; i++) w[i] = weight(x[i], m, s.inv_t);
    if (CUT) {
      int rank[N];
#pragma unroll
      for (int i = 0; i < N; i++) rank[i] = 0;
#pragma unroll
      for (int i = 0; i < N; i++)
#pragma unroll
        for (int j = i + 1; j < N; j++) {
          const bool later = x[j] > x[i];  // equal: the lower index first
          rank[i] += later ? 1 : 0;
          rank[j] += later ? 0 : 1;
        }
      double s1 = 0.0;
#pragma unroll
      for (int i = 0; i < N; i++) s1 += rank[i] < s.k ? w[i] : 0.0;
      const double target = s.p * s1;
      bool kept[N];
#pragma unroll
      for (int i = 0; i < N; i++) {
        double ahead = 0.0;
#pragma unroll
        for (int j = 0; j < N; j++) ahead += rank[j] < rank[i] ? w[j] : 0.0;
        kept[i] = rank[i] == 0 || (rank[i] < s.k && (s.p >= 1.0 || ahead < target) && w[i] >= s.q);
      }
#pragma unroll
      for (int i = 0; i < N; i++) w[i] = kept[i] ? w[i] : 0.0;
    }
    double total = 0.0;
#pragma unroll
    for (int i = 0; i < N; i++) total += w[i];
    const double stop = s.u * total;
    int action = -1;
    float chosen = 0.0f;
    double c = 0.0;
    bool open = true;
#pragma unroll
    for (int i = 0; i < N; i++) {
      c += w[i];
      // the first past the border; until one is, the last that is kept (where rounding put the border at the total)
      if (open && w[i] > 0.0) {
        action = i;
        chosen = x[i];
        open = !(c > stop);
      }
    }
    if (m == -kInf) action = -1;
    write_result(a, r, action, chosen, m, s.inv_t, total);
  }
}

// ----------------------------------------------------- up to 256 actions ---
// G lanes a row (16: four rows a wave), E consecutive actions a lane.  Bound by instructions.  With top-k or top-p the
// row's values are sorted in registers (a bitonic network: the values alone, not their indices, for t and j are all that
// is wanted), weighed in that order and summed along it; the draw then goes over the row as it lies.
template <int G> __device__ __forceinline__ float group_max(float v) {
#pragma unroll
  for (int d = 1; d < G; d <<= 1) v = fmaxf(v, __shfl_xor(v, d, 64));
  return v;
}
// running sums over the lanes of a group, without the lane's own
template <int G> __device__ __forceinline__ double group_before(double v, double* all) {
  const int lane = threadIdx.x & (G - 1);
  double run = v;
#pragma unroll
  for (int d = 1; d < G; d <<= 1) {
    const double o = __hiloint2double(__shfl_up(__double2hiint(run), d, G), __shfl_up(__double2loint(run), d, G));
    if (lane >= d) run += o;
  }
  *all = __hiloint2double(__shfl(__double2hiint(run), G - 1, G), __shfl(__double2loint(run), G - 1, G));
  const double before = __hiloint2double(__shfl_up(__double2hiint(run), 1, G), __shfl_up(__double2loint(run), 1, G));
  return lane ? before : 0.0;
}
template <int G> __device__ __forceinline__ unsigned long long group_ballot(bool b) {
  const unsigned long long m = __ballot(b);
  return G == 64 ? m : (m >> (threadIdx.x & 63 & ~(G - 1))) & ((1ull << (G & 63)) - 1);
}

// descending over index lane * E + e
template <int G, int E> __device__ __forceinline__ void group_sort(float* v) {
  const int lane = threadIdx.x & (G - 1);
#pragma unroll
  for (int size = 2; size <= G * E; size <<= 1) {
#pragma unroll
    for (int d = size >> 1; d >= 1; d >>= 1) {
      if (d >= E) {
        const bool low = !(lane & (d / E));                               // of the pair
        const bool down = size == G * E || !(lane & (size / E));          // this block's direction
        const bool larger = low == down;
#pragma unroll
        for (int e = 0; e < E; e++) {
          const float o = __shfl_xor(v[e], d / E, 64);
          v[e] = larger ? fmaxf(v[e], o) : fminf(v[e], o);
        }
      } else {
#pragma unroll
        for (int e = 0; e < E; e++)
          if (!(e & d)) {
            const bool down = size == G * E ? true : (size >= E ? !(lane & (size / E)) : !(e & size));
            const float hi = fmaxf(v[e], v[e + d]), lo = fminf(v[e], v[e + d]);
            v[e] = down ? hi : lo;
            v[e + d] = down ? lo : hi;
          }
      }
    }
  }
}

template <class T, int G, int E, bool CUT, bool PACKED>
__global__ void __launch_bounds__(kBlock) group_kernel(SampleArgs a) {
  constexpr int kRows = kBlock / G;
  const int lane = threadIdx.x & (G - 1), first = lane * E;
  // (a group whose rows are done goes on with the last row, unwritten: its wave's other groups need its lanes)
  for (uint64_t r0 = (uint64_t)blockIdx.x * kRows; r0 < a.rows; r0 += (uint64_t)gridDim.x * kRows) {
    const uint64_t mine = r0 + threadIdx.x / G;
    const bool live = mine < a.rows;
    const uint64_t r = live ? mine : a.rows - 1;
    const T* row = static_cast<const T*>(a.logits) + (int64_t)r * a.row_stride;
    float x[E];
    if (PACKED && first + E <= a.n) load_logits<T, E>(row + first, x);
    else
#pragma unroll
      for (int e = 0; e < E; e++) x[e] = first + e < a.n ? clean(to_f32(row[(int64_t)(first + e) * a.col_stride])) : -kInf;
    const RowParams s = row_params<CUT>(a, r);
    float m = x[0];
#pragma unroll
    for (int e = 1; e < E; e++) m = fmaxf(m, x[e]);
    m = group_max<G>(m);
    double w[E];
#pragma unroll
    for (int e = 0; e < E; e++) w[e] = weight(x[e], m, s.inv_t);
    if (CUT) {
      if (__any(s.k < a.n || s.p < 1.0)) {
        float v[E];
#pragma unroll
        for (int e = 0; e < E; e++) v[e] = x[e];
        group_sort<G, E>(v);
        double sw[E], sum = 0.0;
#pragma unroll
        for (int e = 0; e < E; e++) {
          sw[e] = first + e < s.k ? weight(v[e], m, s.inv_t) : 0.0;
          sum += sw[e];
        }
        double s1, ahead = group_before<G>(sum, &s1);
        const double target = s.p * s1;
        int count = 0;  // kept: a beginning of the order
        float t = kInf;
#pragma unroll
        for (int e = 0; e < E; e++) {
          const bool in = first + e == 0 || (first + e < s.k && (s.p >= 1.0 || ahead < target) && v[e] > -kInf);
          ahead += sw[e];
          count += __popcll(group_ballot<G>(in));
          if (in) t = v[e];  // descending: the lane's last one kept is its smallest
        }
#pragma unroll
        for (int d = 1; d < G; d <<= 1) t = fminf(t, __shfl_xor(t, d, 64));
        int above = 0, equal = 0;
#pragma unroll
        for (int e = 0; e < E; e++) {
          above += __popcll(group_ballot<G>(x[e] > t));
          equal += x[e] == t ? 1 : 0;
        }
        int before = 0;  // ties at lower indices
#pragma unroll
        for (int d = 1, run = equal; d < G; d <<= 1) {
          const int o = __shfl_up(run, d, G);
          if (lane >= d) run += o;
          before = run - equal;
        }
        const int ties = count - above;
#pragma unroll
        for (int e = 0; e < E; e++) {
          const bool tie = x[e] == t;
          if (x[e] < t || (tie && before >= ties)) w[e] = 0.0;
          before += tie ? 1 : 0;
        }
      }
#pragma unroll
      for (int e = 0; e < E; e++) w[e] = w[e] >= s.q ? w[e] : 0.0;
    }
    double sum = 0.0, total;
#pragma unroll
    for (int e = 0; e < E; e++) sum += w[e];
    double c = group_before<G>(sum, &total);
    const double stop = s.u * total;
    int past = -1, last = -1;  // this lane's first action past the border, its last one kept
    float x_past = 0.0f, x_last = 0.0f;
#pragma unroll
    for (int e = 0; e < E; e++) {
      c += w[e];
      if (w[e] > 0.0) {
        last = first + e;
        x_last = x[e];
        if (past < 0 && c > stop) {
          past = last;
          x_past = x_last;
        }
      }
    }
    const unsigned long long over = group_ballot<G>(past >= 0), kept = group_ballot<G>(last >= 0);
    // rounding may have put the border at the total: the last one kept then
    const int chosen_lane = over ? __ffsll(over) - 1 : (kept ? 63 - __clzll(kept) : 0);
    if (live && lane == chosen_lane) {
      const bool none = m == -kInf;
      write_result(a, r, none ? -1 : (over ? past : last), over ? x_past : x_last, m, s.inv_t, total);
    }
  }
}

// --------------------------------------------------- more than 256 actions ---
// A workgroup a row, which it reads from memory once and again from the caches.  The row is cut into at most SEGMENTS
// stretches of a multiple of 512 actions, a wave each, eight consecutive actions a lane.
//   without a cut   one pass: each segment's largest logit and the sum of its weights relative to that
//   with one        a pass for the largest logit (and, for top-p alone, the sum); a lower bound on what can be kept, so
//                   that the passes after it touch few elements: the k-th largest of the lanes' largest logits, or the
//                   weight below which all actions together weigh less than (1 - p) of the sum; a pass that puts what is
//                   above into BINS bins by m - x, with counts and integer masses (whose order of adding changes nothing);
//                   the bin the border falls into again by finer bins, until it holds one value; and a pass over
//                   what is kept
// then the segment u falls into, and in it the action.
constexpr int kWideSmall = 4096;
constexpr int kLaneRun = 8, kSegment = 64 * kLaneRun;

// low bits of the ordered key that are the same for every value of the type (all clear, or all set below zero)
template <class T> constexpr int kFixedBits = 0;
template <> constexpr int kFixedBits<f16> = 13;
template <> constexpr int kFixedBits<bf16> = 16;

template <int BLOCK, int BINS, int SEGMENTS> struct WideShared {
  double seg_sum[SEGMENTS];
  float seg_max[SEGMENTS];
  int seg_ties[SEGMENTS];
  unsigned long long mass[BINS];
  uint32_t count[BINS];
  double wave_f64[BLOCK / 64];
  unsigned long long wave_u64[BLOCK / 64];
  float wave_f32[2][BLOCK / 64];
  uint32_t wave_u32[BLOCK / 64];
  // the border's bin
  int bin;
  uint32_t bin_count, above_count;
  unsigned long long bin_mass, above_mass;
};

// of one wave's lanes, all lanes the result
__device__ __forceinline__ float wave_max(float v) { return group_max<64>(v); }

template <class T, int BLOCK, int BINS, int SEGMENTS, bool CUT, bool PACKED>
__global__ void __launch_bounds__(BLOCK) wide_kernel(SampleArgs a) {
  constexpr int kWaves = BLOCK / 64;
  __shared__ WideShared<BLOCK, BINS, SEGMENTS> sh;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // turns of 512 actions a segment takes, so that SEGMENTS are enough
  const int turns = (a.n + kSegment * SEGMENTS - 1) / (kSegment * SEGMENTS), seg_len = kSegment * turns;
  const int segments = (a.n + seg_len - 1) / seg_len;

  for (uint64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* row = static_cast<const T*>(a.logits) + (int64_t)r * a.row_stride;
    const RowParams s = row_params<CUT>(a, r);
    // the eight logits of this lane in a turn of a segment
    auto load = [&](int i, float* x) {
      if (PACKED && i + kLaneRun <= a.n) load_logits<T, kLaneRun>(row + i, x);
      else
#pragma unroll
        for (int j = 0; j < kLaneRun; j++) x[j] = i + j < a.n ? clean(to_f32(row[(int64_t)(i + j) * a.col_stride])) : -kInf;
    };
    auto each = [&](auto f) {  // f(segment, first action of this lane, its logits) over the wave's share of the row
      for (int g = wave; g < segments; g += kWaves)
        for (int t = 0; t < turns; t++) {
          const int i = g * seg_len + t * kSegment + lane * kLaneRun;
          float x[kLaneRun];
          load(i, x);
          f(g, x);
        }
    };
    auto block_max = [&](float v, int slot) {
      v = wave_max(v);
      if (lane == 0) sh.wave_f32[slot][wave] = v;
      __syncthreads();
      v = sh.wave_f32[slot][0];
#pragma unroll
      for (int w = 1; w < kWaves; w++) v = fmaxf(v, sh.wave_f32[slot][w]);
      return v;
    };
    auto block_sum = [&](double v) {
      v = wave_sum(v);
      if (lane == 0) sh.wave_f64[wave] = v;
      __syncthreads();
      v = 0.0;
#pragma unroll
      for (int w = 0; w < kWaves; w++) v += sh.wave_f64[w];
      __syncthreads();
      return v;
    };

    float m = -kInf;
    // what is kept: keys above `hi`, and the first `ties` of those in [lo, hi]
    uint32_t lo = 0, hi = 0;
    int ties = 0;
    bool ordered = false;  // some of those in [lo, hi] are left out
    if (!CUT) {
      // largest logit and sum of a segment: a lane's own first, then the wave's
      for (int g = wave; g < segments; g += kWaves) {
        float top = -kInf;
        double sum = 0.0;
        for (int t = 0; t < turns; t++) {
          float x[kLaneRun];
          load(g * seg_len + t * kSegment + lane * kLaneRun, x);
          float here = x[0];
#pragma unroll
          for (int j = 1; j < kLaneRun; j++) here = fmaxf(here, x[j]);
          if (here > top) {
            sum *= weight(top, here, s.inv_t);
            top = here;
          }
#pragma unroll
          for (int j = 0; j < kLaneRun; j++) sum += weight(x[j], top, s.inv_t) * (x[j] > -kInf ? 1.0 : 0.0);
        }
        const float seg_top = wave_max(top);
        sum = wave_sum(top > -kInf ? sum * weight(top, seg_top, s.inv_t) : 0.0);
        if (lane == 0) {
          sh.seg_max[g] = seg_top;
          sh.seg_sum[g] = sum;
        }
      }
      __syncthreads();
      for (int g = threadIdx.x; g < segments; g += BLOCK) m = fmaxf(m, sh.seg_max[g]);
      m = block_max(m, 0);
      for (int g = threadIdx.x; g < segments; g += BLOCK)
        if (sh.seg_max[g] > -kInf) sh.seg_sum[g] *= weight(sh.seg_max[g], m, s.inv_t);
      __syncthreads();
    } else {
      // ---- the largest logit; the smallest finite one; the sum, relative to the lane's own largest
      const bool by_k = s.k < a.n, by_p = s.p < 1.0, sums = by_p && !by_k;
      float top = -kInf, bottom = kInf;
      double sum = 0.0;
      each([&](int, const float* x) {
        float here = x[0];
#pragma unroll
        for (int j = 1; j < kLaneRun; j++) here = fmaxf(here, x[j]);
#pragma unroll
        for (int j = 0; j < kLaneRun; j++) bottom = fminf(bottom, x[j] > -kInf ? x[j] : kInf);
        if (here > top) {
          if (sums) sum *= weight(top, here, s.inv_t);
          top = here;
        }
        if (sums && top > -kInf)
#pragma unroll
          for (int j = 0; j < kLaneRun; j++) sum += weight(x[j], top, s.inv_t);
      });
      m = block_max(top, 0);
      bottom = -block_max(-bottom, 1);
      double s1 = sums ? block_sum(top > -kInf ? sum * weight(top, m, s.inv_t) : 0.0) : 0.0;
      if (m > -kInf) {
        // ---- a bound below everything that can be kept.  Weights below exp(-745) are 0.
        double bound = (double)m - 745.0 / s.inv_t;
        if (sums) bound = fmax(bound, (double)m + log(fmax((1.0 - s.p) * s1 / (double)a.n, 1e-320)) / s.inv_t);
        float from = fminf(m, fmaxf(bottom, (float)(bound - fabs(bound) * 1e-6)));
        if (m == kInf) from = kInf;
        if (by_k && s.k <= BLOCK && m < kInf) {
          // a value that k lanes' largest reach: halving between the smallest and the largest
          float low = from, high = m;
          for (int step = 0; step < 14; step++) {
            const float mid = low + (high - low) * 0.5f;
            if (!(mid > low && mid < high)) break;
            if (__syncthreads_count(top >= mid) >= s.k) low = mid; else high = mid;
          }
          if (__syncthreads_count(top >= low) >= s.k) from = low;
        }
        // ---- bins
        // masses as integers: the sum (at most k where it is not known) below 2^62
        const int scale_bits = 61 - __builtin_amdgcn_frexp_exp(sums ? s1 : (double)s.k);
        const float per = m > from && m < kInf ? (float)(BINS - 1) / (m - from) : 0.0f;
        auto bin_of = [&](float x) { return x == m ? 0 : (int)fminf((m - x) * per, (float)(BINS - 1)); };
        const uint32_t key_from = key_of(from), key_m = key_of(m);
        // the border by counts or by masses: the first bin where what lies up to its end reaches the target
        auto find_bin = [&](bool mass, uint32_t want_count, unsigned long long want_mass) {
          constexpr int kEach = BINS / BLOCK;
          uint32_t c = 0;
          unsigned long long w = 0;
#pragma unroll
          for (int e = 0; e < kEach; e++) {
            c += sh.count[threadIdx.x * kEach + e];
            w += sh.mass[threadIdx.x * kEach + e];
          }
          uint32_t rc = c;
          unsigned long long rw = w;
#pragma unroll
          for (int d = 1; d < 64; d <<= 1) {
            const uint32_t oc = __shfl_up(rc, d, 64);
            const unsigned long long ow = __shfl_up(rw, d, 64);
            if (lane >= d) { rc += oc; rw += ow; }
          }
          if (lane == 63) { sh.wave_u32[wave] = rc; sh.wave_u64[wave] = rw; }
          if (threadIdx.x == 0) sh.bin = -1;
          __syncthreads();
          rc -= c;
          rw -= w;
          for (int v = 0; v < wave; v++) { rc += sh.wave_u32[v]; rw += sh.wave_u64[v]; }
#pragma unroll
          for (int e = 0; e < kEach; e++) {
            const uint32_t bc = sh.count[threadIdx.x * kEach + e];
            const unsigned long long bw = sh.mass[threadIdx.x * kEach + e];
            const bool before = mass ? rw < want_mass : rc < want_count, after = mass ? rw + bw >= want_mass : rc + bc >= want_count;
            if (bc && before && after) {
              sh.bin = threadIdx.x * kEach + e;
              sh.bin_count = bc;
              sh.bin_mass = bw;
              sh.above_count = rc;
              sh.above_mass = rw;
            }
            rc += bc;
            rw += bw;
          }
          __syncthreads();
          return sh.bin;
        };
        auto clear_bins = [&]() {
          for (int b = threadIdx.x; b < BINS; b += BLOCK) { sh.count[b] = 0; sh.mass[b] = 0; }
          __syncthreads();
        };
        auto put_in = [&](int b, float x) {
          atomicAdd(&sh.count[b], 1u);
          atomicAdd(&sh.mass[b], (unsigned long long)__builtin_ldexp(weight(x, m, s.inv_t), scale_bits));
        };
        auto coarse = [&]() {
          clear_bins();
          each([&](int, const float* x) {
#pragma unroll
            for (int j = 0; j < kLaneRun; j++)
              if (x[j] >= from) put_in(bin_of(x[j]), x[j]);
          });
          __syncthreads();
        };
        // the border: [lo, hi] that hold one value (or one action), what is above them, and how many of them are kept
        auto border = [&](bool mass, uint32_t want_count, unsigned long long want_mass) {
          if (find_bin(mass, want_count, want_mass) < 0) return false;
          {
            // the keys of the bin: bin_of falls as the key rises
            const int b = sh.bin;
            uint32_t l = key_from, h = key_m;
            while (l < h) {  // the smallest key whose bin is at most b
              const uint32_t mid = l + (h - l) / 2;
              if (bin_of(value_of(mid)) <= b) h = mid; else l = mid + 1;
            }
            lo = l;
            h = key_m;
            while (l < h) {  // the largest whose bin is at least b
              const uint32_t mid = l + (h - l + 1) / 2;
              if (bin_of(value_of(mid)) >= b) l = mid; else h = mid - 1;
            }
            hi = l;
          }
          while (sh.bin_count > 1 && (hi - lo) >> kFixedBits<T>) {
            const uint32_t above_count = sh.above_count;
            const unsigned long long above_mass = sh.above_mass;
            const int width = 32 - __clz(hi - lo), shift = width > __builtin_ctz(BINS) ? width - __builtin_ctz(BINS) : 0;
            __syncthreads();
            clear_bins();
            each([&](int, const float* x) {
#pragma unroll
              for (int j = 0; j < kLaneRun; j++) {
                const uint32_t key = key_of(x[j]);
                if (key >= lo && key <= hi) put_in((int)((hi - key) >> shift), x[j]);
              }
            });
            __syncthreads();
            find_bin(mass, want_count - above_count, want_mass - above_mass);
            hi -= (uint32_t)sh.bin << shift;
            const uint32_t low = hi - ((1u << shift) - 1);
            lo = low > lo && low <= hi ? low : lo;
            if (threadIdx.x == 0) {
              sh.above_count += above_count;
              sh.above_mass += above_mass;
            }
            __syncthreads();
          }
          // one value: that of the key with the type's fixed bits, in [lo, hi]
          if (mass) {
            const double one = (double)sh.bin_mass / (double)sh.bin_count;
            const double need = ceil((double)(want_mass - sh.above_mass) / one);
            ties = need < (double)sh.bin_count ? (int)need : (int)sh.bin_count;
            if (ties < 1) ties = 1;
          } else {
            ties = (int)(want_count - sh.above_count);
          }
          ordered = (uint32_t)ties < sh.bin_count;
          return true;
        };
        bool cut = false;
        if (by_k || by_p) {
          coarse();
          if (by_k) {
            cut = border(false, (uint32_t)s.k, 0);
            if (by_p) {
              unsigned long long all = 0;  // of the first k
              if (cut) {
                all = sh.above_mass + (unsigned long long)((double)sh.bin_mass / (double)sh.bin_count * (double)ties);
              } else {
                // fewer than k: everything above `from`
                for (int b = threadIdx.x; b < BINS; b += BLOCK) all += sh.mass[b];
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) all += __shfl_xor(all, d, 64);
                if (lane == 0) sh.wave_u64[wave] = all;
                __syncthreads();
                all = 0;
                for (int v = 0; v < kWaves; v++) all += sh.wave_u64[v];
                __syncthreads();
              }
              const unsigned long long want = (unsigned long long)ceil(s.p * (double)all);
              const uint32_t k_lo = lo, k_hi = hi;
              const int k_ties = ties;
              const bool k_cut = cut, k_ordered = ordered;
              if (cut) coarse();  // finer bins have taken their place
              const bool found = border(true, 0, want > 0 ? want : 1);
              // the border by mass counts only where it is the stricter one
              if (k_cut && (!found || hi < k_hi || (hi == k_hi && ties > k_ties))) {
                lo = k_lo; hi = k_hi; ties = k_ties; ordered = k_ordered;
                cut = true;
              } else {
                cut = found;
              }
            }
          } else {
            const unsigned long long want = (unsigned long long)ceil(s.p * __builtin_ldexp(s1, scale_bits));
            cut = border(true, 0, want > 0 ? want : 1);
          }
        }
        if (!cut) {  // everything above the bound
          lo = key_from;
          hi = key_from - 1;
          ties = 0;
          ordered = false;
        }
        __syncthreads();
        // ---- what is kept, by segments
        for (int g = wave; g < segments; g += kWaves) {
          double sum = 0.0;
          int here = 0;
          for (int t = 0; t < turns; t++) {
            float x[kLaneRun];
            load(g * seg_len + t * kSegment + lane * kLaneRun, x);
#pragma unroll
            for (int j = 0; j < kLaneRun; j++) {
              const uint32_t key = key_of(x[j]);
              const bool tie = key >= lo && key <= hi;
              here += tie ? 1 : 0;
              if (key > hi || (tie && !ordered)) {
                const double w = weight(x[j], m, s.inv_t);
                sum += w >= s.q ? w : 0.0;
              }
            }
          }
          sum = wave_sum(sum);
          if (ordered) here = wave_sum(here);
          if (lane == 0) {
            sh.seg_sum[g] = sum;
            sh.seg_ties[g] = here;
          }
        }
        __syncthreads();
      }
    }

    // ---- the segment, and in it the action: one wave's work
    if (wave == 0) {
      int action = -1;
      float chosen = 0.0f;
      double total = 0.0;
      if (m > -kInf) {
        const int per_lane = (segments + 63) / 64, g0 = lane * per_lane, g1 = min(segments, g0 + per_lane);
        // ties are kept by index: how many lie in the segments before.  They weigh the same.
        double tie_weight = 0.0;
        int tie_before = 0;
        if (CUT && ordered) {
          // the value in [lo, hi]: by the type's fixed bits, or (one binary32 value) lo = hi
          const uint32_t mask = (1u << kFixedBits<T>) - 1;
          const float t = value_of(hi & 0x80000000u ? hi & ~mask : (hi + 1 - (mask + 1)) | mask);
          tie_weight = weight(t, m, s.inv_t);
          if (tie_weight < s.q) tie_weight = 0.0;
          int mine = 0;
          for (int g = g0; g < g1; g++) mine += sh.seg_ties[g];
          int run = mine;
#pragma unroll
          for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(run, d, 64);
            if (lane >= d) run += o;
          }
          tie_before = run - mine;
        }
        auto kept_ties = [&](int before, int here) { return before >= ties ? 0 : min(here, ties - before); };
        double sum = 0.0;
        int tb = tie_before;
        for (int g = g0; g < g1; g++) {
          if (CUT && ordered) {
            sh.seg_sum[g] += (double)kept_ties(tb, sh.seg_ties[g]) * tie_weight;
            tb += sh.seg_ties[g];
          }
          sum += sh.seg_sum[g];
        }
        double c = group_before<64>(sum, &total);
        const double stop = s.u * total;
        // the lane's first segment past the border, and its last with anything kept
        int past = -1, last = -1, past_ties = 0, last_ties = 0;
        double past_before = 0.0;
        tb = tie_before;
        for (int g = g0; g < g1; g++) {
          const double v = sh.seg_sum[g];
          if (v > 0.0) {
            last = g;
            last_ties = tb;
            if (past < 0 && c + v > stop) {
              past = g;
              past_ties = tb;
              past_before = c;
            }
          }
          c += v;
          if (CUT && ordered) tb += sh.seg_ties[g];
        }
        const unsigned long long over = __ballot(past >= 0), any = __ballot(last >= 0);
        const int from_lane = over ? __ffsll(over) - 1 : 63 - __clzll(any);
        const int seg = __shfl(over ? past : last, from_lane, 64);
        int seen = __shfl(over ? past_ties : last_ties, from_lane, 64);
        // (rounding may have put the border at the total: then the last action of the last segment)
        double base = over ? __hiloint2double(__shfl(__double2hiint(past_before), from_lane, 64), __shfl(__double2loint(past_before), from_lane, 64))
                           : -__builtin_inf();
        bool found = false;
        for (int t = 0; t < turns && !found; t++) {
          const int i = seg * seg_len + t * kSegment + lane * kLaneRun;
          float x[kLaneRun];
          double w[kLaneRun], mine = 0.0;
          load(i, x);
          int equal = 0;
#pragma unroll
          for (int j = 0; j < kLaneRun; j++) {
            const uint32_t key = key_of(x[j]);
            equal += CUT && key >= lo && key <= hi ? 1 : 0;
          }
          int run = equal;
          if (CUT && ordered) {
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
              const int o = __shfl_up(run, d, 64);
              if (lane >= d) run += o;
            }
          }
          int rank = seen + run - equal;
          if (CUT && ordered) seen += __shfl(run, 63, 64);
#pragma unroll
          for (int j = 0; j < kLaneRun; j++) {
            const uint32_t key = key_of(x[j]);
            bool in = x[j] > -kInf;
            if (CUT) {
              const bool tie = key >= lo && key <= hi;
              in = key > hi || (tie && (!ordered || rank < ties));
              rank += tie ? 1 : 0;
            }
            w[j] = in ? weight(x[j], m, s.inv_t) : 0.0;
            if (CUT && w[j] < s.q) w[j] = 0.0;
            mine += w[j];
          }
          double all, b = base + group_before<64>(mine, &all);
          int p_at = -1, l_at = -1;
          float p_x = 0.0f, l_x = 0.0f;
#pragma unroll
          for (int j = 0; j < kLaneRun; j++) {
            b += w[j];
            if (w[j] > 0.0) {
              l_at = i + j;
              l_x = x[j];
              if (p_at < 0 && b > stop) {
                p_at = l_at;
                p_x = l_x;
              }
            }
          }
          const unsigned long long o = __ballot(p_at >= 0), k = __ballot(l_at >= 0);
          if (o || k) {  // until one is past the border, the last one kept so far
            const int who = o ? __ffsll(o) - 1 : 63 - __clzll(k);
            action = __shfl(o ? p_at : l_at, who, 64);
            chosen = __shfl(o ? p_x : l_x, who, 64);
            found = o != 0;
          }
          base += all;
        }
      }
      if (lane == 0) write_result(a, r, action, chosen, m, s.inv_t, total);
    }
    __syncthreads();
  }
}

}  // namespace

size_t sample_workspace(const SampleArgs&, int) { return 0; }

namespace {

template <class T, bool CUT, bool PACKED> hipError_t launch_rows(const SampleArgs& a, int num_cus, hipStream_t stream) {
  // a launch has fewer than 2^32 threads, and grids beyond what the card holds gain nothing: the workgroups go round
  auto grid = [&](uint64_t per_group) {
    const uint64_t groups = (a.rows + per_group - 1) / per_group, most = (uint64_t)num_cus * 64;
    return dim3((unsigned)(groups < most ? groups : most));
  };
  switch (a.n) {
#define GX_ROW(N) case N: hipLaunchKernelGGL((row_kernel<T, N, CUT, PACKED>), grid(kBlock), dim3(kBlock), 0, stream, a); return hipGetLastError()
    GX_ROW(1); GX_ROW(2); GX_ROW(3); GX_ROW(4); GX_ROW(5); GX_ROW(6); GX_ROW(7); GX_ROW(8);
#undef GX_ROW
    default: break;
  }
#define GX_GROUP(G, E)                                                                                                        \
  if (a.n <= G * E) {                                                                                                         \
    hipLaunchKernelGGL((group_kernel<T, G, E, CUT, PACKED>), grid(kBlock / G), dim3(kBlock), 0, stream, a);                   \
    return hipGetLastError();                                                                                                 \
  }
  GX_GROUP(16, 1) GX_GROUP(16, 2) GX_GROUP(16, 4) GX_GROUP(64, 2) GX_GROUP(64, 4)
#undef GX_GROUP
  if (a.n <= kWideSmall) hipLaunchKernelGGL((wide_kernel<T, 256, 512, 16, CUT, PACKED>), grid(1), dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((wide_kernel<T, 1024, 2048, 1024, CUT, PACKED>), grid(1), dim3(1024), 0, stream, a);
  return hipGetLastError();
}

template <class T> hipError_t launch_typed(const SampleArgs& a, int num_cus, hipStream_t stream) {
  const bool cut = a.temperature || a.top_k || a.top_p || a.min_p || a.greedy_all || (a.top_k_all > 0 && a.top_k_all < a.n) ||
                   a.top_p_all < 1.0f || a.min_p_all > 0.0f;
  const bool packed = a.col_stride == 1;
  if (cut) return packed ? launch_rows<T, true, true>(a, num_cus, stream) : launch_rows<T, true, false>(a, num_cus, stream);
  return packed ? launch_rows<T, false, true>(a, num_cus, stream) : launch_rows<T, false, false>(a, num_cus, stream);
}

}  // namespace

hipError_t launch_sample_logits(const SampleArgs& a, int dtype, void*, int num_cus, hipStream_t stream) {
  if (dtype == GX_F32) return launch_typed<float>(a, num_cus, stream);
  if (dtype == GX_F16) return launch_typed<f16>(a, num_cus, stream);
  return launch_typed<bf16>(a, num_cus, stream);
}

}  // namespace gx
