// What the operators between a policy and a batch share: their arguments as the kernels take them, the element types
// of a policy's tensors, and folds over a wavefront in a fixed order.
#pragma once

#include "gx_device.h"

namespace gx {

// gx_sample as the kernels take it
struct SampleArgs {
  const void* logits;
  uint64_t rows;
  int64_t row_stride, col_stride;
  int32_t n;
  int32_t top_k_all;
  float top_p_all, min_p_all;
  int32_t greedy_all;  // the common temperature is 0
  double inv_t_all;    // 1 / the common temperature
  const float* u;  // nullptr: from the generator, see u_of
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  int32_t* actions;
  float* logprob;  // or nullptr
  uint32_t seed_lo, seed_hi;
  uint64_t tick, env_index_base;
};

// gx_embed as the kernels take it
struct EmbedArgs {
  const void* ids;
  int32_t ids64;  // ids are int64
  int32_t accumulate;
  uint64_t tokens;
  int64_t n_states, dim, table_stride, rows_stride;
  void* table;
  void* rows;
  float scale;
};

using f16 = _Float16;
using bf16 = __bf16;
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(f16 v) { return (float)v; }
__device__ __forceinline__ float to_f32(bf16 v) { return (float)v; }
// to nearest, ties to even
template <class T> __device__ __forceinline__ T from_f32(float v) { return (T)v; }
// the binary32 value as it stands: the compiler would fold a product before the conversion into v_fma_mixlo_f16, which
// skips the product's own rounding and with it the agreement with the plain form
template <> __device__ __forceinline__ f16 from_f32<f16>(float v) {
  asm("" : "+v"(v));
  return (f16)v;
}

// butterfly folds: every lane ends with the same bits, whatever the values
__device__ __forceinline__ double shfl_xor_f64(double v, int mask) {
  return __hiloint2double(__shfl_xor(__double2hiint(v), mask, 64), __shfl_xor(__double2loint(v), mask, 64));
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += shfl_xor_f64(v, d);
  return v;
}
__device__ __forceinline__ int wave_sum(int v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d, 64);
  return v;
}

}  // namespace gx
