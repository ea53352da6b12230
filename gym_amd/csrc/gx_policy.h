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

// ---- lanes of a wavefront ----
// the value of the lane whose number differs in the bits of M
template <int M> __device__ __forceinline__ uint32_t xor_lane(uint32_t v) {
  static_assert(M == 1 || M == 2 || M == 4 || M == 8 || M == 16 || M == 32, "one bit");
  if constexpr (M == 1) return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true);        // quad_perm 1 0 3 2
  else if constexpr (M == 2) return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true);   // quad_perm 2 3 0 1
  else if constexpr (M == 8) return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x128, 0xF, 0xF, true);  // row_ror 8, of 16
  else if constexpr (M == 32) return (uint32_t)__shfl_xor((int)v, 32, 64);
  else return (uint32_t)__builtin_amdgcn_ds_swizzle((int)v, M << 10 | 0x1F);
}
// a value that is the same in every lane, in scalar registers
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ float uniform(float v) { return __uint_as_float(uniform(__float_as_uint(v))); }
__device__ __forceinline__ double uniform(double v) { return __hiloint2double(uniform(__double2hiint(v)), uniform(__double2loint(v))); }
__device__ __forceinline__ unsigned long long uniform(unsigned long long v) {
  return (unsigned long long)uniform((uint32_t)(v >> 32)) << 32 | uniform((uint32_t)v);
}
// Running sums over groups of G lanes, the lane's own included.  Within a row of 16 by shifts that bring zeros in (and
// where a group is less than a row, nothing from the group before); then the last lane of a row into the next (rows 1
// and 3), and lane 31 into the upper half.
template <int CTRL, int ROWS> __device__ __forceinline__ int moved(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, true); }
template <int CTRL, int ROWS> __device__ __forceinline__ double moved(double v) {
  return __hiloint2double(moved<CTRL, ROWS>(__double2hiint(v)), moved<CTRL, ROWS>(__double2loint(v)));
}
template <int G, int D, class T> __device__ __forceinline__ T shifted_in(T v) {
  const T o = moved<0x110 + D, 0xF>(v);
  return G >= 16 || (threadIdx.x & (G - 1)) >= D ? o : (T)0;
}
template <int G, class T> __device__ __forceinline__ T running_sum(T v) {
  if constexpr (G > 1) v += shifted_in<G, 1>(v);
  if constexpr (G > 2) v += shifted_in<G, 2>(v);
  if constexpr (G > 4) v += shifted_in<G, 4>(v);
  if constexpr (G > 8) v += shifted_in<G, 8>(v);
  if constexpr (G > 16) v += moved<0x142, 0xA>(v);  // row_bcast 15
  if constexpr (G > 32) v += moved<0x143, 0xC>(v);  // row_bcast 31
  return v;
}
__device__ __forceinline__ double shfl_xor_f64(double v, int mask) {
  return __hiloint2double(__shfl_xor(__double2hiint(v), mask, 64), __shfl_xor(__double2loint(v), mask, 64));
}
__device__ __forceinline__ double shfl_f64(double v, int lane, int width = 64) {
  return __hiloint2double(__shfl(__double2hiint(v), lane, width), __shfl(__double2loint(v), lane, width));
}
// of the wave, in every lane: the same order of additions, so the same bits, in each
__device__ __forceinline__ double wave_sum(double v) { return shfl_f64(running_sum<64>(v), 63); }
__device__ __forceinline__ int wave_sum(int v) { return __shfl(running_sum<64>(v), 63, 64); }

}  // namespace gx
