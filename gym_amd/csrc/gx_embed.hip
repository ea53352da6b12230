// Embedding of Discrete observations: rows of a table by id, scaled, and the table's gradient (gx_embed).
#include "gx_launch.h"
#include "gx_policy.h"

namespace gx {

namespace {

__device__ __forceinline__ int64_t id_at(const EmbedArgs& a, uint64_t i) {
  return a.ids64 ? static_cast<const int64_t*>(a.ids)[i] : (int64_t) static_cast<const int32_t*>(a.ids)[i];
}

template <class T, class R>
__global__ void __launch_bounds__(kBlock) lookup_kernel(EmbedArgs a) {
  for (uint64_t i = blockIdx.x; i < a.tokens; i += gridDim.x) {
    const int64_t v = id_at(a, i);
    const bool inside = v >= 0 && v < a.n_states;
    const T* from = static_cast<const T*>(a.table) + (inside ? v : 0) * a.table_stride;
    R* to = static_cast<R*>(a.rows) + (int64_t)i * a.rows_stride;
    for (int64_t c = threadIdx.x; c < a.dim; c += kBlock) to[c] = from_f32<R>(inside ? to_f32(from[c]) * a.scale : 0.0f);
  }
}

// a wave per state and 64 columns looks through all ids
template <class T, class R>
__global__ void __launch_bounds__(64) grad_kernel(EmbedArgs a, int64_t col_tiles) {
  for (int64_t g = blockIdx.x; g < a.n_states * col_tiles; g += gridDim.x) {
    const int64_t v = g / col_tiles, c = (g % col_tiles) * 64 + threadIdx.x;
    double sum = 0.0;
    for (uint64_t base = 0; base < a.tokens; base += 64) {
      const uint64_t i = base + threadIdx.x;
      unsigned long long hit = __ballot(i < a.tokens && id_at(a, i) == v);
      while (hit) {
        const int l = __ffsll(hit) - 1;
        hit &= hit - 1;
        if (c < a.dim) sum += (double)to_f32(static_cast<const R*>(a.rows)[(int64_t)(base + l) * a.rows_stride + c]);
      }
    }
    if (c < a.dim) {
      T* to = static_cast<T*>(a.table) + v * a.table_stride + c;
      const double old = a.accumulate ? (double)to_f32(*to) : 0.0;
      *to = from_f32<T>((float)(sum * (double)a.scale + old));
    }
  }
}

template <class F> hipError_t by_types(int table, int rows, F f) {
  auto inner = [&](auto t) {
    if (rows == GX_F32) return f(t, 0.0f);
    if (rows == GX_F16) return f(t, __half());
    return f(t, __hip_bfloat16());
  };
  if (table == GX_F32) return inner(0.0f);
  if (table == GX_F16) return inner(__half());
  return inner(__hip_bfloat16());
}

}  // namespace

hipError_t launch_embed_lookup(const EmbedArgs& a, int table, int rows, int num_cus, hipStream_t stream) {
  const uint64_t most = (uint64_t)num_cus * 32;
  const dim3 grid((unsigned)(a.tokens < most ? a.tokens : most));
  return by_types(table, rows, [&](auto t, auto r) {
    hipLaunchKernelGGL((lookup_kernel<decltype(t), decltype(r)>), grid, dim3(kBlock), 0, stream, a);
    return hipGetLastError();
  });
}

size_t embed_grad_workspace(const EmbedArgs&, int) { return 0; }

hipError_t launch_embed_grad(const EmbedArgs& a, int table, int rows, void*, int num_cus, hipStream_t stream) {
  const int64_t col_tiles = (a.dim + 63) / 64, groups = a.n_states * col_tiles;
  const int64_t most = (int64_t)num_cus * 256;
  const dim3 grid((unsigned)(groups < most ? groups : most));
  return by_types(table, rows, [&](auto t, auto r) {
    hipLaunchKernelGGL((grad_kernel<decltype(t), decltype(r)>), grid, dim3(64), 0, stream, a, col_tiles);
    return hipGetLastError();
  });
}

}  // namespace gx
