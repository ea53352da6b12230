// Embedding of Discrete observations: rows of a table by id, scaled, and the table's gradient (gx_embed).
#include "gx_launch.h"
#include "gx_policy.h"

namespace gx {

namespace {

__device__ __forceinline__ int64_t id_at(const EmbedArgs& a, uint64_t i) {
  return a.ids64 ? static_cast<const int64_t*>(a.ids)[i] : (int64_t) static_cast<const int32_t*>(a.ids)[i];
}

// N consecutive elements, at whatever address: gfx950 loads and stores vectors at any alignment
template <class T, int N> struct Pack { T v[N]; };
template <class T, int N> __device__ __forceinline__ Pack<T, N> load_pack(const T* p) {
  Pack<T, N> x;
  __builtin_memcpy(&x, p, sizeof x);
  return x;
}
template <class T, int N> __device__ __forceinline__ void store_pack(T* p, const Pack<T, N>& x) { __builtin_memcpy(p, &x, sizeof x); }

// ------------------------------------------------------------------ lookup ---
// Bound by the rows it writes.  Eight elements a lane (16 or 32 bytes each way); as many lanes a row as the row has
// such pieces, so a wave takes several rows of a narrow table; kRowsAhead rows a lane, so that many gathers are in flight
// behind the ids.
constexpr int kPiece = 8, kRowsAhead = 4;

template <class T, class R>
__global__ void __launch_bounds__(kBlock) lookup_kernel(EmbedArgs a, int lanes_shift) {
  const int lanes = 1 << lanes_shift, rows = kBlock >> lanes_shift;
  const int lane = threadIdx.x & (lanes - 1), row = threadIdx.x >> lanes_shift;
  for (uint64_t first = (uint64_t)blockIdx.x * (rows * kRowsAhead) + row; first < a.tokens; first += (uint64_t)gridDim.x * (rows * kRowsAhead)) {
    const T* from[kRowsAhead];
#pragma unroll
    for (int k = 0; k < kRowsAhead; k++) {
      const uint64_t i = first + k * rows;
      from[k] = nullptr;
      if (i < a.tokens) {
        const int64_t v = id_at(a, i);
        if (v >= 0 && v < a.n_states) from[k] = static_cast<const T*>(a.table) + v * a.table_stride;
      }
    }
    for (int64_t c = (int64_t)lane * kPiece; c < a.dim; c += (int64_t)lanes * kPiece) {
      if (c + kPiece <= a.dim) {
        Pack<T, kPiece> x[kRowsAhead];
#pragma unroll
        for (int k = 0; k < kRowsAhead; k++) {
          if (from[k]) x[k] = load_pack<T, kPiece>(from[k] + c);
          else
#pragma unroll
            for (int j = 0; j < kPiece; j++) x[k].v[j] = (T)0.0f;
        }
#pragma unroll
        for (int k = 0; k < kRowsAhead; k++) {
          const uint64_t i = first + k * rows;
          if (i >= a.tokens) continue;
          Pack<R, kPiece> y;
#pragma unroll
          for (int j = 0; j < kPiece; j++) y.v[j] = from_f32<R>(from[k] ? to_f32(x[k].v[j]) * a.scale : 0.0f);
          store_pack(static_cast<R*>(a.rows) + (int64_t)i * a.rows_stride + c, y);
        }
      } else {
#pragma unroll
        for (int k = 0; k < kRowsAhead; k++) {
          const uint64_t i = first + k * rows;
          if (i >= a.tokens) continue;
          R* to = static_cast<R*>(a.rows) + (int64_t)i * a.rows_stride;
          for (int64_t d = c; d < a.dim; d++) to[d] = from_f32<R>(from[k] ? to_f32(from[k][d]) * a.scale : 0.0f);
        }
      }
    }
  }
}

// ---------------------------------------------------------------- gradient ---
// table[v] = scale * sum of the rows whose id is v, by sorted tokens:
//   1  the pairs (id, token) are sorted by id, stably, by counting: digits of up to 10 bits, least significant first.
//      Ids outside the table sort behind everything as n_states.  One workgroup sorts up to kSortOne tokens alone, in
//      LDS; more are cut into tiles: counts per tile and digit, running sums over the tiles, and the scatter.
//      The workgroups of the first kernel that have nothing to sort clear the table meanwhile.
//   2  the sorted tokens are cut into chunks of equal length whatever the runs of equal ids, so that one state with most
//      of the tokens is no more work than many.  A group of lanes adds up one chunk: a run that lies inside is written
//      to the table, what a run has in a chunk it enters or leaves at a border goes to the workspace.
//   3  runs over several chunks are joined from those parts, in order, in binary64.
// Every addition's place follows from the ids alone: equal calls, equal bits.
constexpr int kSortOne = 8192, kSortThreads = 1024;  // tokens one workgroup sorts alone
constexpr int kTile = 4096;                          // tokens a workgroup of kBlock threads sorts, 16 a thread
constexpr int kMaxDigit = 10;

struct GradPlan {
  int bits, passes, digit;  // of the key, how many digits, bits of each
  bool one;                 // one workgroup sorts
  uint32_t tiles;
  int lanes_shift;          // lanes of a group: 8 columns each
  int64_t col_tiles;        // groups a row takes
  uint32_t chunk, chunks;   // tokens of a chunk, number of chunks
  size_t keys_a, keys_b, order_a, order_b, counts, totals, parts, bytes;  // offsets into the workspace
};

// a launch has fewer than 2^32 threads: beyond that the workgroups go round
unsigned capped(uint64_t blocks) { return (unsigned)(blocks < (1u << 22) ? blocks : 1u << 22); }

int shift_for(int64_t dim, int most) {
  int s = 0;
  while (s < most && ((int64_t)kPiece << s) < dim) s++;
  return s;
}

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

GradPlan grad_plan(const EmbedArgs& a, int num_cus) {
  GradPlan p{};
  const uint64_t n = a.tokens;
  p.bits = 64 - __builtin_clzll((unsigned long long)a.n_states);  // 0 .. n_states
  p.passes = (p.bits + kMaxDigit - 1) / kMaxDigit;
  p.digit = (p.bits + p.passes - 1) / p.passes;
  p.one = n <= (uint64_t)kSortOne;
  p.tiles = (uint32_t)((n + kTile - 1) / kTile);
  const int64_t pieces = (a.dim + kPiece - 1) / kPiece;
  p.lanes_shift = shift_for(a.dim, 6);
  p.col_tiles = (pieces + (1 << p.lanes_shift) - 1) >> p.lanes_shift;
  // chunks: enough lanes to fill the card (16 waves a compute unit), not fewer than 8 tokens, not more than 512
  const uint64_t want = ((uint64_t)num_cus * 16 * 64 >> p.lanes_shift) / (uint64_t)p.col_tiles;
  uint64_t chunk = want ? (n + want - 1) / want : n;
  chunk = chunk < 8 ? 8 : (chunk > 512 ? 512 : chunk);
  p.chunk = (uint32_t)((chunk + 7) & ~7ull);
  p.chunks = (uint32_t)((n + p.chunk - 1) / p.chunk);
  size_t at = 0;
  auto take = [&](size_t bytes) { size_t o = at; at += up256(bytes); return o; };
  p.keys_a = take(n * 4);
  p.order_a = take(n * 4);
  if (!p.one) {
    if (p.passes > 1) {
      p.keys_b = take(n * 4);
      p.order_b = take(n * 4);
    }
    p.counts = take((size_t)p.tiles * 4 << p.digit);
    p.totals = take((size_t)4 << p.digit);
  }
  if (p.chunks > 1) p.parts = take((size_t)p.chunks * 2 * (size_t)a.dim * 4);
  p.bytes = n ? at : 0;
  return p;
}

__device__ __forceinline__ uint32_t sort_key(const EmbedArgs& a, uint64_t i) {
  const int64_t v = id_at(a, i);
  return v >= 0 && v < a.n_states ? (uint32_t)v : (uint32_t)a.n_states;
}

// clears the table with the workgroups `block` of `blocks`
template <class T>
__device__ __forceinline__ void clear_table(const EmbedArgs& a, uint64_t block, uint64_t blocks) {
  T* table = static_cast<T*>(a.table);
  constexpr int kWide = 16 / sizeof(T);
  if (a.table_stride == a.dim) {  // one stretch: 16 bytes a lane from the first aligned address on
    const uint64_t n = (uint64_t)a.n_states * (uint64_t)a.dim;
    uint64_t head = ((16 - ((uintptr_t)table & 15)) & 15) / sizeof(T);
    head = head < n ? head : n;
    const uint64_t wide = (n - head) / kWide, tail = head + wide * kWide;
    uint4* to = reinterpret_cast<uint4*>(table + head);
    for (uint64_t i = block * blockDim.x + threadIdx.x; i < wide; i += blocks * blockDim.x) to[i] = make_uint4(0, 0, 0, 0);
    if (block == 0) {
      if (threadIdx.x < head) table[threadIdx.x] = (T)0.0f;
      if (tail + threadIdx.x < n) table[tail + threadIdx.x] = (T)0.0f;
    }
    return;
  }
  for (uint64_t v = block; v < (uint64_t)a.n_states; v += blocks)
    for (int64_t c = threadIdx.x; c < a.dim; c += blockDim.x) table[(int64_t)v * a.table_stride + c] = (T)0.0f;
}

template <class T>
__global__ void __launch_bounds__(kBlock) clear_kernel(EmbedArgs a) { clear_table<T>(a, blockIdx.x, gridDim.x); }

// LDS of one wave: its operations are executed in order; this keeps the compiler to that order too
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// lanes of the wave that hold the same digit (among `live` ones)
__device__ __forceinline__ unsigned long long same_digit(uint32_t d, int bits, unsigned long long live) {
  unsigned long long m = live;
  for (int b = 0; b < bits; b++) {
    const unsigned long long ones = __ballot((d >> b) & 1);
    m &= (d >> b) & 1 ? ones : ~ones;
  }
  return m;
}

// Exclusive running sums of n values in LDS by the whole workgroup (n <= 4 x its threads); sums[] holds one per wave.
__device__ __forceinline__ void scan_lds(uint32_t* values, int n, uint32_t* sums) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t v[4], total = 0;
#pragma unroll
  for (int k = 0; k < 4; k++) {
    const int i = (int)threadIdx.x * 4 + k;
    v[k] = i < n ? values[i] : 0;
    total += v[k];
  }
  uint32_t run = total;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t o = __shfl_up(run, d, 64);
    if (lane >= d) run += o;
  }
  if (lane == 63) sums[wave] = run;
  __syncthreads();
  uint32_t base = run - total;
  for (int w = 0; w < wave; w++) base += sums[w];
#pragma unroll
  for (int k = 0; k < 4; k++) {
    const int i = (int)threadIdx.x * 4 + k;
    if (i < n) values[i] = base;
    base += v[k];
  }
  __syncthreads();
}

// Up to kSortOne tokens by one workgroup: digits of 5 bits (the counters of 16 waves fit beside the pairs in LDS), each
// wave owning a contiguous stretch, so that (digit, wave) order keeps equal ids in the order of their tokens.
constexpr int kOneBits = 5;
template <class T>
__global__ void __launch_bounds__(kSortThreads) sort_one_kernel(EmbedArgs a, int bits, uint32_t* keys_out, uint32_t* order_out) {
  if (blockIdx.x) {
    clear_table<T>(a, blockIdx.x - 1, gridDim.x - 1);
    return;
  }
  constexpr int kWaves = kSortThreads / 64, kEach = kSortOne / kSortThreads, kBins = 1 << kOneBits;
  __shared__ uint32_t keys[kSortOne];
  __shared__ uint16_t order[kSortOne];
  __shared__ uint32_t counts[kBins * kWaves];  // [digit][wave]
  __shared__ uint32_t sums[kWaves];
  const int n = (int)a.tokens, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t k[kEach], o[kEach];
  // element e of this lane is token wave * 512 + e * 64 + lane
  const int base = wave * (64 * kEach) + lane;
#pragma unroll
  for (int e = 0; e < kEach; e++) {
    const int i = base + e * 64;
    k[e] = i < n ? sort_key(a, i) : 0xFFFFFFFFu;
    o[e] = i;
  }
  for (int shift = 0; shift < bits; shift += kOneBits) {
    if (threadIdx.x < kBins * kWaves) counts[threadIdx.x] = 0;
    static_assert(kBins * kWaves <= kSortThreads, "one counter a thread");
    __syncthreads();
    uint32_t rank[kEach];
#pragma unroll
    for (int e = 0; e < kEach; e++) {
      const bool live = base + e * 64 < n;
      const uint32_t d = (k[e] >> shift) & (kBins - 1);
      const unsigned long long same = same_digit(d, kOneBits, __ballot(live));
      uint32_t before = 0;
      if (live) before = counts[d * kWaves + wave];
      wave_order();
      rank[e] = before + __popcll(same & ((1ull << lane) - 1));
      if (live && (same & ((1ull << lane) - 1)) == 0) counts[d * kWaves + wave] = before + __popcll(same);
      wave_order();
    }
    __syncthreads();
    scan_lds(counts, kBins * kWaves, sums);
#pragma unroll
    for (int e = 0; e < kEach; e++)
      if (base + e * 64 < n) {
        const uint32_t to = counts[((k[e] >> shift) & (kBins - 1)) * kWaves + wave] + rank[e];
        keys[to] = k[e];
        order[to] = (uint16_t)o[e];
      }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kEach; e++) {
      const int i = base + e * 64;
      if (i < n) {
        k[e] = keys[i];
        o[e] = order[i];
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int e = 0; e < kEach; e++) {
    const int i = base + e * 64;
    if (i < n) {
      keys_out[i] = k[e];
      order_out[i] = o[e];
    }
  }
}

// counts[digit][tile]; the workgroups behind the tiles clear the table
template <class T>
__global__ void __launch_bounds__(kBlock) count_kernel(EmbedArgs a, const uint32_t* keys, uint32_t tiles, int shift, int digit, uint32_t* counts) {
  if (blockIdx.x >= tiles) {
    clear_table<T>(a, blockIdx.x - tiles, gridDim.x - tiles);
    return;
  }
  __shared__ uint32_t bins[1 << kMaxDigit];
  const int n_bins = 1 << digit;
  for (int b = threadIdx.x; b < n_bins; b += kBlock) bins[b] = 0;
  __syncthreads();
  const uint64_t first = (uint64_t)blockIdx.x * kTile;
#pragma unroll
  for (int e = 0; e < kTile / kBlock; e++) {
    const uint64_t i = first + e * kBlock + threadIdx.x;
    if (i < a.tokens) atomicAdd(&bins[((keys ? keys[i] : sort_key(a, i)) >> shift) & (n_bins - 1)], 1u);  // counts: order does not matter
  }
  __syncthreads();
  for (int b = threadIdx.x; b < n_bins; b += kBlock) counts[(size_t)b * tiles + blockIdx.x] = bins[b];
}

// running sums of one digit's counts over the tiles, in place, and the digit's total
__global__ void __launch_bounds__(kBlock) scan_tiles_kernel(uint32_t* counts, uint32_t tiles, uint32_t* totals) {
  __shared__ uint32_t sums[kBlock / 64];
  uint32_t* row = counts + (size_t)blockIdx.x * tiles;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t before = 0;
  for (uint32_t at = 0; at < tiles; at += kBlock * 4) {
    uint32_t v[4], total = 0;
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const uint32_t i = at + threadIdx.x * 4 + k;
      v[k] = i < tiles ? row[i] : 0;
      total += v[k];
    }
    uint32_t run = total;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t o = __shfl_up(run, d, 64);
      if (lane >= d) run += o;
    }
    if (lane == 63) sums[wave] = run;
    __syncthreads();
    uint32_t base = before + run - total, all = 0;
    for (int w = 0; w < kBlock / 64; w++) {
      if (w < wave) base += sums[w];
      all += sums[w];
    }
    before += all;
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const uint32_t i = at + threadIdx.x * 4 + k;
      if (i < tiles) row[i] = base;
      base += v[k];
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = before;
}

__global__ void __launch_bounds__(kBlock) scatter_kernel(EmbedArgs a, const uint32_t* keys, const uint32_t* order, uint32_t tiles, int shift,
                                                         int digit, const uint32_t* counts, const uint32_t* totals, uint32_t* keys_out,
                                                         uint32_t* order_out) {
  constexpr int kWaves = kBlock / 64, kEach = kTile / kBlock;
  __shared__ uint32_t place[1 << kMaxDigit];                // where the digit's next token of this tile goes
  __shared__ uint16_t seen[kWaves][1 << kMaxDigit];         // tokens of the digit in each wave's stretch
  __shared__ uint32_t sums[kWaves];
  const int n_bins = 1 << digit, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int b = threadIdx.x; b < n_bins; b += kBlock) {
    place[b] = totals[b];
#pragma unroll
    for (int w = 0; w < kWaves; w++) seen[w][b] = 0;
  }
  __syncthreads();
  scan_lds(place, n_bins, sums);
  for (int b = threadIdx.x; b < n_bins; b += kBlock) place[b] += counts[(size_t)b * tiles + blockIdx.x];
  const uint64_t first = (uint64_t)blockIdx.x * kTile + wave * (64 * kEach) + lane;
  uint32_t k[kEach], rank[kEach];
#pragma unroll
  for (int e = 0; e < kEach; e++) {
    const uint64_t i = first + e * 64;
    const bool live = i < a.tokens;
    k[e] = live ? (keys ? keys[i] : sort_key(a, i)) : 0;
    const uint32_t d = (k[e] >> shift) & (n_bins - 1);
    const unsigned long long same = same_digit(d, digit, __ballot(live));
    uint32_t before = 0;
    if (live) before = seen[wave][d];
    wave_order();
    rank[e] = before + __popcll(same & ((1ull << lane) - 1));
    if (live && (same & ((1ull << lane) - 1)) == 0) seen[wave][d] = (uint16_t)(before + __popcll(same));
    wave_order();
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < kEach; e++) {
    const uint64_t i = first + e * 64;
    if (i >= a.tokens) continue;
    const uint32_t d = (k[e] >> shift) & (n_bins - 1);
    uint32_t to = place[d] + rank[e];
    for (int w = 0; w < wave; w++) to += seen[w][d];
    keys_out[to] = k[e];
    order_out[to] = order ? order[i] : (uint32_t)i;
  }
}

template <class T>
__device__ __forceinline__ void put(const EmbedArgs& a, uint32_t key, int64_t c, double sum) {
  T* to = static_cast<T*>(a.table) + (int64_t)key * a.table_stride + c;
  const double old = a.accumulate ? (double)to_f32(*to) : 0.0;
  *to = from_f32<T>((float)(sum * (double)a.scale + old));
}

template <class T>
__device__ __forceinline__ void put_piece(const EmbedArgs& a, uint32_t key, int64_t c, int cols, const float* sum) {
  if (cols < kPiece) {
    for (int j = 0; j < kPiece; j++)
      if (j < cols) put<T>(a, key, c + j, (double)sum[j]);
    return;
  }
  T* to = static_cast<T*>(a.table) + (int64_t)key * a.table_stride + c;
  Pack<T, kPiece> y;
  if (a.accumulate) y = load_pack<T, kPiece>(to);
#pragma unroll
  for (int j = 0; j < kPiece; j++)
    y.v[j] = from_f32<T>((float)((double)sum[j] * (double)a.scale + (a.accumulate ? (double)to_f32(y.v[j]) : 0.0)));
  store_pack(to, y);
}

// One group of lanes a chunk and stretch of columns, eight columns a lane, eight rows in flight.
template <class T, class R>
__global__ void __launch_bounds__(kBlock) sum_kernel(EmbedArgs a, int lanes_shift, int64_t col_tiles, uint32_t chunk, uint32_t chunks,
                                                     const uint32_t* keys, const uint32_t* order, float* parts) {
  constexpr int kAhead = 8;
  const int lane = threadIdx.x & ((1 << lanes_shift) - 1);
  const uint64_t groups = (uint64_t)chunks * (uint64_t)col_tiles, stride = (uint64_t)gridDim.x * (kBlock >> lanes_shift);
  for (uint64_t group = (uint64_t)blockIdx.x * (kBlock >> lanes_shift) + (threadIdx.x >> lanes_shift); group < groups; group += stride) {
    const uint64_t which = group / (uint64_t)col_tiles;
    const int64_t c = ((int64_t)(group % (uint64_t)col_tiles) << lanes_shift) * kPiece + (int64_t)lane * kPiece;
    if (c >= a.dim) continue;
    const uint32_t first = (uint32_t)which * chunk;
    const uint32_t n = (uint32_t)a.tokens, end = n - first < chunk ? n : first + chunk;
    const int cols = a.dim - c < kPiece ? (int)(a.dim - c) : kPiece;
    float sum[kPiece] = {};
    uint32_t current = keys[first];
    // a part, not a run: entered from the chunk before, or left into the next one
    bool entered = first > 0 && keys[first - 1] == current;
    const bool left = end < n && keys[end] == keys[end - 1];
    auto flush = [&](bool part, int which_part) {
      if (current >= (uint32_t)a.n_states) return;
      if (!part) {
        put_piece<T>(a, current, c, cols, sum);
        return;
      }
      float* to = parts + ((size_t)which * 2 + which_part) * (size_t)a.dim + c;
      if (cols == kPiece) {
        Pack<float, kPiece> y;
#pragma unroll
        for (int j = 0; j < kPiece; j++) y.v[j] = sum[j];
        store_pack(to, y);
      } else {
#pragma unroll
        for (int j = 0; j < kPiece; j++)
          if (j < cols) to[j] = sum[j];
      }
    };
    for (uint32_t at = first; at < end; at += kAhead) {
      uint32_t key[kAhead];
      Pack<R, kPiece> x[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; k++) {
        const uint32_t i = at + k < end ? at + k : end - 1;
        key[k] = keys[i];
        const R* from = static_cast<const R*>(a.rows) + (int64_t)order[i] * a.rows_stride + c;
        if (cols == kPiece) x[k] = load_pack<R, kPiece>(from);
        else
#pragma unroll
          for (int j = 0; j < kPiece; j++) x[k].v[j] = j < cols ? from[j] : (R)0.0f;
      }
#pragma unroll
      for (int k = 0; k < kAhead; k++) {
        if (at + k >= end) break;
        if (key[k] != current) {
          flush(entered, 0);
          entered = false;
          current = key[k];
#pragma unroll
          for (int j = 0; j < kPiece; j++) sum[j] = 0.0f;
        }
#pragma unroll
        for (int j = 0; j < kPiece; j++) sum[j] += to_f32(x[k].v[j]);
      }
    }
    // the last run: a chunk that a single run enters and leaves has one part, the first
    flush(entered || left, entered ? 0 : 1);
  }
}

// The runs that leave the chunk they begin in: one workgroup each and 64 columns, 16 groups of 16 lanes that take every
// 16th part, then added in order.
template <class T>
__global__ void __launch_bounds__(kBlock) join_kernel(EmbedArgs a, uint32_t chunk, uint32_t chunks, const uint32_t* keys, const float* parts) {
  const uint32_t n = (uint32_t)a.tokens;
  const uint64_t col_tiles = (uint64_t)(a.dim + 63) / 64;
  __shared__ double sums[16][64];
  const int group = threadIdx.x >> 4, lane = threadIdx.x & 15;
  // (uniform over the workgroup throughout; the last chunk has nothing to join)
  for (uint64_t b = blockIdx.x; b < (uint64_t)(chunks - 1) * col_tiles; b += gridDim.x) {
    const uint32_t c0 = (uint32_t)(b / col_tiles);
    const int64_t col0 = (int64_t)(b % col_tiles) * 64;
    const uint32_t end = (c0 + 1) * chunk;
    const uint32_t key = keys[end - 1];
    if (keys[end] != key || key >= (uint32_t)a.n_states) continue;
    if (c0 > 0 && keys[end - chunk - 1] == key) continue;  // began before this chunk
    // the run's last token: the first place in [end, n) with a larger key, by halving
    uint32_t lo = end, hi = n;
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2;
      if (keys[mid] == key) lo = mid + 1; else hi = mid;
    }
    const uint32_t last = (lo - 1) / chunk;  // chunks c0 .. last hold parts of it
    const int64_t c = col0 + lane * 4;
    const int cols = a.dim - c < 4 ? (int)(a.dim - c) : 4;  // may be <= 0
    double sum[4] = {};
    for (uint32_t k = c0 + group; k <= last; k += 16) {
      const float* from = parts + ((size_t)k * 2 + (k == c0 ? 1 : 0)) * (size_t)a.dim + c;
      if (cols == 4) {
        const Pack<float, 4> x = load_pack<float, 4>(from);
#pragma unroll
        for (int j = 0; j < 4; j++) sum[j] += (double)x.v[j];
      } else {
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (j < cols) sum[j] += (double)from[j];
      }
    }
#pragma unroll
    for (int j = 0; j < 4; j++) sums[group][lane * 4 + j] = sum[j];
    __syncthreads();
    if (threadIdx.x < 64 && col0 + threadIdx.x < a.dim) {
      double all = 0.0;
#pragma unroll
      for (int g = 0; g < 16; g++) all += sums[g][threadIdx.x];
      put<T>(a, key, col0 + threadIdx.x, all);
    }
    __syncthreads();
  }
}

template <class F> hipError_t by_type(int dtype, F f) {
  if (dtype == GX_F32) return f(0.0f);
  if (dtype == GX_F16) return f((f16)0.0f);
  return f((bf16)0.0f);
}

}  // namespace

hipError_t launch_embed_lookup(const EmbedArgs& a, int table, int rows, int, hipStream_t stream) {
  const int shift = shift_for(a.dim, 8);
  const uint64_t each = (uint64_t)(kBlock >> shift) * kRowsAhead;
  const dim3 grid(capped((a.tokens + each - 1) / each));
  return by_type(table, [&](auto t) {
    return by_type(rows, [&](auto r) {
      hipLaunchKernelGGL((lookup_kernel<decltype(t), decltype(r)>), grid, dim3(kBlock), 0, stream, a, shift);
      return hipGetLastError();
    });
  });
}

size_t embed_grad_workspace(const EmbedArgs& a, int num_cus) { return grad_plan(a, num_cus).bytes; }

hipError_t launch_embed_grad(const EmbedArgs& a, int table, int rows, void* workspace, int num_cus, hipStream_t stream) {
  const GradPlan p = grad_plan(a, num_cus);
  char* ws = static_cast<char*>(workspace);
  // workgroups that clear the table: 16 KiB each, at most 16 a compute unit
  const uint64_t clear_bytes = a.accumulate ? 0 : (uint64_t)a.n_states * (uint64_t)a.dim * (table == GX_F32 ? 4 : 2);
  uint64_t clear = (clear_bytes + 16383) / 16384;
  if (clear > (uint64_t)num_cus * 16) clear = (uint64_t)num_cus * 16;
  if (a.tokens == 0) {
    if (!clear) return hipSuccess;
    return by_type(table, [&](auto t) {
      hipLaunchKernelGGL(clear_kernel<decltype(t)>, dim3((unsigned)clear), dim3(kBlock), 0, stream, a);
      return hipGetLastError();
    });
  }
  uint32_t* keys = reinterpret_cast<uint32_t*>(ws + p.keys_a);
  uint32_t* order = reinterpret_cast<uint32_t*>(ws + p.order_a);
  float* parts = reinterpret_cast<float*>(ws + p.parts);
  return by_type(table, [&](auto t) -> hipError_t {
    using T = decltype(t);
    if (p.one) {
      hipLaunchKernelGGL(sort_one_kernel<T>, dim3((unsigned)(1 + (clear + 3) / 4)), dim3(kSortThreads), 0, stream, a, p.bits, keys, order);
    } else {
      uint32_t* counts = reinterpret_cast<uint32_t*>(ws + p.counts);
      uint32_t* totals = reinterpret_cast<uint32_t*>(ws + p.totals);
      uint32_t* other_keys = reinterpret_cast<uint32_t*>(ws + p.keys_b);
      uint32_t* other_order = reinterpret_cast<uint32_t*>(ws + p.order_b);
      // the last pass ends in (keys, order)
      const uint32_t *from_keys = nullptr, *from_order = nullptr;
      for (int pass = 0; pass < p.passes; pass++) {
        const bool to_a = (p.passes - 1 - pass) % 2 == 0;
        uint32_t* to_keys = to_a ? keys : other_keys;
        uint32_t* to_order = to_a ? order : other_order;
        const dim3 tiles(p.tiles), first((unsigned)(p.tiles + (pass == 0 ? clear : 0)));
        hipLaunchKernelGGL(count_kernel<T>, first, dim3(kBlock), 0, stream, a, from_keys, p.tiles, pass * p.digit, p.digit, counts);
        hipLaunchKernelGGL(scan_tiles_kernel, dim3(1u << p.digit), dim3(kBlock), 0, stream, counts, p.tiles, totals);
        hipLaunchKernelGGL(scatter_kernel, tiles, dim3(kBlock), 0, stream, a, from_keys, from_order, p.tiles, pass * p.digit, p.digit,
                           counts, totals, to_keys, to_order);
        from_keys = to_keys;
        from_order = to_order;
      }
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const uint64_t groups = (uint64_t)p.chunks * (uint64_t)p.col_tiles, per_block = kBlock >> p.lanes_shift;
    e = by_type(rows, [&](auto r) {
      hipLaunchKernelGGL((sum_kernel<T, decltype(r)>), dim3(capped((groups + per_block - 1) / per_block)), dim3(kBlock), 0, stream, a,
                         p.lanes_shift, p.col_tiles, p.chunk, p.chunks, keys, order, parts);
      return hipGetLastError();
    });
    if (e != hipSuccess || p.chunks < 2) return e;
    hipLaunchKernelGGL(join_kernel<T>, dim3(capped((uint64_t)(p.chunks - 1) * ((uint64_t)(a.dim + 63) / 64))), dim3(kBlock), 0, stream, a, p.chunk, p.chunks,
                       keys, parts);
    return hipGetLastError();
  });
}

}  // namespace gx
