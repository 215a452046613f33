// Global gradient norm over many tensors, and clipping by it.
//
//   norm   = (sum over all tensors and elements of |g|^p)^(1/p)  (p = 1, 2) or max |g|
//   factor = min(1, max_norm / (norm + 1e-6))          g = round(g * factor)
//
// The tensors are cut into tiles of kTile elements; a launch covers up to kListMax tensors through a
// table in its arguments, so a captured graph replays it with no host work.  A workgroup adds up its
// tiles in fp64 (squares of fp32 gradients neither overflow nor lose the small ones, and the
// conversion is free under the loads), leaves one partial value, and a second launch joins the
// partial values in a fixed order: no atomics, and the result does not depend on timing.  A factor of one
// leaves the gradients as they are, so an ordinary step reads them once.
#include <algorithm>

#include "grace_common.h"
#include "grace_lm.h"

namespace grace {
namespace {

constexpr int kBlock = 256;
constexpr int kTile = 4096;
constexpr int kListMax = 240;    // 3.8 KB of kernel arguments
constexpr int kMaxBlocks = 2048;  // partial values per launch
constexpr int64_t kMaxLen = 1 << 29;  // elements per table entry: longer tensors take several

struct List {
  void* p[kListMax];
  uint32_t len[kListMax];        // elements, the type in the upper two bits
  int32_t start[kListMax + 1];   // first tile of each entry
  int32_t n;
};

__device__ __forceinline__ int find_entry(const List& t, int tile) {
  int lo = 0, hi = t.n - 1;  // last entry with start <= tile
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.start[mid] <= tile) lo = mid; else hi = mid - 1;
  }
  return lo;
}

template <int P>
__device__ __forceinline__ double join(double a, double b) {
  if constexpr (P == 0) return (b > a || b != b) ? b : a;  // a NaN stays
  else return a + b;
}
template <int P>
__device__ __forceinline__ double term(float v) {
  const double d = (double)v;
  if constexpr (P == 2) return d * d;
  else return fabs(d);
}

template <int P>
__device__ __forceinline__ double block_join(double v, double* scratch) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = join<P>(v, __shfl_xor(v, o, kWave));
  const int nw = blockDim.x >> 6;
  if (lane_id() == 0) scratch[wave_id()] = v;
  __syncthreads();
  v = scratch[0];
  for (int i = 1; i < nw; ++i) v = join<P>(v, scratch[i]);
  return v;
}

template <typename T, int P>
__device__ __forceinline__ double tile_norm(const T* __restrict__ p, int n) {
  double a = 0.0;
  constexpr int V = 16 / sizeof(T), U = kTile / kBlock / V;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = (u * kBlock + threadIdx.x) * V;
    if (i < n) {
      float x[V];
      load_vec(p + i, x, n - i);
#pragma unroll
      for (int k = 0; k < V; ++k) a = join<P>(a, term<P>(x[k]));
    }
  }
  return a;
}

template <int P>
__global__ __launch_bounds__(kBlock) void norm_part_kernel(List t, double* __restrict__ part) {
  double a = 0.0;
  for (int tile = blockIdx.x; tile < t.start[t.n]; tile += gridDim.x) {
    const int e = find_entry(t, tile);
    const int64_t at = (int64_t)(tile - t.start[e]) * kTile;
    const int n = (int)min((int64_t)(t.len[e] & 0x3fffffffu) - at, (int64_t)kTile);
    double v;
    switch (t.len[e] >> 30) {
      case 0: v = tile_norm<float, P>(static_cast<const float*>(t.p[e]) + at, n); break;
      case 1: v = tile_norm<bf16_t, P>(static_cast<const bf16_t*>(t.p[e]) + at, n); break;
      default: v = tile_norm<half_t, P>(static_cast<const half_t*>(t.p[e]) + at, n); break;
    }
    a = join<P>(a, v);
  }
  __shared__ double scratch[kBlock / kWave];
  a = block_join<P>(a, scratch);
  if (threadIdx.x == 0) part[blockIdx.x] = a;
}

// one workgroup: out[0] = norm, out[1] = factor
template <int P>
__global__ __launch_bounds__(1024) void norm_finish_kernel(const double* __restrict__ part, int64_t n, float max_norm,
                                                           float* __restrict__ out) {
  double a = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += 1024) a = join<P>(a, part[i]);
  __shared__ double scratch[16];
  a = block_join<P>(a, scratch);
  if (threadIdx.x == 0) {
    const double norm = P == 2 ? sqrt(a) : a;
    const double f = (double)max_norm / (norm + 1e-6);
    out[0] = (float)norm;
    out[1] = f > 1.0 ? 1.f : (float)f;  // a NaN stays
  }
}

template <typename T>
__device__ __forceinline__ void tile_scale(T* __restrict__ p, int n, float f) {
  constexpr int V = 16 / sizeof(T), U = kTile / kBlock / V;
  float x[U][V];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = (u * kBlock + threadIdx.x) * V;
    if (i < n) load_vec(p + i, x[u], n - i);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = (u * kBlock + threadIdx.x) * V;
    if (i < n) {
#pragma unroll
      for (int k = 0; k < V; ++k) x[u][k] *= f;
      store_vec(p + i, x[u], n - i);
    }
  }
}

__global__ __launch_bounds__(kBlock) void scale_kernel(List t, const float* __restrict__ factor) {
  const float f = *factor;
  if (f == 1.f) return;
  for (int tile = blockIdx.x; tile < t.start[t.n]; tile += gridDim.x) {
    const int e = find_entry(t, tile);
    const int64_t at = (int64_t)(tile - t.start[e]) * kTile;
    const int n = (int)min((int64_t)(t.len[e] & 0x3fffffffu) - at, (int64_t)kTile);
    switch (t.len[e] >> 30) {
      case 0: tile_scale(static_cast<float*>(t.p[e]) + at, n, f); break;
      case 1: tile_scale(static_cast<bf16_t*>(t.p[e]) + at, n, f); break;
      default: tile_scale(static_cast<half_t*>(t.p[e]) + at, n, f); break;
    }
  }
}

// Calls f(table) for runs of up to kListMax entries.
template <typename F>
void each_table(const GradTensor* g, int64_t n, F&& f) {
  List t;
  t.n = 0;
  int64_t tiles = 0;
  auto send = [&] {
    if (t.n == 0) return;
    t.start[t.n] = (int32_t)tiles;
    f(t);
    t.n = 0;
    tiles = 0;
  };
  for (int64_t i = 0; i < n; ++i) {
    for (int64_t at = 0; at < g[i].len; at += kMaxLen) {
      const int64_t len = std::min(g[i].len - at, kMaxLen), add = (len + kTile - 1) / kTile;
      if (t.n == kListMax || tiles + add > INT32_MAX) send();
      t.p[t.n] = static_cast<char*>(g[i].p) + at * el_bytes(g[i].type);
      t.len[t.n] = (uint32_t)len | ((uint32_t)g[i].type << 30);
      t.start[t.n++] = (int32_t)tiles;
      tiles += add;
    }
  }
  send();
}

unsigned blocks_of(const List& t) { return (unsigned)std::min(t.start[t.n], kMaxBlocks); }

}  // namespace

int64_t gradnorm_parts(const GradTensor* g, int64_t n) {
  int64_t parts = 0;
  each_table(g, n, [&](const List& t) { parts += blocks_of(t); });
  return parts;
}

void gradnorm_partial(const GradTensor* g, int64_t n, NormKind kind, double* part, hipStream_t stream) {
  each_table(g, n, [&](const List& t) {
    const unsigned blocks = blocks_of(t);
    switch (kind) {
      case NormKind::kMax: norm_part_kernel<0><<<blocks, kBlock, 0, stream>>>(t, part); break;
      case NormKind::kL1: norm_part_kernel<1><<<blocks, kBlock, 0, stream>>>(t, part); break;
      case NormKind::kL2: norm_part_kernel<2><<<blocks, kBlock, 0, stream>>>(t, part); break;
    }
    part += blocks;
  });
}

void gradnorm_finish(const double* part, int64_t parts, NormKind kind, float max_norm, float* out, hipStream_t stream) {
  switch (kind) {
    case NormKind::kMax: norm_finish_kernel<0><<<1, 1024, 0, stream>>>(part, parts, max_norm, out); break;
    case NormKind::kL1: norm_finish_kernel<1><<<1, 1024, 0, stream>>>(part, parts, max_norm, out); break;
    case NormKind::kL2: norm_finish_kernel<2><<<1, 1024, 0, stream>>>(part, parts, max_norm, out); break;
  }
}

void grad_scale(const GradTensor* g, int64_t n, const float* factor, hipStream_t stream) {
  each_table(g, n, [&](const List& t) { scale_kernel<<<blocks_of(t), kBlock, 0, stream>>>(t, factor); });
}

}  // namespace grace
