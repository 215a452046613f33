// Global gradient norm over many tensors, and clipping by it.
//
//   norm   = (sum over all tensors and elements of |g|^p)^(1/p)  (p = 1, 2) or max |g|
//   factor = min(1, max_norm / (norm + 1e-6))          g = round(g * factor)
//
// The tensors are cut into tiles of kTileBytes; a launch covers up to kListMax tensors through a
// table in its arguments, so a captured graph replays it with no host work.  A workgroup adds up its
// tiles in fp64 (squares of fp32 gradients neither overflow nor lose the small ones, and the
// conversion is free under the loads) and leaves one partial value; every workgroup of the scaling launch
// joins the partial values itself, in a fixed order: no atomics, no launch in between, and the result does
// not depend on timing.  A factor of one leaves the gradients as they are, so an ordinary step reads
// them once.
#include <algorithm>
#include <type_traits>

#include "grace_common.h"
#include "grace_lm.h"

namespace grace {
namespace {

constexpr int kBlock = 256;
constexpr int kTileBytes = 16384;
constexpr int kListMax = 240;    // 3.8 KB of kernel arguments
// Partial values per launch: eight workgroups a CU, 128 KB of loads in flight.  Half of them take 79 us for 440 MB, twice
// as many 67 us, and 9.6 us for 3.9 us to join them.
constexpr int kMaxBlocks = 2048;
constexpr int64_t kMaxLen = 1 << 29;  // elements per table entry: longer tensors take several

struct List {
  void* p[kListMax];
  uint32_t len[kListMax];        // elements, the type in the upper two bits
  int32_t start[kListMax + 1];   // first tile of each entry
  int32_t n;
};

template <typename T>
constexpr int tile_of() { return kTileBytes / (int)sizeof(T); }

// The table's first tiles, spread over the lanes of a wave, find a tile's entry by ballots: one load's latency for a
// workgroup, where a binary search in the arguments waits for eight loads in a row for every tile.
struct Finder {
  static constexpr int kParts = (kListMax + kWave - 1) / kWave;
  int start[kParts];
  __device__ __forceinline__ explicit Finder(const List& t) {
#pragma unroll
    for (int k = 0; k < kParts; ++k) {
      const int e = k * kWave + lane_id();
      start[k] = e < t.n ? t.start[e] : INT32_MAX;
    }
  }
  // the last entry that starts at the tile or before it
  __device__ __forceinline__ int operator()(int tile) const {
    int e = -1;
#pragma unroll
    for (int k = 0; k < kParts; ++k) e += __popcll(__ballot(start[k] <= tile));
    return e;
  }
};

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

template <typename T, int P, bool ONCE>
__device__ __forceinline__ double tile_norm(const T* __restrict__ p, int n) {
  double a = 0.0;
  constexpr int V = 16 / sizeof(T), U = tile_of<T>() / kBlock / V;
  Bits<T, V> x[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = (u * kBlock + threadIdx.x) * V;
#pragma unroll
    for (int k = 0; k < Bits<T, V>::W; ++k) x[u].w[k] = 0;
    if (i < n) load_bits<ONCE>(p + i, x[u], n - i);
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int k = 0; k < V; ++k) a = join<P>(a, term<P>(bits_at(x[u], k)));
  return a;
}

// Calls f(typed pointer, elements) for a tile.
template <typename F>
__device__ __forceinline__ void on_tile(const List& t, const Finder& find, int tile, F&& f) {
  const int e = find(tile);
  const int64_t k = tile - t.start[e], len = t.len[e] & 0x3fffffffu;
  auto go = [&](auto* p) {
    constexpr int64_t T = tile_of<std::remove_pointer_t<decltype(p)>>();
    f(p + k * T, (int)min(len - k * T, T));
  };
  switch (t.len[e] >> 30) {
    case 0: go(static_cast<float*>(t.p[e])); break;
    case 1: go(static_cast<bf16_t*>(t.p[e])); break;
    default: go(static_cast<half_t*>(t.p[e])); break;
  }
}

// Bound by memory.  ONCE: nontemporal loads.  Gradients of 440 MB take 67 us with them (6.6 TB/s) and 72 us without,
// 219 MB 37 and 40 us; 79 MB, which the 256 MB memory-side cache can still hold from the pass that wrote them, 15.8 and
// 14.9 us.
constexpr int64_t kOnceBytes = 128 << 20;
template <int P, bool ONCE>
__global__ __launch_bounds__(kBlock) void norm_part_kernel(List t, double* __restrict__ part) {
  double a = 0.0;
  const Finder find(t);
  // from the end: whoever reads the gradients next begins at their start, which the memory-side cache still holds
  for (int tile = t.start[t.n] - 1 - (int)blockIdx.x; tile >= 0; tile -= gridDim.x)
    on_tile(t, find, tile, [&](auto* p, int n) {
      a = join<P>(a, tile_norm<std::remove_pointer_t<decltype(p)>, P, ONCE>(p, n));
    });
  __shared__ double scratch[kBlock / kWave];
  a = block_join<P>(a, scratch);
  if (threadIdx.x == 0) part[blockIdx.x] = a;
}

// Norm and factor from the partial values, in every thread of a workgroup of BLOCK threads.
template <int P, int BLOCK>
__device__ __forceinline__ float2 finish(const double* __restrict__ part, int64_t n, float max_norm) {
  __shared__ double scratch[BLOCK / kWave];
  double a = 0.0;
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < n; i += BLOCK) a = join<P>(a, part[i]);
  a = block_join<P>(a, scratch);
  const double norm = P == 2 ? sqrt(a) : a;
  const double f = (double)max_norm / (norm + 1e-6);
  return make_float2((float)norm, f > 1.0 ? 1.f : (float)f);  // a NaN stays
}

// one workgroup: out[0] = norm, out[1] = factor
template <int P>
__global__ __launch_bounds__(1024) void norm_finish_kernel(const double* __restrict__ part, int64_t n, float max_norm,
                                                           float* __restrict__ out) {
  const float2 r = finish<P, 1024>(part, n, max_norm);
  if (threadIdx.x == 0) *reinterpret_cast<float2*>(out) = r;
}

template <typename T>
__device__ __forceinline__ void tile_scale(T* __restrict__ p, int n, float f) {
  constexpr int V = 16 / sizeof(T), U = tile_of<T>() / kBlock / V;
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

__device__ __forceinline__ void scale_tiles(const List& t, float f) {
  if (f == 1.f) return;
  const Finder find(t);
  for (int tile = blockIdx.x; tile < t.start[t.n]; tile += gridDim.x)
    on_tile(t, find, tile, [&](auto* p, int n) { tile_scale(p, n, f); });
}

__global__ __launch_bounds__(kBlock) void scale_kernel(List t, const float* __restrict__ factor) {
  scale_tiles(t, *factor);
}

// With the factor from the partial values; out = nullptr in all launches but the first.  Norm and scaling of 110 million
// gradients: fp32 209 us (6.3 TB/s of two reads and a write), bf16 112 us (5.9); a factor of one 70 and 38 us.
template <int P>
__global__ __launch_bounds__(kBlock) void clip_kernel(List t, const double* __restrict__ part, int64_t n,
                                                      float max_norm, float* __restrict__ out) {
  const float2 r = finish<P, kBlock>(part, n, max_norm);
  if (out != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *reinterpret_cast<float2*>(out) = r;
  scale_tiles(t, r.y);
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
      const int64_t len = std::min(g[i].len - at, kMaxLen), tile = kTileBytes / el_bytes(g[i].type),
                    add = (len + tile - 1) / tile;
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
  int64_t bytes = 0;
  for (int64_t i = 0; i < n; ++i) bytes += g[i].len * el_bytes(g[i].type);
  auto launch = [&](const List& t, unsigned blocks, auto once) {
    constexpr bool ONCE = decltype(once)::value;
    switch (kind) {
      case NormKind::kMax: norm_part_kernel<0, ONCE><<<blocks, kBlock, 0, stream>>>(t, part); break;
      case NormKind::kL1: norm_part_kernel<1, ONCE><<<blocks, kBlock, 0, stream>>>(t, part); break;
      case NormKind::kL2: norm_part_kernel<2, ONCE><<<blocks, kBlock, 0, stream>>>(t, part); break;
    }
  };
  each_table(g, n, [&](const List& t) {
    const unsigned blocks = blocks_of(t);
    if (bytes > kOnceBytes) launch(t, blocks, std::true_type{});
    else launch(t, blocks, std::false_type{});
    part += blocks;
  });
}

void grad_clip(const GradTensor* g, int64_t n, const double* part, int64_t parts, NormKind kind, float max_norm,
               float* out, hipStream_t stream) {
  each_table(g, n, [&](const List& t) {
    const unsigned blocks = blocks_of(t);
    switch (kind) {
      case NormKind::kMax: clip_kernel<0><<<blocks, kBlock, 0, stream>>>(t, part, parts, max_norm, out); break;
      case NormKind::kL1: clip_kernel<1><<<blocks, kBlock, 0, stream>>>(t, part, parts, max_norm, out); break;
      case NormKind::kL2: clip_kernel<2><<<blocks, kBlock, 0, stream>>>(t, part, parts, max_norm, out); break;
    }
    out = nullptr;
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
