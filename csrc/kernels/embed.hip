// Embedding lookup with scaling, and its gradient by sorted tokens.
//
//   forward   out[t, :] = round(scale * w[id_t, :])
//   backward  dw[v, :]  = round(scale * sum_{t : id_t = v, v != pad} dy[t, :])
//
// The backward sorts the tokens by row (a stable LSD radix sort of (row, token) pairs, 8 bits a
// pass) and sums runs of equal rows in that order, so the result does not depend on the launch: no
// floating-point atomics.  The sorted tokens are cut into chunks of kChunk; a wave sums one chunk
// over a slab of columns in fp32 and writes every run that lies inside it.  Runs that cross a chunk
// border (a padding or mask token can fill an eighth of the batch) leave one partial row per chunk,
// and a join launch adds those in chunk order.  Tokens outside [0, vocab) and the padding row sort
// behind all rows (key = vocab) and are left out; the lookup gives NaN rows for the former, so that
// a bad token is loud without a host synchronisation.
#include <algorithm>
#include <type_traits>

#include "grace_common.h"
#include "grace_lm.h"

namespace grace {
namespace {

constexpr int kBlock = 256;
constexpr int kWaves = kBlock / kWave;
constexpr int kVec = 4;     // columns per lane
constexpr int kSlab = kWave * kVec;  // columns per wave
constexpr int kChunk = 32;  // sorted tokens per chunk (at most 64: one per lane)

__device__ __forceinline__ int64_t id_at(const EmbedIds& a, int64_t t) {
  return a.is64 ? static_cast<const int64_t*>(a.ids)[t] : (int64_t) static_cast<const int32_t*>(a.ids)[t];
}

// ---------------------------------------------------------------- forward
// One wave per token: kVec consecutive columns per lane and step.
template <typename TW, typename TO>
__global__ __launch_bounds__(kBlock) void embed_fwd_kernel(EmbedIds ids, const TW* __restrict__ w, int64_t w_stride,
                                                           int64_t d, float scale, TO* __restrict__ out) {
  const int64_t waves = (int64_t)gridDim.x * kWaves;
  for (int64_t t = (int64_t)blockIdx.x * kWaves + wave_id(); t < ids.n; t += waves) {
    const int64_t id = id_at(ids, t);
    const bool ok = id >= 0 && id < ids.vocab;
    const TW* row = w + (ok ? id : 0) * w_stride;
    for (int64_t c = (int64_t)lane_id() * kVec; c < d; c += kWave * kVec) {
      const int left = (int)min(d - c, (int64_t)kVec);
      float x[kVec];
      if (ok) {
        load_vec(row + c, x, left);
#pragma unroll
        for (int i = 0; i < kVec; ++i) x[i] *= scale;
      } else {
#pragma unroll
        for (int i = 0; i < kVec; ++i) x[i] = __uint_as_float(0x7fc00000u);
      }
      store_vec(out + t * d + c, x, left);
    }
  }
}

// ---------------------------------------------------------------- sort
constexpr int kRadix = 256;
constexpr int kPer = 8;            // pairs per thread
constexpr int kSmallWaves = 16;    // one workgroup sorts up to kSmall pairs in LDS
constexpr int kSmall = kSmallWaves * kWave * kPer;
constexpr int kTileWaves = 4;
constexpr int kTile = kTileWaves * kWave * kPer;

__device__ __forceinline__ uint32_t key_at(const EmbedIds& a, int64_t t) {
  const int64_t id = id_at(a, t);
  return (id >= 0 && id < a.vocab && id != a.pad) ? (uint32_t)id : (uint32_t)a.vocab;
}

// Stable rank of each pair among its wave's pairs of the same digit, over kPer rounds of 64; hist
// (this wave's 256 counters, zero on entry) holds the wave's digit counts afterwards.
template <int NB>
__device__ __forceinline__ void wave_rank(const uint32_t (&digit)[kPer], uint32_t (&rank)[kPer], uint32_t* hist) {
  const uint64_t below = (1ull << lane_id()) - 1;
#pragma unroll
  for (int r = 0; r < kPer; ++r) {
    uint64_t same = ~0ull;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const uint64_t one = __ballot((digit[r] >> b) & 1);
      same &= ((digit[r] >> b) & 1) ? one : ~one;
    }
    const int lead = __ffsll((unsigned long long)same) - 1;
    uint32_t old = 0;
    if (lane_id() == lead) old = atomicAdd(&hist[digit[r]], (uint32_t)__popcll(same));
    rank[r] = __shfl(old, lead, kWave) + (uint32_t)__popcll(same & below);
  }
}

// Exclusive prefix of v over the first 256 threads; scratch holds 4 words.  All threads call it.
__device__ __forceinline__ uint32_t scan256(uint32_t v, uint32_t* scratch) {
  uint32_t s = v;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const uint32_t u = __shfl_up(s, o, kWave);
    if (lane_id() >= o) s += u;
  }
  const int w = wave_id();
  __syncthreads();
  if (w < 4 && lane_id() == kWave - 1) scratch[w] = s;
  __syncthreads();
  uint32_t base = 0;
  for (int i = 0; i < w && i < 4; ++i) base += scratch[i];
  return base + s - v;
}

// n <= kSmall: every pass in one workgroup's LDS.
__global__ __launch_bounds__(kSmallWaves* kWave) void sort_small_kernel(EmbedIds ids, int bits, int passes,
                                                                       uint32_t* __restrict__ skey,
                                                                       uint32_t* __restrict__ sval) {
  __shared__ uint2 pair[kSmall];
  __shared__ uint32_t hist[kSmallWaves][kRadix];
  __shared__ uint32_t scratch[4];
  const int w = wave_id(), tid = threadIdx.x, n = (int)ids.n;
  uint32_t key[kPer], val[kPer], digit[kPer], rank[kPer];
  const int first = w * kWave * kPer + lane_id();
#pragma unroll
  for (int r = 0; r < kPer; ++r) {
    const int t = first + r * kWave;
    key[r] = t < n ? key_at(ids, t) : (1u << bits) - 1;  // places behind n stay behind
    val[r] = t;
  }
  for (int p = 0; p < passes; ++p) {
    for (int i = tid; i < kSmallWaves * kRadix; i += kSmallWaves * kWave) (&hist[0][0])[i] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kPer; ++r) digit[r] = (key[r] >> (8 * p)) & (kRadix - 1);
    wave_rank<8>(digit, rank, hist[w]);
    __syncthreads();
    uint32_t total = 0;
    if (tid < kRadix) {
      for (int i = 0; i < kSmallWaves; ++i) {
        const uint32_t c = hist[i][tid];
        hist[i][tid] = total;
        total += c;
      }
    }
    const uint32_t base = scan256(total, scratch);
    if (tid < kRadix)
      for (int i = 0; i < kSmallWaves; ++i) hist[i][tid] += base;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kPer; ++r) pair[hist[w][digit[r]] + rank[r]] = make_uint2(key[r], val[r]);
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kPer; ++r) {
      const uint2 q = pair[first + r * kWave];
      key[r] = q.x;
      val[r] = q.y;
    }
    __syncthreads();
  }
#pragma unroll
  for (int r = 0; r < kPer; ++r) {
    const int t = first + r * kWave;
    if (t < n) {
      skey[t] = key[r];
      sval[t] = val[r];
    }
  }
}

// Digit counts of one tile; in = nullptr: the tokens themselves (first pass).
__global__ __launch_bounds__(kTileWaves* kWave) void sort_count_kernel(EmbedIds ids, const uint32_t* __restrict__ in,
                                                                       int shift, uint32_t* __restrict__ count) {
  __shared__ uint32_t hist[kRadix];
  hist[threadIdx.x] = 0;
  __syncthreads();
  const int64_t t0 = (int64_t)blockIdx.x * kTile;
#pragma unroll
  for (int r = 0; r < kPer; ++r) {
    const int64_t t = t0 + r * kBlock + threadIdx.x;
    if (t < ids.n) atomicAdd(&hist[((in ? in[t] : key_at(ids, t)) >> shift) & (kRadix - 1)], 1u);
  }
  __syncthreads();
  count[(int64_t)blockIdx.x * kRadix + threadIdx.x] = hist[threadIdx.x];
}

// Moves one tile's pairs to their places: each workgroup adds up the counts itself.
__global__ __launch_bounds__(kTileWaves* kWave) void sort_move_kernel(EmbedIds ids, const uint32_t* __restrict__ in_key,
                                                                      const uint32_t* __restrict__ in_val, int shift,
                                                                      const uint32_t* __restrict__ count,
                                                                      uint32_t* __restrict__ out_key,
                                                                      uint32_t* __restrict__ out_val) {
  __shared__ uint32_t hist[kTileWaves][kRadix];
  __shared__ uint32_t scratch[4];
  const int w = wave_id(), tid = threadIdx.x;
  const int64_t t0 = (int64_t)blockIdx.x * kTile + w * kWave * kPer + lane_id();
  for (int i = 0; i < kTileWaves; ++i) hist[i][tid] = 0;
  uint32_t key[kPer], val[kPer], digit[kPer], rank[kPer];
#pragma unroll
  for (int r = 0; r < kPer; ++r) {
    const int64_t t = t0 + r * kWave;
    const bool ok = t < ids.n;
    key[r] = ok ? (in_key ? in_key[t] : key_at(ids, t)) : ~0u;  // places behind n rank behind the last digit's pairs
    val[r] = ok ? (in_val ? in_val[t] : (uint32_t)t) : 0u;
    digit[r] = (key[r] >> shift) & (kRadix - 1);
  }
  __syncthreads();
  wave_rank<8>(digit, rank, hist[w]);
  uint32_t before = 0, total = 0;
  for (unsigned i = 0; i < gridDim.x; ++i) {
    const uint32_t c = count[(int64_t)i * kRadix + tid];
    if (i < blockIdx.x) before += c;
    total += c;
  }
  uint32_t base = scan256(total, scratch) + before;  // its barriers order the ranks before the prefix below
  for (int i = 0; i < kTileWaves; ++i) {
    const uint32_t c = hist[i][tid];
    hist[i][tid] = base;
    base += c;
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kPer; ++r) {
    if (t0 + r * kWave < ids.n) {
      const uint32_t at = hist[w][digit[r]] + rank[r];
      out_key[at] = key[r];
      out_val[at] = val[r];
    }
  }
}

// ---------------------------------------------------------------- sums over runs
struct Runs {
  const uint32_t* key;  // sorted rows, `vocab` for left-out tokens
  const uint32_t* val;  // the tokens in that order
  int64_t n;
  uint32_t vocab;
  float* head;  // [chunks, d]: the part of a run that began in an earlier chunk
  float* tail;  // [chunks, d]: the part of a run that begins here and goes on
};

template <typename TD, typename TG>
__global__ __launch_bounds__(kBlock) void run_sum_kernel(Runs a, const TD* __restrict__ dy, int64_t d, float scale,
                                                         TG* __restrict__ dw) {
  const int64_t c = (int64_t)blockIdx.x * kWaves + wave_id();
  const int64_t begin = c * kChunk;
  if (begin >= a.n) return;
  const int cnt = (int)min((int64_t)kChunk, a.n - begin);
  const int64_t col = (int64_t)blockIdx.y * kSlab + lane_id() * kVec;
  const int left = (int)max(min(d - col, (int64_t)kVec), (int64_t)0);
  const bool in = left > 0;
  const uint32_t before = begin > 0 ? a.key[begin - 1] : a.vocab;
  const uint32_t after = begin + cnt < a.n ? a.key[begin + cnt] : a.vocab;
  uint32_t lk = a.vocab, lv = 0;
  if (lane_id() < cnt) {
    lk = a.key[begin + lane_id()];
    lv = a.val[begin + lane_id()];
  }
  constexpr int U = 8;  // rows in flight
  float acc[kVec] = {};
  uint32_t run = __builtin_amdgcn_readfirstlane(lk);
  bool first = true;  // the run holds the chunk's first place
  auto flush = [&](bool last) {
    if (run < a.vocab && in) {
      if (first && run == before) {
        store_vec(a.head + c * d + col, acc, left);
      } else if (last && run == after) {
        store_vec(a.tail + c * d + col, acc, left);
      } else {
        float o[kVec];
#pragma unroll
        for (int i = 0; i < kVec; ++i) o[i] = acc[i] * scale;
        store_vec(dw + (int64_t)run * d + col, o, left);
      }
    }
  };
  for (int i0 = 0; i0 < cnt; i0 += U) {
    float x[U][kVec];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t k = __builtin_amdgcn_readlane(lk, min(i0 + u, kChunk - 1));
      const uint32_t t = __builtin_amdgcn_readlane(lv, min(i0 + u, kChunk - 1));
#pragma unroll
      for (int i = 0; i < kVec; ++i) x[u][i] = 0.f;
      if (i0 + u < cnt && k < a.vocab && in) load_vec(dy + (int64_t)t * d + col, x[u], left);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i0 + u < cnt) {
        const uint32_t k = __builtin_amdgcn_readlane(lk, i0 + u);
        if (k != run) {
          flush(false);
          run = k;
          first = false;
#pragma unroll
          for (int i = 0; i < kVec; ++i) acc[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < kVec; ++i) acc[i] += x[u][i];
      }
    }
  }
  flush(true);
}

// Adds up the partial rows of the run that begins in chunk blockIdx.x and crosses its end: the
// workgroup's waves take every kWaves-th partial row and meet in LDS in a fixed order.
template <typename TG>
__global__ __launch_bounds__(kBlock) void run_join_kernel(Runs a, int64_t d, float scale, TG* __restrict__ dw) {
  const int64_t c = blockIdx.x, end = (c + 1) * kChunk;
  if (end >= a.n) return;
  const uint32_t run = a.key[end];
  if (run >= a.vocab || a.key[end - 1] != run) return;
  if (c > 0 && a.key[c * kChunk - 1] == run) return;  // it began earlier
  int64_t lo = end, hi = a.n;  // first place behind the run
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (a.key[mid] > run) hi = mid; else lo = mid + 1;
  }
  const int64_t last = (lo - 1) / kChunk;  // the chunk where it ends
  const int64_t col = (int64_t)blockIdx.y * kSlab + lane_id() * kVec;
  const int left = (int)max(min(d - col, (int64_t)kVec), (int64_t)0);
  const bool in = left > 0;
  float acc[kVec] = {};
  if (in) {
    for (int64_t j = c + wave_id(); j <= last; j += kWaves) {
      float x[kVec];
      load_vec((j == c ? a.tail : a.head) + j * d + col, x, left);
#pragma unroll
      for (int i = 0; i < kVec; ++i) acc[i] += x[i];
    }
  }
  __shared__ float part[kWaves][kWave * kVec];
#pragma unroll
  for (int i = 0; i < kVec; ++i) part[wave_id()][lane_id() * kVec + i] = acc[i];
  __syncthreads();
  if (wave_id() == 0 && in) {
    float o[kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      float s = part[0][lane_id() * kVec + i];
      for (int k = 1; k < kWaves; ++k) s += part[k][lane_id() * kVec + i];
      o[i] = s * scale;
    }
    store_vec(dw + (int64_t)run * d + col, o, left);
  }
}

template <typename F>
void by_type(ElType t, F&& f) {
  switch (t) {
    case ElType::kF32: f((float*)nullptr); break;
    case ElType::kBF16: f((bf16_t*)nullptr); break;
    case ElType::kF16: f((half_t*)nullptr); break;
  }
}
int64_t align256(int64_t b) { return (b + 255) & ~(int64_t)255; }

}  // namespace

void embed_forward(const EmbedIds& ids, const void* w, ElType tw, int64_t w_stride, int64_t d, float scale, void* out,
                   ElType to, hipStream_t stream) {
  if (ids.n == 0 || d == 0) return;
  const unsigned grid = (unsigned)std::min<int64_t>((ids.n + kWaves - 1) / kWaves, 1 << 20);
  by_type(tw, [&](auto* tag_w) {
    using TW = std::remove_pointer_t<decltype(tag_w)>;
    by_type(to, [&](auto* tag_o) {
      using TO = std::remove_pointer_t<decltype(tag_o)>;
      embed_fwd_kernel<TW, TO><<<grid, kBlock, 0, stream>>>(ids, (const TW*)w, w_stride, d, scale, (TO*)out);
    });
  });
}

int64_t embed_backward_ws(int64_t n, int64_t vocab, int64_t d) {
  const int64_t chunks = (n + kChunk - 1) / kChunk, tiles = (n + kTile - 1) / kTile;
  return 4 * align256(4 * n) + 2 * align256(4 * chunks * d) + (n > kSmall ? align256(4 * tiles * kRadix) : 0);
}

void embed_backward(const EmbedIds& ids, const void* dy, ElType tdy, int64_t d, float scale, void* dw, ElType tdw,
                    void* ws, hipStream_t stream) {
  if (ids.vocab == 0 || d == 0 || ids.n == 0) return;
  const int64_t n = ids.n, chunks = (n + kChunk - 1) / kChunk;
  char* at = static_cast<char*>(ws);
  auto take = [&](int64_t bytes) {
    char* p = at;
    at += align256(bytes);
    return p;
  };
  uint32_t* key[2] = {(uint32_t*)take(4 * n), (uint32_t*)take(4 * n)};
  uint32_t* val[2] = {(uint32_t*)take(4 * n), (uint32_t*)take(4 * n)};
  float* head = (float*)take(4 * chunks * d);
  float* tail = (float*)take(4 * chunks * d);
  int bits = 1;
  while ((ids.vocab >> bits) != 0) ++bits;  // keys 0 .. vocab
  const int passes = (bits + 7) / 8;
  int now = 0;
  if (n <= kSmall) {
    sort_small_kernel<<<1, kSmallWaves * kWave, 0, stream>>>(ids, bits, passes, key[0], val[0]);
  } else {
    const unsigned tiles = (unsigned)((n + kTile - 1) / kTile);
    uint32_t* count = (uint32_t*)take((int64_t)4 * tiles * kRadix);
    const uint32_t *ik = nullptr, *iv = nullptr;
    for (int p = 0; p < passes; ++p) {
      now = p & 1;
      sort_count_kernel<<<tiles, kTileWaves * kWave, 0, stream>>>(ids, ik, 8 * p, count);
      sort_move_kernel<<<tiles, kTileWaves * kWave, 0, stream>>>(ids, ik, iv, 8 * p, count, key[now], val[now]);
      ik = key[now];
      iv = val[now];
    }
  }
  const Runs runs{key[now], val[now], n, (uint32_t)ids.vocab, head, tail};
  const unsigned slabs = (unsigned)((d + kSlab - 1) / kSlab);
  by_type(tdw, [&](auto* tag_g) {
    using TG = std::remove_pointer_t<decltype(tag_g)>;
    by_type(tdy, [&](auto* tag_d) {
      using TD = std::remove_pointer_t<decltype(tag_d)>;
      run_sum_kernel<TD, TG><<<dim3((unsigned)((chunks + kWaves - 1) / kWaves), slabs), kBlock, 0, stream>>>(
          runs, (const TD*)dy, d, scale, (TG*)dw);
    });
    run_join_kernel<TG><<<dim3((unsigned)chunks, slabs), kBlock, 0, stream>>>(runs, d, scale, (TG*)dw);
  });
}

}  // namespace grace
