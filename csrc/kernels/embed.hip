// Embedding lookup with scaling, and its gradient by sorted tokens.
//
//   forward   out[t, :] = round(scale * w[id_t, :])
//   backward  dw[v, :]  = round(scale * sum_{t : id_t = v, v != pad} dy[t, :])
//
// The backward sums the rows of equal tokens in token order, so the result does not depend on the launch: no
// floating-point atomics.  Two ways there, by the number of tokens n:
//   n <= kFew    one launch: a workgroup per token looks through all tokens, and the first of its kind sums them
//                all; workgroups behind them clear the rows that no token names (the n ids stay in L2)
//   n >  kFew    the tokens are sorted by row (a stable LSD radix sort of (row, token) pairs, 8 bits a
//                pass; up to kSmall pairs in the LDS of one workgroup) and cut into chunks; a wave sums
//                one chunk over a slab of columns in fp32 and writes every run of equal rows inside
//                it.  Runs that cross a chunk's border (a padding or mask token can fill an eighth of a batch)
//                leave one partial row per chunk, which a join launch adds in chunk order.
// There dw is filled with zeros by the workgroups that a sort launch leaves idle, so the fill hides the sort.
// Tokens outside [0, vocab) and the padding row sort behind all rows (key = vocab) and are left out; the
// lookup gives NaN rows for the former, so that a bad token is loud without a host synchronisation.
#include <algorithm>
#include <type_traits>

#include "grace_common.h"
#include "grace_lm.h"

namespace grace {
namespace {

constexpr int kBlock = 256;
constexpr int kWaves = kBlock / kWave;

__device__ __forceinline__ int64_t id_at(const EmbedIds& a, int64_t t) {
  return a.is64 ? static_cast<const int64_t*>(a.ids)[t] : (int64_t) static_cast<const int32_t*>(a.ids)[t];
}

// columns per lane: 16 bytes of the narrower type
template <typename A, typename B>
constexpr int vec_of() { return sizeof(A) == 2 || sizeof(B) == 2 ? 8 : 4; }

// ---------------------------------------------------------------- forward
// 2^lanes_log lanes per token (a wave for wide rows, several tokens a wave for narrow ones), V columns per
// lane and step; the loads of kSteps steps are under way before the first store.  Bound by memory: 65536 fp32 rows of
// 1024 to bf16 take 47 us for at most 339 MB (frequent rows come from the caches); 8 bf16 rows of 768 2.2 us, a launch.
template <typename TW, typename TO>
__global__ __launch_bounds__(kBlock) void embed_fwd_kernel(EmbedIds ids, const TW* __restrict__ w, int64_t w_stride,
                                                           int64_t d, float scale, TO* __restrict__ out,
                                                           int lanes_log) {
  constexpr int V = vec_of<TW, TO>(), kSteps = 2;
  const int lanes = 1 << lanes_log, lane = threadIdx.x & (lanes - 1);
  const int64_t t = (((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * kBlock + threadIdx.x) >> lanes_log;
  if (t >= ids.n) return;
  const int64_t id = id_at(ids, t);
  const bool ok = id >= 0 && id < ids.vocab;
  const TW* row = w + (ok ? id : 0) * w_stride;
  for (int64_t c0 = (int64_t)lane * V; c0 < d; c0 += (int64_t)lanes * V * kSteps) {
    float x[kSteps][V];
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      const int64_t c = c0 + (int64_t)k * lanes * V;
#pragma unroll
      for (int i = 0; i < V; ++i) x[k][i] = __uint_as_float(0x7fc00000u);
      if (ok && c < d) load_vec(row + c, x[k], (int)min(d - c, (int64_t)V));
    }
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      const int64_t c = c0 + (int64_t)k * lanes * V;
      if (c >= d) break;
#pragma unroll
      for (int i = 0; i < V; ++i) x[k][i] *= scale;
      store_vec(out + t * d + c, x[k], (int)min(d - c, (int64_t)V));
    }
  }
}

// ---------------------------------------------------------------- few tokens
constexpr int kFew = 1024;

// Clears those of the rows [r0, r1) that no token names: at most kClearRows of them, 2^lanes_log lanes a row.
constexpr int kClearRows = 1024;
template <typename TG>
__device__ __forceinline__ void clear_rows(const EmbedIds& ids, int64_t r0, int64_t r1, int64_t d, int lanes_log,
                                           TG* __restrict__ dw) {
  constexpr int V = 16 / sizeof(TG);
  __shared__ uint32_t named[kClearRows / 32];
  for (int i = threadIdx.x; i < kClearRows / 32; i += kBlock) named[i] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < (int)ids.n; i += kBlock) {
    const int64_t id = id_at(ids, i);
    if (id >= r0 && id < r1 && id != ids.pad) atomicOr(&named[(id - r0) / 32], 1u << ((id - r0) & 31));
  }
  __syncthreads();
  const int lane = threadIdx.x & ((1 << lanes_log) - 1);
  const float zero[V] = {};
  for (int64_t r = r0 + (threadIdx.x >> lanes_log); r < r1; r += kBlock >> lanes_log) {
    if (named[(r - r0) / 32] >> ((r - r0) & 31) & 1) continue;
    for (int64_t c = (int64_t)lane * V; c < d; c += (int64_t)V << lanes_log)
      store_vec(dw + r * d + c, zero, (int)min(d - c, (int64_t)V));
  }
}

// Workgroup (token t, slab of columns), and behind those the ones that clear.  Each wave looks through a quarter of
// the tokens and notes those of t's row; if t is the first of them the waves sum their notes and meet in LDS
// in token order.  700 tokens of 650 fp32 columns into 10000 rows: 12.6 us for 28 MB, the latency of a search, a sum
// and a meeting one after the other, and of the clearing behind them, which starts when the token workgroups have been
// dispatched (sorting takes three launches).
template <typename TD, typename TG>
__global__ __launch_bounds__(kBlock) void embed_few_kernel(EmbedIds ids, const TD* __restrict__ dy, int64_t d,
                                                           float scale, TG* __restrict__ dw, int slabs, int rows_each,
                                                           int lanes_log) {
  constexpr int V = vec_of<TD, float>(), kSlab = kWave * V, U = 8;
  const int n = (int)ids.n, w = wave_id();
  const int64_t clear = (int64_t)blockIdx.x - (int64_t)n * slabs;
  if (clear >= 0)
    return clear_rows(ids, clear * rows_each, min((clear + 1) * rows_each, ids.vocab), d, lanes_log, dw);
  __shared__ uint16_t note[kWaves][kFew / kWaves];
  __shared__ float part[kWaves][kSlab];
  const int t = blockIdx.x % n;
  const int64_t id = id_at(ids, t);
  if (id < 0 || id >= ids.vocab || id == ids.pad) return;
  const int quarter = (n + kWaves - 1) / kWaves, begin = w * quarter, end = min(begin + quarter, n);
  int found = 0, earlier = 0;
  for (int i0 = begin; i0 < end; i0 += kWave) {
    const int i = i0 + lane_id();
    const bool same = i < end && id_at(ids, i) == id;
    const uint64_t all = __ballot(same);
    if (same) note[w][found + __popcll(all & ((1ull << lane_id()) - 1))] = (uint16_t)i;
    found += __popcll(all);
    earlier |= same && i < t;
  }
  if (__syncthreads_or(earlier)) return;
  const int64_t col = (int64_t)(blockIdx.x / n) * kSlab + lane_id() * V;
  const int left = (int)max(min(d - col, (int64_t)V), (int64_t)0);
  float acc[V] = {};
  for (int j0 = 0; j0 < found; j0 += U) {
    float x[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int from = note[w][min(j0 + u, found - 1)];
#pragma unroll
      for (int i = 0; i < V; ++i) x[u][i] = 0.f;
      if (j0 + u < found && left > 0) load_vec(dy + (int64_t)from * d + col, x[u], left);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] += x[u][i];
  }
#pragma unroll
  for (int i = 0; i < V; ++i) part[w][lane_id() * V + i] = acc[i];
  __syncthreads();
  if (w == 0 && left > 0) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
      for (int k = 1; k < kWaves; ++k) acc[i] += part[k][lane_id() * V + i];
      acc[i] *= scale;
    }
    store_vec(dw + id * d + col, acc, left);
  }
}

// ---------------------------------------------------------------- sort
constexpr int kRadix = 256;
constexpr int kSortWaves = 16;
constexpr int kSortBlock = kSortWaves * kWave;
constexpr int kSmall = kSortBlock * 8;   // pairs that one workgroup sorts in LDS
constexpr int kManyTiles = 64;           // tiles of 2048 pairs before they grow to 8192
// Up to so many tiles each adds up all tiles' counts itself, work that grows with their square: 4 million tokens (512
// tiles, 8 columns) 1042 us and 1045 with a scan of the counts in a launch of its own, 17 million (2048) 1838 and 1451.
constexpr int kScanTiles = 512;

// Memory that a launch clears with the workgroups behind its own: bytes [begin, end) of p (16-byte aligned).
struct Fill {
  void* p;
  int64_t begin, end;
};
constexpr int kFillBlocks = 512;

__device__ __forceinline__ void fill_zero(const Fill& f, int block, int blocks) {
  char* p = static_cast<char*>(f.p);
  const int64_t vecs = (f.end - f.begin) >> 4;
  for (int64_t i = (int64_t)block * kSortBlock + threadIdx.x; i < vecs; i += (int64_t)blocks * kSortBlock)
    reinterpret_cast<uint4*>(p + f.begin)[i] = make_uint4(0, 0, 0, 0);
  const int64_t tail = f.begin + (vecs << 4) + threadIdx.x;
  if (block == 0 && tail < f.end) p[tail] = 0;
}

__device__ __forceinline__ uint32_t key_at(const EmbedIds& a, int64_t t) {
  const int64_t id = id_at(a, t);
  return (id >= 0 && id < a.vocab && id != a.pad) ? (uint32_t)id : (uint32_t)a.vocab;
}

// Stable rank of each pair among its wave's pairs of the same digit, over PER rounds of 64; hist
// (this wave's 256 counters, zero on entry) holds the wave's digit counts afterwards.
template <int PER>
__device__ __forceinline__ void wave_rank(const uint32_t (&digit)[PER], uint32_t (&rank)[PER], uint32_t* hist) {
  constexpr int NB = 8;
  const uint64_t below = (1ull << lane_id()) - 1;
#pragma unroll
  for (int r = 0; r < PER; ++r) {
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

// Turns the waves' digit counts into places: hist[w][q] = base(q) + the counts of the waves before w.  base
// holds q's first place for q = threadIdx.x < 256.  All threads call it between barriers.
__device__ __forceinline__ void place(uint32_t (*hist)[kRadix], uint32_t base) {
  if (threadIdx.x < kRadix) {
#pragma unroll
    for (int i = 0; i < kSortWaves; ++i) {
      const uint32_t c = hist[i][threadIdx.x];
      hist[i][threadIdx.x] = base;
      base += c;
    }
  }
}

// n <= 1024 PER: workgroup 0 sorts, every pass in its LDS; the others clear dw.  4096 tokens, 15 bits: 14.6 us, in which
// 94 MB are cleared at 6.4 TB/s (a fill alone reaches 6.8).
template <int PER>
__global__ __launch_bounds__(kSortBlock) void sort_small_kernel(EmbedIds ids, int bits, int passes,
                                                                uint32_t* __restrict__ skey,
                                                                uint32_t* __restrict__ sval, uint32_t* __restrict__ joins,
                                                                Fill fill) {
  if (blockIdx.x > 0) return fill_zero(fill, blockIdx.x - 1, gridDim.x - 1);
  if (threadIdx.x == 0) *joins = 0;
  __shared__ uint2 pair[kSortBlock * PER];
  __shared__ uint32_t hist[kSortWaves][kRadix];
  __shared__ uint32_t scratch[4];
  const int w = wave_id(), tid = threadIdx.x, n = (int)ids.n;
  uint32_t key[PER], val[PER], digit[PER], rank[PER];
  const int first = w * kWave * PER + lane_id();
#pragma unroll
  for (int r = 0; r < PER; ++r) {
    const int t = first + r * kWave;
    key[r] = t < n ? key_at(ids, t) : (1u << bits) - 1;  // places behind n stay behind
    val[r] = t;
  }
  for (int p = 0; p < passes; ++p) {
#pragma unroll
    for (int i = 0; i < kRadix / kWave; ++i) hist[w][lane_id() + i * kWave] = 0;  // a wave's own counters
#pragma unroll
    for (int r = 0; r < PER; ++r) digit[r] = (key[r] >> (8 * p)) & (kRadix - 1);
    wave_rank(digit, rank, hist[w]);
    __syncthreads();
    uint32_t total = 0;
    if (tid < kRadix) {
#pragma unroll
      for (int i = 0; i < kSortWaves; ++i) total += hist[i][tid];
    }
    place(hist, scan256(total, scratch));
    __syncthreads();
#pragma unroll
    for (int r = 0; r < PER; ++r) pair[hist[w][digit[r]] + rank[r]] = make_uint2(key[r], val[r]);
    __syncthreads();
#pragma unroll
    for (int r = 0; r < PER; ++r) {
      const uint2 q = pair[first + r * kWave];
      key[r] = q.x;
      val[r] = q.y;
    }
  }
#pragma unroll
  for (int r = 0; r < PER; ++r) {
    const int t = first + r * kWave;
    if (t < n) {
      skey[t] = key[r];
      sval[t] = val[r];
    }
  }
}

// Digit counts of every tile of 1024 PER tokens, count[tile][digit]; the workgroups behind the tiles clear a
// share of dw.  in = nullptr: the tokens themselves (the first pass).  65536 tokens: 8.9 us and the move 10.7 us a pass;
// both passes together clear 205 MB in 39 us, 5.2 TB/s.
template <int PER>
__global__ __launch_bounds__(kSortBlock) void sort_count_kernel(EmbedIds ids, int tiles,
                                                                const uint32_t* __restrict__ in, int shift,
                                                                uint32_t* __restrict__ count,
                                                                uint32_t* __restrict__ joins, Fill fill) {
  if ((int)blockIdx.x >= tiles) return fill_zero(fill, blockIdx.x - tiles, gridDim.x - tiles);
  if (blockIdx.x == 0 && threadIdx.x == 0) *joins = 0;
  __shared__ uint32_t hist[kRadix];
  if (threadIdx.x < kRadix) hist[threadIdx.x] = 0;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < PER; ++r) {
    const int64_t t = ((int64_t)blockIdx.x * PER + r) * kSortBlock + threadIdx.x;
    if (t < ids.n) atomicAdd(&hist[((in ? in[t] : key_at(ids, t)) >> shift) & (kRadix - 1)], 1u);
  }
  __syncthreads();
  if (threadIdx.x < kRadix) count[(int64_t)blockIdx.x * kRadix + threadIdx.x] = hist[threadIdx.x];
}

// Of many tiles the counts become places once, a workgroup for each digit: count[tile][digit] turns into the sum over the
// tiles before it, and the row behind the tiles into the digits' totals.
__global__ __launch_bounds__(kSortBlock) void sort_scan_kernel(int tiles, uint32_t* __restrict__ count) {
  __shared__ uint32_t waves[kSortWaves];
  const int w = wave_id();
  uint32_t* at = count + blockIdx.x;
  uint32_t base = 0;
  for (int t0 = 0; t0 < tiles; t0 += kSortBlock) {
    const int t = t0 + threadIdx.x;
    const uint32_t v = t < tiles ? at[(int64_t)t * kRadix] : 0u;
    uint32_t s = v;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
      const uint32_t u = __shfl_up(s, o, kWave);
      if (lane_id() >= o) s += u;
    }
    __syncthreads();  // the last round's sums have been read
    if (lane_id() == kWave - 1) waves[w] = s;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < kSortWaves; ++i) {
      if (i < w) before += waves[i];
      all += waves[i];
    }
    if (t < tiles) at[(int64_t)t * kRadix] = base + before + s - v;
    base += all;
  }
  if (threadIdx.x == 0) at[(int64_t)tiles * kRadix] = base;
}

// Moves one tile's pairs to their places; each workgroup adds up the tiles' counts itself, or finds the sums there
// (scanned).  (Counting the next pass's digits here saves a launch and loses more: a token that fills an eighth of the
// batch sends as many atomics to one address, 42 us for 65536 tokens.)
template <int PER>
__global__ __launch_bounds__(kSortBlock) void sort_move_kernel(EmbedIds ids, int tiles,
                                                               const uint32_t* __restrict__ in_key,
                                                               const uint32_t* __restrict__ in_val, int shift,
                                                               const uint32_t* __restrict__ count, bool scanned,
                                                               uint32_t* __restrict__ out_key,
                                                               uint32_t* __restrict__ out_val, Fill fill) {
  if ((int)blockIdx.x >= tiles) return fill_zero(fill, blockIdx.x - tiles, gridDim.x - tiles);
  __shared__ uint32_t hist[kSortWaves][kRadix];
  __shared__ uint32_t sums[2][kSortBlock / kRadix][kRadix];
  __shared__ uint32_t scratch[4];
  const int w = wave_id(), tid = threadIdx.x;
  const int64_t t0 = (int64_t)blockIdx.x * kSortBlock * PER + w * kWave * PER + lane_id();
  uint32_t key[PER], val[PER], digit[PER], rank[PER];
#pragma unroll
  for (int r = 0; r < PER; ++r) {
    const int64_t t = t0 + r * kWave;
    const bool ok = t < ids.n;
    key[r] = ok ? (in_key ? in_key[t] : key_at(ids, t)) : ~0u;  // places behind n rank behind the last digit's pairs
    val[r] = ok ? (in_val ? in_val[t] : (uint32_t)t) : 0u;
    digit[r] = (key[r] >> shift) & (kRadix - 1);
  }
  uint32_t before = 0, total = 0;
  const int q = tid & (kRadix - 1), group = tid / kRadix;
  if (scanned) {
    if (group == 0) {
      before = count[(int64_t)blockIdx.x * kRadix + q];
      total = count[(int64_t)tiles * kRadix + q];
    }
  } else {
#pragma unroll 4
    for (int i = group; i < tiles; i += kSortBlock / kRadix) {
      const uint32_t c = count[(int64_t)i * kRadix + q];
      if (i < (int)blockIdx.x) before += c;
      total += c;
    }
  }
  sums[0][group][q] = before;
  sums[1][group][q] = total;
#pragma unroll
  for (int i = 0; i < kRadix / kWave; ++i) hist[w][lane_id() + i * kWave] = 0;  // a wave's own counters
  wave_rank(digit, rank, hist[w]);
  __syncthreads();
  before = total = 0;
#pragma unroll
  for (int i = 0; i < kSortBlock / kRadix; ++i) {
    before += sums[0][i][q];
    total += sums[1][i][q];
  }
  place(hist, scan256(tid < kRadix ? total : 0u, scratch) + before);
  __syncthreads();
#pragma unroll
  for (int r = 0; r < PER; ++r) {
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
  int chunk;            // sorted tokens per chunk: 8, 16 or 32
  float* head;  // [chunks, d]: the part of a run that began in an earlier chunk
  float* tail;  // [chunks, d]: the part of a run that begins here and goes on
  uint32_t* joins;      // their number, and then the chunks where such runs begin, in any order
};

// Bound by memory.  ONCE: nontemporal loads of dy.  134 MB of it take 39 us with them and 50 us without; what the
// caches can still hold from the pass that wrote it is read through them.
constexpr int64_t kOnceBytes = 128ll << 20;
template <typename TD, typename TG, bool ONCE>
__global__ __launch_bounds__(kBlock) void run_sum_kernel(Runs a, const TD* __restrict__ dy, int64_t d, float scale,
                                                         TG* __restrict__ dw) {
  constexpr int V = vec_of<TD, float>(), kSlab = kWave * V;
  constexpr int U = 8;  // rows in flight
  const int64_t c = ((int64_t)blockIdx.z * gridDim.x + blockIdx.x) * kWaves + wave_id();
  const int64_t begin = c * a.chunk;
  if (begin >= a.n) return;
  const int cnt = (int)min((int64_t)a.chunk, a.n - begin);
  const int64_t col = (int64_t)blockIdx.y * kSlab + lane_id() * V;
  const int left = (int)max(min(d - col, (int64_t)V), (int64_t)0);
  const bool in = left > 0;
  const uint32_t before = begin > 0 ? a.key[begin - 1] : a.vocab;
  const uint32_t after = begin + cnt < a.n ? a.key[begin + cnt] : a.vocab;
  uint32_t lk = a.vocab, lv = 0;
  if (lane_id() < cnt) {
    lk = a.key[begin + lane_id()];
    lv = a.val[begin + lane_id()];
  }
  float acc[V] = {};
  uint32_t run = __builtin_amdgcn_readfirstlane(lk);
  bool first = true;  // the run holds the chunk's first place
  auto flush = [&](bool last) {
    if (run < a.vocab && in) {
      if (first && run == before) {
        store_vec(a.head + c * d + col, acc, left);
      } else if (last && run == after) {
        store_vec(a.tail + c * d + col, acc, left);
        if (blockIdx.y == 0 && lane_id() == 0) a.joins[1 + atomicAdd(a.joins, 1u)] = (uint32_t)c;
      } else {
        float o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = acc[i] * scale;
        store_vec(dw + (int64_t)run * d + col, o, left);
      }
    }
  };
  for (int i0 = 0; i0 < cnt; i0 += U) {
    Bits<TD, V> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t k = __builtin_amdgcn_readlane(lk, (i0 + u) & (kWave - 1));
      const uint32_t t = __builtin_amdgcn_readlane(lv, (i0 + u) & (kWave - 1));
#pragma unroll
      for (int i = 0; i < Bits<TD, V>::W; ++i) x[u].w[i] = 0;
      if (i0 + u < cnt && k < a.vocab && in) load_bits<ONCE>(dy + (int64_t)t * d + col, x[u], left);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i0 + u < cnt) {
        const uint32_t k = __builtin_amdgcn_readlane(lk, (i0 + u) & (kWave - 1));
        if (k != run) {
          flush(false);
          run = k;
          first = false;
#pragma unroll
          for (int i = 0; i < V; ++i) acc[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] += bits_at(x[u], i);
      }
    }
  }
  flush(true);
}

// Adds up the partial rows of the runs that cross chunks, each in chunk order: the workgroup's waves take
// every kJoinWaves-th partial row and meet in LDS.  An eighth of 65536 tokens the same, 1024 columns: 9.6 us, 4096 tokens
// 4.8 us, bound by the latency of a search and two loads.
constexpr int kJoinWaves = 8, kJoinBlocks = 1024;
template <typename TG>
__global__ __launch_bounds__(kJoinWaves* kWave) void run_join_kernel(Runs a, int64_t d, float scale,
                                                                     TG* __restrict__ dw) {
  constexpr int V = 4, kSlab = kWave * V, U = 8;
  __shared__ float part[kJoinWaves][kSlab];
  const uint32_t joins = a.joins[0], chunks = (uint32_t)((a.n + a.chunk - 1) / a.chunk);
  const int64_t col = (int64_t)blockIdx.y * kSlab + lane_id() * V;
  const int left = (int)max(min(d - col, (int64_t)V), (int64_t)0);
  for (uint32_t k = blockIdx.x; k < joins; k += gridDim.x) {
    const uint32_t c = a.joins[1 + k];
    // the last chunk that begins with the run: 64 places at a time
    uint32_t last = c + 1, end = chunks;
    const uint32_t run = a.key[(int64_t)last * a.chunk];
    while (end - last > 1) {
      const uint32_t step = (end - last + kWave - 1) / kWave;
      const uint64_t p = last + (uint64_t)(lane_id() + 1) * step;
      const uint32_t n = (uint32_t)__popcll(__ballot(p < end && a.key[p * a.chunk] == run));
      last += n * step;
      end = min(end, last + step);
    }
    float acc[V] = {};
    for (uint32_t j0 = c + wave_id(); j0 <= last; j0 += kJoinWaves * U) {
      float x[U][V];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t j = j0 + u * kJoinWaves;
#pragma unroll
        for (int i = 0; i < V; ++i) x[u][i] = 0.f;
        if (j <= last && left > 0) load_vec((j == c ? a.tail : a.head) + (int64_t)j * d + col, x[u], left);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] += x[u][i];
    }
    __syncthreads();  // the last run's parts have been read
#pragma unroll
    for (int i = 0; i < V; ++i) part[wave_id()][lane_id() * V + i] = acc[i];
    __syncthreads();
    if (wave_id() == 0 && left > 0) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int w = 1; w < kJoinWaves; ++w) acc[i] += part[w][lane_id() * V + i];
        acc[i] *= scale;
      }
      store_vec(dw + (int64_t)run * d + col, acc, left);
    }
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
int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// How n tokens are sorted and summed.
struct Plan {
  int per;        // pairs per thread of a sort
  int tiles;
  int chunk;
  int64_t chunks;
};
Plan plan_of(int64_t n) {
  Plan p{};
  if (n <= kSmall) {
    p.per = n <= kSmall / 4 ? 2 : n <= kSmall / 2 ? 4 : 8;
    p.tiles = 1;
  } else {
    p.per = n <= (int64_t)kManyTiles * kSortBlock * 2 ? 2 : 8;
    p.tiles = (int)cdiv(n, kSortBlock * p.per);
  }
  p.chunk = 8;
  while (p.chunk < 32 && n > 1024 * p.chunk) p.chunk *= 2;
  p.chunks = cdiv(n, p.chunk);
  return p;
}

template <typename F>
void by_per(int per, F&& f) {
  if (per == 2) f(std::integral_constant<int, 2>{});
  else if (per == 4) f(std::integral_constant<int, 4>{});
  else f(std::integral_constant<int, 8>{});
}

int passes_of(int64_t vocab, int* bits) {
  *bits = 1;
  while ((vocab >> *bits) != 0) ++*bits;  // keys 0 .. vocab
  return (*bits + 7) / 8;
}

}  // namespace

void embed_forward(const EmbedIds& ids, const void* w, ElType tw, int64_t w_stride, int64_t d, float scale, void* out,
                   ElType to, hipStream_t stream) {
  if (ids.n == 0 || d == 0) return;
  by_type(tw, [&](auto* tag_w) {
    using TW = std::remove_pointer_t<decltype(tag_w)>;
    by_type(to, [&](auto* tag_o) {
      using TO = std::remove_pointer_t<decltype(tag_o)>;
      int log = 0;
      while (log < 6 && ((int64_t)vec_of<TW, TO>() << log) < d) ++log;
      // a dimension of a grid holds less than 2^32 threads
      const int64_t blocks = cdiv(ids.n << log, kBlock), x = std::min<int64_t>(blocks, 1 << 23);
      const dim3 grid((unsigned)x, (unsigned)cdiv(blocks, x));
      embed_fwd_kernel<TW, TO><<<grid, kBlock, 0, stream>>>(ids, (const TW*)w, w_stride, d, scale, (TO*)out, log);
    });
  });
}

int64_t embed_backward_ws(int64_t n, int64_t vocab, int64_t d) {
  if (n <= kFew) return 0;
  const Plan p = plan_of(n);
  return 4 * align256(4 * n) + 2 * align256(4 * p.chunks * d) + align256(4 * (p.chunks + 1)) +
         (n > kSmall ? align256((int64_t)4 * (p.tiles + 1) * kRadix) : 0);
}

void embed_backward(const EmbedIds& ids, const void* dy, ElType tdy, int64_t d, float scale, void* dw, ElType tdw,
                    void* ws, hipStream_t stream) {
  if (ids.vocab == 0 || d == 0 || ids.n == 0) return;
  const int64_t n = ids.n;
  if (n <= kFew) {
    by_type(tdw, [&](auto* tag_g) {
      using TG = std::remove_pointer_t<decltype(tag_g)>;
      by_type(tdy, [&](auto* tag_d) {
        using TD = std::remove_pointer_t<decltype(tag_d)>;
        const int64_t slabs = cdiv(d, kWave * vec_of<TD, float>());
        // 64 KB to clear for a workgroup, but no more than kClearRows rows and no less than one; of rows of 64 bytes
        // and more the ids that it reads for it, 8 KB at most, are an eighth of that
        const int64_t each = std::max<int64_t>(1, std::min<int64_t>(kClearRows, 65536 / (d * (int64_t)sizeof(TG))));
        int log = 0;
        while (log < 8 && ((int64_t)(16 / sizeof(TG)) << log) < d) ++log;
        embed_few_kernel<TD, TG><<<(unsigned)(n * slabs + cdiv(ids.vocab, each)), kBlock, 0, stream>>>(
            ids, (const TD*)dy, d, scale, (TG*)dw, (int)slabs, (int)each, log);
      });
    });
    return;
  }
  const Plan plan = plan_of(n);
  char* at = static_cast<char*>(ws);
  auto take = [&](int64_t bytes) {
    char* p = at;
    at += align256(bytes);
    return p;
  };
  uint32_t* key[2] = {(uint32_t*)take(4 * n), (uint32_t*)take(4 * n)};
  uint32_t* val[2] = {(uint32_t*)take(4 * n), (uint32_t*)take(4 * n)};
  float* head = (float*)take(4 * plan.chunks * d);
  float* tail = (float*)take(4 * plan.chunks * d);
  uint32_t* joins = (uint32_t*)take(4 * (plan.chunks + 1));
  int bits;
  const int passes = passes_of(ids.vocab, &bits);
  const int64_t bytes = ids.vocab * d * el_bytes(tdw);
  int now = 0;
  by_per(plan.per, [&](auto per) {
    constexpr int PER = decltype(per)::value;
    if (n <= kSmall) {
      sort_small_kernel<PER><<<1 + kFillBlocks, kSortBlock, 0, stream>>>(ids, bits, passes, key[0], val[0], joins,
                                                                       Fill{dw, 0, bytes});
      return;
    }
    uint32_t* count = (uint32_t*)take((int64_t)4 * (plan.tiles + 1) * kRadix);
    const int64_t share = align256(cdiv(bytes, 2 * passes));  // of the fill, for each launch
    auto fill = [&](int k) { return Fill{dw, std::min(k * share, bytes), std::min((k + 1) * share, bytes)}; };
    const unsigned grid = plan.tiles + kFillBlocks;
    const bool scanned = plan.tiles > kScanTiles;
    for (int p = 0; p < passes; ++p) {
      const uint32_t *ik = p ? key[now] : nullptr, *iv = p ? val[now] : nullptr;
      now = p & 1;
      sort_count_kernel<PER><<<grid, kSortBlock, 0, stream>>>(ids, plan.tiles, ik, 8 * p, count, joins, fill(2 * p));
      if (scanned) sort_scan_kernel<<<kRadix, kSortBlock, 0, stream>>>(plan.tiles, count);
      sort_move_kernel<PER><<<grid, kSortBlock, 0, stream>>>(ids, plan.tiles, ik, iv, 8 * p, count, scanned, key[now],
                                                            val[now], fill(2 * p + 1));
    }
  });
  const Runs runs{key[now], val[now], n, (uint32_t)ids.vocab, plan.chunk, head, tail, joins};
  by_type(tdw, [&](auto* tag_g) {
    using TG = std::remove_pointer_t<decltype(tag_g)>;
    by_type(tdy, [&](auto* tag_d) {
      using TD = std::remove_pointer_t<decltype(tag_d)>;
      const unsigned slabs = (unsigned)cdiv(d, kWave * vec_of<TD, float>());
      // a dimension of a grid holds less than 2^32 threads
      const int64_t blocks = cdiv(plan.chunks, kWaves), x = std::min<int64_t>(blocks, 1 << 23);
      const dim3 grid((unsigned)x, slabs, (unsigned)cdiv(blocks, x));
      if (n * d * (int64_t)sizeof(TD) >= kOnceBytes)
        run_sum_kernel<TD, TG, true><<<grid, kBlock, 0, stream>>>(runs, (const TD*)dy, d, scale, (TG*)dw);
      else
        run_sum_kernel<TD, TG, false><<<grid, kBlock, 0, stream>>>(runs, (const TD*)dy, d, scale, (TG*)dw);
    });
    run_join_kernel<TG><<<dim3((unsigned)std::min<int64_t>(plan.chunks, kJoinBlocks), (unsigned)cdiv(d, kWave * 4)),
                          kJoinWaves * kWave, 0, stream>>>(runs, d, scale, (TG*)dw);
  });
}

}  // namespace grace
