// Residual norms: the norm after a block, its gate, the scaled residual and the norm before the
// next block in one pass, and their backward.
//
//   u = post ? N(y; pw, pb) : y        s = alpha * x + gate . u        h = N(s; w, b)
//   N(v; w, b) = (v - m) r w + b,  r = 1 / sqrt(mean((v - m)^2) + eps),  m = mean(v) (rms: m = 0)
//
// Backward, with v^ = (v - m) r and a = w . dh:
//   S  = r (a - mean(a) - s^ mean(a s^)) + ds     (rms: without mean(a))
//   dx = alpha S      du = gate . S      dgate = sum S . u      dw = sum dh . s^      db = sum dh
//   dy = du, or with post, a' = pw . du:  ry (a' - mean(a') - y^ mean(a' y^)),
//        dpw = sum du . y^,  dpb = sum du
//
// A row lives in registers (E values per thread), so every input is read once and the variance is
// taken about the mean in a second sweep over registers.  16, 64, 256, 512 or 1024 threads share a row,
// by its width; a workgroup walks over rows with the weights at hand, and rows that need a workgroup's
// barriers are loaded one ahead.  Statistics and sums are fp32; s is rounded to its own
// type only where it is stored, and h is made from the unrounded sum.  The backward reads the stored
// sum if that is fp32; a 16-bit sum is made again from x and y, because its rounding would show in
// the fp32 sums dw (2^-9 of every term against 2^-24).
// Column sums (dw, db, dgate, dpw, dpb): every workgroup adds up its rows in registers and leaves one
// partial row; a second launch adds the partial rows in a fixed order.
//
// Bound by memory: a copy runs at 5.2 TB/s.  64 million values in whole vectors, forward and backward: bf16 widths of
// 64 to 16384 at 4.7-5.5 and 4.0-4.4 TB/s, fp32 at 4.7-5.5 and 4.1-4.9.  With a norm behind the block and a gate, rms and
// without biases: up to 8192 columns 4.4-5.5 and 3.1-4.9, wider ones 3.8-4.2 and, for want of registers, 2.5 (bf16) and
// 4.2 (fp32).  With both biases more registers are short: up to 8192 columns 3.5-5.4 and 2.9-4.8 in whole vectors, 12000
// columns 3.1-3.3 and 0.8 (bf16) and 1.8 (fp32).  An fp32 stream with a bf16 block up to 8192 columns: 4.9-5.6 and 4.4-4.6.
#pragma once

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "grace_common.h"
#include "grace_lm.h"

namespace grace {
namespace resnorm {

constexpr int kCUs = 256;

template <int TPR>
constexpr int block_of() { return TPR < 256 ? 256 : TPR; }

// Values per load: 16 bytes of the narrower type where the rows are whole vectors.  A row that ends inside one is
// taken by single values, or pairs of 16 bits, so that a wave's accesses are aligned and next to each other: wide ones
// of 16-bit values at odd addresses run at half the rate, and the branches of a partial vector cost registers and waits
// (bf16, forward and backward: 1100 columns 3.8 and 4.2 TB/s as pairs, 3.6 and 2.8 as single values, 2.3 and 2.4 as
// vectors; 651 columns 4.1 and 3.7 as single values, 3.5 and 3.8 as vectors).
template <typename TY>
constexpr int vec_of() { return sizeof(TY) == 2 ? 8 : 4; }
template <typename TY, typename F>
void by_vec(int d, F&& f) {
  using std::integral_constant;
  if (d % vec_of<TY>() == 0) f(integral_constant<int, vec_of<TY>()>{});
  else if (sizeof(TY) == 2 && d % 2 == 0) f(integral_constant<int, sizeof(TY) == 2 ? 2 : 1>{});
  else f(integral_constant<int, 1>{});
}

struct FwdArgs {
  NormShape n;
  const void *x, *y;
  NormParam gate, weight, bias, post_weight, post_bias;
  void *h, *s;
  float* stats;
};

// How the workgroups of the backward share the rows.  A gate's sums end with its group of rows: long
// groups are cut into parts (one partial row of dgate per part), of short groups a workgroup takes
// whole ones and writes their dgate itself.
struct Split {
  int64_t groups;      // groups of rows (1 without a gate whose sums are wanted)
  int64_t group_rows;
  int64_t parts;       // workgroups per group, or 1
  int64_t per_block;   // groups per workgroup, or 1
  int64_t blocks;
};

enum { kDw, kDb, kDg, kDpw, kDpb, kSums };
enum { kGateNone, kGateParts, kGateGroups, kGateRows };  // dgate: not wanted, partial rows, per group, per row

struct BwdArgs {
  NormShape n;
  Split split;
  const void *s, *x, *y, *dh, *ds;  // s = nullptr: made again from x and y
  const float* stats;
  NormParam gate, weight, post_weight, post_bias;
  void *dx, *dy, *dgate;
  bool dgate_f32;
  bool once;  // nontemporal stores
  bool want[kSums];
  int dgate_mode;
  float* part;  // [sums][blocks][d]
};

// ---------------------------------------------------------------- a row in registers
// Sum over the wave, in every lane.  DPP steps: a tenth of the latency of LDS permutes.
__device__ __forceinline__ float dpp_sum(float v) {
#define GRACE_DPP(ctrl, rows) \
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, rows, 0xf, true))
  GRACE_DPP(0x111, 0xf);  // within rows of 16 lanes: shifted by 1, 2, 4, 8
  GRACE_DPP(0x112, 0xf);
  GRACE_DPP(0x114, 0xf);
  GRACE_DPP(0x118, 0xf);
  GRACE_DPP(0x142, 0xa);  // lane 15 of a row to the next one
  GRACE_DPP(0x143, 0xc);  // lane 31 to the upper half
#undef GRACE_DPP
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// Sum over 16 lanes, in each of them: rotations within the row of lanes.
__device__ __forceinline__ float dpp_sum16(float v) {
#define GRACE_ROR(n) v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + n, 0xf, 0xf, true))
  GRACE_ROR(8);
  GRACE_ROR(4);
  GRACE_ROR(2);
  GRACE_ROR(1);
#undef GRACE_ROR
  return v;
}

// Sums over the TPR threads of a row.  More than one wave: one barrier a sum, on two buffers in turn
// (a wave can be at most one barrier ahead of another).
template <int TPR>
struct RowSum {
  static constexpr int W = TPR / kWave;
  float* scratch;  // [2][2 W]
  int turn = 0;
  __device__ __forceinline__ void operator()(float& a, float& b) {
    a = TPR == 16 ? dpp_sum16(a) : dpp_sum(a);
    b = TPR == 16 ? dpp_sum16(b) : dpp_sum(b);
    if constexpr (W > 1) {
      float* q = scratch + turn * 2 * W;
      turn ^= 1;
      if (lane_id() == 0) {
        q[2 * wave_id()] = a;
        q[2 * wave_id() + 1] = b;
      }
      __syncthreads();
      a = q[0];
      b = q[1];
#pragma unroll
      for (int i = 1; i < W; ++i) {
        a += q[2 * i];
        b += q[2 * i + 1];
      }
    }
  }
  __device__ __forceinline__ void operator()(float& a) {
    float b = 0.f;
    (*this)(a, b);
  }
};

template <typename T, int V, int J>
struct Raw {
  Bits<T, V> v[J];
};

// The width is a multiple of V.
template <int TPR, int V, int J>
struct Row {
  int t, d;
  __device__ __forceinline__ Row(int t, int d) : t(t), d(d) {}
  __device__ __forceinline__ int col(int j) const { return (j * TPR + t) * V; }
  __device__ __forceinline__ bool in(int j) const { return col(j) < d; }  // vector j is inside the width

  // as stored; zero outside the width, or everywhere without a pointer
  template <typename T>
  __device__ __forceinline__ void load(const void* p, int64_t at, Raw<T, V, J>& r) const {
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int i = 0; i < Bits<T, V>::W; ++i) r.v[j].w[i] = 0;
    // asked once of 4 to 16 narrow accesses, but of every wide one: two or four of them run better so
    const bool there = p != nullptr;
    if (V < 4 && !there) return;
#pragma unroll
    for (int j = 0; j < J; ++j)
      if ((V < 4 || there) && in(j)) load_bits(static_cast<const T*>(p) + at + col(j), r.v[j]);
  }
  // Before the first use of r: 16-bit values in narrow accesses are widened behind this, not where each is loaded, which
  // would make every load wait for the one before it.
  template <typename T>
  __device__ __forceinline__ void arrive(Raw<T, V, J>& r) const {
    if constexpr (V < 4 && sizeof(T) == 2) {
#pragma unroll
      for (int j = 0; j < J; ++j) asm volatile("" : "+v"(r.v[j].w[0]));
    }
  }
  template <typename T>
  __device__ __forceinline__ void widened(const void* p, int64_t at, float (&o)[J][V]) const {
    Raw<T, V, J> r;
    load<T>(p, at, r);
    arrive(r);
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) o[j][i] = bits_at(r.v[j], i);
  }
  // widened; zero outside the width
  template <typename TY>
  __device__ __forceinline__ void param(const NormParam& p, int64_t at, float (&o)[J][V]) const {
    if (p.f32) widened<float>(p.p, at, o);
    else widened<TY>(p.p, at, o);
  }
  template <typename T>
  __device__ __forceinline__ void store(void* p, int64_t at, const float (&v)[J][V], bool once) const {
    // narrow accesses leave lines in parts, for the cache to join (fp32, 130 columns: 280 us past it, 235 us through it)
    if constexpr (V > 2) {
      if (once) {
#pragma unroll
        for (int j = 0; j < J; ++j)
          if (in(j)) store_vec<true>(static_cast<T*>(p) + at + col(j), v[j]);
        return;
      }
    }
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (in(j)) store_vec<false>(static_cast<T*>(p) + at + col(j), v[j]);
  }
  // mean and 1 / deviation of v, which is zero outside the width
  __device__ __forceinline__ void stats(const float (&v)[J][V], bool rms, float eps, RowSum<TPR>& sum, float& mean,
                                        float& rstd) const {
    float a = 0.f;
    mean = 0.f;
    if (!rms) {
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) a += v[j][i];
      sum(a);
      mean = a / (float)d;
    }
    a = 0.f;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if (in(j)) {
#pragma unroll
        for (int i = 0; i < V; ++i) a = fmaf(v[j][i] - mean, v[j][i] - mean, a);
      }
    }
    sum(a);
    rstd = 1.f / sqrtf(a / (float)d + eps);
  }
  // zero outside the width
  __device__ __forceinline__ void trim(float (&v)[J][V]) const {
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (!in(j)) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[j][i] = 0.f;
      }
  }
};

// Where the weights and the gate of a workgroup's rows are, each thread's own values of them.
//   registers  backward of rows of a wave or less, forward of rows of 1024 threads
//   LDS        where they cost no registers: the registers decide how many rows a CU has in flight.  A thread reads
//              what it wrote, or what the other row slots wrote to the same place, the same bits: no barriers.  An
//              array takes 4 KB for rows of 64 threads and 16 values, 16 KB for 512 threads, 32 KB for 1024; the gate
//              takes that for every row slot, for their rows may have different ones.
//   memory     from the caches: backward of rows of 16 values for each of 1024 threads, whose registers and LDS hold no
//              more, and forward of some rows of a wave
enum Home { kInRegisters, kInLds, kInMemory };

enum { kW, kB, kPw, kPb, kG, kParams };

template <int K, int TPR, int V, int J, Home HOME>
struct Params {
  static constexpr int kFloats = HOME == kInLds ? TPR * V * J : 0;  // of LDS, for each array
  static constexpr int kAccess = V < 4 ? V : 4;                     // values of an LDS access
  struct alignas(4 * kAccess) Part {
    float v[kAccess];
  };
  float r[HOME == kInRegisters ? K : 1][J][V];
  Part* lds;
  Part* own;  // the row slot's
  __device__ __forceinline__ explicit Params(float* p)
      : lds(reinterpret_cast<Part*>(p) + threadIdx.x % TPR), own(lds + threadIdx.x / TPR * (J * V / kAccess) * TPR) {}
  __device__ __forceinline__ Part& part(int place, int j, int i, bool slot = false) const {
    return (slot ? own : lds)[((place * J + j) * (V / kAccess) + i / kAccess) * TPR];
  }
  // k: the array (a constant), place: its place in LDS, from + at: where it is in memory
  template <typename TY>
  __device__ __forceinline__ void set(int k, int place, const Row<TPR, V, J>& row, const NormParam& from, int64_t at) {
    if constexpr (HOME == kInMemory) return;
    float v[J][V];
    row.template param<TY>(from, at, v);
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int i = 0; i < V; i += kAccess) {
        Part q;
#pragma unroll
        for (int m = 0; m < kAccess; ++m) q.v[m] = v[j][i + m];
        if constexpr (HOME == kInLds) {
          part(place, j, i, k == kG) = q;
        } else {
#pragma unroll
          for (int m = 0; m < kAccess; ++m) r[k][j][i + m] = q.v[m];
        }
      }
  }
  template <typename TY>
  __device__ __forceinline__ void get(int k, int place, const Row<TPR, V, J>& row, const NormParam& from, int64_t at,
                                      float (&v)[J][V]) const {
    if constexpr (HOME == kInMemory) {
      int64_t none = 0;  // which the compiler can't see: it would keep narrow ones in registers, 16 for each array
      if constexpr (V < 4) asm volatile("" : "+s"(none));
      row.template param<TY>(from, at + none, v);
    } else {
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int i = 0; i < V; i += kAccess) {
          if constexpr (HOME == kInLds) {
            const Part q = part(place, j, i, k == kG);
#pragma unroll
            for (int m = 0; m < kAccess; ++m) v[j][i + m] = q.v[m];
          } else {
#pragma unroll
            for (int m = 0; m < kAccess; ++m) v[j][i + m] = r[k][j][i + m];
          }
        }
    }
  }
};

// Column sums of a thread's own values, in registers or, where those are short, in LDS (places as Params').
template <int TPR, int V, int J, bool LDS>
struct ColumnSum {
  using Lds = Params<1, TPR, V, J, kInLds>;
  float r[LDS ? 1 : J][V];
  Lds at;
  __device__ __forceinline__ explicit ColumnSum(float* p) : at(p) { clear(); }
  __device__ __forceinline__ void clear() { each([](float, int, int) { return 0.f; }); }
  __device__ __forceinline__ void add(const float (&x)[J][V]) {
    each([&](float a, int j, int i) { return a + x[j][i]; });
  }
  __device__ __forceinline__ void fma(const float (&x)[J][V], const float (&y)[J][V]) {
    each([&](float a, int j, int i) { return fmaf(x[j][i], y[j][i], a); });
  }
  __device__ __forceinline__ void get(float (&v)[J][V]) {
    each([&](float a, int j, int i) { return v[j][i] = a; });
  }
  template <typename F>
  __device__ __forceinline__ void each(F&& f) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if constexpr (LDS) {
#pragma unroll
        for (int i = 0; i < V; i += Lds::kAccess) {
          typename Lds::Part q = at.part(0, j, i);
#pragma unroll
          for (int m = 0; m < Lds::kAccess; ++m) q.v[m] = f(q.v[m], j, i + m);
          at.part(0, j, i) = q;
        }
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) r[j][i] = f(r[j][i], j, i);
      }
    }
  }
};

// the workgroup's slot of rows; known to be the same in a wave where it is
template <int TPR>
__device__ __forceinline__ int row_slot() {
  if constexpr (block_of<TPR>() == TPR) return 0;
  else if constexpr (TPR < kWave) return threadIdx.x / TPR;
  else return __builtin_amdgcn_readfirstlane(threadIdx.x / TPR);
}

// Which arrays there are, and their places in LDS (-1: not there).
struct ParamPlaces {
  int at[kParams], n = 0;
  __host__ __device__ __forceinline__ ParamPlaces(const void* w, const void* b, const void* gate, const void* pw,
                                                  const void* pb) {
    const void* p[kParams] = {w, b, pw, pb, gate};
#pragma unroll
    for (int k = 0; k < kParams; ++k) at[k] = p[k] != nullptr ? n++ : -1;
  }
};

// Forward: at most five arrays in LDS, 80 KB; 1024 threads would take 160 KB.  Theirs are in registers, of which 8 values a
// thread take 82 to 97; with 16 values 128 do not hold them, and 60 to 186 are spilled (12000 columns, all five arrays: 3.3
// TB/s in bf16, 3.1 in fp32).  fp32 rows of 16 values a thread take them from the caches, when their sums are done: 4096 rows of 768 take 10.4 us and 11.3 with LDS,
// which is filled before the first row; in 16 bits (64 million values in rows of 650) 3.6 TB/s and 4.4 with LDS.
template <typename TY, int E, int TPR>
constexpr Home forward_home() {
  return TPR == 1024 ? kInRegisters : E == 16 && sizeof(TY) == 4 ? kInMemory : kInLds;
}
// Backward: at most four arrays in LDS, 128 KB.
template <int E, int TPR>
constexpr Home backward_home() { return TPR <= kWave ? kInRegisters : E == 8 ? kInLds : kInMemory; }

// Rows of 16 values for each of 1024 threads with a post norm or a gate: two of the sums in LDS, 128 KB, for the
// weights are not there.  All of them in 128 registers would spill: 12000 columns with both, backward,
// 0.8 TB/s for 2.5 in bf16 and 2.0 for 4.2 in fp32.
template <int E, int TPR, bool POST, bool GATED>
constexpr bool sums_in_lds() { return backward_home<E, TPR>() == kInMemory && (POST || GATED); }

#define GRACE_EACH(body)          \
  _Pragma("unroll") for (int j = 0; j < J; ++j) \
  _Pragma("unroll") for (int i = 0; i < V; ++i) { body; }

// ---------------------------------------------------------------- forward
template <typename TX, typename TY, int E, int TPR, int V>
__global__ __launch_bounds__(block_of<TPR>()) void resnorm_fwd_kernel(FwdArgs g) {
  constexpr int J = E / V, kSlots = block_of<TPR>() / TPR;
  __shared__ float scratch[TPR > kWave ? 4 * TPR / kWave : 1];
  RowSum<TPR> sum{scratch};
  const NormShape& n = g.n;
  const Row<TPR, V, J> row(threadIdx.x % TPR, n.d);
  const uint32_t rows = (uint32_t)n.rows, step = gridDim.x * kSlots, gate_rows = (uint32_t)n.gate_rows;
  uint32_t r = blockIdx.x * kSlots + row_slot<TPR>();
  if (r >= rows) return;
  constexpr bool AHEAD = TPR > kWave;
  Raw<TY, V, J> ry;
  Raw<TX, V, J> rx;
  auto fetch = [&](uint32_t q) {
    row.load(g.y, (int64_t)q * n.d, ry);
    row.load(g.x, (int64_t)q * n.d, rx);
  };
  fetch(r);
  extern __shared__ __align__(16) float dyn[];
  Params<kParams, TPR, V, J, forward_home<TY, E, TPR>()> params(dyn);
  const ParamPlaces places(g.weight.p, g.bias.p, g.gate.p, n.post ? g.post_weight.p : nullptr,
                           n.post ? g.post_bias.p : nullptr);
  auto put = [&](int k, const NormParam& from) {
    if (places.at[k] >= 0) params.template set<TY>(k, places.at[k], row, from, 0);
  };
  put(kW, g.weight);
  put(kB, g.bias);
  put(kPw, g.post_weight);
  put(kPb, g.post_bias);
  auto take = [&](int k, const NormParam& from, float(&v)[J][V]) {
    params.template get<TY>(k, places.at[k], row, from, 0, v);
  };
  uint32_t gate_now = ~0u;
  for (;;) {
    const int64_t at = (int64_t)r * n.d;
    float u[J][V], x[J][V], p[J][V], mean, rstd;
    // a gate that stays is not loaded again: a load here would make the row wait for the last one's stores
    if (g.gate.p != nullptr && r / gate_rows != gate_now) {
      gate_now = r / gate_rows;
      params.template set<TY>(kG, places.at[kG], row, g.gate, (int64_t)gate_now * n.d);
    }
    row.arrive(ry);
    row.arrive(rx);
    GRACE_EACH(u[j][i] = bits_at(ry.v[j], i); x[j][i] = bits_at(rx.v[j], i))
    const bool more = rows - r > step;
    if (AHEAD && more) fetch(r + step);
    if (n.post) {
      row.stats(u, n.rms, n.eps, sum, mean, rstd);
      if (g.stats != nullptr && row.t == 0) {
        g.stats[2 * n.rows + r] = mean;
        g.stats[3 * n.rows + r] = rstd;
      }
      GRACE_EACH(u[j][i] = (u[j][i] - mean) * rstd)
      if (g.post_weight.p != nullptr) {
        take(kPw, g.post_weight, p);
        GRACE_EACH(u[j][i] *= p[j][i])
      }
      if (g.post_bias.p != nullptr) {
        take(kPb, g.post_bias, p);
        GRACE_EACH(u[j][i] += p[j][i])
      }
    }
    if (g.gate.p != nullptr) {
      params.template get<TY>(kG, places.at[kG], row, g.gate, (int64_t)gate_now * n.d, p);
      GRACE_EACH(u[j][i] *= p[j][i])
    }
    if (g.x != nullptr) GRACE_EACH(u[j][i] = fmaf(n.alpha, x[j][i], u[j][i]))
    row.trim(u);
    if (g.s != nullptr) row.template store<TX>(g.s, at, u, false);
    row.stats(u, n.rms, n.eps, sum, mean, rstd);
    if (g.stats != nullptr && row.t == 0) {
      g.stats[r] = mean;
      g.stats[n.rows + r] = rstd;
    }
    GRACE_EACH(u[j][i] = (u[j][i] - mean) * rstd)
    if (g.weight.p != nullptr) {
      take(kW, g.weight, p);
      GRACE_EACH(u[j][i] *= p[j][i])
    }
    if (g.bias.p != nullptr) {
      take(kB, g.bias, p);
      GRACE_EACH(u[j][i] += p[j][i])
    }
    row.template store<TY>(g.h, at, u, false);
    if (!more) return;
    r += step;
    if (!AHEAD) fetch(r);
  }
}

// ---------------------------------------------------------------- backward
template <typename TY, int V>
__device__ __forceinline__ void store_param(void* p, bool f32, int64_t at, const float (&v)[V]) {
  if (f32) store_vec(static_cast<float*>(p) + at, v);
  else store_vec(static_cast<TY*>(p) + at, v);
}

// Sums acc over the workgroup's row slots and hands each vector to out(column, values); acc
// is left as it is.  red: [slots][TPR * E] floats for more than one slot.
template <int TPR, int V, int J, typename F>
__device__ __forceinline__ void over_slots(const float (&acc)[J][V], const Row<TPR, V, J>& row, float* red, F&& out) {
  if constexpr (block_of<TPR>() > TPR) {
    constexpr int kSlots = block_of<TPR>() / TPR, kRow = TPR * V * J;
    __syncthreads();  // red has been read
    GRACE_EACH(red[(threadIdx.x / TPR) * kRow + row.col(j) + i] = acc[j][i])
    __syncthreads();
    for (int c = threadIdx.x * V; c < row.d; c += block_of<TPR>() * V) {
      float v[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        v[i] = red[c + i];
#pragma unroll
        for (int k = 1; k < kSlots; ++k) v[i] += red[k * kRow + c + i];
      }
      out(c, v);
    }
  } else {
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (row.in(j)) out(row.col(j), acc[j]);
  }
}

// BIAS: one of the two biases is there.  Four waves to a SIMD hold 128 registers each: a few of them spilled cost less
// than the fourth wave (fp32, 1536 columns, gate and post norm: 332 us, 362 us with three waves of 131 registers).  Single
// values in rows of 512 threads, odd widths of 2049 to 4095, pay more for it: 63 to 199 registers are spilled (bf16, 3001
// columns: 3.3 TB/s, with gate, post norm and biases 1.2).
template <typename TX, typename TY, int E, int TPR, int V, bool POST, bool GATED, bool BIAS>
__global__ __launch_bounds__(block_of<TPR>(),
                             TPR == 512 || (TPR == 256 && V > 1) ? 4 : 1) void resnorm_bwd_kernel(BwdArgs g) {
  constexpr int J = E / V, kSlots = block_of<TPR>() / TPR;
  // The next row's loads are issued before this row's sums, where registers hold them: 1024 threads have 128 each, and a
  // single 16-bit value takes as much of them as two in a vector.
  constexpr bool kShort = sizeof(TY) == 2 ? V < (TPR == 1024 ? 4 : 2) : TPR == 1024 && (POST || GATED);
  constexpr bool AHEAD = TPR > kWave && E == 8 && !kShort;
  __shared__ float scratch[TPR > kWave ? 4 * TPR / kWave : 1];
  __shared__ float red[kSlots > 1 ? kSlots * TPR * E : 1];
  RowSum<TPR> sum{scratch};
  const NormShape& n = g.n;
  const Row<TPR, V, J> row(threadIdx.x % TPR, n.d);
  extern __shared__ __align__(16) float dyn[];
  constexpr bool kLds = sums_in_lds<E, TPR, POST, GATED>();
  ColumnSum<TPR, V, J, kLds> dw(dyn);
  ColumnSum<TPR, V, J, kLds && POST> dpw(dyn + TPR * E);
  ColumnSum<TPR, V, J, kLds && !POST> dg(dyn + TPR * E);
  ColumnSum<TPR, V, J, false> db(dyn), dpb(dyn);
  Params<2 + 2 * POST, TPR, V, J, backward_home<E, TPR>()> params(dyn);
  constexpr int W = 0, G = 1, PW = 2, PB = 3;  // the places in registers
  const ParamPlaces places(g.weight.p, nullptr, g.gate.p, POST ? g.post_weight.p : nullptr,
                           POST && BIAS ? g.post_bias.p : nullptr);
  if (g.weight.p != nullptr) params.template set<TY>(W, places.at[kW], row, g.weight, 0);
  if constexpr (POST) {
    if (g.post_weight.p != nullptr) params.template set<TY>(PW, places.at[kPw], row, g.post_weight, 0);
    if constexpr (BIAS)
      if (g.post_bias.p != nullptr) params.template set<TY>(PB, places.at[kPb], row, g.post_bias, 0);
  }
  const bool again = sizeof(TX) == 2 && g.s == nullptr;
  const void* sx = again ? g.x : g.s;
  const void* y_read = POST || GATED || again ? g.y : nullptr;
  const float inv_d = 1.f / (float)n.d;
  const uint32_t part = (uint32_t)(blockIdx.x % g.split.parts);
  const uint32_t g0 = (uint32_t)(blockIdx.x / g.split.parts * g.split.per_block);
  const uint32_t g1 = (uint32_t)min((int64_t)g0 + g.split.per_block, g.split.groups);
  const uint32_t group_rows = (uint32_t)g.split.group_rows, gate_rows = (uint32_t)n.gate_rows;
  const uint32_t chunk = (uint32_t)((g.split.group_rows + g.split.parts - 1) / g.split.parts);
  uint32_t gate_now = ~0u;
  Raw<TX, V, J> rs, rds;
  Raw<TY, V, J> ry, rdh;
  auto fetch = [&](uint32_t r) {
    const int64_t at = (int64_t)r * n.d;
    row.load(sx, at, rs);
    row.load(g.dh, at, rdh);
    row.load(y_read, at, ry);
    row.load(g.ds, at, rds);
  };
  for (uint32_t grp = g0; grp < g1; ++grp) {
    const uint32_t r_end = grp * group_rows + (uint32_t)min((uint64_t)(part + 1) * chunk, (uint64_t)group_rows);
    const uint32_t r_begin = grp * group_rows + (uint32_t)min((uint64_t)part * chunk, (uint64_t)group_rows) + row_slot<TPR>();
    if (AHEAD && r_begin < r_end) fetch(r_begin);
    for (uint32_t r = r_begin; r < r_end; r += kSlots) {
      const int64_t at = (int64_t)r * n.d;
      if constexpr (!AHEAD) fetch(r);
      const float mean = g.stats[r], rstd = g.stats[n.rows + r];
      const float pmean = POST ? g.stats[2 * n.rows + r] : 0.f, prstd = POST ? g.stats[3 * n.rows + r] : 1.f;
      if constexpr (GATED) {
        if (r / gate_rows != gate_now) {
          gate_now = r / gate_rows;
          params.template set<TY>(G, places.at[kG], row, g.gate, (int64_t)gate_now * n.d);
        }
      }
      float S[J][V], hat[J][V], phat[J][V], ds[J][V], p[J][V];
      // u of the forward, without its gate, from phat
      auto made_u = [&](float(&u)[J][V]) {
        GRACE_EACH(u[j][i] = phat[j][i])
        if constexpr (POST) {
          if (g.post_weight.p != nullptr) {
            params.template get<TY>(PW, places.at[kPw], row, g.post_weight, 0, p);
            GRACE_EACH(u[j][i] *= p[j][i])
          }
          if constexpr (BIAS) {
            if (g.post_bias.p != nullptr) {
              params.template get<TY>(PB, places.at[kPb], row, g.post_bias, 0, p);
              GRACE_EACH(u[j][i] += p[j][i])
            }
          }
        }
      };
      float c1 = 0.f, c2 = 0.f;
      row.arrive(ry);
      row.arrive(rs);
      row.arrive(rdh);
      row.arrive(rds);
      GRACE_EACH(phat[j][i] = bits_at(ry.v[j], i); hat[j][i] = bits_at(rs.v[j], i); S[j][i] = bits_at(rdh.v[j], i);
                 ds[j][i] = bits_at(rds.v[j], i))
      if (AHEAD && r + kSlots < r_end) fetch(r + kSlots);
      // outside the width everything stays zero: a large mean there would make an infinity of zero, and NaN of the sums
      if constexpr (POST) GRACE_EACH(phat[j][i] = (phat[j][i] - (row.in(j) ? pmean : 0.f)) * prstd)
      if (again) {
        float u[J][V];
        made_u(u);
        if constexpr (GATED) {
          params.template get<TY>(G, places.at[kG], row, g.gate, (int64_t)gate_now * n.d, p);
          GRACE_EACH(u[j][i] *= p[j][i])
        }
        GRACE_EACH(hat[j][i] = fmaf(n.alpha, hat[j][i], u[j][i]))
      }
      GRACE_EACH(hat[j][i] = (hat[j][i] - (row.in(j) ? mean : 0.f)) * rstd)
      dw.fma(S, hat);
      if constexpr (BIAS) db.add(S);
      if (g.weight.p != nullptr) {
        params.template get<TY>(W, places.at[kW], row, g.weight, 0, p);
        GRACE_EACH(S[j][i] *= p[j][i])
      }
      GRACE_EACH(c1 += S[j][i]; c2 = fmaf(S[j][i], hat[j][i], c2))
      sum(c1, c2);
      c1 = n.rms ? 0.f : c1 * inv_d;
      c2 *= inv_d;
      GRACE_EACH(S[j][i] = rstd * (S[j][i] - c1 - hat[j][i] * c2))
      if (g.dh == nullptr) GRACE_EACH(S[j][i] = 0.f)
      GRACE_EACH(S[j][i] += ds[j][i])
      row.trim(S);
      if (g.dx != nullptr) {
        GRACE_EACH(ds[j][i] = n.alpha * S[j][i])
        row.template store<TX>(g.dx, at, ds, g.once);
      }
      if constexpr (GATED) {
        float u[J][V];
        made_u(u);
        params.template get<TY>(G, places.at[kG], row, g.gate, (int64_t)gate_now * n.d, p);
        GRACE_EACH(u[j][i] *= S[j][i]; S[j][i] *= p[j][i])
        if (g.dgate_mode == kGateRows) {
#pragma unroll
          for (int j = 0; j < J; ++j)
            if (row.in(j)) store_param<TY>(g.dgate, g.dgate_f32, at + row.col(j), u[j]);
        } else {
          dg.add(u);
        }
      }
      if constexpr (POST) {
        c1 = c2 = 0.f;
        dpw.fma(S, phat);
        if constexpr (BIAS) dpb.add(S);
        if (g.post_weight.p != nullptr) {
          params.template get<TY>(PW, places.at[kPw], row, g.post_weight, 0, p);
          GRACE_EACH(S[j][i] *= p[j][i])
        }
        GRACE_EACH(c1 += S[j][i]; c2 = fmaf(S[j][i], phat[j][i], c2))
        sum(c1, c2);
        c1 = n.rms ? 0.f : c1 * inv_d;
        c2 *= inv_d;
        GRACE_EACH(S[j][i] = prstd * (S[j][i] - c1 - phat[j][i] * c2))
      }
      row.template store<TY>(g.dy, at, S, g.once);
    }
    if constexpr (GATED) {
      if (g.dgate_mode == kGateGroups) {
        float v[J][V];
        dg.get(v);
        over_slots(v, row, red, [&](int c, const float(&v)[V]) {
          store_param<TY>(g.dgate, g.dgate_f32, (int64_t)grp * n.d + c, v);
        });
        dg.clear();
      }
    }
  }
  const int64_t plane = g.split.blocks * n.d;
  auto leave = [&](int which, auto& sum) {
    if (!g.want[which]) return;
    float* to = g.part + which * plane + blockIdx.x * (int64_t)n.d;
    float acc[J][V];
    sum.get(acc);
    over_slots(acc, row, red, [&](int c, const float(&v)[V]) { store_vec(to + c, v); });
  };
  leave(kDw, dw);
  if constexpr (BIAS) leave(kDb, db);
  if constexpr (GATED) leave(kDg, dg);
  if constexpr (POST) {
    leave(kDpw, dpw);
    if constexpr (BIAS) leave(kDpb, dpb);
  }
}

// ---------------------------------------------------------------- launches
// Values per thread and threads per row, by the row's width.  Narrow rows share a wave by fours (64 bf16 columns,
// forward and backward: 4.7 and 4.3 TB/s, with a wave for each row 0.9 and 1.6); more than 16 values to a thread
// would spill, and a row is spread over no more waves than it needs, for each sum waits for all of them.
template <typename F>
void by_width(int d, F&& f) {
  using std::integral_constant;
  if (d <= 16 * 8) f(integral_constant<int, 8>{}, integral_constant<int, 16>{});
  else if (d <= 16 * 16) f(integral_constant<int, 16>{}, integral_constant<int, 16>{});
  else if (d <= 64 * 8) f(integral_constant<int, 8>{}, integral_constant<int, 64>{});
  else if (d <= 64 * 16) f(integral_constant<int, 16>{}, integral_constant<int, 64>{});
  else if (d <= 256 * 8) f(integral_constant<int, 8>{}, integral_constant<int, 256>{});
  else if (d <= 512 * 8) f(integral_constant<int, 8>{}, integral_constant<int, 512>{});
  else if (d <= 1024 * 8) f(integral_constant<int, 8>{}, integral_constant<int, 1024>{});
  else f(integral_constant<int, 16>{}, integral_constant<int, 1024>{});
}

// More than 64 KB of dynamic LDS has to be asked for, once for each kernel and device.
template <auto Kernel>
void allow_lds(unsigned bytes) {
  if (bytes <= 60 * 1024) return;
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev > 63) dev = 63;
  if (done.load(std::memory_order_relaxed) >> dev & 1) return;
  if (hipFuncSetAttribute(reinterpret_cast<const void*>(Kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                          140 * 1024) == hipSuccess && dev < 63)
    done.fetch_or(1ull << dev, std::memory_order_relaxed);
}

// Workgroups of a kernel with so many arrays in LDS that the chip holds at a time; asked for once.
template <auto Kernel>
unsigned resident(int block, int arrays, unsigned lds) {
  static std::atomic<unsigned> known[kParams + 16];
  unsigned n = known[arrays].load(std::memory_order_relaxed);
  if (n > 0) return n;
  int per_cu = 0;
  if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, Kernel, block, lds) != hipSuccess || per_cu < 1) {
    (void)hipGetLastError();
    per_cu = 1;
  }
  n = (unsigned)per_cu * kCUs;
  known[arrays].store(n, std::memory_order_relaxed);
  return n;
}

template <typename TX, typename TY>
void launch_forward(const FwdArgs& a, hipStream_t stream) {
  auto launch = [&](auto e, auto tpr, auto v) {
    constexpr int E = decltype(e)::value, TPR = decltype(tpr)::value, V = decltype(v)::value, B = block_of<TPR>();
    constexpr auto kernel = resnorm_fwd_kernel<TX, TY, E, TPR, V>;
    const ParamPlaces places(a.weight.p, a.bias.p, a.gate.p, a.n.post ? a.post_weight.p : nullptr,
                             a.n.post ? a.post_bias.p : nullptr);
    // the gate's row is its row slot's own
    const int arrays = places.n + (places.at[kG] >= 0 ? B / TPR - 1 : 0);
    const unsigned lds = arrays * Params<1, TPR, V, E / V, forward_home<TY, E, TPR>()>::kFloats * 4;
    allow_lds<kernel>(lds);
    // a last, half-empty round of workgroups would cost as much as a full one
    const unsigned grid =
        (unsigned)std::min<int64_t>((a.n.rows + B / TPR - 1) / (B / TPR), resident<kernel>(B, arrays, lds));
    kernel<<<grid, B, lds, stream>>>(a);
  };
  by_width(a.n.d, [&](auto e, auto tpr) {
    by_vec<TY>(a.n.d, [&](auto v) { launch(e, tpr, v); });
  });
}

template <typename TX, typename TY>
void launch_backward(const BwdArgs& a, hipStream_t stream) {
  const bool bias = a.want[kDb] || a.want[kDpb] || a.post_bias.p != nullptr;
  auto choose = [&](auto post, auto gated, auto biased, auto v) {
    constexpr bool POST = decltype(post)::value, GATED = decltype(gated)::value, BIAS = decltype(biased)::value;
    constexpr int V = decltype(v)::value;
    by_width(a.n.d, [&](auto e, auto tpr) {
      constexpr int E = decltype(e)::value, TPR = decltype(tpr)::value;
      constexpr auto kernel = resnorm_bwd_kernel<TX, TY, E, TPR, V, POST, GATED, BIAS>;
      const ParamPlaces places(a.weight.p, nullptr, a.gate.p, POST ? a.post_weight.p : nullptr,
                               POST && BIAS ? a.post_bias.p : nullptr);
      const unsigned lds = sums_in_lds<E, TPR, POST, GATED>()
                               ? 2 * TPR * E * 4
                               : places.n * Params<1, TPR, V, E / V, backward_home<E, TPR>()>::kFloats * 4;
      allow_lds<kernel>(lds);
      kernel<<<(unsigned)a.split.blocks, block_of<TPR>(), lds, stream>>>(a);
    });
  };
  // a form without biases for whole vectors only (16 bf16 values for each of 64 threads, gate and post norm: 209
  // registers, two waves to a SIMD; with biases 266 and one)
  auto by_bias = [&](auto post, auto gated) {
    by_vec<TY>(a.n.d, [&](auto v) {
      if constexpr (decltype(v)::value == vec_of<TY>())
        if (!bias) return choose(post, gated, std::false_type{}, v);
      choose(post, gated, std::true_type{}, v);
    });
  };
  auto by_gate = [&](auto post) {
    if (a.gate.p != nullptr) by_bias(post, std::true_type{});
    else by_bias(post, std::false_type{});
  };
  if (a.n.post) by_gate(std::true_type{});
  else by_gate(std::false_type{});
}

// one translation unit per pair of types (resnorm_*.hip)
#define GRACE_RESNORM_DECLARE(prefix, TX, TY)                                             \
  prefix template void launch_forward<TX, TY>(const FwdArgs&, hipStream_t);     \
  prefix template void launch_backward<TX, TY>(const BwdArgs&, hipStream_t);

}  // namespace resnorm
}  // namespace grace
