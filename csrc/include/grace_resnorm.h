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
// taken about the mean in a second sweep over registers.  64, 256, 512 or 1024 threads share a row,
// by its width; a workgroup walks over rows with the weights in registers, and rows that need a
// workgroup's barriers are loaded one ahead.  Statistics and sums are fp32; s is rounded to its own
// type only where it is stored, and h is made from the unrounded sum.  The backward reads the stored
// sum if that is fp32; a 16-bit sum is made again from x and y, because its rounding would show in
// the fp32 sums dw (2^-9 of every term against 2^-24).
// Column sums (dw, db, dgate, dpw, dpb): every workgroup adds up its rows in registers and leaves one
// partial row; a second launch adds the partial rows in a fixed order.
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

// values per load: 16 bytes of the narrower type
template <typename TX, typename TY>
constexpr int vec_of() { return sizeof(TY) == 2 ? 8 : 4; }

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

// Sums over the TPR threads of a row.  More than one wave: one barrier a sum, on two buffers in turn
// (a wave can be at most one barrier ahead of another).
template <int TPR>
struct RowSum {
  static constexpr int W = TPR / kWave;
  float* scratch;  // [2][2 W]
  int turn = 0;
  __device__ __forceinline__ void operator()(float& a, float& b) {
    a = dpp_sum(a);
    b = dpp_sum(b);
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

template <int TPR, int V, int J>
struct Row {
  int t, d;
  int left[J];  // values of vector j inside the width (at most 0: none)
  __device__ __forceinline__ Row(int t, int d) : t(t), d(d) {
#pragma unroll
    for (int j = 0; j < J; ++j) left[j] = min(d - (j * TPR + t) * V, V);
  }
  __device__ __forceinline__ int col(int j) const { return (j * TPR + t) * V; }

  // as stored; zero outside the width, or everywhere without a pointer
  template <typename T>
  __device__ __forceinline__ void load(const void* p, int64_t at, Raw<T, V, J>& r) const {
#pragma unroll
    for (int j = 0; j < J; ++j) {
#pragma unroll
      for (int i = 0; i < Bits<T, V>::W; ++i) r.v[j].w[i] = 0;
      if (p != nullptr && left[j] > 0) load_bits(static_cast<const T*>(p) + at + col(j), r.v[j], left[j]);
    }
  }
  template <typename TY>
  __device__ __forceinline__ void param(const NormParam& p, int64_t at, float none, float (&o)[J][V]) const {
#pragma unroll
    for (int j = 0; j < J; ++j) {
#pragma unroll
      for (int i = 0; i < V; ++i) o[j][i] = none;
      if (p.p == nullptr || left[j] <= 0) continue;
      if (p.f32) load_vec(static_cast<const float*>(p.p) + at + col(j), o[j], left[j]);
      else load_vec(static_cast<const TY*>(p.p) + at + col(j), o[j], left[j]);
    }
  }
  template <typename T>
  __device__ __forceinline__ void store(void* p, int64_t at, const float (&v)[J][V], bool once) const {
    if (once) {
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (left[j] > 0) store_vec<true>(static_cast<T*>(p) + at + col(j), v[j], left[j]);
    } else {
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (left[j] > 0) store_vec(static_cast<T*>(p) + at + col(j), v[j], left[j]);
    }
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
      if (left[j] >= V) {
#pragma unroll
        for (int i = 0; i < V; ++i) a = fmaf(v[j][i] - mean, v[j][i] - mean, a);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (i < left[j]) a = fmaf(v[j][i] - mean, v[j][i] - mean, a);
      }
    }
    sum(a);
    rstd = 1.f / sqrtf(a / (float)d + eps);
  }
  // zero outside the width
  __device__ __forceinline__ void trim(float (&v)[J][V]) const {
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (left[j] < V) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[j][i] = i < left[j] ? v[j][i] : 0.f;
      }
  }
};

// The weights (and in the backward the gate) of a workgroup's rows, each thread's own values.  Rows that
// take a workgroup keep them in LDS, where they cost no registers: the registers decide how many such
// rows a CU has in flight.  Only the thread that wrote a value reads it, so there are no barriers.
// 16384 columns would take 64 KB an array, so rows of 16 values a thread keep them in registers.
template <int K, int TPR, int V, int J, bool LDS>
struct Params {
  static constexpr bool kLds = LDS;
  static constexpr int kFloats = kLds ? TPR * V * J : 0;  // of LDS, for each array
  float r[kLds ? 1 : K][J][V];
  float4* lds;
  __device__ __forceinline__ explicit Params(float* p) : lds(reinterpret_cast<float4*>(p) + threadIdx.x) {}
  // k: the array (a constant), at: its place in LDS
  __device__ __forceinline__ void set(int k, int at, const float (&v)[J][V]) {
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        if constexpr (kLds) {
          lds[((at * J + j) * (V / 4) + i / 4) * TPR] = make_float4(v[j][i], v[j][i + 1], v[j][i + 2], v[j][i + 3]);
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q) r[k][j][i + q] = v[j][i + q];
        }
      }
  }
  __device__ __forceinline__ void get(int k, int at, float (&v)[J][V]) const {
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        if constexpr (kLds) {
          const float4 q = lds[((at * J + j) * (V / 4) + i / 4) * TPR];
          v[j][i] = q.x;
          v[j][i + 1] = q.y;
          v[j][i + 2] = q.z;
          v[j][i + 3] = q.w;
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q) v[j][i + q] = r[k][j][i + q];
        }
      }
  }
};

// the workgroup's slot of rows, known to be the same in a wave
template <int TPR>
__device__ __forceinline__ int row_slot() {
  return block_of<TPR>() == TPR ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / TPR);
}

enum { kW, kB, kPw, kPb, kG, kParams };

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

template <int E, int TPR>
constexpr bool lds_forward() { return TPR > kWave && TPR < 1024; }  // at most five arrays: 80 KB
template <int E, int TPR>
constexpr bool lds_backward() { return TPR > kWave && E == 8; }  // at most four: 128 KB

#define GRACE_EACH(body)          \
  _Pragma("unroll") for (int j = 0; j < J; ++j) \
  _Pragma("unroll") for (int i = 0; i < V; ++i) { body; }

// ---------------------------------------------------------------- forward
template <typename TX, typename TY, int E, int TPR>
__global__ __launch_bounds__(block_of<TPR>()) void resnorm_fwd_kernel(FwdArgs g) {
  constexpr int V = vec_of<TX, TY>(), J = E / V, kSlots = block_of<TPR>() / TPR;
  __shared__ float scratch[TPR > kWave ? 4 * TPR / kWave : 1];
  RowSum<TPR> sum{scratch};
  const NormShape& n = g.n;
  const Row<TPR, V, J> row(threadIdx.x % TPR, n.d);
  const uint32_t rows = (uint32_t)n.rows, step = gridDim.x * kSlots, gate_rows = (uint32_t)n.gate_rows;
  uint32_t r = blockIdx.x * kSlots + row_slot<TPR>();
  if (r >= rows) return;
  // Rows of one wave: many are in flight anyway, and few registers (78 for 160) let all 4096 rows of a
  // small batch run at once; their weights come from the caches.
  constexpr bool AHEAD = TPR > kWave;
  Raw<TY, V, J> ry;
  Raw<TX, V, J> rx;
  auto fetch = [&](uint32_t q) {
    row.load(g.y, (int64_t)q * n.d, ry);
    row.load(g.x, (int64_t)q * n.d, rx);
  };
  fetch(r);
  extern __shared__ __align__(16) float dyn[];
  Params<kParams, TPR, V, J, lds_forward<E, TPR>()> params(dyn);
  const ParamPlaces at_lds(g.weight.p, g.bias.p, g.gate.p, n.post ? g.post_weight.p : nullptr,
                           n.post ? g.post_bias.p : nullptr);
  {
    float v[J][V];
    auto put = [&](int k, const NormParam& p, float none) {
      if (!AHEAD || at_lds.at[k] < 0) return;
      row.template param<TY>(p, 0, none, v);
      params.set(k, at_lds.at[k], v);
    };
    put(kW, g.weight, 1.f);
    put(kB, g.bias, 0.f);
    put(kPw, g.post_weight, 1.f);
    put(kPb, g.post_bias, 0.f);
  }
  auto take = [&](int k, const NormParam& from, float(&v)[J][V]) {
    if constexpr (AHEAD) params.get(k, at_lds.at[k], v);
    else row.template param<TY>(from, 0, 0.f, v);
  };
  uint32_t gate_now = ~0u;
  for (;;) {
    const int64_t at = (int64_t)r * n.d;
    float u[J][V], x[J][V], p[J][V], gate[J][V], mean, rstd;
    // a gate that stays is not loaded again: a load here would make the row wait for the last one's stores
    if (g.gate.p != nullptr && (!AHEAD || r / gate_rows != gate_now)) {
      gate_now = r / gate_rows;
      row.template param<TY>(g.gate, (int64_t)gate_now * n.d, 1.f, gate);
      if (AHEAD) params.set(kG, at_lds.at[kG], gate);
    }
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
      if (AHEAD) params.get(kG, at_lds.at[kG], gate);
      GRACE_EACH(u[j][i] *= gate[j][i])
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
__device__ __forceinline__ void store_param(void* p, bool f32, int64_t at, const float (&v)[V], int n) {
  if (f32) store_vec(static_cast<float*>(p) + at, v, n);
  else store_vec(static_cast<TY*>(p) + at, v, n);
}

// Sums acc over the workgroup's row slots and hands each vector to out(column, values, count); acc
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
      out(c, v, min(row.d - c, V));
    }
  } else {
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (row.left[j] > 0) out(row.col(j), acc[j], row.left[j]);
  }
}

// BIAS: one of the two biases is there
template <typename TX, typename TY, int E, int TPR, bool POST, bool GATED, bool BIAS>
__global__ __launch_bounds__(block_of<TPR>(), TPR == 512 ? 4 : 1) void resnorm_bwd_kernel(BwdArgs g) {
  constexpr int V = vec_of<TX, TY>(), J = E / V, kSlots = block_of<TPR>() / TPR;
  constexpr bool AHEAD = TPR > kWave;  // the next row's loads are issued before this row's sums
  __shared__ float scratch[TPR > kWave ? 4 * TPR / kWave : 1];
  __shared__ float red[kSlots > 1 ? kSlots * TPR * E : 1];
  RowSum<TPR> sum{scratch};
  const NormShape& n = g.n;
  const Row<TPR, V, J> row(threadIdx.x % TPR, n.d);
  float dw[J][V], db[J][V], dg[J][V], dpw[J][V], dpb[J][V];
  GRACE_EACH(dw[j][i] = db[j][i] = dg[j][i] = dpw[j][i] = dpb[j][i] = 0.f)
  extern __shared__ __align__(16) float dyn[];
  Params<2 + 2 * POST, TPR, V, J, lds_backward<E, TPR>()> params(dyn);
  constexpr int W = 0, G = 1, PW = 2, PB = 3;  // the places in registers
  const ParamPlaces at_lds(g.weight.p, nullptr, g.gate.p, POST ? g.post_weight.p : nullptr,
                           POST && BIAS ? g.post_bias.p : nullptr);
  {
    float v[J][V];
    if (g.weight.p != nullptr) {
      row.template param<TY>(g.weight, 0, 1.f, v);
      params.set(W, at_lds.at[kW], v);
    }
    if constexpr (POST) {
      if (g.post_weight.p != nullptr) {
        row.template param<TY>(g.post_weight, 0, 1.f, v);
        params.set(PW, at_lds.at[kPw], v);
      }
      if constexpr (BIAS) {
        if (g.post_bias.p != nullptr) {
          row.template param<TY>(g.post_bias, 0, 0.f, v);
          params.set(PB, at_lds.at[kPb], v);
        }
      }
    }
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
          float v[J][V];
          row.template param<TY>(g.gate, (int64_t)gate_now * n.d, 1.f, v);
          params.set(G, at_lds.at[kG], v);
        }
      }
      float S[J][V], hat[J][V], phat[J][V], ds[J][V], p[J][V];
      // u of the forward, without its gate, from phat
      auto made_u = [&](float(&u)[J][V]) {
        GRACE_EACH(u[j][i] = phat[j][i])
        if constexpr (POST) {
          if (g.post_weight.p != nullptr) {
            params.get(PW, at_lds.at[kPw], p);
            GRACE_EACH(u[j][i] *= p[j][i])
          }
          if constexpr (BIAS) {
            if (g.post_bias.p != nullptr) {
              params.get(PB, at_lds.at[kPb], p);
              GRACE_EACH(u[j][i] += p[j][i])
            }
          }
        }
      };
      float c1 = 0.f, c2 = 0.f;
      GRACE_EACH(phat[j][i] = bits_at(ry.v[j], i); hat[j][i] = bits_at(rs.v[j], i); S[j][i] = bits_at(rdh.v[j], i);
                 ds[j][i] = bits_at(rds.v[j], i))
      if (AHEAD && r + kSlots < r_end) fetch(r + kSlots);
      if constexpr (POST) GRACE_EACH(phat[j][i] = (phat[j][i] - pmean) * prstd)
      if (again) {
        float u[J][V];
        made_u(u);
        if constexpr (GATED) {
          params.get(G, at_lds.at[kG], p);
          GRACE_EACH(u[j][i] *= p[j][i])
        }
        GRACE_EACH(hat[j][i] = fmaf(n.alpha, hat[j][i], u[j][i]))
      }
      GRACE_EACH(hat[j][i] = (hat[j][i] - mean) * rstd; dw[j][i] = fmaf(S[j][i], hat[j][i], dw[j][i]))
      if constexpr (BIAS) GRACE_EACH(db[j][i] += S[j][i])
      if (g.weight.p != nullptr) {
        params.get(W, at_lds.at[kW], p);
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
        params.get(G, at_lds.at[kG], p);
        GRACE_EACH(u[j][i] *= S[j][i]; dg[j][i] = g.dgate_mode == kGateRows ? u[j][i] : dg[j][i] + u[j][i];
                   S[j][i] *= p[j][i])
        if (g.dgate_mode == kGateRows) {
#pragma unroll
          for (int j = 0; j < J; ++j)
            if (row.left[j] > 0) store_param<TY>(g.dgate, g.dgate_f32, at + row.col(j), dg[j], row.left[j]);
        }
      }
      if constexpr (POST) {
        c1 = c2 = 0.f;
        GRACE_EACH(dpw[j][i] = fmaf(S[j][i], phat[j][i], dpw[j][i]))
        if constexpr (BIAS) GRACE_EACH(dpb[j][i] += S[j][i])
        if (g.post_weight.p != nullptr) {
          params.get(PW, at_lds.at[kPw], p);
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
        over_slots(dg, row, red, [&](int c, const float(&v)[V], int k) {
          store_param<TY>(g.dgate, g.dgate_f32, (int64_t)grp * n.d + c, v, k);
        });
        GRACE_EACH(dg[j][i] = 0.f)
      }
    }
  }
  const int64_t plane = g.split.blocks * n.d;
  auto leave = [&](int which, const float(&acc)[J][V]) {
    if (!g.want[which]) return;
    float* to = g.part + which * plane + blockIdx.x * (int64_t)n.d;
    over_slots(acc, row, red, [&](int c, const float(&v)[V], int k) { store_vec(to + c, v, k); });
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
// Values per thread and threads per row, by the row's width.
template <typename F>
void by_width(int d, F&& f) {
  using std::integral_constant;
  if (d <= 64 * 8) f(integral_constant<int, 8>{}, integral_constant<int, 64>{});
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

// Workgroups of a kernel that the chip holds at a time.
template <auto Kernel>
unsigned resident(int block, unsigned lds) {
  static std::atomic<uint64_t> last{0};  // lds + 1 in the upper half, the answer in the lower
  const uint64_t key = (uint64_t)lds + 1, known = last.load(std::memory_order_relaxed);
  if (known >> 32 == key) return (unsigned)known;
  int per_cu = 0;
  if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, Kernel, block, lds) != hipSuccess || per_cu < 1) {
    (void)hipGetLastError();
    per_cu = 1;
  }
  const unsigned n = (unsigned)per_cu * kCUs;
  last.store(key << 32 | n, std::memory_order_relaxed);
  return n;
}

template <typename TX, typename TY>
void launch_forward(const FwdArgs& a, hipStream_t stream) {
  by_width(a.n.d, [&](auto e, auto tpr) {
    constexpr int E = decltype(e)::value, TPR = decltype(tpr)::value, B = block_of<TPR>();
    const ParamPlaces places(a.weight.p, a.bias.p, a.gate.p, a.n.post ? a.post_weight.p : nullptr,
                             a.n.post ? a.post_bias.p : nullptr);
    constexpr int V = vec_of<TX, TY>();
    const unsigned lds = places.n * Params<1, TPR, V, E / V, lds_forward<E, TPR>()>::kFloats * 4;
    allow_lds<resnorm_fwd_kernel<TX, TY, E, TPR>>(lds);
    // a last, half-empty round of workgroups would cost as much as a full one
    const unsigned grid = (unsigned)std::min<int64_t>((a.n.rows + B / TPR - 1) / (B / TPR),
                                                      resident<resnorm_fwd_kernel<TX, TY, E, TPR>>(B, lds));
    resnorm_fwd_kernel<TX, TY, E, TPR><<<grid, B, lds, stream>>>(a);
  });
}

template <typename TX, typename TY>
void launch_backward(const BwdArgs& a, hipStream_t stream) {
  const bool bias = a.want[kDb] || a.want[kDpb] || a.post_bias.p != nullptr;
  auto choose = [&](auto post, auto gated, auto biased) {
    constexpr bool POST = decltype(post)::value, GATED = decltype(gated)::value, BIAS = decltype(biased)::value;
    by_width(a.n.d, [&](auto e, auto tpr) {
      constexpr int E = decltype(e)::value, TPR = decltype(tpr)::value, V = vec_of<TX, TY>();
      const ParamPlaces places(a.weight.p, nullptr, a.gate.p, POST ? a.post_weight.p : nullptr,
                               POST && BIAS ? a.post_bias.p : nullptr);
      const unsigned lds = places.n * Params<1, TPR, V, E / V, lds_backward<E, TPR>()>::kFloats * 4;
      allow_lds<resnorm_bwd_kernel<TX, TY, E, TPR, POST, GATED, BIAS>>(lds);
      resnorm_bwd_kernel<TX, TY, E, TPR, POST, GATED, BIAS>
          <<<(unsigned)a.split.blocks, block_of<TPR>(), lds, stream>>>(a);
    });
  };
  auto by_bias = [&](auto post, auto gated) {
    if (bias) choose(post, gated, std::true_type{});
    else choose(post, gated, std::false_type{});
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
