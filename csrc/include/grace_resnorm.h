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
#include <type_traits>

#include "grace_common.h"
#include "grace_lm.h"

namespace grace {
namespace resnorm {

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
  Pack<T, V> v[J];
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
      for (int i = 0; i < V; ++i) r.v[j].v[i] = (T)0.f;
      const T* q = static_cast<const T*>(p) + at + col(j);
      if (p != nullptr && left[j] >= V) r.v[j] = *reinterpret_cast<const Pack<T, V>*>(q);
      else if (p != nullptr && left[j] > 0) {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (i < left[j]) r.v[j].v[i] = q[i];
      }
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
  __device__ __forceinline__ void store(void* p, int64_t at, const float (&v)[J][V]) const {
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (left[j] > 0) store_vec(static_cast<T*>(p) + at + col(j), v[j], left[j]);
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

// the workgroup's slot of rows, known to be the same in a wave
template <int TPR>
__device__ __forceinline__ int row_slot() {
  return block_of<TPR>() == TPR ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / TPR);
}

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
  Raw<TY, V, J> ry;
  Raw<TX, V, J> rx;
  row.load(g.y, (int64_t)r * n.d, ry);
  row.load(g.x, (int64_t)r * n.d, rx);
  float w[J][V], b[J][V], pw[J][V], pb[J][V], gate[J][V];
  row.template param<TY>(g.weight, 0, 1.f, w);
  row.template param<TY>(g.bias, 0, 0.f, b);
  if (n.post) {
    row.template param<TY>(g.post_weight, 0, 1.f, pw);
    row.template param<TY>(g.post_bias, 0, 0.f, pb);
  }
  uint32_t gate_now = ~0u;
  for (;;) {
    const int64_t at = (int64_t)r * n.d;
    if (g.gate.p != nullptr && r / gate_rows != gate_now) {
      gate_now = r / gate_rows;
      row.template param<TY>(g.gate, (int64_t)gate_now * n.d, 1.f, gate);
    }
    float u[J][V], x[J][V], mean, rstd;
    GRACE_EACH(u[j][i] = (float)ry.v[j].v[i]; x[j][i] = (float)rx.v[j].v[i])
    const bool more = rows - r > step;
    if (more) {
      row.load(g.y, at + (int64_t)step * n.d, ry);
      row.load(g.x, at + (int64_t)step * n.d, rx);
    }
    if (n.post) {
      row.stats(u, n.rms, n.eps, sum, mean, rstd);
      if (g.stats != nullptr && row.t == 0) {
        g.stats[2 * n.rows + r] = mean;
        g.stats[3 * n.rows + r] = rstd;
      }
      GRACE_EACH(u[j][i] = (u[j][i] - mean) * rstd * pw[j][i] + pb[j][i])
    }
    if (g.gate.p != nullptr) GRACE_EACH(u[j][i] *= gate[j][i])
    if (g.x != nullptr) GRACE_EACH(u[j][i] = fmaf(n.alpha, x[j][i], u[j][i]))
    row.trim(u);
    if (g.s != nullptr) row.template store<TX>(g.s, at, u);
    row.stats(u, n.rms, n.eps, sum, mean, rstd);
    if (g.stats != nullptr && row.t == 0) {
      g.stats[r] = mean;
      g.stats[n.rows + r] = rstd;
    }
    GRACE_EACH(u[j][i] = (u[j][i] - mean) * rstd * w[j][i] + b[j][i])
    row.template store<TY>(g.h, at, u);
    if (!more) return;
    r += step;
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

template <typename TX, typename TY, int E, int TPR, bool POST, bool GATED>
__global__ __launch_bounds__(block_of<TPR>()) void resnorm_bwd_kernel(BwdArgs g) {
  constexpr int V = vec_of<TX, TY>(), J = E / V, kSlots = block_of<TPR>() / TPR;
  constexpr bool AHEAD = TPR > kWave;  // the next row's loads are issued before this row's sums
  __shared__ float scratch[TPR > kWave ? 4 * TPR / kWave : 1];
  __shared__ float red[kSlots > 1 ? kSlots * TPR * E : 1];
  RowSum<TPR> sum{scratch};
  const NormShape& n = g.n;
  const Row<TPR, V, J> row(threadIdx.x % TPR, n.d);
  float dw[J][V], db[J][V], dg[J][V], dpw[J][V], dpb[J][V], w[J][V], pw[J][V], pb[J][V], gate[J][V];
  GRACE_EACH(dw[j][i] = db[j][i] = dg[j][i] = dpw[j][i] = dpb[j][i] = 0.f)
  row.template param<TY>(g.weight, 0, 1.f, w);
  if constexpr (POST) {
    row.template param<TY>(g.post_weight, 0, 1.f, pw);
    row.template param<TY>(g.post_bias, 0, 0.f, pb);
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
          row.template param<TY>(g.gate, (int64_t)gate_now * n.d, 1.f, gate);
        }
      }
      float S[J][V], hat[J][V], phat[J][V], ds[J][V];
      float c1 = 0.f, c2 = 0.f;
      GRACE_EACH(phat[j][i] = (float)ry.v[j].v[i]; hat[j][i] = (float)rs.v[j].v[i]; S[j][i] = (float)rdh.v[j].v[i];
                 ds[j][i] = (float)rds.v[j].v[i])
      if (AHEAD && r + kSlots < r_end) fetch(r + kSlots);
      if constexpr (POST) GRACE_EACH(phat[j][i] = (phat[j][i] - pmean) * prstd)
      if (again) {
        GRACE_EACH(float u = phat[j][i]; if constexpr (POST) u = u * pw[j][i] + pb[j][i];
                   if constexpr (GATED) u *= gate[j][i]; hat[j][i] = fmaf(n.alpha, hat[j][i], u))
      }
      GRACE_EACH(hat[j][i] = (hat[j][i] - mean) * rstd; dw[j][i] = fmaf(S[j][i], hat[j][i], dw[j][i]);
                 db[j][i] += S[j][i]; S[j][i] *= w[j][i]; c1 += S[j][i]; c2 = fmaf(S[j][i], hat[j][i], c2))
      sum(c1, c2);
      c1 = n.rms ? 0.f : c1 * inv_d;
      c2 *= inv_d;
      GRACE_EACH(S[j][i] = rstd * (S[j][i] - c1 - hat[j][i] * c2))
      if (g.dh == nullptr) GRACE_EACH(S[j][i] = 0.f)
      GRACE_EACH(S[j][i] += ds[j][i])
      row.trim(S);
      if (g.dx != nullptr) {
        GRACE_EACH(ds[j][i] = n.alpha * S[j][i])
        row.template store<TX>(g.dx, at, ds);
      }
      if constexpr (GATED) {
        GRACE_EACH(float u = phat[j][i]; if constexpr (POST) u = u * pw[j][i] + pb[j][i]; u *= S[j][i];
                   dg[j][i] = g.dgate_mode == kGateRows ? u : dg[j][i] + u; S[j][i] *= gate[j][i])
        if (g.dgate_mode == kGateRows) {
#pragma unroll
          for (int j = 0; j < J; ++j)
            if (row.left[j] > 0) store_param<TY>(g.dgate, g.dgate_f32, at + row.col(j), dg[j], row.left[j]);
        }
      }
      if constexpr (POST) {
        c1 = c2 = 0.f;
        GRACE_EACH(dpw[j][i] = fmaf(S[j][i], phat[j][i], dpw[j][i]); dpb[j][i] += S[j][i]; S[j][i] *= pw[j][i];
                   c1 += S[j][i]; c2 = fmaf(S[j][i], phat[j][i], c2))
        sum(c1, c2);
        c1 = n.rms ? 0.f : c1 * inv_d;
        c2 *= inv_d;
        GRACE_EACH(S[j][i] = prstd * (S[j][i] - c1 - phat[j][i] * c2))
      }
      row.template store<TY>(g.dy, at, S);
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
  leave(kDb, db);
  if constexpr (GATED) leave(kDg, dg);
  if constexpr (POST) {
    leave(kDpw, dpw);
    leave(kDpb, dpb);
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

template <typename TX, typename TY>
void launch_forward(const FwdArgs& a, unsigned max_blocks, hipStream_t stream) {
  by_width(a.n.d, [&](auto e, auto tpr) {
    constexpr int E = decltype(e)::value, TPR = decltype(tpr)::value, B = block_of<TPR>();
    const unsigned grid = (unsigned)std::min<int64_t>((a.n.rows + B / TPR - 1) / (B / TPR), max_blocks);
    resnorm_fwd_kernel<TX, TY, E, TPR><<<grid, B, 0, stream>>>(a);
  });
}

template <typename TX, typename TY>
void launch_backward(const BwdArgs& a, hipStream_t stream) {
  const bool post = a.n.post, gated = a.gate.p != nullptr;
  by_width(a.n.d, [&](auto e, auto tpr) {
    constexpr int E = decltype(e)::value, TPR = decltype(tpr)::value, B = block_of<TPR>();
    const unsigned grid = (unsigned)a.split.blocks;
    if (post && gated) resnorm_bwd_kernel<TX, TY, E, TPR, true, true><<<grid, B, 0, stream>>>(a);
    else if (post) resnorm_bwd_kernel<TX, TY, E, TPR, true, false><<<grid, B, 0, stream>>>(a);
    else if (gated) resnorm_bwd_kernel<TX, TY, E, TPR, false, true><<<grid, B, 0, stream>>>(a);
    else resnorm_bwd_kernel<TX, TY, E, TPR, false, false><<<grid, B, 0, stream>>>(a);
  });
}

// one translation unit per block type (resnorm_f32.hip, resnorm_bf16.hip, resnorm_f16.hip)
#define GRACE_RESNORM_DECLARE(prefix, TX, TY)                                             \
  prefix template void launch_forward<TX, TY>(const FwdArgs&, unsigned, hipStream_t);     \
  prefix template void launch_backward<TX, TY>(const BwdArgs&, hipStream_t);

}  // namespace resnorm
}  // namespace grace
