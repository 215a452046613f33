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
// taken about the mean in a second sweep over registers.  64, 256 or 1024 threads share a row, by its
// width.  Statistics and sums are fp32; s is rounded to its own type only where it is stored, h is
// made from the unrounded sum.  The backward reads the stored s: in 16 bits s^ then carries that one
// rounding, which is below the rounding of dx.
// Column sums (dw, db, dgate, dpw, dpb): every workgroup adds up its rows in registers and leaves one
// partial row; a second launch adds the partial rows in a fixed order.
#pragma once

#include <algorithm>
#include <type_traits>

#include "grace_common.h"
#include "grace_lm.h"

namespace grace {
namespace resnorm {

constexpr int kVec = 4;          // values per load

template <int TPR>
constexpr int block_of() { return TPR < 256 ? 256 : TPR; }

struct FwdArgs {
  NormShape n;
  const void *x, *y;
  NormParam gate, weight, bias, post_weight, post_bias;
  void *h, *s;
  float* stats;
};

template <typename TY, int V>
__device__ __forceinline__ void load_param(const NormParam& p, int64_t at, float (&o)[V], int n) {
  if (p.f32) load_vec(static_cast<const float*>(p.p) + at, o, n);
  else load_vec(static_cast<const TY*>(p.p) + at, o, n);
}

// values of vector j that lie inside the width (at most 0: none)
template <int TPR, int J>
__device__ __forceinline__ void row_left(int t, int d, int (&left)[J]) {
#pragma unroll
  for (int j = 0; j < J; ++j) left[j] = min(d - (j * TPR + t) * kVec, kVec);
}

// Sums of a and b over the TPR threads of a row; scratch: 2 * TPR / 64 floats, for TPR > 64.
template <int TPR>
__device__ __forceinline__ void row_sum2(float& a, float& b, float* scratch) {
  a = wave_sum(a);
  b = wave_sum(b);
  if constexpr (TPR > kWave) {
    constexpr int W = TPR / kWave;
    __syncthreads();  // the last sums have been read
    if (lane_id() == 0) {
      scratch[2 * wave_id()] = a;
      scratch[2 * wave_id() + 1] = b;
    }
    __syncthreads();
    a = scratch[0];
    b = scratch[1];
#pragma unroll
    for (int i = 1; i < W; ++i) {
      a += scratch[2 * i];
      b += scratch[2 * i + 1];
    }
  }
}

// mean and 1 / deviation of the row v (zero outside the width)
template <int TPR, int V, int J>
__device__ __forceinline__ void row_stats(const float (&v)[J][V], const int (&left)[J], int d, bool rms, float eps,
                                          float* scratch, float& mean, float& rstd) {
  float a = 0.f, b = 0.f;
  mean = 0.f;
  if (!rms) {
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) a += v[j][i];
    row_sum2<TPR>(a, b, scratch);
    mean = a / (float)d;
  }
  a = b = 0.f;
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
  row_sum2<TPR>(a, b, scratch);
  rstd = 1.f / sqrtf(a / (float)d + eps);
}

template <typename TX, typename TY, int E, int TPR>
__global__ __launch_bounds__(block_of<TPR>()) void resnorm_fwd_kernel(FwdArgs g) {
  constexpr int V = kVec, J = E / V, kSlots = block_of<TPR>() / TPR;
  __shared__ float scratch[2 * (TPR > kWave ? TPR / kWave : 1)];
  const NormShape& n = g.n;
  const int t = threadIdx.x % TPR, d = n.d;
  const int64_t slots = (int64_t)gridDim.x * kSlots;
  int left[J];
  row_left<TPR>(t, d, left);
  for (int64_t r = (int64_t)blockIdx.x * kSlots + threadIdx.x / TPR; r < n.rows; r += slots) {
    const int64_t at = r * d;
    float u[J][V], mean, rstd;
#pragma unroll
    for (int j = 0; j < J; ++j) {
#pragma unroll
      for (int i = 0; i < V; ++i) u[j][i] = 0.f;
      if (left[j] > 0) load_vec(static_cast<const TY*>(g.y) + at + (j * TPR + t) * V, u[j], left[j]);
    }
    if (n.post) {
      row_stats<TPR>(u, left, d, n.rms, n.eps, scratch, mean, rstd);
      if (g.stats && t == 0) {
        g.stats[2 * n.rows + r] = mean;
        g.stats[3 * n.rows + r] = rstd;
      }
#pragma unroll
      for (int j = 0; j < J; ++j) {
        if (left[j] <= 0) continue;
        const int c = (j * TPR + t) * V;
        float p[V];
#pragma unroll
        for (int i = 0; i < V; ++i) u[j][i] = (u[j][i] - mean) * rstd;
        if (g.post_weight.p) {
          load_param<TY>(g.post_weight, c, p, left[j]);
#pragma unroll
          for (int i = 0; i < V; ++i) u[j][i] *= p[i];
        }
        if (g.post_bias.p) {
          load_param<TY>(g.post_bias, c, p, left[j]);
#pragma unroll
          for (int i = 0; i < V; ++i) u[j][i] += p[i];
        }
      }
    }
    const int64_t gate_at = g.gate.p ? (r / n.gate_rows) * d : 0;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if (left[j] <= 0) continue;
      const int c = (j * TPR + t) * V;
      float p[V];
      if (g.gate.p) {
        load_param<TY>(g.gate, gate_at + c, p, left[j]);
#pragma unroll
        for (int i = 0; i < V; ++i) u[j][i] *= p[i];
      }
      if (g.x) {
        load_vec(static_cast<const TX*>(g.x) + at + c, p, left[j]);
#pragma unroll
        for (int i = 0; i < V; ++i) u[j][i] = fmaf(n.alpha, p[i], u[j][i]);
      }
      if (g.s) store_vec(static_cast<TX*>(g.s) + at + c, u[j], left[j]);
    }
    row_stats<TPR>(u, left, d, n.rms, n.eps, scratch, mean, rstd);
    if (g.stats && t == 0) {
      g.stats[r] = mean;
      g.stats[n.rows + r] = rstd;
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if (left[j] <= 0) continue;
      const int c = (j * TPR + t) * V;
      float p[V];
#pragma unroll
      for (int i = 0; i < V; ++i) u[j][i] = (u[j][i] - mean) * rstd;
      if (g.weight.p) {
        load_param<TY>(g.weight, c, p, left[j]);
#pragma unroll
        for (int i = 0; i < V; ++i) u[j][i] *= p[i];
      }
      if (g.bias.p) {
        load_param<TY>(g.bias, c, p, left[j]);
#pragma unroll
        for (int i = 0; i < V; ++i) u[j][i] += p[i];
      }
      store_vec(static_cast<TY*>(g.h) + at + c, u[j], left[j]);
    }
  }
}

// ---------------------------------------------------------------- backward
// How the workgroups share the rows.  A gate's sums end with its group of rows: long groups are cut
// into parts (one partial row of dgate per part), of short groups a workgroup takes whole ones and
// writes their dgate itself.
struct Split {
  int64_t groups;      // groups of rows (1 without a gate whose sums are wanted)
  int64_t group_rows;
  int64_t parts;       // workgroups per group, or 1
  int64_t per_block;   // groups per workgroup, or 1
  int64_t blocks;
};

enum { kDw, kDb, kDg, kDpw, kDpb, kSums };

struct BwdArgs {
  NormShape n;
  Split split;
  const void *s, *y, *dh, *ds;
  const float* stats;
  NormParam gate, weight, post_weight, post_bias;
  void *dx, *dy, *dgate;
  bool dgate_f32;
  bool want[kSums];
  int dgate_mode;  // 0: none, 1: partial rows, 2: written per group, 3: a gate of the rows' own shape
  float* part;     // [sums][blocks][d]
};

template <typename TY, int V>
__device__ __forceinline__ void store_param(void* p, bool f32, int64_t at, const float (&v)[V], int n) {
  if (f32) store_vec(static_cast<float*>(p) + at, v, n);
  else store_vec(static_cast<TY*>(p) + at, v, n);
}

// Sums acc over the workgroup's row slots and hands each vector to out(column, values, count); acc
// is left as it is.  red: [slots][TPR * E] floats for more than one slot.
template <int TPR, int V, int J, typename F>
__device__ __forceinline__ void over_slots(const float (&acc)[J][V], const int (&left)[J], int d, float* red, F&& out) {
  const int t = threadIdx.x % TPR;
  if constexpr (block_of<TPR>() > TPR) {
    constexpr int kSlots = block_of<TPR>() / TPR, kRow = TPR * V * J;
    __syncthreads();  // red has been read
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) red[(threadIdx.x / TPR) * kRow + (j * TPR + t) * V + i] = acc[j][i];
    __syncthreads();
    for (int c = threadIdx.x * V; c < d; c += block_of<TPR>() * V) {
      float v[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        v[i] = red[c + i];
#pragma unroll
        for (int k = 1; k < kSlots; ++k) v[i] += red[k * kRow + c + i];
      }
      out(c, v, min(d - c, V));
    }
  } else {
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (left[j] > 0) out((j * TPR + t) * V, acc[j], left[j]);
  }
}

// FULL: with gate or post norm
template <typename TX, typename TY, int E, int TPR, bool FULL>
__global__ __launch_bounds__(block_of<TPR>()) void resnorm_bwd_kernel(BwdArgs g) {
  constexpr int V = kVec, J = E / V, kSlots = block_of<TPR>() / TPR;
  __shared__ float scratch[2 * (TPR > kWave ? TPR / kWave : 1)];
  __shared__ float red[kSlots > 1 ? kSlots * TPR * E : 1];
  const NormShape& n = g.n;
  const int t = threadIdx.x % TPR, slot = threadIdx.x / TPR, d = n.d;
  int left[J];
  row_left<TPR>(t, d, left);
  float dw[J][V], db[J][V], dg[FULL ? J : 1][V], dpw[FULL ? J : 1][V], dpb[FULL ? J : 1][V];
#pragma unroll
  for (int j = 0; j < J; ++j) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      dw[j][i] = db[j][i] = 0.f;
      if constexpr (FULL) dg[j][i] = dpw[j][i] = dpb[j][i] = 0.f;
    }
  }
  const float inv_d = 1.f / (float)d;
  const int64_t part = blockIdx.x % g.split.parts;
  const int64_t g0 = (blockIdx.x / g.split.parts) * g.split.per_block;
  const int64_t g1 = min(g0 + g.split.per_block, g.split.groups);
  const int64_t chunk = (g.split.group_rows + g.split.parts - 1) / g.split.parts;
  for (int64_t grp = g0; grp < g1; ++grp) {
    const int64_t r_end = grp * g.split.group_rows + min((part + 1) * chunk, g.split.group_rows);
    for (int64_t r = grp * g.split.group_rows + part * chunk + slot; r < r_end; r += kSlots) {
      const int64_t at = r * d;
      const float mean = g.stats[r], rstd = g.stats[n.rows + r];
      float S[J][V], hat[J][V];
      float c1 = 0.f, c2 = 0.f;
#pragma unroll
      for (int j = 0; j < J; ++j) {
#pragma unroll
        for (int i = 0; i < V; ++i) S[j][i] = hat[j][i] = 0.f;
        if (left[j] <= 0 || !g.dh) continue;
        const int c = (j * TPR + t) * V;
        float p[V];
        load_vec(static_cast<const TX*>(g.s) + at + c, hat[j], left[j]);
        load_vec(static_cast<const TY*>(g.dh) + at + c, S[j], left[j]);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          hat[j][i] = (hat[j][i] - mean) * rstd;
          dw[j][i] = fmaf(S[j][i], hat[j][i], dw[j][i]);
          db[j][i] += S[j][i];
        }
        if (g.weight.p) {
          load_param<TY>(g.weight, c, p, left[j]);
#pragma unroll
          for (int i = 0; i < V; ++i) S[j][i] *= p[i];
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
          c1 += S[j][i];
          c2 = fmaf(S[j][i], hat[j][i], c2);
        }
      }
      if (g.dh) {
        row_sum2<TPR>(c1, c2, scratch);
        c1 = n.rms ? 0.f : c1 * inv_d;
        c2 *= inv_d;
      }
#pragma unroll
      for (int j = 0; j < J; ++j) {
        if (left[j] <= 0) continue;
        const int c = (j * TPR + t) * V;
        float p[V];
#pragma unroll
        for (int i = 0; i < V; ++i) S[j][i] = rstd * (S[j][i] - c1 - hat[j][i] * c2);
        if (!g.dh || left[j] < V) {  // no norm gradient, or the places behind the width
#pragma unroll
          for (int i = 0; i < V; ++i) S[j][i] = g.dh && i < left[j] ? S[j][i] : 0.f;
        }
        if (g.ds) {
          load_vec(static_cast<const TX*>(g.ds) + at + c, p, left[j]);
#pragma unroll
          for (int i = 0; i < V; ++i) S[j][i] += p[i];
        }
        if (g.dx) {
#pragma unroll
          for (int i = 0; i < V; ++i) p[i] = n.alpha * S[j][i];
          store_vec(static_cast<TX*>(g.dx) + at + c, p, left[j]);
        }
        if constexpr (!FULL) store_vec(static_cast<TY*>(g.dy) + at + c, S[j], left[j]);
      }
      if constexpr (FULL) {
        const float pmean = n.post ? g.stats[2 * n.rows + r] : 0.f, prstd = n.post ? g.stats[3 * n.rows + r] : 1.f;
        const int64_t gate_at = g.gate.p ? (r / n.gate_rows) * d : 0;
        c1 = c2 = 0.f;
#pragma unroll
        for (int j = 0; j < J; ++j) {
          if (left[j] <= 0) continue;
          const int c = (j * TPR + t) * V;
          float p[V], pw[V], u[V];
          load_vec(static_cast<const TY*>(g.y) + at + c, hat[j], left[j]);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            hat[j][i] = (hat[j][i] - pmean) * prstd;
            u[i] = hat[j][i];
            pw[i] = 1.f;
          }
          if (n.post && g.post_weight.p) {
            load_param<TY>(g.post_weight, c, pw, left[j]);
#pragma unroll
            for (int i = 0; i < V; ++i) u[i] *= pw[i];
          }
          if (n.post && g.post_bias.p) {
            load_param<TY>(g.post_bias, c, p, left[j]);
#pragma unroll
            for (int i = 0; i < V; ++i) u[i] += p[i];
          }
          if (g.gate.p) {
            load_param<TY>(g.gate, gate_at + c, p, left[j]);
#pragma unroll
            for (int i = 0; i < V; ++i) {
              u[i] *= S[j][i];
              dg[j][i] += u[i];
              S[j][i] *= p[i];
            }
            if (g.dgate_mode == 3) store_param<TY>(g.dgate, g.dgate_f32, at + c, u, left[j]);
          }
          if (n.post) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
              dpw[j][i] = fmaf(S[j][i], hat[j][i], dpw[j][i]);
              dpb[j][i] += S[j][i];
              S[j][i] *= pw[i];
              c1 += S[j][i];
              c2 = fmaf(S[j][i], hat[j][i], c2);
            }
          }
        }
        if (n.post) {
          row_sum2<TPR>(c1, c2, scratch);
          c1 = n.rms ? 0.f : c1 * inv_d;
          c2 *= inv_d;
        }
#pragma unroll
        for (int j = 0; j < J; ++j) {
          if (left[j] <= 0) continue;
          if (n.post) {
#pragma unroll
            for (int i = 0; i < V; ++i) S[j][i] = prstd * (S[j][i] - c1 - hat[j][i] * c2);
          }
          store_vec(static_cast<TY*>(g.dy) + at + (j * TPR + t) * V, S[j], left[j]);
        }
      }
    }
    if constexpr (FULL) {
      if (g.dgate_mode == 2) {
        over_slots<TPR>(dg, left, d, red, [&](int c, const float(&v)[V], int k) {
          store_param<TY>(g.dgate, g.dgate_f32, grp * d + c, v, k);
        });
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
          for (int i = 0; i < V; ++i) dg[j][i] = 0.f;
      }
    }
  }
  const int64_t plane = g.split.blocks * d;
  auto leave = [&](int which, const auto& acc) {
    if (!g.want[which]) return;
    float* to = g.part + which * plane + blockIdx.x * (int64_t)d;
    over_slots<TPR>(acc, left, d, red, [&](int c, const float(&v)[V], int k) { store_vec(to + c, v, k); });
  };
  leave(kDw, dw);
  leave(kDb, db);
  if constexpr (FULL) {
    leave(kDg, dg);
    leave(kDpw, dpw);
    leave(kDpb, dpb);
  }
}

// Threads per row and values per thread, by the row's width.
template <typename F>
void by_width(int d, bool full, F&& f) {
  using std::integral_constant;
  if (d <= 64 * 16) f(integral_constant<int, 16>{}, integral_constant<int, 64>{});
  else if (d <= 256 * 16) f(integral_constant<int, 16>{}, integral_constant<int, 256>{});
  else f(integral_constant<int, 16>{}, integral_constant<int, 1024>{});
}

template <typename TX, typename TY>
void launch_forward(const FwdArgs& a, hipStream_t stream) {
  by_width(a.n.d, false, [&](auto e, auto tpr) {
    constexpr int E = decltype(e)::value, TPR = decltype(tpr)::value, B = block_of<TPR>();
    const unsigned grid = (unsigned)std::min<int64_t>((a.n.rows + B / TPR - 1) / (B / TPR), 1 << 20);
    resnorm_fwd_kernel<TX, TY, E, TPR><<<grid, B, 0, stream>>>(a);
  });
}

template <typename TX, typename TY>
void launch_backward(const BwdArgs& a, bool full, hipStream_t stream) {
  by_width(a.n.d, full, [&](auto e, auto tpr) {
    constexpr int E = decltype(e)::value, TPR = decltype(tpr)::value;
    const unsigned grid = (unsigned)a.split.blocks;
    if (full) resnorm_bwd_kernel<TX, TY, E, TPR, true><<<grid, block_of<TPR>(), 0, stream>>>(a);
    else resnorm_bwd_kernel<TX, TY, E, TPR, false><<<grid, block_of<TPR>(), 0, stream>>>(a);
  });
}

// one translation unit per block type (resnorm_f32.hip, resnorm_bf16.hip, resnorm_f16.hip)
#define GRACE_RESNORM_DECLARE(prefix, TX, TY)                                        \
  prefix template void launch_forward<TX, TY>(const FwdArgs&, hipStream_t);          \
  prefix template void launch_backward<TX, TY>(const BwdArgs&, bool, hipStream_t);

}  // namespace resnorm
}  // namespace grace
