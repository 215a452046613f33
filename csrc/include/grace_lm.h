// Launchers of the language-model training kernels: embedding (embed.hip), residual norms
// (resnorm.hip) and the global gradient norm (gradnorm.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "grace_vec.h"

namespace grace {

// ---------------------------------------------------------------- embedding (embed.hip)
struct EmbedIds {
  const void* ids;  // [n] int64 or int32, contiguous
  bool is64;
  int64_t n;
  int64_t vocab;
  int64_t pad;  // row without a gradient, or -1
};

// slabs of columns are a grid's second dimension, or a factor of its first, which holds less than 2^32 threads
constexpr int64_t kEmbedMaxWidth = 1 << 21;

// out[t, :] = round(scale * w[ids[t], :]); rows of w are w_stride elements apart
void embed_forward(const EmbedIds& ids, const void* w, ElType tw, int64_t w_stride, int64_t d, float scale, void* out,
                   ElType to, hipStream_t stream);

// bytes of workspace that embed_backward needs
int64_t embed_backward_ws(int64_t n, int64_t vocab, int64_t d);

// dw[v, :] = round(scale * sum of dy[t, :] over ids[t] == v), every row of dw [vocab, d] (16-byte aligned)
// written; n > 0
void embed_backward(const EmbedIds& ids, const void* dy, ElType tdy, int64_t d, float scale, void* dw, ElType tdw,
                    void* ws, hipStream_t stream);

// ---------------------------------------------------------------- residual norm (resnorm.hip)
//   u = post ? N(y; post_weight, post_bias) : y
//   s = alpha * x + gate . u         (x = nullptr: s = gate . u)
//   h = N(s; weight, bias)
// N is a layer norm, or a root-mean-square norm (rms).  Rows are contiguous; x, s and their gradients
// have type tx, y, h and theirs ty.  A parameter or gate is fp32 or of type ty.
struct NormParam {
  const void* p;  // nullptr: none (one for a weight or gate, zero for a bias)
  bool f32;
};
struct NormShape {
  int64_t rows;
  int64_t gate_rows;  // consecutive rows that share one row of the gate (rows: one gate for all)
  int d;
  float alpha, eps;
  bool rms, post;
  ElType tx, ty;
};
constexpr int kNormMaxWidth = 16384;

// stats: [2, rows] fp32 (mean, 1 / deviation of s), with post [4, rows] (and those of y); may be null.
// s may be null (not written).
void resnorm_forward(const NormShape& n, const void* x, const void* y, NormParam gate, NormParam weight, NormParam bias,
                     NormParam post_weight, NormParam post_bias, void* h, void* s, float* stats, hipStream_t stream);

struct NormGrads {
  void *dx, *dy;                                    // dx may be null, or equal to dy
  void *dgate, *dweight, *dbias, *dpost_weight, *dpost_bias;  // nullptr: not wanted; of their parameter's type
  bool bias_f32, post_bias_f32;
};
int64_t resnorm_backward_ws(const NormShape& n);  // bytes
// s: the sum as it was stored, of type tx = fp32, or y itself without x, gate and post; or nullptr: made again
// from x (may be null) and y.  dh or ds may be null (a zero gradient).  y may be null where only s is read.
void resnorm_backward(const NormShape& n, const void* s, const void* x, const void* y, const float* stats, NormParam gate,
                      NormParam weight, NormParam post_weight, NormParam post_bias, const void* dh, const void* ds,
                      const NormGrads& g, void* ws, hipStream_t stream);

// ---------------------------------------------------------------- global gradient norm (gradnorm.hip)
struct GradTensor {
  void* p;  // dense memory of len elements
  int64_t len;
  ElType type;
};
enum class NormKind : int { kMax = 0, kL1 = 1, kL2 = 2 };

int64_t gradnorm_parts(const GradTensor* g, int64_t n);  // partial values that the next call writes
void gradnorm_partial(const GradTensor* g, int64_t n, NormKind kind, double* part, hipStream_t stream);
// out[0] = norm, out[1] = min(1, max_norm / (norm + 1e-6)), from any number of partial values
void gradnorm_finish(const double* part, int64_t parts, NormKind kind, float max_norm, float* out, hipStream_t stream);
// both at once from the partial values: out as above, and g *= out[1]; no tensors: neither
void grad_clip(const GradTensor* g, int64_t n, const double* part, int64_t parts, NormKind kind, float max_norm,
               float* out, hipStream_t stream);
// g *= *factor (a device value); one leaves the memory untouched.  No two tensors may overlap.
void grad_scale(const GradTensor* g, int64_t n, const float* factor, hipStream_t stream);

}  // namespace grace
