// Launchers of the residual norms (the kernels, and the mathematics: grace_resnorm.h).
#include "grace_resnorm.h"

namespace grace {

namespace resnorm {
GRACE_RESNORM_DECLARE(extern, float, float)
GRACE_RESNORM_DECLARE(extern, bf16_t, bf16_t)
GRACE_RESNORM_DECLARE(extern, float, bf16_t)
GRACE_RESNORM_DECLARE(extern, half_t, half_t)
GRACE_RESNORM_DECLARE(extern, float, half_t)
}  // namespace resnorm

namespace {

using namespace resnorm;

// Rows per row slot of a workgroup before another workgroup is added, where there is one for each CU: 4096 fp32 rows of
// 768 take 11.1 + 3.9 us (backward and fold) with two and 12.8 + 5.0 us with one, 735 fp16 rows of 651 10.8 and 8.3 us.
constexpr int kMinRows = 2;

struct FoldArgs {
  const float* part;
  int64_t blocks;
  int d;
  int sums;            // outputs below: the wanted sums in turn
  int which[kSums];
  void* out[kSums];
  bool f32[kSums];
  int64_t rows[kSums];  // output rows (more than one: dgate's groups)
};

// One workgroup adds 64 columns of one output row.  16 lanes read the columns of a partial row, so the
// workgroup's 64 slices have 64 x kAhead rows in flight: the launch is one or two latencies long (3.9 us for 512
// partial rows of two sums of 768 columns, 9 us for 512 of three of 4096).
constexpr int kFoldCols = 64, kFoldSlices = 64, kAhead = 4;
template <typename TY>
__global__ __launch_bounds__(1024) void resnorm_fold_kernel(FoldArgs a) {
  int64_t row = blockIdx.y;
  int k = 0;
  while (k + 1 < a.sums && row >= a.rows[k]) row -= a.rows[k++];
  const int64_t per = a.blocks / a.rows[k];
  const int slice = threadIdx.x / 16, lane = threadIdx.x % 16;
  const int c = blockIdx.x * kFoldCols + lane * 4, left = min(a.d - c, 4);
  float v[4] = {};
  if (left > 0) {
    const float* p = a.part + ((int64_t)a.which[k] * a.blocks + row * per) * a.d + c;
    for (int64_t i = slice; i < per; i += kFoldSlices * kAhead) {
      float x[kAhead][4];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
#pragma unroll
        for (int q = 0; q < 4; ++q) x[u][q] = 0.f;
        if (i + u * kFoldSlices < per) load_vec(p + (i + u * kFoldSlices) * a.d, x[u], left);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] += x[u][q];
    }
  }
  __shared__ float red[kFoldSlices][kFoldCols];
#pragma unroll
  for (int q = 0; q < 4; ++q) red[slice][lane * 4 + q] = v[q];
  // 16 waves: 16 sums of 4 slices, then the first wave joins those
  const int col = lane_id(), w = wave_id();
  __syncthreads();
  float s = red[4 * w][col] + red[4 * w + 1][col] + red[4 * w + 2][col] + red[4 * w + 3][col];
  __syncthreads();
  red[w][col] = s;
  __syncthreads();
  const int at = blockIdx.x * kFoldCols + col;
  if (w == 0 && at < a.d) {
#pragma unroll
    for (int i = 1; i < 16; ++i) s += red[i][col];
    if (a.f32[k]) static_cast<float*>(a.out[k])[row * a.d + at] = s;
    else static_cast<TY*>(a.out[k])[row * a.d + at] = (TY)s;
  }
}

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// row slots of a workgroup, and the workgroups that the chip holds at a time
struct Shape {
  int slots, resident;
};
Shape shape_of(int d) {
  Shape s{};
  by_width(d, [&](auto, auto tpr) {
    constexpr int TPR = decltype(tpr)::value;
    s = {block_of<TPR>() / TPR, kCUs * 1024 / block_of<TPR>()};
  });
  return s;
}

Split split_rows(const NormShape& n, bool grouped) {
  const Shape shape = shape_of(n.d);
  const int64_t one = cdiv(n.rows, shape.slots), several = cdiv(n.rows, (int64_t)shape.slots * kMinRows);
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>(shape.resident, std::max(several, std::min<int64_t>(one, kCUs))));
  Split s{1, n.rows, most, 1, most};
  if (grouped && n.gate_rows < n.rows) {
    s.groups = n.rows / n.gate_rows;
    s.group_rows = n.gate_rows;
    s.parts = std::max<int64_t>(1, most / s.groups);
    s.per_block = s.parts > 1 ? 1 : cdiv(s.groups, most);
    s.blocks = s.parts > 1 ? s.groups * s.parts : cdiv(s.groups, s.per_block);
  }
  return s;
}

// A backward that moves more than twice the 256 MB memory-side cache stores past it, for what it writes first is
// gone from there when it ends: 64 million fp32 values in rows of 1024 take 214 us for 218 us, with gate and post
// norm 316 for 327 (32768 bf16 rows of 4096: the same).  The forward loses by it: 219 us for 205 us there.
bool moves_much(const NormShape& n) { return n.rows * n.d * (el_bytes(n.tx) + el_bytes(n.ty)) * 2 > (512ll << 20); }

template <typename F>
void by_types(const NormShape& n, F&& f) {
  using std::integral_constant;
  if (n.ty == ElType::kF32) return f((float*)nullptr, (float*)nullptr);
  if (n.ty == ElType::kBF16)
    return n.tx == ElType::kF32 ? f((float*)nullptr, (bf16_t*)nullptr) : f((bf16_t*)nullptr, (bf16_t*)nullptr);
  return n.tx == ElType::kF32 ? f((float*)nullptr, (half_t*)nullptr) : f((half_t*)nullptr, (half_t*)nullptr);
}

}  // namespace

void resnorm_forward(const NormShape& n, const void* x, const void* y, NormParam gate, NormParam weight, NormParam bias,
                     NormParam post_weight, NormParam post_bias, void* h, void* s, float* stats, hipStream_t stream) {
  if (n.rows == 0 || n.d == 0) return;
  const FwdArgs a{n, x, y, gate, weight, bias, post_weight, post_bias, h, s, stats};
  by_types(n, [&](auto* tag_x, auto* tag_y) {
    using TX = std::remove_pointer_t<decltype(tag_x)>;
    using TY = std::remove_pointer_t<decltype(tag_y)>;
    launch_forward<TX, TY>(a, stream);
  });
}

int64_t resnorm_backward_ws(const NormShape& n) {
  const int64_t blocks = std::max(split_rows(n, false).blocks, split_rows(n, true).blocks);
  return kSums * blocks * n.d * (int64_t)sizeof(float);
}

void resnorm_backward(const NormShape& n, const void* s, const void* x, const void* y, const float* stats, NormParam gate,
                      NormParam weight, NormParam post_weight, NormParam post_bias, const void* dh, const void* ds,
                      const NormGrads& g, void* ws, hipStream_t stream) {
  if (n.rows == 0 || n.d == 0) return;
  const bool own_rows = n.gate_rows == 1 && n.rows > 1;  // the gate has the rows' own shape
  BwdArgs a{};
  a.n = n;
  a.split = split_rows(n, g.dgate != nullptr && !own_rows);
  a.s = s;
  a.x = x;
  a.y = y;
  a.dh = dh;
  a.ds = ds;
  a.stats = stats;
  a.gate = gate;
  a.weight = weight;
  a.post_weight = post_weight;
  a.post_bias = post_bias;
  a.dx = g.dx == g.dy ? nullptr : g.dx;
  a.dy = g.dy;
  a.dgate = g.dgate;
  a.dgate_f32 = gate.f32;
  a.dgate_mode = g.dgate == nullptr ? kGateNone
                 : own_rows         ? kGateRows
                 : a.split.groups > 1 && a.split.parts == 1 ? kGateGroups : kGateParts;
  a.once = moves_much(n);
  a.part = static_cast<float*>(ws);
  void* const outs[kSums] = {g.dweight, g.dbias, a.dgate_mode == kGateParts ? g.dgate : nullptr, g.dpost_weight, g.dpost_bias};
  FoldArgs f{};
  f.part = a.part;
  f.blocks = a.split.blocks;
  f.d = n.d;
  const bool f32[kSums] = {weight.f32, g.bias_f32, gate.f32, post_weight.f32, g.post_bias_f32};
  int64_t out_rows = 0;
  for (int k = 0; k < kSums; ++k) {
    a.want[k] = outs[k] != nullptr;
    if (!outs[k]) continue;
    f.which[f.sums] = k;
    f.out[f.sums] = outs[k];
    f.f32[f.sums] = f32[k];
    f.rows[f.sums] = k == kDg ? a.split.groups : 1;
    out_rows += f.rows[f.sums++];
  }
  by_types(n, [&](auto* tag_x, auto* tag_y) {
    using TX = std::remove_pointer_t<decltype(tag_x)>;
    using TY = std::remove_pointer_t<decltype(tag_y)>;
    launch_backward<TX, TY>(a, stream);
    if (f.sums > 0)
      resnorm_fold_kernel<TY><<<dim3((unsigned)cdiv(n.d, kWave), (unsigned)out_rows), 1024, 0, stream>>>(f);
  });
}

}  // namespace grace
