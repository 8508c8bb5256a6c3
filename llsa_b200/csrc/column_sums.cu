// Parameter gradients from column sums per sample (column_sums.cuh).
#include "column_sums.cuh"

namespace llsa {

namespace {

constexpr uint32_t kCols = 32, kLanes = 32;

// blockIdx.y: 32 columns; blockIdx.x: a sample, or (the last one, with `overall`) all of them.  Thread (column, lane) adds every 32nd part;
// the lanes are added in order through shared memory.  Parts are few and far: what counts is how many loads are on their way, and that nothing beside them is
// slow (a part's sample divided out of its number: layer norm's backward of 2 x 8192 rows of 2048 channels 58.8 us, 53.5 so).  Eight columns to a CTA of
// 128 lanes took 62.2.
__global__ void __launch_bounds__(kCols * kLanes)
column_grads_kernel(ColumnParts P, ColumnParts S, uint32_t B, int C, ParamView w, ParamView bias, ParamView s, float plus, ColumnGrads g, int overall) {
  __shared__ float s_sum[2][kLanes][kCols];
  const uint32_t col = threadIdx.x % kCols, lane = threadIdx.x / kCols;
  const int c = (int) (blockIdx.y * kCols + col);
  const bool all = overall && blockIdx.x == gridDim.x - 1;
  const int64_t b = blockIdx.x;
  float sum[2] = {0.f, 0.f};
  const auto add = [&](const ColumnParts& parts, int which, float& to) {
    const uint32_t chunks = (uint32_t) parts.chunks, n = all ? B * chunks : chunks;
    const float* p = parts.p + (all ? 0 : b * chunks * 2 * C) + which * C + c;
    if (all && s.p) {
      // the sample of part i goes along with i
      const uint32_t dq = kLanes / chunks, dr = kLanes % chunks;
      uint32_t q = lane / chunks, r = lane % chunks;
#pragma unroll 4
      for (uint32_t i = lane; i < n; i += kLanes) {
        to = fmaf(plus + s.at(q, c, 0.f), p[(int64_t) i * 2 * C], to);
        q += dq, r += dr;
        if (r >= chunks) r -= chunks, ++q;
      }
    } else {
#pragma unroll 8
      for (uint32_t i = lane; i < n; i += kLanes) to += p[(int64_t) i * 2 * C];
    }
  };
  pdl_wait();
  pdl_trigger();
  if (c < C) {
    if (all ? g.weight.p : g.scale.p) add(P, 0, sum[0]);
    if (all ? g.bias.p != nullptr : g.shift.p || (g.scale.p && bias.p)) add(S, 1, sum[1]);
  }
  s_sum[0][lane][col] = sum[0];
  s_sum[1][lane][col] = sum[1];
  __syncthreads();
  if (lane || c >= C) return;
  sum[0] = sum[1] = 0.f;
#pragma unroll
  for (uint32_t k = 0; k < kLanes; ++k) {
    sum[0] += s_sum[0][k][col];
    sum[1] += s_sum[1][k][col];
  }
  if (all) {
    if (g.weight.p) g.weight.put(c, sum[0]);
    if (g.bias.p) g.bias.put(c, sum[1]);
  } else {
    if (g.scale.p) g.scale.put(b * C + c, fmaf(w.at(0, c, 1.f), sum[0], bias.at(0, c, 0.f) * sum[1]));
    if (g.shift.p) g.shift.put(b * C + c, sum[1]);
  }
}

}  // namespace

int make_param(ParamView* v, const LlsaTensor* t, const char* name, int dtype, int64_t B, int64_t C) {
  v->p = nullptr;
  v->ld = 0;
  v->is_bf16 = 0;
  if (!t) return LLSA_OK;
  LLSA_REQUIRE(t->ptr, LLSA_ERR_NULL, "%s: null tensor", name);
  LLSA_REQUIRE(t->dtype == LLSA_F32 || t->dtype == dtype, LLSA_ERR_DTYPE, "%s: must be f32 or of the data's type", name);
  if (B) LLSA_REQUIRE(t->ndim == 2 && t->shape[0] == B && t->shape[1] == C, LLSA_ERR_SHAPE, "%s: must be [%lld,%lld]", name, (long long) B, (long long) C);
  else LLSA_REQUIRE(t->ndim == 1 && t->shape[0] == C, LLSA_ERR_SHAPE, "%s: must be [%lld]", name, (long long) C);
  LLSA_REQUIRE(C == 1 || t->stride[t->ndim - 1] == 1, LLSA_ERR_STRIDE, "%s: innermost stride must be 1", name);
  v->p = t->ptr;
  v->ld = B ? t->stride[0] : 0;
  v->is_bf16 = t->dtype == LLSA_BF16;
  return LLSA_OK;
}

int check_grad(const LlsaTensor* t, const char* name, int dtype, int ndim, const int64_t* shape) {
  LLSA_REQUIRE(t->ptr, LLSA_ERR_NULL, "%s: null tensor", name);
  LLSA_REQUIRE(t->dtype == LLSA_F32 || t->dtype == dtype, LLSA_ERR_DTYPE, "%s: must be f32 or of the data's type", name);
  return check_contig(t, name, t->dtype, ndim, shape);
}

int finish_column_grads(const ColumnParts& P, const ColumnParts& S, int64_t B, int64_t C, const ParamView& w, const ParamView& bias, const ParamView& s, float plus,
                        const ColumnGrads& g, cudaStream_t st) {
  const int per_sample = g.scale.p || g.shift.p, overall = g.weight.p || g.bias.p;
  const int64_t slots = (per_sample ? B : 0) + overall;
  if (slots == 0) return LLSA_OK;
  launch_pdl(column_grads_kernel, dim3((unsigned) slots, (unsigned) ((C + kCols - 1) / kCols)), dim3(kCols * kLanes), 0, st, P, S, (uint32_t) B, (int) C, w, bias,
             s, plus, g, overall);
  LLSA_LAUNCH_OK("column_grads_kernel");
  return LLSA_OK;
}

int clear_column_grads(const ColumnGrads& g, int64_t B, int64_t C, cudaStream_t st) {
  const GradView* const v[4] = {&g.scale, &g.shift, &g.weight, &g.bias};
  for (int i = 0; i < 4; ++i)
    if (v[i]->p && (i >= 2 || B)) LLSA_CUDA_OK(cudaMemsetAsync(v[i]->p, 0, (size_t) ((i < 2 ? B : 1) * C * (v[i]->is_bf16 ? 2 : 4)), st));
  return LLSA_OK;
}

}  // namespace llsa
