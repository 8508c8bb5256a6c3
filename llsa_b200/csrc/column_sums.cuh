// Column sums per sample and the parameter gradients that come from them: shared by the layer norm's and the projection's backward.
#pragma once
#include <algorithm>

#include "common.cuh"

namespace llsa {

// A parameter that a kernel reads element by element: [C] (ld 0) or [B, C], fp32 or bf16, or absent
struct ParamView {
  const void* p;
  int64_t ld;
  int is_bf16;
  __device__ __forceinline__ float at(uint32_t b, int c, float absent) const {
    if (!p) return absent;
    const int64_t i = b * ld + c;
    return is_bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]) : reinterpret_cast<const float*>(p)[i];
  }
};
// The gradient of one, contiguous, rounded once when it is written
struct GradView {
  void* p;
  int is_bf16;
  __device__ __forceinline__ void put(int64_t i, float v) const {
    if (is_bf16) reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
    else reinterpret_cast<float*>(p)[i] = v;
  }
};
// per sample [B, C]: scale, shift; over all samples [C]: weight, bias
struct ColumnGrads {
  GradView scale, shift, weight, bias;
};

// B = 0: a vector [C]; else [B, C] with any row stride.  dtype: f32 or the data's.
int make_param(ParamView* v, const LlsaTensor* t, const char* name, int dtype, int64_t B, int64_t C);
int check_grad(const LlsaTensor* t, const char* name, int dtype, int ndim, const int64_t* shape);
inline GradView make_grad(const LlsaTensor* t) {
  GradView g;
  g.p = t ? t->ptr : nullptr;
  g.is_bf16 = t && t->dtype == LLSA_BF16;
  return g;
}

// The sums P and S of parts of a sample's rows: P in partial[B * chunks][0][C] of one array, S in [B * chunks][1][C] of the same or another one
struct ColumnParts {
  const float* p;
  int64_t chunks;
};
// With P_b, S_b the sums of a sample's parts, added in order:
//   scale_b = w P_b + bias S_b,  shift_b = S_b,  weight = sum_b f_b P_b,  bias = sum_b f_b S_b          (those that are wanted)
// f_b = plus + s_b, 1 where there is no s
int finish_column_grads(const ColumnParts& P, const ColumnParts& S, int64_t B, int64_t C, const ParamView& w, const ParamView& bias, const ParamView& s, float plus,
                        const ColumnGrads& grads, cudaStream_t st);
// The same of no rows at all
int clear_column_grads(const ColumnGrads& grads, int64_t B, int64_t C, cudaStream_t st);

}  // namespace llsa
