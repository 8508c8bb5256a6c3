// What the projection's kernels share: the epilogue's operands, the activations, and the interface between linear.cu and the matrix products.
#pragma once
#include "column_sums.cuh"
#include "common.cuh"

namespace llsa {

enum Activation { kActNone = 0, kActGeluTanh = 1, kActSilu = 2 };

// A matrix with unit stride along one of its dimensions: element (i, j) at p[i * ld + j]
template <typename T>
struct Mat {
  T* p;
  int64_t ld;
};

// What stands behind the product z of a forward: y = residual + gate act(z + bias); `pre`, if given, keeps z + bias for the backward (in the data's type, as it is as
// large as y: a half step of each term of the gate's gradient).
template <typename T>
struct Epilogue {
  const T* bias;
  Mat<const T> residual;
  Mat<const T> gate;            // row = sample
  uint32_t rows_per_gate;
  Mat<T> y;
  Mat<T> pre;
  int act;
};

constexpr float kGelu2 = 1.5957691216057308f, kGelu3 = 0.044715f;      // 2 sqrt(2 / pi)
// 1 / (1 + e^-t)
__device__ __forceinline__ float sigmoid(float t) { return 1.f / (1.f + expf(-t)); }
// gelu_tanh: z (1 + tanh(u)) / 2 = z sigmoid(2 u), u = sqrt(2 / pi) (z + 0.044715 z^3): no cancellation for negative z
__device__ __forceinline__ float activate(float z, int act) {
  if (act == kActGeluTanh) return z * sigmoid(kGelu2 * z * fmaf(kGelu3 * z, z, 1.f));
  if (act == kActSilu) return z * sigmoid(z);
  return z;
}
// The derivative; beyond |z| = 1e4 it is 0 or 1, and z^2 and an infinite z are kept out of its products with 0
__device__ __forceinline__ float activate_grad(float z, int act) {
  if (act == kActNone) return 1.f;
  if (fabsf(z) > 1e4f) z = copysignf(1e4f, z);
  const bool gelu = act == kActGeluTanh;
  const float q = z * z, s = sigmoid(gelu ? kGelu2 * z * fmaf(kGelu3, q, 1.f) : z);
  const float du = gelu ? kGelu2 * fmaf(3.f * kGelu3, q, 1.f) : 1.f;
  return fmaf(z * s * (1.f - s), du, s);
}

// D[i, j] = sum_k A(i, k) B(j, k), k < K.  a_k: A(i, k) at a.p[i * ld + k] (else at a.p[k * ld + i]); b_k alike.
template <typename T>
struct Product {
  Mat<const T> a, b;
  int a_k, b_k;
  int64_t M, N, K;
  int split;                   // parts of the sum over k, one after another in `partial`; 1: none
  int64_t samples = 0;         // bf16: that many products of these sizes, their operands and results one behind the other (parts: `split` of each)
};

// bf16, on tcgen05 (linear_tc.cu).  Operands: rows on 16-byte boundaries.  The forward and the input's gradient (A along k), with their epilogue;
int linear_tc_product(const Product<__nv_bfloat16>& p, const Epilogue<__nv_bfloat16>& e, int wait_limit, int32_t* status, cudaStream_t st);
// (with samples: the input's gradient alone, B along i or j).
// dz = dy act'(z) with z computed once more, e.y = dz (rows on 16-byte boundaries), and the column sums of dz: sums[group][1][N], linear_tc_slope_groups of them;
int linear_tc_slope(const Product<__nv_bfloat16>& p, const Epilogue<__nv_bfloat16>& e, const Mat<const __nv_bfloat16>& dy, float* sums, int wait_limit,
                    int32_t* status, cudaStream_t st);
int64_t linear_tc_slope_groups(int64_t M, int64_t N, int64_t K);
// the weight's gradient (both operands across), in p.split parts of [M][ld], ld a multiple of 8; the number of parts to take
int linear_tc_parts(const Product<__nv_bfloat16>& p, float* partial, int64_t ld, int wait_limit, int32_t* status, cudaStream_t st);
// `turned`: the parts are better taken of the transposed result, A and B changing places
int linear_tc_split(int64_t M, int64_t N, int64_t K, int64_t samples, bool* turned);

}  // namespace llsa
