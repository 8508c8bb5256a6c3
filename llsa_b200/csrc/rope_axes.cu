// Rotary positions over several axes (rows and columns of an image; time, rows and columns of a clip), without a table.
//
// The channels are cut into one part per axis (models/rope_dit_transformer_2d.py:71-109: axes_dims_rope); pair i of axis a's d_a channels turns by
//   angle(n, a, i) = pos[n, a] theta^(-2 i / d_a),     y[2c] = cos x[2c] - sin x[2c+1],  y[2c+1] = sin x[2c] + cos x[2c+1]
// (triton/rope.py:37-47); the backward pass is the rotation by -angle.  The angle is a product in 64 bits, kept in units of pi, so that whole turns
// come off exactly (t - 2 rint(t / 2)) and sine and cosine see a number in [-1, 1]: positions of a million cost no precision.  A thread owns 16 bytes of
// channels of one token, computes their sines once and turns that token's rows of several heads and samples with them: the arithmetic is
// spread over B H rows, and what is left is one read of x and one write of y.
//
// Bound by memory.  bf16 [8, 6, 16384, 64] (201 MB moved): 32.7 us, 6.2 TB/s; fp32 [2, 12, 16384, 128] (403 MB): 61.6 us, 6.5 TB/s.  With the first
// rows loaded behind the sines instead of before them, and the row's place divided out of its number, 40.0 us; batches of four rows 33.8, of
// eight 33.4; half the CTAs 32.9.
#include <math.h>

#include <algorithm>

#include "common.cuh"
#include "vec.cuh"

namespace llsa {

namespace {

using bf16 = __nv_bfloat16;

constexpr int kMaxPairs = 256, kMaxAxes = 4;

struct AxesTable {
  double turn[kMaxPairs];           // theta^(-2 i / d_a) / pi
  int end[kMaxAxes];                // first pair behind axis a
};

struct Positions {
  const void* p;
  int64_t sb, sn;                   // sb 0: the same for every sample
  int kind;                         // LlsaDtype
  __device__ __forceinline__ double at(int64_t b, int64_t n, int a) const {
    const int64_t i = b * sb + n * sn + a;
    if (kind == LLSA_I64) return (double) reinterpret_cast<const int64_t*>(p)[i];
    if (kind == LLSA_I32) return (double) reinterpret_cast<const int32_t*>(p)[i];
    return (double) reinterpret_cast<const float*>(p)[i];
  }
};

// Grid: x over (token, 16 bytes), y over parts of the B H rows of a token (per sample: of its H heads, times B).
template <typename T, int N, int U>
__global__ void __launch_bounds__(256)
rope_axes_kernel(View<const T> x, View<T> y, Positions pos, const __grid_constant__ AxesTable table, int axes, float sign, int64_t S, int lanes, uint32_t H,
                 uint32_t rows, uint32_t per, uint32_t parts) {
  using V = Vec<T, N>;
  pdl_wait();
  pdl_trigger();
  const int64_t i = blockIdx.x * (int64_t) blockDim.x + threadIdx.x;
  const int64_t n = i / lanes;
  const int c = (int) (i - n * lanes) * N;
  if (n >= S) return;
  // per sample: blockIdx.y = sample * parts + part, rows = H;  else blockIdx.y = part, rows = B H
  const uint32_t b0 = blockIdx.y / parts, first = (blockIdx.y - b0 * parts) * per, end = min(rows, first + per);
  // rows of the batch that starts at r: their first loads are on their way while the sines are computed
  uint32_t b = b0 + first / H, h = first % H;
  const auto load = [&](typename V::type (&raw)[U], T* (&to)[U], uint32_t r) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (r + u < end) {
        raw[u] = *reinterpret_cast<const typename V::type*>(x.row(b, h, n) + c);
        to[u] = y.row(b, h, n) + c;
        if (++h == H) h = 0, ++b;
      }
  };
  typename V::type raw[U];
  T* to[U];
  load(raw, to, first);
  float sn[N / 2], cs[N / 2];
#pragma unroll
  for (int j = 0; j < N / 2; ++j) {
    const int pair = c / 2 + j;
    int a = 0;
    while (a + 1 < axes && pair >= table.end[a]) ++a;
    const double t = pos.at(b0, n, a) * table.turn[pair];
    sincospif((float) (t - 2.0 * rint(t * 0.5)), &sn[j], &cs[j]);
    sn[j] *= sign;
  }
  for (uint32_t r = first; r < end; r += U) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (r + u < end) {
        float v[N], w[N];
        V::unpack(raw[u], v);
#pragma unroll
        for (int j = 0; j < N / 2; ++j) {
          w[2 * j] = fmaf(cs[j], v[2 * j], -sn[j] * v[2 * j + 1]);
          w[2 * j + 1] = fmaf(sn[j], v[2 * j], cs[j] * v[2 * j + 1]);
        }
        *reinterpret_cast<typename V::type*>(to[u]) = V::pack(w);
      }
    if (r + U < end) load(raw, to, r + U);
  }
}

bool rows_aligned(const LlsaTensor* t, int64_t per16) {
  if ((uintptr_t) t->ptr % 16 || t->shape[3] % per16) return false;
  for (int i = 0; i < 3; ++i)
    if (t->shape[i] != 1 && t->stride[i] % per16) return false;
  return true;
}

template <typename T, int N>
int launch(const LlsaTensor* x, const LlsaTensor* y, const Positions& pos, const AxesTable& table, int axes, bool inverse, cudaStream_t st) {
  constexpr int U = 6;                                // rows on their way at once
  const int64_t B = x->shape[0], H = x->shape[1], S = x->shape[2], D = x->shape[3];
  const int64_t lanes = D / N, blocks = (S * lanes + 255) / 256;
  const int64_t rows = pos.sb ? H : B * H, samples = pos.sb ? B : 1;
  // two rounds of CTAs on every SM, so that one's sines are computed behind another's loads; at least one batch of rows each
  int64_t parts = std::min((148 * 16 + blocks * samples - 1) / (blocks * samples), (rows + U - 1) / U);
  parts = std::max<int64_t>(parts, 1);
  const int64_t per = ((rows + parts - 1) / parts + U - 1) / U * U;
  parts = (rows + per - 1) / per;
  LLSA_REQUIRE(blocks <= INT32_MAX && rows <= INT32_MAX && samples * parts <= 65535, LLSA_ERR_SHAPE, "rope_axes: too many tokens, or too many samples with positions of their own");
  launch_pdl(rope_axes_kernel<T, N, U>, dim3((unsigned) blocks, (unsigned) (samples * parts)), dim3(256), 0, st, make_view<const T>(x), make_view<T>(y), pos,
             table, axes, inverse ? -1.f : 1.f, S, (int) lanes, (uint32_t) H, (uint32_t) rows, (uint32_t) per, (uint32_t) parts);
  LLSA_LAUNCH_OK("rope_axes_kernel");
  return LLSA_OK;
}

}  // namespace
}  // namespace llsa

using namespace llsa;

extern "C" int llsa_rope_axes(const LlsaTensor* x, const LlsaTensor* positions, int n_axes, const int32_t* axes_dims, double theta, int inverse,
                              const LlsaTensor* y, void* stream) {
  LLSA_REQUIRE(x && positions && axes_dims && y && x->ptr && positions->ptr && y->ptr, LLSA_ERR_NULL, "rope_axes: null argument");
  LLSA_REQUIRE(is_float_dtype(x->dtype) && y->dtype == x->dtype, LLSA_ERR_DTYPE, "rope_axes: x and y must both be f32 or both bf16");
  LLSA_REQUIRE(positions->dtype == LLSA_I32 || positions->dtype == LLSA_I64 || positions->dtype == LLSA_F32, LLSA_ERR_DTYPE,
               "rope_axes: positions must be i32, i64 or f32");
  LLSA_REQUIRE(x->ndim == 4 && y->ndim == 4, LLSA_ERR_SHAPE, "rope_axes: x and y must be [B,H,N,D]");
  const int64_t B = x->shape[0], H = x->shape[1], N = x->shape[2], D = x->shape[3];
  for (int i = 0; i < 4; ++i) LLSA_REQUIRE(x->shape[i] == y->shape[i], LLSA_ERR_SHAPE, "rope_axes: x and y differ in dimension %d", i);
  LLSA_REQUIRE(x->stride[3] == 1 && y->stride[3] == 1, LLSA_ERR_STRIDE, "rope_axes: innermost strides must be 1");
  LLSA_REQUIRE(n_axes >= 1 && n_axes <= kMaxAxes, LLSA_ERR_ARG, "rope_axes: %d axes, supported are 1 to %d", n_axes, kMaxAxes);
  LLSA_REQUIRE(theta > 0 && isfinite(theta), LLSA_ERR_ARG, "rope_axes: theta must be a positive number");
  AxesTable table;
  int64_t sum = 0;
  for (int a = 0; a < n_axes; ++a) {
    LLSA_REQUIRE(axes_dims[a] >= 2 && axes_dims[a] % 2 == 0, LLSA_ERR_ARG, "rope_axes: axis %d has %d channels, must be a positive even number", a, axes_dims[a]);
    sum += axes_dims[a];
  }
  LLSA_REQUIRE(sum == D, LLSA_ERR_SHAPE, "rope_axes: the axes have %lld channels together, x has %lld", (long long) sum, (long long) D);
  LLSA_REQUIRE(D <= 2 * kMaxPairs, LLSA_ERR_SHAPE, "rope_axes: %lld channels, supported are up to %d", (long long) D, 2 * kMaxPairs);
  int pair = 0;
  for (int a = 0; a < kMaxAxes; ++a) {
    if (a < n_axes)
      for (int i = 0; i < axes_dims[a] / 2; ++i) table.turn[pair++] = pow(theta, -2.0 * i / axes_dims[a]) / M_PI;
    table.end[a] = pair;
  }
  for (; pair < kMaxPairs; ++pair) table.turn[pair] = 0;
  const bool per_sample = positions->ndim == 3;
  LLSA_REQUIRE(positions->ndim == 2 || per_sample, LLSA_ERR_SHAPE, "rope_axes: positions must be [N,A] or [B,N,A]");
  const int64_t* ps = positions->shape + (per_sample ? 1 : 0);
  LLSA_REQUIRE((!per_sample || positions->shape[0] == B) && ps[0] == N && ps[1] == n_axes, LLSA_ERR_SHAPE, "rope_axes: positions must be [%lld,%d] or [%lld,%lld,%d]",
               (long long) N, n_axes, (long long) B, (long long) N, n_axes);
  const int64_t* pst = positions->stride + (per_sample ? 1 : 0);
  LLSA_REQUIRE(n_axes == 1 || pst[1] == 1, LLSA_ERR_STRIDE, "rope_axes: innermost stride of positions must be 1");
  Positions pos;
  pos.p = positions->ptr;
  pos.sb = per_sample && B > 1 ? positions->stride[0] : 0;      // samples that share their positions are turned together
  pos.sn = pst[0];
  pos.kind = positions->dtype;
  if (B * H * N == 0) return LLSA_OK;
  const cudaStream_t st = (cudaStream_t) stream;
  const int64_t per16 = x->dtype == LLSA_F32 ? 4 : 8;
  const bool wide = rows_aligned(x, per16) && rows_aligned(y, per16);
  if (x->dtype == LLSA_F32)
    return wide ? launch<float, 4>(x, y, pos, table, n_axes, inverse, st) : launch<float, 2>(x, y, pos, table, n_axes, inverse, st);
  return wide ? launch<bf16, 8>(x, y, pos, table, n_axes, inverse, st) : launch<bf16, 2>(x, y, pos, table, n_axes, inverse, st);
}
