// Layer norm with an optional learned weight and bias and an optional scale and shift per sample (adaLN), forward and backward
// (models/rope_dit_transformer_2d.py:295-337, :600-640: norm(x) * (1 + scale) + shift).
//
//   h = (x - mean) rstd,   y = h A + T,   A = w (1 + s_b),  T = bias (1 + s_b) + t_b          (absent: w = 1, bias = s = t = 0)
//   g = dy A,   dx = rstd (g - mean_c(g) - h mean_c(g h))
//   P_b = sum_n dy h,  S_b = sum_n dy;   dt_b = S_b,  ds_b = w P_b + bias S_b,  dw = sum_b (1 + s_b) P_b,  dbias = sum_b (1 + s_b) S_b
//
// so the four parameter gradients come from two column sums per sample.  A group of 1 to 32 warps owns a row; the row stays in registers between
// the sums (mean first, then the squares of the centred values: no cancellation) and A, T of the sample stay there from row to row.  All sums are
// fp32; results are rounded once.  Column sums go through registers, shared memory and one partial per CTA to a second kernel that adds
// them in a fixed order: the same bits from run to run.
#include "column_sums.cuh"
#include "common.cuh"

namespace llsa {

namespace {

using bf16 = __nv_bfloat16;

template <typename T, int VEC>
struct Pack;
template <>
struct Pack<bf16, 4> {
  using type = uint2;
  static __device__ __forceinline__ void unpack(uint2 r, float* v) {
    v[0] = bf16_lo(r.x); v[1] = bf16_hi(r.x); v[2] = bf16_lo(r.y); v[3] = bf16_hi(r.y);
  }
  static __device__ __forceinline__ uint2 pack(const float* v) { return make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])); }
};
template <>
struct Pack<float, 4> {
  using type = float4;
  static __device__ __forceinline__ void unpack(float4 r, float* v) { v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w; }
  static __device__ __forceinline__ float4 pack(const float* v) { return make_float4(v[0], v[1], v[2], v[3]); }
};
template <typename T>
struct Pack<T, 1> {
  using type = T;
  static __device__ __forceinline__ void unpack(T r, float* v) { v[0] = to_f32<T>(r); }
  static __device__ __forceinline__ T pack(const float* v) { return from_f32<T>(v[0]); }
};

// [B,N,C] tensor with unit channel stride
template <typename T>
struct Rows {
  T* p;
  int64_t sb, sn;
  __device__ __forceinline__ T* row(uint32_t b, uint32_t n) const { return p + b * sb + n * sn; }
};

// w, bias [C]; scale, shift [B, C] with a row stride of their own; each may be absent
struct NormParams {
  ParamView w, bias, scale, shift;
};

// The part of a row that one thread of a group of `threads` holds: R vectors of VEC channels, `threads` vectors apart
template <typename T, int VEC, int R>
struct Slice {
  using P = Pack<T, VEC>;
  typename P::type raw[R];
  __device__ __forceinline__ void load(const T* row, int t, int threads, int C) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int c = (i * threads + t) * VEC;
      if (c < C) raw[i] = *reinterpret_cast<const typename P::type*>(row + c);
    }
  }
  __device__ __forceinline__ void values(float (&v)[R * VEC], int t, int threads, int C) const {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      P::unpack(raw[i], v + i * VEC);
      if ((i * threads + t) * VEC >= C)
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i * VEC + j] = 0.f;
    }
  }
  static __device__ __forceinline__ void store(T* row, const float (&v)[R * VEC], int t, int threads, int C) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int c = (i * threads + t) * VEC;
      if (c < C) *reinterpret_cast<typename P::type*>(row + c) = P::pack(v + i * VEC);
    }
  }
};

// Sums of N values over a group: a warp, or `warps` warps of the CTA (then every thread of the CTA calls).  Two buffers in turn: a warp that
// is one sum ahead writes the other one, and it cannot be two ahead.
template <bool MULTI, int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float (*s_red)[32][2], int& turn, int warps) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  if constexpr (MULTI) {
    const int warp = threadIdx.x >> 5, first = warp / warps * warps;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) s_red[turn][warp][i] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0.f;
    for (int w = 0; w < warps; ++w)
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += s_red[turn][first + w][i];
    turn ^= 1;
  }
}

// TPB: threads of a CTA; MULTI: more than one warp to a row
template <typename T, int VEC, int R, bool MULTI, int TPB>
__global__ void __launch_bounds__(TPB)
layer_norm_fwd_kernel(Rows<const T> x, NormParams par, float eps, Rows<T> y, float2* __restrict__ stats, uint32_t M, uint32_t N, int C, int warps) {
  constexpr int E = R * VEC;
  __shared__ float s_red[2][32][2];
  const int threads = 32 * warps, group = threadIdx.x / threads, t = threadIdx.x - group * threads, groups = blockDim.x / threads;
  const float inv_c = 1.f / (float) C;
  int turn = 0;
  pdl_wait();
  pdl_trigger();
  float a[E], sh[E];
  uint32_t cur = ~0u;
  const uint64_t step = (uint64_t) gridDim.x * groups;
  Slice<T, VEC, R> next;
  uint64_t r = (uint64_t) blockIdx.x * groups + group;
  uint32_t b = 0, n = 0;
  if (r < M) {
    b = (uint32_t) r / N; n = (uint32_t) r - b * N;
    next.load(x.row(b, n), t, threads, C);
  }
  for (uint64_t base = (uint64_t) blockIdx.x * groups; base < M; base += step) {      // the same number of rounds for every group of the CTA
    const bool valid = r < M;
    const uint32_t rb = b, rn = n;
    float v[E];
    next.values(v, t, threads, C);
    if (r + step < M) {
      b = (uint32_t) (r + step) / N; n = (uint32_t) (r + step) - b * N;
      next.load(x.row(b, n), t, threads, C);
    }
    if (valid && rb != cur) {
      cur = rb;
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const int c = (i * threads + t) * VEC + j;
          if (c < C) {
            const float up = 1.f + par.scale.at(rb, c, 0.f);
            a[i * VEC + j] = par.w.at(0, c, 1.f) * up;
            sh[i * VEC + j] = fmaf(par.bias.at(0, c, 0.f), up, par.shift.at(rb, c, 0.f));
          }
        }
    }
    float s[1] = {0.f}, q[1] = {0.f};
#pragma unroll
    for (int i = 0; i < E; ++i) s[0] += v[i];
    group_sum<MULTI>(s, s_red, turn, warps);
    const float mean = s[0] * inv_c;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      v[i] -= mean;
      if (((i / VEC) * threads + t) * VEC < C) q[0] = fmaf(v[i], v[i], q[0]);
    }
    group_sum<MULTI>(q, s_red, turn, warps);
    const float rstd = rsqrtf(fmaf(q[0], inv_c, eps));
    if (valid) {
#pragma unroll
      for (int i = 0; i < E; ++i) v[i] = fmaf(v[i] * rstd, a[i], sh[i]);
      Slice<T, VEC, R>::store(y.row(rb, rn), v, t, threads, C);
      if (stats && t == 0) stats[r] = make_float2(mean, rstd);
    }
    r += step;
  }
}

// A CTA takes rows [s * per, (s + 1) * per) of sample b, chunk = b * chunks + s, and leaves its two column sums in partial[chunk][2][C].
template <typename T, int VEC, int R, bool MULTI, int TPB, bool SUMS>
__global__ void __launch_bounds__(TPB)
layer_norm_bwd_kernel(Rows<const T> dy, Rows<const T> x, NormParams par, const float2* __restrict__ stats, Rows<T> dx, float* __restrict__ partial,
                      uint32_t N, uint32_t chunks, uint32_t per, int C, int warps) {
  constexpr int E = R * VEC;
  __shared__ float s_red[2][32][2];
  __shared__ float s_col[SUMS ? 4096 : 1];
  const int threads = 32 * warps, group = threadIdx.x / threads, t = threadIdx.x - group * threads, groups = blockDim.x / threads;
  const float inv_c = 1.f / (float) C;
  const uint32_t b = blockIdx.x / chunks, first = (blockIdx.x - b * chunks) * per, end = min(N, first + per);
  int turn = 0;
  pdl_wait();
  pdl_trigger();
  float a[E], p[SUMS ? E : 1], sum[SUMS ? E : 1];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int c = (i * threads + t) * VEC + j;
      a[i * VEC + j] = c < C ? par.w.at(0, c, 1.f) * (1.f + par.scale.at(b, c, 0.f)) : 0.f;
      if constexpr (SUMS) p[i * VEC + j] = sum[i * VEC + j] = 0.f;
    }
  uint32_t n = first + group;
  Slice<T, VEC, R> nx, ng;
  float2 nst = make_float2(0.f, 0.f);
  if (n < end) {
    nx.load(x.row(b, n), t, threads, C);
    ng.load(dy.row(b, n), t, threads, C);
    nst = stats[(uint64_t) b * N + n];
  }
  for (uint32_t base = first; base < end; base += groups, n += groups) {
    const bool valid = n < end;
    float h[E], g[E];
    nx.values(h, t, threads, C);
    ng.values(g, t, threads, C);
    const float mean = nst.x, rstd = nst.y;
    if (n + groups < end) {
      nx.load(x.row(b, n + groups), t, threads, C);
      ng.load(dy.row(b, n + groups), t, threads, C);
      nst = stats[(uint64_t) b * N + n + groups];
    }
    float m[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < E; ++i) {
      h[i] = (h[i] - mean) * rstd;
      if constexpr (SUMS)
        if (valid) {
          p[i] = fmaf(g[i], h[i], p[i]);
          sum[i] += g[i];
        }
      g[i] *= a[i];
      m[0] += g[i];
      m[1] = fmaf(g[i], h[i], m[1]);
    }
    group_sum<MULTI>(m, s_red, turn, warps);
    m[0] *= inv_c;
    m[1] *= inv_c;
    if (valid) {
#pragma unroll
      for (int i = 0; i < E; ++i) g[i] = rstd * (g[i] - m[0] - h[i] * m[1]);
      Slice<T, VEC, R>::store(dx.row(b, n), g, t, threads, C);
    }
  }
  if constexpr (SUMS) {
    float* out = partial + (int64_t) blockIdx.x * 2 * C;
    if (groups == 1) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int c = ((i / VEC) * threads + t) * VEC + i % VEC;
        if (c < C) {
          out[c] = p[i];
          out[C + c] = sum[i];
        }
      }
    } else {
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < E; ++i) {
          const int c = ((i / VEC) * threads + t) * VEC + i % VEC;
          if (c < C) s_col[group * C + c] = which ? sum[i] : p[i];
        }
        __syncthreads();
        for (int c = threadIdx.x; c < C; c += blockDim.x) {
          float u = 0.f;
          for (int k = 0; k < groups; ++k) u += s_col[k * C + c];
          out[which * C + c] = u;
        }
      }
    }
  }
}

// Warps of a group and vectors of a thread: the fewest warps whose threads hold at most 16 channels each.
struct Split {
  int vec, r, warps, threads;
};
inline Split split_of(int64_t C, bool vec4) {
  Split s;
  s.vec = vec4 ? 4 : 1;
  s.warps = 1;
  while ((C + s.vec * 32 * s.warps - 1) / (s.vec * 32 * s.warps) * s.vec > 16) s.warps *= 2;
  s.r = (int) ((C + s.vec * 32 * s.warps - 1) / (s.vec * 32 * s.warps));
  if (!vec4) s.r = (s.r + 3) / 4 * 4;
  s.threads = s.warps > 8 ? 32 * s.warps : 256;
  return s;
}

template <typename T>
bool rows_vec4(const LlsaTensor* t) {
  const int64_t bytes = 4 * sizeof(T);
  return t->shape[2] % 4 == 0 && (uintptr_t) t->ptr % bytes == 0 && (t->shape[0] == 1 || t->stride[0] % 4 == 0) && (t->shape[1] == 1 || t->stride[1] % 4 == 0);
}
template <typename T>
Rows<T> make_rows(const LlsaTensor* t) {
  Rows<T> r;
  r.p = (T*) t->ptr;
  r.sb = t->stride[0];
  r.sn = t->stride[1];
  return r;
}

int check_rows(const LlsaTensor* t, const char* name, int dtype, const int64_t* shape) {
  LLSA_REQUIRE(t && t->ptr, LLSA_ERR_NULL, "%s: null tensor", name);
  LLSA_REQUIRE(t->dtype == dtype, LLSA_ERR_DTYPE, "%s: dtype %d, expected %d", name, t->dtype, dtype);
  LLSA_REQUIRE(t->ndim == 3 && t->shape[0] == shape[0] && t->shape[1] == shape[1] && t->shape[2] == shape[2], LLSA_ERR_SHAPE,
               "%s: must be [B,N,C] = [%lld,%lld,%lld]", name, (long long) shape[0], (long long) shape[1], (long long) shape[2]);
  LLSA_REQUIRE(shape[2] == 1 || t->stride[2] == 1, LLSA_ERR_STRIDE, "%s: innermost stride %lld, must be 1", name, (long long) t->stride[2]);
  return LLSA_OK;
}

// The input's sizes: [B,N,C], at most 2^31 - 1 rows of at most 16384 channels
int check_input(const LlsaTensor* x, const char* name) {
  LLSA_REQUIRE(x && x->ptr, LLSA_ERR_NULL, "%s: null tensor", name);
  LLSA_REQUIRE(is_float_dtype(x->dtype), LLSA_ERR_DTYPE, "%s: must be f32 or bf16", name);
  LLSA_REQUIRE(x->ndim == 3, LLSA_ERR_SHAPE, "%s: must be [B,N,C]", name);
  LLSA_REQUIRE(x->shape[2] >= 1 && x->shape[2] <= 16384, LLSA_ERR_SHAPE, "%s: %lld channels, supported are 1 to 16384", name, (long long) x->shape[2]);
  LLSA_REQUIRE(x->shape[0] * x->shape[1] <= INT32_MAX, LLSA_ERR_SHAPE, "%s: more than 2^31 - 1 rows", name);
  return check_rows(x, name, x->dtype, x->shape);
}

// Rows a CTA of the backward takes, and CTAs per sample.  Where nothing is summed over a sample, all rows are one sample.
struct Chunks {
  int64_t B, N, chunks, per;
};
Chunks chunks_of(int64_t B, int64_t N, int64_t C) {
  const Split s = split_of(C, C % 4 == 0);
  const int64_t groups = s.threads / (32 * s.warps), ctas = 148 * (s.threads > 256 ? 1 : 3);
  Chunks c;
  c.B = B;
  c.N = N;
  c.chunks = std::max<int64_t>(1, std::min((ctas + B - 1) / B, (N + 4 * groups - 1) / (4 * groups)));
  c.per = (N + c.chunks - 1) / c.chunks;
  c.per = (c.per + groups - 1) / groups * groups;
  c.chunks = (N + c.per - 1) / c.per;
  return c;
}

// The kernel for a split: rows of one warp, of several warps of 256 threads, or (above 4096 channels) of up to 1024 threads, whose threads hold 16 channels each.
#define LLSA_NORM_CASE(V_, R_, ...)                                                                 \
  if (sp.vec == V_ && sp.r <= R_) {                                                                 \
    constexpr int VEC = V_, R = R_;                                                                 \
    if (sp.warps == 1) { constexpr bool MULTI = false; constexpr int TPB = 256; __VA_ARGS__; }      \
    else { constexpr bool MULTI = true; constexpr int TPB = 256; __VA_ARGS__; }                     \
  }
#define LLSA_NORM_KERNEL(...)                                                                       \
  if (sp.threads > 256) {                                                                           \
    constexpr bool MULTI = true;                                                                    \
    constexpr int TPB = 1024;                                                                       \
    if (sp.vec == 4) { constexpr int VEC = 4, R = 4; __VA_ARGS__; }                                 \
    else { constexpr int VEC = 1, R = 16; __VA_ARGS__; }                                            \
  } else                                                                                            \
    LLSA_NORM_CASE(4, 1, __VA_ARGS__)                                                               \
  else LLSA_NORM_CASE(4, 2, __VA_ARGS__)                                                            \
  else LLSA_NORM_CASE(4, 3, __VA_ARGS__)                                                            \
  else LLSA_NORM_CASE(4, 4, __VA_ARGS__)                                                            \
  else LLSA_NORM_CASE(1, 4, __VA_ARGS__)                                                            \
  else LLSA_NORM_CASE(1, 8, __VA_ARGS__)                                                            \
  else LLSA_NORM_CASE(1, 12, __VA_ARGS__)                                                           \
  else LLSA_NORM_CASE(1, 16, __VA_ARGS__)

template <typename T>
int launch_fwd(const LlsaTensor* x, const NormParams& par, float eps, const LlsaTensor* y, float2* stats, cudaStream_t st) {
  const uint32_t M = (uint32_t) (x->shape[0] * x->shape[1]), N = (uint32_t) x->shape[1];
  const int C = (int) x->shape[2];
  const Split sp = split_of(C, rows_vec4<T>(x) && rows_vec4<T>(y));
  const int64_t groups = sp.threads / (32 * sp.warps);
  const int64_t grid = std::min<int64_t>((M + groups - 1) / groups, 148 * (sp.threads > 256 ? 2 : 4));
  const Rows<const T> xr = make_rows<const T>(x);
  const Rows<T> yr = make_rows<T>(y);
  LLSA_NORM_KERNEL(launch_pdl(layer_norm_fwd_kernel<T, VEC, R, MULTI, TPB>, dim3((unsigned) grid), dim3(sp.threads), 0, st, xr, par, eps, yr, stats, M, N, C,
                              sp.warps))
  LLSA_LAUNCH_OK("layer_norm_fwd_kernel");
  return LLSA_OK;
}

template <typename T, bool SUMS>
int launch_bwd(const LlsaTensor* dy, const LlsaTensor* x, const NormParams& par, const float2* stats, const LlsaTensor* dx, float* partial,
               const Chunks& ch, cudaStream_t st) {
  const int C = (int) x->shape[2];
  const Split sp = split_of(C, rows_vec4<T>(x) && rows_vec4<T>(dy) && rows_vec4<T>(dx));
  const Rows<const T> gr = make_rows<const T>(dy), xr = make_rows<const T>(x);
  const Rows<T> dr = make_rows<T>(dx);
  const unsigned grid = (unsigned) (ch.B * ch.chunks);
  LLSA_NORM_KERNEL(launch_pdl(layer_norm_bwd_kernel<T, VEC, R, MULTI, TPB, SUMS>, dim3(grid), dim3(sp.threads), 0, st, gr, xr, par, stats, dr, partial,
                              (uint32_t) ch.N, (uint32_t) ch.chunks, (uint32_t) ch.per, C, sp.warps))
  LLSA_LAUNCH_OK("layer_norm_bwd_kernel");
  return LLSA_OK;
}

int params_of(NormParams* par, const LlsaTensor* x, const LlsaTensor* weight, const LlsaTensor* bias, const LlsaTensor* scale, const LlsaTensor* shift) {
  const int64_t B = x->shape[0], C = x->shape[2];
  int rc;
  if ((rc = make_param(&par->w, weight, "weight", x->dtype, 0, C))) return rc;
  if ((rc = make_param(&par->bias, bias, "bias", x->dtype, 0, C))) return rc;
  if ((rc = make_param(&par->scale, scale, "scale", x->dtype, B, C))) return rc;
  return make_param(&par->shift, shift, "shift", x->dtype, B, C);
}

}  // namespace
}  // namespace llsa

using namespace llsa;

extern "C" int llsa_layer_norm_fwd(const LlsaTensor* x, const LlsaTensor* weight, const LlsaTensor* bias, const LlsaTensor* scale,
                                   const LlsaTensor* shift, float eps, const LlsaTensor* y, const LlsaTensor* stats, void* stream) {
  int rc = check_input(x, "x");
  if (rc) return rc;
  if ((rc = check_rows(y, "y", x->dtype, x->shape))) return rc;
  NormParams par;
  if ((rc = params_of(&par, x, weight, bias, scale, shift))) return rc;
  const int64_t shape[3] = {x->shape[0], x->shape[1], 2};
  if (stats && (rc = check_contig(stats, "stats", LLSA_F32, 3, shape))) return rc;
  LLSA_REQUIRE(eps >= 0.f, LLSA_ERR_ARG, "layer_norm: eps %g is negative or not a number", (double) eps);
  if (shape[0] * shape[1] == 0) return LLSA_OK;
  float2* st = stats ? (float2*) stats->ptr : nullptr;
  return x->dtype == LLSA_F32 ? launch_fwd<float>(x, par, eps, y, st, (cudaStream_t) stream)
                              : launch_fwd<__nv_bfloat16>(x, par, eps, y, st, (cudaStream_t) stream);
}

extern "C" int64_t llsa_layer_norm_bwd_partial_elems(int64_t B, int64_t N, int64_t C, int per_sample) {
  if (B <= 0 || N <= 0 || C <= 0 || C > 16384) return 0;
  const Chunks c = chunks_of(per_sample ? B : 1, per_sample ? N : B * N, C);
  return c.B * c.chunks * 2 * C;
}

extern "C" int llsa_layer_norm_bwd(const LlsaTensor* dy, const LlsaTensor* x, const LlsaTensor* weight, const LlsaTensor* bias,
                                   const LlsaTensor* scale, const LlsaTensor* stats, const LlsaTensor* dx, const LlsaTensor* dweight,
                                   const LlsaTensor* dbias, const LlsaTensor* dscale, const LlsaTensor* dshift, const LlsaTensor* partial,
                                   void* stream) {
  int rc = check_input(x, "x");
  if (rc) return rc;
  if ((rc = check_rows(dy, "dy", x->dtype, x->shape)) || (rc = check_rows(dx, "dx", x->dtype, x->shape))) return rc;
  const int64_t B = x->shape[0], N = x->shape[1], C = x->shape[2];
  NormParams par;
  if ((rc = params_of(&par, x, weight, bias, scale, nullptr))) return rc;
  const int64_t shape[3] = {B, N, 2};
  if ((rc = check_contig(stats, "stats", LLSA_F32, 3, shape))) return rc;
  const bool sums = dweight || dbias || dscale || dshift;
  const LlsaTensor* const vecs[2] = {dweight, dbias};
  const LlsaTensor* const mats[2] = {dscale, dshift};
  const char* const vname[2] = {"dweight", "dbias"};
  const char* const mname[2] = {"dscale", "dshift"};
  const int64_t vs[1] = {C}, ms[2] = {B, C};
  for (int i = 0; i < 2; ++i) {
    if (vecs[i] && (rc = check_grad(vecs[i], vname[i], x->dtype, 1, vs))) return rc;
    if (mats[i] && (rc = check_grad(mats[i], mname[i], x->dtype, 2, ms))) return rc;
  }
  // the rows of a sample are summed apart where its modulation has a gradient, or weighs the rest
  const bool per_sample = scale || dshift;
  if (sums) {
    LLSA_REQUIRE(partial && partial->ptr, LLSA_ERR_NULL, "partial: null tensor");
    LLSA_REQUIRE(partial->dtype == LLSA_F32 && partial->ndim == 1 && is_contiguous(partial) &&
                     partial->shape[0] >= llsa_layer_norm_bwd_partial_elems(B, N, C, per_sample),
                 LLSA_ERR_WORKSPACE, "partial: must be f32 and hold llsa_layer_norm_bwd_partial_elems() elements");
  }
  const ColumnGrads grads = {make_grad(dscale), make_grad(dshift), make_grad(dweight), make_grad(dbias)};
  if (B * N == 0) return sums ? clear_column_grads(grads, B, C, (cudaStream_t) stream) : LLSA_OK;
  const Chunks ch = chunks_of(per_sample ? B : 1, per_sample ? N : B * N, C);
  LLSA_REQUIRE(ch.B * ch.chunks <= INT32_MAX, LLSA_ERR_SHAPE, "layer_norm_bwd: too many samples");
  // one sample of all rows: needs rows that follow one another
  LlsaTensor f[3] = {*dy, *x, *dx};
  if (!per_sample && B > 1)
    for (LlsaTensor& t : f) {
      LLSA_REQUIRE(N == 1 || t.stride[0] == N * t.stride[1], LLSA_ERR_STRIDE, "layer_norm_bwd: samples must follow one another where nothing is per sample");
      if (N == 1) t.stride[1] = t.stride[0];
      t.shape[1] = B * N;
      t.shape[0] = 1;
    }
  float* part = sums ? (float*) partial->ptr : nullptr;
  const float2* sv = (const float2*) stats->ptr;
  const cudaStream_t st = (cudaStream_t) stream;
  if (x->dtype == LLSA_F32)
    rc = sums ? launch_bwd<float, true>(&f[0], &f[1], par, sv, &f[2], part, ch, st) : launch_bwd<float, false>(&f[0], &f[1], par, sv, &f[2], part, ch, st);
  else
    rc = sums ? launch_bwd<__nv_bfloat16, true>(&f[0], &f[1], par, sv, &f[2], part, ch, st)
              : launch_bwd<__nv_bfloat16, false>(&f[0], &f[1], par, sv, &f[2], part, ch, st);
  if (rc || !sums) return rc;
  return finish_column_grads(part, ch.B, ch.chunks, C, par.w, par.bias, par.scale, grads, st);
}
