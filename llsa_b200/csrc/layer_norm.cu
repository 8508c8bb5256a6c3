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
// Reading and writing the rows once each is what there is to do; what costs beside it is a row's chain of sums and the instructions around it, some 200 a
// warp, so the pairs of values share instructions, a row is on its way while another is worked on, and enough warps fit an SM.
#include "column_sums.cuh"
#include "common.cuh"
#include "vec.cuh"

namespace llsa {

namespace {

using bf16 = __nv_bfloat16;

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

// The part of a row that one thread of a group of `threads` holds: R vectors of VEC channels, `threads` vectors apart.
//   kWhole   vectors of four on their boundaries; R is no larger than C asks for, and only the last one may lie behind the row's end
//   kLoose   the same, with any of them behind the end
//   kShifted rows of any length, whose vectors of four begin `m` channels in front of the row, on their boundary; those over the row's ends go element by element.
//            R is no larger than C + 3 asks for: only the first vector begins in front of the row, only the last two may lie behind its end
//   kSingle  element by element
enum Form { kWhole, kLoose, kShifted, kSingle };
template <typename T, int FORM, int R>
struct Slice {
  static constexpr int VEC = FORM == kSingle ? 1 : 4, E = R * VEC;
  using P = Vec<T, VEC>;
  typename P::type raw[R];
  static __device__ __forceinline__ int channel(int e, int t, int threads, int m) { return ((e / VEC) * threads + t) * VEC + e % VEC - (FORM == kShifted ? m : 0); }
  static __device__ __forceinline__ bool there(int e, int c, int C) {
    if (FORM == kWhole) return e / VEC < R - 1 || c < C;
    if (FORM == kShifted) return (e / VEC > 0 || c >= 0) && (e / VEC < R - 2 || c < C);
    return c < C;
  }
  // All of a shifted vector
  static __device__ __forceinline__ bool all_there(int i, int c, int C) { return (i > 0 || c >= 0) && (i < R - 2 || c + VEC <= C); }
  __device__ __forceinline__ void load(const T* row, int t, int threads, int C, int m) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int c = channel(i * VEC, t, threads, m);
      if (FORM != kShifted ? there(i * VEC, c, C) : all_there(i, c, C)) {
        raw[i] = *reinterpret_cast<const typename P::type*>(row + c);
      } else if (FORM == kShifted) {
        T* u = reinterpret_cast<T*>(&raw[i]);
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (there(i * VEC + j, c + j, C)) u[j] = row[c + j];
      }
    }
  }
  // The values in pairs, for instructions that take two; zeros where there is none
  __device__ __forceinline__ void values(float2 (&v)[E / 2], int t, int threads, int C, int m) const {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      float u[VEC];
      P::unpack(raw[i], u);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int e = i * VEC + j;
        const float x = there(e, channel(e, t, threads, m), C) ? u[j] : 0.f;
        if (e & 1) v[e / 2].y = x;
        else v[e / 2].x = x;
      }
    }
  }
  static __device__ __forceinline__ void store(T* row, const float2 (&v)[E / 2], int t, int threads, int C, int m) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int c = channel(i * VEC, t, threads, m);
      const typename P::type w = P::pack(reinterpret_cast<const float*>(v) + i * VEC);
      if (FORM != kShifted ? there(i * VEC, c, C) : all_there(i, c, C)) {
        *reinterpret_cast<typename P::type*>(row + c) = w;
      } else if (FORM == kShifted) {
        const T* u = reinterpret_cast<const T*>(&w);
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (there(i * VEC + j, c + j, C)) row[c + j] = u[j];
      }
    }
  }
};
// A parameter's part beside a slice; `absent` where it or the channel is not there.  One look at its type, not one for every channel
template <typename S>
__device__ __forceinline__ void load_param(float (&v)[S::E], const ParamView& p, uint32_t b, float absent, int t, int threads, int C, int m) {
  if (p.p && p.is_bf16) {
    const bf16* row = reinterpret_cast<const bf16*>(p.p) + b * p.ld;
#pragma unroll
    for (int e = 0; e < S::E; ++e) {
      const int c = S::channel(e, t, threads, m);
      v[e] = S::there(e, c, C) ? __bfloat162float(row[c]) : absent;
    }
  } else if (p.p) {
    const float* row = reinterpret_cast<const float*>(p.p) + b * p.ld;
#pragma unroll
    for (int e = 0; e < S::E; ++e) {
      const int c = S::channel(e, t, threads, m);
      v[e] = S::there(e, c, C) ? row[c] : absent;
    }
  } else {
#pragma unroll
    for (int e = 0; e < S::E; ++e) v[e] = absent;
  }
}
// Four channels of one, of which those of a shifted vector are there or not one by one
template <int FORM>
__device__ __forceinline__ void load_param4(float (&v)[4], const ParamView& p, uint32_t b, float absent, int c, int C) {
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = absent;
  if (!p.p || c >= C) return;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (FORM == kWhole || (unsigned) (c + j) < (unsigned) C)
      v[j] = p.is_bf16 ? __bfloat162float(reinterpret_cast<const bf16*>(p.p)[b * p.ld + c + j]) : reinterpret_cast<const float*>(p.p)[b * p.ld + c + j];
}
template <typename T>
__device__ __forceinline__ int shift_of(const T* row) { return (int) ((uintptr_t) row / sizeof(T) & 3); }

// Sums of N values over a group: a warp, or `warps` warps of the CTA that meet at a barrier of their own.  Two buffers in turn: a warp that is one sum
// ahead writes the other one, and it cannot be two ahead.
template <bool MULTI, int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float (*s_red)[32][2], int& turn, int warps, int group) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  if constexpr (MULTI) {
    const int warp = threadIdx.x >> 5, first = group * warps;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) s_red[turn][warp][i] = v[i];
    asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(32 * warps) : "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0.f;
    for (int w = 0; w < warps; ++w)
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += s_red[turn][first + w][i];
    turn ^= 1;
  }
}

// CTAs that an SM should hold, by threads, by values of a thread and their type: registers are what decides (fp32, 12 values: four CTAs 75 us, three 71.5;
// shifted, 16 values: bf16 three 87.5 us, two 100, fp32 49.5 and 45.6; 20 values: fp32 44 and 34)
constexpr int fwd_ctas(int tpb, int form, int e, int bytes) {
  return tpb > 256 ? 1 : form == kWhole ? (bytes == 2 || e <= 8 ? 4 : 3) : form == kShifted ? (e <= 8 ? 4 : e > 16 ? 2 : bytes == 2 ? 3 : 2) : e <= 12 ? 4 : 3;
}
constexpr int bwd_ctas(int tpb) { return tpb > 256 ? 1 : 2; }

// TPB: threads of a CTA; MULTI: more than one warp to a row.  A CTA takes rows [blockIdx.x * per, + per): neighbours, so that a group's sample, and with it A and
// T, changes rarely.  (Rows a grid apart had them loaded for nearly every row: 8 x 16384 rows of 384 channels 77 us, 44 so.)
// Measured (bf16 unless said): 8 x 16384 rows of 384 channels 39.6 us (5.1 TB/s), in fp32 71.5 (5.6); 8 x 16384 of 768 92.7; 2 x 8192 of 2048 35.6; with A and T
// in registers, which spill, 43.6, 81.7, 105 and 40.6.  Shifted, 8 x 16384 rows of 390: 75 (every vector looked at 94); 4 x 4096 of 770: 26 (31).  Two rows on
// their way are worth 1 us of the first and cost 12 of the 768 channels' 93.
template <typename T, int FORM, int R, bool MULTI, int TPB>
__global__ void __launch_bounds__(TPB, fwd_ctas(TPB, FORM, R * (FORM == kSingle ? 1 : 4), sizeof(T)))
layer_norm_fwd_kernel(Rows<const T> x, NormParams par, float eps, Rows<T> y, float2* __restrict__ stats, uint32_t M, uint32_t N, uint32_t per, int C, int warps) {
  using S = Slice<T, FORM, R>;
  constexpr int E = S::E;
  // vectors: A and T lie in shared memory, each thread's own, and leave their registers to the rows (512 threads have the registers, and would need more than
  // 48 KB); rows of one warp have two on their way
  constexpr bool KEEP = FORM == kWhole || (FORM == kShifted && TPB == 256);
  constexpr int DEPTH = FORM == kWhole && R <= 3 && !MULTI && sizeof(T) == 2 ? 2 : 1;
  __shared__ float s_red[2][32][2];
  __shared__ float4 s_par[KEEP ? 2 * R * TPB : 1];
  const int threads = MULTI ? 32 * warps : 32, group = threadIdx.x / threads, t = threadIdx.x - group * threads, groups = TPB / threads;
  const float inv_c = 1.f / (float) C;
  const uint32_t end = min(M, (blockIdx.x + 1) * per);
  int turn = 0, m = 0;
  pdl_wait();
  pdl_trigger();
  float2 a[E / 2], sh[E / 2];
  uint32_t cur = ~0u, r = blockIdx.x * per + group, b = r / N, n = r - b * N;
  S raw[DEPTH];
  uint32_t sb[DEPTH], sn[DEPTH];                               // whose they are
  const auto fetch = [&](int d) {                              // the next row into place d
    sb[d] = b, sn[d] = n;
    if (r < end) raw[d].load(x.row(b, n), t, threads, C, m);
    r += groups;
    n += groups;
    if (n >= N) {
      const uint32_t q = n / N;
      b += q;
      n -= q * N;
    }
  };
  if (FORM == kShifted && r < end) m = shift_of(x.row(b, n));  // of all the group's rows: they are a multiple of four apart
  const uint32_t mine = r < end ? (end - r + groups - 1) / groups : 0;
#pragma unroll
  for (int d = 0; d < DEPTH; ++d) fetch(d);
  for (uint32_t i0 = 0; i0 < mine; i0 += DEPTH) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      if (d && i0 + d >= mine) break;
      const uint32_t rb = sb[d], rn = sn[d];
      float2 v[E / 2];
      raw[d].values(v, t, threads, C, m);
      fetch(d);
      if (rb != cur) {
        cur = rb;
        if constexpr (KEEP) {
#pragma unroll 1
          for (int i = 0; i < R; ++i) {
            const int c = S::channel(4 * i, t, threads, m);
            float u[4], w[4], bias[4], shift[4];
            load_param4<FORM>(u, par.scale, rb, 0.f, c, C);
            load_param4<FORM>(w, par.w, 0, 1.f, c, C);
            load_param4<FORM>(bias, par.bias, 0, 0.f, c, C);
            load_param4<FORM>(shift, par.shift, rb, 0.f, c, C);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              w[j] *= 1.f + u[j];
              bias[j] = fmaf(bias[j], 1.f + u[j], shift[j]);
            }
            s_par[2 * i * TPB + threadIdx.x] = make_float4(w[0], w[1], w[2], w[3]);
            s_par[(2 * i + 1) * TPB + threadIdx.x] = make_float4(bias[0], bias[1], bias[2], bias[3]);
          }
        } else {
          float u[E], w[E];
          load_param<S>(u, par.scale, rb, 0.f, t, threads, C, m);
          load_param<S>(w, par.w, 0, 1.f, t, threads, C, m);
#pragma unroll
          for (int e = 0; e < E; ++e) reinterpret_cast<float*>(a)[e] = w[e] * (1.f + u[e]);
          load_param<S>(w, par.bias, 0, 0.f, t, threads, C, m);
#pragma unroll
          for (int e = 0; e < E; ++e) reinterpret_cast<float*>(sh)[e] = w[e] * (1.f + u[e]);
          load_param<S>(u, par.shift, rb, 0.f, t, threads, C, m);
#pragma unroll
          for (int e = 0; e < E; ++e) reinterpret_cast<float*>(sh)[e] += u[e];
        }
      }
      float2 s2 = v[0];
#pragma unroll
      for (int i = 1; i < E / 2; ++i) s2 = __fadd2_rn(s2, v[i]);
      float s[1] = {s2.x + s2.y};
      group_sum<MULTI>(s, s_red, turn, warps, group);
      const float mean = s[0] * inv_c;
      float2 q2 = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < E / 2; ++i) {
        v[i] = __fadd2_rn(v[i], make_float2(-mean, -mean));
        float2 u = v[i];                                         // what is not there stays out of the squares
        if (!S::there(2 * i, S::channel(2 * i, t, threads, m), C)) u.x = 0.f;
        if (!S::there(2 * i + 1, S::channel(2 * i + 1, t, threads, m), C)) u.y = 0.f;
        q2 = __ffma2_rn(u, u, q2);
      }
      float q[1] = {q2.x + q2.y};
      group_sum<MULTI>(q, s_red, turn, warps, group);
      const float rstd = rsqrtf(fmaf(q[0], inv_c, eps));
#pragma unroll
      for (int i = 0; i < E / 2; ++i) {
        float2 ai = a[i], ti = sh[i];
        if constexpr (KEEP) {
          const float4 pa = s_par[i / 2 * 2 * TPB + threadIdx.x], pt = s_par[(i / 2 * 2 + 1) * TPB + threadIdx.x];
          ai = i & 1 ? make_float2(pa.z, pa.w) : make_float2(pa.x, pa.y);
          ti = i & 1 ? make_float2(pt.z, pt.w) : make_float2(pt.x, pt.y);
        }
        v[i] = __ffma2_rn(__fmul2_rn(v[i], make_float2(rstd, rstd)), ai, ti);
      }
      S::store(y.row(rb, rn), v, t, threads, C, m);
      if (stats && t == 0) stats[(uint64_t) rb * N + rn] = make_float2(mean, rstd);
    }
  }
}

// A CTA takes rows [s * per, (s + 1) * per) of sample b, chunk = b * chunks + s, and leaves its two column sums in partial[chunk][2][C] (NULL: none are wanted).
// Of shifted rows every group holds other channels in a thread than its neighbour: the sums meet by channel in shared memory.
// Measured, the parameters' gradients included (bf16 unless said): 8 x 16384 rows of 384 channels 58.4 us (5.2 TB/s), in fp32 99.6 (6.1); 8 x 16384 of 768 123.6;
// 2 x 8192 of 2048 53.5; shifted, 3 x 5377 of 1155 in fp32 56, 8 x 16384 of 390 122.  With one row on its way instead of two 68.3 and 131.5 (384 and 768); of 16 values to a
// thread, or of fp32, two rows spill (2048: 84.7, fp32 115).
template <typename T, int FORM, int R, bool MULTI, int TPB>
__global__ void __launch_bounds__(TPB, bwd_ctas(TPB))
layer_norm_bwd_kernel(Rows<const T> dy, Rows<const T> x, NormParams par, const float2* __restrict__ stats, Rows<T> dx, float* __restrict__ partial,
                      uint32_t N, uint32_t chunks, uint32_t per, int C, int warps) {
  using S = Slice<T, FORM, R>;
  constexpr int E = S::E;
  constexpr int DEPTH = FORM == kWhole && R <= 3 && sizeof(T) == 2 ? 2 : 1;       // rows on their way
  __shared__ float s_red[2][32][2];
  __shared__ float s_col[TPB > 512 ? 1 : 16 * TPB];
  const int threads = MULTI ? 32 * warps : 32, group = threadIdx.x / threads, t = threadIdx.x - group * threads, groups = TPB / threads;
  const float inv_c = 1.f / (float) C;
  const uint32_t b = blockIdx.x / chunks, first = (blockIdx.x - b * chunks) * per, end = min(N, first + per);
  int turn = 0, m = 0;
  pdl_wait();
  pdl_trigger();
  float2 a[E / 2], p[E / 2], sum[E / 2];
  uint32_t n = first + group;
  if (FORM == kShifted) m = shift_of(x.row(b, n));
  {
    float u[E], w[E];
    load_param<S>(u, par.scale, b, 0.f, t, threads, C, m);
    load_param<S>(w, par.w, 0, 1.f, t, threads, C, m);
#pragma unroll
    for (int e = 0; e < E; ++e) reinterpret_cast<float*>(a)[e] = S::there(e, S::channel(e, t, threads, m), C) ? w[e] * (1.f + u[e]) : 0.f;
  }
#pragma unroll
  for (int i = 0; i < E / 2; ++i) p[i] = sum[i] = make_float2(0.f, 0.f);
  S rx[DEPTH], rg[DEPTH];
  float2 rst[DEPTH];
  uint32_t ahead = n;
  const auto fetch = [&](int d) {                              // the next row into place d
    if (ahead < end) {
      rx[d].load(x.row(b, ahead), t, threads, C, m);
      rg[d].load(dy.row(b, ahead), t, threads, C, m);
      rst[d] = stats[(uint64_t) b * N + ahead];
    }
    ahead += groups;
  };
#pragma unroll
  for (int d = 0; d < DEPTH; ++d) fetch(d);
  while (n < end) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      if (d && n >= end) break;
      const uint32_t rn = n;
      const float2 rs = rst[d];
      float2 h[E / 2], g[E / 2];
      rx[d].values(h, t, threads, C, m);
      rg[d].values(g, t, threads, C, m);
      const float2 minus = make_float2(-rs.x, -rs.x), r2 = make_float2(rs.y, rs.y);
      n += groups;
      fetch(d);
      float2 m1 = make_float2(0.f, 0.f), m2 = m1;
#pragma unroll
      for (int i = 0; i < E / 2; ++i) {
        h[i] = __fmul2_rn(__fadd2_rn(h[i], minus), r2);
        p[i] = __ffma2_rn(g[i], h[i], p[i]);
        sum[i] = __fadd2_rn(sum[i], g[i]);
        g[i] = __fmul2_rn(g[i], a[i]);                           // 0 where nothing is there
        m1 = __fadd2_rn(m1, g[i]);
        m2 = __ffma2_rn(g[i], h[i], m2);
      }
      float s[2] = {m1.x + m1.y, m2.x + m2.y};
      group_sum<MULTI>(s, s_red, turn, warps, group);
      const float2 k1 = make_float2(-s[0] * inv_c, -s[0] * inv_c), k2 = make_float2(-s[1] * inv_c, -s[1] * inv_c);
#pragma unroll
      for (int i = 0; i < E / 2; ++i) g[i] = __fmul2_rn(r2, __ffma2_rn(h[i], k2, __fadd2_rn(g[i], k1)));
      S::store(dx.row(b, rn), g, t, threads, C, m);
    }
  }
  if (!partial) return;
  float* out = partial + (int64_t) blockIdx.x * 2 * C;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const float* mine = reinterpret_cast<const float*>(which ? sum : p);
    if (TPB > 512 || groups == 1) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int c = S::channel(e, t, threads, m);
        if (S::there(e, c, C)) out[which * C + c] = mine[e];
      }
    } else {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int c = S::channel(e, t, threads, m);
        if (S::there(e, c, C)) s_col[group * C + c] = mine[e];
      }
      __syncthreads();
      for (int c = threadIdx.x; c < C; c += TPB) {
        float u = 0.f;
        for (int k = 0; k < groups; ++k) u += s_col[k * C + c];
        out[which * C + c] = u;
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ choice of the kernel
// The fewest warps to a row whose threads hold at most 16 channels each, but for one case.
struct Split {
  int form, r, warps, threads;
};
// whole: rows on the boundaries of their vectors; alike: all of a call's rows begin equally far behind one, and four rows on again
Split split_of(int64_t C, bool whole, bool alike, bool fwd) {
  Split s;
  s.form = whole ? kWhole : alike && C + 3 <= 2048 ? kShifted : kSingle;
  const int64_t vec = s.form == kSingle ? 1 : 4, span = C + (s.form == kShifted ? 3 : 0);
  s.warps = 1;
  while ((span + vec * 32 * s.warps - 1) / (vec * 32 * s.warps) * vec > 16) s.warps *= 2;
  s.r = (int) ((span + vec * 32 * s.warps - 1) / (vec * 32 * s.warps));
  // rows a multiple of four apart begin alike: four groups at least
  s.threads = s.form == kShifted && s.warps == 4 ? 512 : 256;
  // forward: two warps, with 20 values a thread, have two CTAs to an SM where four warps of 512 threads have one.  They hold up to 1277 channels behind the boundary.
  // us, two warps / four, 16384 rows in fp32, 32768 in bf16: 1029 channels 30.8 / 41.2, 60.9 / 98.7; 1155 32.0 / 41.0, 59.5 / 93.6; 1277 33.6 / 41.0, 60.4 / 95.0; four
  // warps take 41.2 and 93.8 for 1281, which two do not hold.  (Backward: bf16 63 / 69, fp32 78 / 56 at 3 x 5377 x 1155.)
  if (fwd && s.threads == 512 && span <= 1280) {
    s.warps = 2;
    s.r = 5;
    s.threads = 256;
  }
  if (s.warps > 8) {
    s.threads = 1024;
    s.warps = 32;
    if (s.form == kWhole) s.form = kLoose;
  }
  return s;
}
template <typename T, typename... Ts>
Split split_for(bool fwd, const LlsaTensor* x, Ts... others) {
  const LlsaTensor* const t[] = {x, others...};
  const int64_t es = sizeof(T);
  bool whole = true, alike = true;
  for (const LlsaTensor* u : t) {
    const int64_t sb = u->shape[0] == 1 ? 0 : u->stride[0], sn = u->shape[1] == 1 ? 0 : u->stride[1];
    whole = whole && u->shape[2] % 4 == 0 && (uintptr_t) u->ptr % (4 * es) == 0 && sb % 4 == 0 && sn % 4 == 0;
    const int64_t sn0 = x->shape[1] == 1 ? 0 : x->stride[1], sb0 = x->shape[0] == 1 ? 0 : x->stride[0];
    alike = alike && ((uintptr_t) u->ptr / es) % 4 == ((uintptr_t) x->ptr / es) % 4 && sn % 4 == sn0 % 4 && sb % 4 == sb0 % 4 &&
            (x->shape[0] == 1 || sb % 4 == (x->shape[1] * u->stride[1]) % 4) && (x->shape[1] > 1 || sb % 4 == u->stride[1] % 4);
  }
  return split_of(x->shape[2], whole, alike, fwd);
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
  const int64_t ctas = 148 * (C > 4096 ? 1 : 2);               // what the SMs hold at once
  Chunks c;
  c.B = B;
  c.N = N;
  c.chunks = std::max<int64_t>(1, std::min((ctas + B - 1) / B, (N + 15) / 16));
  c.per = ((N + c.chunks - 1) / c.chunks + 7) / 8 * 8;
  c.chunks = (N + c.per - 1) / c.per;
  return c;
}

// The kernel for a split.  Rows of one warp; of several warps of 256 threads; of 512, which has four groups of four; of all of 1024, above 4096 channels.
#define LLSA_NORM_R(F_, R_, W_, T_, ...)                                                                        \
  if (sp.form == F_ && (F_ == kWhole || F_ == kShifted ? sp.r == R_ : sp.r <= R_) && (sp.warps > 1) == W_ && sp.threads == T_) { \
    constexpr int FORM = F_, R = R_, TPB = T_;                                                                  \
    constexpr bool MULTI = W_;                                                                                  \
    __VA_ARGS__;                                                                                                \
  }
#define LLSA_NORM_KERNEL(...)                                                                                   \
  LLSA_NORM_R(kWhole, 1, false, 256, __VA_ARGS__)                                                               \
  else LLSA_NORM_R(kWhole, 2, false, 256, __VA_ARGS__)                                                          \
  else LLSA_NORM_R(kWhole, 3, false, 256, __VA_ARGS__)                                                          \
  else LLSA_NORM_R(kWhole, 4, false, 256, __VA_ARGS__)                                                          \
  else LLSA_NORM_R(kWhole, 3, true, 256, __VA_ARGS__)                                                           \
  else LLSA_NORM_R(kWhole, 4, true, 256, __VA_ARGS__)                                                           \
  else LLSA_NORM_R(kLoose, 4, true, 1024, __VA_ARGS__)                                                          \
  else LLSA_NORM_R(kShifted, 1, false, 256, __VA_ARGS__)                                                        \
  else LLSA_NORM_R(kShifted, 2, false, 256, __VA_ARGS__)                                                        \
  else LLSA_NORM_R(kShifted, 3, false, 256, __VA_ARGS__)                                                        \
  else LLSA_NORM_R(kShifted, 4, false, 256, __VA_ARGS__)                                                        \
  else LLSA_NORM_R(kShifted, 3, true, 256, __VA_ARGS__)                                                         \
  else LLSA_NORM_R(kShifted, 4, true, 256, __VA_ARGS__)                                                         \
  else LLSA_NORM_R(kShifted, 5, true, 256, __VA_ARGS__)                                                         \
  else LLSA_NORM_R(kShifted, 3, true, 512, __VA_ARGS__)                                                         \
  else LLSA_NORM_R(kShifted, 4, true, 512, __VA_ARGS__)                                                         \
  else LLSA_NORM_R(kSingle, 16, false, 256, __VA_ARGS__)                                                        \
  else LLSA_NORM_R(kSingle, 16, true, 256, __VA_ARGS__)                                                         \
  else LLSA_NORM_R(kSingle, 16, true, 1024, __VA_ARGS__)                                                        \
  else LLSA_REQUIRE(false, LLSA_ERR_SHAPE, "layer_norm: no kernel for %d channels", C);

// Rows that follow one another as one sample: where nothing is per sample, A and T are loaded once
bool flatten(LlsaTensor* t) {
  const int64_t B = t->shape[0], N = t->shape[1];
  if (B > 1 && N > 1 && t->stride[0] != N * t->stride[1]) return false;
  if (N == 1) t->stride[1] = t->stride[0];
  t->shape[0] = 1;
  t->shape[1] = B * N;
  return true;
}

template <typename T>
int launch_fwd(const LlsaTensor* x, const NormParams& par, float eps, const LlsaTensor* y, float2* stats, cudaStream_t st) {
  const uint32_t M = (uint32_t) (x->shape[0] * x->shape[1]), N = (uint32_t) x->shape[1];
  const int C = (int) x->shape[2];
  const Split sp = split_for<T>(true, x, y);
  const int64_t groups = sp.threads / (32 * sp.warps);
  const Rows<const T> xr = make_rows<const T>(x);
  const Rows<T> yr = make_rows<T>(y);
  LLSA_NORM_KERNEL({
    // as many CTAs as the SMs hold at once, an equal share of rows each
    const int64_t most = 148 * fwd_ctas(TPB, FORM, R * (FORM == kSingle ? 1 : 4), sizeof(T)), per = ((M + most - 1) / most + groups - 1) / groups * groups, grid = (M + per - 1) / per;
    launch_pdl(layer_norm_fwd_kernel<T, FORM, R, MULTI, TPB>, dim3((unsigned) grid), dim3(TPB), 0, st, xr, par, eps, yr, stats, M, N, (uint32_t) per, C, sp.warps);
  })
  LLSA_LAUNCH_OK("layer_norm_fwd_kernel");
  return LLSA_OK;
}

template <typename T>
int launch_bwd(const LlsaTensor* dy, const LlsaTensor* x, const NormParams& par, const float2* stats, const LlsaTensor* dx, float* partial,
               const Chunks& ch, cudaStream_t st) {
  const int C = (int) x->shape[2];
  const Split sp = split_for<T>(false, x, dy, dx);
  const Rows<const T> gr = make_rows<const T>(dy), xr = make_rows<const T>(x);
  const Rows<T> dr = make_rows<T>(dx);
  const unsigned grid = (unsigned) (ch.B * ch.chunks);
  LLSA_NORM_KERNEL(launch_pdl(layer_norm_bwd_kernel<T, FORM, R, MULTI, TPB>, dim3(grid), dim3(TPB), 0, st, gr, xr, par, stats, dr, partial, (uint32_t) ch.N,
                              (uint32_t) ch.chunks, (uint32_t) ch.per, C, sp.warps))
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
  LlsaTensor fx = *x, fy = *y;
  if (!scale && !shift && flatten(&fx) && flatten(&fy)) x = &fx, y = &fy;
  return x->dtype == LLSA_F32 ? launch_fwd<float>(x, par, eps, y, st, (cudaStream_t) stream)
                              : launch_fwd<bf16>(x, par, eps, y, st, (cudaStream_t) stream);
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
    for (LlsaTensor& t : f)
      LLSA_REQUIRE(flatten(&t), LLSA_ERR_STRIDE, "layer_norm_bwd: samples must follow one another where nothing is per sample");
  float* part = sums ? (float*) partial->ptr : nullptr;
  const float2* sv = (const float2*) stats->ptr;
  const cudaStream_t st = (cudaStream_t) stream;
  if (x->dtype == LLSA_F32)
    rc = launch_bwd<float>(&f[0], &f[1], par, sv, &f[2], part, ch, st);
  else
    rc = launch_bwd<bf16>(&f[0], &f[1], par, sv, &f[2], part, ch, st);
  if (rc || !sums) return rc;
  return finish_column_grads({part, ch.chunks}, {part, ch.chunks}, ch.B, C, par.w, par.bias, par.scale, 1.f, grads, st);
}
