// A projection with its epilogue, forward and backward: y = residual + gate_b act(x w^T + bias)
// (models/rope_dit_transformer_2d.py:205-213, :254-258, :640-711: to_q / to_k / to_v, to_out and the feed-forward with adaLN-zero's gates).
//
//   z = x w^T + bias,  dz = dy gate_b act'(z),  dx = dz w,  dw = dz^T x,  dbias = sum dz,  dgate_b = sum_n dy z,  dresidual = dy
//
// This file: checks, the products of fp32 data, and the passes around the products (dz and its column sums, the sum of a split product's parts).  bf16 data:
// linear_tc.cu.
#include <string.h>

#include "linear.cuh"
#include "tc05.cuh"
#include "vec.cuh"

namespace llsa {

namespace {

using bf16 = __nv_bfloat16;

// ------------------------------------------------------------------------------------------------ scalar products
// fp32 data: one multiply-add per product, as fp32 asks; the tensor cores round their operands to fewer bits.  A CTA of TH x TH threads owns a tile of
// TH TM x TH TM outputs (TH = 16, or 8 for CTAs of two warps), a thread TM x TM of them.  Steps of 16 along k: the next step's operands are on their way in
// registers while this one's are multiplied from shared memory, where either stands as 16 rows of neighbours in i or j (turned on the way in if memory has it
// along k), so that a thread's fours are one load.  TM^2 multiply-adds a k against TM / 2 such loads: the FMA pipe is what bounds it, with two CTAs to an SM.
// 16384 x 384 -> 1536: 437 us forward, 468 dx, 390 dw (44, 41 and 50 TFLOP/s; cuBLAS 500 forward, 406 dw).  2048 x 384 -> 384: 31 us, 192 tiles of 64 x 64 on
// 148 SMs, of which 44 have two, and there shared memory is the pace (cuBLAS 27); operands four steps ahead instead of one change nothing.
template <int TM, int TH, bool ALONG_K>
struct Operand {
  static constexpr int kRows = TH * TM, kK = 16, kLd = kRows + 4, kFloats = kK * kLd, kThreads = TH * TH;
  static constexpr int kVecs = kRows * kK / 4, kMine = (kVecs + kThreads - 1) / kThreads;
  float4 x[kMine];
  // The place of the thread's u-th row (t: its number along the tile)
  static __device__ __forceinline__ int row(int t, int u) { return TM >= 4 ? (u / 4) * 4 * TH + 4 * t + u % 4 : 2 * t + u; }
  static __device__ __forceinline__ void place(int v, int& r, int& k) {
    r = ALONG_K ? v / 4 : v % (kRows / 4) * 4;
    k = ALONG_K ? v % 4 * 4 : v / (kRows / 4);
  }
  const float* src[kMine];      // of the next step
  int have[kMine];              // rows, or columns of the four, that are there
  __device__ __forceinline__ void begin(const Mat<const float>& m, int64_t row0, int64_t rows, int64_t k0) {
#pragma unroll
    for (int q = 0; q < kMine; ++q) {
      const int v = q * kThreads + threadIdx.x;
      int r, k;
      place(v, r, k);
      const int64_t i = row0 + r, left = max((int64_t) 0, min((int64_t) 4, rows - i));
      src[q] = ALONG_K ? m.p + i * m.ld + k0 + k : m.p + (k0 + k) * m.ld + i;
      have[q] = kVecs % kThreads && v >= kVecs ? 0 : ALONG_K ? (left ? 4 : 0) : (int) left;
    }
  }
  // `left` k's are left
  __device__ __forceinline__ void load(int64_t ld, int vec, int left) {
#pragma unroll
    for (int q = 0; q < kMine; ++q) {
      int r, k;
      place(q * kThreads + threadIdx.x, r, k);
      const int n = ALONG_K ? min(have[q], left - k) : k < left ? have[q] : 0;
      x[q] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (vec && n >= 4) {
        x[q] = __ldg(reinterpret_cast<const float4*>(src[q]));
      } else {
        if (n > 0) x[q].x = __ldg(src[q]);
        if (n > 1) x[q].y = __ldg(src[q] + 1);
        if (n > 2) x[q].z = __ldg(src[q] + 2);
        if (n > 3) x[q].w = __ldg(src[q] + 3);
      }
      src[q] += ALONG_K ? kK : kK * ld;
    }
  }
  __device__ __forceinline__ void put(float* buf) const {
#pragma unroll
    for (int q = 0; q < kMine; ++q) {
      const int v = q * kThreads + threadIdx.x;
      if (kVecs % kThreads && v >= kVecs) break;
      int r, k;
      place(v, r, k);
      if constexpr (ALONG_K) {
        float* to = buf + k * kLd + r;
        to[0] = x[q].x;
        to[kLd] = x[q].y;
        to[2 * kLd] = x[q].z;
        to[3 * kLd] = x[q].w;
      } else {
        *reinterpret_cast<float4*>(buf + k * kLd + r) = x[q];
      }
    }
  }
  static __device__ __forceinline__ void read(const float* buf, int t, int k, float (&u)[TM]) {
    if constexpr (TM >= 4) {
#pragma unroll
      for (int i = 0; i < TM; i += 4) {
        const float4 f = *reinterpret_cast<const float4*>(buf + k * kLd + i * TH + 4 * t);
        u[i] = f.x; u[i + 1] = f.y; u[i + 2] = f.z; u[i + 3] = f.w;
      }
    } else {
      const float2 f = *reinterpret_cast<const float2*>(buf + k * kLd + 2 * t);
      u[0] = f.x; u[1] = f.y;
    }
  }
};

// S > 1: a cluster of S CTAs takes a tile, an S-th of the sum each; they leave their sums in shared memory, and every one adds an S-th of the rows up, in order
template <int TM, int TH, int S, bool A_K, bool B_K, bool PARTIAL>
__global__ void __launch_bounds__(TH * TH, TH == 16 ? 2 : 4)
product_kernel(Product<float> p, Epilogue<float> e, float* __restrict__ partial, int64_t partial_ld, int64_t tiles_n, int64_t per_split, int vec_a, int vec_b) {
  using A = Operand<TM, TH, A_K>;
  using B = Operand<TM, TH, B_K>;
  constexpr int BM = TH * TM, BK = 16;
  __shared__ __align__(16) float s_ab[4][A::kFloats];
  float(*s_a)[A::kFloats] = s_ab, (*s_b)[A::kFloats] = s_ab + 2;
  const int tx = threadIdx.x % TH, ty = threadIdx.x / TH;
  const uint32_t tile = blockIdx.x / S, rank = blockIdx.x % S;
  const int64_t i0 = tile / tiles_n * BM, j0 = tile % tiles_n * BM;
  const int64_t k_first = (S > 1 ? rank : blockIdx.y) * per_split, k_end = min(p.K, k_first + per_split);
  float2 acc[TM][TM / 2];                                    // two neighbours an instruction, the same multiply-adds
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TM / 2; ++j) acc[i][j] = make_float2(0.f, 0.f);
  pdl_wait();
  pdl_trigger();
  A a;
  B b;
  a.begin(p.a, i0, p.M, k_first);
  b.begin(p.b, j0, p.N, k_first);
  int buf = 0, left = (int) (k_end - k_first);               // of a part, or of the features: fewer than 2^31
  a.load(p.a.ld, vec_a, left);
  b.load(p.b.ld, vec_b, left);
  for (; left > 0; buf ^= 1) {
    a.put(s_a[buf]);
    b.put(s_b[buf]);
    __syncthreads();                                         // and the other buffer's readers are through
    left -= BK;
    if (left > 0) {
      a.load(p.a.ld, vec_a, left);
      b.load(p.b.ld, vec_b, left);
    }
#pragma unroll
    for (int k = 0; k < BK; ++k) {
      float u[TM], v[TM];
      A::read(s_a[buf], ty, k, u);
      B::read(s_b[buf], tx, k, v);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TM / 2; ++j) acc[i][j] = __ffma2_rn(make_float2(u[i], u[i]), make_float2(v[2 * j], v[2 * j + 1]), acc[i][j]);
    }
  }
  if constexpr (S > 1) {
    static_assert(TM % S == 0 && 4 * A::kFloats >= BM * A::kLd, "rows of a thread in equal shares; a tile of sums where the operands stood");
    float* sums = &s_ab[0][0];
    __syncthreads();                                         // the last step's readers are through
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TM / 2; j += 2)
        *reinterpret_cast<float4*>(sums + A::row(ty, i) * A::kLd + B::row(tx, 2 * j)) = make_float4(acc[i][j].x, acc[i][j].y, acc[i][j + 1].x, acc[i][j + 1].y);
    tc::cluster_sync_all();
#pragma unroll
    for (int i = 0; i < TM; ++i)
      if (i / (TM / S) == rank)
#pragma unroll
        for (int j = 0; j < TM / 2; j += 2) {
          float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (uint32_t q = 0; q < S; ++q) {
            float4 u;
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(u.x), "=f"(u.y), "=f"(u.z), "=f"(u.w)
                         : "r"(tc::at_rank(sums + A::row(ty, i) * A::kLd + B::row(tx, 2 * j), q)) : "memory");
            t.x += u.x, t.y += u.y, t.z += u.z, t.w += u.w;
          }
          acc[i][j] = make_float2(t.x, t.y);
          acc[i][j + 1] = make_float2(t.z, t.w);
        }
    tc::cluster_sync_all();                                  // nobody's sums are read any more
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int64_t r = i0 + A::row(ty, i);
    if (r >= p.M || (S > 1 && i / (TM / S) != rank)) continue;
    const int64_t sample = !PARTIAL && e.gate.p ? (uint32_t) r / e.rows_per_gate : 0;
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      const int64_t c = j0 + B::row(tx, j);
      if (c >= p.N) continue;
      const float d = j & 1 ? acc[i][j / 2].y : acc[i][j / 2].x;
      if constexpr (PARTIAL) {
        partial[(blockIdx.y * p.M + r) * partial_ld + c] = d;
      } else {
        float z = d + (e.bias ? e.bias[c] : 0.f);
        if (e.pre.p) e.pre.p[r * e.pre.ld + c] = z;
        z = activate(z, e.act);
        if (e.gate.p) z *= e.gate.p[sample * e.gate.ld + c];
        if (e.residual.p) z += e.residual.p[r * e.residual.ld + c];
        e.y.p[r * e.y.ld + c] = z;
      }
    }
  }
}

template <bool A_K, bool B_K, bool PARTIAL>
int launch_product(const Product<float>& p, const Epilogue<float>& e, float* partial, int64_t ld, cudaStream_t st) {
  auto tiles = [&](int64_t b) { return (p.M + b - 1) / b * ((p.N + b - 1) / b); };
  auto vec = [](const Mat<const float>& m) { return (uintptr_t) m.p % 16 == 0 && m.ld % 4 == 0; };
  // split: parts of the sum, a CTA each: along y in memory, or the `cluster` CTAs of a tile
  auto go = [&](auto kernel, int64_t b, unsigned threads, int64_t split, unsigned cluster) {
    const int64_t per = ((p.K + split - 1) / split + 15) / 16 * 16;
    launch_pdl_cluster(kernel, dim3((unsigned) (tiles(b) * cluster), (unsigned) (PARTIAL ? split : 1)), dim3(threads), cluster, 0, st, p, e, partial, ld,
                       (p.N + b - 1) / b, per, (int) vec(p.a), (int) vec(p.b));
  };
  LLSA_REQUIRE(tiles(32) <= INT32_MAX / 8, LLSA_ERR_SHAPE, "linear: too many outputs");
  const int64_t t = tiles(64), steps = (p.K + 15) / 16;
  if constexpr (PARTIAL) {
    // parts in tiles of 64 x 64 that two warps hold, which fill four to an SM evenly (dw of 16384 x 384 -> 1536 390 us, in tiles of 128 x 128 446; of
    // 2048 x 384 -> 384 24 and 29)
    if (t * p.split >= 148) go(product_kernel<8, 8, 1, A_K, B_K, true>, 64, 64, p.split, 1);
    else go(product_kernel<2, 16, 1, A_K, B_K, true>, 32, 256, p.split, 1);
  } else {
    // the largest tile that still gives every SM one (forward of 16384 x 384 -> 1536 in tiles of two warps 469 us, 437 so: operands are turned on the way in);
    // where there are few, their sums in 2 to 8 parts of 16 steps at least, of 4 where not every SM has a tile.  us, without and so: 512 x 1536 -> 384 60 / 28
    // (cuBLAS 36), 300 x 389 -> 771 28 / 19 (17), dx of 2048 x 384 -> 1536 107 / 79; 2048 x 384 -> 384 would be 31 / 33, 8 x 256 -> 384 8 / 10
    int64_t S = 1;
    while (S < 8 && t * S * 2 <= 148 * 6 && steps / (2 * S) >= (t >= 148 ? 16 : 4)) S *= 2;
    if (t * S < 148 && steps < 32) S = 1;
    if (tiles(128) >= 148) go(product_kernel<8, 16, 1, A_K, B_K, false>, 128, 256, 1, 1);
    else if (S == 8) go(product_kernel<8, 8, 8, A_K, B_K, false>, 64, 64, S, 8);
    else if (S == 4) go(product_kernel<8, 8, 4, A_K, B_K, false>, 64, 64, S, 4);
    else if (S == 2) go(product_kernel<8, 8, 2, A_K, B_K, false>, 64, 64, S, 2);
    else if (t >= 148) go(product_kernel<4, 16, 1, A_K, B_K, false>, 64, 256, 1, 1);
    else go(product_kernel<2, 16, 1, A_K, B_K, false>, 32, 256, 1, 1);
  }
  LLSA_LAUNCH_OK("product_kernel");
  return LLSA_OK;
}

// ------------------------------------------------------------------------------------------------ dz and its column sums
// dz = dy gate act'(z) and, per column and part of a sample's rows, P = sum dy z and S = sum dz (column_sums.cuh).  bf16 data: act' by linear_tc_slope.  A
// thread owns V neighbouring columns and every (256 / tx)th row of its CTA's; U rows are on their way at once.
template <typename T>
struct FrontArgs {
  Mat<const T> dy, pre, gate;
  Mat<T> dz;                   // p NULL: not written
  float* partial;              // NULL: no sums
  uint32_t N, chunks, per;     // rows of a sample, CTAs along them, rows of a CTA
  int F, act, tx;              // tx: threads along the columns, a power of two
};
template <typename T, int V>
__global__ void __launch_bounds__(256, 2)
linear_dz_kernel(FrontArgs<T> a) {
  constexpr int U = 8;
  using P = Vec<T, V>;
  using Raw = typename P::type;
  extern __shared__ float s_part[];                        // [2][256 / tx][tx * V]
  const int tx = a.tx, lanes = 256 / tx, col = threadIdx.x % tx, lane = threadIdx.x / tx, c = (blockIdx.y * tx + col) * V;
  const uint32_t b = blockIdx.x / a.chunks, first = (blockIdx.x - b * a.chunks) * a.per, end = min(a.N, first + a.per);
  pdl_wait();
  pdl_trigger();
  float p[V], s[V], gate[V];
#pragma unroll
  for (int i = 0; i < V; ++i) p[i] = s[i] = 0.f;
  if (c < a.F) {
#pragma unroll
    for (int i = 0; i < V; ++i) gate[i] = a.gate.p ? to_f32<T>(a.gate.p[b * a.gate.ld + c + i]) : 1.f;
    for (uint32_t n0 = first + lane; n0 < end; n0 += U * lanes) {
      Raw dy[U], pre[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (n0 + u * lanes < end) {
          const int64_t r = (int64_t) b * a.N + n0 + u * lanes;
          dy[u] = *reinterpret_cast<const Raw*>(a.dy.p + r * a.dy.ld + c);
          if (a.pre.p) pre[u] = *reinterpret_cast<const Raw*>(a.pre.p + r * a.pre.ld + c);
        }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (n0 + u * lanes < end) {
          float g[V], z[V], d[V];
          P::unpack(dy[u], g);
          if (a.pre.p) P::unpack(pre[u], z);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            d[i] = __fmul_rn(g[i], gate[i]);      // never contracted: the sums' bits do not depend on what else is asked for
            if (a.pre.p) {
              p[i] = fmaf(g[i], z[i], p[i]);
              if constexpr (sizeof(T) == 4) d[i] *= activate_grad(z[i], a.act);
            }
            s[i] = __fadd_rn(s[i], d[i]);
          }
          if (a.dz.p) *reinterpret_cast<Raw*>(a.dz.p + ((int64_t) b * a.N + n0 + u * lanes) * a.dz.ld + c) = P::pack(d);
        }
    }
  }
  if (!a.partial) return;
  const int width = tx * V;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    s_part[lane * width + col * V + i] = p[i];
    s_part[(lanes + lane) * width + col * V + i] = s[i];
  }
  __syncthreads();
  for (int k = threadIdx.x; k < 2 * width; k += 256) {
    const int which = k / width, at = k - which * width;
    if (blockIdx.y * width + at >= a.F) continue;
    float u = 0.f;
    for (int j = 0; j < lanes; ++j) u += s_part[(which * lanes + j) * width + at];
    a.partial[((int64_t) blockIdx.x * 2 + which) * a.F + blockIdx.y * width + at] = u;
  }
}

template <typename T, int V>
int launch_dz(FrontArgs<T>& f, int64_t blocks, int tx, cudaStream_t st) {
  f.tx = tx;
  const int64_t cols = (f.F + tx * V - 1) / (tx * V);
  LLSA_REQUIRE(blocks <= INT32_MAX && cols <= 65535, LLSA_ERR_SHAPE, "linear_bwd: too many samples or features");
  launch_pdl(linear_dz_kernel<T, V>, dim3((unsigned) blocks, (unsigned) cols), dim3(256), (size_t) (f.partial ? 2 * 256 * V * 4 : 0), st, f);
  LLSA_LAUNCH_OK("linear_dz_kernel");
  return LLSA_OK;
}

// ------------------------------------------------------------------------------------------------ parts of a split product
// out[r, c] = sum of the parts' (r, c), or, TURNED, of their (c, r).  A CTA takes 32 x 32 of them through shared memory, 8 rows of threads; the parts are
// added in order, four on their way at once.
template <typename T, bool TURNED>
__global__ void __launch_bounds__(256)
sum_parts_kernel(const float* __restrict__ partial, int64_t ld, int split, int64_t rows, int64_t cols, T* __restrict__ out) {
  __shared__ float s_tile[32][33];
  const int x = threadIdx.x % 32, y = threadIdx.x / 32;
  const int64_t r0 = blockIdx.y * (int64_t) 32, c0 = blockIdx.x * (int64_t) 32;
  const int64_t part = (TURNED ? cols : rows) * ld, prow = TURNED ? c0 : r0, pcol = (TURNED ? r0 : c0) + x;
  const int64_t prows = TURNED ? cols : rows, pcols = TURNED ? rows : cols;
  pdl_wait();
  pdl_trigger();
  float u[4] = {0.f, 0.f, 0.f, 0.f};
  if (pcol < pcols) {
#pragma unroll 4
    for (int s = 0; s < split; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (prow + y + 8 * i < prows) u[i] += partial[s * part + (prow + y + 8 * i) * ld + pcol];
  }
  if constexpr (TURNED) {
#pragma unroll
    for (int i = 0; i < 4; ++i) s_tile[y + 8 * i][x] = u[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = s_tile[x][y + 8 * i];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (r0 + y + 8 * i < rows && c0 + x < cols) out[(r0 + y + 8 * i) * cols + c0 + x] = from_f32<T>(u[i]);
}

template <typename T>
int sum_parts(const float* partial, int64_t ld, int split, bool turned, int64_t rows, int64_t cols, T* out, cudaStream_t st) {
  const dim3 grid((unsigned) ((cols + 31) / 32), (unsigned) ((rows + 31) / 32));
  LLSA_REQUIRE(grid.y <= 65535, LLSA_ERR_SHAPE, "linear_bwd: too many features");
  if (turned) launch_pdl(sum_parts_kernel<T, true>, grid, dim3(256), 0, st, partial, ld, split, rows, cols, out);
  else launch_pdl(sum_parts_kernel<T, false>, grid, dim3(256), 0, st, partial, ld, split, rows, cols, out);
  LLSA_LAUNCH_OK("sum_parts_kernel");
  return LLSA_OK;
}

// ------------------------------------------------------------------------------------------------ a gate by samples
// Of long samples the gate is applied to what is small instead of to dy.  With G_b = dy_b^T x_b (the parts of dw, taken sample by sample) and S_b = sum_n dy:
//   dx_b = dy_b (gate_b w),   dw = sum_b gate_b G_b,   dgate_b = rowsum(w G_b) + bias S_b,   dbias = sum_b gate_b S_b
// so that the product of the forward is not kept, dz is neither written nor rounded, and what passes through memory for it is B weights and parts.  gate_b w is
// rounded to bf16, as the tensor cores take their operands: a half step in dx beside the one of dx itself, where a rounded dz would put it into dx and dw.
// us, 131072 rows in 8 samples, 1536 -> 384, forward and backward: 490 with z kept and dz written, 465 so.
__global__ void __launch_bounds__(256)
gated_weight_kernel(Mat<const bf16> w, Mat<const bf16> gate, bf16* __restrict__ out, int F, int K) {      // out [B][F][K]; K a multiple of 8
  const int64_t i = blockIdx.x * (int64_t) blockDim.x + threadIdx.x, b = blockIdx.y;
  const int per = K / 8;
  pdl_wait();
  pdl_trigger();
  if (i >= (int64_t) F * per) return;
  const int f = (int) (i / per), k = (int) (i % per) * 8;
  float v[8];
  Vec<bf16, 8>::unpack(*reinterpret_cast<const uint4*>(w.p + f * w.ld + k), v);
  const float g = __bfloat162float(gate.p[b * gate.ld + f]);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] *= g;
  *reinterpret_cast<uint4*>(out + (b * F + f) * K + k) = Vec<bf16, 8>::pack(v);
}

// dw = sum_b gate_b (sum of sample b's parts), and of each CTA's share of the input features rowsum(w G_b) in pg[B][share][0][F].  out, pg: NULL where not wanted.
// A CTA takes 16 rows of 128 columns of the parts ([F][K], or TURNED [K][F]), 512 bytes of a row to a warp; its threads hold 2 x 4 values, and two samples' parts
// are on their way at once, in order.  (57 MB of parts, 1536 x 384 in 24: 31 us in tiles of 32 x 32, 62 and more with more of those 128-byte pieces on their
// way; so 18.)  F and K are multiples of 8.
constexpr int kPartRows = 16, kPartCols = 128;
template <bool TURNED>
__global__ void __launch_bounds__(256, 2)
gated_parts_kernel(const float* __restrict__ partial, int64_t ld, int per_sample, int B, int64_t F, int64_t K, Mat<const bf16> gate, Mat<const bf16> w,
                   bf16* __restrict__ out, float* __restrict__ pg) {
  constexpr int kAtOnce = 2, kAhead = 4;
  __shared__ float4 s_sum[kAtOnce][8][kPartCols / 4];
  __shared__ float s_out[TURNED ? kPartCols : 1][kPartRows + 1];
  const int x = threadIdx.x % 32, y = threadIdx.x / 32;
  const int64_t rows = TURNED ? K : F, cols = TURNED ? F : K, part = rows * ld, r0 = blockIdx.x * (int64_t) kPartRows, c0 = blockIdx.y * (int64_t) kPartCols,
                c = c0 + 4 * x, share = TURNED ? blockIdx.x : blockIdx.y, shares = TURNED ? gridDim.x : gridDim.y;
  const bool there[2] = {r0 + y < rows && c < cols, r0 + y + 8 < rows && c < cols};
  pdl_wait();
  pdl_trigger();
  float wv[2][4], acc[2][4] = {};
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t r = r0 + y + 8 * i;
      wv[i][j] = pg && there[i] ? __bfloat162float(TURNED ? w.p[(c + j) * w.ld + r] : w.p[r * w.ld + c + j]) : 0.f;
    }
  for (int b0 = 0; b0 < B; b0 += kAtOnce) {
    float u[kAtOnce][2][4] = {}, g[kAtOnce][TURNED ? 4 : 2];
#pragma unroll
    for (int q = 0; q < kAtOnce; ++q)
#pragma unroll
      for (int j = 0; j < (TURNED ? 4 : 2); ++j)
        g[q][j] = b0 + q < B && there[TURNED ? 0 : j] ? __bfloat162float(gate.p[(b0 + q) * gate.ld + (TURNED ? c + j : r0 + y + 8 * j)]) : 0.f;
    for (int s = 0; s < per_sample; s += kAhead) {
      float4 v[kAtOnce][kAhead][2];
#pragma unroll
      for (int q = 0; q < kAtOnce; ++q)
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          const float* p = partial + ((int64_t) (b0 + q) * per_sample + s + j) * part + (r0 + y) * ld + c;
          const bool some = b0 + q < B && s + j < per_sample;
#pragma unroll
          for (int i = 0; i < 2; ++i) v[q][j][i] = some && there[i] ? *reinterpret_cast<const float4*>(p + 8 * i * ld) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
      for (int q = 0; q < kAtOnce; ++q)
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            u[q][i][0] += v[q][j][i].x;
            u[q][i][1] += v[q][j][i].y;
            u[q][i][2] += v[q][j][i].z;
            u[q][i][3] += v[q][j][i].w;
          }
    }
#pragma unroll
    for (int q = 0; q < kAtOnce; ++q)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (b0 + q < B && there[i]) acc[i][j] = fmaf(g[q][TURNED ? j : i], u[q][i][j], acc[i][j]);
    if (!pg) continue;
    if constexpr (TURNED) {
      if (b0) __syncthreads();
#pragma unroll
      for (int q = 0; q < kAtOnce; ++q) {
        float t[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) t[j] = fmaf(wv[1][j], u[q][1][j], wv[0][j] * u[q][0][j]);
        s_sum[q][y][x] = make_float4(t[0], t[1], t[2], t[3]);
      }
      __syncthreads();
      const int q = threadIdx.x / kPartCols, col = threadIdx.x % kPartCols;
      if (b0 + q < B && c0 + col < F) {
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) t += reinterpret_cast<const float*>(&s_sum[q][k][0])[col];
        pg[((int64_t) (b0 + q) * shares + share) * 2 * F + c0 + col] = t;
      }
    } else {
#pragma unroll
      for (int q = 0; q < kAtOnce; ++q)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float t = 0.f;
#pragma unroll
          for (int j = 0; j < 4; ++j) t = fmaf(wv[i][j], u[q][i][j], t);
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
          const int64_t f = r0 + y + 8 * i;
          if (x == 0 && b0 + q < B && f < F) pg[((int64_t) (b0 + q) * shares + share) * 2 * F + f] = t;
        }
    }
  }
  if (!out) return;
  if constexpr (TURNED) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s_out[4 * x + j][y + 8 * i] = acc[i][j];
    __syncthreads();
    const int64_t f = c0 + threadIdx.x / 2, k = r0 + threadIdx.x % 2 * 8;
    if (f < F && k < K) *reinterpret_cast<uint4*>(out + f * K + k) = Vec<bf16, 8>::pack(&s_out[threadIdx.x / 2][threadIdx.x % 2 * 8]);
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (there[i]) *reinterpret_cast<uint2*>(out + (r0 + y + 8 * i) * K + c) = Vec<bf16, 4>::pack(acc[i]);
  }
}

// ------------------------------------------------------------------------------------------------ checks and plan
// A matrix with unit column stride
int check_matrix(const LlsaTensor* t, const char* name, int dtype, int64_t rows, int64_t cols) {
  LLSA_REQUIRE(t && t->ptr, LLSA_ERR_NULL, "%s: null tensor", name);
  LLSA_REQUIRE(t->dtype == dtype, LLSA_ERR_DTYPE, "%s: dtype %d, expected %d", name, t->dtype, dtype);
  LLSA_REQUIRE(t->ndim == 2 && t->shape[0] == rows && t->shape[1] == cols, LLSA_ERR_SHAPE, "%s: must be [%lld,%lld]", name, (long long) rows, (long long) cols);
  LLSA_REQUIRE(cols == 1 || t->stride[1] == 1, LLSA_ERR_STRIDE, "%s: innermost stride %lld, must be 1", name, (long long) t->stride[1]);
  return LLSA_OK;
}

// Rows on 16-byte boundaries that do not overlap, such as those of one that stands for all: tensor maps are specified for strides that reach past a row
bool rows16(const LlsaTensor* t) {
  return (uintptr_t) t->ptr % 16 == 0 && (t->shape[0] == 1 || (t->stride[0] * (int64_t) dtype_size(t->dtype) % 16 == 0 && t->stride[0] >= t->shape[1]));
}

struct Plan {
  int64_t M, K, F, B, N;       // rows, input and output features, samples (1 without a gate), rows of a sample
  int dtype;
  bool write_dz, sums;         // the pass over dy: leaves dz / column sums
  bool slope;                  // bf16 with an activation: that pass is a product
  int vec, tx;                 // its columns of a thread, threads along the columns
  int64_t dz_ld, chunks, per;
  int split;                   // dw: parts of the sum over the rows, of [F][part_ld], or turned [K][part_ld]
  bool turned;
  int64_t part_ld;
  bool by_sample;              // the gate is applied to the weight and to the parts of dw
  int64_t k_tiles;
  size_t o_dz, o_cols, o_parts, o_wg, o_pg, bytes;
};

// Long samples: twice as many rows as input features, where the B weights and parts hold no more bytes than z and dz; rows on 16-byte boundaries throughout;
// samples that a grid's second dimension takes.  us, forward and backward in a graph, so / with z kept: samples x rows, features: 8 x 16384, 1536 -> 384 461 / 488;
// 8 x 4096, 384 -> 1536 171 / 233; 64 x 1024, 64 -> 512 148 / 152; 4 x 2048, 1024 -> 1024 84 to 91 / 84; beside the line 16 x 512, 256 -> 1024 68 / 66; 2 x 1024,
// 256 -> 256 26 to 29 / 27.  Of many samples the parts of a narrow dw are added by few CTAs, one pair of samples after another (gated_parts_kernel), and z kept would be
// the faster way: 32 x 1024, 384 -> 384 98 / 90; 64 x 512, 256 -> 1024 203 / 169; 256 x 512, 256 -> 256 389 / 204; 1024 x 512, 64 -> 64 1003 / 227.
bool by_sample(const LlsaLinearArgs* a, const Plan& p) {
  return p.dtype == LLSA_BF16 && a->gate && p.N >= 512 && p.N >= 2 * p.K && p.K % 8 == 0 && p.F % 8 == 0 && p.B <= 65535;
}

int check_common(const LlsaLinearArgs* a, Plan* p) {
  LLSA_REQUIRE(a && a->x && a->x->ptr && a->weight && a->weight->ptr, LLSA_ERR_NULL, "linear: null argument");
  LLSA_REQUIRE(is_float_dtype(a->x->dtype), LLSA_ERR_DTYPE, "x: must be f32 or bf16");
  LLSA_REQUIRE(a->x->ndim == 2 && a->weight->ndim == 2, LLSA_ERR_SHAPE, "linear: x must be [M,K] and weight [F,K]");
  p->dtype = a->x->dtype;
  p->M = a->x->shape[0];
  p->K = a->x->shape[1];
  p->F = a->weight->shape[0];
  LLSA_REQUIRE(p->K >= 1 && p->F >= 1 && p->K <= (1 << 20) && p->F <= (1 << 20), LLSA_ERR_SHAPE, "linear: 1 to 2^20 features are supported");
  LLSA_REQUIRE(p->M <= INT32_MAX, LLSA_ERR_SHAPE, "linear: more than 2^31 - 1 rows");
  int rc;
  if ((rc = check_matrix(a->x, "x", p->dtype, p->M, p->K)) || (rc = check_matrix(a->weight, "weight", p->dtype, p->F, p->K))) return rc;
  if (p->dtype == LLSA_BF16) LLSA_REQUIRE(rows16(a->x) && rows16(a->weight), LLSA_ERR_STRIDE, "linear: rows of x and weight must start on 16-byte boundaries, and not overlap");
  LLSA_REQUIRE(a->activation >= kActNone && a->activation <= kActSilu, LLSA_ERR_ARG, "linear: activation %d is not known", a->activation);
  p->B = 1;
  if (a->gate) {
    LLSA_REQUIRE(a->gate->ptr, LLSA_ERR_NULL, "gate: null tensor");
    LLSA_REQUIRE(a->activation == kActNone, LLSA_ERR_ARG, "linear: a gate goes with no activation");
    LLSA_REQUIRE(a->gate->ndim == 2 && (p->M == 0 || (a->gate->shape[0] >= 1 && p->M % a->gate->shape[0] == 0)), LLSA_ERR_SHAPE,
                 "gate: must be [B,F], B a divisor of the rows of x");
    if ((rc = check_matrix(a->gate, "gate", p->dtype, a->gate->shape[0], p->F))) return rc;
    p->B = std::max<int64_t>(1, a->gate->shape[0]);
  }
  p->N = p->M / p->B;
  const int64_t bs[1] = {p->F};
  if (a->bias && (rc = check_contig(a->bias, "bias", p->dtype, 1, bs))) return rc;
  if (a->pre) {
    const int64_t s[2] = {p->M, p->F};
    if ((rc = check_contig(a->pre, "pre", p->dtype, 2, s))) return rc;
  }
  return LLSA_OK;
}

// What the backward does, from the shapes and from which results are asked for
void plan_bwd(const LlsaLinearArgs* a, Plan* p) {
  const int es = (int) dtype_size(p->dtype);
  if (p->M == 0) {             // no product to split and nothing to keep
    p->write_dz = p->sums = p->slope = p->by_sample = false;
    p->bytes = 0;
    return;
  }
  // dy itself is dz without an activation and a gate, where the tensor cores can read it
  p->write_dz = a->activation != kActNone || a->gate || (p->dtype == LLSA_BF16 && !(a->dy && rows16(a->dy)));
  p->by_sample = by_sample(a, *p);
  if (p->by_sample) p->write_dz = false;
  p->sums = p->by_sample ? a->dbias || (a->dgate && a->bias) : a->dbias || a->dgate;
  p->dz_ld = (p->F + 7) / 8 * 8;
  p->slope = p->dtype == LLSA_BF16 && a->activation != kActNone;
  if (p->slope) {
    p->chunks = linear_tc_slope_groups(p->M, p->F, p->K);
  } else {
    // a CTA: tx threads along the columns, the width of 16, 32 or 64 that leaves the fewest idle; along the rows as many CTAs as the SMs hold at once, two,
    // or of 16 rows a thread at least (U = 8 loads on their way a thread; 131072 x 384 sums in 26 us, with four and six CTAs and U = 4 51 and 54)
    p->vec = p->F % 8 == 0 && a->dy && rows16(a->dy) ? 16 / es : 1;
    int64_t idle = INT64_MAX;
    for (int tx : {64, 32, 16}) {
      const int64_t w = tx * p->vec, left = (p->F + w - 1) / w * w;
      if (left < idle) {
        idle = left;
        p->tx = tx;
      }
    }
    const int64_t cols = (p->F + p->tx * p->vec - 1) / (p->tx * p->vec), lanes = 256 / p->tx;
    p->chunks = std::max<int64_t>(1, std::min(148 * 2 / (cols * p->B), (p->N + 16 * lanes - 1) / (16 * lanes)));
    p->per = std::max<int64_t>(1, (p->N + p->chunks - 1) / p->chunks);
    p->chunks = std::max<int64_t>(1, (p->N + p->per - 1) / p->per);
  }
  const int64_t tiles = (p->F + 63) / 64 * ((p->K + 63) / 64);
  p->turned = false;
  p->split = p->dtype == LLSA_BF16 ? linear_tc_split(p->F, p->K, p->by_sample ? p->N : p->M, p->by_sample ? p->B : 0, &p->turned) : (int) std::max<int64_t>(1, std::min(148 * 4 / tiles, (p->M + 127) / 128));      // one wave of four CTAs to an SM
  p->part_ld = ((p->turned ? p->F : p->K) + 7) / 8 * 8;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += (bytes + 255) / 256 * 256;
    return o;
  };
  p->o_dz = take(p->write_dz ? (size_t) (p->M * p->dz_ld * es) : 0);
  p->o_cols = take(p->sums ? (size_t) (p->B * p->chunks * 2 * p->F * 4) : 0);
  const bool parts = a->dweight || (p->by_sample && a->dgate);
  p->o_parts = take(parts ? (size_t) ((p->by_sample ? p->B : 1) * p->split * (p->turned ? p->K : p->F) * p->part_ld * 4) : 0);
  p->k_tiles = p->turned ? (p->K + kPartRows - 1) / kPartRows : (p->K + kPartCols - 1) / kPartCols;
  p->o_wg = take(p->by_sample && a->dx ? (size_t) (p->B * p->F * p->K * es) : 0);
  p->o_pg = take(p->by_sample && a->dgate ? (size_t) (p->B * p->k_tiles * 2 * p->F * 4) : 0);
  p->bytes = at;
}

template <typename T>
Mat<T> mat(const LlsaTensor* t) {
  Mat<T> m;
  m.p = t ? (T*) t->ptr : nullptr;
  m.ld = !t ? 0 : t->shape[0] == 1 ? (t->shape[1] + 7) / 8 * 8 : t->stride[0];      // one row: a stride that a tensor map takes
  return m;
}

int product(const Product<float>& p, const Epilogue<float>& e, const LlsaLinearArgs*, cudaStream_t st) {
  return p.b_k ? launch_product<true, true, false>(p, e, nullptr, 0, st) : launch_product<true, false, false>(p, e, nullptr, 0, st);
}
int product(const Product<bf16>& p, const Epilogue<bf16>& e, const LlsaLinearArgs* a, cudaStream_t st) {
  return linear_tc_product(p, e, a->wait_limit, a->status, st);
}
int product_parts(const Product<float>& p, float* partial, int64_t ld, const LlsaLinearArgs*, cudaStream_t st) {
  return launch_product<false, false, true>(p, Epilogue<float>{}, partial, ld, st);
}
int product_parts(const Product<bf16>& p, float* partial, int64_t ld, const LlsaLinearArgs* a, cudaStream_t st) {
  return linear_tc_parts(p, partial, ld, a->wait_limit, a->status, st);
}

template <typename T>
int forward(const LlsaLinearArgs* a, const Plan& p, cudaStream_t st) {
  Epilogue<T> e = {};
  e.bias = a->bias ? (const T*) a->bias->ptr : nullptr;
  e.residual = mat<const T>(a->residual);
  e.gate = mat<const T>(a->gate);
  e.rows_per_gate = (uint32_t) p.N;
  e.y = mat<T>(a->y);
  e.pre = mat<T>(a->pre);
  e.act = a->activation;
  return product(Product<T>{mat<const T>(a->x), mat<const T>(a->weight), 1, 1, p.M, p.F, p.K, 1}, e, a, st);
}

int slope(const LlsaLinearArgs* a, const Plan& p, const Mat<bf16>& dz, float* sums, cudaStream_t st) {
  Epilogue<bf16> e = {};
  e.bias = a->bias ? (const bf16*) a->bias->ptr : nullptr;
  e.y = dz;
  e.act = a->activation;
  return linear_tc_slope(Product<bf16>{mat<const bf16>(a->x), mat<const bf16>(a->weight), 1, 1, p.M, p.F, p.K, 1}, e, mat<const bf16>(a->dy), sums, a->wait_limit,
                         a->status, st);
}
int slope(const LlsaLinearArgs*, const Plan&, const Mat<float>&, float*, cudaStream_t) { return LLSA_ERR_ARG; }      // not asked for

int backward_by_sample(const LlsaLinearArgs* a, const Plan& p, cudaStream_t st) {
  char* ws = (char*) a->workspace;
  const Mat<const bf16> dy = mat<const bf16>(a->dy), x = mat<const bf16>(a->x), w = mat<const bf16>(a->weight), gate = mat<const bf16>(a->gate);
  float* cols = p.sums ? (float*) (ws + p.o_cols) : nullptr;
  int rc;
  if (p.sums) {
    FrontArgs<bf16> f = {};
    f.dy = dy;
    f.partial = cols;
    f.N = (uint32_t) p.N; f.chunks = (uint32_t) p.chunks; f.per = (uint32_t) p.per;
    f.F = (int) p.F;
    rc = p.vec > 1 ? launch_dz<bf16, 8>(f, p.B * p.chunks, p.tx, st) : launch_dz<bf16, 1>(f, p.B * p.chunks, p.tx, st);
    if (rc) return rc;
  }
  if (a->dx) {
    bf16* wg = (bf16*) (ws + p.o_wg);
    launch_pdl(gated_weight_kernel, dim3((unsigned) ((p.F * (p.K / 8) + 255) / 256), (unsigned) p.B), dim3(256), 0, st, w, gate, wg, (int) p.F, (int) p.K);
    LLSA_LAUNCH_OK("gated_weight_kernel");
    Epilogue<bf16> e = {};
    e.y = mat<bf16>(a->dx);
    Product<bf16> d = {dy, {wg, p.K}, 1, 0, p.N, p.K, p.F, 1};
    d.samples = p.B;
    if ((rc = product(d, e, a, st))) return rc;
  }
  float* pg = a->dgate ? (float*) (ws + p.o_pg) : nullptr;
  if (a->dweight || a->dgate) {
    float* parts = (float*) (ws + p.o_parts);
    Product<bf16> d = p.turned ? Product<bf16>{x, dy, 0, 0, p.K, p.F, p.N, p.split} : Product<bf16>{dy, x, 0, 0, p.F, p.K, p.N, p.split};
    d.samples = p.B;
    if ((rc = product_parts(d, parts, p.part_ld, a, st))) return rc;
    const int64_t height = p.turned ? p.K : p.F, width = p.turned ? p.F : p.K;
    const dim3 grid((unsigned) ((height + kPartRows - 1) / kPartRows), (unsigned) ((width + kPartCols - 1) / kPartCols));
    bf16* dw = a->dweight ? (bf16*) a->dweight->ptr : nullptr;
    launch_pdl(p.turned ? gated_parts_kernel<true> : gated_parts_kernel<false>, grid, dim3(256), 0, st, (const float*) parts, p.part_ld, p.split, (int) p.B, p.F, p.K,
               gate, w, dw, pg);
    LLSA_LAUNCH_OK("gated_parts_kernel");
  }
  if (!a->dgate && !a->dbias) return LLSA_OK;
  const ParamView none = {nullptr, 0, 0}, factor = {a->gate->ptr, gate.ld, 1};
  ParamView bias;
  if ((rc = make_param(&bias, a->bias, "bias", p.dtype, 0, p.F))) return rc;
  return finish_column_grads({pg, p.k_tiles}, {cols, p.chunks}, p.B, p.F, none, bias, factor, 0.f,
                             {make_grad(a->dgate), make_grad(nullptr), make_grad(nullptr), make_grad(a->dbias)}, st);
}

template <typename T>
int backward(const LlsaLinearArgs* a, const Plan& p, cudaStream_t st) {
  char* ws = (char*) a->workspace;
  Mat<const T> dz = mat<const T>(a->dy);
  if (p.write_dz || p.sums) {
    FrontArgs<T> f = {};
    f.dy = dz;
    if (p.write_dz) {
      f.dz.p = (T*) (ws + p.o_dz);
      f.dz.ld = p.dz_ld;
      dz.p = f.dz.p;
      dz.ld = f.dz.ld;
    }
    f.partial = p.sums ? (float*) (ws + p.o_cols) : nullptr;
    int rc;
    if (p.slope) {
      rc = slope(a, p, f.dz, f.partial, st);
    } else {
      if (a->activation != kActNone || a->dgate) f.pre = mat<const T>(a->pre);
      f.gate = mat<const T>(a->gate);
      f.N = (uint32_t) p.N; f.chunks = (uint32_t) p.chunks; f.per = (uint32_t) p.per;
      f.F = (int) p.F;
      f.act = a->activation;
      rc = p.vec > 1 ? launch_dz<T, 16 / sizeof(T)>(f, p.B * p.chunks, p.tx, st) : launch_dz<T, 1>(f, p.B * p.chunks, p.tx, st);
    }
    if (rc) return rc;
    if (p.sums) {
      const ParamView none = {nullptr, 0, 0};
      rc = finish_column_grads({f.partial, p.chunks}, {f.partial, p.chunks}, p.B, p.F, none, none, none, 1.f,
                               {make_grad(a->dgate), make_grad(nullptr), make_grad(nullptr), make_grad(a->dbias)}, st);
      if (rc) return rc;
    }
  }
  if (a->dx) {
    Epilogue<T> e = {};
    e.y = mat<T>(a->dx);
    const int rc = product(Product<T>{dz, mat<const T>(a->weight), 1, 0, p.M, p.K, p.F, 1}, e, a, st);
    if (rc) return rc;
  }
  if (a->dweight) {
    float* parts = (float*) (ws + p.o_parts);
    const Mat<const T> x = mat<const T>(a->x);
    const int rc = p.turned ? product_parts(Product<T>{x, dz, 0, 0, p.K, p.F, p.M, p.split}, parts, p.part_ld, a, st)
                            : product_parts(Product<T>{dz, x, 0, 0, p.F, p.K, p.M, p.split}, parts, p.part_ld, a, st);
    if (rc) return rc;
    return sum_parts<T>(parts, p.part_ld, p.split, p.turned, p.F, p.K, (T*) a->dweight->ptr, st);
  }
  return LLSA_OK;
}

}  // namespace
}  // namespace llsa

using namespace llsa;

extern "C" int llsa_linear_fwd(const LlsaLinearArgs* a, void* stream) {
  Plan p;
  int rc = check_common(a, &p);
  if (rc) return rc;
  if (a->residual && (rc = check_matrix(a->residual, "residual", p.dtype, p.M, p.F))) return rc;
  LLSA_REQUIRE(!a->gate || a->residual, LLSA_ERR_ARG, "linear: a gate goes with a residual");
  LLSA_REQUIRE(!a->pre || a->gate || p.dtype == LLSA_F32, LLSA_ERR_ARG, "linear: bf16 products are kept for a gate only");
  if ((rc = check_matrix(a->y, "y", p.dtype, p.M, p.F))) return rc;
  if (p.M == 0) return LLSA_OK;
  return p.dtype == LLSA_F32 ? forward<float>(a, p, (cudaStream_t) stream) : forward<bf16>(a, p, (cudaStream_t) stream);
}

extern "C" int llsa_linear_keeps_product(const LlsaLinearArgs* a) {
  Plan p;
  if (check_common(a, &p)) return -1;
  return p.dtype == LLSA_F32 ? a->activation != kActNone || a->gate : a->gate && !by_sample(a, p);
}

extern "C" int64_t llsa_linear_bwd_workspace_bytes(const LlsaLinearArgs* a) {
  Plan p;
  if (check_common(a, &p)) return -1;
  plan_bwd(a, &p);
  return (int64_t) p.bytes;
}

extern "C" int llsa_linear_bwd(const LlsaLinearArgs* a, void* stream) {
  Plan p;
  int rc = check_common(a, &p);
  if (rc) return rc;
  plan_bwd(a, &p);
  if ((rc = check_matrix(a->dy, "dy", p.dtype, p.M, p.F))) return rc;
  LLSA_REQUIRE(!p.by_sample || rows16(a->dy), LLSA_ERR_STRIDE, "dy: rows must start on 16-byte boundaries, and not overlap, for a gate of long samples");
  LLSA_REQUIRE(!p.by_sample || !a->dx || rows16(a->dx), LLSA_ERR_STRIDE, "dx: rows must start on 16-byte boundaries, and not overlap, for a gate of long samples");
  LLSA_REQUIRE(!p.by_sample || !a->dweight || (uintptr_t) a->dweight->ptr % 16 == 0, LLSA_ERR_STRIDE, "dweight: must start on a 16-byte boundary for a gate of long samples");
  LLSA_REQUIRE(p.M == 0 || a->pre || !((a->dgate && !p.by_sample) || (p.dtype == LLSA_F32 && a->activation != kActNone)), LLSA_ERR_NULL, "pre: null tensor");
  if (a->dx && (rc = check_matrix(a->dx, "dx", p.dtype, p.M, p.K))) return rc;
  const int64_t ws[2] = {p.F, p.K}, gs[2] = {p.B, p.F}, bs[1] = {p.F};
  if (a->dweight && (rc = check_contig(a->dweight, "dweight", p.dtype, 2, ws))) return rc;
  if (a->dbias && (rc = check_grad(a->dbias, "dbias", p.dtype, 1, bs))) return rc;
  if (a->dgate) {
    LLSA_REQUIRE(a->gate, LLSA_ERR_NULL, "gate: null tensor");
    if ((rc = check_grad(a->dgate, "dgate", p.dtype, 2, gs))) return rc;
  }
  LLSA_REQUIRE(p.bytes == 0 || (a->workspace && ((uintptr_t) a->workspace & 255) == 0 && a->workspace_bytes >= (int64_t) p.bytes), LLSA_ERR_WORKSPACE,
               "workspace: llsa_linear_bwd_workspace_bytes() bytes on a 256-byte boundary are needed");
  if (p.M == 0) {
    if (a->dweight) LLSA_CUDA_OK(cudaMemsetAsync(a->dweight->ptr, 0, (size_t) (p.F * p.K) * dtype_size(p.dtype), (cudaStream_t) stream));
    return clear_column_grads({make_grad(a->dgate), make_grad(nullptr), make_grad(nullptr), make_grad(a->dbias)}, a->gate ? a->gate->shape[0] : 0, p.F,
                              (cudaStream_t) stream);
  }
  if (p.by_sample) return backward_by_sample(a, p, (cudaStream_t) stream);
  return p.dtype == LLSA_F32 ? backward<float>(a, p, (cudaStream_t) stream) : backward<bf16>(a, p, (cudaStream_t) stream);
}
