// The projection's matrix products on tcgen05 (bf16): D[i, j] = sum_k A(i, k) B(j, k), fp32 sums in tensor memory, and what stands behind them.
//
//   forward   A = x, B = w, both along k in memory:  y = residual + gate act(D + bias)
//   slope     the same product again:                dz = dy act'(D + bias), and its column sums.  z is not kept between the passes: writing it and
//             reading it back costs 4 bytes a value, computing it again K / 750 ns a value and SM; it is never rounded
//   forward   A = dz, B = w taken across:            dx
//   parts     A = dz, B = x, both taken across:      dw, in parts of the sum over the tokens, which a second kernel adds in order
//
// An operand whose rows run along k is a K-major tile, one whose rows run along i or j an MN-major tile, and TMA fills either from a row-major
// matrix with 128-byte swizzled rows of 64 (tc05.cuh).  Ragged edges are zeros that TMA fills in.
// A persistent CTA per SM walks tiles of 128 x BN, columns fastest (neighbours in time share rows of A in L2).  Warp 8 keeps a ring of k-steps of 64 filled;
// warp 9 issues the products into one of two accumulators in tensor memory; warps 0-7 empty the other one, so that a tile's epilogue runs under the
// next tile's products.  The epilogue goes in chunks of 64 columns, alternate chunks to either warpgroup, thread = row: a chunk is finished in
// a 128 x 64 buffer of shared memory (two per warpgroup), which a warp of movers (10, 11) has filled with the residual or dy by TMA beforehand and stores
// by TMA afterwards.  Written straight from the registers, 32 bytes of each of 32 rows an instruction, the stores were the kernel's pace: 590 us
// for 131072 x 384 -> 1536 with GELU.  Matrices whose rows TMA cannot take go through the same buffers with loads and stores of the warp.
// Every mbarrier wait is bounded; tiles behind one that ran out are written as NaN (and the status word says so).
#include <string.h>

#include "linear.cuh"
#include "tc05.cuh"
#include "tma.cuh"

namespace llsa {

namespace {

using bf16 = __nv_bfloat16;

constexpr int kBM = 128, kBK = 64, kThreads = 384, kEpilogueWarps = 8;
constexpr int kChunk = 64, kChunkElems = kBM * kChunk;      // a chunk of the epilogue: 16 KB of bf16

enum Kind { kForward, kSlope, kParts };

struct ProductMaps {
  CUtensorMap a, b, in, y;      // in: residual or dy
};

template <int BN, int KIND>
struct Tile {
  static constexpr int kStageElems = (kBM + BN) * kBK;
  static constexpr int kStages = KIND == kParts ? (BN == 256 ? 4 : BN == 192 ? 5 : BN == 128 ? 6 : 8) : BN == 256 ? 3 : BN == 192 ? 4 : BN == 128 ? (KIND == kSlope ? 4 : 5) : 6;
  static constexpr int kTmemCols = BN == 64 ? 128 : BN == 128 ? 256 : 512;
  static constexpr int kBuffers = KIND == kParts ? 0 : 4;
  static constexpr size_t kSmem = ((size_t) kStages * kStageElems + (size_t) kBuffers * kChunkElems) * 2 + 1024;
};

struct Bars {
  uint64_t full[8], empty[8], ready[2], free_[2], avail[4], done[4];      // avail, done: warpgroup * 2 + buffer
};

struct Outputs {
  Epilogue<bf16> e;
  Mat<const bf16> in;        // residual or dy
  float* partial;            // parts: [part][M][ld]; slope: [CTAs of a column][2][N], the sums in the second row
  int64_t ld;
  int64_t M, N;
  int tma_in, tma_y, vec_gate;
};

__device__ __forceinline__ void stg256(void* p, const uint32_t* r) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]),
               "r"(r[7])
               : "memory");
}

// ------------------------------------------------------------------------------------------------ activations, two values an instruction
__device__ __forceinline__ float2 two(float x) { return make_float2(x, x); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float clamp_nan(float x, float m) {      // to [-m, m]; NaN stays
  asm("min.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(m));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(-m));
  return x;
}
constexpr float kLog2e = 1.4426950408889634f;
// 1 / (1 + 2^t)
__device__ __forceinline__ float2 logistic2(float2 t) {
  const float2 d = __fadd2_rn(make_float2(ex2(t.x), ex2(t.y)), two(1.f));
  return make_float2(rcp(d.x), rcp(d.y));
}
template <int ACT>
__device__ __forceinline__ float2 activate2(float2 z) {
  if constexpr (ACT == kActNone) return z;
  float2 t;
  if constexpr (ACT == kActGeluTanh) t = __fmul2_rn(z, __ffma2_rn(__fmul2_rn(z, z), two(-kGelu2 * kGelu3 * kLog2e), two(-kGelu2 * kLog2e)));
  else t = __fmul2_rn(z, two(-kLog2e));
  return __fmul2_rn(z, logistic2(t));
}
template <int ACT>
__device__ __forceinline__ float2 slope2(float2 z) {      // s + z s (1 - s) u'(z)
  z = make_float2(clamp_nan(z.x, 1e4f), clamp_nan(z.y, 1e4f));      // 0 or 1 beyond; z^2 stays finite
  const float2 q = __fmul2_rn(z, z);
  float2 t;
  if constexpr (ACT == kActGeluTanh) t = __fmul2_rn(z, __ffma2_rn(q, two(-kGelu2 * kGelu3 * kLog2e), two(-kGelu2 * kLog2e)));
  else t = __fmul2_rn(z, two(-kLog2e));
  const float2 s = logistic2(t);
  float2 w = __fmul2_rn(__fmul2_rn(z, s), __ffma2_rn(s, two(-1.f), two(1.f)));
  if constexpr (ACT == kActGeluTanh) w = __fmul2_rn(w, __ffma2_rn(q, two(3.f * kGelu3 * kGelu2), two(kGelu2)));
  return __fadd2_rn(w, s);
}

// ------------------------------------------------------------------------------------------------ pieces of the epilogue
__device__ __forceinline__ void unpack8(const uint4& x, float2 (&v)[4]) {
  v[0] = make_float2(bf16_lo(x.x), bf16_hi(x.x)); v[1] = make_float2(bf16_lo(x.y), bf16_hi(x.y));
  v[2] = make_float2(bf16_lo(x.z), bf16_hi(x.z)); v[3] = make_float2(bf16_lo(x.w), bf16_hi(x.w));
}
__device__ __forceinline__ uint4 pack8(const float2 (&v)[4]) {
  return make_uint4(pack_bf16(v[0].x, v[0].y), pack_bf16(v[1].x, v[1].y), pack_bf16(v[2].x, v[2].y), pack_bf16(v[3].x, v[3].y));
}
// Eight elements of a row of which n are there
__device__ __forceinline__ uint4 load8(const bf16* p, int n, bool vec) {
  if (vec && n >= 8) return ldg128(p);
  const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = (2 * i < n ? (uint32_t) h[2 * i] : 0u) | (2 * i + 1 < n ? (uint32_t) h[2 * i + 1] << 16 : 0u);
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint16_t* element(bf16* buf, int row, int col) {      // of a swizzled chunk
  return reinterpret_cast<uint16_t*>(buf) + tc::swz(row, col >> 3) + (col & 7);
}
// A wait on a partner that gives up on nothing but this wait itself: the epilogue and its mover, who carry on behind a tile that went missing
__device__ __forceinline__ bool steady_wait(uint64_t* bar, uint32_t parity, volatile tc::WaitCtl* c) {
  for (int i = 0; i < tc::kWaitPolls; ++i)
    if (__all_sync(0xffffffffu, tc::mbar_try_wait(bar, parity))) return true;
  c->abort = 1;
  return false;
}

// The chunks of 64 columns of a CTA's tiles that one warpgroup owns, in order
template <int BN>
struct Chunks {
  int item, c, q;               // the item, the chunk behind the last one that was given out, the items before
  int tiles_n, items;
  int64_t N;
  int64_t i0, j0;               // of the chunk that was given out
  __device__ __forceinline__ Chunks(int tiles_n_, int items_, int64_t n) : item(blockIdx.x), c(0), q(0), tiles_n(tiles_n_), items(items_), N(n) {}
  __device__ __forceinline__ bool next(int wg) {
    for (; item < items; item += gridDim.x, c = 0, ++q)
      for (; c < BN / kChunk; ++c) {
        const int64_t j = (int64_t) (item % tiles_n) * BN + c * kChunk;
        if (((q * (BN / kChunk) + c) & 1) != wg || j >= N) continue;
        i0 = (int64_t) (item / tiles_n) * kBM;
        j0 = j;
        ++c;
        return true;
      }
    return false;
  }
};

// ------------------------------------------------------------------------------------------------ kernel
// items: (part, row tile, column tile), columns fastest.  k_blocks: steps of 64; per_split: those of a part.
template <int BN, bool A_MN, bool B_MN, int KIND, int ACT>
__global__ void __launch_bounds__(kThreads, 1)
product_tc_kernel(const __grid_constant__ ProductMaps maps, const __grid_constant__ Outputs out, int k_blocks, int per_split, int tiles_n, int tiles, int items,
                  int wait_limit, int32_t* status) {
  using T = Tile<BN, KIND>;
  extern __shared__ unsigned char smem_dyn[];
  __shared__ Bars bars;
  __shared__ uint32_t s_tmem;
  __shared__ tc::WaitCtl s_ctl;
  __shared__ float s_sum[KIND == kSlope ? kEpilogueWarps : 1][kChunk];
  bf16* ring = reinterpret_cast<bf16*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
  bf16* buffers = ring + T::kStages * T::kStageElems;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile tc::WaitCtl* ctl = &s_ctl;
  if (tid == 0) {
    s_ctl.abort = 0;
    s_ctl.limit = wait_limit > 0 ? wait_limit : tc::kWaitPolls;
    for (int i = 0; i < T::kStages; ++i) { tc::mbar_init(&bars.full[i], 1); tc::mbar_init(&bars.empty[i], 1); }
    for (int i = 0; i < 2; ++i) { tc::mbar_init(&bars.ready[i], 1); tc::mbar_init(&bars.free_[i], kEpilogueWarps); }
    for (int i = 0; i < 4; ++i) { tc::mbar_init(&bars.avail[i], 1); tc::mbar_init(&bars.done[i], 4); }
    tc::fence_mbar_init();
  }
  pdl_wait();
  if (warp == 0) tc::tmem_alloc(&s_tmem, T::kTmemCols);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  pdl_trigger();
  const uint32_t tmem = s_tmem;

  if (warp == 8) {
    // ---------------------------------------------------------------- TMA producer
    int st = 0;
    uint32_t ph = 1;
    bool ok = true;
    for (int item = blockIdx.x; ok && item < items; item += gridDim.x) {
      const int split = item / tiles, t = item - split * tiles, i0 = t / tiles_n * kBM, j0 = t % tiles_n * BN;
      const int k_end = min(k_blocks, (split + 1) * per_split);
      for (int kb = split * per_split; kb < k_end; ++kb) {
        if (!(ok = tc::warp_wait(&bars.empty[st], ph, ctl))) break;
        bf16* a = ring + st * T::kStageElems;
        bf16* b = a + kBM * kBK;
        tma::expect_tx_w(&bars.full[st], T::kStageElems * 2);
        if constexpr (A_MN) {
#pragma unroll
          for (int g = 0; g < kBM / 64; ++g) tma::load_2d_w(a + g * 64 * kBK, &maps.a, &bars.full[st], i0 + 64 * g, kb * kBK);
        } else {
          tma::load_2d_w(a, &maps.a, &bars.full[st], kb * kBK, i0);
        }
        if constexpr (B_MN) {
#pragma unroll
          for (int g = 0; g < BN / 64; ++g) tma::load_2d_w(b + g * 64 * kBK, &maps.b, &bars.full[st], j0 + 64 * g, kb * kBK);
        } else {
          tma::load_2d_w(b, &maps.b, &bars.full[st], kb * kBK, j0);
        }
        if (++st == T::kStages) { st = 0; ph ^= 1; }
      }
    }
  } else if (warp == 9) {
    // ---------------------------------------------------------------- products
    const uint32_t idesc = tc::instr_desc(kBM, BN, A_MN, B_MN);
    // K-major: 8 rows of 128 bytes follow one another; MN-major: 64 columns further on stands 64 rows (8 KB) behind
    const uint64_t da = tc::smem_desc(tc::smem_u32(ring), A_MN ? 8192 : 16, 1024), db = tc::smem_desc(tc::smem_u32(ring + kBM * kBK), B_MN ? 8192 : 16, 1024);
    const uint32_t hi_a = (uint32_t) (da >> 32), hi_b = (uint32_t) (db >> 32), lo_a = (uint32_t) da, lo_b = (uint32_t) db;
    constexpr uint32_t kStep = (T::kStageElems * 2) >> 4;
    int st = 0, acc = 0;
    uint32_t ph = 0, acc_ph = 1;
    bool ok = true;
    for (int item = blockIdx.x; ok && item < items; item += gridDim.x) {
      const int split = item / tiles, first = split * per_split, k_end = min(k_blocks, first + per_split);
      if (!(ok = tc::warp_wait(&bars.free_[acc], acc_ph, ctl))) break;
      for (int kb = first; kb < k_end; ++kb) {
        if (!(ok = tc::warp_wait(&bars.full[st], ph, ctl))) break;
        tc::fence_after_sync();
        tc::umma_ss_k64<A_MN ? 128 : 2, B_MN ? 128 : 2>(tmem + acc * BN, lo_a + st * kStep, hi_a, lo_b + st * kStep, hi_b, idesc, kb > first);
        tc::umma_commit_w(&bars.empty[st]);
        if (++st == T::kStages) { st = 0; ph ^= 1; }
      }
      if (!ok) break;
      tc::umma_commit_w(&bars.ready[acc]);
      acc ^= 1;
      if (acc == 0) acc_ph ^= 1;
    }
  } else if (warp >= 10) {
    // ---------------------------------------------------------------- movers: a chunk's residual or dy in, its result out
    if constexpr (KIND != kParts) {
      const int wg = warp - 10;
      Chunks<BN> head(tiles_n, items, out.N), tail(tiles_n, items, out.N);
      auto prepare = [&](int b) {                              // the buffer for the chunk at `head`
        uint64_t* bar = &bars.avail[wg * 2 + b];
        if (out.tma_in) {
          tma::expect_tx_w(bar, kChunkElems * 2);
          tma::load_2d_w(buffers + (wg * 2 + b) * kChunkElems, &maps.in, bar, (int) head.j0, (int) head.i0);
        } else if (lane == 0) {
          tma::mbar_arrive(bar);
        }
      };
      for (int b = 0; b < 2; ++b)
        if (head.next(wg)) prepare(b);
      uint32_t ph = 0;
      for (int b = 0; tail.next(wg); ph ^= b, b ^= 1) {
        if (!steady_wait(&bars.done[wg * 2 + b], ph, ctl)) break;
        if (out.tma_y) {
          tma::store_2d_w(&maps.y, (int) tail.j0, (int) tail.i0, tc::smem_u32(buffers + (wg * 2 + b) * kChunkElems));
          tma::reduce_commit_w();
          tma::reduce_wait_read();
          __syncwarp();
        }
        if (head.next(wg)) prepare(b);
      }
      tma::reduce_wait_all();
    }
  } else {
    // ---------------------------------------------------------------- epilogue; thread = row
    const int wg = warp >> 2, row = (warp & 3) * 32 + lane;
    int acc = 0, q = 0;
    uint32_t ph = 0;
    bool ok = true;
    auto accumulator_read = [&] {
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) tma::mbar_arrive(&bars.free_[acc]);
    };
    if constexpr (KIND == kParts) {
      constexpr int kCols = BN / 2;                            // a warpgroup half the columns, straight to memory: one tile or two per CTA
      for (int item = blockIdx.x; item < items; item += gridDim.x) {
        const int split = item / tiles, t = item - split * tiles;
        const int64_t r = (int64_t) (t / tiles_n) * kBM + row, j0 = (int64_t) (t % tiles_n) * BN + wg * kCols;
        ok = ok && __all_sync(0xffffffffu, tc::bounded_wait(&bars.ready[acc], ph, ctl));
        tc::fence_after_sync();
        const uint32_t src = tmem + ((uint32_t) ((warp & 3) * 32) << 16) + acc * BN + wg * kCols;
#pragma unroll 1
        for (int c = 0; c < kCols; c += 32) {
          float v[32];
          if (ok) {
            tc::tmem_ld32_async(src + c, v);
            tc::tmem_ld_wait(v);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(0x7fffffffu);
          }
          if (c + 32 == kCols) accumulator_read();
          if (r < out.M) {
            float* p = out.partial + ((int64_t) split * out.M + r) * out.ld + j0 + c;
#pragma unroll
            for (int i = 0; i < 32; i += 8)
              if (j0 + c + i < out.ld) stg256(p + i, reinterpret_cast<const uint32_t*>(v + i));      // ld is a multiple of 8
          }
        }
        acc ^= 1;
        if (acc == 0) ph ^= 1;
      }
    } else {
      constexpr int kChunks = BN / kChunk;
      const Epilogue<bf16>& e = out.e;
      float2 sums[KIND == kSlope ? kChunk / 2 : 1];            // slope: of this thread's rows; its columns stay the same (the grid is a multiple of tiles_n, BN = 128)
#pragma unroll
      for (int i = 0; i < (KIND == kSlope ? kChunk / 2 : 1); ++i) sums[i] = two(0.f);
      int seq = 0;
      for (int item = blockIdx.x; item < items; item += gridDim.x, ++q) {
        const int64_t i0 = (int64_t) (item / tiles_n) * kBM, r = i0 + row, jt = (int64_t) (item % tiles_n) * BN;
        const int64_t sample = KIND == kForward && e.gate.p && r < out.M ? (uint32_t) r / e.rows_per_gate : 0;
        ok = ok && __all_sync(0xffffffffu, tc::bounded_wait(&bars.ready[acc], ph, ctl));
        tc::fence_after_sync();
        bool read = false;
#pragma unroll 1
        for (int c = (q * kChunks + wg) & 1; c < kChunks; c += 2) {
          const int64_t j0 = jt + c * kChunk;
          if (j0 >= out.N) break;
          const int cols = (int) min((int64_t) kChunk, out.N - j0);
          float v[kChunk];
          if (ok) {
            const uint32_t src = tmem + ((uint32_t) ((warp & 3) * 32) << 16) + acc * BN + c * kChunk;
            tc::tmem_ld32_async(src, reinterpret_cast<float(&)[32]>(v[0]));
            tc::tmem_ld32_async(src + 32, reinterpret_cast<float(&)[32]>(v[32]));
            tc::tmem_ld_wait(reinterpret_cast<float(&)[32]>(v[0]));
            tc::tmem_ld_wait(reinterpret_cast<float(&)[32]>(v[32]));
          } else {
#pragma unroll
            for (int i = 0; i < kChunk; ++i) v[i] = __uint_as_float(0x7fffffffu);
          }
          if (c + 2 >= kChunks || j0 + 2 * kChunk >= out.N) {
            accumulator_read();
            read = true;
          }
          bf16* buf = buffers + (wg * 2 + (seq & 1)) * kChunkElems;
          if (!steady_wait(&bars.avail[wg * 2 + (seq & 1)], (uint32_t) (seq >> 1) & 1, ctl)) break;
          if (out.in.p && !out.tma_in) {                       // a warp's own rows, a row at a time
            for (int k = 0; k < 32; ++k) {
              const int64_t rr = i0 + (warp & 3) * 32 + k;
              const uint16_t* src = reinterpret_cast<const uint16_t*>(out.in.p + rr * out.in.ld + j0);
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int col = lane + 32 * h;
                *element(buf, (warp & 3) * 32 + k, col) = rr < out.M && col < cols ? src[col] : (uint16_t) 0;
              }
            }
            __syncwarp();
          }
#pragma unroll
          for (int g = 0; g < kChunk / 8; ++g) {
            float2 z[4], t[4];
            uint4* place = reinterpret_cast<uint4*>(buf + tc::swz(row, g));
#pragma unroll
            for (int i = 0; i < 4; ++i) z[i] = make_float2(v[8 * g + 2 * i], v[8 * g + 2 * i + 1]);
            if (e.bias) {
              unpack8(load8(e.bias + j0 + 8 * g, cols - 8 * g, true), t);
#pragma unroll
              for (int i = 0; i < 4; ++i) z[i] = __fadd2_rn(z[i], t[i]);
            }
            if constexpr (KIND == kForward) {
              if constexpr (ACT != kActNone) {
#pragma unroll
                for (int i = 0; i < 4; ++i) z[i] = activate2<ACT>(z[i]);
              } else {
                if (e.pre.p && r < out.M) {                    // kept for the gate's gradient
                  const uint4 w = pack8(z);
                  bf16* p = e.pre.p + r * e.pre.ld + j0 + 8 * g;
                  if (cols >= 8 * g + 8 && (e.pre.ld & 7) == 0) *reinterpret_cast<uint4*>(p) = w;
                  else
                    for (int i = 0; i < 8; ++i)
                      if (8 * g + i < cols) p[i] = __float2bfloat16_rn(i & 1 ? z[i / 2].y : z[i / 2].x);
                }
                if (e.gate.p) {
                  unpack8(load8(e.gate.p + sample * e.gate.ld + j0 + 8 * g, cols - 8 * g, out.vec_gate), t);
#pragma unroll
                  for (int i = 0; i < 4; ++i) z[i] = __fmul2_rn(z[i], t[i]);
                }
              }
              if (out.in.p) {
                unpack8(*place, t);
#pragma unroll
                for (int i = 0; i < 4; ++i) z[i] = __fadd2_rn(z[i], t[i]);
              }
            } else {
              unpack8(*place, t);
#pragma unroll
              for (int i = 0; i < 4; ++i) z[i] = __fmul2_rn(t[i], slope2<ACT>(z[i]));
              if (r < out.M)
#pragma unroll
                for (int i = 0; i < 4; ++i) sums[4 * g + i] = __fadd2_rn(sums[4 * g + i], z[i]);
            }
            *place = pack8(z);
          }
          tc::fence_async_smem();                              // what TMA stores from here, and loads into here next
          if (!out.tma_y) {
            __syncwarp();
            for (int k = 0; k < 32; ++k) {
              const int64_t rr = i0 + (warp & 3) * 32 + k;
              uint16_t* dst = reinterpret_cast<uint16_t*>(e.y.p + rr * e.y.ld + j0);
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int col = lane + 32 * h;
                if (rr < out.M && col < cols) dst[col] = *element(buf, (warp & 3) * 32 + k, col);
              }
            }
            tc::fence_async_smem();
          }
          __syncwarp();
          if (lane == 0) tma::mbar_arrive(&bars.done[wg * 2 + (seq & 1)]);
          ++seq;
        }
        if (!read) accumulator_read();
        acc ^= 1;
        if (acc == 0) ph ^= 1;
      }
      if constexpr (KIND == kSlope) {
        // 64 sums of 32 rows -> two columns a lane: each step hands half of what is left to the lane opposite
        float s[kChunk];
#pragma unroll
        for (int i = 0; i < kChunk / 2; ++i) { s[2 * i] = sums[i].x; s[2 * i + 1] = sums[i].y; }
#pragma unroll
        for (int o = 16, n = 32; o > 0; o >>= 1, n >>= 1) {
          const bool upper = lane & o;
#pragma unroll
          for (int i = 0; i < n; ++i) {
            const float give = upper ? s[i] : s[i + n], keep = upper ? s[i + n] : s[i];
            s[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
          }
        }
        s_sum[warp][2 * lane] = s[0];
        s_sum[warp][2 * lane + 1] = s[1];
        asm volatile("bar.sync %0, 128;" ::"r"(1 + wg) : "memory");
        const int64_t j = (int64_t) (blockIdx.x % tiles_n) * BN + wg * kChunk + row;
        if (out.partial && row < kChunk && j < out.N) {
          float u = 0.f;
#pragma unroll
          for (int k = 0; k < 4; ++k) u += s_sum[wg * 4 + k][row];
          out.partial[((int64_t) (blockIdx.x / tiles_n) * 2 + 1) * out.N + j] = u;
        }
      }
    }
  }
  if (ctl->abort) tc::abort_drain();
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  if (warp == 0) tc::tmem_dealloc(tmem, T::kTmemCols);
  if (tid == 0 && s_ctl.abort && status) atomicOr(status, LLSA_DEV_WAIT_EXPIRED);
}

// ------------------------------------------------------------------------------------------------ choice of the tile
// Cycles of a k-step of 64 by tile width: the products' (BN / 2 per 16 of k) or what the tile's operands take from shared memory at 128 bytes a cycle.
int64_t step_cycles(int bn) { return 4 * std::max(bn / 2, (kBM + bn) / 4); }
// Cycles of a tile outside its products where nothing hides them: fill of the ring and the last epilogue
constexpr int64_t kTileCycles = 1500;

struct Choice {
  int bn, split;
};
// The tile width, and with `parts` the number of parts, that a count of waves of 148 CTAs says is the fastest
Choice choose(int64_t M, int64_t N, int64_t k_blocks, bool parts) {
  Choice best = {64, 1};
  int64_t least = INT64_MAX;
  for (int bn : {64, 128, 192, 256}) {
    const int64_t tiles = (M + kBM - 1) / kBM * ((N + bn - 1) / bn);
    const int64_t most = parts ? std::max<int64_t>(1, std::min<int64_t>(k_blocks / 4, 148 / std::max<int64_t>(1, std::min<int64_t>(tiles, 148)))) : 1;
    for (int64_t s = 1; s <= most; ++s) {
      const int64_t waves = (tiles * s + 147) / 148, steps = (k_blocks + s - 1) / s;
      // a part's tile is written and read again once, at about 40 bytes a cycle of the SM
      const int64_t cost = waves * (steps * step_cycles(bn) + (parts ? kBM * bn * 8 / 40 : 0)) + kTileCycles + 4 * bn;
      if (cost < least) {
        least = cost;
        best = {bn, (int) s};
      }
    }
  }
#ifdef LLSA_BN
  if (LLSA_BN) best.bn = LLSA_BN;
#endif
  return best;
}

int matrix_map(CUtensorMap* m, const void* base, int64_t ld, int64_t rows, int64_t cols, uint32_t box_rows) {
  const uint64_t dims[2] = {(uint64_t) cols, (uint64_t) rows}, strides[1] = {(uint64_t) ld * 2};
  return tma::make_map(m, base, 2, dims, strides, box_rows);
}
template <typename T>
bool rows16(const Mat<T>& m) { return m.p && ((uintptr_t) m.p & 15) == 0 && m.ld % 8 == 0; }

template <int BN, bool A_MN, bool B_MN, int KIND, int ACT>
int launch(const Product<bf16>& p, Outputs& out, int64_t row_groups, int wait_limit, int32_t* status, cudaStream_t st) {
  using T = Tile<BN, KIND>;
  ProductMaps maps;
  int rc = A_MN ? matrix_map(&maps.a, p.a.p, p.a.ld, p.K, p.M, kBK) : matrix_map(&maps.a, p.a.p, p.a.ld, p.M, p.K, kBM);
  if (rc) return rc;
  rc = B_MN ? matrix_map(&maps.b, p.b.p, p.b.ld, p.K, p.N, kBK) : matrix_map(&maps.b, p.b.p, p.b.ld, p.N, p.K, BN);
  if (rc) return rc;
  maps.in = maps.y = maps.a;
  if (KIND != kParts) {
    out.tma_in = rows16(out.in);
    out.tma_y = rows16(out.e.y);
    out.vec_gate = rows16(out.e.gate);
    if (out.tma_in && (rc = matrix_map(&maps.in, out.in.p, out.in.ld, p.M, p.N, kBM))) return rc;
    if (out.tma_y && (rc = matrix_map(&maps.y, out.e.y.p, out.e.y.ld, p.M, p.N, kBM))) return rc;
  }
  const auto kernel = product_tc_kernel<BN, A_MN, B_MN, KIND, ACT>;
  LLSA_SMEM_LIMIT(kernel, T::kSmem);
  const int64_t tiles_n = (p.N + BN - 1) / BN, tiles = (p.M + kBM - 1) / kBM * tiles_n, k_blocks = (p.K + kBK - 1) / kBK;
  const int64_t per = (k_blocks + p.split - 1) / p.split, items = tiles * p.split;
  LLSA_REQUIRE(items <= INT32_MAX && p.M <= INT32_MAX - kBM && p.N <= INT32_MAX - BN && p.K <= INT32_MAX - kBK, LLSA_ERR_SHAPE, "linear: too many outputs");
  const int64_t grid = KIND == kSlope ? tiles_n * row_groups : std::min<int64_t>(items, 148);
  launch_pdl(kernel, dim3((unsigned) grid), dim3(kThreads), T::kSmem, st, maps, out, (int) k_blocks, (int) per, (int) tiles_n, (int) tiles, (int) items, wait_limit,
             status);
  LLSA_LAUNCH_OK("product_tc_kernel");
  return LLSA_OK;
}

template <bool A_MN, bool B_MN, int KIND, int ACT>
int launch_width(int bn, const Product<bf16>& p, Outputs& out, int wait_limit, int32_t* status, cudaStream_t st) {
  switch (bn) {
    case 64: return launch<64, A_MN, B_MN, KIND, ACT>(p, out, 0, wait_limit, status, st);
    case 128: return launch<128, A_MN, B_MN, KIND, ACT>(p, out, 0, wait_limit, status, st);
    case 192: return launch<192, A_MN, B_MN, KIND, ACT>(p, out, 0, wait_limit, status, st);
    default: return launch<256, A_MN, B_MN, KIND, ACT>(p, out, 0, wait_limit, status, st);
  }
}

Outputs outputs(const Product<bf16>& p, const Epilogue<bf16>& e, const Mat<const bf16>& in) {
  Outputs out = {};
  out.e = e;
  out.in = in;
  out.M = p.M;
  out.N = p.N;
  return out;
}

}  // namespace

int linear_tc_product(const Product<bf16>& p, const Epilogue<bf16>& e, int wait_limit, int32_t* status, cudaStream_t st) {
  Outputs out = outputs(p, e, e.residual);
  const int bn = choose(p.M, p.N, (p.K + kBK - 1) / kBK, false).bn;
  if (!p.b_k) return launch_width<false, true, kForward, kActNone>(bn, p, out, wait_limit, status, st);
  if (e.act == kActGeluTanh) return launch_width<false, false, kForward, kActGeluTanh>(bn, p, out, wait_limit, status, st);
  if (e.act == kActSilu) return launch_width<false, false, kForward, kActSilu>(bn, p, out, wait_limit, status, st);
  return launch_width<false, false, kForward, kActNone>(bn, p, out, wait_limit, status, st);
}

int64_t linear_tc_slope_groups(int64_t M, int64_t N) {
  const int64_t rows = (M + kBM - 1) / kBM, tiles_n = (N + 127) / 128;
  return std::max<int64_t>(1, std::min(rows, 148 / tiles_n));
}

int linear_tc_slope(const Product<bf16>& p, const Epilogue<bf16>& e, const Mat<const bf16>& dy, float* sums, int wait_limit, int32_t* status, cudaStream_t st) {
  Outputs out = outputs(p, e, dy);
  out.partial = sums;
  const int64_t groups = linear_tc_slope_groups(p.M, p.N);
  return e.act == kActGeluTanh ? launch<128, false, false, kSlope, kActGeluTanh>(p, out, groups, wait_limit, status, st)
                               : launch<128, false, false, kSlope, kActSilu>(p, out, groups, wait_limit, status, st);
}

int linear_tc_split(int64_t M, int64_t N, int64_t K) {
  const int64_t k_blocks = (K + kBK - 1) / kBK;
  const int s = choose(M, N, k_blocks, true).split;
  const int64_t per = (k_blocks + s - 1) / s;
  return (int) ((k_blocks + per - 1) / per);      // no part without a share
}

int linear_tc_parts(const Product<bf16>& p, float* partial, int64_t ld, int wait_limit, int32_t* status, cudaStream_t st) {
  Outputs out = outputs(p, {}, {});
  out.partial = partial;
  out.ld = ld;
  return launch_width<true, true, kParts, kActNone>(choose(p.M, p.N, (p.K + kBK - 1) / kBK, true).bn, p, out, wait_limit, status, st);
}

}  // namespace llsa
