// The projection's matrix products on tcgen05 (linear_tc.cu): the kernel and its launch.
#pragma once
#include <string.h>

#include "linear.cuh"
#include "tc05.cuh"
#include "tma.cuh"

namespace llsa {
namespace linear_tc {

using bf16 = __nv_bfloat16;

constexpr int kBM = 128, kBK = 64;
// Roles: G warpgroups of epilogue, the producer, the warp that issues the products, a mover to each warpgroup.  Three warpgroups hide the latencies of a long
// epilogue; two leave 32 KB more to the ring, which a long sum needs.  us, two / three, 131072 rows, tiles of 256 x 256: 384 -> 1536 with GELU 177 / 164, gated
// onto a residual 203 / 177, plain 136 / 149; 1536 -> 384 plain 150 / 159, gated 157 / 177.  Four leave a ring of three steps: GELU 183 where three take 167.
template <int G>
struct Roles {
  static constexpr int kEpilogueWarps = 4 * G, kProducer = kEpilogueWarps, kIssuer = kProducer + 1, kMover = kIssuer + 1, kThreads = 32 * (kMover + G);
};
constexpr int kChunk = 64, kChunkElems = kBM * kChunk;      // a chunk of the epilogue: 16 KB of bf16

enum Kind { kForward, kSlope, kParts };

struct ProductMaps {
  CUtensorMap a, b, in, y;      // in: residual or dy
};

// A CTA's share: 128 rows of A and, of a pair, half the columns of B (MN-major in whole groups of 64)
template <int BN, bool PAIR, bool B_MN, int KIND, int G>
struct Tile {
  static constexpr int kBCols = PAIR ? BN / 2 : BN, kBElems = (B_MN ? (kBCols + 63) / 64 * 64 : kBCols) * kBK;
  static constexpr int kStageElems = kBM * kBK + kBElems;
  // what 227 KB hold beside the epilogue's buffers
  static constexpr int kRoom = (KIND == kParts ? 225 : 225 - 32 * G) * 512, kStages = kRoom / kStageElems < 8 ? kRoom / kStageElems : 8;
  static constexpr int kTmemCols = BN == 64 ? 128 : BN == 128 ? 256 : 512;
  static constexpr int kBuffers = KIND == kParts ? 0 : 2 * G;
  static constexpr size_t kSmem = ((size_t) kStages * kStageElems + (size_t) kBuffers * kChunkElems) * 2 + 1024;
};

template <int G>
struct Bars {
  uint64_t full[8], empty[8], ready[2], free_[2], avail[2 * G], done[2 * G];      // avail, done: warpgroup * 2 + buffer
};

struct Outputs {
  Epilogue<bf16> e;
  Mat<const bf16> in;        // residual or dy
  float* partial;            // parts: [part][M][ld]; slope: [CTAs of a column][2][N], the sums in the second row
  int64_t ld;
  int64_t M, N;              // M: of a sample, where there are several
  int vec_pre;
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
// s + z s (1 - s) u'(z).  Beyond +-7 (SiLU: +-30) the slope is 1 or within 4e-14 (3e-12) of 0, and z stays there: 2^t then stays below 2^52 and both of a pair's
// reciprocals come from one.  The special functions, 16 a cycle, are what paces the kernel: three for two values instead of four.  A NaN stands in for itself
// alone: it goes in with the last factor, and the shared reciprocal sees a number in its place.
template <int ACT>
__device__ __forceinline__ float2 slope2(float2 z) {
  constexpr float kFar = ACT == kActGeluTanh ? 7.f : 30.f;
  z = make_float2(clamp_nan(z.x, kFar), clamp_nan(z.y, kFar));
  const float2 c = make_float2(fmaxf(z.x, -kFar), fmaxf(z.y, -kFar)), q = __fmul2_rn(c, c);
  float2 t;
  if constexpr (ACT == kActGeluTanh) t = __fmul2_rn(c, __ffma2_rn(q, two(-kGelu2 * kGelu3 * kLog2e), two(-kGelu2 * kLog2e)));
  else t = __fmul2_rn(c, two(-kLog2e));
  const float2 d = __fadd2_rn(make_float2(ex2(t.x), ex2(t.y)), two(1.f));
  const float r = rcp(d.x * d.y);
  const float2 s = make_float2(r * d.y, r * d.x);
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
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 x;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(a) : "memory");
  return x;
}
__device__ __forceinline__ void sts128(uint32_t a, const uint4& x) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w) : "memory");
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

// The tiles of a CTA (or pair), in order: every `units`th, columns fastest.  No division on the way: a role's warp has nothing to hide it behind
struct Walk {
  int item, i, j;               // tile: row i, column j
  int units, di, dj, tiles_n;
  __device__ __forceinline__ Walk(int unit, int units_, int tiles_n_) : item(unit), units(units_), tiles_n(tiles_n_) {
    i = unit / tiles_n;
    j = unit - i * tiles_n;
    di = units / tiles_n;
    dj = units - di * tiles_n;
  }
  __device__ __forceinline__ void step() {
    item += units;
    i += di;
    j += dj;
    if (j >= tiles_n) { j -= tiles_n; ++i; }
  }
};
// The chunks of 64 columns of a CTA's tiles that one warpgroup owns, in order: one of G of all its tiles' chunks; of a tile of the slope, which has at most
// three, always the same one (its column sums stay in registers)
template <int BN, int KIND, int G>
struct Chunks {
  static constexpr int kChunks = BN / kChunk;
  static_assert(KIND != kSlope || kChunks <= G, "one chunk of a tile to a warpgroup");
  Walk w;
  int c, wg, first, items, N;   // the next chunk of the tile; the warpgroup of the tile's first chunk
  __device__ __forceinline__ Chunks(const Walk& walk, int wg_, int items_, int n) : w(walk), c(wg_), wg(wg_), first(0), items(items_), N(n) {}
  __device__ __forceinline__ void next_tile() {
    w.step();
    if (KIND != kSlope) first = (first + kChunks) % G;
    c = wg - first + (wg < first ? G : 0);
  }
  __device__ __forceinline__ bool in_tile() const { return c < kChunks && w.j * BN + c * kChunk < N; }
  // Moves to the next owned chunk with columns in it, which stays at (w.i, j0()) until it is taken; false: none is left
  __device__ __forceinline__ bool find() {
    for (; w.item < items; next_tile())
      if (in_tile()) return true;
    return false;
  }
  __device__ __forceinline__ int j0() const { return w.j * BN + c * kChunk; }
  __device__ __forceinline__ void take() { c += G; }
};

// ------------------------------------------------------------------------------------------------ kernel
// items: (part, row tile, column tile), columns fastest.  k_blocks: steps of 64; per_split: those of a part.
// IN: the epilogue reads a tile (residual, dy); GATED: it multiplies by a gate and may keep z
// TMA: the movers bring and store the epilogue's tiles; else the epilogue's warps do, for rows that are on no 16-byte boundary.
// SAMPLES: the maps have a third dimension, the sample; row tiles, or the parts of a sum over rows, are a sample's each, `per_sample` of them
template <int BN, bool PAIR, bool A_MN, bool B_MN, int KIND, int ACT, bool IN, bool GATED, int G, bool SAMPLES, bool TMA>
__global__ void __launch_bounds__(Roles<G>::kThreads, 1)
product_tc_kernel(const __grid_constant__ ProductMaps maps, const __grid_constant__ Outputs out, int k_blocks, int per_split, int tiles_n, int tiles, int items,
                  int per_sample, int wait_limit, int32_t* status) {
  using T = Tile<BN, PAIR, B_MN, KIND, G>;
  using R = Roles<G>;
  extern __shared__ unsigned char smem_dyn[];
  __shared__ Bars<G> bars;
  __shared__ uint32_t s_tmem;
  __shared__ tc::WaitCtl s_ctl;
  __shared__ __align__(16) uint16_t s_col[KIND == kParts ? 1 : 2][G][2 * kChunk];      // bias and gate of a warpgroup's chunk
  bf16* ring = reinterpret_cast<bf16*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
  bf16* buffers = ring + T::kStages * T::kStageElems;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile tc::WaitCtl* ctl = &s_ctl;
  const int rank = PAIR ? blockIdx.x & 1 : 0, unit = blockIdx.x >> PAIR, units = gridDim.x >> PAIR;      // units: CTAs, or pairs
  const int row0 = rank * kBM;                                 // of a tile of kBM << PAIR rows
  [[maybe_unused]] const int rows_m = tiles / tiles_n;         // rows of tiles
  if (tid == 0) {
    s_ctl.abort = 0;
    s_ctl.limit = wait_limit > 0 ? wait_limit : tc::kWaitPolls;
    for (int i = 0; i < T::kStages; ++i) { tc::mbar_init(&bars.full[i], 1); tc::mbar_init(&bars.empty[i], 1); }
    for (int i = 0; i < 2; ++i) { tc::mbar_init(&bars.ready[i], 1); tc::mbar_init(&bars.free_[i], R::kEpilogueWarps << PAIR); }
    for (int i = 0; i < 2 * G; ++i) { tc::mbar_init(&bars.avail[i], 1); tc::mbar_init(&bars.done[i], 4); }
    tc::fence_mbar_init();
  }
  pdl_wait();
  if (warp == 0) {
    if constexpr (PAIR) tc::tmem_alloc_pair(&s_tmem, T::kTmemCols);
    else tc::tmem_alloc(&s_tmem, T::kTmemCols);
  }
  tc::fence_before_sync();
  if constexpr (PAIR) tc::cluster_sync_all();                  // the other CTA's barriers are there
  else __syncthreads();
  tc::fence_after_sync();
  pdl_trigger();
  const uint32_t tmem = s_tmem;

  if (warp == R::kProducer) {
    // ---------------------------------------------------------------- TMA producer: this CTA's operands; of a pair, on the barriers of rank 0
    int st = 0;
    uint32_t ph = 1;
    bool ok = true;
    for (Walk w(unit, units, tiles_n); ok && w.item < items; w.step()) {
      const int split = KIND == kParts ? w.item / tiles : 0, sample = SAMPLES ? (KIND == kParts ? split : w.i) / per_sample : 0;
      const int i0 = (w.i - (KIND == kParts ? split * rows_m : sample * per_sample)) * (kBM << PAIR) + row0, j0 = w.j * BN + rank * T::kBCols;
      const int part = KIND == kParts ? split - sample * per_sample : 0, k_end = min(k_blocks, (part + 1) * per_split);
      for (int kb = part * per_split; kb < k_end; ++kb) {
        if (!(ok = tc::warp_wait(&bars.empty[st], ph, ctl))) break;
        bf16* a = ring + st * T::kStageElems;
        bf16* b = a + kBM * kBK;
        uint64_t* bar = &bars.full[st];
        if (rank == 0) tma::expect_tx_w(bar, (T::kStageElems * 2) << PAIR);
        const uint32_t to = PAIR ? tc::at_rank(bar, 0) : 0;
        auto load = [&](bf16* dst, const CUtensorMap* map, int c0, int c1) {
          if constexpr (SAMPLES && PAIR) tma::load_3d_pair_w(dst, map, to, c0, c1, sample);
          else if constexpr (SAMPLES) tma::load_3d_w(dst, map, bar, c0, c1, sample);
          else if constexpr (PAIR) tma::load_2d_pair_w(dst, map, to, c0, c1);
          else tma::load_2d_w(dst, map, bar, c0, c1);
        };
        if constexpr (A_MN) {
#pragma unroll
          for (int g = 0; g < kBM / 64; ++g) load(a + g * 64 * kBK, &maps.a, i0 + 64 * g, kb * kBK);
        } else {
          load(a, &maps.a, kb * kBK, i0);
        }
        if constexpr (B_MN) {
#pragma unroll
          for (int g = 0; g < (T::kBCols + 63) / 64; ++g) load(b + g * 64 * kBK, &maps.b, j0 + 64 * g, kb * kBK);
        } else {
          load(b, &maps.b, kb * kBK, j0);
        }
        if (++st == T::kStages) { st = 0; ph ^= 1; }
      }
    }
  } else if (warp == R::kIssuer) {
    // ---------------------------------------------------------------- products; of a pair, by rank 0
    const uint32_t idesc = tc::instr_desc(kBM << PAIR, BN, A_MN, B_MN);
    // K-major: 8 rows of 128 bytes follow one another; MN-major: 64 columns further on stands 64 rows (8 KB) behind
    const uint64_t da = tc::smem_desc(tc::smem_u32(ring), A_MN ? 8192 : 16, 1024), db = tc::smem_desc(tc::smem_u32(ring + kBM * kBK), B_MN ? 8192 : 16, 1024);
    const uint32_t hi_a = (uint32_t) (da >> 32), hi_b = (uint32_t) (db >> 32), lo_a = (uint32_t) da, lo_b = (uint32_t) db;
    constexpr uint32_t kStep = (T::kStageElems * 2) >> 4;
    constexpr int kAS = A_MN ? 128 : 2, kBS = B_MN ? 128 : 2;
    auto commit = [](uint64_t* bar) {
      if constexpr (PAIR) tc::umma_commit_pair_w(bar);
      else tc::umma_commit_w(bar);
    };
    int st = 0, acc = 0;
    uint32_t ph = 0, acc_ph = 1;
    bool ok = true;
    for (int item = unit; ok && rank == 0 && item < items; item += units) {
      const int split = KIND == kParts ? item / tiles : 0, first = (SAMPLES && KIND == kParts ? split % per_sample : split) * per_split, k_end = min(k_blocks, first + per_split);
      if (!(ok = tc::warp_wait(&bars.free_[acc], acc_ph, ctl))) break;
      for (int kb = first; kb < k_end; ++kb) {
        if (!(ok = tc::warp_wait(&bars.full[st], ph, ctl))) break;
        tc::fence_after_sync();
        if constexpr (PAIR) tc::umma_pair_ss_k64<kAS, kBS>(tmem + acc * BN, lo_a + st * kStep, hi_a, lo_b + st * kStep, hi_b, idesc, kb > first);
        else tc::umma_ss_k64<kAS, kBS>(tmem + acc * BN, lo_a + st * kStep, hi_a, lo_b + st * kStep, hi_b, idesc, kb > first);
        commit(&bars.empty[st]);
        if (++st == T::kStages) { st = 0; ph ^= 1; }
      }
      if (!ok) break;
      commit(&bars.ready[acc]);
      acc ^= 1;
      if (acc == 0) acc_ph ^= 1;
    }
  } else if (warp >= R::kMover) {
    // ---------------------------------------------------------------- movers: a chunk's residual or dy in, its result out
    if constexpr (KIND != kParts) {
      const int wg = warp - R::kMover;
      Chunks<BN, KIND, G> head(Walk(unit, units, tiles_n), wg, items, (int) out.N), tail(head);
      auto prepare = [&](int b) {                              // the buffer for the chunk at `head`
        uint64_t* bar = &bars.avail[wg * 2 + b];
        if (IN && TMA) {
          tma::expect_tx_w(bar, kChunkElems * 2);
          tma::load_2d_w(buffers + (wg * 2 + b) * kChunkElems, &maps.in, bar, head.j0(), head.w.i * (kBM << PAIR) + row0);
        } else if (lane == 0) {
          tma::mbar_arrive(bar);
        }
        head.take();
      };
      for (int b = 0; b < 2; ++b)
        if (head.find()) prepare(b);
      uint32_t ph = 0;
      for (int b = 0; tail.find(); ph ^= b, b ^= 1, tail.take()) {
        if (!steady_wait(&bars.done[wg * 2 + b], ph, ctl)) break;
        const bf16* buf = buffers + (wg * 2 + b) * kChunkElems;
        const int sample = SAMPLES ? tail.w.i / per_sample : 0, i0 = (tail.w.i - sample * per_sample) * (kBM << PAIR) + row0;
        const bool store = TMA && i0 < out.M;
        if (store) {
          if constexpr (SAMPLES) tma::store_3d_w(&maps.y, tail.j0(), i0, sample, tc::smem_u32(buf));
          else tma::store_2d_w(&maps.y, tail.j0(), i0, tc::smem_u32(buf));
          tma::reduce_commit_w();
        }
        if (store) tma::reduce_wait_read();
        __syncwarp();
        if (head.find()) prepare(b);
      }
      tma::reduce_wait_all();
    }
  } else {
    // ---------------------------------------------------------------- epilogue; thread = row
    const int wg = warp >> 2, row = (warp & 3) * 32 + lane;
    int acc = 0;
    uint32_t ph = 0;
    bool ok = true;
    auto accumulator_read = [&] {
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR) tc::arrive_remote(tc::at_rank(&bars.free_[acc], 0));
        else tma::mbar_arrive(&bars.free_[acc]);
      }
    };
    if constexpr (KIND == kParts) {
      for (Walk w(unit, units, tiles_n); w.item < items; w.step()) {
        const int split = w.item / tiles;
        const int64_t r = (int64_t) (w.i - split * rows_m) * (kBM << PAIR) + row0 + row, j0 = (int64_t) w.j * BN;
        ok = ok && __all_sync(0xffffffffu, tc::bounded_wait(&bars.ready[acc], ph, ctl));
        tc::fence_after_sync();
        const uint32_t src = tmem + ((uint32_t) ((warp & 3) * 32) << 16) + acc * BN;
#pragma unroll 1
        for (int c = 32 * wg; c < BN; c += 32 * G) {     // straight to memory: a tile or two per CTA
          float v[32];
          if (ok) {
            tc::tmem_ld32_async(src + c, v);
            tc::tmem_ld_wait(v);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(0x7fffffffu);
          }
          if (r < out.M) {
            float* p = out.partial + ((int64_t) split * out.M + r) * out.ld + j0 + c;
#pragma unroll
            for (int i = 0; i < 32; i += 8)
              if (j0 + c + i < out.ld) stg256(p + i, reinterpret_cast<const uint32_t*>(v + i));      // ld is a multiple of 8
          }
        }
        accumulator_read();
        acc ^= 1;
        if (acc == 0) ph ^= 1;
      }
    } else {
      const Epilogue<bf16>& e = out.e;
      const int t = tid & 127, M = (int) out.M, N = (int) out.N;
      float2 sums[KIND == kSlope ? 8 : 1];                     // slope: of this thread's 16 columns and its rows, before they are rounded
#pragma unroll
      for (int i = 0; i < (KIND == kSlope ? 8 : 1); ++i) sums[i] = two(0.f);
      int seq = 0;
      for (Chunks<BN, KIND, G> own(Walk(unit, units, tiles_n), wg, items, N); own.w.item < items; own.next_tile()) {
        const int i0 = own.w.i * (kBM << PAIR) + row0, r = i0 + row;
        uint32_t sample = 0;                                   // of the first row
        bool mixed = false;                                    // more samples than one in these rows: a thread reads its own row's gate
        if (GATED && i0 < M) {
          sample = (uint32_t) i0 / e.rows_per_gate;
          mixed = (uint32_t) min(i0 + kBM - 1, M - 1) / e.rows_per_gate != sample;
        }
        // bias (half of the threads) and gate (the others) of the warpgroup's one or two chunks, on their way while the products end
        uint16_t col[2] = {0, 0};
        const bf16* src_col = t < kChunk ? e.bias : GATED && !mixed ? e.gate.p + sample * e.gate.ld : nullptr;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int j = own.j0() + k * G * kChunk + (t & (kChunk - 1));
          if (src_col && own.c + k * G < BN / kChunk && j < N) col[k] = reinterpret_cast<const uint16_t*>(src_col)[j];
        }
        ok = ok && __all_sync(0xffffffffu, tc::bounded_wait(&bars.ready[acc], ph, ctl));
        tc::fence_after_sync();
        bool read = false;
#pragma unroll 1
        for (int k0 = 0; own.in_tile(); own.take(), k0 = 1) {
          const int j0 = own.j0(), cols = min(kChunk, N - j0), b = seq & 1;
          const bool last = own.c + G >= BN / kChunk || j0 + G * kChunk >= N;
          bf16* buf = buffers + (wg * 2 + b) * kChunkElems;
          s_col[b][wg][t] = col[k0];
          asm volatile("bar.sync %0, 128;" ::"r"(1 + wg) : "memory");
          if (!steady_wait(&bars.avail[wg * 2 + b], (uint32_t) (seq >> 1) & 1, ctl)) break;
          if constexpr (IN && !TMA) {                             // a warp's own rows, a row at a time
#pragma unroll 1
            for (int k = 0; k < 32; k += 8) {                  // eight on their way at once
              uint16_t u[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const int64_t rr = i0 + (warp & 3) * 32 + k + i / 2;
                const int x = lane + 32 * (i & 1);
                u[i] = rr < M && x < cols ? reinterpret_cast<const uint16_t*>(out.in.p + rr * out.in.ld + j0)[x] : (uint16_t) 0;
              }
#pragma unroll
              for (int i = 0; i < 16; ++i) *element(buf, (warp & 3) * 32 + k + i / 2, lane + 32 * (i & 1)) = u[i];
            }
            __syncwarp();
          }
          // chunk c of this thread's row of the buffer stands at at ^ 16 c
          const uint32_t at = tc::smem_u32(buf) + row * 128 + ((row & 7) << 4), col_at = tc::smem_u32(&s_col[b][wg][0]);
          if (!ok) {                                           // the products never came
#pragma unroll
            for (int g = 0; g < 8; ++g) sts128(at ^ (g << 4), make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu));
          } else if constexpr (KIND == kSlope) {
            // Spread as the accumulators of small products are (tc05.cuh: tmem_ld_16x64), not a row to a thread: a thread then has 16 columns and not 64, whose
            // sums fit its registers and whose bias it unpacks once for four rows.  The buffer's 8 x 8 pieces go through ldmatrix and stmatrix
            const uint32_t src = tmem + ((uint32_t) ((warp & 3) * 32) << 16) + acc * BN + own.c * kChunk;
            uint32_t bias[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) bias[j] = *reinterpret_cast<const uint32_t*>(&s_col[b][wg][8 * j + 2 * (lane & 3)]);
#pragma unroll 1
            for (int h = 0; h < 32; h += 16) {
              float v[32];
              tc::tmem_ld_16x64(src + ((uint32_t) h << 16), v);
              if (h) accumulator_read();                       // a tile has one chunk for this warpgroup
              if (i0 + kBM > M) {                              // rows that are not there: zeros times an infinite weight are no numbers, which the sums would keep
                const int lo = i0 + (warp & 3) * 32 + h + (lane >> 2);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                  if (lo >= M) v[4 * j] = v[4 * j + 1] = 0.f;
                  if (lo + 8 >= M) v[4 * j + 2] = v[4 * j + 3] = 0.f;
                }
              }
              // this lane's row of the pieces it addresses: rows 0-7 or 8-15 (lane bit 3) of columns j or j + 1 (bit 4)
              const int pr = (warp & 3) * 32 + h + (lane & 15);
              const uint32_t piece = tc::smem_u32(buf) + pr * 128 + ((pr & 7) << 4);
#pragma unroll
              for (int j = 0; j < 8; j += 2) {
                uint32_t d[4];
                const uint32_t a = piece ^ ((j + (lane >> 4)) << 4);
                asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3]) : "r"(a) : "memory");
#pragma unroll
                for (int i = 0; i < 4; ++i) {                  // (rows, columns): (low, j), (high, j), (low, j + 1), (high, j + 1)
                  const int jj = j + i / 2;
                  const float2 z = __fadd2_rn(make_float2(v[4 * jj + 2 * (i & 1)], v[4 * jj + 2 * (i & 1) + 1]), make_float2(bf16_lo(bias[jj]), bf16_hi(bias[jj])));
                  const float2 dz = __fmul2_rn(make_float2(bf16_lo(d[i]), bf16_hi(d[i])), slope2<ACT>(z));
                  sums[jj] = __fadd2_rn(sums[jj], dz);
                  d[i] = pack_bf16(dz.x, dz.y);
                }
                asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(d[0]), "r"(d[1]), "r"(d[2]), "r"(d[3]) : "memory");
              }
            }
            read = true;
          } else {
            const uint32_t src = tmem + ((uint32_t) ((warp & 3) * 32) << 16) + acc * BN + own.c * kChunk;
            // In a loop where an activation makes it long: two warps a scheduler, and every instruction fetched once a chunk is waited for
#pragma unroll (ACT == kActNone && !GATED ? 2 : 1)
            for (int x = 0; x < kChunk; x += 32) {
              float v[32];
              tc::tmem_ld32_async(src + x, v);
              tc::tmem_ld_wait(v);
              if (last && x + 32 == kChunk) accumulator_read();
#pragma unroll
              for (int g = 0; g < 4; ++g) {
                float2 z[4], u[4];
                const uint32_t place = (at ^ (x << 1)) ^ (g << 4);
                unpack8(lds128(col_at + 2 * x + 16 * g), u);
#pragma unroll
                for (int i = 0; i < 4; ++i) z[i] = __fadd2_rn(make_float2(v[8 * g + 2 * i], v[8 * g + 2 * i + 1]), u[i]);
#pragma unroll
                for (int i = 0; i < 4; ++i) z[i] = activate2<ACT>(z[i]);
                if constexpr (GATED) {
                  if (e.pre.p && r < M) {                    // kept for the gate's gradient
                    uint16_t* to = reinterpret_cast<uint16_t*>(e.pre.p + (int64_t) r * e.pre.ld + j0 + x + 8 * g);
                    const uint4 p = pack8(z);
                    if (out.vec_pre && x + 8 * g + 8 <= cols) *reinterpret_cast<uint4*>(to) = p;
                    else
#pragma unroll
                      for (int i = 0; i < 8; ++i)
                        if (x + 8 * g + i < cols) to[i] = (uint16_t) ((i < 2 ? p.x : i < 4 ? p.y : i < 6 ? p.z : p.w) >> (16 * (i & 1)));
                  }
                  if (!mixed) {
                    unpack8(lds128(col_at + 2 * kChunk + 2 * x + 16 * g), u);
                  } else {
                    const uint16_t* own = reinterpret_cast<const uint16_t*>(e.gate.p + (int64_t) ((uint32_t) min(r, M - 1) / e.rows_per_gate) * e.gate.ld + j0);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                      const int k = x + 8 * g + 2 * i;
                      u[i] = make_float2(k < cols ? bf16_lo(own[k]) : 0.f, k + 1 < cols ? bf16_lo(own[k + 1]) : 0.f);
                    }
                  }
#pragma unroll
                  for (int i = 0; i < 4; ++i) z[i] = __fmul2_rn(z[i], u[i]);
                }
                if constexpr (IN) {
                  unpack8(lds128(place), u);
#pragma unroll
                  for (int i = 0; i < 4; ++i) z[i] = __fadd2_rn(z[i], u[i]);
                }
                sts128(place, pack8(z));
              }
            }
            read = last;
          }
          tc::fence_async_smem();                              // what TMA stores from here, and loads into here next
          if constexpr (!TMA) {
            __syncwarp();
#pragma unroll 1
            for (int k = 0; k < 32; k += 8) {
              uint16_t u[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) u[i] = *element(buf, (warp & 3) * 32 + k + i / 2, lane + 32 * (i & 1));
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const int64_t rr = i0 + (warp & 3) * 32 + k + i / 2;
                const int x = lane + 32 * (i & 1);
                if (rr < M && x < cols) reinterpret_cast<uint16_t*>(e.y.p + rr * e.y.ld + j0)[x] = u[i];
              }
            }
            tc::fence_async_smem();
          }
          __syncwarp();
          if (lane == 0) tma::mbar_arrive(&bars.done[wg * 2 + b]);
          ++seq;
        }
        if (!read) accumulator_read();
        acc ^= 1;
        if (acc == 0) ph ^= 1;
      }
      if constexpr (KIND == kSlope) {
        // the columns of a CTA stay the same (its units are a multiple of tiles_n): one sum over its rows.  Lanes 4 apart have the same columns
#pragma unroll
        for (int i = 0; i < 8; ++i) {
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) {
            sums[i].x += __shfl_xor_sync(0xffffffffu, sums[i].x, o);
            sums[i].y += __shfl_xor_sync(0xffffffffu, sums[i].y, o);
          }
        }
        float* s_sum = reinterpret_cast<float*>(ring);         // the last product has read the ring
        asm volatile("bar.sync %0, 128;" ::"r"(1 + wg) : "memory");
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (lane < 4) *reinterpret_cast<float2*>(s_sum + warp * kChunk + 8 * i + 2 * lane) = sums[i];
        asm volatile("bar.sync %0, 128;" ::"r"(1 + wg) : "memory");
        const int j = unit % tiles_n * BN + wg * kChunk + row;
        if (out.partial && wg < BN / kChunk && row < kChunk && j < N) {
          float u = 0.f;
#pragma unroll
          for (int k = 0; k < 4; ++k) u += s_sum[(wg * 4 + k) * kChunk + row];
          if (ctl->abort) u = __uint_as_float(0x7fffffffu);      // tiles are missing, and copies may still land in the ring
          out.partial[((int64_t) ((unit / tiles_n) << PAIR | rank) * 2 + 1) * N + j] = u;
        }
      }
    }
  }
  if (ctl->abort) tc::abort_drain();
  __syncwarp();
  tc::fence_before_sync();
  if constexpr (PAIR) tc::cluster_sync_all();                  // and nothing of the other CTA arrives here any more
  else __syncthreads();
  tc::fence_after_sync();
  if (warp == 0) {
    if constexpr (PAIR) tc::tmem_dealloc_pair(tmem, T::kTmemCols);
    else tc::tmem_dealloc(tmem, T::kTmemCols);
  }
  if (tid == 0 && s_ctl.abort && status) atomicOr(status, LLSA_DEV_WAIT_EXPIRED);
}

// ------------------------------------------------------------------------------------------------ launch
struct Choice {
  int bn;
  bool pair;
  int split = 1;
  int64_t cost = 0;             // cycles, as choose() counts them
};
// Slope: units (CTAs or pairs) that share a column of tiles
inline int64_t slope_rows(int64_t M, int64_t N, int bn, bool pair) {
  const int64_t rows = pair ? 2 * kBM : kBM, tiles_n = (N + bn - 1) / bn;
  return std::max<int64_t>(1, std::min((M + rows - 1) / rows, (pair ? 74 : 148) / tiles_n));
}

// samples: 0 for a matrix, else that many of them, `apart` elements from one to the next
inline int matrix_map(CUtensorMap* m, const void* base, int64_t ld, int64_t rows, int64_t cols, uint32_t box_rows, int64_t samples, int64_t apart) {
  const uint64_t dims[3] = {(uint64_t) cols, (uint64_t) rows, (uint64_t) samples}, strides[2] = {(uint64_t) ld * 2, (uint64_t) apart * 2};
  return tma::make_map(m, base, samples ? 3 : 2, dims, strides, box_rows);
}
// Rows of `cols` on 16-byte boundaries that do not overlap
template <typename T>
inline bool rows16(const Mat<T>& m, int64_t cols) { return m.p && ((uintptr_t) m.p & 15) == 0 && m.ld % 8 == 0 && m.ld >= cols; }

template <int BN, bool PAIR, bool A_MN, bool B_MN, int KIND, int ACT, bool IN, bool GATED, int G, bool SAMPLES, bool TMA>
int launch(const Product<bf16>& p, Outputs& out, int wait_limit, int32_t* status, cudaStream_t st) {
  using T = Tile<BN, PAIR, B_MN, KIND, G>;
  using R = Roles<G>;
  ProductMaps maps;
  int rc = A_MN ? matrix_map(&maps.a, p.a.p, p.a.ld, p.K, p.M, kBK, p.samples, p.K * p.a.ld) : matrix_map(&maps.a, p.a.p, p.a.ld, p.M, p.K, kBM, p.samples, p.M * p.a.ld);
  if (rc) return rc;
  rc = B_MN ? matrix_map(&maps.b, p.b.p, p.b.ld, p.K, p.N, kBK, p.samples, p.K * p.b.ld) : matrix_map(&maps.b, p.b.p, p.b.ld, p.N, p.K, T::kBCols, 0, 0);
  if (rc) return rc;
  maps.in = maps.y = maps.a;
  if (KIND != kParts) {
    out.vec_pre = rows16(out.e.pre, p.N);
    if (IN && TMA && (rc = matrix_map(&maps.in, out.in.p, out.in.ld, p.M, p.N, kBM, 0, 0))) return rc;
    if (TMA && (rc = matrix_map(&maps.y, out.e.y.p, out.e.y.ld, p.M, p.N, kBM, p.samples, p.M * out.e.y.ld))) return rc;
  }
  const auto kernel = product_tc_kernel<BN, PAIR, A_MN, B_MN, KIND, ACT, IN, GATED, G, SAMPLES, TMA>;
  LLSA_SMEM_LIMIT(kernel, T::kSmem);
  constexpr int64_t kRows = kBM << PAIR, kUnits = PAIR ? 74 : 148;
  const int64_t tiles_n = (p.N + BN - 1) / BN, k_blocks = (p.K + kBK - 1) / kBK, tiles_m = (p.M + kRows - 1) / kRows;
  // samples: of their own row tiles, or (parts) of their own parts of the sum
  const int64_t tiles = tiles_m * tiles_n * (SAMPLES && KIND != kParts ? p.samples : 1), parts = p.split * (SAMPLES && KIND == kParts ? p.samples : 1);
  LLSA_REQUIRE(p.N <= INT32_MAX / 2, LLSA_ERR_SHAPE, "linear: too many features");
  const int64_t per = (k_blocks + p.split - 1) / p.split, items = tiles * parts;
  LLSA_REQUIRE(items <= INT32_MAX / 4 && p.M <= INT32_MAX - 2 * kBM && p.N <= INT32_MAX - BN && p.K <= INT32_MAX - kBK, LLSA_ERR_SHAPE, "linear: too many outputs");
  const int64_t units = KIND == kSlope ? tiles_n * slope_rows(p.M, p.N, BN, PAIR) : std::min(items, kUnits);
  launch_pdl_cluster(kernel, dim3((unsigned) (units << PAIR)), dim3(R::kThreads), PAIR ? 2u : 1u, T::kSmem, st, maps, out, (int) k_blocks, (int) per, (int) tiles_n,
                     (int) tiles, (int) items, (int) (KIND == kParts ? p.split : tiles_m), wait_limit, status);
  LLSA_LAUNCH_OK("product_tc_kernel");
  return LLSA_OK;
}

// The tiles that are built: 128 x 64 (not slope) and 128 x 128 of one CTA, 256 x 192 and 256 x 256 (not slope) of a pair
template <bool A_MN, bool B_MN, int KIND, int ACT, bool IN, bool GATED, int G, bool SAMPLES, bool TMA>
int launch_tile(const Choice& c, const Product<bf16>& p, Outputs& out, int wait_limit, int32_t* status, cudaStream_t st) {
  if (c.pair) {
    if constexpr (KIND != kSlope)
      if (c.bn == 256) return launch<256, true, A_MN, B_MN, KIND, ACT, IN, GATED, G, SAMPLES, TMA>(p, out, wait_limit, status, st);
    return launch<192, true, A_MN, B_MN, KIND, ACT, IN, GATED, G, SAMPLES, TMA>(p, out, wait_limit, status, st);
  }
  if constexpr (KIND != kSlope)
    if (c.bn == 64) return launch<64, false, A_MN, B_MN, KIND, ACT, IN, GATED, G, SAMPLES, TMA>(p, out, wait_limit, status, st);
  return launch<128, false, A_MN, B_MN, KIND, ACT, IN, GATED, G, SAMPLES, TMA>(p, out, wait_limit, status, st);
}
template <bool A_MN, bool B_MN, int KIND, int ACT, bool IN, bool GATED, int G, bool SAMPLES = false>
int launch_choice(const Choice& c, const Product<bf16>& p, Outputs& out, int wait_limit, int32_t* status, cudaStream_t st) {
  if constexpr (KIND == kParts || SAMPLES) return launch_tile<A_MN, B_MN, KIND, ACT, IN, GATED, G, SAMPLES, true>(c, p, out, wait_limit, status, st);
  return (!IN || rows16(out.in, p.N)) && rows16(out.e.y, p.N) ? launch_tile<A_MN, B_MN, KIND, ACT, IN, GATED, G, SAMPLES, true>(c, p, out, wait_limit, status, st)
                                                    : launch_tile<A_MN, B_MN, KIND, ACT, IN, GATED, G, SAMPLES, false>(c, p, out, wait_limit, status, st);
}
// A forward with a long epilogue: by the length of its sums
template <int ACT, bool IN, bool GATED>
int launch_long(const Choice& c, const Product<bf16>& p, Outputs& out, int wait_limit, int32_t* status, cudaStream_t st) {
  return p.K <= 12 * kBK ? launch_choice<false, false, kForward, ACT, IN, GATED, 3>(c, p, out, wait_limit, status, st)
                         : launch_choice<false, false, kForward, ACT, IN, GATED, 2>(c, p, out, wait_limit, status, st);
}

// y of a product of two K-major operands, by what stands behind it (linear_tc_forward.cu)
int launch_forward(const Choice& c, const Product<bf16>& p, Outputs& out, int wait_limit, int32_t* status, cudaStream_t st);

}  // namespace linear_tc
}  // namespace llsa
