// The projection's matrix products on tcgen05 (bf16): D[i, j] = sum_k A(i, k) B(j, k), fp32 sums in tensor memory.
//
// One kernel for the forward (A = x, B = w, both along k in memory), the input's gradient (A = dz, B = w taken across) and the weight's gradient (A =
// dz, B = x, both taken across): an operand whose rows run along k is a K-major tile, one whose rows run along i or j an MN-major tile, and
// TMA fills either from a row-major matrix with 128-byte swizzled rows of 64 (tc05.cuh).  Ragged edges are zeros that TMA fills in.
// A persistent CTA per SM walks tiles of 128 x BN: warp 8 keeps a ring of k-steps of 64 filled, warp 9 issues the products into one of two
// accumulators in tensor memory, and warps 0-7 empty the other one (bias, activation, gate, residual; thread = row, a warpgroup half the columns), so that a
// tile's epilogue runs under the next tile's products.  A sum that is too long and has too few tiles (the weight's gradient: k is the number
// of tokens) is cut into parts, fp32 partial tiles that a second kernel adds in order.
// Every mbarrier wait is bounded; tiles behind one that ran out are written as NaN (and the status word says so).
#include <string.h>

#include "linear.cuh"
#include "tc05.cuh"
#include "tma.cuh"

namespace llsa {

namespace {

using bf16 = __nv_bfloat16;

constexpr int kBM = 128, kBK = 64, kThreads = 320, kEpilogueWarps = 8;

struct ProductMaps {
  CUtensorMap a, b;
};

template <int BN>
struct Tile {
  static constexpr int kStageElems = (kBM + BN) * kBK;
  static constexpr int kStages = BN == 256 ? 4 : BN == 192 ? 5 : BN == 128 ? 6 : 8;
  static constexpr int kTmemCols = BN == 64 ? 128 : BN == 128 ? 256 : 512;
  static constexpr size_t kSmem = (size_t) kStages * kStageElems * 2 + 1024;
};

template <int BN>
struct Bars {
  uint64_t full[Tile<BN>::kStages], empty[Tile<BN>::kStages], ready[2], free_[2];
};

struct Outputs {
  Epilogue<bf16> e;
  float* partial;            // PARTIAL: [split][M][ld]
  int64_t ld;
  int64_t M, N;
  int vec_y, vec_r, vec_pre; // rows on 32-byte boundaries
};

__device__ __forceinline__ void ldg256(const void* p, uint32_t (&r)[8]) {
  asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "l"(p));
}
__device__ __forceinline__ void stg256(void* p, const uint32_t* r) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]),
               "r"(r[7])
               : "memory");
}

// 16 of a row's columns, as values
__device__ __forceinline__ void load_row16(const bf16* p, int vec, int n, float (&v)[16]) {
  if (vec && n == 16) {
    uint32_t w[8];
    ldg256(p, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) { v[2 * i] = bf16_lo(w[i]); v[2 * i + 1] = bf16_hi(w[i]); }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = i < n ? __bfloat162float(p[i]) : 0.f;
  }
}
__device__ __forceinline__ void store_row16(uint16_t* p, int vec, int n, const uint32_t (&w)[8]) {
  if (vec && n == 16) {
    stg256(p, w);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < n) p[i] = (uint16_t) (w[i / 2] >> (16 * (i & 1)));
  }
}

template <bool PARTIAL>
__device__ __forceinline__ void finish16(const Outputs& o, int64_t split, int64_t r, int64_t sample, int64_t c0, float (&v)[16]) {
  const int n = (int) min((int64_t) 16, o.N - c0);
  if (n <= 0) return;
  if constexpr (PARTIAL) {
    float* p = o.partial + (split * o.M + r) * o.ld + c0;
#pragma unroll
    for (int i = 0; i < 16; i += 8)
      if (c0 + i < o.ld) stg256(p + i, reinterpret_cast<const uint32_t*>(v + i));      // ld is a multiple of 8
  } else {
    const Epilogue<bf16>& e = o.e;
    uint32_t w[8];
    float t[16];
    if (e.bias) {
      load_row16(e.bias + c0, ((uintptr_t) (e.bias + c0) & 31) == 0, n, t);
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] += t[i];
    }
    if (e.pre.p) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        w[i] = e.act != kActNone ? (uint32_t) half_bits(v[2 * i]) | (uint32_t) half_bits(v[2 * i + 1]) << 16 : pack_bf16(v[2 * i], v[2 * i + 1]);
      store_row16(reinterpret_cast<uint16_t*>(e.pre.p + r * e.pre.ld + c0), o.vec_pre, n, w);
    }
    if (e.act != kActNone)
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = activate<true>(v[i], e.act);
    if (e.gate.p) {
      const bf16* g = e.gate.p + sample * e.gate.ld + c0;
      load_row16(g, ((uintptr_t) g & 31) == 0, n, t);
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] *= t[i];
    }
    if (e.residual.p) {
      load_row16(e.residual.p + r * e.residual.ld + c0, o.vec_r, n, t);
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] += t[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
    store_row16(reinterpret_cast<uint16_t*>(e.y.p + r * e.y.ld + c0), o.vec_y, n, w);
  }
}

// items: tiles times parts of the sum, (part, row tile, column tile), columns fastest: neighbours in time share rows of A in L2
template <int BN, bool A_MN, bool B_MN, bool PARTIAL>
__global__ void __launch_bounds__(kThreads, 1)
product_tc_kernel(const __grid_constant__ ProductMaps maps, const __grid_constant__ Outputs out, int k_blocks, int per_split, int tiles_n, int tiles, int items,
                  int wait_limit, int32_t* status) {
  using T = Tile<BN>;
  extern __shared__ unsigned char smem_dyn[];
  __shared__ Bars<BN> bars;
  __shared__ uint32_t s_tmem;
  __shared__ tc::WaitCtl s_ctl;
  bf16* ring = reinterpret_cast<bf16*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile tc::WaitCtl* ctl = &s_ctl;
  if (tid == 0) {
    s_ctl.abort = 0;
    s_ctl.limit = wait_limit > 0 ? wait_limit : tc::kWaitPolls;
    for (int i = 0; i < T::kStages; ++i) { tc::mbar_init(&bars.full[i], 1); tc::mbar_init(&bars.empty[i], 1); }
    for (int i = 0; i < 2; ++i) { tc::mbar_init(&bars.ready[i], 1); tc::mbar_init(&bars.free_[i], kEpilogueWarps); }
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
  } else {
    // ---------------------------------------------------------------- epilogue; thread = row, warpgroup = half the columns
    const int wg = warp >> 2, row = (warp & 3) * 32 + lane;
    constexpr int kCols = BN / 2;
    int acc = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int item = blockIdx.x; item < items; item += gridDim.x) {
      const int split = item / tiles, t = item - split * tiles;
      const int64_t r = (int64_t) (t / tiles_n) * kBM + row, j0 = (int64_t) (t % tiles_n) * BN + wg * kCols;
      const int64_t sample = !PARTIAL && out.e.gate.p && r < out.M ? (uint32_t) r / out.e.rows_per_gate : 0;
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
        if (c + 32 == kCols) {                               // all of it has been read
          tc::fence_before_sync();
          __syncwarp();
          if (lane == 0) tma::mbar_arrive(&bars.free_[acc]);
        }
        if (r < out.M) {
          finish16<PARTIAL>(out, split, r, sample, j0 + c, reinterpret_cast<float(&)[16]>(v[0]));
          finish16<PARTIAL>(out, split, r, sample, j0 + c + 16, reinterpret_cast<float(&)[16]>(v[16]));
        }
      }
      acc ^= 1;
      if (acc == 0) ph ^= 1;
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
  return best;
}

int matrix_map(CUtensorMap* m, const Mat<const bf16>& t, int64_t rows, int64_t cols, uint32_t box_rows) {
  const uint64_t dims[2] = {(uint64_t) cols, (uint64_t) rows}, strides[1] = {(uint64_t) t.ld * 2};
  return tma::make_map(m, t.p, 2, dims, strides, box_rows);
}

template <int BN, bool A_MN, bool B_MN, bool PARTIAL>
int launch(const Product<bf16>& p, const Outputs& out, int wait_limit, int32_t* status, cudaStream_t st) {
  ProductMaps maps;
  int rc = A_MN ? matrix_map(&maps.a, p.a, p.K, p.M, kBK) : matrix_map(&maps.a, p.a, p.M, p.K, kBM);
  if (rc) return rc;
  rc = B_MN ? matrix_map(&maps.b, p.b, p.K, p.N, kBK) : matrix_map(&maps.b, p.b, p.N, p.K, BN);
  if (rc) return rc;
  const auto kernel = product_tc_kernel<BN, A_MN, B_MN, PARTIAL>;
  LLSA_SMEM_LIMIT(kernel, Tile<BN>::kSmem);
  const int64_t tiles_n = (p.N + BN - 1) / BN, tiles = (p.M + kBM - 1) / kBM * tiles_n, k_blocks = (p.K + kBK - 1) / kBK;
  const int64_t per = (k_blocks + p.split - 1) / p.split, parts = p.split, items = tiles * parts;
  LLSA_REQUIRE(items <= INT32_MAX && p.M <= INT32_MAX - kBM && p.N <= INT32_MAX - BN && p.K <= INT32_MAX - kBK, LLSA_ERR_SHAPE, "linear: too many outputs");
  launch_pdl(kernel, dim3((unsigned) std::min<int64_t>(items, 148)), dim3(kThreads), Tile<BN>::kSmem, st, maps, out, (int) k_blocks, (int) per, (int) tiles_n,
             (int) tiles, (int) items, wait_limit, status);
  LLSA_LAUNCH_OK("product_tc_kernel");
  return LLSA_OK;
}

template <bool A_MN, bool B_MN, bool PARTIAL>
int launch_width(int bn, const Product<bf16>& p, const Outputs& out, int wait_limit, int32_t* status, cudaStream_t st) {
  switch (bn) {
    case 64: return launch<64, A_MN, B_MN, PARTIAL>(p, out, wait_limit, status, st);
    case 128: return launch<128, A_MN, B_MN, PARTIAL>(p, out, wait_limit, status, st);
    case 192: return launch<192, A_MN, B_MN, PARTIAL>(p, out, wait_limit, status, st);
    default: return launch<256, A_MN, B_MN, PARTIAL>(p, out, wait_limit, status, st);
  }
}

int rows32(const void* p, int64_t ld) { return ((uintptr_t) p & 31) == 0 && ld % 16 == 0; }

}  // namespace

int linear_tc_product(const Product<bf16>& p, const Epilogue<bf16>& e, int wait_limit, int32_t* status, cudaStream_t st) {
  Outputs out = {};
  out.e = e;
  out.M = p.M;
  out.N = p.N;
  out.vec_y = rows32(e.y.p, e.y.ld);
  out.vec_r = rows32(e.residual.p, e.residual.ld);
  out.vec_pre = rows32(e.pre.p, e.pre.ld);
  const int bn = choose(p.M, p.N, (p.K + kBK - 1) / kBK, false).bn;
  return p.b_k ? launch_width<false, false, false>(bn, p, out, wait_limit, status, st) : launch_width<false, true, false>(bn, p, out, wait_limit, status, st);
}

int linear_tc_split(int64_t M, int64_t N, int64_t K) {
  const int64_t k_blocks = (K + kBK - 1) / kBK;
  const int s = choose(M, N, k_blocks, true).split;
  const int64_t per = (k_blocks + s - 1) / s;
  return (int) ((k_blocks + per - 1) / per);      // no part without a share
}

int linear_tc_parts(const Product<bf16>& p, float* partial, int64_t ld, int wait_limit, int32_t* status, cudaStream_t st) {
  Outputs out = {};
  out.partial = partial;
  out.ld = ld;
  out.M = p.M;
  out.N = p.N;
  return launch_width<true, true, true>(choose(p.M, p.N, (p.K + kBK - 1) / kBK, true).bn, p, out, wait_limit, status, st);
}

}  // namespace llsa
