// The projection's matrix products on tcgen05 (bf16): D[i, j] = sum_k A(i, k) B(j, k), fp32 sums in tensor memory, and what stands behind them.
//
//   forward   A = x, B = w, both along k in memory:  y = residual + gate act(D + bias)
//   slope     the same product again:                dz = dy act'(D + bias), and its column sums.  z is not kept between the passes: that would cost 4 bytes a
//             value of memory traffic and 2 of storage (123 us and 400 MB at 131072 x 1536), and z would be rounded.  dz is rounded to bf16, which is how the
//             tensor cores take it in the next two products (a half step of each term: dx and dw are 2.35e-3 off in the norm where one rounding leaves
//             1.66e-3); its column sums take it unrounded
//   forward   A = dz, B = w taken across:            dx
//   parts     A = dz, B = x, both taken across:      dw, in parts of the sum over the tokens, which a second kernel adds in order
//
// An operand whose rows run along k is a K-major tile, one whose rows run along i or j an MN-major tile, and TMA fills either from a row-major
// matrix with 128-byte swizzled rows of 64 (tc05.cuh).  Ragged edges are zeros that TMA fills in.
// A persistent CTA per SM walks tiles of 128 x BN, or a pair of them (a cluster of two) tiles of 256 x BN, columns fastest (neighbours in time share rows of A in
// L2).  The SM takes 64 bytes a cycle from L2, which is the pace of a 128 x 128 tile twice over; a pair keeps half of B in either CTA and multiplies both
// halves, 256 x 256 at the pace of the tensor cores.  One warp keeps a ring of k-steps of 64 filled; another (of a pair, rank 0's) issues the products
// into one of two accumulators in tensor memory; two or three warpgroups empty the other one, so that a tile's epilogue runs under the
// next tile's products.  The epilogue goes in chunks of 64 columns, dealt out to the warpgroups in turn: a chunk is finished in a 128 x 64 buffer of
// shared memory (two per warpgroup), which the warpgroup's mover warp has filled with the residual or dy by TMA beforehand and stores by TMA
// afterwards.  Matrices whose rows TMA cannot take go through the same buffers with loads and stores of the warp.
//
// us, 131072 rows, 384 -> 1536 | 1536 -> 384 (cuBLAS: 145 | 142 to 149 forward, 145 | 175 dw): plain 133 | 133, with GELU 167, gated onto a residual 171 | 157,
// dx 146 | 144, dw 126 | 133, slope with its column sums 241: 1.0 to 1.2 PFLOP/s where there is little epilogue.  An activation's epilogue is paced by the 16
// special functions a cycle (89 us of GELU's 167; its instructions do not all hide under the products).  With the results stored straight from registers, 32
// bytes of each of 32 rows an instruction, GELU took 590; with tiles of one CTA instead of pairs 271 (plain 217).
// Every mbarrier wait is bounded; tiles behind one that ran out are written as NaN (and the status word says so).
#include "linear_tc.cuh"

namespace llsa {

using namespace linear_tc;

namespace {

// ------------------------------------------------------------------------------------------------ choice of the tile
// Cycles of a k-step of 64: the products' (BN / 2 per 16 of k), or what the SM's port to L2 takes for the operands at 64 bytes a cycle: 128 rows of A and BN
// of B, of a pair BN / 2.  The port is the pace of everything but the pair of 256 x 256.
int64_t step_cycles(int bn, bool pair) { return std::max(2 * bn, 256 + (pair ? bn : 2 * bn)); }

// The tile, and with `parts` the number of parts, that a count of waves over 148 SMs says is the fastest.  in: the epilogue reads a tile as well
// samples: that many products of these sizes
Choice choose(int64_t M, int64_t N, int64_t k_blocks, int kind, bool in, bool act, int64_t samples = 1) {
  Choice best = {128, false, 1, INT64_MAX};
  int64_t least = INT64_MAX;
  for (const Choice c : {Choice{64, false}, Choice{128, false}, Choice{192, true}, Choice{256, true}}) {
    if (kind == kSlope && c.bn != 128 && c.bn != 192) continue;
    const int64_t units = c.pair ? 74 : 148, rows = c.pair ? 2 * kBM : kBM, tiles = (M + rows - 1) / rows * ((N + c.bn - 1) / c.bn) * samples;
    const int64_t most = kind == kParts ? std::max<int64_t>(1, std::min<int64_t>(k_blocks / 4, 4 * units / tiles)) : 1;
    for (int64_t s = 1; s <= most; ++s) {
      const int64_t waves = (tiles * s + units - 1) / units, steps = (k_blocks + s - 1) / s;
      // beside the steps: the epilogue's tile through the same port, a part written and read again (about 40 bytes a cycle of the SM); an activation takes two of
      // the 16 special functions a cycle for a value; and once the first tile's fill and the last one's epilogue, which nothing hides
      const int64_t products = steps * step_cycles(c.bn, c.pair) + (in ? 4 * c.bn : 0) + (kind == kParts ? kBM * c.bn * 8 / 40 : 0);
      const int64_t tile = std::max<int64_t>(products, (act ? 16 : 6) * c.bn);
      const int64_t cost = waves * tile + 1500 + 8 * c.bn;
      if (cost < least) {
        least = cost;
        best = {c.bn, c.pair, (int) s, cost};
      }
    }
  }
  return best;
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
  const Choice c = choose(p.M, p.N, (p.K + kBK - 1) / kBK, kForward, e.residual.p != nullptr, e.act != kActNone, std::max<int64_t>(1, p.samples));
  if (p.samples) return launch_choice<false, true, kForward, kActNone, false, false, 2, true>(c, p, out, wait_limit, status, st);
  if (!p.b_k) return launch_choice<false, true, kForward, kActNone, false, false, 2>(c, p, out, wait_limit, status, st);
  return launch_forward(c, p, out, wait_limit, status, st);
}

int64_t linear_tc_slope_groups(int64_t M, int64_t N, int64_t K) {
  const Choice c = choose(M, N, (K + kBK - 1) / kBK, kSlope, true, true);
  return slope_rows(M, N, c.bn, c.pair) << c.pair;
}

int linear_tc_slope(const Product<bf16>& p, const Epilogue<bf16>& e, const Mat<const bf16>& dy, float* sums, int wait_limit, int32_t* status, cudaStream_t st) {
  Outputs out = outputs(p, e, dy);
  out.partial = sums;
  const Choice c = choose(p.M, p.N, (p.K + kBK - 1) / kBK, kSlope, true, true);
  return e.act == kActGeluTanh ? launch_choice<false, false, kSlope, kActGeluTanh, true, false, 3>(c, p, out, wait_limit, status, st)
                               : launch_choice<false, false, kSlope, kActSilu, true, false, 3>(c, p, out, wait_limit, status, st);
}

int linear_tc_split(int64_t M, int64_t N, int64_t K, int64_t samples, bool* turned) {
  const int64_t k_blocks = (K + kBK - 1) / kBK, n = std::max<int64_t>(1, samples);
  const Choice c = choose(M, N, k_blocks, kParts, false, false, n), d = choose(N, M, k_blocks, kParts, false, false, n);
  *turned = d.cost < c.cost;
  const int s = *turned ? d.split : c.split;
  const int64_t per = (k_blocks + s - 1) / s;
  return (int) ((k_blocks + per - 1) / per);      // no part without a share
}

int linear_tc_parts(const Product<bf16>& p, float* partial, int64_t ld, int wait_limit, int32_t* status, cudaStream_t st) {
  Outputs out = outputs(p, {}, {});
  out.partial = partial;
  out.ld = ld;
  const Choice c = choose(p.M, p.N, (p.K + kBK - 1) / kBK, kParts, false, false, std::max<int64_t>(1, p.samples));
  return p.samples ? launch_choice<true, true, kParts, kActNone, false, false, 2, true>(c, p, out, wait_limit, status, st)
                   : launch_choice<true, true, kParts, kActNone, false, false, 2>(c, p, out, wait_limit, status, st);
}

}  // namespace llsa
