// The forward products of the projection (linear_tc.cu), one kernel for each epilogue: without an activation plain, onto a residual, or gated onto it; with
// one plain or onto a residual.  A flag that a kernel looks up costs a branch per eight columns, some 15 cycles of a warp that has nothing to hide them.
#include "linear_tc.cuh"

namespace llsa {
namespace linear_tc {

int launch_forward(const Choice& c, const Product<bf16>& p, Outputs& out, int wait_limit, int32_t* status, cudaStream_t st) {
  const bool in = out.in.p != nullptr;
  if (out.e.act == kActGeluTanh)
    return in ? launch_long<kActGeluTanh, true, false>(c, p, out, wait_limit, status, st)
              : launch_long<kActGeluTanh, false, false>(c, p, out, wait_limit, status, st);
  if (out.e.act == kActSilu)
    return in ? launch_long<kActSilu, true, false>(c, p, out, wait_limit, status, st)
              : launch_long<kActSilu, false, false>(c, p, out, wait_limit, status, st);
  if (out.e.gate.p) return launch_long<kActNone, true, true>(c, p, out, wait_limit, status, st);
  return in ? launch_long<kActNone, true, false>(c, p, out, wait_limit, status, st)
            : launch_choice<false, false, kForward, kActNone, false, false, 2>(c, p, out, wait_limit, status, st);
}

}  // namespace linear_tc
}  // namespace llsa
