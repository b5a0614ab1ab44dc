// Instantiations of the decode kernel over 4-bit pages.
#include "int4_decode.cuh"

#include "host.h"

namespace {

// MINB: resident CTAs per SM the registers are held to.  A CTA's 5 warps share 4
// register files, so 2 CTAs leave 168 registers a thread, 3 leave 128 and 4 leave
// 96.  State per thread grows with D/16 x NT: 24 accumulator and query registers
// fit 4 CTAs, 48 fit 3, 96 fit 2 (with spills of 0.1 to 0.3 KB a thread).  Other
// counts were timed at D 128 with groups of up to 8 and D 64 with 32 heads.
template <typename T, int D, int NT, int HS, int MINB>
void take(pabh::Int4Kernel* o) {
  o->ops = pabh::kernel_ops<&pab::decode_int4_kernel<T, D, NT, HS, MINB>>();
  o->parts = pab::kQ4Consumers / HS;
  o->min_ctas = MINB;
}

template <typename T>
bool select(int D, int G, pabh::Int4Kernel* o) {
  const int nt = G <= 8 ? 1 : (G <= 16 ? 2 : 4);
  switch (D * 16 + nt) {
    case 64 * 16 + 1: take<T, 64, 1, 1, 4>(o); return true;
    case 64 * 16 + 2: take<T, 64, 2, 1, 3>(o); return true;
    case 64 * 16 + 4: take<T, 64, 2, 2, 3>(o); return G <= 32;   // 16 heads per warp pair
    case 128 * 16 + 1: take<T, 128, 1, 1, 3>(o); return true;
    case 128 * 16 + 2: take<T, 128, 2, 1, 2>(o); return true;
    case 128 * 16 + 4: take<T, 128, 2, 2, 2>(o); return G <= 32;  // 16 heads per warp pair
    case 256 * 16 + 1: take<T, 256, 1, 1, 2>(o); return true;
    default: return false;
  }
}

}  // namespace

bool pabh::select_int4_kernel(int dtype, int D, int G, Int4Kernel* o) {
  return dtype == PAB200_DTYPE_BF16 ? select<__nv_bfloat16>(D, G, o) : select<__half>(D, G, o);
}
