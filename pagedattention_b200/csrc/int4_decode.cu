// Instantiations of the decode kernel over 4-bit pages.
#include "host.h"

namespace {

template <typename T, int D, int NT, int ST, bool PAIR>
pabh::KernelOps ops_of() {
  return pabh::kernel_ops<&pab::decode_int4_kernel<T, D, NT, ST, PAIR>>();
}

template <typename T, int ST>
bool select(int D, int nt, bool pair, pabh::KernelOps* o) {
  if (pair) {  // groups of 17-32 heads at D 128: two warps per ring, 16 heads each
    if (D != 128 || nt != 2) return false;
    *o = ops_of<T, 128, 2, ST, true>();
    return true;
  }
  switch (D * 16 + nt) {
    case 64 * 16 + 1: *o = ops_of<T, 64, 1, ST, false>(); return true;
    case 64 * 16 + 2: *o = ops_of<T, 64, 2, ST, false>(); return true;
    case 64 * 16 + 4: *o = ops_of<T, 64, 4, ST, false>(); return true;
    case 128 * 16 + 1: *o = ops_of<T, 128, 1, ST, false>(); return true;
    case 128 * 16 + 2: *o = ops_of<T, 128, 2, ST, false>(); return true;
    case 256 * 16 + 1: *o = ops_of<T, 256, 1, ST, false>(); return true;
    default: return false;
  }
}

template <typename T>
bool select_st(int D, int nt, int st, bool pair, pabh::KernelOps* o) {
  switch (st) {
    case 32: return select<T, 32>(D, nt, pair, o);
    case 64: return select<T, 64>(D, nt, pair, o);
    default: return false;
  }
}

}  // namespace

bool pabh::select_int4_kernel(int dtype, int D, int nt, int st, bool pair, KernelOps* o) {
  return dtype == PAB200_DTYPE_BF16 ? select_st<__nv_bfloat16>(D, nt, st, pair, o)
                                    : select_st<__half>(D, nt, st, pair, o);
}
