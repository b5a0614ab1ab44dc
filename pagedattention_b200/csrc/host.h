// Host-side pieces shared by the translation units of libpab200.so: error
// text, alignment checks, launch configuration and the decode kernel handle.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

#include "decode.cuh"
#include "pab200.h"

#define PAB200_EXPORT extern "C" __attribute__((visibility("default")))

namespace pabh {

// Records the calling thread's error text and returns `code`.
int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int cuda_fail(cudaError_t e, const char* what);

// SM count of the current device (148 if it cannot be queried).
int device_sm_count_current();

inline size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

inline bool aligned(const void* p, size_t a) {
  return (reinterpret_cast<uintptr_t>(p) % a) == 0;
}

struct KernelOps {
  void* fn;  // decode kernel (for attributes / occupancy)
  cudaError_t (*launch)(dim3, dim3, size_t, cudaStream_t, bool, const CUtensorMap&,
                        const CUtensorMap&, const pab::DecodeParams&);
};

// Launch configuration; `pdl` lets the grid start while the previous kernel
// in the stream finishes (programmatic dependent launch): the kernel waits
// with griddepcontrol.wait before it reads that kernel's output.
struct LaunchCfg {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  LaunchCfg(dim3 grid, dim3 block, size_t smem, cudaStream_t s, bool pdl) {
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 1 : 0;
  }
};

template <auto Kernel>
cudaError_t launch_decode(dim3 grid, dim3 block, size_t smem, cudaStream_t s, bool pdl,
                          const CUtensorMap& k, const CUtensorMap& v,
                          const pab::DecodeParams& p) {
  LaunchCfg lc(grid, block, smem, s, pdl);
  return cudaLaunchKernelEx(&lc.cfg, Kernel, k, v, p);
}

template <auto Kernel>
KernelOps kernel_ops() {
  return KernelOps{reinterpret_cast<void*>(Kernel), &launch_decode<Kernel>};
}

// The decode kernel over 4-bit pages for these sizes (int4_decode.cu).
struct Int4Kernel {
  KernelOps ops;
  int parts;     // token parts of a stage, joined at the end of a head
  int min_ctas;  // resident CTAs per SM its registers allow
};
bool select_int4_kernel(int dtype, int D, int G, Int4Kernel* o);

// A selection of pages inside a decode call: the whole contexts' lengths and
// table width, and the launch of the kernels that write the call's tables and
// lengths (programmatically dependent on the planner before them, which touches
// nothing of theirs; the last of them starts the decode grid's dependency).
struct Selection {
  const int32_t* lens;
  int64_t l_sb, l_sh;
  int32_t max_blocks;
  int (*launch)(const void* what, cudaStream_t s);
  const void* what;
};
// pab200_decode() over the tables that `sel` writes.
int decode_selected(const pab200_decode_args* a, const Selection& sel, void* workspace,
                    size_t workspace_bytes, void* stream);

}  // namespace pabh
