// Pieces of the kernels that take the rows of a batch's tokens: which tokens
// one warp takes, which page they go to, and 8-element row accesses.
#pragma once

#include "decode.cuh"

namespace pab {

// Where the rows of (sequence, kv head) pairs live: block table, lengths and
// the cut of a token axis into sequences (null: one token per sequence).
struct TokenMap {
  const int32_t* bt;
  const int32_t* cu;
  int64_t bt_sb, bt_sh, bt_si, l_sb, l_sh, num_pages;
  int32_t num_tokens, bt_mul, bt_add, B, Hkv, bs, log2_bs, maxb;
};

// Positions are cut into runs of 2^k (a page, or a tile of one); one warp takes
// the tokens of one run.  Sequence s owns run slots [first_slot(s),
// first_slot(s + 1)), at least as many as the runs its tokens touch wherever
// they start: floor((n - 2) / 2^k) + 2 <= floor(cu[s+1] / 2^k) - floor(cu[s] /
// 2^k) + 2.
__host__ __device__ __forceinline__ int64_t num_slots(int64_t tokens, int B, bool cu, int k) {
  return cu ? (tokens >> k) + 2 * int64_t(B) : B;
}

struct TokenRun {
  int s;         // sequence
  int t0;        // its first token
  int n;         // its tokens (0: none, or offsets that make no sense)
  int run;       // this slot's run, counted from the run its first token is in
};

__device__ __forceinline__ TokenRun find_run(const TokenMap& m, int slot, int k) {
  TokenRun r;
  if (!m.cu) {
    r.s = r.t0 = slot;
    r.n = slot < m.B ? 1 : 0;
    r.run = 0;
    return r;
  }
  int lo = 0, hi = m.B - 1;  // last s with first_slot(s) <= slot
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if ((m.cu[mid] >> k) + 2 * mid <= slot)
      lo = mid;
    else
      hi = mid - 1;
  }
  r.s = lo;
  r.t0 = m.cu[lo];
  const int end = m.cu[lo + 1];
  r.n = r.t0 < 0 || end > m.num_tokens || end < r.t0 ? 0 : end - r.t0;
  r.run = slot - (r.t0 >> k) - 2 * lo;
  if (r.run < 0) r.n = 0;
  return r;
}

// Page of table column i of (s, h), or -1 with *flags raised.
__device__ __forceinline__ int64_t find_page(const TokenMap& m, int s, int h, int64_t i,
                                             uint32_t* flags) {
  if (i >= m.maxb) {
    *flags |= kStatusAppendFull;
    return -1;
  }
  const int64_t pid = static_cast<int64_t>(m.bt[s * m.bt_sb + h * m.bt_sh + i * m.bt_si]) * m.bt_mul +
                      static_cast<int64_t>(h) * m.bt_add;
  if (pid < 0 || pid >= m.num_pages) {
    *flags |= kStatusBadPage;
    return -1;
  }
  return pid;
}

// Minimum / maximum of two pairs of T, NaN if either is NaN.
template <typename T>
__device__ __forceinline__ uint32_t min2_nan(uint32_t a, uint32_t b);
template <typename T>
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b);
template <>
__device__ __forceinline__ uint32_t min2_nan<__nv_bfloat16>(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <>
__device__ __forceinline__ uint32_t max2_nan<__nv_bfloat16>(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <>
__device__ __forceinline__ uint32_t min2_nan<__half>(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <>
__device__ __forceinline__ uint32_t max2_nan<__half>(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Eight elements of a row as they are; `vec`: the row may be read in 16 bytes.
template <typename T>
__device__ __forceinline__ uint4 load_row8(const T* p, bool vec) {
  if (vec) return __ldg(reinterpret_cast<const uint4*>(p));
  const uint16_t* u = reinterpret_cast<const uint16_t*>(p);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = u[2 * i] | static_cast<uint32_t>(u[2 * i + 1]) << 16;
  return make_uint4(w[0], w[1], w[2], w[3]);
}

}  // namespace pab
