// Pieces of the kernels that take new rows of a batch: which sequence a token
// belongs to, which page it goes to, and 8-element row accesses.
#pragma once

#include "decode.cuh"

namespace pab {

// Where the rows of (sequence, kv head) pairs live: block table, lengths and
// the cut of a token axis into sequences (null: one token per sequence).
struct TokenMap {
  const int32_t* bt;
  const int32_t* cu;
  int64_t bt_sb, bt_sh, bt_si, l_sb, l_sh, num_pages, num_tokens;
  int32_t bt_mul, bt_add, B, Hkv, bs, maxb;
};

// Sequence of token i and its place j among that sequence's tokens; false for
// a token in no sequence.
__device__ __forceinline__ bool find_token(const TokenMap& m, int64_t i, int* s, int* j) {
  if (!m.cu) {
    *s = static_cast<int>(i);
    *j = 0;
    return i < m.B;
  }
  int lo = 0, hi = m.B;  // first s with cu[s + 1] > i
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (m.cu[mid + 1] > i)
      hi = mid;
    else
      lo = mid + 1;
  }
  if (lo >= m.B) return false;
  *s = lo;
  *j = static_cast<int>(i - m.cu[lo]);
  return *j >= 0;
}

// Page of position pos of (s, h), or -1 with *flags raised.
__device__ __forceinline__ int64_t find_page(const TokenMap& m, int s, int h, int64_t pos,
                                             uint32_t* flags) {
  const int64_t i = pos / m.bs;
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

// fp32 minimum / maximum that return NaN if either is NaN.
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Eight elements of a row.
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vec, float (&f)[8]) {
  if (vec) {
    unpack8<T>(*reinterpret_cast<const uint4*>(p), f);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = static_cast<float>(p[i]);
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]),
                                            pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
}

}  // namespace pab
