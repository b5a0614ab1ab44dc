// 4-bit page cache: append (quantise) and read-back.
#include "host.h"
#include "int4.cuh"
#include "tokens.cuh"

namespace pab {

struct Int4AppendParams {
  TokenMap map;
  uint8_t* cache[2];       // keys, values
  const void* rows[2];
  int32_t* lens;
  uint32_t* status;
  int64_t r_st, r_sh;      // strides of the new rows (elements)
  int32_t vec;             // rows may be read in 16-byte units
};

// Quantises 8 of the 64 elements of a group held by 8 consecutive lanes:
// returns their code word, and the group's (scale, minimum) pair.  The code is
// the quotient (x - lo) / s rounded to the nearest integer, ties to even: the
// product with the reciprocal is within one of it, and the remainder
// x - lo - c s, exact in fp32, settles the rest.
template <typename T>
__device__ __forceinline__ uint32_t int4_quantise(const float (&f)[8], uint32_t* pair) {
  float lo = f[0], hi = f[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = min_nan(lo, f[i]);
    hi = max_nan(hi, f[i]);
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  const float range = hi - lo;
  const bool finite = fabsf(range) <= 3.4028235e38f;  // false for NaN and infinities
  *pair = pack2<T>(finite ? __fdiv_rn(range, 15.f) : __int_as_float(0x7fffffff),
                   finite ? lo : __int_as_float(0x7fffffff));
  const float s = unpack2<T>(*pair).x;
  uint32_t word = 0;
  if (finite && s > 0.f) {
    const float inv = __frcp_rn(s);
    const bool tiny = s < 1e-37f;  // the reciprocal overflows
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = f[i] - lo;
      float c = rintf(tiny ? __fdiv_rn(a, s) : a * inv);
      c = fminf(c, 15.f);
      const float r = 2.f * fmaf(-c, s, a);
      const int ci = static_cast<int>(c);
      int d = 0;
      if (r > s || (r == s && (ci & 1))) d = 1;
      if (r < -s || (r == -s && (ci & 1))) d = -1;
      const int q = min(max(ci + d, 0), 15);
      word |= static_cast<uint32_t>(q) << (4 * (i / 2 + 4 * (i % 2)));
    }
  }
  return word;
}

// One lane per 8 elements: D/8 lanes hold a row; blockIdx.y 0 keys, 1 values.
template <typename T, int D>
__global__ void __launch_bounds__(256) int4_append_kernel(const Int4AppendParams p) {
  constexpr int LR = D / 8;
  const TokenMap& m = p.map;
  const int kv = blockIdx.y;
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / LR;
  const int e = threadIdx.x % LR, g = e / 8, o = e % 8;
  const int64_t i = row / m.Hkv;
  const int h = static_cast<int>(row - i * m.Hkv);
  uint32_t flags = 0;
  int64_t pid = -1;
  int r = 0;
  float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  int s, j;
  if (i < m.num_tokens && find_token(m, i, &s, &j)) {
    const int L = p.lens[s * m.l_sb + h * m.l_sh];
    if (L < 0) {
      flags |= kStatusNegative;
    } else {
      const int64_t pos = static_cast<int64_t>(L) + j;
      pid = find_page(m, s, h, pos, &flags);
      r = static_cast<int>(pos % m.bs);
    }
    load8<T>(static_cast<const T*>(p.rows[kv]) + i * p.r_st + h * p.r_sh + e * 8, p.vec != 0, f);
  }
  uint32_t pair;
  const uint32_t word = int4_quantise<T>(f, &pair);
  if (flags && p.status) atomicOr(p.status, flags);
  if (pid < 0) return;
  uint8_t* page = p.cache[kv] + pid * (static_cast<int64_t>(m.bs) * int4_row_bytes(D));
  *reinterpret_cast<uint32_t*>(page + (kv ? int4_value_word(D, r, g, o) : int4_key_word(D, r, g, o))) = word;
  if (o == 0) *reinterpret_cast<uint32_t*>(page + int4_pair(D, m.bs, r, g)) = pair;
}

// The lengths of one sequence, after its rows are written: each grows by the
// number of new tokens before the first that had no place.  A length shared by
// the sequence's heads grows by the least of theirs.  One warp per sequence.
__global__ void __launch_bounds__(128) int4_lengths_kernel(const Int4AppendParams p) {
  const TokenMap& m = p.map;
  const int lane = threadIdx.x & 31;
  const int s = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (s >= m.B) return;
  int64_t n = 1;
  if (m.cu) {
    n = static_cast<int64_t>(m.cu[s + 1]) - m.cu[s];
    if (m.cu[s] < 0 || m.cu[s + 1] > m.num_tokens) n = 0;
  }
  if (n <= 0) return;
  int64_t least = n;
  for (int h = 0; h < m.Hkv; ++h) {
    int32_t* lp = p.lens + s * m.l_sb + h * m.l_sh;
    const int64_t L = *lp;
    int64_t got = L < 0 ? 0 : n;
    uint32_t flags = 0;
    for (int64_t pg = L / m.bs + lane; got > 0 && pg * m.bs < L + n; pg += 32)
      if (find_page(m, s, h, pg * m.bs, &flags) < 0) {
        const int64_t before = pg * m.bs - L;
        got = before < 0 ? 0 : before;
        break;
      }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const int64_t x = __shfl_xor_sync(0xffffffffu, got, o);
      got = x < got ? x : got;
    }
    if (m.l_sh != 0) {
      if (lane == 0) *lp = static_cast<int32_t>(L + got);
    } else {
      least = got < least ? got : least;
    }
  }
  if (m.l_sh == 0 && lane == 0) p.lens[s * m.l_sb] += static_cast<int32_t>(least);
}

struct Int4ReadParams {
  TokenMap map;
  const uint8_t* cache[2];
  void* out[2];
  const int32_t* lens;
  const int32_t* starts;   // [B] first position read, or null: 0
  uint32_t* status;
  int64_t o_st, o_sh, start_sb;
};

// lo + s c of 8 elements, rounded to T.  The rounding of s may put code 15 of a
// range as wide as T's past T's largest value: such a value saturates.
template <typename T>
__device__ __forceinline__ uint4 int4_values(uint32_t word, float2 sl) {
  constexpr float kMax = std::is_same<T, __half>::value ? 65504.f : 3.38953139e38f;
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = fmaf(sl.x, static_cast<float>((word >> (4 * (i / 2 + 4 * (i % 2)))) & 15u), sl.y);
    if (v[i] > kMax) v[i] = kMax;  // a NaN stays
  }
  return make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]),
                    pack2<T>(v[6], v[7]));
}

template <typename T, int D>
__global__ void __launch_bounds__(256) int4_read_kernel(const Int4ReadParams p) {
  constexpr int LR = D / 8;
  const TokenMap& m = p.map;
  const int kv = blockIdx.y;
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / LR;
  const int e = threadIdx.x % LR, g = e / 8, o = e % 8;
  const int64_t i = row / m.Hkv;
  const int h = static_cast<int>(row - i * m.Hkv);
  int s, j;
  if (i >= m.num_tokens || !find_token(m, i, &s, &j)) return;
  const int L = p.lens[s * m.l_sb + h * m.l_sh];
  const int64_t pos = static_cast<int64_t>(p.starts ? p.starts[s * p.start_sb] : 0) + j;
  uint4 v = make_uint4(0u, 0u, 0u, 0u);
  if (pos >= 0 && pos < L) {
    uint32_t flags = 0;
    const int64_t pid = find_page(m, s, h, pos, &flags);
    if (flags && p.status)
      atomicOr(p.status, flags & kStatusAppendFull ? kStatusClamp : flags);
    if (pid >= 0) {
      const int r = static_cast<int>(pos % m.bs);
      const uint8_t* page = p.cache[kv] + pid * (static_cast<int64_t>(m.bs) * int4_row_bytes(D));
      const uint32_t word = *reinterpret_cast<const uint32_t*>(
          page + (kv ? int4_value_word(D, r, g, o) : int4_key_word(D, r, g, o)));
      const uint32_t pair = *reinterpret_cast<const uint32_t*>(page + int4_pair(D, m.bs, r, g));
      v = int4_values<T>(word, unpack2<T>(pair));
    }
  }
  *reinterpret_cast<uint4*>(static_cast<T*>(p.out[kv]) + i * p.o_st + h * p.o_sh + e * 8) = v;
}

}  // namespace pab

namespace {

using pabh::aligned;
using pabh::fail;

// The checks that append and read-back share; fills the token map.
int check_int4(const pab200_int4_rows_args* a, pab::TokenMap* m) {
  if (!a) return fail(PAB200_ERR_INVALID_ARGUMENT, "args is null");
  if (a->dtype != PAB200_DTYPE_BF16 && a->dtype != PAB200_DTYPE_F16)
    return fail(PAB200_ERR_UNSUPPORTED, "dtype %d: rows must be bf16 or f16", a->dtype);
  const int D = a->head_size, bs = a->block_size;
  if (D != 64 && D != 128 && D != 256)
    return fail(PAB200_ERR_UNSUPPORTED, "head_size %d: supported 64, 128, 256", D);
  if (bs != 8 && bs != 16 && bs != 32 && bs != 64)
    return fail(PAB200_ERR_UNSUPPORTED, "block_size %d: supported 8, 16, 32, 64", bs);
  if (a->num_seqs < 0 || a->num_kv_heads < 1 || a->max_blocks < 0 || a->num_pages < 0 ||
      a->num_tokens < 0)
    return fail(PAB200_ERR_INVALID_ARGUMENT,
                "need num_seqs, max_blocks, num_pages, num_tokens >= 0, num_kv_heads >= 1");
  if (!a->cu_tokens && a->num_tokens != a->num_seqs)
    return fail(PAB200_ERR_INVALID_ARGUMENT,
                "without cu_tokens there is one token per sequence: num_tokens %lld, num_seqs %d",
                static_cast<long long>(a->num_tokens), a->num_seqs);
  if (int64_t(a->max_blocks) * bs >= (int64_t(1) << 31) || a->num_tokens >= (int64_t(1) << 31) ||
      a->num_tokens * a->num_kv_heads * (D / 8) / 256 >= (int64_t(1) << 31) - 1)
    return fail(PAB200_ERR_UNSUPPORTED, "max_blocks*block_size or num_tokens too large (>= 2^31)");
  if (a->num_seqs == 0 || a->num_tokens == 0) return PAB200_OK;
  if (!a->k_rows || !a->v_rows || !a->seqlens)
    return fail(PAB200_ERR_INVALID_ARGUMENT, "k_rows, v_rows or seqlens is null");
  if (a->max_blocks > 0 && a->num_pages > 0 && (!a->k_cache || !a->v_cache || !a->block_table))
    return fail(PAB200_ERR_INVALID_ARGUMENT, "k_cache, v_cache or block_table is null");
  if (!aligned(a->k_cache, 16) || !aligned(a->v_cache, 16))
    return fail(PAB200_ERR_ALIGNMENT, "k_cache and v_cache must be 16-byte aligned");
  if (!aligned(a->k_rows, 2) || !aligned(a->v_rows, 2))
    return fail(PAB200_ERR_ALIGNMENT, "k_rows and v_rows must be 2-byte aligned");
  *m = pab::TokenMap{};
  m->bt = a->block_table;
  m->cu = a->cu_tokens;
  m->bt_sb = a->bt_stride_b;
  m->bt_sh = a->bt_stride_h;
  m->bt_si = a->bt_stride_i;
  m->l_sb = a->seqlens_stride_b;
  m->l_sh = a->seqlens_stride_h;
  m->num_pages = a->num_pages;
  m->num_tokens = a->num_tokens;
  m->bt_mul = a->bt_page_mul;
  m->bt_add = a->bt_page_add;
  m->B = a->num_seqs;
  m->Hkv = a->num_kv_heads;
  m->bs = bs;
  m->maxb = a->num_pages > 0 ? a->max_blocks : 0;
  return PAB200_OK;
}

bool rows_vec(const pab200_int4_rows_args* a) {
  return aligned(a->k_rows, 16) && aligned(a->v_rows, 16) && a->row_stride_t % 8 == 0 &&
         a->row_stride_h % 8 == 0;
}

dim3 rows_grid(const pab200_int4_rows_args* a) {
  const int64_t threads = a->num_tokens * a->num_kv_heads * (a->head_size / 8);
  return dim3(static_cast<unsigned>((threads + 255) / 256), 2);
}

template <typename T>
void launch_append(const pab::Int4AppendParams& p, int D, dim3 grid, cudaStream_t s) {
  switch (D) {
    case 64: pab::int4_append_kernel<T, 64><<<grid, 256, 0, s>>>(p); break;
    case 128: pab::int4_append_kernel<T, 128><<<grid, 256, 0, s>>>(p); break;
    default: pab::int4_append_kernel<T, 256><<<grid, 256, 0, s>>>(p); break;
  }
}

template <typename T>
void launch_read(const pab::Int4ReadParams& p, int D, dim3 grid, cudaStream_t s) {
  switch (D) {
    case 64: pab::int4_read_kernel<T, 64><<<grid, 256, 0, s>>>(p); break;
    case 128: pab::int4_read_kernel<T, 128><<<grid, 256, 0, s>>>(p); break;
    default: pab::int4_read_kernel<T, 256><<<grid, 256, 0, s>>>(p); break;
  }
}

}  // namespace

PAB200_EXPORT size_t pab200_int4_page_bytes(int32_t head_size, int32_t block_size) {
  if ((head_size != 64 && head_size != 128 && head_size != 256) ||
      (block_size != 8 && block_size != 16 && block_size != 32 && block_size != 64))
    return 0;
  return size_t(block_size) * pab::int4_row_bytes(head_size);
}

PAB200_EXPORT int pab200_kv_append_int4(const pab200_int4_rows_args* a, int32_t increment,
                                        void* stream) {
  pab::Int4AppendParams p{};
  const int rc = check_int4(a, &p.map);
  if (rc || a->num_seqs == 0 || a->num_tokens == 0) return rc;
  p.cache[0] = static_cast<uint8_t*>(a->k_cache);
  p.cache[1] = static_cast<uint8_t*>(a->v_cache);
  p.rows[0] = a->k_rows;
  p.rows[1] = a->v_rows;
  p.lens = a->seqlens;
  p.status = a->status;
  p.r_st = a->row_stride_t;
  p.r_sh = a->row_stride_h;
  p.vec = rows_vec(a);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->dtype == PAB200_DTYPE_BF16)
    launch_append<__nv_bfloat16>(p, a->head_size, rows_grid(a), s);
  else
    launch_append<__half>(p, a->head_size, rows_grid(a), s);
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess && increment) {
    pab::int4_lengths_kernel<<<(a->num_seqs + 3) / 4, 128, 0, s>>>(p);
    e = cudaGetLastError();
  }
  return e == cudaSuccess ? PAB200_OK : pabh::cuda_fail(e, "4-bit append launch");
}

PAB200_EXPORT int pab200_kv_read_int4(const pab200_int4_rows_args* a, const int32_t* starts,
                                      int64_t starts_stride, void* stream) {
  pab::Int4ReadParams p{};
  const int rc = check_int4(a, &p.map);
  if (rc || a->num_seqs == 0 || a->num_tokens == 0) return rc;
  if (!rows_vec(a))
    return fail(PAB200_ERR_ALIGNMENT, "rows must be 16-byte aligned with strides that are multiples of 8");
  p.cache[0] = static_cast<const uint8_t*>(a->k_cache);
  p.cache[1] = static_cast<const uint8_t*>(a->v_cache);
  p.out[0] = a->k_rows;
  p.out[1] = a->v_rows;
  p.lens = a->seqlens;
  p.starts = starts;
  p.start_sb = starts_stride;
  p.status = a->status;
  p.o_st = a->row_stride_t;
  p.o_sh = a->row_stride_h;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->dtype == PAB200_DTYPE_BF16)
    launch_read<__nv_bfloat16>(p, a->head_size, rows_grid(a), s);
  else
    launch_read<__half>(p, a->head_size, rows_grid(a), s);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? PAB200_OK : pabh::cuda_fail(e, "4-bit read launch");
}
