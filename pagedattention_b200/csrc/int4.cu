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
  int32_t increment;
  int32_t log2_run;        // tokens a warp takes: one 8-token tile, or two of a page
};

// Codes of a group whose scale is below T's normal numbers (rounded coarsely,
// so that quotients pass 15), 0 or NaN (no codes), as in int4_codes_of.
template <typename T>
__device__ __noinline__ uint32_t int4_quantise_tiny(uint4 x, uint32_t pair) {
  const uint32_t v[4] = {x.x, x.y, x.z, x.w};
  const float2 sl = unpack2<T>(pair);
  uint32_t word = 0;
  for (int i = 0; i < 8 && sl.x > 0.f; ++i) {
    const float2 f = unpack2<T>(v[i / 2]);
    const float q = rintf(__fdiv_rn((i & 1 ? f.y : f.x) - sl.y, sl.x));
    word |= static_cast<uint32_t>(fminf(q, 15.f)) << (4 * (i / 2 + 4 * (i % 2)));
  }
  return word;
}

// (minimum, -maximum) of the 64 elements of a group, 8 in each of 8 consecutive
// lanes, of the rows of N rounds: lane o of the 8 gets round o % N.  A 16-bit
// float changes sign by its top bit, so one comparison serves both; a step
// across lanes also halves the rounds that a lane goes on with.
template <typename T, int N>
__device__ __forceinline__ uint32_t group_ranges(const uint4 (&x)[N], int o) {
  uint32_t v[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t lo = min2_nan<T>(min2_nan<T>(x[i].x, x[i].y), min2_nan<T>(x[i].z, x[i].w));
    const uint32_t hi = max2_nan<T>(max2_nan<T>(x[i].x, x[i].y), max2_nan<T>(x[i].z, x[i].w)) ^ 0x80008000u;
    v[i] = min2_nan<T>(__byte_perm(lo, hi, 0x5410), __byte_perm(lo, hi, 0x7632));
  }
#pragma unroll
  for (int b = 1; b < 8; b <<= 1) {
    const bool up = o & b;
#pragma unroll
    for (int j = 0; 2 * j < N / b; ++j) {
      if (N / b > 1) {
        const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? v[2 * j] : v[2 * j + 1], b);
        v[j] = min2_nan<T>(up ? v[2 * j + 1] : v[2 * j], got);
      } else {
        v[0] = min2_nan<T>(v[0], __shfl_xor_sync(0xffffffffu, v[0], b));
      }
    }
    if (N / b == 0) v[0] = min2_nan<T>(v[0], __shfl_xor_sync(0xffffffffu, v[0], b));
  }
  return v[0];
}

// Smallest scale whose quotients stay at 15 (1 + 2^-8) at most: the normal
// numbers of fp16; of bf16, those whose reciprocal is finite.
template <typename T>
__device__ constexpr float int4_least_scale() {
  return std::is_same<T, __half>::value ? 6.103515625e-5f : 1e-36f;
}

// A group's (scale, minimum) pair and 1 / scale from its (minimum, -maximum).
template <typename T>
__device__ __forceinline__ uint32_t int4_scale(uint32_t both, float* inv) {
  const float2 lh = unpack2<T>(both);
  const float range = -lh.y - lh.x;
  const bool finite = fabsf(range) <= 3.4028235e38f;  // false for NaN and infinities
  const float nan = __int_as_float(0x7fffffff);
  const uint32_t pair = pack2<T>(finite ? __fdiv_rn(range, 15.f) : nan, finite ? lh.x : nan);
  const float s = unpack2<T>(pair).x;
  *inv = s >= int4_least_scale<T>() ? __frcp_rn(s) : 0.f;
  return pair;
}

// Code word of 8 elements (element i in nibble i / 2 + 4 (i % 2)).
//
// A code is the quotient a / s, a = x - lo, rounded to the nearest integer, ties
// to even.  The quotient is formed as q0 = a (1/s) corrected once by its
// remainder, q0 + (a - q0 s)(1/s), which is the correctly rounded a / s (P.
// Markstein, IBM J. Res. Dev. 34, 1990), so that exact ties, common among 16-bit
// inputs, stay ties; adding 1.5 * 2^23 rounds it.
template <typename T>
__device__ __forceinline__ uint32_t int4_codes_of(const uint4& x, uint32_t pair, float inv) {
  if (inv == 0.f) return int4_quantise_tiny<T>(x, pair);
  const float2 sl = unpack2<T>(pair);
  constexpr float kMagic = 12582912.f;  // 1.5 * 2^23
  const uint32_t v[4] = {x.x, x.y, x.z, x.w};
  uint32_t c[8];  // 0x4b400000 + code
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2<T>(v[i]);
    const float a0 = f.x - sl.y, a1 = f.y - sl.y;
    const float q0 = a0 * inv, q1 = a1 * inv;
    c[2 * i] = __float_as_uint(fmaf(fmaf(-q0, sl.x, a0), inv, q0) + kMagic);
    c[2 * i + 1] = __float_as_uint(fmaf(fmaf(-q1, sl.x, a1), inv, q1) + kMagic);
  }
  // c0 + 16 c2 + 256 c4 + 4096 c6: the constant leaves the low 16 bits alone
  const uint32_t even = ((c[6] * 16u + c[4]) * 16u + c[2]) * 16u + c[0];
  const uint32_t odd = ((c[7] * 16u + c[5]) * 16u + c[3]) * 16u + c[1];
  return __byte_perm(even, odd, 0x5410);
}

// 4 x 4 transpose of the words of 4 lanes that differ in lane bits A and B:
// lane (a, b) with w[j] ends with w[i] = the word j = 2 a + b of lane i.
template <int A, int B>
__device__ __forceinline__ void transpose4(uint32_t (&w)[4], bool a, bool b) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {  // exchange w[j] / w[j + 2] with the lane across A
    const uint32_t got = __shfl_xor_sync(0xffffffffu, a ? w[j] : w[j + 2], A);
    if (a)
      w[j] = got;
    else
      w[j + 2] = got;
  }
#pragma unroll
  for (int j = 0; j < 4; j += 2) {
    const uint32_t got = __shfl_xor_sync(0xffffffffu, b ? w[j] : w[j + 1], B);
    if (b)
      w[j] = got;
    else
      w[j + 1] = got;
  }
}

// Quantises the tokens [r0, r1) (rows of an 8-token tile; FULL: all 8, in 16-byte
// reads) of one (sequence, kv head) into its page (`off` bytes into both caches),
// the tile starting at row `tile`.  `src0`: offset of row 0's elements.
//
// A warp holds the tile as D/8 lanes per row: 256/D rows at a time, in D/32
// rounds.  The divisions for a round's scales are made by one lane of each
// group's 8 and handed round.  Keys: a row's words fill D/2 contiguous bytes.
// Values: a tile's words are [octet][pair][parity][group]; with D = 128 the lanes
// of one octet (2 groups x 2 row parities) hold 4 rounds = 4 pairs of words,
// which a 4 x 4 transpose turns into 16 contiguous bytes per lane, 512 per warp.
template <typename T, int D, bool FULL>
__device__ __forceinline__ void append_tile(const Int4AppendParams& p, int64_t off, int tile, int r0,
                                            int r1, int64_t src0) {
  constexpr int LR = D / 8, RP = 32 / LR, ROUNDS = 8 / RP;
  const int lane = threadIdx.x & 31, e = lane % LR, rr = lane / LR, g = e / 8, o = e % 8;
  const int bs = p.map.bs;
  uint4 x[2][ROUNDS];
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    const T* row = static_cast<const T*>(p.rows[kv]) + src0 + rr * p.r_st + e * 8;
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i, row += RP * p.r_st) {
      const int r = i * RP + rr;
      x[kv][i] = make_uint4(0u, 0u, 0u, 0u);
      if (FULL)
        x[kv][i] = load_row8<T>(row, true);
      else if (r >= r0 && r < r1)
        x[kv][i] = load_row8<T>(row, p.vec != 0);
    }
  }
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    uint8_t* page = p.cache[kv] + off;
    float inv;
    const uint32_t pair = int4_scale<T>(group_ranges<T, ROUNDS>(x[kv], o), &inv);
    const int mr = o % ROUNDS * RP + rr;  // the row this lane has scaled
    if (o < ROUNDS && (FULL || (mr >= r0 && mr < r1)))
      *reinterpret_cast<uint32_t*>(page + int4_pair(D, bs, tile + mr, g)) = pair;
    uint32_t w[ROUNDS];
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
      const int from = (lane & 24) + i;
      const uint32_t pi = __shfl_sync(0xffffffffu, pair, from);
      const float vi = __shfl_sync(0xffffffffu, inv, from);
      w[i] = int4_codes_of<T>(x[kv][i], pi, vi);
    }
    if constexpr (FULL && D == 128) {
      if (kv == 1) {
        // lanes of octet o: parity rr (bit 16), group g (bit 8); round i = pair i
        transpose4<16, 8>(w, rr != 0, g != 0);
        uint8_t* at = page + (tile >> 3) * (4 * D) + (o * 4 + rr * 2 + g) * 16;
        *reinterpret_cast<uint4*>(at) = make_uint4(w[0], w[1], w[2], w[3]);
        continue;
      }
    }
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
      const int r = i * RP + rr;
      if (FULL || (r >= r0 && r < r1))
        *reinterpret_cast<uint32_t*>(page + (kv ? int4_value_word(D, tile + r, g, o)
                                                : int4_key_word(D, tile + r, g, o))) = w[i];
    }
  }
}

// Ragged runs of tokens: one warp per (run of 8 or 16 positions, kv head).
//
// Reads 2 bytes per element and writes 9/16: 32,375 tokens of 8 kv heads, D 128,
// move 170 MB, 26 us at a copy's 6.55 TB/s.  It takes 43 (4.0 TB/s): issue binds
// it (73 % of the slots), about 1,190 warp instructions per 8-token tile; without
// any arithmetic the same loads and stores take 29, the ranges and the codes about
// 7 each.  64 registers (4 CTAs per SM, a few spilled) 42.8, 80 registers 44.4.
template <typename T, int D>
__global__ void __launch_bounds__(256, D == 256 ? 2 : 4) int4_append_kernel(const Int4AppendParams p, int warps) {
  const TokenMap& m = p.map;
  const int wid = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (wid >= warps) return;
  const int slot = wid / m.Hkv, h = wid - slot * m.Hkv;
  const int k = p.log2_run;
  const TokenRun t = find_run(m, slot, k);
  if (t.n == 0) return;
  const int L = p.lens[t.s * m.l_sb + h * m.l_sh];
  uint32_t flags = 0;
  if (L < 0) {
    flags = kStatusNegative;
  } else {
    const int64_t pos0 = ((static_cast<int64_t>(L) >> k) + t.run) << k;  // the run's position
    const int64_t over = static_cast<int64_t>(L) + t.n - pos0;
    if (over <= 0) return;
    const int a = L > pos0 ? static_cast<int>(L - pos0) : 0;  // its new rows: [a, end)
    const int end = over < (1 << k) ? static_cast<int>(over) : 1 << k;
    const int64_t pid = find_page(m, t.s, h, pos0 >> m.log2_bs, &flags);
    if (pid >= 0) {
      const int64_t off = pid * (static_cast<int64_t>(m.bs) * int4_row_bytes(D));
      const int tile = static_cast<int>(pos0) & (m.bs - 1);
      int64_t src0 = (t.t0 + pos0 - L) * p.r_st + h * p.r_sh;
#pragma unroll 1
      for (int r = 0; r < end; r += 8, src0 += 8 * p.r_st) {
        if (a <= r && end >= r + 8 && p.vec)
          append_tile<T, D, true>(p, off, tile + r, 0, 8, src0);
        else if (a < r + 8)
          append_tile<T, D, false>(p, off, tile + r, a - r, end - r, src0);
      }
    }
  }
  if (flags && p.status && (threadIdx.x & 31) == 0) atomicOr(p.status, flags);
}

// One token per sequence: one CTA per sequence, a warp per kv head, and the
// length, which every warp has read by then, in the same launch.  A chain of
// dependent loads (length, table, row): 4.4 us for 64 sequences of 8 kv heads.
template <typename T, int D>
__global__ void __launch_bounds__(256) int4_append_step_kernel(const Int4AppendParams p) {
  const TokenMap& m = p.map;
  const int s = blockIdx.x, lane = threadIdx.x & 31;
  uint32_t flags = 0;
  bool all = true;
  for (int h = threadIdx.x >> 5; h < m.Hkv; h += blockDim.x >> 5) {
    int32_t* lp = p.lens + s * m.l_sb + h * m.l_sh;
    const int L = *lp;
    uint32_t f = L < 0 ? kStatusNegative : 0u;
    const int64_t pid = L < 0 ? -1 : find_page(m, s, h, L >> m.log2_bs, &f);
    if (pid >= 0) {
      const int row = L & (m.bs - 1);
      append_tile<T, D, false>(p, pid * (static_cast<int64_t>(m.bs) * int4_row_bytes(D)), row & ~7,
                               row & 7, (row & 7) + 1,
                               (static_cast<int64_t>(s) - (row & 7)) * p.r_st + h * p.r_sh);
    }
    if (pid >= 0 && m.l_sh != 0 && p.increment && lane == 0) *lp = L + 1;
    all = all && pid >= 0;
    flags |= f;
  }
  if (flags && p.status && lane == 0) atomicOr(p.status, flags);
  if (m.l_sh == 0) {
    const bool ok = __syncthreads_and(all) != 0;  // every warp has read the length
    if (ok && p.increment && threadIdx.x == 0) p.lens[s * m.l_sb] += 1;
  }
}

// The lengths of ragged runs, after the rows: each grows by the number of new
// tokens before the first that had no place.  A length shared by the
// sequence's heads grows by the least of theirs.  One warp per sequence.
__global__ void __launch_bounds__(128) int4_lengths_kernel(const Int4AppendParams p) {
  const TokenMap& m = p.map;
  const int lane = threadIdx.x & 31;
  const int s = blockIdx.x * 4 + (threadIdx.x >> 5);
  // The rows' kernel has read every length; and whatever waits for this grid can
  // count on the rows.
  grid_dependency_wait();
  if (s >= m.B) return;
  const int t0 = m.cu[s], t1 = m.cu[s + 1];
  if (t0 < 0 || t1 > m.num_tokens || t1 <= t0) return;
  const int64_t n = t1 - t0;
  int64_t least = n;
  // Heads whose ids come from one table entry of a pool are in range together.
  const bool alike = m.l_sh == 0 && m.bt_sh == 0 && m.bt_add == 1 && m.bt_mul == m.Hkv &&
                     m.num_pages % m.Hkv == 0;
  const int heads = alike ? 1 : m.Hkv;
  for (int h = 0; h < heads; ++h) {
    int32_t* lp = p.lens + s * m.l_sb + h * m.l_sh;
    const int64_t L = *lp;
    int64_t got = L < 0 ? 0 : n;
    uint32_t flags = 0;
    if (L >= 0)
      for (int64_t pg = (L >> m.log2_bs) + lane; (pg << m.log2_bs) < L + n; pg += 32)
        if (find_page(m, s, h, pg, &flags) < 0) {
          const int64_t before = (pg << m.log2_bs) - L;
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
  int32_t zero_rest;       // rows of no sequence become zeros
  int32_t log2_run;        // as in Int4AppendParams
};

// lo + s c of 8 elements: c, s and lo are exact in T, so one packed fma rounds
// once.  The rounding of s may put code 15 of a range as wide as T's past T's
// largest value: such a value saturates.
template <typename T>
__device__ __forceinline__ uint4 int4_values(uint32_t word, uint32_t pair) {
  uint32_t r[4];
  int4_codes<T>(word, r);
  const uint32_t s = __byte_perm(pair, pair, 0x1010), lo = __byte_perm(pair, pair, 0x3232);
  constexpr uint32_t kMax = std::is_same<T, __half>::value ? 0x7bff7bffu : 0x7f7f7f7fu;
#pragma unroll
  for (int m = 0; m < 4; ++m) r[m] = min2_nan<T>(fma2<T>(s, r[m], lo), kMax);
  return make_uint4(r[0], r[1], r[2], r[3]);
}

// One warp per (run of 8 or 16 positions, kv head), lanes as in append_tile: the
// rounds of a tile of which every row is wanted differ by constant offsets.
// 32,375 tokens of 8 kv heads, D 128 (170 MB, 26 us at a copy's rate): 32 us,
// 5.3 TB/s; waits for loads, 58 % of the issue slots busy.  More CTAs per SM with
// fewer registers: 32.6 to 34.3.
template <typename T, int D>
__global__ void __launch_bounds__(256) int4_read_kernel(const Int4ReadParams p, int warps) {
  constexpr int LR = D / 8, RP = 32 / LR, ROUNDS = 8 / RP;
  const TokenMap& m = p.map;
  const int wid = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (wid >= warps) return;
  const int slot = wid / m.Hkv, h = wid - slot * m.Hkv, k = p.log2_run, run = 1 << k;
  const int lane = threadIdx.x & 31, e = lane % LR, rr = lane / LR, g = e / 8, o = e % 8;
  const int64_t column = h * p.o_sh + e * 8;
  if (p.zero_rest && m.cu) {
    // Slots past the last sequence's: rows from cu[B]; the slots before the
    // first sequence's: rows up to cu[0].  Without sequences all rows lie behind.
    const int first = m.cu[0], last = m.B > 0 ? max(m.cu[m.B], 0) : 0;
    const int past = slot - ((last >> k) + 2 * m.B);
    const int64_t z0 = (past >= 0 ? last : 0) + (static_cast<int64_t>(past >= 0 ? past : slot) << k);
    const int64_t z1 = past >= 0 ? m.num_tokens : min(first, m.num_tokens);
    for (int64_t r = z0 + rr; r < z1 && r < z0 + run; r += RP)
#pragma unroll
      for (int kv = 0; kv < 2; ++kv)
        *reinterpret_cast<uint4*>(static_cast<T*>(p.out[kv]) + r * p.o_st + column) =
            make_uint4(0u, 0u, 0u, 0u);
    if (past >= 0) return;
  }
  const TokenRun t = find_run(m, slot, k);
  if (t.n == 0) return;
  const int L = p.lens[t.s * m.l_sb + h * m.l_sh];
  const int64_t start = p.starts ? p.starts[t.s * p.start_sb] : 0;
  const int64_t pos0 = ((start >> k) + t.run) << k;  // the run's position (start may be < 0)
  const int64_t over = start + t.n - pos0;
  if (over <= 0) return;
  const int a = start > pos0 ? static_cast<int>(start - pos0) : 0;  // its rows: [a, end)
  const int end = over < run ? static_cast<int>(over) : run;
  const int64_t left = L - pos0;
  const int have = left < 0 ? 0 : (left < end ? static_cast<int>(left) : end);  // rows from here on hold no token
  uint32_t flags = 0;
  int64_t pid = -1;
  if (pos0 >= 0 && a < have) {
    pid = find_page(m, t.s, h, pos0 >> m.log2_bs, &flags);
    if (flags && p.status && lane == 0)
      atomicOr(p.status, flags & kStatusAppendFull ? kStatusClamp : flags);
  }
  const int tile = (static_cast<int>(pos0) & (m.bs - 1)) + rr;  // this lane's first row of the page
  const int64_t off = pid * (static_cast<int64_t>(m.bs) * int4_row_bytes(D));
  int64_t to = (t.t0 + pos0 - start + rr) * p.o_st + column;
#pragma unroll 1
  for (int r = 0; r < end; r += 8, to += 8 * p.o_st) {
    if (a >= r + 8) continue;
    uint32_t w[2][ROUNDS], pr[2][ROUNDS];
    const bool full = pid >= 0 && a <= r && have >= r + 8;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const uint8_t* page = p.cache[kv] + off;
      const uint8_t* code = page + (kv ? int4_value_word(D, tile + r, g, o) : int4_key_word(D, tile + r, g, o));
      const uint8_t* pairs = page + int4_pair(D, m.bs, tile + r, g);
#pragma unroll
      for (int i = 0; i < ROUNDS; ++i) {
        const int row = r + i * RP + rr;
        w[kv][i] = pr[kv][i] = 0u;
        if (full || (pid >= 0 && row >= a && row < have)) {
          // a round's rows lie RP further: 128 bytes of keys, 16 of values and pairs
          w[kv][i] = __ldg(reinterpret_cast<const uint32_t*>(code + i * (kv ? 16 : 128)));
          pr[kv][i] = __ldg(reinterpret_cast<const uint32_t*>(pairs + i * 16));
        }
      }
    }
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      T* out = static_cast<T*>(p.out[kv]) + to;
#pragma unroll
      for (int i = 0; i < ROUNDS; ++i, out += RP * p.o_st) {
        const int row = r + i * RP + rr;
        if (full || (row >= a && row < end))
          *reinterpret_cast<uint4*>(out) = int4_values<T>(w[kv][i], pr[kv][i]);
      }
    }
  }
}

}  // namespace pab

namespace {

using pabh::aligned;
using pabh::fail;

// Whether a call has rows to write; `rest`: rows of no sequence too.
bool any_rows(const pab200_int4_rows_args* a, bool rest) {
  return a->num_tokens > 0 && (a->num_seqs > 0 || rest);
}

// The checks that append and read-back share; fills the token map.
int check_int4(const pab200_int4_rows_args* a, pab::TokenMap* m, bool rest) {
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
  if (int64_t(a->max_blocks) * bs >= (int64_t(1) << 31) || a->num_tokens >= (int64_t(1) << 30) ||
      (pab::num_slots(a->num_tokens, a->num_seqs, a->cu_tokens != nullptr, 3) + 8) * a->num_kv_heads >=
          (int64_t(1) << 31))
    return fail(PAB200_ERR_UNSUPPORTED,
                "max_blocks*block_size, or num_tokens*num_kv_heads/8, too large (>= 2^31)");
  if (!any_rows(a, rest)) return PAB200_OK;
  const bool seqs = a->num_seqs > 0;
  if (!a->k_rows || !a->v_rows || (seqs && !a->seqlens))
    return fail(PAB200_ERR_INVALID_ARGUMENT, "k_rows, v_rows or seqlens is null");
  if (seqs && a->max_blocks > 0 && a->num_pages > 0 && (!a->k_cache || !a->v_cache || !a->block_table))
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
  m->num_tokens = static_cast<int32_t>(a->num_tokens);
  m->bt_mul = a->bt_page_mul;
  m->bt_add = a->bt_page_add;
  m->B = a->num_seqs;
  m->Hkv = a->num_kv_heads;
  m->bs = bs;
  m->log2_bs = bs == 8 ? 3 : (bs == 16 ? 4 : (bs == 32 ? 5 : 6));
  m->maxb = a->num_pages > 0 ? a->max_blocks : 0;
  return PAB200_OK;
}

bool rows_vec(const pab200_int4_rows_args* a) {
  return aligned(a->k_rows, 16) && aligned(a->v_rows, 16) && a->row_stride_t % 8 == 0 &&
         a->row_stride_h % 8 == 0;
}

// Positions a warp takes (log2): two tiles of a page where there are pages of two,
// which shares the search for the run and its page (32,375 tokens of 8 kv heads,
// D 128, pages of 16: append 50 us with one tile per warp, 44 with two at 80
// registers; read-back 34 and 32).
int log2_run(const pab200_int4_rows_args* a) { return a->block_size >= 16 ? 4 : 3; }

// Warps of a kernel over (run, kv head) pairs.
int run_warps(const pab200_int4_rows_args* a, int k) {
  // two slots more: the read-back's rows behind the last sequence
  const int more = a->cu_tokens ? 2 : 0;
  return static_cast<int>(
      (pab::num_slots(a->num_tokens, a->num_seqs, a->cu_tokens != nullptr, k) + more) *
      a->num_kv_heads);
}

template <typename T, int D>
void launch_append(const pab::Int4AppendParams& p, int warps, cudaStream_t s) {
  if (p.map.cu) {
    pab::int4_append_kernel<T, D><<<(warps + 7) / 8, 256, 0, s>>>(p, warps);
  } else {
    const int per_cta = p.map.Hkv < 8 ? p.map.Hkv : 8;
    pab::int4_append_step_kernel<T, D><<<p.map.B, per_cta * 32, 0, s>>>(p);
  }
}

template <typename T>
void launch_append_d(const pab::Int4AppendParams& p, int D, int warps, cudaStream_t s) {
  switch (D) {
    case 64: launch_append<T, 64>(p, warps, s); break;
    case 128: launch_append<T, 128>(p, warps, s); break;
    default: launch_append<T, 256>(p, warps, s); break;
  }
}

template <typename T>
void launch_read(const pab::Int4ReadParams& p, int D, int warps, cudaStream_t s) {
  const int grid = (warps + 7) / 8;
  switch (D) {
    case 64: pab::int4_read_kernel<T, 64><<<grid, 256, 0, s>>>(p, warps); break;
    case 128: pab::int4_read_kernel<T, 128><<<grid, 256, 0, s>>>(p, warps); break;
    default: pab::int4_read_kernel<T, 256><<<grid, 256, 0, s>>>(p, warps); break;
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
  const int rc = check_int4(a, &p.map, false);
  if (rc || !any_rows(a, false)) return rc;
  if (increment && a->num_seqs > 1 && a->seqlens_stride_b == 0)
    return fail(PAB200_ERR_INVALID_ARGUMENT,
                "sequences share a length (seqlens_stride_b is 0): it cannot be advanced for each");
  p.cache[0] = static_cast<uint8_t*>(a->k_cache);
  p.cache[1] = static_cast<uint8_t*>(a->v_cache);
  p.rows[0] = a->k_rows;
  p.rows[1] = a->v_rows;
  p.lens = a->seqlens;
  p.status = a->status;
  p.r_st = a->row_stride_t;
  p.r_sh = a->row_stride_h;
  p.vec = rows_vec(a);
  p.increment = increment ? 1 : 0;
  p.log2_run = log2_run(a);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->dtype == PAB200_DTYPE_BF16)
    launch_append_d<__nv_bfloat16>(p, a->head_size, run_warps(a, p.log2_run), s);
  else
    launch_append_d<__half>(p, a->head_size, run_warps(a, p.log2_run), s);
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess && increment && a->cu_tokens) {
    // scheduled while the rows' kernel drains; waits for it before any length
    pabh::LaunchCfg lc(dim3((a->num_seqs + 3) / 4), dim3(128), 0, s, true);
    e = cudaLaunchKernelEx(&lc.cfg, pab::int4_lengths_kernel, p);
  }
  return e == cudaSuccess ? PAB200_OK : pabh::cuda_fail(e, "4-bit append launch");
}

PAB200_EXPORT int pab200_kv_read_int4(const pab200_int4_rows_args* a, const int32_t* starts,
                                      int64_t starts_stride, int32_t zero_rest, void* stream) {
  pab::Int4ReadParams p{};
  const int rc = check_int4(a, &p.map, zero_rest != 0);
  if (rc || !any_rows(a, zero_rest != 0)) return rc;
  if (!rows_vec(a))
    return fail(PAB200_ERR_ALIGNMENT, "rows must be 16-byte aligned with strides that are multiples of 8");
  p.cache[0] = static_cast<const uint8_t*>(a->k_cache);
  p.cache[1] = static_cast<const uint8_t*>(a->v_cache);
  p.out[0] = a->k_rows;
  p.out[1] = a->v_rows;
  p.lens = a->seqlens;
  p.starts = starts;
  p.start_sb = starts_stride;
  p.zero_rest = zero_rest ? 1 : 0;
  p.status = a->status;
  p.o_st = a->row_stride_t;
  p.o_sh = a->row_stride_h;
  p.log2_run = log2_run(a);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->dtype == PAB200_DTYPE_BF16)
    launch_read<__nv_bfloat16>(p, a->head_size, run_warps(a, p.log2_run), s);
  else
    launch_read<__half>(p, a->head_size, run_warps(a, p.log2_run), s);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? PAB200_OK : pabh::cuda_fail(e, "4-bit read launch");
}
