// Page-sparse decode: key bounds of pages, selection of pages by a query, and
// the decode over the selected pages.
#include "host.h"
#include "int4.cuh"
#include "tokens.cuh"

namespace pab {

struct BoundsParams {
  TokenMap map;
  void* bounds;            // [pages][2][D]: minimum, maximum
  const void* rows;
  const int32_t* lens;     // lengths before the new tokens
  uint32_t* status;
  int64_t r_st, r_sh;
  int32_t vec;
};

// One warp per (page, kv head): the minimum and maximum of the page's new rows,
// D/8 lanes per row and 256/D rows at a time, joined with the page's bounds when
// it began before.  Comparisons work on the 16-bit pairs as they are.  Bound by
// reading the rows: 32,375 tokens of 8 kv heads, D 128 (66 MB, and 8 MB of bounds
// to write): 12.3 us from L2, 19 from HBM; one token each of 64 sequences 2.7 us, a
// chain of dependent loads.
template <typename T, int D>
__global__ void __launch_bounds__(256) page_bounds_kernel(const BoundsParams p, int warps) {
  constexpr int LR = D / 8, RP = 32 / LR;
  const TokenMap& m = p.map;
  const int lane = threadIdx.x & 31;
  const int wid = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (wid >= warps) return;
  const int slot = wid / m.Hkv, h = wid - slot * m.Hkv;
  const TokenRun t = find_run(m, slot, m.log2_bs);
  if (t.n == 0) return;
  const int L = p.lens[t.s * m.l_sb + h * m.l_sh];
  uint32_t flags = 0;
  const int64_t pg = (static_cast<int64_t>(L) >> m.log2_bs) + t.run;
  const int64_t pos0 = pg << m.log2_bs;                 // the page's position
  const int64_t end = static_cast<int64_t>(L) + t.n - pos0;
  if (L >= 0 && end <= 0) return;
  const int64_t pid = L < 0 ? -1 : find_page(m, t.s, h, pg, &flags);
  if (pid < 0) {
    if (p.status && lane == 0) atomicOr(p.status, L < 0 ? kStatusNegative : flags);
    return;
  }
  const int r0 = L > pos0 ? static_cast<int>(L - pos0) : 0;  // first new row, and the end
  const int r1 = end < m.bs ? static_cast<int>(end) : m.bs;
  const int e = lane % LR, rr = lane / LR;
  const T* rows = static_cast<const T*>(p.rows) + (t.t0 + pos0 - L) * p.r_st + h * p.r_sh + e * 8;
  constexpr uint32_t kInf = std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u;
  uint32_t mn[4], mx[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    mn[i] = kInf;
    mx[i] = kInf | 0x80008000u;
  }
  auto take = [&](const uint4& lo, const uint4& hi) {
    mn[0] = min2_nan<T>(mn[0], lo.x);
    mn[1] = min2_nan<T>(mn[1], lo.y);
    mn[2] = min2_nan<T>(mn[2], lo.z);
    mn[3] = min2_nan<T>(mn[3], lo.w);
    mx[0] = max2_nan<T>(mx[0], hi.x);
    mx[1] = max2_nan<T>(mx[1], hi.y);
    mx[2] = max2_nan<T>(mx[2], hi.z);
    mx[3] = max2_nan<T>(mx[3], hi.w);
  };
  T* out = static_cast<T*>(p.bounds) + pid * (2 * D) + e * 8;
  if (r0 > 0) take(*reinterpret_cast<const uint4*>(out), *reinterpret_cast<const uint4*>(out + D));
  constexpr int U = 8;  // rows in flight per lane
  for (int r = r0 + rr; r < r1; r += RP * U) {
    uint4 x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int ru = r + u * RP < r1 ? r + u * RP : r;  // past the end: row r again
      x[u] = load_row8<T>(rows + ru * p.r_st, p.vec != 0);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) take(x[u], x[u]);
  }
#pragma unroll
  for (int o = LR; o < 32; o <<= 1)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      mn[i] = min2_nan<T>(mn[i], __shfl_xor_sync(0xffffffffu, mn[i], o));
      mx[i] = max2_nan<T>(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], o));
    }
  if (rr != 0) return;
  *reinterpret_cast<uint4*>(out) = make_uint4(mn[0], mn[1], mn[2], mn[3]);
  *reinterpret_cast<uint4*>(out + D) = make_uint4(mx[0], mx[1], mx[2], mx[3]);
}

// N consecutive 32-bit words (aligned to min(N, 4) words), read once.
template <int N>
__device__ __forceinline__ void ld_global_words(const void* p, uint32_t (&w)[N]) {
  if constexpr (N == 1) {
    w[0] = __ldg(static_cast<const uint32_t*>(p));
  } else if constexpr (N == 2) {
    const uint2 v = __ldg(static_cast<const uint2*>(p));
    w[0] = v.x;
    w[1] = v.y;
  } else {
    const uint4 v = __ldg(static_cast<const uint4*>(p));
    w[0] = v.x;
    w[1] = v.y;
    w[2] = v.z;
    w[3] = v.w;
  }
}

struct SelectParams {
  const void* q;
  const void* bounds;
  const int32_t* lens;
  const int32_t* bt;
  int32_t* tables;     // [B][Hkv][keep]
  int32_t* out_lens;   // [B][Hkv]
  float2* scores;      // [B * Hkv][maxb]: score, sum of its terms' sizes
  uint32_t* status;
  int64_t q_sb, q_sh, l_sb, l_sh, bt_sb, bt_sh, bt_si, num_pages;
  int32_t bt_mul, bt_add, B, Hkv, G, bs, maxb, keep, sink, recent, chunk;
  int32_t chained;     // the decode grid of the same call follows
};

__device__ __forceinline__ int clamped_length(const SelectParams& p, int s, int h) {
  const int L = p.lens[s * p.l_sb + h * p.l_sh];
  const int64_t cap = static_cast<int64_t>(p.maxb) * p.bs;
  return L < 0 ? 0 : (L > cap ? static_cast<int>(cap) : L);
}

// A page's score is the sum over the group and the head elements of max(q * min,
// q * max), the upper bound of the group's summed scores; by definition in 64 bits,
// rounded to fp32.  Where nothing is infinite that is the sum over the elements of
// max * (sum of the group's positive query parts) + min * (sum of the negative ones).  Which
// pages rank next to the border must not hang on the order of an fp32 sum, but
// 64-bit conversions and sums bound the kernel (24,400 pages of 8 kv heads, D
// 128: 100 MB of bounds, 15 us at a copy's rate; 36 to 40 us in 64 bits, 26 as
// below, about 3.8 TB/s).  So this kernel sums in fp32, with the sum A of the terms' sizes beside it: an fp32
// score is within kScoreError * A of the rounded 64-bit one (at most 17 rounded
// products and sums per lane, 5 sums over the warp, the rounding of the query
// sums, of the 64-bit score and of A: 25 * 2^-24).  The selection settles the few
// pages that this leaves open in 64 bits.
constexpr float kScoreError = 32.f / 16777216.f;

// Positive and negative parts of the query, summed over the group in 64 bits.
template <typename T>
__device__ __forceinline__ double2 query_parts(const SelectParams& p, const T* q, int d) {
  double up = 0.0, dn = 0.0;
#pragma unroll 8
  for (int g = 0; g < p.G; ++g) {
    const float x = static_cast<float>(q[g * p.q_sh + d]);
    up += x > 0.f ? x : 0.f;
    dn += x > 0.f ? 0.f : x;  // a NaN makes this one NaN
  }
  return make_double2(up, dn);
}

// blockIdx.x: chunk of p.chunk pages, 8 warps of p.chunk / 8 (at most 64), a
// whole warp per page.  A warp lives for dozens of pages with the next four on
// their way while it sums four (two to eight pages at a time and chunks of 64 to
// 512 pages: all 25 to 30 us at the size above).
template <typename T, int D>
__global__ void __launch_bounds__(256, 4) page_scores_kernel(const SelectParams p) {
  constexpr int V = D / 32;                         // elements per lane
  constexpr int W = V / 2;                          // 32-bit words of them
  constexpr int U = 4;                              // pages at a time
  __shared__ float qs[2][D];
  grid_launch_dependents();
  const int u = blockIdx.y, s = u / p.Hkv, h = u - s * p.Hkv;
  const int lane = threadIdx.x & 31, per = p.chunk / 8;
  const int c0 = p.sink + blockIdx.x * p.chunk, w0 = c0 + (threadIdx.x >> 5) * per;
  // The table entries, the query and the length are loaded together, before it
  // is known whether the chunk holds a page.
  int id[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int i = 32 * j + lane;
    id[j] = i < per && w0 + i < p.maxb ? p.bt[s * p.bt_sb + h * p.bt_sh + (w0 + i) * p.bt_si] : 0;
  }
  const T* q = static_cast<const T*>(p.q) + s * p.q_sb + static_cast<int64_t>(h) * p.G * p.q_sh;
  for (int d = threadIdx.x; d < D; d += 256) {
    const double2 x = query_parts<T>(p, q, d);
    qs[0][d] = static_cast<float>(x.x);
    qs[1][d] = static_cast<float>(x.y);
  }
  const int n = (clamped_length(p, s, h) + p.bs - 1) / p.bs;
  const int c1 = min(c0 + p.chunk, n - p.recent);
  if (n <= p.keep || c0 >= c1) {
    grid_dependency_wait();
    return;
  }
  const int count = min(per, c1 - w0);
  // This warp's pages: ids, -1 for one out of range.
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t pid = static_cast<int64_t>(id[j]) * p.bt_mul + static_cast<int64_t>(h) * p.bt_add;
    const bool ok = pid >= 0 && pid < p.num_pages;
    if (!ok && 32 * j + lane < count && p.status) atomicOr(p.status, kStatusBadPage);
    id[j] = ok ? static_cast<int>(pid) : -1;
  }
  __syncthreads();
  float up[V], dn[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    up[i] = qs[0][lane * V + i];
    dn[i] = qs[1][lane * V + i];
  }
  struct Pages {
    uint32_t mn[U][W], mx[U][W];
    int bad;  // bit v: page v has no bounds
  };
  auto load = [&](int t, Pages& x) {
    x.bad = 0;
#pragma unroll
    for (int v = 0; v < U; ++v) {
      const int pid = __shfl_sync(0xffffffffu, t + v < 32 ? id[0] : id[1], (t + v) & 31);
      if (pid < 0) x.bad |= 1 << v;
      // past the end: any page will do
      const T* b = static_cast<const T*>(p.bounds) +
                   static_cast<int64_t>(t + v < count && pid >= 0 ? pid : 0) * (2 * D) + lane * V;
      ld_global_words<W>(b, x.mn[v]);
      ld_global_words<W>(b + D, x.mx[v]);
    }
  };
  // Four sums over the warp at once: lanes of the upper half go on with pages 2
  // and 3, of every half's upper half with the odd one.
  const bool h16 = lane & 16, h8 = lane & 8;
  auto warp_sums = [&](const float (&a)[U]) {
    const float g0 = __shfl_xor_sync(0xffffffffu, h16 ? a[0] : a[2], 16);
    const float g1 = __shfl_xor_sync(0xffffffffu, h16 ? a[1] : a[3], 16);
    const float b0 = (h16 ? a[2] : a[0]) + g0, b1 = (h16 ? a[3] : a[1]) + g1;
    float r = (h8 ? b1 : b0) + __shfl_xor_sync(0xffffffffu, h8 ? b0 : b1, 8);
    r += __shfl_xor_sync(0xffffffffu, r, 4);
    r += __shfl_xor_sync(0xffffffffu, r, 2);
    return r + __shfl_xor_sync(0xffffffffu, r, 1);
  };
  float2* out = p.scores + static_cast<int64_t>(u) * p.maxb + w0;
  auto score = [&](int t, const Pages& x) {
    float a[U], size[U];
#pragma unroll
    for (int v = 0; v < U; ++v) {
      a[v] = size[v] = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const float2 lo = unpack2<T>(x.mn[v][i]), hi = unpack2<T>(x.mx[v][i]);
        a[v] = fmaf(hi.x, up[2 * i], a[v]);
        a[v] = fmaf(lo.x, dn[2 * i], a[v]);
        a[v] = fmaf(hi.y, up[2 * i + 1], a[v]);
        a[v] = fmaf(lo.y, dn[2 * i + 1], a[v]);
        size[v] = fmaf(fabsf(hi.x), up[2 * i], size[v]);
        size[v] = fmaf(fabsf(lo.x), -dn[2 * i], size[v]);
        size[v] = fmaf(fabsf(hi.y), up[2 * i + 1], size[v]);
        size[v] = fmaf(fabsf(lo.y), -dn[2 * i + 1], size[v]);
      }
    }
    const float r = warp_sums(a), z = warp_sums(size);
    const int v = (h16 ? 2 : 0) + (h8 ? 1 : 0);
    if ((lane & 7) == 0 && t + v < count)
      out[t + v] = x.bad >> v & 1 ? make_float2(-INFINITY, 0.f) : make_float2(r, z);
  };
  Pages x, y;
  if (count > 0) load(0, x);
  for (int t = 0; t < count; t += 2 * U) {
    if (t + U < count) load(t + U, y);
    score(t, x);
    if (t + U >= count) break;
    if (t + 2 * U < count) load(t + 2 * U, x);
    score(t + U, y);
  }
  // In a decode call the planner runs beside this kernel: what waits for this
  // grid must be able to count on the planner's end too.
  grid_dependency_wait();
}

// Sum over the lanes of a warp, in every lane.
__device__ __forceinline__ double warp_sum(double a) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  return a;
}

// The score of bounds `b` term by term, for infinities: the query's parts would
// multiply an infinite bound that the maximum leaves aside by 0.  NaN where a
// query element of 0 meets an infinite bound.
template <typename T, int D>
__device__ __forceinline__ float term_score(const SelectParams& p, const T* q, const T* b) {
  double a = 0.0;
#pragma unroll 1
  for (int d = threadIdx.x & 31; d < D; d += 32)
#pragma unroll 1
    for (int g = 0; g < p.G; ++g) {
      const double x = static_cast<float>(q[g * p.q_sh + d]);
      const double u = x * static_cast<float>(b[d]), v = x * static_cast<float>(b[D + d]);
      a += u != u || v != v ? u + v : (u > v ? u : v);
    }
  return static_cast<float>(warp_sum(a));
}

// The score of page `pid` by its definition, in every lane of a warp; `q`: the
// group's queries, `qs`: their parts in 64 bits.
template <typename T, int D>
__device__ __forceinline__ float exact_score(const SelectParams& p, int64_t pid, const T* q,
                                             const double* qs) {
  if (pid < 0 || pid >= p.num_pages) return -INFINITY;
  const T* b = static_cast<const T*>(p.bounds) + pid * (2 * D);
  double a = 0.0;
  for (int d = threadIdx.x & 31; d < D; d += 32) {
    a = fma(static_cast<double>(static_cast<float>(b[D + d])), qs[d], a);
    a = fma(static_cast<double>(static_cast<float>(b[d])), qs[D + d], a);
  }
  a = warp_sum(a);
  // finite 16-bit bounds and queries have a sum far inside 64 bits' range
  if (!(fabs(a) <= 1e300)) return term_score<T, D>(p, q, b);
  return static_cast<float>(a);
}

// Order-preserving key of a score: larger scores have larger keys, -0 and +0
// the same, NaN the largest; and the score of a key.
__device__ __forceinline__ uint32_t score_key(float f) {
  if (f != f) return 0xffffffffu;
  const uint32_t b = __float_as_uint(f + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_score(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// The larger of two numbers, NaN if either is.
__device__ __forceinline__ float fmax_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Sums of x.x and of x.y over the block's threads before this one, and the
// totals (`warp_sum` is free again after the next barrier).
template <int NTH>
__device__ __forceinline__ int2 block_scan(int2 x, int2* warp_sum, int2* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto scan = [&](int2 v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, v.x, o), b = __shfl_up_sync(0xffffffffu, v.y, o);
      if (lane >= o) {
        v.x += a;
        v.y += b;
      }
    }
    return v;
  };
  const int2 v = scan(x);
  if (lane == 31) warp_sum[warp] = v;
  __syncthreads();
  const int2 w = scan(lane < NTH / 32 ? warp_sum[lane] : make_int2(0, 0));
  *total = make_int2(__shfl_sync(0xffffffffu, w.x, 31), __shfl_sync(0xffffffffu, w.y, 31));
  const int before_x = __shfl_sync(0xffffffffu, w.x, warp ? warp - 1 : 0);
  const int before_y = __shfl_sync(0xffffffffu, w.y, warp ? warp - 1 : 0);
  return make_int2((warp ? before_x : 0) + v.x - x.x, (warp ? before_y : 0) + v.y - x.y);
}

// One CTA per (sequence, kv head): the pages to attend to, ascending.
//
// The k-th largest fp32 score T is found by counting: the range between the
// smallest and the largest key is cut into NTH bins (the scores fill their own
// range, so that no bin is crowded and the shared-memory counters do not
// serialise); when the bin that holds the k-th has at most NTH keys, they are
// compared with one another, else it becomes the range.  With e the bound of the
// scores' errors, the true k-th lies within e of T: pages above T + 2 e are kept,
// pages below T - 2 e are not, and unless exactly as many as are still wanted lie
// between, those are scored in 64 bits and ranked, equal ones by page.  (A score
// or a size that is not finite leaves every page open.)  A thread owns
// consecutive pages, so that one scan places them in order.  About 12 us for 32
// units of up to 8,192 pages.  The kernel is a
// chain of short steps run once by few CTAs: loops are kept rolled, since cold
// instructions cost as much as the steps.
template <typename T, int D, int NTH>
__global__ void __launch_bounds__(NTH) select_pages_kernel(const SelectParams p) {
  constexpr int kLog2Bins = NTH == 1024 ? 10 : 8;
  constexpr int kHeld = NTH * 8;  // keys kept in shared memory (padded: no bank conflicts)
  constexpr int kFew = 64;        // open pages compared directly
  __shared__ uint32_t keys[kHeld + kHeld / 32];
  __shared__ int hist[NTH];
  __shared__ uint32_t list[NTH];
  __shared__ double qs[2 * D];
  __shared__ int2 sums[3][32];
  __shared__ uint32_t sh_lo[32], sh_hi[32];
  __shared__ float sh_size[32];
  __shared__ uint32_t sh_key;
  __shared__ int sh_bin, sh_rank, sh_count, sh_listed;
  // The decode grid of the same call waits for the tables; whatever follows a
  // selection on its own may read its lengths first, so that has to start later.
  if (p.chained) grid_launch_dependents();
  const int u = blockIdx.x, s = u / p.Hkv, h = u - s * p.Hkv;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int L = clamped_length(p, s, h);
  const int raw = p.lens[s * p.l_sb + h * p.l_sh];
  const int n = (L + p.bs - 1) / p.bs;
  const int32_t* bt = p.bt + s * p.bt_sb + h * p.bt_sh;
  int32_t* out = p.tables + static_cast<int64_t>(u) * p.keep;
  hist[tid] = 0;
  const T* q = static_cast<const T*>(p.q) + s * p.q_sb + static_cast<int64_t>(h) * p.G * p.q_sh;
  if (n > p.keep) {  // the query's parts, while the scores are still summed
    for (int d = tid; d < D; d += NTH) {
      const double2 x = query_parts<T>(p, q, d);
      qs[d] = x.x;
      qs[D + d] = x.y;
    }
  }
  grid_dependency_wait();  // the scores; nothing of this call is written before
  if (tid == 0) {
    if (raw != L && p.status) atomicOr(p.status, raw < 0 ? kStatusNegative : kStatusClamp);
    p.out_lens[u] = n <= p.keep ? L : (p.keep - 1) * p.bs + L - (n - 1) * p.bs;
  }
  if (n <= p.keep) {
    for (int i = tid; i < p.keep; i += NTH) out[i] = i < n ? bt[i * p.bt_si] : -1;
    return;
  }
  const int c0 = p.sink, m = n - p.sink - p.recent;  // candidates, of which k are kept
  const int k = p.keep - p.sink - p.recent;
  for (int i = tid; i < p.sink + p.recent; i += NTH) {
    const bool first = i < p.sink;
    out[first ? i : p.keep - p.recent + i - p.sink] =
        bt[(first ? i : n - p.recent + i - p.sink) * p.bt_si];
  }
  if (k == 0) return;
  float2* sc = p.scores + static_cast<int64_t>(u) * p.maxb + c0;
  uint32_t lo = 0xffffffffu, hi = 0u;
  float size = 0.f;
#pragma unroll 4
  for (int i = tid; i < m; i += NTH) {
    const float2 x = __ldcg(sc + i);
    const uint32_t key = score_key(x.x);
    if (i < kHeld) keys[i + (i >> 5)] = key;
    lo = min(lo, key);
    hi = max(hi, key);
    size = fmax_nan(size, x.y);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    size = fmax_nan(size, __shfl_xor_sync(0xffffffffu, size, o));
  }
  if (lane == 0) sh_size[warp] = size;
  // This thread's pages, in order, with their keys.
  const int per = (m + NTH - 1) / NTH;
  const int i0 = min(tid * per, m), i1 = min(i0 + per, m);
  auto key_of = [&](int i) { return i < kHeld ? keys[i + (i >> 5)] : score_key(__ldcg(&sc[i].x)); };
  uint32_t khi = 0xffffffffu, klo = 0u;  // keys above khi are kept, below klo not
  bool sure = true, exact = false;       // exact: the search is among the open pages
  auto open = [&](uint32_t x) { return !sure || (x <= khi && x >= klo); };
  // The keys the search is among: all, or the 64-bit ones (in place of the
  // sizes, read by then) of the open pages.
  auto walk = [&](auto&& fn) {
#pragma unroll 1
    for (int i = i0; i < i1; ++i) {
      const uint32_t x = key_of(i);
      if (!exact)
        fn(x);
      else if (open(x))
        fn(score_key(__ldcg(&sc[i].y)));
    }
  };
  int rank = k, want = 0, opened = 0;
  int2 before = make_int2(0, 0), total;
  bool few = false;
#pragma unroll 1
  for (;;) {
    // The rank-th largest key, left in lo, with its rank among the equal ones.
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    if (lane == 0) {
      sh_lo[warp] = lo;
      sh_hi[warp] = hi;
    }
    __syncthreads();
    lo = __reduce_min_sync(0xffffffffu, sh_lo[lane % (NTH / 32)]);
    hi = __reduce_max_sync(0xffffffffu, sh_hi[lane % (NTH / 32)]);
#pragma unroll 1
    while (lo < hi) {
      const int bits = 32 - __clz(hi - lo);
      const int shift = bits > kLog2Bins ? bits - kLog2Bins : 0;
      walk([&](uint32_t x) {
        if (x >= lo && x <= hi) atomicAdd(&hist[(x - lo) >> shift], 1);
      });
      if (tid == 0) sh_listed = 0;
      __syncthreads();
      // thread t looks at bin NTH - 1 - t: how many keys lie in the bins above it
      const int mine = hist[NTH - 1 - tid];
      const int above = block_scan<NTH>(make_int2(mine, 0), sums[0], &total).x;
      if (above < rank && rank <= above + mine) {
        sh_bin = NTH - 1 - tid;
        sh_rank = rank - above;
        sh_count = mine;
      }
      hist[NTH - 1 - tid] = 0;
      __syncthreads();
      rank = sh_rank;
      lo += static_cast<uint32_t>(sh_bin) << shift;
      const uint32_t span = (1u << shift) - 1u;  // lo + span may pass the largest key
      if (hi - lo > span) hi = lo + span;
      const int count = sh_count;
      if (lo < hi && count <= NTH) {
        walk([&](uint32_t x) {
          if (x >= lo && x <= hi) list[atomicAdd(&sh_listed, 1)] = x;
        });
        __syncthreads();
        if (tid < count) {
          const uint32_t x = list[tid];
          int above_x = 0, equal_x = 0;
          for (int i = 0; i < count; ++i) {
            above_x += list[i] > x;
            equal_x += list[i] == x;
          }
          // equal keys all write the same two words
          if (above_x < rank && rank <= above_x + equal_x) {
            sh_key = x;
            sh_rank = rank - above_x;
          }
        }
        __syncthreads();
        lo = hi = sh_key;
        rank = sh_rank;
      }
    }
    if (exact) break;
    for (int w = 0; w < NTH / 32; ++w) size = fmax_nan(size, sh_size[w]);
    const float t = key_score(lo), e2 = 2.f * (size * kScoreError + 1e-37f);
    sure = e2 <= 3e38f && t == t;
    if (sure) {
      khi = score_key(t + e2);
      klo = score_key(t - e2);
    }
    int2 cnt = make_int2(0, 0);
#pragma unroll 1
    for (int i = i0; i < i1; ++i) {
      const uint32_t x = key_of(i);
      cnt.x += sure && x > khi;
      cnt.y += open(x);
    }
    before = block_scan<NTH>(cnt, sums[1], &total);
    want = k - total.x;  // of the open pages
    opened = total.y;
    if (want == opened) break;
    few = opened <= kFew;
    // The open pages' 64-bit scores, a warp each.
    if (opened <= NTH) {
      int at = before.y;
#pragma unroll 1
      for (int i = i0; i < i1; ++i)
        if (open(key_of(i))) list[at++] = static_cast<uint32_t>(i);
    }
    __syncthreads();
    const int todo = opened <= NTH ? opened : m;
#pragma unroll 1
    for (int j = warp; j < todo; j += NTH / 32) {
      const int i = opened <= NTH ? static_cast<int>(list[j]) : j;
      if (opened > NTH && !open(key_of(i))) continue;
      const int64_t pid = static_cast<int64_t>(bt[(c0 + i) * p.bt_si]) * p.bt_mul +
                          static_cast<int64_t>(h) * p.bt_add;
      const float x = exact_score<T, D>(p, pid, q, qs);
      if (lane == 0) {
        if (few)
          list[kFew + j] = score_key(x);
        else
          __stcg(&sc[i].y, x);
      }
    }
    __syncthreads();
    if (few) break;
    exact = true;
    rank = want;
    lo = 0xffffffffu;
    hi = 0u;
    walk([&](uint32_t x) {
      lo = min(lo, x);
      hi = max(hi, x);
    });
  }
  // Pages above khi and, of the open ones: all; of a few, those with fewer than
  // `want` before them; of many, those above lo and the first `rank` equal to it.
  int at = before.x + before.y, ties = 0;
  if (few) {
    if (tid < opened) {
      const uint32_t x = list[kFew + tid];
      int ahead = 0;
      for (int i = 0; i < opened; ++i)
        ahead += list[kFew + i] > x || (list[kFew + i] == x && i < tid);
      hist[tid] = ahead < want;
    }
    __syncthreads();
    at = before.x;
    for (int i = 0; i < before.y; ++i) at += hist[i];
  } else if (exact) {
    int2 cnt = make_int2(0, 0);
    walk([&](uint32_t y) {
      cnt.x += y > lo;
      cnt.y += y == lo;
    });
    const int2 b = block_scan<NTH>(cnt, sums[2], &total);
    ties = rank - b.y;  // left for this thread's pages
    at = before.x + b.x + min(b.y, rank);
  }
  int j = before.y;
#pragma unroll 1
  for (int i = i0; i < i1; ++i) {
    const uint32_t x = key_of(i);
    bool take = sure && x > khi;
    if (open(x)) {
      take = true;
      if (few) {
        take = hist[j++] != 0;
      } else if (exact) {
        const uint32_t y = score_key(__ldcg(&sc[i].y));
        take = y > lo || (y == lo && ties-- > 0);
      }
    }
    // exactly k are taken; the bound keeps a unit inside its table all the same
    if (take && at < k) out[p.sink + at++] = bt[(c0 + i) * p.bt_si];
  }
}

}  // namespace pab

namespace {

using pabh::aligned;
using pabh::fail;

int check_head(int dtype, int D, int bs) {
  if (dtype != PAB200_DTYPE_BF16 && dtype != PAB200_DTYPE_F16)
    return fail(PAB200_ERR_UNSUPPORTED, "dtype %d: bf16 or f16", dtype);
  if (D != 64 && D != 128 && D != 256)
    return fail(PAB200_ERR_UNSUPPORTED, "head_size %d: supported 64, 128, 256", D);
  if (bs != 8 && bs != 16 && bs != 32 && bs != 64)
    return fail(PAB200_ERR_UNSUPPORTED, "block_size %d: supported 8, 16, 32, 64", bs);
  return PAB200_OK;
}

int check_select(const pab200_select_args* a) {
  if (!a) return fail(PAB200_ERR_INVALID_ARGUMENT, "args is null");
  int rc = check_head(a->dtype, a->head_size, a->block_size);
  if (rc) return rc;
  if (a->num_seqs < 1 || a->num_kv_heads < 1 || a->num_q_heads < 1 ||
      a->num_q_heads % a->num_kv_heads != 0)
    return fail(PAB200_ERR_INVALID_ARGUMENT,
                "num_seqs, num_q_heads, num_kv_heads must be >= 1, num_q_heads %% num_kv_heads == 0");
  if (a->max_blocks < 0 || a->num_pages < 0)
    return fail(PAB200_ERR_INVALID_ARGUMENT, "max_blocks and num_pages must be >= 0");
  if (a->num_sink < 0 || a->num_recent < 1 ||
      int64_t(a->num_sink) + a->num_recent > a->num_selected)
    return fail(PAB200_ERR_INVALID_ARGUMENT,
                "need num_sink >= 0, num_recent >= 1, num_sink + num_recent <= num_selected");
  const int64_t units = int64_t(a->num_seqs) * a->num_kv_heads;
  if (units > 65535 || int64_t(a->max_blocks) * a->block_size >= (int64_t(1) << 31) ||
      units * a->num_selected >= (int64_t(1) << 31) ||
      int64_t(a->num_selected) * a->block_size >= (int64_t(1) << 31))
    return fail(PAB200_ERR_UNSUPPORTED,
                "num_seqs*num_kv_heads above 65535, or max_blocks or num_selected too large");
  if (!a->q || !a->seqlens || !a->tables || !a->selected_lens)
    return fail(PAB200_ERR_INVALID_ARGUMENT, "q, seqlens, tables or selected_lens is null");
  if (a->max_blocks > 0 && a->num_pages > 0 && (!a->page_bounds || !a->block_table))
    return fail(PAB200_ERR_INVALID_ARGUMENT, "page_bounds or block_table is null");
  if (!aligned(a->page_bounds, 16) || !aligned(a->q, 2))
    return fail(PAB200_ERR_ALIGNMENT, "page_bounds must be 16-byte aligned");
  return PAB200_OK;
}

size_t scores_bytes(const pab200_select_args* a) {
  return pabh::align256(size_t(a->num_seqs) * a->num_kv_heads * (a->max_blocks > 0 ? a->max_blocks : 1) * 8);
}

template <typename T>
cudaError_t launch_scores(const pab::SelectParams& p, int D, const cudaLaunchConfig_t* cfg) {
  switch (D) {
    case 64: return cudaLaunchKernelEx(cfg, pab::page_scores_kernel<T, 64>, p);
    case 128: return cudaLaunchKernelEx(cfg, pab::page_scores_kernel<T, 128>, p);
    default: return cudaLaunchKernelEx(cfg, pab::page_scores_kernel<T, 256>, p);
  }
}

template <typename T, int D>
cudaError_t launch_selection_d(const pab::SelectParams& p, bool small, const cudaLaunchConfig_t* cfg) {
  return small ? cudaLaunchKernelEx(cfg, pab::select_pages_kernel<T, D, 256>, p)
               : cudaLaunchKernelEx(cfg, pab::select_pages_kernel<T, D, 1024>, p);
}

template <typename T>
cudaError_t launch_selection(const pab::SelectParams& p, int D, bool small,
                             const cudaLaunchConfig_t* cfg) {
  switch (D) {
    case 64: return launch_selection_d<T, 64>(p, small, cfg);
    case 128: return launch_selection_d<T, 128>(p, small, cfg);
    default: return launch_selection_d<T, 256>(p, small, cfg);
  }
}

// `chained`: between the planner and the decode grid of one call.
int launch_select(const pab200_select_args* a, void* scores, bool chained, cudaStream_t s) {
  pab::SelectParams p{};
  p.q = a->q;
  p.bounds = a->page_bounds;
  p.lens = a->seqlens;
  p.bt = a->block_table;
  p.tables = a->tables;
  p.out_lens = a->selected_lens;
  p.scores = static_cast<float2*>(scores);
  p.status = a->status;
  p.q_sb = a->q_stride_b;
  p.q_sh = a->q_stride_h;
  p.l_sb = a->seqlens_stride_b;
  p.l_sh = a->seqlens_stride_h;
  p.bt_sb = a->bt_stride_b;
  p.bt_sh = a->bt_stride_h;
  p.bt_si = a->bt_stride_i;
  p.num_pages = a->num_pages;
  p.bt_mul = a->bounds_page_mul;
  p.bt_add = a->bounds_page_add;
  p.B = a->num_seqs;
  p.Hkv = a->num_kv_heads;
  p.G = a->num_q_heads / a->num_kv_heads;
  p.bs = a->block_size;
  p.maxb = a->num_pages > 0 ? a->max_blocks : 0;
  p.keep = a->num_selected;
  p.sink = a->num_sink;
  p.recent = a->num_recent;
  p.chained = chained;
  const unsigned units = static_cast<unsigned>(p.B * p.Hkv);
  const bool scored = p.maxb > p.keep;
  if (scored) {
    // Pages per CTA: what gives every SM about four CTAs, in whole steps of the
    // 8 warps, at most 64 pages per warp.
    const int64_t pages = int64_t(units) * p.maxb;
    int64_t each = pages / (4 * pabh::device_sm_count_current());
    each = (each + 63) / 64 * 64;
    const int chunk = each < 64 ? 64 : (each > 512 ? 512 : static_cast<int>(each));
    p.chunk = chunk;
    const dim3 grid((p.maxb + chunk - 1) / chunk, units);
    pabh::LaunchCfg sc(grid, dim3(256), 0, s, chained);
    const cudaError_t e = a->dtype == PAB200_DTYPE_BF16
                              ? launch_scores<__nv_bfloat16>(p, a->head_size, &sc.cfg)
                              : launch_scores<__half>(p, a->head_size, &sc.cfg);
    if (e != cudaSuccess) return pabh::cuda_fail(e, "page scores launch");
  }
  // Scheduled while the scores drain; waits for them before it reads any.
  // 256 threads while shared memory holds all of their keys (8 per thread), so that
  // several units share an SM.
  const bool small = p.maxb <= 2048;
  pabh::LaunchCfg lc(dim3(units), dim3(small ? 256 : 1024), 0, s, scored || chained);
  const cudaError_t err = a->dtype == PAB200_DTYPE_BF16
                              ? launch_selection<__nv_bfloat16>(p, a->head_size, small, &lc.cfg)
                              : launch_selection<__half>(p, a->head_size, small, &lc.cfg);
  if (err != cudaSuccess) return pabh::cuda_fail(err, "page selection launch");
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? PAB200_OK : pabh::cuda_fail(e, "page selection launch");
}

// The decode over the selected tables.
pab200_decode_args selected_decode(const pab200_decode_args* a, const pab200_select_args* sel) {
  pab200_decode_args d = *a;
  d.seqlens = sel->selected_lens;
  d.block_table = sel->tables;
  d.max_blocks = sel->num_selected;
  d.seqlens_stride_b = sel->num_kv_heads;
  d.seqlens_stride_h = 1;
  d.bt_stride_b = int64_t(sel->num_kv_heads) * sel->num_selected;
  d.bt_stride_h = sel->num_selected;
  d.bt_stride_i = 1;
  return d;
}

int check_sparse(const pab200_decode_args* a, const pab200_select_args* sel) {
  if (!a) return fail(PAB200_ERR_INVALID_ARGUMENT, "args is null");
  const int rc = check_select(sel);
  if (rc) return rc;
  if (a->q != sel->q || a->dtype != sel->dtype || a->num_seqs != sel->num_seqs ||
      a->num_q_heads != sel->num_q_heads || a->num_kv_heads != sel->num_kv_heads ||
      a->head_size != sel->head_size || a->block_size != sel->block_size ||
      a->q_stride_b != sel->q_stride_b || a->q_stride_h != sel->q_stride_h)
    return fail(PAB200_ERR_INVALID_ARGUMENT,
                "the selection and the decode must have the same query and sizes");
  return PAB200_OK;
}

}  // namespace

PAB200_EXPORT size_t pab200_select_pages_workspace_size(const pab200_select_args* a) {
  return check_select(a) ? 0 : scores_bytes(a);
}

PAB200_EXPORT int pab200_select_pages(const pab200_select_args* a, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  const int rc = check_select(a);
  if (rc) return rc;
  if (!workspace || workspace_bytes < scores_bytes(a))
    return fail(PAB200_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", scores_bytes(a),
                workspace ? workspace_bytes : size_t(0));
  if (!aligned(workspace, 256)) return fail(PAB200_ERR_ALIGNMENT, "workspace must be 256-byte aligned");
  return launch_select(a, workspace, false, static_cast<cudaStream_t>(stream));
}

PAB200_EXPORT size_t pab200_decode_sparse_workspace_size(const pab200_decode_args* a,
                                                         const pab200_select_args* sel) {
  if (check_sparse(a, sel)) return 0;
  const pab200_decode_args d = selected_decode(a, sel);
  const size_t need = pab200_decode_workspace_size(&d);
  return need == 0 ? 0 : pabh::align256(need) + scores_bytes(sel);
}

PAB200_EXPORT int pab200_decode_sparse(const pab200_decode_args* a, const pab200_select_args* sel,
                                       void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_sparse(a, sel);
  if (rc) return rc;
  const pab200_decode_args d = selected_decode(a, sel);
  const size_t need = pab200_decode_workspace_size(&d);
  if (need == 0) return fail(PAB200_ERR_INVALID_ARGUMENT, "%s", pab200_last_error());
  const size_t at = pabh::align256(need), all = at + scores_bytes(sel);
  if (!workspace || workspace_bytes < all)
    return fail(PAB200_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", all,
                workspace ? workspace_bytes : size_t(0));
  if (!aligned(workspace, 256)) return fail(PAB200_ERR_ALIGNMENT, "workspace must be 256-byte aligned");
  struct What {
    const pab200_select_args* sel;
    void* scores;
  };
  const What what{sel, static_cast<uint8_t*>(workspace) + at};
  pabh::Selection in{};
  in.lens = sel->seqlens;
  in.l_sb = sel->seqlens_stride_b;
  in.l_sh = sel->seqlens_stride_h;
  in.max_blocks = sel->num_pages > 0 ? sel->max_blocks : 0;
  in.launch = [](const void* w, cudaStream_t s) {
    const What* x = static_cast<const What*>(w);
    return launch_select(x->sel, x->scores, true, s);
  };
  in.what = &what;
  return pabh::decode_selected(&d, in, workspace, need, stream);
}

namespace {

template <typename T>
void launch_bounds(const pab::BoundsParams& p, int D, int warps, cudaStream_t s) {
  const int grid = (warps + 7) / 8;
  switch (D) {
    case 64: pab::page_bounds_kernel<T, 64><<<grid, 256, 0, s>>>(p, warps); break;
    case 128: pab::page_bounds_kernel<T, 128><<<grid, 256, 0, s>>>(p, warps); break;
    default: pab::page_bounds_kernel<T, 256><<<grid, 256, 0, s>>>(p, warps); break;
  }
}

}  // namespace

PAB200_EXPORT int pab200_update_page_bounds(const pab200_page_bounds_args* a, void* stream) {
  if (!a) return fail(PAB200_ERR_INVALID_ARGUMENT, "args is null");
  int rc = check_head(a->dtype, a->head_size, a->block_size);
  if (rc) return rc;
  if (a->num_seqs < 0 || a->num_kv_heads < 1 || a->max_blocks < 0 || a->num_pages < 0 ||
      a->num_tokens < 0)
    return fail(PAB200_ERR_INVALID_ARGUMENT,
                "need num_seqs, max_blocks, num_pages, num_tokens >= 0, num_kv_heads >= 1");
  if (!a->cu_tokens && a->num_tokens != a->num_seqs)
    return fail(PAB200_ERR_INVALID_ARGUMENT,
                "without cu_tokens there is one token per sequence: num_tokens %lld, num_seqs %d",
                static_cast<long long>(a->num_tokens), a->num_seqs);
  const int bs = a->block_size, log2_bs = bs == 8 ? 3 : (bs == 16 ? 4 : (bs == 32 ? 5 : 6));
  const int64_t warps =
      pab::num_slots(a->num_tokens, a->num_seqs, a->cu_tokens != nullptr, log2_bs) * a->num_kv_heads;
  if (int64_t(a->max_blocks) * bs >= (int64_t(1) << 31) || a->num_tokens >= (int64_t(1) << 30) ||
      warps >= (int64_t(1) << 31) - 8)
    return fail(PAB200_ERR_UNSUPPORTED, "max_blocks*block_size or num_tokens too large (>= 2^31)");
  if (a->num_seqs == 0 || a->num_tokens == 0) return PAB200_OK;
  if (!a->k_rows || !a->seqlens) return fail(PAB200_ERR_INVALID_ARGUMENT, "k_rows or seqlens is null");
  if (a->max_blocks > 0 && a->num_pages > 0 && (!a->page_bounds || !a->block_table))
    return fail(PAB200_ERR_INVALID_ARGUMENT, "page_bounds or block_table is null");
  if (!aligned(a->page_bounds, 16) || !aligned(a->k_rows, 2))
    return fail(PAB200_ERR_ALIGNMENT, "page_bounds must be 16-byte aligned");
  pab::BoundsParams p{};
  p.map.bt = a->block_table;
  p.map.cu = a->cu_tokens;
  p.map.bt_sb = a->bt_stride_b;
  p.map.bt_sh = a->bt_stride_h;
  p.map.bt_si = a->bt_stride_i;
  p.map.l_sb = a->seqlens_stride_b;
  p.map.l_sh = a->seqlens_stride_h;
  p.map.num_pages = a->num_pages;
  p.map.num_tokens = static_cast<int32_t>(a->num_tokens);
  p.map.bt_mul = a->bounds_page_mul;
  p.map.bt_add = a->bounds_page_add;
  p.map.B = a->num_seqs;
  p.map.Hkv = a->num_kv_heads;
  p.map.bs = bs;
  p.map.log2_bs = log2_bs;
  p.map.maxb = a->num_pages > 0 ? a->max_blocks : 0;
  p.bounds = a->page_bounds;
  p.rows = a->k_rows;
  p.lens = a->seqlens;
  p.status = a->status;
  p.r_st = a->row_stride_t;
  p.r_sh = a->row_stride_h;
  p.vec = aligned(a->k_rows, 16) && a->row_stride_t % 8 == 0 && a->row_stride_h % 8 == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->dtype == PAB200_DTYPE_BF16)
    launch_bounds<__nv_bfloat16>(p, a->head_size, static_cast<int>(warps), s);
  else
    launch_bounds<__half>(p, a->head_size, static_cast<int>(warps), s);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? PAB200_OK : pabh::cuda_fail(e, "page bounds launch");
}
