// Page-sparse decode: key bounds of pages, selection of pages by a query, and
// the decode over the selected pages.
#include "host.h"
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
// it began before.  Comparisons work on the 16-bit pairs as they are.
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

struct SelectParams {
  const void* q;
  const void* bounds;
  const int32_t* lens;
  const int32_t* bt;
  int32_t* tables;     // [B][Hkv][keep]
  int32_t* out_lens;   // [B][Hkv]
  float* scores;       // [B * Hkv][maxb]
  uint32_t* status;
  int64_t q_sb, q_sh, l_sb, l_sh, bt_sb, bt_sh, bt_si, num_pages;
  int32_t bt_mul, bt_add, B, Hkv, G, bs, maxb, keep, sink, recent;
};

__device__ __forceinline__ int clamped_length(const SelectParams& p, int s, int h) {
  const int L = p.lens[s * p.l_sb + h * p.l_sh];
  const int64_t cap = static_cast<int64_t>(p.maxb) * p.bs;
  return L < 0 ? 0 : (L > cap ? static_cast<int>(cap) : L);
}

// Score of every candidate page of a (sequence, kv head): sum over the head
// elements of max * (sum of the group's positive query parts) + min * (sum of
// the negative ones), the upper bound of the group's summed scores.  Summed in
// 64 bits and rounded once, so that the order of the sum cannot change which
// pages rank next to the border.
template <typename T, int D>
__global__ void __launch_bounds__(256) page_scores_kernel(const SelectParams p) {
  constexpr int LP = D / 8, PW = 32 / LP;  // lanes per page, pages per warp step
  __shared__ double qs[2][D];
  const int u = blockIdx.y, s = u / p.Hkv, h = u - s * p.Hkv;
  const int L = clamped_length(p, s, h);
  const int n = (L + p.bs - 1) / p.bs;
  if (n <= p.keep) return;
  const T* q = static_cast<const T*>(p.q) + s * p.q_sb + static_cast<int64_t>(h) * p.G * p.q_sh;
  for (int d = threadIdx.x; d < D; d += 256) {
    double up = 0.0, dn = 0.0;
    for (int g = 0; g < p.G; ++g) {
      const double x = static_cast<double>(static_cast<float>(q[g * p.q_sh + d]));
      up += x > 0.0 ? x : 0.0;
      dn += x < 0.0 ? x : (x > 0.0 ? 0.0 : x);
    }
    qs[0][d] = up;
    qs[1][d] = dn;
  }
  __syncthreads();
  const int lane = threadIdx.x & 31, e = lane % LP;
  double up[8], dn[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    up[i] = qs[0][e * 8 + i];
    dn[i] = qs[1][e * 8 + i];
  }
  const int warps = gridDim.x * 8;
  uint32_t flags = 0;
  const int c1 = n - p.recent;
  for (int c0 = p.sink + (blockIdx.x * 8 + (threadIdx.x >> 5)) * PW; c0 < c1; c0 += warps * PW) {
    const int c = c0 + lane / LP;
    double sum = 0.0;
    bool bad = false;
    if (c < c1) {
      const int64_t pid = static_cast<int64_t>(p.bt[s * p.bt_sb + h * p.bt_sh + c * p.bt_si]) * p.bt_mul +
                          static_cast<int64_t>(h) * p.bt_add;
      bad = pid < 0 || pid >= p.num_pages;
      if (!bad) {
        const T* b = static_cast<const T*>(p.bounds) + pid * (2 * D) + e * 8;
        float mn[8], mx[8];
        unpack8<T>(__ldg(reinterpret_cast<const uint4*>(b)), mn);
        unpack8<T>(__ldg(reinterpret_cast<const uint4*>(b + D)), mx);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          sum = fma(static_cast<double>(mx[i]), up[i], fma(static_cast<double>(mn[i]), dn[i], sum));
      }
    }
#pragma unroll
    for (int o = 1; o < LP; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (bad) flags |= kStatusBadPage;
    if (e == 0 && c < c1) p.scores[static_cast<int64_t>(u) * p.maxb + c] = bad ? -INFINITY : static_cast<float>(sum);
  }
  if (flags && p.status) atomicOr(p.status, flags);
}

// Order-preserving key of a score: larger scores have larger keys, -0 and +0
// the same, NaN the largest.
__device__ __forceinline__ uint32_t score_key(float f) {
  if (f != f) return 0xffffffffu;
  const uint32_t b = __float_as_uint(f + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Sum of x over the block's threads before this one, and the total.
__device__ __forceinline__ int block_scan(int x, int* warp_sum, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int v = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  __syncthreads();
  if (lane == 31) warp_sum[warp] = v;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) {
    if (w < warp) before += warp_sum[w];
    all += warp_sum[w];
  }
  *total = all;
  return before + v - x;
}

// One CTA per (sequence, kv head): the pages to attend to, ascending.  Radix
// selection of the k-th largest key, 8 bits a pass; the pages above it, and
// the first of those equal to it, are kept.
__global__ void __launch_bounds__(1024) select_pages_kernel(const SelectParams p) {
  __shared__ int hist[256];
  __shared__ int warp_sum[32];
  __shared__ uint32_t sh_prefix;
  __shared__ int sh_rank;
  const int u = blockIdx.x, s = u / p.Hkv, h = u - s * p.Hkv;
  const int tid = threadIdx.x;
  const int L = clamped_length(p, s, h);
  const int raw = p.lens[s * p.l_sb + h * p.l_sh];
  if (tid == 0 && raw != L && p.status) atomicOr(p.status, raw < 0 ? kStatusNegative : kStatusClamp);
  const int n = (L + p.bs - 1) / p.bs;
  const int32_t* bt = p.bt + s * p.bt_sb + h * p.bt_sh;
  int32_t* out = p.tables + static_cast<int64_t>(u) * p.keep;
  if (n <= p.keep) {
    for (int i = tid; i < p.keep; i += 1024) out[i] = i < n ? bt[i * p.bt_si] : -1;
    if (tid == 0) p.out_lens[u] = L;
    return;
  }
  const float* sc = p.scores + static_cast<int64_t>(u) * p.maxb;
  const int c0 = p.sink, c1 = n - p.recent;
  const int k = p.keep - p.sink - p.recent;  // candidates kept
  uint32_t prefix = 0;
  int rank = k;  // the rank-th largest key is looked for among keys that begin with prefix
  if (k > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int c = c0 + tid; c < c1; c += 1024) {
        const uint32_t key = score_key(sc[c]);
        if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8)))
          atomicAdd(&hist[(key >> shift) & 255u], 1);
      }
      __syncthreads();
      if (tid < 32) {  // bins from the top: lane l holds bins 255 - 8 l .. 248 - 8 l
        int sum = 0;
        for (int i = 0; i < 8; ++i) sum += hist[255 - (tid * 8 + i)];
        int v = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, v, o);
          if (tid >= o) v += y;
        }
        int before = v - sum;
        if (before < rank && rank <= v) {
          for (int i = 0; i < 8; ++i) {
            const int bin = 255 - (tid * 8 + i);
            if (rank <= before + hist[bin]) {
              sh_prefix = prefix | static_cast<uint32_t>(bin) << shift;
              sh_rank = rank - before;
              break;
            }
            before += hist[bin];
          }
        }
      }
      __syncthreads();
      prefix = sh_prefix;
      rank = sh_rank;
      __syncthreads();
    }
  }
  // Keys above `prefix` are kept, of the equal ones the first `rank`.
  int kept = 0, equal = 0;
  for (int b0 = c0; b0 < c1 && k > 0; b0 += 1024) {
    const int c = b0 + tid;
    const uint32_t key = c < c1 ? score_key(sc[c]) : 0u;
    const bool eq = c < c1 && key == prefix;
    int total;
    const int eq_before = equal + block_scan(eq, warp_sum, &total);
    equal += total;
    const bool take = c < c1 && (key > prefix || (eq && eq_before < rank));
    const int at = kept + block_scan(take, warp_sum, &total);
    kept += total;
    if (take) out[p.sink + at] = bt[c * p.bt_si];
  }
  for (int i = tid; i < p.sink; i += 1024) out[i] = bt[i * p.bt_si];
  for (int i = tid; i < p.recent; i += 1024) out[p.keep - p.recent + i] = bt[(c1 + i) * p.bt_si];
  if (tid == 0) p.out_lens[u] = (p.keep - 1) * p.bs + L - (n - 1) * p.bs;
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
  return pabh::align256(size_t(a->num_seqs) * a->num_kv_heads * (a->max_blocks > 0 ? a->max_blocks : 1) * 4);
}

template <typename T>
void launch_scores(const pab::SelectParams& p, int D, dim3 grid, cudaStream_t s) {
  switch (D) {
    case 64: pab::page_scores_kernel<T, 64><<<grid, 256, 0, s>>>(p); break;
    case 128: pab::page_scores_kernel<T, 128><<<grid, 256, 0, s>>>(p); break;
    default: pab::page_scores_kernel<T, 256><<<grid, 256, 0, s>>>(p); break;
  }
}

int launch_select(const pab200_select_args* a, void* scores, cudaStream_t s) {
  pab::SelectParams p{};
  p.q = a->q;
  p.bounds = a->page_bounds;
  p.lens = a->seqlens;
  p.bt = a->block_table;
  p.tables = a->tables;
  p.out_lens = a->selected_lens;
  p.scores = static_cast<float*>(scores);
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
  const unsigned units = static_cast<unsigned>(p.B * p.Hkv);
  if (p.maxb > p.keep) {
    const int per_cta = 8 * 32 / (a->head_size / 8) * 4;
    unsigned chunks = static_cast<unsigned>((p.maxb + per_cta - 1) / per_cta);
    const unsigned most = (8u * pabh::device_sm_count_current() + units - 1) / units;
    if (chunks > most) chunks = most;
    if (a->dtype == PAB200_DTYPE_BF16)
      launch_scores<__nv_bfloat16>(p, a->head_size, dim3(chunks, units), s);
    else
      launch_scores<__half>(p, a->head_size, dim3(chunks, units), s);
  }
  pab::select_pages_kernel<<<units, 1024, 0, s>>>(p);
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
  return launch_select(a, workspace, static_cast<cudaStream_t>(stream));
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
  rc = launch_select(sel, static_cast<uint8_t*>(workspace) + at, static_cast<cudaStream_t>(stream));
  if (rc) return rc;
  return pabh::decode_after(&d, workspace, need, stream);
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
