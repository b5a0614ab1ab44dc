// Decode attention over 4-bit pages (int4.cuh).
//
//   score_t = scale * sum_g [ s_tg (q_g . c_tg) + lo_tg sum(q_g) ]
//   out_d   = sum_t p_t [ (lo_tg + 8 s_tg) + s_tg (c_td - 8) ] / sum_t p_t
//
// A quarter of the bytes of 16-bit pages but the same products, and codes to
// widen before the matrix instructions can take them: instruction issue bounds
// the kernel, not HBM, so everything is laid out for few instructions per code.
//   * One producer warp per CTA walks the CTA's page range (the planner's equal
//     cut of all pages), reads the block table one stage ahead and fills a ring of
//     128-token stages: four pages of a cache per copy (rows gathered through a
//     tensor map, pages up to 2 KB), or one untiled bulk copy per page.  Four
//     consumer warps share every stage, 32 tokens each (groups of more than 16
//     heads: two pairs, each warp 16 heads and 64 tokens), and do nothing but
//     arithmetic.
//   * Keys enter the MMA as fp16 subnormals, the nibbles as they stand (one
//     mask per pair); the query is brought to fp16 by a power of two per head,
//     which loses nothing of a bf16 or fp16 query that matters, and the score is
//     scaled back in fp32.
//   * Scales and minima never touch the codes: the keys' multiply the partial
//     scores of their group, the values' scale multiplies the probability, which
//     is rounded to fp16 once, and the rest of the value is summed apart in fp32.
//     The scales carry a power of two that follows the largest scale seen, so that
//     the fp16 product keeps its bits for small values and unlikely tokens, and
//     stays in range for bf16's scales (products of probability and scale more than
//     2^24 below the largest scale lose bits).
//     How the values' codes enter depends on T.
//     fp16: as c - 8, so that the rounding of p s is multiplied by s (c - 8), about
//     |x|, not by s c, about the group's range: the output keeps fp16's 11 bits.
//     bf16: as they stand, like the keys': an fp16 p s is eight times finer than
//     the bf16 output needs, and than a bf16 p s (error against 64 bits 0.0017,
//     0.0023 with bf16 c - 8; 4 contexts of 32768 to 131072 tokens 3 us less of 111).
//     Since sums of codes >= 0 only grow, and the tensor cores cut their fp32 sums
//     short, the accumulators are emptied into shared memory every kFlush chunks of
//     32 tokens.
//   * The softmax's reference point moves only when a score exceeds it by
//     kRaise (log2 units): no shuffles or rescaling in most stages.
// At the end of a head (or of the CTA's part of it) the consumers' states are
// joined through shared memory and written: the output, or one partial state
// for the reduce kernels of decode.cuh.
//
// Measured (bf16, 8 kv heads of 4 query heads, D 128, pages of 16): 64 sequences
// of 4096 tokens (303 MB) 75.5 us, 4.0 TB/s of the 6.55 a copy reaches (pages of 32
// and 64, which take bulk copies: 75.8 and 74.6).  About 600 warp instructions per 32
// tokens and head keep the issue slots a good half and the ALU pipe 55 to 60 % busy;
// the copies alone take 59 us, the arithmetic alone about 70.  The pairs of
// int4_value_pairs cost 4 instructions instead of 5: 76.3 -> 74.8.  Without a producing warp (the last warp of a stage refills its slot)
// 15 us more, with 4 CTAs per SM at 96 registers (which spill) 12 more.  Handing
// CTAs that end early the last chunks of others, as decode.cuh does, costs one more
// join per chunk and instructions that the producer has to fetch: 5 us with that
// code in place but unused, 6 to 13 with 1 to 4 chunks.  One copy of the emptying
// and of the join in the loop instead of two: 77.3 -> 76.1.
#pragma once

#include <type_traits>

#include "decode.cuh"
#include "int4.cuh"

namespace pab {

constexpr int kQ4Consumers = 4;                       // consumer warps per CTA
constexpr int kQ4Threads = (kQ4Consumers + 1) * 32;
constexpr int kQ4Stage = 128;                         // tokens per ring stage
constexpr int kQ4MaxDepth = 4;
constexpr int kQ4NoHead = 1 << 27;                    // in a stage record: no next head
constexpr int kQ4Early = 1024;                        // heads whose prefix a CTA keeps itself

// Shared memory: ring, then joining buffer, then barriers, records, prefix.
__host__ __device__ constexpr int q4_stage_bytes(int D) { return 2 * kQ4Stage * int4_row_bytes(D); }
__host__ __device__ constexpr int q4_join_floats(int D, int G, int parts) {
  return parts * G * (D + 4) + ((parts * G * 2 + 3) & ~3);
}
__host__ __device__ constexpr size_t q4_smem(int D, int G, int parts, int depth) {
  return 128 + size_t(depth) * q4_stage_bytes(D) + size_t(q4_join_floats(D, G, parts)) * 4 +
         kQ4MaxDepth * (16 + 16) + 16 + (2 * kQ4Early + 1 + 32) * 4;
}

template <typename T, int D, int NT, int HS, int MINB>
__global__ void __launch_bounds__(kQ4Threads, MINB)
    decode_int4_kernel(const __grid_constant__ CUtensorMap kmap,
                       const __grid_constant__ CUtensorMap vmap,
                       const __grid_constant__ DecodeParams p) {
  constexpr int NG = D / kInt4Group;           // quantisation groups per row
  constexpr int KS = D / 16;                   // k-steps of the scores, d-tiles of the output
  constexpr int PARTS = kQ4Consumers / HS;     // token parts of a stage
  constexpr int PT = kQ4Stage / PARTS;         // tokens per part, in chunks of 32
  constexpr int MT = 2;                        // 16-token tiles per chunk
  constexpr int STAGE_BYTES = q4_stage_bytes(D), KV_BYTES = STAGE_BYTES / 2;
  // Probability x scale must stay below 65504, a probability stays below
  // 2^kRaise = 7.46, and scales are brought to 2^13 at most (fp16's largest, 2 *
  // 65504 / 15, stay as they are).
  constexpr bool kHalf = std::is_same<T, __half>::value;
  constexpr float kRaise = 2.9f;
  constexpr int kFlush = 32;  // bf16: chunks between two emptyings of the accumulators
  // Reference point of an empty state: below every score, and finite, so that
  // a score of -inf has probability 0.
  constexpr float kNoScore = -3e38f;
  constexpr float kFar = 9.094947017729282e-13f;  // 2^-40

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_addr(smem_raw);
  const uint32_t base = (raw_addr + 127u) & ~127u;
  uint8_t* const smem = smem_raw + (base - raw_addr);
  const int depth = p.depth, G = p.G, Hkv = p.Hkv, bs = p.bs;
  float* const join = reinterpret_cast<float*>(smem + depth * STAGE_BYTES);
  float* const join_ml = join + PARTS * G * (D + 4);
  uint8_t* const tail = reinterpret_cast<uint8_t*>(join + q4_join_floats(D, G, PARTS));
  const uint32_t full = smem_addr(tail), empty = full + kQ4MaxDepth * 8;
  int4* const record = reinterpret_cast<int4*>(tail + kQ4MaxDepth * 16);
  // consumers' own barriers: states deposited, states read
  const uint32_t joined = full + kQ4MaxDepth * 32, drained = joined + 8;
  int* const cum_sm = reinterpret_cast<int*>(tail + kQ4MaxDepth * 32 + 16);
  int* const len_sm = cum_sm + kQ4Early + 1;
  int* const wsum = len_sm + kQ4Early;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n_heads = p.B * Hkv, cap = p.maxb * bs;
  const int log2_bs = __ffs(bs) - 1;
  auto head_len = [&](int hd) {
    const int s = hd / Hkv, h = hd - s * Hkv;
    const int L = p.lens[s * p.l_sb + h * p.l_sh];
    return L < 0 ? 0 : (L > cap ? cap : L);
  };
  grid_launch_dependents();
  if (tid == 0) {
    for (int i = 0; i < depth; ++i) {
      mbar_init(full + i * 8, 1);
      mbar_init(empty + i * 8, kQ4Consumers);
    }
    mbar_init(joined, kQ4Consumers);
    mbar_init(drained, kQ4Consumers);
    fence_mbar_init();
    if (p.gather) {
      tma_prefetch_desc(&kmap);
      tma_prefetch_desc(&vmap);
    }
  }
  // The page-count prefix of all heads, computed by this CTA like the planner
  // computes it for the reduce kernel (up to kQ4Early heads; more: the
  // planner's).  The host launches the planner without programmatic
  // dependence, so the lengths are final here.
  const bool early = p.early != 0;
  int total;
  if (early) {
    const int per = (n_heads + kQ4Threads - 1) / kQ4Threads;
    const int h0 = min(tid * per, n_heads), h1 = min(h0 + per, n_heads);
    int sum = 0, s = h0 / Hkv, h = h0 - s * Hkv;
#pragma unroll 1
    for (int hd = h0; hd < h1; ++hd) {
      int L = p.lens[s * p.l_sb + h * p.l_sh];
      L = L < 0 ? 0 : (L > cap ? cap : L);
      len_sm[hd] = L;
      sum += (L + bs - 1) >> log2_bs;
      if (++h == Hkv) {
        h = 0;
        ++s;
      }
    }
    int x = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) wsum[warp] = x;
    __syncthreads();
    int run = x - sum;
    for (int w = 0; w < warp; ++w) run += wsum[w];
#pragma unroll 1
    for (int hd = h0; hd < h1; ++hd) {
      cum_sm[hd] = run;
      run += (len_sm[hd] + bs - 1) >> log2_bs;
    }
    if (tid == kQ4Threads - 1) cum_sm[n_heads] = run;
    __syncthreads();
    total = cum_sm[n_heads];
  } else {
    grid_dependency_wait();
    total = p.cum[n_heads];
    __syncthreads();
  }
  const int64_t units = (static_cast<int64_t>(total) + p.unit_pages - 1) / p.unit_pages;
  const int W = static_cast<int>(units < p.total_warps ? units : p.total_warps);
  const int u = blockIdx.x;
  const int gs = u < W ? static_cast<int>(static_cast<int64_t>(u) * total / W) : 0;
  const int ge = u < W ? static_cast<int>(static_cast<int64_t>(u + 1) * total / W) : 0;

  if (warp == kQ4Consumers) {
    // ------------------------------------------------------------ producer
    const int log2_pps = 7 - log2_bs, pps = 1 << log2_pps;  // pages per stage (2..16)
    const int pb = int4_row_bytes(D) << log2_bs;
    const uint64_t policy = l2_policy_evict_first();
    auto prefix = [&](int hd) { return early ? cum_sm[hd] : p.cum[hd]; };
    bool bad_seen = false, timeout = false;
    int issued = 0, slot = 0;
    uint32_t phase = 1;  // of `empty`: the first round finds every slot free
    // Largest head whose first page is <= P.
    auto find_head = [&](int P) -> int {
      int lo = 0, hi = n_heads;
      while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32;
        const int x = lo + lane * step;
        const unsigned mask = __ballot_sync(0xffffffffu, x < hi && prefix(x) <= P);
        lo += (31 - __clz(mask)) * step;
        hi = lo + step < hi ? lo + step : hi;
      }
      return lo;
    };
    if (gs < ge) {
      int head = find_head(gs);
      int c_lo = prefix(head), c_hi = prefix(head + 1), gp = gs;
      int nx_head = 0, nx_np = 0, nx_tok = 0, nx_flags = 0, nx_raw = 0;
      int64_t nx_add = 0;
      const int32_t* c_bt = p.bt;
      int c_h = 0, c_len = 0;
      auto enter_head = [&]() {
        const int s = head / Hkv;
        c_h = head - s * Hkv;
        c_bt = p.bt + s * p.bt_sb + c_h * p.bt_sh;
        c_len = early ? len_sm[head] : head_len(head);
      };
      enter_head();
      // The next stage, its block-table entries on their way.
      auto prepare = [&]() -> bool {
        if (gp >= ge) return false;
        if (gp >= c_hi) {
          do {
            ++head;
            c_lo = c_hi;
            c_hi = prefix(head + 1);
          } while (gp >= c_hi);
          enter_head();
        }
        const int lp = gp - c_lo;
        int np = pps;
        if (c_hi - gp < np) np = c_hi - gp;
        if (ge - gp < np) np = ge - gp;
        nx_head = head;
        nx_np = np;
        const int left = c_len - (lp << log2_bs);
        nx_tok = left < np << log2_bs ? left : np << log2_bs;
        // 1: the head's first stage in the range, 2: its last, 4: the whole head
        // is in the range
        nx_flags = (gp == c_lo || gp == gs ? 1 : 0) |
                   (gp + np == c_hi || gp + np == ge ? 2 : 0) |
                   (c_lo >= gs && c_hi <= ge ? 4 : 0);
        nx_add = static_cast<int64_t>(c_h) * p.bt_add;
        if (lane < np) nx_raw = c_bt[static_cast<int64_t>(lp + lane) * p.bt_si];
        gp += np;
        return true;
      };
      // Rows per gathering copy: four pages of one cache.
      const int quads = pps >> 2;
      bool more = prepare();
      while (more) {
        const int np = nx_np;
        int4 rec = make_int4(nx_head, nx_tok, nx_flags, 0);
        const int64_t pid = static_cast<int64_t>(nx_raw) * p.bt_mul + nx_add;
        const bool ok = lane < np && pid >= 0 && pid < p.num_pages;
        const uint32_t bad = __ballot_sync(0xffffffffu, lane < np && !ok);
        bad_seen |= bad != 0;
        more = prepare();
        // the next stage's head, while it fits beside the flags
        rec.z |= (more && nx_head < kQ4NoHead ? nx_head : kQ4NoHead) << 3;
        if (!__all_sync(0xffffffffu, mbar_wait(empty + slot * 8, phase, kWaitLimitNs))) {
          timeout = true;
          break;
        }
        const uint32_t st = base + slot * STAGE_BYTES, bar = full + slot * 8;
        if (p.gather) {
          // Pages that are not there (past np, or rejected) read as zeros.
          const int row = ok ? static_cast<int>(pid) : static_cast<int>(p.num_pages);
          const int quad = lane & 3, kv = lane >> 2;
          int32_t r[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) r[i] = __shfl_sync(0xffffffffu, row, quad * 4 + i);
          if (lane == 0) {
            record[slot] = rec;
            mbar_arrive_expect_tx(bar, static_cast<uint32_t>(2 * pb * ((np + 3) & ~3)));
          }
          __syncwarp();
          if (kv < 2 && quad < quads && quad * 4 < np)
            tma_gather4(st + kv * KV_BYTES + quad * 4 * pb, kv ? &vmap : &kmap, 0, r, bar, policy);
        } else {
          if (bad) {
            // A rejected page id has no copy: zeros (codes, scales and minima)
            // stand in, written before the arrival that publishes the stage.
            uint8_t* const sp = smem + slot * STAGE_BYTES;
            for (int g = 0; g < np; ++g) {
              if (!(bad >> g & 1u)) continue;
              for (int i = lane; i < pb / 8; i += 32) {
                const int half = pb / 16;
                uint4* z = reinterpret_cast<uint4*>(sp + (i < half ? 0 : KV_BYTES) + g * pb);
                z[i < half ? i : i - half] = make_uint4(0u, 0u, 0u, 0u);
              }
            }
            fence_proxy_async_smem();  // before the copies that refill this slot later
            __syncwarp();
          }
          if (lane == 0) {
            record[slot] = rec;
            mbar_arrive_expect_tx(bar, static_cast<uint32_t>(2 * pb * (np - __popc(bad))));
          }
          __syncwarp();
          const int pg = lane & 15, kv = lane >> 4;
          const int64_t src = __shfl_sync(0xffffffffu, pid, pg);
          if (pg < np && !(bad >> pg & 1u))
            bulk_load(st + kv * KV_BYTES + pg * pb, (kv ? p.v_pages : p.k_pages) + src * pb,
                      static_cast<uint32_t>(pb), bar, policy);
        }
        ++issued;
        if (++slot == depth) {
          slot = 0;
          phase ^= 1;
        }
      }
    }
    // The end record, in a free slot.
    bool ended = false;
    if (!timeout) {
      if (!__all_sync(0xffffffffu, mbar_wait(empty + slot * 8, phase, kWaitLimitNs))) {
        timeout = true;
      } else {
        ended = true;
        if (lane == 0) {
          record[slot] = make_int4(-1, 0, 0, 0);
          mbar_arrive(full + slot * 8);
        }
      }
    }
    // No copy of this CTA is in flight when it ends, whatever the consumers
    // did (the end record's slot was waited for above).
    for (int j = max(issued - depth + (ended ? 1 : 0), 0); j < issued; ++j)
      mbar_wait(full + (j % depth) * 8, (j / depth) & 1, kWaitLimitNs);
    grid_dependency_wait();  // the planner has reset the status word
    if (lane == 0 && (bad_seen || timeout))
      atomicOr(p.status, (bad_seen ? kStatusBadPage : 0u) | (timeout ? kStatusTimeout : 0u));
    return;
  }

  // ------------------------------------------------------------- consumers
  // Heads of length 0 get zeros (an empty state in state mode).
  for (int hd = u * kQ4Consumers + warp; hd < n_heads; hd += gridDim.x * kQ4Consumers) {
    if ((early ? len_sm[hd] : head_len(hd)) != 0) continue;
    const int s = hd / Hkv, h = hd - s * Hkv;
    for (int g = 0; g < G; ++g) {
      const int64_t row = static_cast<int64_t>(s) * Hkv * G + h * G + g;
      for (int c = lane * 4; c < D; c += 128) {
        if (p.state_o)
          *reinterpret_cast<float4*>(p.state_o + row * D + c) = make_float4(0.f, 0.f, 0.f, 0.f);
        else
          *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + s * p.o_sb + (h * G + g) * p.o_sh + c) =
              make_uint2(0u, 0u);
      }
      if (p.state_o && lane == 0) p.state_lse[row] = -INFINITY;
    }
  }
  const int lr = lane >> 2, lc = lane & 3;
  const int part = warp / HS, g_lo = (warp % HS) * NT * 8;
  const int tok0 = part * PT;                  // this warp's first token of a stage
  // Byte offsets of an 8-token tile's codes and (scale, minimum) pairs from the
  // part's first: a page holds whole tiles, and a part begins with a page or
  // with half of one.  Keys and values place lanes alike.
  const int page_bytes = int4_row_bytes(D) << log2_bs;
  auto code_off = [&](int t8) {
    return ((t8 * 8) >> log2_bs) * page_bytes + ((t8 * 8) & (bs - 1)) * (D / 2);
  };
  auto pair_off = [&](int t8) {
    return ((t8 * 8) >> log2_bs) * page_bytes + ((t8 * 8) & (bs - 1)) * (NG * 4);
  };
  const uint32_t part_base = base + (tok0 >> log2_bs) * page_bytes;
  uint32_t code_at = part_base + (tok0 & (bs - 1)) * (D / 2) + lane * (D / 8);
  uint32_t pair_at = part_base + bs * (D / 2) + ((tok0 & (bs - 1)) + lr) * (NG * 4);

  uint32_t qb[KS][NT][2];
  float qsum[NT][NG][2];   // scale_log2 x sum of the query over a group, heads 2 lc + e
  float qmul[NT][2];       // what a sum of (query x code) products is multiplied by
  // Tokens of a chunk from which on its scores are taken as they are: 32.  Where a
  // head tile's scores are in units of 1 / kFar, more than any, with bit nt set.
  int whole = 32;
  float acc[KS][NT][4], mid[NT][NG][2], m_ref[NT][2], l_sum[NT][2];
  // The scales' power of two and the largest scale it allows.  bf16: chunks since
  // the accumulators were emptied, and the reference points then (`emptied`: there
  // is something in shared memory).
  float nu = 1.f, s_lim = -1.f, m_then[NT][2];
  int chunks = 0;
  bool emptied = false;

  // The query group of head hd, as fp16 scaled by a power of two per head that
  // brings its largest element to 2^10..2^11 (elements paired with the nibbles
  // at bits 0..3 are 16 times larger), and a fresh state.
  auto start_head = [&](int hd) {
    const int s = hd / Hkv, h = hd - s * Hkv;
    whole = 32;
    const T* qp = static_cast<const T*>(p.q) + s * p.q_sb + static_cast<int64_t>(h) * G * p.q_sh;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int g = g_lo + nt * 8 + lr;
      uint32_t raw[KS][2];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        raw[ks][0] = raw[ks][1] = 0u;
        if (g < G) {
          const T* row = qp + g * p.q_sh + (ks >> 2) * 64 + lc * 16 + (ks & 3) * 4;
          raw[ks][0] = *reinterpret_cast<const uint32_t*>(row);
          raw[ks][1] = *reinterpret_cast<const uint32_t*>(row + 2);
        }
      }
      float big = 0.f, sum[NG];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const float2 a = unpack2<T>(raw[ks][0]), b = unpack2<T>(raw[ks][1]);
        big = fmaxf(fmaxf(big, fmaxf(fabsf(a.x), fabsf(a.y))), fmaxf(fabsf(b.x), fabsf(b.y)));
      }
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
      // exponent of the largest element; 0 and non-finite elements: no scaling
      int ex = static_cast<int>(__float_as_uint(big) >> 23) - 127;
      if (big == 0.f || ex > 127) ex = 10;
      if (ex < -110) ex = -110;
      const float up = __uint_as_float(static_cast<uint32_t>(137 - ex) << 23);      // 2^(10 - ex)
      // 2^(ex - 10), what the scaled query's sums and products are multiplied by;
      // where a head's largest element passes 2^64, 2^-40 of it for all of the tile
      // (that keeps it, the codes' weight and the sums inside fp32).
      const bool is_far = !kHalf && __any_sync(0xffffffffu, ex > 64);
      if (is_far) whole |= 0x7ffffff0 | 1 << nt;
      const float down = __uint_as_float(static_cast<uint32_t>(117 + ex) << 23) * (is_far ? kFar : 1.f);
#pragma unroll
      for (int gi = 0; gi < NG; ++gi) {
        sum[gi] = 0.f;
#pragma unroll
        for (int ks = 4 * gi; ks < 4 * gi + 4; ++ks) {
          const float2 a = unpack2<T>(raw[ks][0]), b = unpack2<T>(raw[ks][1]);
          qb[ks][nt][0] = pack2<__half>(a.x * up * 16.f, a.y * up * 16.f);
          qb[ks][nt][1] = pack2<__half>(b.x * up, b.y * up);
          sum[gi] += (a.x * up + a.y * up) + (b.x * up + b.y * up);
        }
        sum[gi] += __shfl_xor_sync(0xffffffffu, sum[gi], 1);
        sum[gi] += __shfl_xor_sync(0xffffffffu, sum[gi], 2);
        sum[gi] *= down;
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        // 2^20: the codes' weight
        qmul[nt][e] = __shfl_sync(0xffffffffu, down * 1048576.f, lc * 8 + e * 4) * p.scale_log2;
        m_ref[nt][e] = kNoScore;
        l_sum[nt][e] = 0.f;
#pragma unroll
        for (int gi = 0; gi < NG; ++gi) {
          qsum[nt][gi][e] = __shfl_sync(0xffffffffu, sum[gi], lc * 8 + e * 4) * p.scale_log2;
          mid[nt][gi][e] = 0.f;
        }
      }
#pragma unroll
      for (int dt = 0; dt < KS; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[dt][nt][i] = 0.f;
    }
    s_lim = -1.f;
    chunks = 0;
    emptied = false;
  };

  // The queries of the head after this one on their way to L1 while the last
  // stage of this one is computed: lane l touches every 32nd sector.
  auto fetch_queries = [&](int hd) {
    if (hd >= kQ4NoHead) return;
    const int s = hd / Hkv, h = hd - s * Hkv;
    const T* qp = static_cast<const T*>(p.q) + s * p.q_sb + static_cast<int64_t>(h) * G * p.q_sh;
    constexpr int kPerRow = D * 2 / 32;  // sectors
    for (int i = lane; i < G * kPerRow; i += 32) {
      uint32_t x;
      asm volatile("ld.global.ca.u32 %0, [%1];"
                   : "=r"(x)
                   : "l"(qp + (i / kPerRow) * p.q_sh + (i % kPerRow) * 16));
    }
  };
  uint32_t joins = 0;  // heads finished so far
  // Adds the accumulators, in units of the output, to this lane's elements of the
  // joining buffer (or puts them there), with `mid` (the sums of the values'
  // other part) at a head's end.  False if the buffer did not become free: every
  // consumer has read the last head's states by then (a fresh barrier's previous
  // phase counts as complete).
  auto deposit = [&](bool last) -> bool {
    if (!emptied && !__all_sync(0xffffffffu, mbar_wait(drained, (joins & 1) ^ 1, kWaitLimitNs)))
      return false;
    // bf16: codes entered as c 2^-24 (even ones of a word) or c 2^-20 (odd ones).
    // Undone in two steps, as 2^24 / nu passes fp32's range for the largest scales.
    const float down = __uint_as_float((254u << 23) - __float_as_uint(nu));
    const float w0 = kHalf ? 1.f : 16777216.f, w1 = kHalf ? 1.f : 1048576.f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int g = g_lo + nt * 8 + lc * 2 + e;
        float* row = join + (part * G + g) * (D + 4) + lr * 8;
        const float keep = emptied ? fast_exp2(m_then[nt][e] - m_ref[nt][e]) : 0.f;
        m_then[nt][e] = m_ref[nt][e];
#pragma unroll
        for (int gi = 0; gi < NG; ++gi) {
          float v = 0.f;
          if (last) {
            v = mid[nt][gi][e];
            v += __shfl_xor_sync(0xffffffffu, v, 4);
            v += __shfl_xor_sync(0xffffffffu, v, 8);
            v += __shfl_xor_sync(0xffffffffu, v, 16);
          }
          // accumulator (tile 4 gi + m, register e + 2 j): element 64 gi + 8 lr + 2 m + j
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            // odd codes entered with the even ones below them
            if constexpr (kHalf) {
              acc[gi * 4 + 2 * half + 1][nt][e] -= 0.0625f * acc[gi * 4 + 2 * half][nt][e];
              acc[gi * 4 + 2 * half + 1][nt][e + 2] -= 0.0625f * acc[gi * 4 + 2 * half][nt][e + 2];
            } else {
              acc[gi * 4 + 2 * half + 1][nt][e] -= acc[gi * 4 + 2 * half][nt][e];
              acc[gi * 4 + 2 * half + 1][nt][e + 2] -= acc[gi * 4 + 2 * half][nt][e + 2];
            }
            float4 x = make_float4(fmaf(acc[gi * 4 + 2 * half][nt][e] * w0, down, v),
                                   fmaf(acc[gi * 4 + 2 * half][nt][e + 2] * w0, down, v),
                                   fmaf(acc[gi * 4 + 2 * half + 1][nt][e] * w1, down, v),
                                   fmaf(acc[gi * 4 + 2 * half + 1][nt][e + 2] * w1, down, v));
            float4* at = reinterpret_cast<float4*>(row + gi * 64 + half * 4);
            if (g < G) {
              if (emptied) {
                const float4 old = *at;
                x = make_float4(fmaf(old.x, keep, x.x), fmaf(old.y, keep, x.y),
                                fmaf(old.z, keep, x.z), fmaf(old.w, keep, x.w));
              }
              *at = x;
            }
            acc[gi * 4 + 2 * half][nt][e] = acc[gi * 4 + 2 * half][nt][e + 2] = 0.f;
            acc[gi * 4 + 2 * half + 1][nt][e] = acc[gi * 4 + 2 * half + 1][nt][e + 2] = 0.f;
          }
        }
      }
    return true;
  };
  // Joins the deposited states of head hd and writes the output (whole) or the
  // partial state of this CTA's segment.
  auto finish_head = [&](int hd, bool whole, int slot) -> bool {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float l = l_sum[nt][e];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        const int g = g_lo + nt * 8 + lc * 2 + e;
        if (lr == 0 && g < G) {
          join_ml[(part * G + g) * 2] = m_ref[nt][e];
          join_ml[(part * G + g) * 2 + 1] = l;
        }
      }
    __syncwarp();
    if (lane == 0) mbar_arrive(joined);
    if (!__all_sync(0xffffffffu, mbar_wait(joined, joins & 1, kWaitLimitNs))) return false;
    ++joins;
    const int s = hd / Hkv, h = hd - s * Hkv;
    for (int idx = tid; idx < G * (D / 4); idx += kQ4Consumers * 32) {
      const int g = idx / (D / 4), c = (idx - g * (D / 4)) * 4;
      float M = -INFINITY, L = 0.f, wt[PARTS];
#pragma unroll
      for (int w = 0; w < PARTS; ++w) M = fmaxf(M, join_ml[(w * G + g) * 2]);
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < PARTS; ++w) {
        wt[w] = fast_exp2(join_ml[(w * G + g) * 2] - M);
        L += wt[w] * join_ml[(w * G + g) * 2 + 1];
        const float4 a = *reinterpret_cast<const float4*>(join + (w * G + g) * (D + 4) + c);
        o.x = fmaf(wt[w], a.x, o.x);
        o.y = fmaf(wt[w], a.y, o.y);
        o.z = fmaf(wt[w], a.z, o.z);
        o.w = fmaf(wt[w], a.w, o.w);
      }
      if (whole) {
        const float inv = 1.f / L;
        const int64_t row = static_cast<int64_t>(s) * Hkv * G + h * G + g;
        if (p.state_o) {
          *reinterpret_cast<float4*>(p.state_o + row * D + c) =
              make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
          if (c == 0) p.state_lse[row] = (M + __log2f(L)) * kLn2;
        } else {
          *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + s * p.o_sb + (h * G + g) * p.o_sh + c) =
              make_uint2(pack2<T>(o.x * inv, o.y * inv), pack2<T>(o.z * inv, o.w * inv));
        }
      } else {
        float* ps = p.part + static_cast<int64_t>(slot) * p.slot_floats;
        __stcg(reinterpret_cast<float4*>(ps + g * D + c), o);
        if (c == 0) {
          __stcg(ps + G * D + g, M);
          __stcg(ps + G * D + G + g, L);
        }
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(drained);
    return true;
  };

  bool timeout = false;
  uint32_t phase = 0;
  for (int slot = 0;;) {
    if (!__all_sync(0xffffffffu, mbar_wait(full + slot * 8, phase, kWaitLimitNs))) {
      timeout = true;
      break;
    }
    const int4 rec = record[slot];
    if (rec.x < 0) break;
    if (rec.z & 1) start_head(rec.x);
    if (rec.z & 2) fetch_queries(rec.z >> 3);
#pragma unroll
    for (int ch = 0; ch < PT / 32; ++ch) {
      const int ntok = rec.y - tok0 - ch * 32;  // valid tokens from here (may be <= 0 or > 32)
      if (ntok <= 0) break;
      // Scores in log2 units, lanes over (token row lr of an 8-token tile,
      // heads 2 lc and 2 lc + 1).
      float sc[MT][NT][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        uint32_t wa[D / 32], wb[D / 32], ma[NG], mb[NG];
        const int t8 = ch * 4 + 2 * mt;
        ld_shared_words<D / 32>(code_at + code_off(t8), wa);
        ld_shared_words<D / 32>(code_at + code_off(t8 + 1), wb);
        ld_shared_words<NG>(pair_at + pair_off(t8), ma);
        ld_shared_words<NG>(pair_at + pair_off(t8 + 1), mb);
        float t[NT][4], z[NT][4];
#pragma unroll
        for (int gi = 0; gi < NG; ++gi) {
          float sg[NT][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) sg[nt][i] = 0.f;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            uint32_t ra[4], rb[4];
            int4_raw_pairs(wa[gi * 2 + j], ra);
            int4_raw_pairs(wb[gi * 2 + j], rb);
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
              const uint32_t a[4] = {ra[2 * hf], rb[2 * hf], ra[2 * hf + 1], rb[2 * hf + 1]};
              const int ks = gi * 4 + j * 2 + hf;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                mma_16816<__half>(sg[nt], a, qb[ks][nt][0], qb[ks][nt][1]);
            }
          }
          const float2 fa = unpack2<T>(ma[gi]), fb = unpack2<T>(mb[gi]);  // scale, minimum
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 f = i < 2 ? fa : fb;
              if (gi == 0) {
                t[nt][i] = f.x * sg[nt][i];
                z[nt][i] = f.y * qsum[nt][gi][i & 1];
              } else {
                t[nt][i] = fmaf(f.x, sg[nt][i], t[nt][i]);
                z[nt][i] = fmaf(f.y, qsum[nt][gi][i & 1], z[nt][i]);
              }
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[mt][nt][i] = fmaf(t[nt][i], qmul[nt][i & 1], z[nt][i]);
      }
      const bool ragged = ntok < whole;
      if (ragged) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (!kHalf && whole >> nt & 1) sc[mt][nt][i] *= 1.f / kFar;
              if (mt * 16 + lr + (i >> 1) * 8 >= ntok) sc[mt][nt][i] = -INFINITY;
            }
      }
      // The reference point of the softmax.
      float mx[NT][2];
      bool up = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          mx[nt][e] = fmaxf(sc[0][nt][e], sc[0][nt][e + 2]);
#pragma unroll
          for (int mt = 1; mt < MT; ++mt)
            mx[nt][e] = fmaxf(mx[nt][e], fmaxf(sc[mt][nt][e], sc[mt][nt][e + 2]));
          up |= mx[nt][e] > m_ref[nt][e] + kRaise;
        }
      if (__any_sync(0xffffffffu, up)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float m = mx[nt][e];
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
            const float mn = fmaxf(m_ref[nt][e], m);
            const float alpha = fast_exp2(m_ref[nt][e] - mn);
            m_ref[nt][e] = mn;
            l_sum[nt][e] *= alpha;
#pragma unroll
            for (int gi = 0; gi < NG; ++gi) mid[nt][gi][e] *= alpha;
#pragma unroll
            for (int dt = 0; dt < KS; ++dt) {
              acc[dt][nt][e] *= alpha;
              acc[dt][nt][e + 2] *= alpha;
            }
          }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = e; i < 4; i += 2) {
              sc[mt][nt][i] = fast_exp2(sc[mt][nt][i] - m_ref[nt][e]);
              l_sum[nt][e] += sc[mt][nt][i];
            }
        }
      // The values' scales and minima; rows past the end may hold anything: zeros.
      uint32_t ma[MT][NG], mb[MT][NG];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const int t8 = ch * 4 + 2 * mt;
        ld_shared_words<NG>(pair_at + KV_BYTES + pair_off(t8), ma[mt]);
        ld_shared_words<NG>(pair_at + KV_BYTES + pair_off(t8 + 1), mb[mt]);
        if (ragged) {
          const bool oka = mt * 16 + lr < ntok, okb = mt * 16 + 8 + lr < ntok;
#pragma unroll
          for (int gi = 0; gi < NG; ++gi) {
            ma[mt][gi] = oka ? ma[mt][gi] : 0u;
            mb[mt][gi] = okb ? mb[mt][gi] : 0u;
          }
        }
      }
      {
        uint32_t big = ma[0][0];  // pairs (scale, minimum): the low half counts
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int gi = 0; gi < NG; ++gi) {
            if (mt + gi) big = max2<T>(big, ma[mt][gi]);
            big = max2<T>(big, mb[mt][gi]);
          }
        const float s_max = unpack2<T>(big).x;
        if (__any_sync(0xffffffffu, s_max > s_lim)) {
          // Scales are >= 0 (or NaN, which stays out): their bits order them.
          const uint32_t bits = __reduce_max_sync(0xffffffffu, s_max > 0.f ? __float_as_uint(s_max) : 0u);
          // four times the power of two above the largest becomes 2^13; fp16: none
          // shrinks, as 2^kRaise times its largest scale is still in range
          const uint32_t ex = min(max((bits >> 23) + 3u, 16u), kHalf ? 140u : 255u);
          const float nu_new = __uint_as_float((267u - ex) << 23);
          const float f = s_lim < 0.f ? 0.f : nu_new * __uint_as_float((254u << 23) - __float_as_uint(nu));
          nu = nu_new;
          s_lim = kHalf && ex == 140u ? INFINITY : __uint_as_float(ex << 23);
#pragma unroll
          for (int dt = 0; dt < KS; ++dt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int i = 0; i < 4; ++i) acc[dt][nt][i] *= f;
        }
      }
      // O^T += V^T P^T on the codes.
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        if (ragged && mt * 16 >= ntok) break;
        uint32_t wa[D / 32], wb[D / 32];
        const int t8 = ch * 4 + 2 * mt;
        ld_shared_words<D / 32>(code_at + KV_BYTES + code_off(t8), wa);
        ld_shared_words<D / 32>(code_at + KV_BYTES + code_off(t8 + 1), wb);
#pragma unroll
        for (int gi = 0; gi < NG; ++gi) {
          // (scale, value of the code that enters as 0)
          float2 fa = kHalf ? int4_centre<T>(ma[mt][gi]) : unpack2<T>(ma[mt][gi]);
          float2 fb = kHalf ? int4_centre<T>(mb[mt][gi]) : unpack2<T>(mb[mt][gi]);
          fa.x *= nu;
          fb.x *= nu;
          uint32_t pg[NT][2];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            pg[nt][0] = movmatrix_trans(pack2<__half>(sc[mt][nt][0] * fa.x, sc[mt][nt][1] * fa.x));
            pg[nt][1] = movmatrix_trans(pack2<__half>(sc[mt][nt][2] * fb.x, sc[mt][nt][3] * fb.x));
#pragma unroll
            for (int e = 0; e < 2; ++e)
              mid[nt][gi][e] = fmaf(sc[mt][nt][e], fa.y, fmaf(sc[mt][nt][e + 2], fb.y, mid[nt][gi][e]));
          }
          uint32_t xa[4], ya[4], xb[4], yb[4];
          // The octet's words of two consecutive tokens -> pairs (even token,
          // odd token) of one element: even elements x, odd elements y.
          int4_value_pairs<kHalf>(__byte_perm(wa[gi], wa[NG + gi], 0x5410), xa);
          int4_value_pairs<kHalf>(__byte_perm(wa[gi], wa[NG + gi], 0x7632), ya);
          int4_value_pairs<kHalf>(__byte_perm(wb[gi], wb[NG + gi], 0x5410), xb);
          int4_value_pairs<kHalf>(__byte_perm(wb[gi], wb[NG + gi], 0x7632), yb);
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            const uint32_t a[4] = {xa[m], ya[m], xb[m], yb[m]};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma_16816<__half>(acc[gi * 4 + m][nt], a, pg[nt][0], pg[nt][1]);
          }
        }
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(empty + slot * 8);  // the slot may be refilled
    code_at += STAGE_BYTES;
    pair_at += STAGE_BYTES;
    if (++slot == depth) {
      slot = 0;
      phase ^= 1;
      code_at -= depth * STAGE_BYTES;
      pair_at -= depth * STAGE_BYTES;
    }
    const bool last = (rec.z & 2) != 0;
    chunks += PT / 32;
    if (last || (!kHalf && chunks >= kFlush)) {
      if (!deposit(last) || (last && !finish_head(rec.x, (rec.z & 4) != 0, rec.x + u))) {
        timeout = true;
        break;
      }
      chunks = 0;
      emptied = !kHalf;  // (a last deposit: start_head resets it)
    }
  }
  grid_dependency_wait();  // the reduce kernel follows the planner too
  if (timeout && lane == 0) atomicOr(p.status, kStatusTimeout);
}

}  // namespace pab
