// Attention weights per cached key, and the eviction of keys by them; the page copy of a forked sequence.
//
// AttnWeightsKernel adds to w[key] the softmax weights that the six query heads of a kv head's group gave the key in the
// decode call just made: w[key] += sum_g 2^(s_g - M_g - log2 L_g), s_g = q_g.k * scale in log2 units. The call's
// partials give M_g and L_g (joined in unit order), so one pass over K is enough; it reads K again (the part kernels
// keep no scores) and is HBM-bound: half of the cache bytes plus 8 B per key and kv head. Scores are computed in fp32
// from the fp16 query and the exact codes (f16 MMA on exact fp16 integers, the block scale applied in fp32), so a
// weight is as exact as fp32 sums make it; the part kernels' 16-bit query planes would cost 2e-5 of a weight.
// The shape of the decode kernels without their V side: one CTA per split-K unit, a ring of K pages filled by TMA
// (no multicast), eight warps on two pages at a time, 16 keys of a page per warp, the last of a page's warps refills its
// stage. No order-dependent sums: each key is added to once per call.
//
// EvictSelectKernel, one CTA per (layer, sequence, kv head): the n_keep keys to keep, ascending. The first n_sink and the
// last n_recent are kept, of the rest the largest weights; ties go to the lowest index, NaN counts as less than
// everything. A radix select over the order-preserving bits finds the smallest kept weight and how many keys of exactly
// that weight are kept; a last pass in index order writes the kept indices and moves the weights to the front.
//
// EvictMoveKernel moves the kept rows to slots 0 .. n_keep - 1, in place where the sequence has its pages to itself: kept
// index i is at least i, so with chunks of slots in ascending order a chunk's sources lie at or behind its slots, and
// only the chunk's own reads have to come before its writes. Pages that another sequence shares are replaced by fresh
// ones (the host lists them) and stay as they were.
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

#include "decode_ring.cuh"
#include "kernels.cuh"
#include "ptx.cuh"

namespace yahkv {
namespace {

// ----------------------------------------------------------------------------------------------------------------
// attention weights
// ----------------------------------------------------------------------------------------------------------------
constexpr int kKeyGroups = 4;                      // 16 keys of a page each
constexpr int kPageSets = 2;                       // pages in work at a time: warp w takes those of parity w / 4
constexpr int kWeightWarps = kKeyGroups * kPageSets;
constexpr int kWeightThreads = kWeightWarps * 32;
constexpr int kBoxBytes = kPageTokens * 128;       // one swizzled TMA box: 64 token rows x 128 B

// Shared memory: ring of K boxes | ring of block scales | query operands (quantized formats) | barriers, counters, abort
// flag. fp16: three stages of 32 KB and two CTAs per SM, the query operands in registers. Quantized formats issue more
// instructions per byte: three CTAs, q8_0 with 4 x 17 KB, q4_0 with 6 x 9 KB, the query operands in shared memory, so that
// 80 registers do (with two CTAs and the operands in registers the kernel spilled: 120 us against TODO us).
template <int kFmt>
struct WeightSmem {
  static constexpr int kBoxes = CodeBytes(kFmt) / 128;
  static constexpr int kStages = kFmt == kFmtF16 ? 3 : kFmt == kFmtQ8 ? 4 : 6;
  static constexpr int kCtas = kFmt == kFmtF16 ? 2 : 3;
  static constexpr int kScaleBytes = RecordScaleBytes(kFmt, 0);
  static constexpr int kTx = kBoxes * kBoxBytes + kScaleBytes;
  static constexpr int kScaleOff = kStages * kBoxes * kBoxBytes;
  static constexpr int kQOff = kScaleOff + kStages * kScaleBytes;   // [8 blocks][32 lanes] 16 bytes
  static constexpr int kBarOff = kQOff + (kFmt == kFmtF16 ? 0 : kBlocksPerRow * 32 * 16);
  static constexpr int kDoneOff = kBarOff + 8 * kStages;
  static constexpr int kFillOff = kDoneOff + 4 * kStages;
  static constexpr int kAbortOff = kFillOff + 4 * kStages;
  static constexpr int kNormOff = kAbortOff + 4;
  static constexpr int kBytes = (kNormOff + 4 * 8 + 127) / 128 * 128;
  static_assert(kCtas * (kBytes + 1024) <= 228 * 1024, "resident CTAs per SM");
  static_assert(kPageSets <= kStages, "a set never waits for a stage it holds itself");
};
constexpr int kStatusSmemMisaligned = 2;

// Four bytes u -> fp16 pairs (0, 1), (2, 3) of u - bias (0x6400 | u is 1024 + u; bias_h = 1024 + bias).
__device__ __forceinline__ void Bytes4(std::uint32_t u, __half2 bias_h, std::uint32_t& h01, std::uint32_t& h23) {
  const std::uint32_t a = __byte_perm(u, 0x64646464U, 0x4140), b = __byte_perm(u, 0x64646464U, 0x4342);
  const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), bias_h), y = __hsub2(*reinterpret_cast<const __half2*>(&b), bias_h);
  h01 = *reinterpret_cast<const std::uint32_t*>(&x), h23 = *reinterpret_cast<const std::uint32_t*>(&y);
}
__device__ __forceinline__ float HalfOf(const uint2& v, int i) {   // fp16 number i of four, i a constant after unrolling
  const std::uint32_t w = i < 2 ? v.x : v.y;
  const __half2 h = *reinterpret_cast<const __half2*>(&w);
  return (i & 1) ? __high2float(h) : __low2float(h);
}
// D(16 x 8, f32) = A(16 x 16, f16) . B(16 x 8, f16), no accumulator input
__device__ __forceinline__ void MmaF16Zero(float (&d)[4], std::uint32_t a0, std::uint32_t a1, std::uint32_t a2, std::uint32_t a3,
                                           std::uint32_t b0, std::uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0F));
}

template <int kFmt>
__global__ void __launch_bounds__(kWeightThreads, WeightSmem<kFmt>::kCtas)
    AttnWeightsKernel(const __grid_constant__ CUtensorMap kmap, PoolView pool, int layer,
                      const std::int32_t* __restrict__ tables, int table_stride, const DecodeUnit* __restrict__ units,
                      const CombineItem* __restrict__ items, const __half* __restrict__ q, float scale_log2,
                      const float* __restrict__ partial_ml, float* __restrict__ weights, long long weights_stride, int* status) {
  using L = WeightSmem<kFmt>;
  extern __shared__ __align__(1024) std::uint8_t smem[];
  ChainedKernelEntry();
  float* norm_s = reinterpret_cast<float*>(smem + L::kNormOff);   // M + log2 L per query head
  std::uint64_t* full_bar = reinterpret_cast<std::uint64_t*>(smem + L::kBarOff);
  int* done_cnt = reinterpret_cast<int*>(smem + L::kDoneOff);
  int* fill_cnt = reinterpret_cast<int*>(smem + L::kFillOff);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kAbortOff);
  if ((SmemAddr(smem) & 1023U) != 0) {   // never seen; a misaligned swizzle would corrupt results
    if (threadIdx.x == 0) atomicExch(status, kStatusSmemMisaligned);
    return;
  }
  const DecodeUnit u = units[blockIdx.x];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int kw = warp & (kKeyGroups - 1), par = warp / kKeyGroups;
  const int n_pages = u.page_end - u.page_begin;
  if (n_pages <= 0) return;
  const std::int32_t* row = tables + static_cast<std::size_t>(u.seq) * table_stride + u.page_begin;

  // Gather of one page's K into a ring stage; a whole converged warp calls it, one elected lane issues. Once a wait has
  // given up nothing more is fetched.
  auto issue = [&](int s, std::int32_t page) {
    if (*abort_flag != 0) return;
    page = min(max(page, 0), pool.num_pages - 1);   // never trust a table entry read from memory
    const std::size_t rec = (static_cast<std::size_t>(layer) * pool.num_pages + page) * kKvHeads + u.kvh;
    if (ElectOne()) {
      fill_cnt[s] += 1;
      MbarArriveExpectTx(&full_bar[s], L::kTx);
#pragma unroll
      for (int b = 0; b < L::kBoxes; ++b)
        TmaLoad2D(smem + (s * L::kBoxes + b) * kBoxBytes, &kmap, b * 128, static_cast<int>(rec * kPageTokens), &full_bar[s]);
      if constexpr (L::kScaleBytes > 0)
        BulkLoad(smem + L::kScaleOff + s * L::kScaleBytes, pool.kscales + rec * (kPageTokens * kBlocksPerRow), L::kScaleBytes, &full_bar[s]);
    }
  };
  if (warp == 0) {
    if (lane == 0) {
      PrefetchTensorMap(&kmap);
      for (int s = 0; s < L::kStages; ++s) {
        MbarInit(&full_bar[s], 1);
        done_cnt[s] = 0;
        fill_cnt[s] = 0;
      }
      *abort_flag = 0;
      FenceBarrierInit();
    }
    __syncwarp();
    for (int i = 0; i < L::kStages && i < n_pages; ++i) issue(i, __ldg(row + i));
  }

  // M + log2 L of the six heads from the partials of the decode call, warp h < 6 for head h
  if (warp < kGroup) {
    const CombineItem it = items[u.batch * kKvHeads + u.kvh];
    const float* ml = partial_ml + static_cast<std::size_t>(it.first_partial) * kPartialMlFloats + 2 * warp;
    float m = -INFINITY, l = 0.0F;
    for (int i = lane; i < it.n_partials; i += 32) m = fmaxf(m, ml[static_cast<std::size_t>(i) * kPartialMlFloats]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFU, m, o));
    for (int i = lane; i < it.n_partials; i += 32) {
      const float mi = ml[static_cast<std::size_t>(i) * kPartialMlFloats];
      l += mi == -INFINITY ? 0.0F : exp2f(mi - m) * ml[static_cast<std::size_t>(i) * kPartialMlFloats + 1];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xFFFFFFFFU, l, o);
    if (lane == 0) norm_s[warp] = m + log2f(l);
  }
  // S[key][head] = K[key][dim] . Q^T[dim][head]: A = 16 keys as ldmatrix hands them over, B = the query, column g = head g.
  // fp16: dims 16 s + 2t, + 1 and 16 s + 8 + 2t, + 1 of step s. Codes: a 16-byte piece is 16 codes (q8_0) or a block's 32
  // nibbles (q4_0), lane t has its bytes 4t .. 4t + 3: elements 4t .. of a 32-element block and 16 + 4t ..
  std::uint32_t qa[kFmt == kFmtF16 ? 32 : 1];
  if constexpr (kFmt == kFmtF16) {
    const __half* src = q + (static_cast<std::size_t>(u.batch) * kQHeads + u.kvh * kGroup + min(g, kGroup - 1)) * kHeadDim;
#pragma unroll
    for (int i = 0; i < 32; ++i) qa[i] = g < kGroup ? __ldg(reinterpret_cast<const std::uint32_t*>(src + 8 * i + 2 * t)) : 0U;
  } else {   // warp b lays out block b: lane (g, t) dims 32 b + 4t .. + 3 and 32 b + 16 + 4t .. + 3 of head g
    const __half* src = q + (static_cast<std::size_t>(u.batch) * kQHeads + u.kvh * kGroup + min(g, kGroup - 1)) * kHeadDim + 32 * warp;
    uint2 lo = __ldg(reinterpret_cast<const uint2*>(src + 4 * t)), hi = __ldg(reinterpret_cast<const uint2*>(src + 16 + 4 * t));
    if (g >= kGroup) lo = hi = make_uint2(0, 0);
    *reinterpret_cast<uint4*>(smem + L::kQOff + (warp * 32 + lane) * 16) = make_uint4(lo.x, lo.y, hi.x, hi.y);
    static_assert(kWeightWarps == kBlocksPerRow, "a warp per block");
  }
  __syncthreads();   // barriers initialised, norms visible
  // this thread's results are heads 2t, 2t + 1 of keys g and g + 8; the padding heads weigh nothing
  const float norm0 = t < 3 ? norm_s[2 * t] : INFINITY, norm1 = t < 3 ? norm_s[2 * t + 1] : INFINITY;
  float* w_out = weights + (static_cast<std::size_t>(u.seq) * kKvHeads + u.kvh) * static_cast<std::size_t>(weights_stride);
  const __half2 bias = __half2half2(__ushort_as_half(kFmt == kFmtQ8 ? 0x6480 : 0x6408));
  // ldmatrix rows: matrices = (keys 0-7 | 8-15 of the group) x (16-byte pieces 2x | 2x + 1); piece p of row r sits at p ^ (r % 8)
  const int lm_key = kw * 16 + (lane & 7) + ((lane >> 3) & 1) * 8;
  const std::uint32_t lm0 = lm_key * 128 + (((lane >> 4) ^ (lm_key & 7)) << 4);

  bool alive = true;
  for (int i = par; i < n_pages; i += kPageSets) {
    const int s = i % L::kStages, gen = i / L::kStages;
    std::int32_t refill_page = 0;
    if (lane == 0 && i + L::kStages < n_pages) refill_page = __ldg(row + i + L::kStages);
    alive = RingWait(alive, fill_cnt + s, &full_bar[s], gen, abort_flag);
    const std::uint32_t k_base = SmemAddr(smem + s * L::kBoxes * kBoxBytes);
    float sc[4] = {0.0F, 0.0F, 0.0F, 0.0F};   // (key g, head 2t), (g, 2t + 1), (g + 8, 2t), (g + 8, 2t + 1)
    if constexpr (kFmt == kFmtF16) {
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        std::uint32_t w[4];
        LdMatrixX4(k_base + (x >> 2) * kBoxBytes + (lm0 ^ (static_cast<std::uint32_t>(x & 3) << 5)), w);
        MmaF16(sc, w[0], w[1], w[2], w[3], qa[2 * x], qa[2 * x + 1]);
      }
    } else {
      const std::uint8_t* scales = smem + L::kScaleOff + s * L::kScaleBytes + (kw * 16 + g) * (kBlocksPerRow * 2);
      const std::uint32_t q_base = SmemAddr(smem + L::kQOff) + lane * 16;
#pragma unroll
      for (int dh = 0; dh < 2; ++dh) {   // blocks 4 dh .. + 3; scales fetched per half to keep registers low
        const uint2 d0 = *reinterpret_cast<const uint2*>(scales + dh * 8);
        const uint2 d1 = *reinterpret_cast<const uint2*>(scales + 8 * (kBlocksPerRow * 2) + dh * 8);
        // one block of 32 elements: two k-steps into a fresh accumulator, then the keys' scales
        auto block = [&](int b, std::uint32_t lo0, std::uint32_t lo1, std::uint32_t hi0, std::uint32_t hi1) {
          std::uint32_t qb[4], a0, a1, a2, a3;
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(qb[0]), "=r"(qb[1]), "=r"(qb[2]), "=r"(qb[3])
                       : "r"(q_base + (4 * dh + b) * 512));
          float acc[4];
          Bytes4(lo0, bias, a0, a2);
          Bytes4(lo1, bias, a1, a3);
          MmaF16Zero(acc, a0, a1, a2, a3, qb[0], qb[1]);
          Bytes4(hi0, bias, a0, a2);
          Bytes4(hi1, bias, a1, a3);
          MmaF16(acc, a0, a1, a2, a3, qb[2], qb[3]);
          const float s0 = HalfOf(d0, b), s1 = HalfOf(d1, b);
          sc[0] = fmaf(s0, acc[0], sc[0]), sc[1] = fmaf(s0, acc[1], sc[1]);
          sc[2] = fmaf(s1, acc[2], sc[2]), sc[3] = fmaf(s1, acc[3], sc[3]);
        };
        if constexpr (kFmt == kFmtQ8) {
#pragma unroll
          for (int b = 0; b < 4; ++b) {   // pieces 2b, 2b + 1 of box dh: one block
            std::uint32_t w[4];
            LdMatrixX4(k_base + dh * kBoxBytes + (lm0 ^ (static_cast<std::uint32_t>(b) << 5)), w);
            block(b, w[0] ^ kQ8FlipWord, w[1] ^ kQ8FlipWord, w[2] ^ kQ8FlipWord, w[3] ^ kQ8FlipWord);
          }
        } else {
#pragma unroll
          for (int x = 0; x < 2; ++x) {   // a piece is a block
            std::uint32_t w[4];
            LdMatrixX4(k_base + (lm0 ^ (static_cast<std::uint32_t>(2 * dh + x) << 5)), w);
#pragma unroll
            for (int k = 0; k < 2; ++k)
              block(2 * x + k, w[2 * k] & 0x0F0F0F0FU, w[2 * k + 1] & 0x0F0F0F0FU, (w[2 * k] >> 4) & 0x0F0F0F0FU,
                    (w[2 * k + 1] >> 4) & 0x0F0F0F0FU);
          }
        }
      }
    }
    // the stage is in registers: the last of the page's four warps refills it
    const bool last = RingRelease(&done_cnt[s], lane, kKeyGroups);
    if (last && i + L::kStages < n_pages) issue(s, __shfl_sync(0xFFFFFFFFU, refill_page, 0));
    float p0 = exp2f(fmaf(sc[0], scale_log2, -norm0)) + exp2f(fmaf(sc[1], scale_log2, -norm1));
    float p1 = exp2f(fmaf(sc[2], scale_log2, -norm0)) + exp2f(fmaf(sc[3], scale_log2, -norm1));
    p0 += __shfl_xor_sync(0xFFFFFFFFU, p0, 1), p1 += __shfl_xor_sync(0xFFFFFFFFU, p1, 1);
    p0 += __shfl_xor_sync(0xFFFFFFFFU, p0, 2), p1 += __shfl_xor_sync(0xFFFFFFFFU, p1, 2);
    // lanes t = 0 and 1 add keys g and g + 8: one addition per key and call, so the order of CTAs does not matter
    const int key = (u.page_begin + i) * kPageTokens + kw * 16 + 8 * t + g;
    if (t < 2 && key < u.n_keys) atomicAdd(w_out + key, t == 0 ? p0 : p1);
  }
  if (!alive && lane == 0) atomicExch(status, kStatusWaitTimeout);
  __syncthreads();
  RingDrainAfterAbort(abort_flag, fill_cnt, full_bar, L::kStages);
}

// ----------------------------------------------------------------------------------------------------------------
// selection
// ----------------------------------------------------------------------------------------------------------------
constexpr int kSelectThreads = 1024;
constexpr int kSelectPer = 4;                                  // keys per thread and turn of the last pass
constexpr int kSelectTile = kSelectThreads * kSelectPer;
constexpr int kSelectCache = 36 * 1024;                        // keys whose words are kept in shared memory (144 KB)
// Histograms: a lane counts into copy lane % 8, copies an odd number of words apart, so that equal weights (zeros above
// all) meet four at a time and not 32 at a time. (One histogram with the lanes of equal bins joined by match.any first:
// 33 us for 128 rows of 14,000 keys against TODO us.)
constexpr int kHistCopies = 8, kHistBins = 2048, kHistStride = kHistBins + 1;

// Order-preserving bits of a weight: larger weight, larger word; NaN below everything, -0 equal to +0.
__device__ __forceinline__ std::uint32_t OrderOf(float w) {
  if (w != w) return 0U;
  const std::uint32_t b = __float_as_uint(w == 0.0F ? 0.0F : w);
  return (b & 0x80000000U) != 0 ? ~b : b | 0x80000000U;
}
// Exclusive prefix sum over the CTA's threads; *total receives the sum. scan_s: one int per warp. Two barriers inside.
__device__ __forceinline__ int CtaScan(int v, int* scan_s, int lane, int warp, int* total) {
  int sum = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int x = __shfl_up_sync(0xFFFFFFFFU, sum, d);
    if (lane >= d) sum += x;
  }
  if (lane == 31) scan_s[warp] = sum;
  __syncthreads();
  if (warp == 0) {
    int x = scan_s[lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(0xFFFFFFFFU, x, d);
      if (lane >= d) x += y;
    }
    scan_s[lane] = x;
  }
  __syncthreads();
  *total = scan_s[31];
  return (warp > 0 ? scan_s[warp - 1] : 0) + sum - v;
}

__global__ void __launch_bounds__(kSelectThreads)
    EvictSelectKernel(const EvictSeq* __restrict__ seqs, int n_seqs, int kv_head_begin, int n_keep, int n_sink, int n_recent,
                      float* __restrict__ weights, long long weights_stride, long long layer_stride, int n_cache,
                      std::int32_t* __restrict__ kept) {
  extern __shared__ std::uint32_t select_smem[];
  int* hist = reinterpret_cast<int*>(select_smem);
  std::uint32_t* word_s = select_smem + kHistCopies * kHistStride;   // [n_cache] words of the first keys to choose from
  __shared__ int scan_s[kSelectThreads / 32];
  __shared__ std::uint32_t prefix_s;
  __shared__ int want_s;
  ChainedKernelEntry();
  const int b = blockIdx.x, h = kv_head_begin + blockIdx.y, layer = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const EvictSeq es = seqs[b];
  std::int32_t* out = kept + ((static_cast<std::size_t>(layer) * n_seqs + b) * kKvHeads + h) * static_cast<std::size_t>(n_keep);
  if (es.n_keys <= n_keep) {   // nothing to evict: the sequence stays as it is
    for (int i = tid; i < n_keep; i += kSelectThreads) out[i] = i < es.n_keys ? i : -1;
    return;
  }
  float* w = weights + static_cast<std::size_t>(layer) * layer_stride +
             (static_cast<std::size_t>(es.seq) * kKvHeads + h) * static_cast<std::size_t>(weights_stride);
  const int lo = n_sink, n_mid = es.n_keys - n_recent - n_sink;   // the keys to choose from are lo .. lo + n_mid - 1
  const int n_choose = n_keep - n_sink - n_recent;                // fewer than n_mid
  const int n_held = min(n_mid, n_cache);
  int want = n_choose;
  // the want-th largest word, eleven, eleven and ten bits at a time; the first pass fills the cache
  std::uint32_t prefix = 0, mask = 0;
  if (want > 0) {
    const int shifts[3] = {21, 10, 0}, bits[3] = {11, 11, 10};
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
      for (int i = tid; i < kHistCopies * kHistStride; i += kSelectThreads) hist[i] = 0;
      __syncthreads();
      const std::uint32_t bin_mask = (1U << bits[pass]) - 1U;
      for (int i0 = 0; i0 < n_mid; i0 += kSelectTile) {
        std::uint32_t o[kSelectPer];
        bool on[kSelectPer];
#pragma unroll
        for (int k = 0; k < kSelectPer; ++k) {
          const int i = i0 + k * kSelectThreads + tid;
          on[k] = i < n_mid;
          o[k] = !on[k] ? 0U : pass > 0 && i < n_held ? word_s[i] : OrderOf(w[lo + i]);
        }
#pragma unroll
        for (int k = 0; k < kSelectPer; ++k) {
          const int i = i0 + k * kSelectThreads + tid;
          if (pass == 0 && i < n_held) word_s[i] = o[k];
          if (on[k] && (o[k] & mask) == prefix) atomicAdd(&hist[(lane % kHistCopies) * kHistStride + ((o[k] >> shifts[pass]) & bin_mask)], 1);
        }
      }
      __syncthreads();
      // counts from the largest bin down; two bins per thread
      const int top = kHistBins - 1 - 2 * tid;
      int c0 = 0, c1 = 0;
#pragma unroll
      for (int c = 0; c < kHistCopies; ++c) c0 += hist[c * kHistStride + top], c1 += hist[c * kHistStride + top - 1];
      int total;
      const int before = CtaScan(c0 + c1, scan_s, lane, warp, &total);
      if (before < want && before + c0 >= want) {
        prefix_s = prefix | (static_cast<std::uint32_t>(top) << shifts[pass]);
        want_s = want - before;
      } else if (before + c0 < want && before + c0 + c1 >= want) {
        prefix_s = prefix | (static_cast<std::uint32_t>(top - 1) << shifts[pass]);
        want_s = want - before - c0;
      }
      __syncthreads();
      prefix = prefix_s, want = want_s;
      mask |= bin_mask << shifts[pass];
      __syncthreads();
    }
  }
  // prefix is the smallest kept word and `want` keys of exactly that word are kept, the lowest indices. In index order, a
  // kept key's slot is the number of keys kept before it; a thread takes four neighbouring keys.
  int base_gt = 0, base_eq = 0;
  for (int i0 = 0; i0 < es.n_keys; i0 += kSelectTile) {
    const int at = i0 + kSelectPer * tid;
    float wi[kSelectPer];
    bool gt[kSelectPer], eq[kSelectPer];
    int count = 0;   // keys above the border in the low half, keys on it in the high half: at most 4096 of each
#pragma unroll
    for (int k = 0; k < kSelectPer; ++k) {
      const int i = at + k, m = i - lo;
      const bool in = i < es.n_keys, middle = in && m >= 0 && m < n_mid;
      wi[k] = in ? w[i] : 0.0F;
      const std::uint32_t o = middle ? OrderOf(wi[k]) : 0U;
      gt[k] = in && (!middle || (n_choose > 0 && o > prefix));
      eq[k] = middle && n_choose > 0 && o == prefix;
      count += (gt[k] ? 1 : 0) + (eq[k] ? 1 << 16 : 0);
    }
    int total;
    const int before = CtaScan(count, scan_s, lane, warp, &total);   // behind its barriers every weight of the tile has been read
    int gt_before = base_gt + (before & 0xFFFF), eq_before = base_eq + (before >> 16);
#pragma unroll
    for (int k = 0; k < kSelectPer; ++k) {
      if (gt[k] || (eq[k] && eq_before < want)) {
        const int slot = gt_before + min(eq_before, want);
        if (slot < n_keep) out[slot] = at + k, w[slot] = wi[k];
      }
      gt_before += gt[k] ? 1 : 0, eq_before += eq[k] ? 1 : 0;
    }
    base_gt += total & 0xFFFF, base_eq += total >> 16;
    __syncthreads();
  }
  for (int i = n_keep + tid; i < es.n_keys; i += kSelectThreads) w[i] = 0.0F;   // slots of keys to come
}

// ----------------------------------------------------------------------------------------------------------------
// moving the kept rows
// ----------------------------------------------------------------------------------------------------------------
constexpr int kMoveThreads = 512;
constexpr int kMovePer = 4;   // 16-byte pieces of codes per thread and chunk

// One CTA per (layer, sequence, kv head, side): chunks of whole rows (128 of q8_0), so that a row's bytes are asked for
// together, 32 KB at a time, and the next chunk's loads are in flight while a chunk is written.
template <int kFmt>
__global__ void __launch_bounds__(kMoveThreads)
    EvictMoveKernel(PoolView pool, const std::int32_t* __restrict__ tables, int table_stride, const EvictSeq* __restrict__ seqs,
                    int n_seqs, const std::int32_t* __restrict__ dst_pages, int n_keep, const std::int32_t* __restrict__ kept) {
  constexpr int kPieces = CodeBytes(kFmt) / 16;                     // of a row
  constexpr int kRows = kMoveThreads * kMovePer / kPieces;          // of a chunk
  constexpr bool kScales = kFmt != kFmtF16;
  static_assert(!kScales || kRows <= kMoveThreads, "one thread per row's scales");
  ChainedKernelEntry();
  const int b = blockIdx.x, side = blockIdx.y & 1, h = pool.kv_head_begin + (blockIdx.y >> 1), layer = blockIdx.z;
  const EvictSeq es = seqs[b];
  if (es.n_keys <= n_keep) return;
  const int tid = threadIdx.x;
  const std::int32_t* idx = kept + ((static_cast<std::size_t>(layer) * n_seqs + b) * kKvHeads + h) * static_cast<std::size_t>(n_keep);
  const std::int32_t* table = tables + static_cast<std::size_t>(es.seq) * table_stride;
  const std::int32_t* dst = dst_pages + es.first_dst;
  uint4* codes = reinterpret_cast<uint4*>(side == 0 ? pool.kcodes : pool.vcodes);
  uint4* scales = reinterpret_cast<uint4*>(side == 0 ? pool.kscales : pool.vscales);
  // row of the pools, in rows of one kv head
  auto row_of = [&](std::int32_t page, int tok) -> std::size_t {
    page = min(max(page, 0), pool.num_pages - 1);   // never trust a table entry read from memory
    return ((static_cast<std::size_t>(layer) * pool.num_pages + page) * kKvHeads + h) * kPageTokens + tok;
  };
  auto source = [&](int slot) -> std::size_t {
    const int i = min(max(__ldg(idx + slot), 0), es.n_keys - 1);
    return row_of(__ldg(table + i / kPageTokens), i % kPageTokens);
  };
  auto target = [&](int slot) -> std::size_t { return row_of(__ldg(dst + slot / kPageTokens), slot % kPageTokens); };
  uint4 v[kMovePer], sc = make_uint4(0, 0, 0, 0);
  auto load = [&](int c0) {
    std::size_t at[kMovePer];
#pragma unroll
    for (int k = 0; k < kMovePer; ++k) at[k] = source(min(c0 + (tid + k * kMoveThreads) / kPieces, n_keep - 1));
#pragma unroll
    for (int k = 0; k < kMovePer; ++k) v[k] = codes[at[k] * kPieces + tid % kPieces];
    if (kScales && tid < kRows) sc = scales[source(min(c0 + tid, n_keep - 1))];
  };
  static_assert(kMoveThreads % kPieces == 0, "a thread keeps its piece of a row");
  load(0);
  for (int c0 = 0; c0 < n_keep; c0 += kRows) {
    uint4 mine[kMovePer];
    const uint4 my_sc = sc;
#pragma unroll
    for (int k = 0; k < kMovePer; ++k) mine[k] = v[k];
    __syncthreads();   // every row of the chunk is in registers: its slots may be written
    if (c0 + kRows < n_keep) load(c0 + kRows);   // sources at or behind the next chunk's first slot
#pragma unroll
    for (int k = 0; k < kMovePer; ++k) {
      const int slot = c0 + (tid + k * kMoveThreads) / kPieces;
      if (slot < n_keep) codes[target(slot) * kPieces + tid % kPieces] = mine[k];
    }
    if (kScales && tid < kRows && c0 + tid < n_keep) scales[target(c0 + tid)] = my_sc;
  }
}

// Page src -> page dst, every layer, all kv heads, both sides: the partly filled last page of a forked prefix.
__global__ void __launch_bounds__(256) CopyPageKernel(PoolView pool, int src, int dst) {
  ChainedKernelEntry();
  const int layer = blockIdx.x, what = blockIdx.y;   // 0, 1: K, V codes; 2, 3: K, V scales
  const std::size_t bytes = static_cast<std::size_t>(kKvHeads) * (what < 2 ? RecordCodeBytes(pool.fmt) : RecordScaleBytes(pool.fmt, what - 2));
  std::uint8_t* base = what == 0   ? pool.kcodes
                       : what == 1 ? pool.vcodes
                                   : reinterpret_cast<std::uint8_t*>(what == 2 ? pool.kscales : pool.vscales);
  const uint4* from = reinterpret_cast<const uint4*>(base + (static_cast<std::size_t>(layer) * pool.num_pages + src) * bytes);
  uint4* to = reinterpret_cast<uint4*>(base + (static_cast<std::size_t>(layer) * pool.num_pages + dst) * bytes);
  for (std::size_t i = static_cast<std::size_t>(blockIdx.z) * 256 + threadIdx.x; i < bytes / 16; i += 256ULL * gridDim.z) to[i] = from[i];
}

int SelectSmem(int n_cache) { return 4 * (kHistCopies * kHistStride + n_cache); }

template <int kFmt>
cudaError_t LaunchWeights(const DecodeLaunch& a, float* weights, long long weights_stride, cudaStream_t stream) {
  return LaunchChained(AttnWeightsKernel<kFmt>, a.n_units, kWeightThreads, WeightSmem<kFmt>::kBytes, stream, *a.kmap, a.pool, a.layer,
                       a.tables_dev, a.table_stride, a.units_dev, a.items_dev, static_cast<const __half*>(a.q_dev), a.scale_log2,
                       a.partial_ml, weights, weights_stride, a.status_dev);
}

}  // namespace

cudaError_t ConfigureEvictKernels() {
  cudaError_t e = cudaFuncSetAttribute(AttnWeightsKernel<kFmtF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, WeightSmem<kFmtF16>::kBytes);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(AttnWeightsKernel<kFmtQ8>, cudaFuncAttributeMaxDynamicSharedMemorySize, WeightSmem<kFmtQ8>::kBytes);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(AttnWeightsKernel<kFmtQ4>, cudaFuncAttributeMaxDynamicSharedMemorySize, WeightSmem<kFmtQ4>::kBytes);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(EvictSelectKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SelectSmem(kSelectCache));
  return e;
}

cudaError_t LaunchAttnWeights(const DecodeLaunch& a, float* weights, long long weights_stride, cudaStream_t stream) {
  if (a.n_units <= 0) return cudaSuccess;
  if (a.pool.fmt == kFmtF16) return LaunchWeights<kFmtF16>(a, weights, weights_stride, stream);
  return a.pool.fmt == kFmtQ8 ? LaunchWeights<kFmtQ8>(a, weights, weights_stride, stream)
                              : LaunchWeights<kFmtQ4>(a, weights, weights_stride, stream);
}

cudaError_t LaunchEvict(const EvictLaunch& a, cudaStream_t stream) {
  if (a.n_seqs <= 0) return cudaSuccess;
  const dim3 per_row(static_cast<unsigned>(a.n_seqs), static_cast<unsigned>(a.pool.kv_head_count), static_cast<unsigned>(a.pool.n_layers));
  // words of the keys in shared memory, as many as the longest sequence has (what does not fit is read again per pass)
  const int n_cache = std::min(a.max_keys, kSelectCache);
  cudaError_t e = LaunchChained(EvictSelectKernel, per_row, kSelectThreads, SelectSmem(n_cache), stream, a.seqs_dev,
                                a.n_seqs, a.pool.kv_head_begin, a.n_keep, a.n_sink, a.n_recent, a.weights, a.weights_stride,
                                a.layer_stride, n_cache, a.kept);
  if (e != cudaSuccess) return e;
  const dim3 grid(per_row.x, 2 * per_row.y, per_row.z);
  const auto move = a.pool.fmt == kFmtF16 ? EvictMoveKernel<kFmtF16> : a.pool.fmt == kFmtQ8 ? EvictMoveKernel<kFmtQ8> : EvictMoveKernel<kFmtQ4>;
  return LaunchChained(move, grid, kMoveThreads, 0, stream, a.pool, a.tables_dev, a.table_stride, a.seqs_dev, a.n_seqs,
                       a.dst_pages_dev, a.n_keep, a.kept);
}

cudaError_t LaunchCopyPage(const PoolView& pool, int src, int dst, cudaStream_t stream) {
  return LaunchChained(CopyPageKernel, dim3(static_cast<unsigned>(pool.n_layers), 4, 4), 256, 0, stream, pool, src, dst);
}

}  // namespace yahkv
