// Attention weights per cached key, and the eviction of keys by them; the page copy of a forked sequence.
//
// AttnWeightsKernel adds to w[key] the softmax weights that the six query heads of a kv head's group gave the key in the
// decode call just made: w[key] += sum_g 2^(s_g - M_g - log2 L_g). The part kernel has kept the scores s_g (log2 units: the
// kScores variants in decode_attn.cu and decode_f16.cu), its partials give M_g and L_g, so the pass
// reads 96 B per key and adds to 16 B. (Reading K again and making the scores anew cost 56 us on a q8_0 batch of 291,000
// keys beside a part kernel of 113; this pass takes 5 and keeping the scores 20, with fp16 pages 3.) No sum depends on the order of CTAs: each key is added to once per call.
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

#include "kernels.cuh"
#include "ptx.cuh"

namespace yahkv {
namespace {

// ----------------------------------------------------------------------------------------------------------------
// attention weights
// ----------------------------------------------------------------------------------------------------------------
constexpr int kWeightThreads = 256;
constexpr int kWeightPages = kWeightThreads / kPageTokens;   // pages per turn, a thread per key

__global__ void __launch_bounds__(kWeightThreads)
    AttnWeightsKernel(const DecodeUnit* __restrict__ units, const CombineItem* __restrict__ items,
                      const float* __restrict__ partial_ml, const float* __restrict__ scores, float* __restrict__ weights,
                      long long weights_stride) {
  __shared__ float norm_s[kGroup];   // M + log2 L per query head
  ChainedKernelEntry();
  const DecodeUnit u = units[blockIdx.x];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n_pages = u.page_end - u.page_begin;
  // the scores of the first turn are on their way while the norms are made
  float s[kGroup];
  auto load = [&](int i) {
    const float* src = scores + (static_cast<std::size_t>(u.pad) + i) * (kGroup * kPageTokens) + threadIdx.x % kPageTokens;
#pragma unroll
    for (int h = 0; h < kGroup; ++h) s[h] = i < n_pages ? src[h * kPageTokens] : -INFINITY;
  };
  int i = threadIdx.x / kPageTokens;
  load(i);
  if (warp < kGroup) {
    const CombineItem it = items[u.batch * kKvHeads + u.kvh];
    const float* ml = partial_ml + static_cast<std::size_t>(it.first_partial) * kPartialMlFloats + 2 * warp;
    float m = -INFINITY, l = 0.0F;
    for (int k = lane; k < it.n_partials; k += 32) m = fmaxf(m, ml[static_cast<std::size_t>(k) * kPartialMlFloats]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFU, m, o));
    for (int k = lane; k < it.n_partials; k += 32) {
      const float mk = ml[static_cast<std::size_t>(k) * kPartialMlFloats];
      l += mk == -INFINITY ? 0.0F : exp2f(mk - m) * ml[static_cast<std::size_t>(k) * kPartialMlFloats + 1];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xFFFFFFFFU, l, o);
    if (lane == 0) norm_s[warp] = m + log2f(l);
  }
  __syncthreads();
  float norm[kGroup];
#pragma unroll
  for (int h = 0; h < kGroup; ++h) norm[h] = norm_s[h];
  float* w_out = weights + (static_cast<std::size_t>(u.seq) * kKvHeads + u.kvh) * static_cast<std::size_t>(weights_stride);
  for (; i < n_pages; i += kWeightPages) {
    float p = 0.0F;
#pragma unroll
    for (int h = 0; h < kGroup; ++h) p += exp2f(s[h] - norm[h]);
    const int key = (u.page_begin + i) * kPageTokens + threadIdx.x % kPageTokens;
    load(i + kWeightPages);
    // one addition per key and call, so the order of CTAs does not matter; nothing waits for it
    if (key < u.n_keys) atomicAdd(w_out + key, p);
  }
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
// 33 us for 128 rows of 14,000 keys against 26.)
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

}  // namespace

cudaError_t ConfigureEvictKernels() {
  const auto e = LoadKernels(AttnWeightsKernel, CopyPageKernel, EvictMoveKernel<kFmtF16>, EvictMoveKernel<kFmtQ8>, EvictMoveKernel<kFmtQ4>);
  if (e != cudaSuccess) return e;
  return cudaFuncSetAttribute(EvictSelectKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SelectSmem(kSelectCache));
}

cudaError_t LaunchAttnWeights(const DecodeLaunch& a, float* weights, long long weights_stride, cudaStream_t stream) {
  if (a.n_units <= 0) return cudaSuccess;
  return LaunchChained(AttnWeightsKernel, a.n_units, kWeightThreads, 0, stream, a.units_dev, a.items_dev, a.partial_ml, a.scores_dev,
                       weights, weights_stride);
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
