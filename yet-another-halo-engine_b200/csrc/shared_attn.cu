// Decode attention over a prefix that the rows of a batch share: the prefix pass, computed once for all of a group's
// rows, and the combine that joins it with what every row has behind the prefix.
//
// With K = [K_p; K_b] (prefix; the row's own suffix) a row's attention is the join of two softmax partials,
//   o = (2^(m_p - M) A_p + 2^(m_b - M) A_b) / (2^(m_p - M) l_p + 2^(m_b - M) l_b),   A = sum_i 2^(s_i - m) v_i,
// and for the prefix the rows of a group of B sequences x 6 query heads are one [6 B x 256] x [256 x P] product per kv
// head: every cache byte of the prefix is read once per call instead of B times. The suffixes run through the decode
// kernels of the cache formats (one split-K unit list that starts behind the prefix).
//
// SharedPrefixKernel: one CTA pair (a cluster of two on the two SMs of a TPC, tcgen05 cta_group::2) per kv head, 256
// group rows (128 per CTA) and a run of 64-token pages, one page = one key tile. The layout of the prefill kernel's
// pair: Q in tensor memory as the A operand (group row r of the CTA = lane r), S = Q K^T (M 256, N 64, K 256) double-
// buffered in tensor memory, two softmax warpgroups of one thread per row taking alternate tiles, P as fp16 through
// shared memory, O += P V (M 256, N 256, K 64) in 256 tensor-memory columns, S two tiles ahead of P V. No causal mask: a
// shared page is full and visible to every row. Every part leaves its unnormalised accumulator and (max, sum) per row.
//
// Operands. fp16 pages are the operands as they lie in the pool: a page of one kv head is 64 rows of 512 B, and each CTA
// of the pair loads half of it (keys 32 rank .. + 31 of K, dims 128 rank .. + 127 of V) by TMA with 128-byte swizzle,
// no multicast. q8_0 / q4_0 pages are loaded as codes and block scales by eight more warps (two groups taking alternate
// tiles, a tile ahead in registers) which write each CTA's half as the same fp16 tiles: the code is an exact fp16 integer,
// the product with the block's fp16 scale is rounded once to fp16, the values the prefill pass works on too. Rounding
// K and V to 11 bits (the codes have 8 and the scales 11) costs about 2e-4 of an output's size each, as much as the fp16
// rounding of the output itself; exact products would need a second MMA per operand.
//
// What bounds it. fp16 pages: HBM as long as a group has at most 42 rows (a 64-key tile is 64 KB and takes the pair's
// tensor pipes 1,024 clocks whatever the number of rows): 16 rows x 65536 in 53 us with launch and drain = 5.1 TB/s; with
// more rows a second pair re-reads the pages from L2 and the tensor pipe bounds (96 rows x 32768 in 75 us: 0.75 us a tile at
// the 1.6 GHz the power cap leaves, 70 % of the pipe over the whole kernel, 6 us of it prologue and epilogue). Quantized
// pages: a tile takes 0.9 us for any number of rows, two thirds of it tensor time (16 x 65536 of q4_0 57 us, 96 x 32768
// 80); with the conversion's stores left out it takes 0.79, and eight more instructions per 16 bytes cost a tenth.
//
// Why pairs. Single CTAs of 128 rows double the bytes that an SM converts or fetches per tile, and the parts that the
// combine joins. They are a little faster for groups of at most 21 rows, whose second CTA has no rows (21 x 262144 of
// q8_0: 166 us against 204; 16 x 65536: 53 against 57, but the combine 14 against 10) and slower for all others (64 x
// 32768 of q8_0: 75 us against 59, 42 x 65536 of fp16: 77 against 57).
#include <cuda_fp16.h>

#include <cmath>
#include <type_traits>

#include "kernels.cuh"
#include "ptx.cuh"
#include "umma.cuh"

namespace yahkv {
namespace {

constexpr int kTileM = kPrefillTileRows;   // 128 group rows per CTA, 256 per pair
constexpr int kTileN = kPageTokens;        // keys per tile: one page
constexpr int kSoftmaxThreads = 256;       // warps 0-7: two warpgroups of one thread per row
constexpr int kWarpTma = 8, kWarpMma = 9;
constexpr int kDequantWarps = 4;           // per group; warps 10-17 are two groups, quantized pages only
constexpr int kDequantGroups = 2;          // tiles alternate between them
constexpr int kWarpDequant = 10;
constexpr int kKHalfBytes = (kTileN / 2) * kHeadDim * 2;   // fp16 half tiles, 16 KB each
constexpr int kVHalfBytes = kTileN * (kHeadDim / 2) * 2;
constexpr int kKBlockBytes = (kTileN / 2) * 128;           // one [32 keys][64 dims] box
constexpr int kVBlockBytes = kTileN * 128;                 // one [64 keys][64 dims] box
constexpr int kPBytes = kTileM * kTileN * 2;
constexpr int kTmemCols = 512, kColS = 0, kColO = 128, kColQ = 384;   // S 2 x 64, O 256, Q 128 columns
constexpr float kLazyRescale = 8.0F;
constexpr int kStatusAbort = 5;
constexpr int kOutPitch = kHeadDim * 4 + 16;   // an output row in shared memory: four banks further per row
constexpr int kMaxStages = 5;

template <int kFmt>
struct Shape {
  static constexpr bool kQuant = kFmt != kFmtF16;
  // fp16 half tiles of K and of V in flight, each with barriers of its own: S runs two tiles ahead of P V, so K is done
  // with long before V is, and the stage of K(j + 3) must not wait for P(j) V(j) (one ring for both: the conversion of a
  // tile and its products took turns, 3,500 clocks per q4_0 tile against 2,400 with two)
  static constexpr int kKStages = kQuant ? 3 : 5;
  static constexpr int kVStages = kQuant ? 4 : 5;
  static constexpr int kThreads = kSoftmaxThreads + 64 + (kQuant ? 32 * kDequantWarps * kDequantGroups : 0);
  static constexpr int kSmemK = 0;
  static constexpr int kSmemV = kSmemK + kKStages * kKHalfBytes;
  static constexpr int kSmemP = kSmemV + kVStages * kVHalfBytes;
  static constexpr int kSmemBars = kSmemP + 2 * kPBytes;
  static_assert(kTileM * kOutPitch <= kSmemBars, "the output rows take the place of the tiles");
  static constexpr int kBarBytes = 512;
  static constexpr int kBytes = kSmemBars + kBarBytes + 3 * kTileM * 4;   // barriers, then the max / sum exchange
  static_assert(kBytes <= 232448, "shared memory of one CTA");
};

// As in the prefill kernel: "leader" barriers are used in CTA 0 of the pair only, "both" are waited on by each CTA on
// its own copy, "local" inside one CTA.
struct SharedBars {
  std::uint64_t q_full;                  // leader: softmax warps of both CTAs -> MMA
  std::uint64_t k_full[kMaxStages];      // leader: TMA (fp16 pages) or the dequantizing warps of both CTAs -> MMA
  std::uint64_t v_full[kMaxStages];
  std::uint64_t k_empty[kMaxStages];     // both: MMA -> the stage's writer: S(j) is complete
  std::uint64_t v_empty[kMaxStages];     // both: P(j) V(j) is complete
  std::uint64_t s_full[2];               // both
  std::uint64_t s_free[2];               // leader
  std::uint64_t p_full[2];               // leader
  std::uint64_t m_posted[2];             // local
  std::uint64_t pv_done[2];              // both
  std::uint64_t o_done;                  // both
  std::uint32_t tmem_base;
  int abort_flag;
  int converted[2];                      // local: per group of dequantizing warps, tiles up to this one are converted
};

// Eight values of a row as fp16: exact integer codes times the block scale, one rounding. kLimit: a product that the
// rounded scale takes beyond fp16 (127 x 516 for a block of 65,504) is the largest number, not infinity; with a scale that
// is no number it is none either. Asked for only where a scale has all of kLimitBits, as every one has that is large enough
// (limiting all of them: 72 us instead of 66 for 16 rows x 65536 of q4_0).
template <int kFmt>
constexpr std::uint32_t kLimitBits = kFmt == kFmtQ8 ? 0x6000U : 0x7000U;   // 512 (codes to -128) and 8192 (to -8) as fp16
template <bool kLimit>
__device__ __forceinline__ uint4 ScaleCodes(const std::uint32_t (&h)[4], std::uint16_t scale) {
  const __half2 d = __half2half2(__ushort_as_half(scale));
  const __half2 most = __half2half2(__ushort_as_half((scale & 0x7FFFU) < 0x7C00U ? 0x7BFF : 0x7C00));
  uint4 o;
  std::uint32_t* w = &o.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&h[i]), d);
    if (kLimit) v = __hmax2_nan(__hmin2_nan(v, most), __hneg2(most));
    w[i] = *reinterpret_cast<const std::uint32_t*>(&v);
  }
  return o;
}
// Four bytes u = code + 128 -> fp16 pairs (0, 1), (2, 3) of the codes: 0x6400 | u is 1024 + u.
__device__ __forceinline__ void Bytes4ToHalf2(std::uint32_t u, std::uint32_t& h01, std::uint32_t& h23) {
  const std::uint32_t a = __byte_perm(u, 0x64646464U, 0x4140), b = __byte_perm(u, 0x64646464U, 0x4342);
  const __half2 bias = __half2half2(__ushort_as_half(0x6480));   // 1152
  const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), bias), y = __hsub2(*reinterpret_cast<const __half2*>(&b), bias);
  h01 = *reinterpret_cast<const std::uint32_t*>(&x), h23 = *reinterpret_cast<const std::uint32_t*>(&y);
}
// Four bytes holding 0 .. 15 -> fp16 pairs of n - 8.
__device__ __forceinline__ void Nibs4ToHalf2(std::uint32_t n, std::uint32_t& h01, std::uint32_t& h23) {
  const std::uint32_t a = __byte_perm(n, 0x64646464U, 0x4140), b = __byte_perm(n, 0x64646464U, 0x4342);
  const __half2 bias = __half2half2(__ushort_as_half(0x6408));   // 1032
  const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), bias), y = __hsub2(*reinterpret_cast<const __half2*>(&b), bias);
  h01 = *reinterpret_cast<const std::uint32_t*>(&x), h23 = *reinterpret_cast<const std::uint32_t*>(&y);
}
// What a dequantizing thread takes of a row at a time, one load and one block scale: 16 dims = two chunks of 8, 16 bytes of
// fp16 each. Item m of q8_0: 16 bytes of codes, chunks 2 m and 2 m + 1. Of q4_0: 8 bytes, whose low nibbles are chunk
// 4 (m / 2) + m % 2 and whose high nibbles are two chunks further (elements 0-15 of a block are the low nibbles of its
// 16 bytes). (A chunk at a time, with a load and a scale each: 67 us a call against 66 for 16 rows x 65536 of q4_0.)
template <int kFmt>
struct Item;
template <>
struct Item<kFmtQ8> {
  using Codes = uint4;
  static constexpr int kBytes = 16, kSecond = 1;   // of codes; chunks from the first to the second
  static __device__ __forceinline__ int First(int m) { return 2 * m; }
};
template <>
struct Item<kFmtQ4> {
  using Codes = uint2;
  static constexpr int kBytes = 8, kSecond = 2;
  static __device__ __forceinline__ int First(int m) { return 4 * (m >> 1) + (m & 1); }
};
template <bool kFlipped, bool kLimit>   // kFlipped: the bytes are code + 128 already
__device__ __forceinline__ void DequantItem(const uint4& codes, std::uint16_t scale, uint4 (&out)[2]) {
  const std::uint32_t flip = kFlipped ? 0U : kQ8FlipWord;
  std::uint32_t h[4];
  Bytes4ToHalf2(codes.x ^ flip, h[0], h[1]);
  Bytes4ToHalf2(codes.y ^ flip, h[2], h[3]);
  out[0] = ScaleCodes<kLimit>(h, scale);
  Bytes4ToHalf2(codes.z ^ flip, h[0], h[1]);
  Bytes4ToHalf2(codes.w ^ flip, h[2], h[3]);
  out[1] = ScaleCodes<kLimit>(h, scale);
}
template <bool kFlipped, bool kLimit>
__device__ __forceinline__ void DequantItem(const uint2& codes, std::uint16_t scale, uint4 (&out)[2]) {
  std::uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    Nibs4ToHalf2((codes.x >> (4 * i)) & 0x0F0F0F0FU, h[0], h[1]);
    Nibs4ToHalf2((codes.y >> (4 * i)) & 0x0F0F0F0FU, h[2], h[3]);
    out[i] = ScaleCodes<kLimit>(h, scale);
  }
}

// Codes that are read once: past L1.
__device__ __forceinline__ void LoadStream(const std::uint8_t* p, uint2& v) {
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
}
__device__ __forceinline__ void LoadStream(const std::uint8_t* p, uint4& v) {
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
}

template <int kFmt>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Shape<kFmt>::kThreads, 1)
    SharedPrefixKernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, PoolView pool,
                       int layer, const std::int32_t* __restrict__ tables, int table_stride,
                       const PrefixTile* __restrict__ tiles, const std::int32_t* __restrict__ rows,
                       const __half* __restrict__ q, float scale_log2, float* __restrict__ part_acc,
                       float* __restrict__ part_ml, int* status) {
  using S = Shape<kFmt>;
  extern __shared__ __align__(1024) std::uint8_t smem[];
  SharedBars* bars = reinterpret_cast<SharedBars*>(smem + S::kSmemBars);
  static_assert(sizeof(SharedBars) <= S::kBarBytes, "the max / sum exchange follows the barriers");
  volatile int* abort_flag = &bars->abort_flag;
  const std::uint32_t rank = ClusterCtaRank();   // 0 = leader: its MMA warp issues for the pair
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if ((SmemAddr(smem) & 1023U) != 0) {   // the same in both CTAs: either both leave or neither does
    ChainedKernelEntryBefore();
    if (threadIdx.x == 0) atomicExch(status, kStatusAbort);
    return;
  }
  // Barriers and tensor memory are set up while the kernels before this one in the stream still run (programmatic
  // dependent launch); nothing of theirs is read before ChainedKernelEntryBefore. The suffix kernel runs beside this one.
  if (threadIdx.x == 0) {
    MbarInit(&bars->q_full, 2 * kSoftmaxThreads / 32);
    for (int s = 0; s < S::kKStages; ++s) {
      MbarInit(&bars->k_full[s], S::kQuant ? 2 * kDequantWarps : 1);
      MbarInit(&bars->k_empty[s], 1);
    }
    for (int s = 0; s < S::kVStages; ++s) {
      MbarInit(&bars->v_full[s], S::kQuant ? 2 * kDequantWarps : 1);
      MbarInit(&bars->v_empty[s], 1);
    }
    for (int g = 0; g < 2; ++g) {
      MbarInit(&bars->s_full[g], 1);
      MbarInit(&bars->s_free[g], 2 * kSoftmaxThreads / 64);
      MbarInit(&bars->p_full[g], 2 * kSoftmaxThreads / 64);
      MbarInit(&bars->m_posted[g], kSoftmaxThreads / 64);
      MbarInit(&bars->pv_done[g], 1);
    }
    MbarInit(&bars->o_done, 1);
    bars->abort_flag = 0;
    bars->converted[0] = bars->converted[1] = 0;
    FenceBarrierInit();
  }
  if (warp == kWarpMma) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(SmemAddr(&bars->tmem_base)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  TcFenceBefore();
  ClusterSync();
  TcFenceAfter();
  const std::uint32_t tmem = bars->tmem_base;
  ChainedKernelEntryBefore();
  const PrefixTile tile = tiles[blockIdx.x];
  const int n_tiles = tile.page_end - tile.page_begin;   // at least one, the same in both CTAs
  const std::int32_t* table = tables + static_cast<std::size_t>(tile.seq) * table_stride + tile.page_begin;

  if (warp == kWarpTma) {
    // ------------------------------ producer of fp16 pages: this CTA's half of every page ------------------------------
    if constexpr (!S::kQuant) {
      const bool elected = ElectOne();
      if (elected) {
        PrefetchTensorMap(&kmap);
        PrefetchTensorMap(&vmap);
      }
      static_assert(S::kKStages == S::kVStages, "one stage index for both");
      constexpr int kRing = S::kKStages;
      bool ok = true;
      int s = 0, issued_k = 0, issued_v = 0;
      std::uint32_t ph = 1;
      std::int32_t next_page = __ldg(table);
      for (int j = 0; j < n_tiles && ok; ++j) {
        const std::int32_t page = min(max(next_page, 0), pool.num_pages - 1);   // never trust a table entry read from memory
        if (j + 1 < n_tiles) next_page = __ldg(table + j + 1);
        const std::size_t rec = (static_cast<std::size_t>(layer) * pool.num_pages + page) * kKvHeads + tile.kvh;
        const int y = static_cast<int>(rec * kPageTokens);
        if (j >= kRing) ok = WaitOrAbort(&bars->k_empty[s], ph, abort_flag);
        if (!ok) break;
        if (elected) {
          const std::uint32_t full = MapToCta(SmemAddr(&bars->k_full[s]), 0);
          if (rank == 0) MbarArriveExpectTx(&bars->k_full[s], 2 * kKHalfBytes);
#pragma unroll
          for (int kb = 0; kb < 4; ++kb)   // keys 32 rank .. + 31, 64 dims per box
            TmaLoad2DPair(smem + S::kSmemK + s * kKHalfBytes + kb * kKBlockBytes, &kmap, kb * 64,
                          y + static_cast<int>(rank) * (kTileN / 2), full);
        }
        issued_k = j + 1;
        if (j >= kRing) ok = WaitOrAbort(&bars->v_empty[s], ph, abort_flag);
        if (!ok) break;
        if (elected) {
          const std::uint32_t full = MapToCta(SmemAddr(&bars->v_full[s]), 0);
          if (rank == 0) MbarArriveExpectTx(&bars->v_full[s], 2 * kVHalfBytes);
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)   // all 64 keys, dims 128 rank + 64 kb .. + 63
            TmaLoad2DPair(smem + S::kSmemV + s * kVHalfBytes + kb * kVBlockBytes, &vmap, (static_cast<int>(rank) * 2 + kb) * 64,
                          y, full);
        }
        issued_v = j + 1;
        if (++s == kRing) s = 0, ph ^= 1U;
      }
      // After a wait that gave up, the copies still in flight get one more bounded wait each (the last fill of a stage
      // says which phase is outstanding), so that none lands in shared memory after the CTA has left it. The bytes of
      // both CTAs are counted on the leader's barriers, and both CTAs meet at the cluster barrier below.
      if (*abort_flag != 0 && rank == 0) {
        for (int x = 0; x < kRing; ++x) {
          const int k_fills = issued_k / kRing + (x < issued_k % kRing ? 1 : 0), v_fills = issued_v / kRing + (x < issued_v % kRing ? 1 : 0);
          if (k_fills > 0) MbarWait(&bars->k_full[x], static_cast<std::uint32_t>(k_fills - 1) & 1U, 20000000ULL);
          if (v_fills > 0) MbarWait(&bars->v_full[x], static_cast<std::uint32_t>(v_fills - 1) & 1U, 20000000ULL);
        }
      }
    } else {
      // Quantized pages are loaded by the dequantizing warps, one tile of theirs ahead; this warp brings the pages after
      // that into L2: the pair's two CTAs a half each, kAhead tiles before they are converted. It follows the counter of
      // converted tiles and no mbarrier: nothing waits for this warp, so a barrier could be two phases ahead of it.
      constexpr int kAhead = 6;
      const bool elected = ElectOne();
      volatile int* converted = bars->converted;
      for (int j = 2; j < n_tiles; ++j) {
        bool ok = true;
        if (const int done = j - kAhead; done >= 0) {
          const std::uint64_t t0 = GlobalTimerNs();
          while (max(converted[0], converted[1]) <= done && ok) ok = *abort_flag == 0 && GlobalTimerNs() - t0 < kWaitLimitNs;
        }
        if (!__all_sync(0xFFFFFFFFU, ok)) break;
        const std::int32_t page = min(max(__ldg(table + j), 0), pool.num_pages - 1);
        const std::size_t row = ((static_cast<std::size_t>(layer) * pool.num_pages + page) * kKvHeads + tile.kvh) * kPageTokens + rank * (kTileN / 2);
        if (elected) {
          PrefetchL2(pool.kcodes + row * CodeBytes(kFmt), (kTileN / 2) * CodeBytes(kFmt));
          PrefetchL2(pool.vcodes + row * CodeBytes(kFmt), (kTileN / 2) * CodeBytes(kFmt));
          PrefetchL2(pool.kscales + row * kBlocksPerRow, (kTileN / 2) * kBlocksPerRow * 2);
          PrefetchL2(pool.vscales + row * kBlocksPerRow, (kTileN / 2) * kBlocksPerRow * 2);
        }
      }
    }
  } else if (warp == kWarpMma) {
    // ------------------------------ MMA issuer (leader CTA only): S(0), S(1), then S(j + 2), P(j) V(j) ------------------------------
    if (rank == 0) {
      const bool elected = ElectOne();
      constexpr std::uint32_t idesc_s = InstrDesc(2 * kTileM, kTileN, false);
      constexpr std::uint32_t idesc_o = InstrDesc(2 * kTileM, kHeadDim, true);
      const std::uint32_t k_lo0 = DescLo(SmemAddr(smem + S::kSmemK), 16);
      const std::uint32_t v_lo0 = DescLo(SmemAddr(smem + S::kSmemV), kVBlockBytes);
      const std::uint32_t p_lo0 = DescLo(SmemAddr(smem + S::kSmemP), 16);
      const std::uint32_t q_col = tmem + kColQ, o_col = tmem + kColO;
      int ks = 0, vs = 0;
      std::uint32_t kph = 0, vph = 0;
      auto issue_s = [&](int j) -> bool {
        if (!WaitOrAbort<true>(&bars->k_full[ks], kph, abort_flag)) return false;
        if (j >= 2 && !WaitOrAbort<true>(&bars->s_free[j & 1], static_cast<std::uint32_t>((j - 2) >> 1) & 1U, abort_flag))
          return false;
        TcFenceAfter();
        const std::uint32_t lo = k_lo0 + ks * (kKHalfBytes >> 4);
        const std::uint32_t s_col = tmem + kColS + (j & 1) * kTileN;
        if (elected) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            UmmaF16Ts2(s_col, q_col + i * 8, lo + (((i >> 2) * kKBlockBytes + (i & 3) * 32) >> 4), idesc_s, i > 0);
          UmmaCommitPair(&bars->s_full[j & 1]);
          UmmaCommitPair(&bars->k_empty[ks]);
        }
        if (++ks == S::kKStages) ks = 0, kph ^= 1U;
        return true;
      };
      auto issue_pv = [&](int j) -> bool {
        if (!WaitOrAbort<true>(&bars->v_full[vs], vph, abort_flag)) return false;
        if (!WaitOrAbort<true>(&bars->p_full[j & 1], static_cast<std::uint32_t>(j >> 1) & 1U, abort_flag)) return false;
        TcFenceAfter();
        const std::uint32_t plo = p_lo0 + (j & 1) * (kPBytes >> 4);
        const std::uint32_t lo = v_lo0 + vs * (kVHalfBytes >> 4);
        if (elected) {
#pragma unroll
          for (int k16 = 0; k16 < kTileN / 16; ++k16)
            UmmaF16Ss2(o_col, plo + k16 * (32 >> 4), lo + k16 * ((16 * 128) >> 4), idesc_o, j > 0 || k16 > 0);
          UmmaCommitPair(&bars->v_empty[vs]);
          UmmaCommitPair(&bars->pv_done[j & 1]);
        }
        if (++vs == S::kVStages) vs = 0, vph ^= 1U;
        return true;
      };
      bool ok = WaitOrAbort<true>(&bars->q_full, 0, abort_flag);
      if (ok && n_tiles > 0) ok = issue_s(0);
      if (ok && n_tiles > 1) ok = issue_s(1);
      for (int j = 0; j < n_tiles && ok; ++j) {
        if (j + 2 < n_tiles) ok = issue_s(j + 2);
        if (ok) ok = issue_pv(j);
      }
      if (ok && elected) UmmaCommitPair(&bars->o_done);
    }
  } else if (S::kQuant && warp >= kWarpDequant) {
    // ------------------------------ dequantizing warps: pages -> fp16 half tiles ------------------------------
    // A group holds the codes of its next tile in registers: they are loaded (past L1) as soon as the tile before has been
    // converted, two tile periods ahead. Staging them in shared memory by TMA first cost 32 KB more of shared-memory
    // traffic per tile and CTA: 60 us against 58 for 16 rows x 65536 of q8_0, 85 against 82 for 96 rows x 32768.
    if constexpr (S::kQuant) {
      using It = Item<kFmt>;
      const int group = (warp - kWarpDequant) / kDequantWarps, w = (warp - kWarpDequant) % kDequantWarps;
      // Items of a thread: K 32 keys x 16 items, key k_key0 + 8 i; V 64 keys x 8 items (this CTA's half row), key
      // v_key0 + 16 i. Eight lanes store four items of two keys at once: chunk c of a key lies at c ^ (key % 8), so the
      // eight fall on different banks with neighbouring keys where an item's chunks are 0, 2, 4, 6 (q8_0), and with
      // keys two apart where they are 0, 1, 4, 5 (q4_0).
      const int kb = (lane >> 2) & 1;
      const int k_key0 = kFmt == kFmtQ8 ? 2 * w + kb : 4 * (w >> 1) + (w & 1) + 2 * kb;   // 0 .. 7 over the group
      const int v_key0 = k_key0 + 8 * (lane >> 4);
      const int km = (lane & 3) | ((lane >> 3) << 2), vm = (lane & 3) | (((lane >> 3) & 1) << 2);
      const int vm_row = static_cast<int>(rank) * 8 + vm;   // the item in its row
      const int kc = It::First(km), vc = It::First(vm);
      typename It::Codes kw[4], vw[4];
      std::uint16_t ksc[4], vsc[4];
      auto row_of = [&](std::int32_t page) -> std::size_t {
        page = min(max(page, 0), pool.num_pages - 1);   // never trust a table entry read from memory
        return ((static_cast<std::size_t>(layer) * pool.num_pages + page) * kKvHeads + tile.kvh) * kPageTokens;
      };
      auto fetch_k = [&](std::size_t row) {
        const std::size_t k_row = row + rank * (kTileN / 2) + k_key0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          LoadStream(pool.kcodes + (k_row + 8 * i) * CodeBytes(kFmt) + km * It::kBytes, kw[i]);
          ksc[i] = __ldg(pool.kscales + (k_row + 8 * i) * kBlocksPerRow + (km >> 1));
        }
      };
      auto fetch_v = [&](std::size_t row) {
        const std::size_t v_row = row + v_key0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          LoadStream(pool.vcodes + (v_row + 16 * i) * CodeBytes(kFmt) + vm_row * It::kBytes, vw[i]);
          vsc[i] = __ldg(pool.vscales + (v_row + 16 * i) * kBlocksPerRow + (vm_row >> 1));
        }
      };
      auto large = [](const std::uint16_t (&sc)[4]) {   // the same answer in the whole warp
        const std::uint32_t bits = static_cast<std::uint32_t>(sc[0]) | sc[1] | sc[2] | sc[3];
        return __any_sync(0xFFFFFFFFU, (bits & kLimitBits<kFmt>) == kLimitBits<kFmt>);
      };
      if (group < n_tiles) {
        const std::size_t row = row_of(__ldg(table + group));
        fetch_k(row);
        fetch_v(row);
      }
      std::int32_t next_page = group + kDequantGroups < n_tiles ? __ldg(table + group + kDequantGroups) : 0;
      for (int j = group; j < n_tiles; j += kDequantGroups) {
        const int ks = j % S::kKStages, vs = j % S::kVStages;
        bool ok = true;
        if (j >= S::kKStages)
          ok = WaitOrAbort<true>(&bars->k_empty[ks], static_cast<std::uint32_t>(j / S::kKStages - 1) & 1U, abort_flag);
        ok = __all_sync(0xFFFFFFFFU, ok);
        if (!ok) break;
        std::uint8_t* kd = smem + S::kSmemK + ks * kKHalfBytes;
        std::uint8_t* vd = smem + S::kSmemV + vs * kVHalfBytes;
        auto convert_k = [&](auto limit) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = k_key0 + 8 * i;
            uint4 o[2];
            DequantItem<false, limit.value>(kw[i], ksc[i], o);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int c = kc + x * It::kSecond;
              *reinterpret_cast<uint4*>(kd + (c >> 3) * kKBlockBytes + key * 128 + (((c & 7) ^ (key & 7)) << 4)) = o[x];
            }
          }
        };
        if (large(ksc)) convert_k(std::true_type());
        else convert_k(std::false_type());
        FenceProxyAsync();   // the tensor core reads the tiles through the async proxy
        __syncwarp();
        if (lane == 0) MbarArriveCluster(MapToCta(SmemAddr(&bars->k_full[ks]), 0));
        if (w == 0 && lane == 0) *const_cast<volatile int*>(&bars->converted[group]) = j + 1;
        const bool more = j + kDequantGroups < n_tiles;
        const std::size_t next_row = row_of(next_page);
        if (more) fetch_k(next_row);
        if (j >= S::kVStages) ok = WaitOrAbort<true>(&bars->v_empty[vs], static_cast<std::uint32_t>(j / S::kVStages - 1) & 1U, abort_flag);
        ok = __all_sync(0xFFFFFFFFU, ok);
        if (!ok) break;
        auto convert_v = [&](auto limit) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = v_key0 + 16 * i;
            uint4 o[2];
            DequantItem<true, limit.value>(vw[i], vsc[i], o);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int c = vc + x * It::kSecond;
              *reinterpret_cast<uint4*>(vd + (c >> 3) * kVBlockBytes + key * 128 + (((c & 7) ^ (key & 7)) << 4)) = o[x];
            }
          }
        };
        if (large(vsc)) convert_v(std::true_type());
        else convert_v(std::false_type());
        FenceProxyAsync();
        __syncwarp();
        if (lane == 0) MbarArriveCluster(MapToCta(SmemAddr(&bars->v_full[vs]), 0));
        if (more) fetch_v(next_row);
        if (j + 2 * kDequantGroups < n_tiles) next_page = __ldg(table + j + 2 * kDequantGroups);
      }
    }
  } else if (warp < kWarpTma) {
    // ------------------ softmax, correction, epilogue: two warpgroups of one thread per group row ------------------
    const int r = threadIdx.x & (kTileM - 1);
    const int hc = threadIdx.x >> 7;
    const std::uint32_t lane_addr = tmem + (static_cast<std::uint32_t>((warp & 3) * 32) << 16);
    const bool valid = r < tile.n_rows;
    {   // this thread's 128 dims of the row's query -> tensor memory; rows past the group are zero
      const int gr = tile.row0 + (valid ? r : 0);
      const std::int32_t b = valid ? __ldg(rows + tile.row_list + gr / kGroup) : 0;
      const uint4* src = reinterpret_cast<const uint4*>(
          q + (static_cast<std::size_t>(b) * kQHeads + tile.kvh * kGroup + gr % kGroup) * kHeadDim + hc * (kHeadDim / 2));
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        std::uint32_t qr[32];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint4 v = valid ? __ldg(src + part * 8 + i) : make_uint4(0, 0, 0, 0);
          qr[4 * i] = v.x, qr[4 * i + 1] = v.y, qr[4 * i + 2] = v.z, qr[4 * i + 3] = v.w;
        }
        TmemSt32(lane_addr + kColQ + hc * 64 + part * 32, qr);
      }
      TmemWaitSt();
      TcFenceBefore();
      __syncwarp();
      if (lane == 0) MbarArriveCluster(MapToCta(SmemAddr(&bars->q_full), 0));
    }
    // Tiles alternate between the two warpgroups; the reference maximum travels from the group of tile j to the group
    // of tile j + 1 through shared memory, each group keeps its own partial row sum.
    float m_mine = -INFINITY, l_mine = 0.0F;
    float* mref = reinterpret_cast<float*>(smem + S::kSmemBars + S::kBarBytes);   // [128 rows]
    bool ok = true;
    for (int j = hc; j < n_tiles; j += 2) {
      ok = WaitOrAbort(&bars->s_full[hc], static_cast<std::uint32_t>(j >> 1) & 1U, abort_flag);
      ok = __all_sync(0xFFFFFFFFU, ok);
      if (!ok) break;
      TcFenceAfter();
      std::uint32_t sraw[64];
      TmemLd32(lane_addr + kColS + hc * kTileN, *reinterpret_cast<std::uint32_t(*)[32]>(&sraw[0]));
      TmemLd32(lane_addr + kColS + hc * kTileN + 32, *reinterpret_cast<std::uint32_t(*)[32]>(&sraw[32]));
      TmemWaitLd();
      TcFenceBefore();
      __syncwarp();
      if (lane == 0) MbarArriveCluster(MapToCta(SmemAddr(&bars->s_free[hc]), 0));
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < kTileN; ++c) mx[c & 3] = fmaxf(mx[c & 3], __uint_as_float(sraw[c]));
      const float tmax = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale_log2;   // log2 units from here on
      float m_ref = -INFINITY;
      if (j >= 1) {
        ok = WaitOrAbort(&bars->m_posted[hc ^ 1], static_cast<std::uint32_t>((j - 1) >> 1) & 1U, abort_flag);
        ok = __all_sync(0xFFFFFFFFU, ok);
        if (!ok) break;
        m_ref = mref[r];
      }
      if (m_mine != m_ref) {
        l_mine *= Exp2Fast(m_mine - m_ref);
        m_mine = m_ref;
      }
      const bool need = tmax > m_ref + kLazyRescale;
      if (__any_sync(0xFFFFFFFFU, need)) {
        if (j >= 1) {   // O may be rescaled only once P(j-1) V(j-1) has completed
          ok = WaitOrAbort(&bars->pv_done[hc ^ 1], static_cast<std::uint32_t>((j - 1) >> 1) & 1U, abort_flag);
          ok = __all_sync(0xFFFFFFFFU, ok);
          if (!ok) break;
          TcFenceAfter();
        }
        const float m_new = need ? tmax : m_ref;
        const float alpha = m_new == -INFINITY ? 1.0F : Exp2Fast(m_ref - m_new);
        m_mine = m_ref = m_new;
        l_mine *= alpha;
        if (j >= 1) {
#pragma unroll 1
          for (int c0 = 0; c0 < kHeadDim; c0 += 16) {   // 16 columns at a time: the 64 scores stay in registers
            std::uint32_t o[16];
            TmemLd16(lane_addr + kColO + c0, o);
            TmemWaitLd();
#pragma unroll
            for (int c = 0; c < 16; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * alpha);
            TmemSt16(lane_addr + kColO + c0, o);
          }
          TmemWaitSt();
        }
      }
      mref[r] = m_ref;
      __syncwarp();
      if (lane == 0) MbarArrive(&bars->m_posted[hc]);
      const float neg_m = m_ref == -INFINITY ? 0.0F : -m_ref;
      float ls[4] = {0.0F, 0.0F, 0.0F, 0.0F};
      std::uint32_t pk[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const float p0 = Exp2Fast(fmaf(__uint_as_float(sraw[2 * i]), scale_log2, neg_m));
        const float p1 = Exp2Fast(fmaf(__uint_as_float(sraw[2 * i + 1]), scale_log2, neg_m));
        ls[i & 3] += p0 + p1;
        const __half2 h = __floats2half2_rn(p0, p1);
        pk[i] = *reinterpret_cast<const std::uint32_t*>(&h);
      }
      l_mine += (ls[0] + ls[1]) + (ls[2] + ls[3]);
      if (j >= 2) {
        ok = WaitOrAbort(&bars->pv_done[hc], static_cast<std::uint32_t>((j - 2) >> 1) & 1U, abort_flag);
        ok = __all_sync(0xFFFFFFFFU, ok);
        if (!ok) break;
      }
      {
        std::uint8_t* prow = smem + S::kSmemP + hc * kPBytes + (r >> 3) * 1024 + (r & 7) * 128;
#pragma unroll
        for (int c = 0; c < 8; ++c)
          *reinterpret_cast<uint4*>(prow + ((c ^ (r & 7)) << 4)) = make_uint4(pk[4 * c], pk[4 * c + 1], pk[4 * c + 2], pk[4 * c + 3]);
      }
      FenceProxyAsync();
      TcFenceBefore();
      __syncwarp();
      if (lane == 0) MbarArriveCluster(MapToCta(SmemAddr(&bars->p_full[hc]), 0));
    }
    // ---- epilogue: the part's unnormalised rows and their (max, sum) ----
    if (ok && n_tiles > 0) {
      ok = WaitOrAbort(&bars->o_done, 0, abort_flag);
      ok = __all_sync(0xFFFFFFFFU, ok);
    }
    float* xsum = mref + kTileM;   // [2 groups][128 rows]
    NamedBarrierSync(1, kSoftmaxThreads);
    if (n_tiles > 0) {
      const float m_fin = mref[r];
      if (m_mine != m_fin) l_mine *= Exp2Fast(m_mine - m_fin);
    }
    xsum[hc * kTileM + r] = l_mine;
    NamedBarrierSync(1, kSoftmaxThreads);
    if (ok && n_tiles > 0) {
      TcFenceAfter();
      // The rows go through shared memory (the tiles have been read) and out as bulk copies, a thread its own 512 B: a
      // thread's 16-byte stores would hit 32 lines per instruction.
      const std::size_t row = static_cast<std::size_t>(tile.part_row0) + r;
      if (hc == 0 && valid) *reinterpret_cast<float2*>(part_ml + 2 * row) = make_float2(mref[r], l_mine + xsum[kTileM + r]);
      std::uint8_t* mine = smem + r * kOutPitch + hc * (kHeadDim / 2) * 4;
#pragma unroll 1
      for (int c0 = 0; c0 < kHeadDim / 2; c0 += 32) {
        std::uint32_t o[32];
        TmemLd32(lane_addr + kColO + hc * (kHeadDim / 2) + c0, o);
        TmemWaitLd();
#pragma unroll
        for (int c = 0; c < 8; ++c)
          *reinterpret_cast<uint4*>(mine + (c0 + 4 * c) * 4) = make_uint4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
      }
      FenceProxyAsync();
      if (valid) {
        BulkStore(part_acc + row * kHeadDim + hc * (kHeadDim / 2), mine, (kHeadDim / 2) * 4);
        BulkStoreWait();
      }
    }
  }
  // ---- teardown: every role of both CTAs arrives here, also after an abort ----
  TcFenceBefore();
  ClusterSync();
  if (threadIdx.x == 0 && bars->abort_flag != 0) atomicExch(status, kStatusAbort);
  if (warp == kWarpMma) {
    TcFenceAfter();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

// Joins the prefix parts and the suffix units of one (batch row, query head), prefix first, each in order:
// out = (sum w_i A_i) / (sum w_i l_i) * sigmoid(gate), w_i = 2^(m_i - M). Two warps per head, half of the output dims
// each: lane i weighs partials i, i + 32, ... and holds four dims, so nothing is exchanged but by shuffles. The merge is
// latency-bound, so the first rows are fetched before their weights are known. (A CTA per head with its barriers: 12 us
// on 96 rows of nine partials against 5.)
constexpr int kCombineWarps = 8;
constexpr int kCombineEarly = 12;
__global__ void __launch_bounds__(32 * kCombineWarps)
    SharedCombineKernel(const PrefixItem* __restrict__ prefix_items, const float* __restrict__ prefix_acc,
                        const float* __restrict__ prefix_ml, const CombineItem* __restrict__ items,
                        const float* __restrict__ partial_acc, const float* __restrict__ partial_ml,
                        const float* __restrict__ gate, void* out, int out_f32, int n_heads) {
  ChainedKernelEntry();
  const int task = blockIdx.x * kCombineWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int head = task >> 1, dim0 = (task & 1) * (kHeadDim / 2) + 4 * lane;
  if (head >= n_heads) return;
  const int b = head / kQHeads, hh = head % kQHeads, kvh = hh / kGroup, j = hh % kGroup;
  const PrefixItem pi = prefix_items[b * kKvHeads + kvh];
  const CombineItem it = items[b * kKvHeads + kvh];
  const int np = pi.n_parts, n = np + it.n_partials;
  if (n <= 0) return;   // a kv head outside the context's range
  auto ml_of = [&](int i) {
    return i < np ? *reinterpret_cast<const float2*>(prefix_ml + 2 * (pi.first + static_cast<std::size_t>(i) * pi.stride + j))
                  : *reinterpret_cast<const float2*>(partial_ml + (static_cast<std::size_t>(it.first_partial) + (i - np)) * kPartialMlFloats + 2 * j);
  };
  auto row_of = [&](int i) {
    return *reinterpret_cast<const float4*>(
        (i < np ? prefix_acc + (pi.first + static_cast<std::size_t>(i) * pi.stride + j) * kHeadDim
                : partial_acc + (static_cast<std::size_t>(it.first_partial) + (i - np)) * kPartialAccFloats + j * kHeadDim) + dim0);
  };
  const float2 first = lane < n ? ml_of(lane) : make_float2(-INFINITY, 0.0F);
  float4 early[kCombineEarly];
#pragma unroll
  for (int i = 0; i < kCombineEarly; ++i)
    if (i < n) early[i] = row_of(i);
  float M = first.x;
  for (int i = lane + 32; i < n; i += 32) M = fmaxf(M, ml_of(i).x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xFFFFFFFFU, M, o));
  float A[4] = {0.0F, 0.0F, 0.0F, 0.0F}, L = 0.0F;
  auto add = [&](float w, float wl, int i, const float4& x) {
    const float wi = __shfl_sync(0xFFFFFFFFU, w, i);
    L += __shfl_sync(0xFFFFFFFFU, wl, i);
    A[0] = fmaf(wi, x.x, A[0]), A[1] = fmaf(wi, x.y, A[1]), A[2] = fmaf(wi, x.z, A[2]), A[3] = fmaf(wi, x.w, A[3]);
  };
  for (int i0 = 0; i0 < n; i0 += 32) {
    const float2 ml = i0 == 0 ? first : i0 + lane < n ? ml_of(i0 + lane) : make_float2(-INFINITY, 0.0F);
    const float w = ml.x == -INFINITY ? 0.0F : Exp2Fast(ml.x - M);
    const float wl = w * ml.y;
    const int m = min(n - i0, 32);
    int i = 0;
    if (i0 == 0) {
#pragma unroll
      for (; i < kCombineEarly; ++i)
        if (i < m) add(w, wl, i, early[i]);
    }
#pragma unroll 8
    for (; i < m; ++i) add(w, wl, i, row_of(i0 + i));
  }
  const float inv = 1.0F / L;
  const std::size_t at = (static_cast<std::size_t>(b) * kQHeads + hh) * kHeadDim + dim0;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    float o = A[c] * inv;
    if (gate != nullptr) o *= 1.0F / (1.0F + expf(-gate[at + c]));
    if (out_f32)
      static_cast<float*>(out)[at + c] = o;
    else
      static_cast<__half*>(out)[at + c] = __float2half_rn(o);
  }
}

template <int kFmt>
cudaError_t Configure(int* pairs) {
  cudaError_t e = cudaFuncSetAttribute(SharedPrefixKernel<kFmt>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<kFmt>::kBytes);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(2, 1, 1), cfg.blockDim = dim3(Shape<kFmt>::kThreads, 1, 1), cfg.dynamicSmemBytes = Shape<kFmt>::kBytes;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 2, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
  cfg.attrs = &attr, cfg.numAttrs = 1;
  return cudaOccupancyMaxActiveClusters(pairs, SharedPrefixKernel<kFmt>, &cfg);
}

template <int kFmt>
cudaError_t Launch(const DecodeLaunch& a, const SharedLaunch& p, cudaStream_t stream) {
  return LaunchChained(SharedPrefixKernel<kFmt>, p.n_tiles, Shape<kFmt>::kThreads, Shape<kFmt>::kBytes, stream, *p.kmap, *p.vmap,
                       a.pool, a.layer, a.tables_dev, a.table_stride, p.tiles_dev, p.rows_dev,
                       static_cast<const __half*>(a.q_dev), a.scale_log2, p.part_acc, p.part_ml, a.status_dev);
}

}  // namespace

cudaError_t ConfigureSharedKernels(int fmt, int* max_active_pairs) {
  if (cudaError_t e = LoadKernels(SharedCombineKernel); e != cudaSuccess) return e;
  return fmt == kFmtF16  ? Configure<kFmtF16>(max_active_pairs)
         : fmt == kFmtQ8 ? Configure<kFmtQ8>(max_active_pairs)
                         : Configure<kFmtQ4>(max_active_pairs);
}

cudaError_t LaunchSharedPrefix(const DecodeLaunch& a, const SharedLaunch& p, cudaStream_t stream) {
  if (p.n_tiles <= 0) return cudaSuccess;
  if ((p.n_tiles & 1) != 0) return cudaErrorInvalidValue;   // tiles come as pairs, one cluster each
  if (a.pool.fmt == kFmtF16) return Launch<kFmtF16>(a, p, stream);
  return a.pool.fmt == kFmtQ8 ? Launch<kFmtQ8>(a, p, stream) : Launch<kFmtQ4>(a, p, stream);
}

cudaError_t LaunchSharedCombine(const DecodeLaunch& a, const SharedLaunch& p, cudaStream_t stream) {
  if (a.n_seqs <= 0) return cudaSuccess;
  const int heads = a.n_seqs * kQHeads;
  return LaunchChained(SharedCombineKernel, (2 * heads + kCombineWarps - 1) / kCombineWarps, 32 * kCombineWarps, 0, stream,
                       p.prefix_items_dev, p.part_acc, p.part_ml, a.items_dev, a.partial_acc, a.partial_ml, a.gate_dev, a.out_dev,
                       a.out_f32, heads);
}

}  // namespace yahkv
