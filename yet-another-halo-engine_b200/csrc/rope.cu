// Rotary positions for head rows of 256 dims: any even rotated part, half or interleaved pairs, scaled frequencies,
// optionally behind the head RMS norm, at positions that are device-resident data.
//
// Pair p < R / 2 of a row at position n is turned by n f_p:  (a, b) -> (a c - b s, a s + b c), c + i s = m e^(i n f_p), with
// a, b at dims (p, p + R / 2) or (2p, 2p + 1) and m the scaling's magnitude. The host evaluates e^(i n f_p) in double
// precision for n = 0 .. 1023 and for the multiples of 1024 (times m) and rounds each once to fp32; the kernel multiplies
// the two, e^(i n f) = e^(i 1024 (n / 1024) f) e^(i (n % 1024) f): two roundings more than a full table (a relative 1e-7)
// for a thousandth of its size, so that the angles of a million positions stay in cache. HBM-bound: every row is read and
// written once.
//
// One warp per token and a few of its heads (the angles stay in registers), lane l holding dims 8 l .. 8 l + 7. With
// R / 2 a multiple of 8 the other half of a pair is the same register of another lane (a shuffle); otherwise the row
// goes through shared memory. Interleaved pairs never leave their lane.
#include <cuda_fp16.h>

#include "kernels.cuh"
#include "ptx.cuh"

namespace yahkv {
namespace {

constexpr int kRopeRowWarps = 8;

template <bool kF32>
__device__ __forceinline__ void LoadRow8(const void* base, std::size_t at, float (&x)[8]) {
  if constexpr (kF32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + at);
    const float4 a = p[0], b = p[1];
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
    const uint4 raw = *reinterpret_cast<const uint4*>(static_cast<const __half*>(base) + at);
    const __half2* h = reinterpret_cast<const __half2*>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(h[i]);
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
  }
}
template <bool kF32>
__device__ __forceinline__ void StoreRow8(void* base, std::size_t at, const float (&x)[8]) {
  if constexpr (kF32) {
    float4* p = reinterpret_cast<float4*>(static_cast<float*>(base) + at);
    p[0] = make_float4(x[0], x[1], x[2], x[3]), p[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    __half2 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<uint4*>(static_cast<__half*>(base) + at) = *reinterpret_cast<const uint4*>(h);
  }
}

// The angles of this lane's eight dims: cs[j] belongs to dim 8 lane + j. Neighbouring dims are neighbouring pairs (half) or
// share them (interleaved), so a lane's entries are one run of the tables, read 16 bytes at a time where it is aligned.
__device__ __forceinline__ float2 TurnOf(float2 x, float2 y) {
  return make_float2(fmaf(x.x, y.x, -(x.y * y.y)), fmaf(x.x, y.y, x.y * y.x));
}
__device__ __forceinline__ void LaneAngles(const RopeRowsLaunch& a, long long pos, int lane, float2 (&cs)[8]) {
  const int half = a.rotary_dim / 2;
  const float2* hi = a.tab_hi + (pos >> kRopeLowBits) * half;
  const float2* lo = a.tab_lo + (pos & ((1 << kRopeLowBits) - 1)) * half;
  if (a.interleaved) {
    if ((half & 3) == 0 && 8 * lane < a.rotary_dim) {
      const float4* h4 = reinterpret_cast<const float4*>(hi + 4 * lane);
      const float4* l4 = reinterpret_cast<const float4*>(lo + 4 * lane);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4 x = __ldg(h4 + i), y = __ldg(l4 + i);
        cs[4 * i] = cs[4 * i + 1] = TurnOf(make_float2(x.x, x.y), make_float2(y.x, y.y));
        cs[4 * i + 2] = cs[4 * i + 3] = TurnOf(make_float2(x.z, x.w), make_float2(y.z, y.w));
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      cs[2 * i] = make_float2(1.0F, 0.0F);
      if (8 * lane + 2 * i < a.rotary_dim) cs[2 * i] = TurnOf(__ldg(hi + 4 * lane + i), __ldg(lo + 4 * lane + i));
      cs[2 * i + 1] = cs[2 * i];
    }
    return;
  }
  if ((half & 7) == 0 && 8 * lane < a.rotary_dim) {   // the lane's dims lie in one half
    const int p0 = 8 * lane < half ? 8 * lane : 8 * lane - half;
    const float4* h4 = reinterpret_cast<const float4*>(hi + p0);
    const float4* l4 = reinterpret_cast<const float4*>(lo + p0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 x = __ldg(h4 + i), y = __ldg(l4 + i);
      cs[2 * i] = TurnOf(make_float2(x.x, x.y), make_float2(y.x, y.y));
      cs[2 * i + 1] = TurnOf(make_float2(x.z, x.w), make_float2(y.z, y.w));
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int d = 8 * lane + j;
    cs[j] = make_float2(1.0F, 0.0F);
    if (d < a.rotary_dim) {
      const int p = d < half ? d : d - half;
      cs[j] = TurnOf(__ldg(hi + p), __ldg(lo + p));
    }
  }
}

enum PairMode { kInterleavedPairs, kHalfPairs, kAnyPairs };
// The other half of the pairs of this lane's dims.
//   kInterleavedPairs  rotary_dim a multiple of 8: neighbours in the lane
//   kHalfPairs         rotary_dim / 2 a multiple of 8: the same register of the lane rotary_dim / 16 away
//   kAnyPairs          any even rotary_dim, either layout: through shared memory
template <int kMode>
__device__ __forceinline__ void PairOf(const float (&x)[8], float (&other)[8], float* row_s, int half, bool interleaved, int lane) {
  if constexpr (kMode == kInterleavedPairs) {
#pragma unroll
    for (int j = 0; j < 8; ++j) other[j] = x[j ^ 1];
  } else if constexpr (kMode == kHalfPairs) {
    const int src = 8 * lane < half ? lane + half / 8 : lane - half / 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) other[j] = __shfl_sync(0xFFFFFFFFU, x[j], src & 31);
  } else {
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 8; ++j) row_s[8 * lane + j] = x[j];
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int d = 8 * lane + j;
      other[j] = d >= 2 * half ? 0.0F : interleaved ? row_s[d ^ 1] : row_s[d < half ? d + half : d - half];
    }
  }
}

// kHeads rows of one token per warp, all loaded before anything else is waited for. With w the norm weights (or 1) and
// o(d) the other dim of d's pair, out_d = inv (x_d (w_d cos) + x_o (w_o (-/+ sin))): the two products in parentheses are
// made once per token, so a row costs two multiplications and an fma per dim, and the sum of its squares.
template <bool kInF32, bool kOutF32, int kHeads, int kMode>
__global__ void __launch_bounds__(32 * kRopeRowWarps) RopeRowsKernel(const RopeRowsLaunch a) {
  __shared__ float row_s[kRopeRowWarps][kMode == kAnyPairs ? kHeadDim : 1];
  ChainedKernelEntry();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long task = static_cast<long long>(blockIdx.x) * kRopeRowWarps + warp;
  const int head_groups = (a.n_heads + kHeads - 1) / kHeads;
  const long long token = task / head_groups;
  const int h0 = static_cast<int>(task % head_groups) * kHeads;
  if (token >= a.n_tokens) return;
  long long pos = __ldg(a.positions + token);
  const std::size_t x_at = static_cast<std::size_t>(token) * a.x_stride + static_cast<std::size_t>(h0) * kHeadDim + 8 * lane;
  const std::size_t out_at = static_cast<std::size_t>(token) * a.out_stride + static_cast<std::size_t>(h0) * kHeadDim + 8 * lane;
  float x[kHeads][8];
#pragma unroll
  for (int h = 0; h < kHeads; ++h)
    if (h0 + h < a.n_heads) LoadRow8<kInF32>(a.x, x_at + h * kHeadDim, x[h]);
  const int half = a.rotary_dim / 2;
  if (pos < 0 || pos >= a.max_positions) {   // reported, and turned by the nearest angle there is
    if (lane == 0) atomicExch(a.status, kStatusRopePosition);
    pos = pos < 0 ? 0 : a.max_positions - 1;
  }
  float2 cs[8];
  LaneAngles(a, pos, lane, cs);
#pragma unroll
  for (int j = 0; j < 8; ++j)   // the first dim of a pair takes -sin
    if (a.interleaved ? (j & 1) == 0 : 8 * lane + j < half) cs[j].y = -cs[j].y;
  if (a.weight != nullptr) {
    float w[8], wo[8];
    LoadRow8<true>(a.weight, 8 * lane, w);
    PairOf<kMode>(w, wo, row_s[warp], half, a.interleaved, lane);
#pragma unroll
    for (int j = 0; j < 8; ++j) cs[j].x *= w[j], cs[j].y *= wo[j];
  }
  // a dim that is not rotated must not see its neighbour, not even times zero
  const bool turns = 8 * lane < a.rotary_dim;
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
    if (h0 + h >= a.n_heads) break;   // the whole warp at once
    float inv = 1.0F;
    if (a.weight != nullptr) {
      float acc = 0.0F;
#pragma unroll
      for (int j = 0; j < 8; ++j) acc = fmaf(x[h][j], x[h][j], acc);
#pragma unroll
      for (int m = 16; m >= 1; m >>= 1) acc += __shfl_xor_sync(0xFFFFFFFFU, acc, m);
      inv = rsqrtf(fmaf(acc, 1.0F / kHeadDim, a.eps));
    }
    float other[8];
    PairOf<kMode>(x[h], other, row_s[warp], half, a.interleaved, lane);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[h][j] *= cs[j].x;
      if (kMode == kAnyPairs ? 8 * lane + j < a.rotary_dim : turns) x[h][j] = fmaf(other[j], cs[j].y, x[h][j]);
      if (a.weight != nullptr) x[h][j] *= inv;
    }
    StoreRow8<kOutF32>(a.out, out_at + h * kHeadDim, x[h]);
  }
}

template <bool kInF32, bool kOutF32, int kHeads>
auto KernelOf(bool interleaved, int rotary_dim) {
  return interleaved && rotary_dim % 8 == 0      ? RopeRowsKernel<kInF32, kOutF32, kHeads, kInterleavedPairs>
         : !interleaved && rotary_dim % 16 == 0 ? RopeRowsKernel<kInF32, kOutF32, kHeads, kHalfPairs>
                                                : RopeRowsKernel<kInF32, kOutF32, kHeads, kAnyPairs>;
}
template <bool kInF32, bool kOutF32, int kHeads>
cudaError_t Launch(const RopeRowsLaunch& a, cudaStream_t stream) {
  const long long tasks = static_cast<long long>(a.n_tokens) * ((a.n_heads + kHeads - 1) / kHeads);
  const long long grid = (tasks + kRopeRowWarps - 1) / kRopeRowWarps;
  if (grid > 0x7FFFFFFFLL) return cudaErrorInvalidValue;
  return LaunchChained(KernelOf<kInF32, kOutF32, kHeads>(a.interleaved, a.rotary_dim), static_cast<unsigned>(grid), 32 * kRopeRowWarps, 0, stream, a);
}
template <bool kInF32, bool kOutF32>
cudaError_t LaunchHeads(const RopeRowsLaunch& a, cudaStream_t stream) {
  // Few rows: one per warp, so that the call fills the device. Many: four rows of a token share the angles.
  return static_cast<long long>(a.n_tokens) * a.n_heads < 148 * 64 ? Launch<kInF32, kOutF32, 1>(a, stream)
                                                                   : Launch<kInF32, kOutF32, 4>(a, stream);
}

}  // namespace

cudaError_t LoadRopeRows(bool interleaved, int rotary_dim) {
  cudaError_t e = LoadKernels(KernelOf<true, true, 1>(interleaved, rotary_dim), KernelOf<true, true, 4>(interleaved, rotary_dim));
  if (e == cudaSuccess) e = LoadKernels(KernelOf<true, false, 1>(interleaved, rotary_dim), KernelOf<true, false, 4>(interleaved, rotary_dim));
  if (e == cudaSuccess) e = LoadKernels(KernelOf<false, true, 1>(interleaved, rotary_dim), KernelOf<false, true, 4>(interleaved, rotary_dim));
  if (e == cudaSuccess) e = LoadKernels(KernelOf<false, false, 1>(interleaved, rotary_dim), KernelOf<false, false, 4>(interleaved, rotary_dim));
  return e;
}

cudaError_t LaunchRopeRows(const RopeRowsLaunch& a, cudaStream_t stream) {
  if (a.n_tokens <= 0 || a.n_heads <= 0) return cudaSuccess;
  if (a.x_f32) return a.out_f32 ? LaunchHeads<true, true>(a, stream) : LaunchHeads<true, false>(a, stream);
  return a.out_f32 ? LaunchHeads<false, true>(a, stream) : LaunchHeads<false, false>(a, stream);
}

}  // namespace yahkv
