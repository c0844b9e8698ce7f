// Device code of the routing scan that more than one translation unit uses: the mask bytes of a thread as
// bits and the block-wide scan of visual counts.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace ffnk {

constexpr int kRouteThreads = 256;
constexpr int kRoutePerThread = 32;                             // two 128-bit loads of mask bytes
constexpr int kRouteTile = kRouteThreads * kRoutePerThread;     // 8192 tokens per tile

// The 32 mask bytes of one thread as a bit mask (bit i = token base + i is visual), how many of
// the 32 tokens exist, and how many runs start among them (a token whose modality differs from its
// predecessor's; token 0 always).
struct ThreadTokens {
  uint32_t bits;
  int valid;
  int nruns;
};

// 32 mask bytes (eight words) -> 32 bits.  Four bytes at a time: the high bit of every non-zero byte, then
// one multiply that lines the bits of positions 0, 8, 16, 24 up at 24..27 (no two partial products share
// a bit position).
__device__ __forceinline__ uint32_t mask_words_to_bits(const uint32_t (&w)[kRoutePerThread / 4]) {
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < kRoutePerThread / 4; ++i) {
    const uint32_t nz = (((w[i] & 0x7F7F7F7Fu) + 0x7F7F7F7Fu) | w[i]) & 0x80808080u;
    bits |= ((((nz >> 7) * 0x01020408u) >> 24) & 0xFu) << (4 * i);
  }
  return bits;
}

__device__ __forceinline__ ThreadTokens load_thread_tokens(const uint8_t* __restrict__ mask, int M, int base) {
  uint32_t w[kRoutePerThread / 4] = {};
  int valid = M - base;
  valid = valid < 0 ? 0 : (valid > kRoutePerThread ? kRoutePerThread : valid);
  if (valid == kRoutePerThread && ((reinterpret_cast<uintptr_t>(mask) & 15) == 0)) {
    const uint4 v0 = *reinterpret_cast<const uint4*>(mask + base);
    const uint4 v1 = *reinterpret_cast<const uint4*>(mask + base + 16);
    w[0] = v0.x; w[1] = v0.y; w[2] = v0.z; w[3] = v0.w;
    w[4] = v1.x; w[5] = v1.y; w[6] = v1.z; w[7] = v1.w;
  } else {
#pragma unroll    // fully unrolled: the words stay in registers
    for (int i = 0; i < kRoutePerThread; ++i)
      if (i < valid) w[i >> 2] |= static_cast<uint32_t>(mask[base + i]) << (8 * (i & 3));
  }
  ThreadTokens t;
  t.bits = mask_words_to_bits(w);
  t.valid = valid;
  t.nruns = 0;
  if (valid > 0) {
    const uint32_t prev = base > 0 ? (mask[base - 1] != 0 ? 1u : 0u) : ((t.bits & 1u) ^ 1u);
    const uint32_t vmask = valid == 32 ? 0xFFFFFFFFu : ((1u << valid) - 1u);
    t.nruns = __popc((t.bits ^ ((t.bits << 1) | prev)) & vmask);
  }
  return t;
}

// Block-wide scan of the per-thread visual counts.  Returns the number of visual tokens before
// this thread inside the tile; *tile_v = visual tokens of the tile.  Contains one __syncthreads().
__device__ __forceinline__ int block_exclusive_scan(int nv, int* s_warp, int* tile_v) {
  const int tid = threadIdx.x;
  int incl = nv;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int n = __shfl_up_sync(0xFFFFFFFFu, incl, o);
    if ((tid & 31) >= o) incl += n;
  }
  if ((tid & 31) == 31) s_warp[tid >> 5] = incl;
  __syncthreads();
  int warp_off = 0, total = 0;
#pragma unroll
  for (int i = 0; i < kRouteThreads / 32; ++i) {
    const int c = s_warp[i];
    if (i < (tid >> 5)) warp_off += c;
    total += c;
  }
  *tile_v = total;
  return warp_off + incl - nv;
}

}  // namespace ffnk
