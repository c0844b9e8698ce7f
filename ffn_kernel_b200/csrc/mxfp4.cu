// Quantisation to MXFP4 and back (the format: mxfp4.cuh).
//
//   mx_quantize_rows_kernel    x contiguous along the blocks: weights in nn.Linear storage, activations; with
//                              routing lists the rows come out in routed order
//   mx_route_quantize_kernel   routing, the copy into routed order and the quantisation of the activations in one
//                              launch, for masks of up to 32768 tokens
//   mx_quantize_cols_kernel    x contiguous across the blocks: [in, out] weights
//   mx_dequantize_kernel       codes and scales -> bf16 / fp16 / fp32
//
// All are bound by HBM: a value is read once and leaves as 4.25 bits (or the reverse); the arithmetic is an
// integer maximum over 32 values, one product and one conversion instruction per value pair.
#include "ffnk_internal.h"
#include "mxfp4.cuh"
#include "ptx.cuh"
#include "route.cuh"

namespace ffnk {

template <int T> struct MxType;
template <> struct MxType<FFNK_BF16> { using t = __nv_bfloat16; };
template <> struct MxType<FFNK_FP16> { using t = __half; };
template <> struct MxType<FFNK_FP32> { using t = float; };

constexpr int kQuantThreads = 256;
constexpr int kQuantPerSm = 4;        // resident CTAs the row kernels are compiled for
constexpr int kChunksMax = 2;         // warp steps of a row in flight together (for few rows one, on more warps)

// One chunk of a row: the lanes of a block share its maximum by shuffles, each rounds its own values.
template <typename T>
__device__ __forceinline__ void quantize_chunk(const MxRaw& raw, int chunk, int cols, uint8_t* codes_row, uint8_t* scale_row,
                                               int k_atoms, int lane) {
  using L = MxLane<T>;
  uint32_t m = absmax_bits<T>(raw);
#pragma unroll
  for (int o = 1; o < L::lanes_per_block; o <<= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  const uint32_t byte = mx_scale_byte(m);
  const float inv = mx_inverse_scale(byte);
  uint32_t code[L::values / 8];
#pragma unroll
  for (int j = 0; j < L::values / 8; ++j) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = raw_value<T>(raw, 8 * j + i);
    code[j] = mx_round8(v, byte, inv);
  }
  const int c = chunk * L::chunk + lane * L::values;
  if (c < ((cols + 31) & ~31)) {
    if constexpr (L::values == 16) *reinterpret_cast<uint2*>(codes_row + c / 2) = make_uint2(code[0], code[1]);
    else *reinterpret_cast<uint32_t*>(codes_row + c / 2) = code[0];
  }
  const int block = c >> 5;
  if (lane % L::lanes_per_block == 0 && (block >> 2) < k_atoms)
    scale_row[static_cast<int64_t>(block >> 2) * kMxAtomBytes + (block & 3)] = static_cast<uint8_t>(byte);
}

// The rows of one warp, `n` <= kChunksMax chunks from chunk `first` on; the next row's loads are in flight while one
// is rounded.  `row(i)` names the i-th row's source and destination (source < 0: no further row).
struct MxRowRef {
  int src, dst;
};
template <typename T, class Rows>
__device__ __forceinline__ void quantize_rows(const T* x, int64_t ldx, int align, int cols, int first, int n, uint8_t* codes,
                                              uint8_t* scales, int lane, Rows&& row) {
  const int64_t ld = mx_code_ld(cols);
  const int k_atoms = static_cast<int>(mx_k_atoms(cols));
  MxRowRef now = row(0), next = row(1);
  MxRaw raw[kChunksMax];
  auto load = [&](const MxRowRef& r) {
#pragma unroll
    for (int u = 0; u < kChunksMax; ++u)
      if (u < n && r.src >= 0) raw[u] = load_lane(x + r.src * ldx, (first + u) * MxLane<T>::chunk + lane * MxLane<T>::values, cols, align);
  };
  load(now);
  for (int i = 2; now.src >= 0; ++i) {
    MxRaw cur[kChunksMax];
#pragma unroll
    for (int u = 0; u < kChunksMax; ++u) cur[u] = raw[u];
    load(next);
    const MxRowRef after = row(i);
#pragma unroll
    for (int u = 0; u < kChunksMax; ++u)
      if (u < n)                                       // warp-uniform
        quantize_chunk<T>(cur[u], first + u, cols, codes + now.dst * ld, scales + mx_scale_word(now.dst, 0, k_atoms), k_atoms, lane);
    now = next;
    next = after;
  }
}

// blockIdx.y: which group of `per_warp` chunks of every row.
// Plain (perm == nullptr): row r of x -> row r; the scale bytes of the rows that fill the last atom are zeroed.
// Routed: rows in routed order (visual rows first, text rows from the next multiple of 256), none beyond them.
// Measured: 32768 x 4096 bf16 52.6 us = 6.46 TB/s, 0.99 of a plain copy; 11008 x 4096 fp32 32.3 us = 6.32 TB/s.  (Loads of
// one row at a time, without the next row in flight, and 16-byte loads: 78 us; with 64-bit index divisions 118 us.)
template <typename T>
__global__ void __launch_bounds__(kQuantThreads, kQuantPerSm) mx_quantize_rows_kernel(
    const T* __restrict__ x, int64_t ldx, int rows, int cols, const int* __restrict__ perm, const int* __restrict__ counts,
    uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int align, int per_warp) {
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int chunks = (cols + MxLane<T>::chunk - 1) / MxLane<T>::chunk;
  const int first = blockIdx.y * per_warp, n = min(per_warp, chunks - first);
  const int step = gridDim.x * (kQuantThreads / 32);
  const int r0 = blockIdx.x * (kQuantThreads / 32) + (threadIdx.x >> 5);
  if (perm) {
    const int Mv = counts[0], cap = counts[2], text_base = ((Mv + 255) >> 8) << 8;
    quantize_rows(x, ldx, align, cols, first, n, codes, scales, lane, [&](int i) {
      const int64_t r = r0 + static_cast<int64_t>(i) * step;
      if (r >= rows) return MxRowRef{-1, 0};
      const int k = static_cast<int>(r);
      return k < Mv ? MxRowRef{perm[k], k} : MxRowRef{perm[cap + (k - Mv)], text_base + (k - Mv)};
    });
    return;
  }
  quantize_rows(x, ldx, align, cols, first, n, codes, scales, lane, [&](int i) {
    const int64_t r = r0 + static_cast<int64_t>(i) * step;
    return r < rows ? MxRowRef{static_cast<int>(r), static_cast<int>(r)} : MxRowRef{-1, 0};
  });
  // rows that only fill the last atom
  const int k_atoms = static_cast<int>(mx_k_atoms(cols));
  const int a0 = first * (MxLane<T>::chunk / 128), a1 = min(k_atoms, (first + n) * (MxLane<T>::chunk / 128));
  for (int64_t r = rows + r0; r < mx_row_atoms(rows) * 128; r += step)
    for (int a = a0 + lane; a < a1; a += 32) *reinterpret_cast<uint32_t*>(scales + mx_scale_word(r, a, k_atoms)) = 0u;
}

// Routing and quantisation of the activations in one launch (M <= kMxRouteTokens).  Every CTA keeps the whole mask as bits
// with the visual tokens before each word (8 KiB of shared memory), so a warp knows where a token's row goes without any
// list: the tokens are taken in their own order, and each leaves its entry of the lists on the way.  (A compaction of the
// whole mask in every CTA, as for the copy of bf16 rows, was bound by its shared-memory stores: 8192 x 4096 34 us, now
// 20, from cold caches.  A routing kernel and then mx_quantize_rows_kernel take as long from 16384 tokens on, 35 us and
// 68 us at 32768, in three launches.)
// WORDS: words of 32 tokens a thread, consecutive.
constexpr int kMxRouteWords = 4;
constexpr int kMxRouteTokens = kRouteThreads * 32 * kMxRouteWords;
constexpr int kMxBesideTokens = 1024;        // few tokens: the product starts beside this kernel (mx_route_quantize)
template <int WORDS>
__global__ void __launch_bounds__(kRouteThreads, kQuantPerSm) mx_route_quantize_kernel(
    const uint8_t* __restrict__ mask, int M, int cap, int* __restrict__ perm, int* __restrict__ counts,
    const __nv_bfloat16* __restrict__ x, int64_t ldx, int cols, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
    int align, int per_warp) {
  __shared__ uint32_t s_bits[kRouteThreads * WORDS];   // token 32 i + k is visual: bit k of word i
  __shared__ int s_before[kRouteThreads * WORDS];      // visual tokens before word i
  __shared__ int s_warp[kRouteThreads / 32];
  __shared__ int s_runs;
  const int tid = threadIdx.x, lane = tid & 31;
  const bool writer = blockIdx.x == 0 && blockIdx.y == 0;
  griddep_launch_dependents();
  const int words = (M + kRouteThreads * 32 - 1) / (kRouteThreads * 32);
  uint32_t bits[WORDS] = {};
  int count = 0, runs = 0;
#pragma unroll
  for (int w = 0; w < WORDS; ++w) {
    if (w < words) {
      const ThreadTokens tt = load_thread_tokens(mask, M, (tid * words + w) * 32);
      bits[w] = tt.bits;
      count += __popc(tt.bits);
      runs += tt.nruns;
    }
  }
  if (tid == 0) s_runs = 0;
  int Mv = 0;
  int before = block_exclusive_scan(count, s_warp, &Mv);
#pragma unroll
  for (int w = 0; w < WORDS; ++w) {
    if (w < words) {
      s_bits[tid * words + w] = bits[w];
      s_before[tid * words + w] = before;
      before += __popc(bits[w]);
    }
  }
  if (writer) {
    const int wr = __reduce_add_sync(0xFFFFFFFFu, runs);
    if (lane == 0 && wr) atomicAdd(&s_runs, wr);
  }
  __syncthreads();
  if (writer && tid == 0) {
    counts[0] = Mv;
    counts[1] = M - Mv;
    counts[2] = cap;
    counts[3] = M;
    counts[4] = s_runs;
  }
  const int text_base = ((Mv + 255) >> 8) << 8;
  const int chunks = (cols + MxLane<__nv_bfloat16>::chunk - 1) / MxLane<__nv_bfloat16>::chunk;
  const int first = blockIdx.y * per_warp, n = min(per_warp, chunks - first);
  const int step = gridDim.x * (kRouteThreads / 32), r0 = blockIdx.x * (kRouteThreads / 32) + (tid >> 5);
  const bool lists = blockIdx.y == 0 && lane == 0;
  quantize_rows(x, ldx, align, cols, first, n, codes, scales, lane, [&](int i) {
    const int t = r0 + i * step;
    if (t >= M) return MxRowRef{-1, 0};
    const uint32_t word = s_bits[t >> 5];
    const int visual = s_before[t >> 5] + __popc(word & ((1u << (t & 31)) - 1u));
    const bool v = (word >> (t & 31)) & 1u;
    if (lists) perm[v ? visual : cap + (t - visual)] = t;
    return MxRowRef{t, v ? visual : text_base + (t - visual)};
  });
}

// x(r, c) at x[c * ldc + r]: blocks run across the contiguous dimension.  A CTA takes 64 (fp32) or 128 (16-bit types)
// rows x one atom of four blocks; a thread reads the 32 values of one block of one row, or of two neighbouring rows at
// once, so that a warp reads 128 contiguous bytes a column; the codes go through shared memory so that a row leaves as
// 64 contiguous bytes.  `pairs`: the 16-bit columns are 4-byte aligned.
// Bound by HBM once the inner tiles did without a predicate and a 64-bit product a load (uniform column addresses) and the
// maximum is one instruction for two values: 11008 x 4096 fp32 37.9 -> 32.9 us = 6.2 TB/s, bf16 34.5 -> 20.7 us = 5.5 TB/s.
// Four CTAs an SM, for which fp32 spills 8 bytes: three without a spill take 34.3 us where four take 31.5.
template <typename T> struct MxCols {
  static constexpr int per_thread = 4 / sizeof(T);
  static constexpr int rows = 64 * per_thread;
};
template <typename T>
__global__ void __launch_bounds__(kQuantThreads, 4) mx_quantize_cols_kernel(const T* __restrict__ x, int64_t ldc, int64_t rows,
                                                                         int64_t cols, uint8_t* __restrict__ codes,
                                                                         uint8_t* __restrict__ scales, bool pairs) {
  constexpr int P = MxCols<T>::per_thread, R = MxCols<T>::rows;
  __shared__ uint4 s_code[R][5];             // four blocks a row, one piece of padding against bank conflicts
  __shared__ __align__(4) uint8_t s_scale[R][4];
  const int tid = threadIdx.x;
  const int64_t ld = mx_code_ld(cols), k_atoms = mx_k_atoms(cols);
  const int64_t row_tiles = mx_row_atoms(rows) * (128 / R);
  const int64_t tiles = row_tiles * k_atoms;
  const int lr = (tid & 63) * P, b = __shfl_sync(0xFFFFFFFFu, tid >> 6, 0);     // a warp has one block
  for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int64_t atom = t / row_tiles, r0 = (t - atom * row_tiles) * R;
    uint32_t w[32];                          // one fp32, or two 16-bit values of neighbouring rows
    if (pairs && r0 + R <= rows && atom * 128 + 128 <= cols) {       // the same for the whole CTA
      // uniform addresses of the columns, one offset a lane
      const T* base = x + (atom * 128 + b * 32) * ldc + r0;
#pragma unroll
      for (int i = 0; i < 32; ++i)
        w[i] = __ldg(reinterpret_cast<const uint32_t*>(reinterpret_cast<const char*>(base + i * ldc) + lr * static_cast<int>(sizeof(T))));
    } else {
      const int64_t r = r0 + lr, c0 = atom * 128 + b * 32;
      const T* src = x + c0 * ldc + r;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        w[i] = 0;
        if (c0 + i < cols) {
          if constexpr (P == 1) {
            if (r < rows) w[i] = reinterpret_cast<const uint32_t*>(src)[i * ldc];
          } else {
            const unsigned short* q = reinterpret_cast<const unsigned short*>(src) + i * ldc;
            if (r < rows) w[i] = q[0] | (r + 1 < rows ? static_cast<uint32_t>(q[1]) << 16 : 0u);
          }
        }
      }
    }
    uint32_t top = 0;                        // largest magnitude, of both rows side by side where there are two
    if constexpr (P == 1) {
      float t = 0.0f;
#pragma unroll
      for (int i = 0; i < 32; i += 2) t = max_abs3(t, __uint_as_float(w[i]), __uint_as_float(w[i + 1]));
      top = __float_as_uint(t) & 0x7FFFFFFFu;
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) top = __vmaxu2(top, w[i] & 0x7FFF7FFFu);
    }
#pragma unroll
    for (int h = 0; h < P; ++h) {
      MxRaw one;
      one.w[0] = top;
      const uint32_t m = __float_as_uint(raw_value<T>(one, h));
      float v[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        one.w[0] = w[i];
        v[i] = raw_value<T>(one, h);
      }
      const uint32_t byte = mx_scale_byte(m);
      const float inv = mx_inverse_scale(byte);
      uint32_t c[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float a[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] = v[8 * j + i];
        c[j] = mx_round8(a, byte, inv);
      }
      s_code[lr + h][b] = make_uint4(c[0], c[1], c[2], c[3]);
      s_scale[lr + h][b] = static_cast<uint8_t>(byte);
    }
    __syncthreads();
    for (int i = tid; i < R * 4; i += kQuantThreads) {
      const int64_t wr = r0 + (i >> 2), block = atom * 4 + (i & 3);
      if (wr < rows && block * 16 < ld) *reinterpret_cast<uint4*>(codes + wr * ld + block * 16) = s_code[i >> 2][i & 3];
    }
    if (tid < R)
      *reinterpret_cast<uint32_t*>(scales + mx_scale_word(r0 + tid, atom, k_atoms)) = *reinterpret_cast<const uint32_t*>(s_scale[tid]);
    __syncthreads();
  }
}

__device__ __forceinline__ void mx_put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void mx_put(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void mx_put(float* p, float v) { *p = v; }

// Up to six matrices in one launch (blockIdx.z).  gate[i] >= 0: matrix i belongs to a modality, and is left out when
// counts[gate] says that modality has no token.
struct MxDequantJob {
  const uint8_t* codes[6];
  const uint8_t* scales[6];
  void* out[6];
  int64_t rows[6], cols[6], ldo[6];
  int gate[6];
  const int* counts;
};

// 32 bytes of output a lane, one 256-bit store: 16 values of a 16-bit type or 8 of fp32.  A warp takes units of `per_warp`
// chunks of a row, the units of a row to neighbouring warps, so that a CTA writes several KiB in a row; the next unit's codes and
// scales are in flight while one is written.
// Measured: 11008 x 4096 to bf16 21.4 us = 5.3 TB/s, to fp32 38.2 us = 5.3 TB/s (four fifths and nine tenths of it writes).
// chunks of a unit: 2 KiB of a 16-bit type, 8 KiB of fp32 (11008 x 4096: 1 / 2 / 4 / 8 chunks of bf16 23.7 / 21.2 / 22.0 / 24.7 us, of
// fp32 41.3 / 40.1 / 40.0 / 38.4)
template <typename T> constexpr int kDequantChunks = sizeof(T) == 4 ? 8 : 2;
template <typename T>
__global__ void __launch_bounds__(kQuantThreads, kQuantPerSm) mx_dequantize_kernel(const __grid_constant__ MxDequantJob job, int per_warp) {
  using L = MxLane<T>;
  const int w = blockIdx.z;
  if (job.gate[w] >= 0 && job.counts[job.gate[w]] == 0) return;
  const uint8_t* __restrict__ codes = job.codes[w];
  const uint8_t* __restrict__ scales = job.scales[w];
  T* __restrict__ out = static_cast<T*>(job.out[w]);
  const int64_t rows = job.rows[w];
  const int cols = static_cast<int>(job.cols[w]);
  const int lane = threadIdx.x & 31;
  const int64_t ldo = job.ldo[w];
  const bool vec = ((reinterpret_cast<uintptr_t>(out) | static_cast<uintptr_t>(ldo * sizeof(T))) & 31) == 0;
  const int64_t ld = mx_code_ld(cols);
  const int k_atoms = static_cast<int>(mx_k_atoms(cols));
  const int width = per_warp * L::chunk, groups = (cols + width - 1) / width;
  const int warps = gridDim.x * (kQuantThreads / 32), w0 = blockIdx.x * (kQuantThreads / 32) + (threadIdx.x >> 5);
  const int row_step = warps / groups, group_step = warps - row_step * groups;
  int64_t r = w0 / groups;
  int g = w0 - static_cast<int>(r) * groups;
  uint32_t code[kDequantChunks<T>][L::values / 8] = {}, byte[kDequantChunks<T>] = {};
  auto load = [&]() {
    if (r >= rows) return;
    const uint8_t* scale_row = scales + mx_scale_word(r, 0, k_atoms);
#pragma unroll
    for (int u = 0; u < kDequantChunks<T>; ++u) {
      const int c = g * width + u * L::chunk + lane * L::values;
      if (u < per_warp && c < cols) {
        if constexpr (L::values == 16) {
          const uint2 q = __ldg(reinterpret_cast<const uint2*>(codes + r * ld + c / 2));
          code[u][0] = q.x;
          code[u][1] = q.y;
        } else {
          code[u][0] = __ldg(reinterpret_cast<const uint32_t*>(codes + r * ld + c / 2));
        }
        byte[u] = __ldg(scale_row + static_cast<int64_t>(c >> 7) * kMxAtomBytes + ((c >> 5) & 3));
      }
    }
  };
  load();
  while (r < rows) {
    uint32_t cur[kDequantChunks<T>][L::values / 8], sb[kDequantChunks<T>];
#pragma unroll
    for (int u = 0; u < kDequantChunks<T>; ++u) {
#pragma unroll
      for (int j = 0; j < L::values / 8; ++j) cur[u][j] = code[u][j];
      sb[u] = byte[u];
    }
    const int c0 = g * width + lane * L::values;
    T* row = out + r * ldo;
    r += row_step;
    g += group_step;
    if (g >= groups) {
      g -= groups;
      ++r;
    }
    load();
#pragma unroll
    for (int u = 0; u < kDequantChunks<T>; ++u) {
      const int c = c0 + u * L::chunk;
      if (u >= per_warp || c >= cols) break;
      const float s = mx_scale_value(sb[u]);
      __align__(32) T e[L::values];
#pragma unroll
      for (int j = 0; j < L::values / 8; ++j) {
        float v[8];
        mx_unpack8(cur[u][j], v);
#pragma unroll
        for (int i = 0; i < 8; ++i) mx_put(&e[8 * j + i], mul_keep_subnormals(v[i], s));
      }
      T* o = row + c;
      if (vec && c + L::values <= cols) {
        const uint32_t* q = reinterpret_cast<const uint32_t*>(e);
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(o), "r"(q[0]), "r"(q[1]), "r"(q[2]), "r"(q[3]),
                     "r"(q[4]), "r"(q[5]), "r"(q[6]), "r"(q[7])
                     : "memory");
      } else {
#pragma unroll
        for (int i = 0; i < L::values; ++i)
          if (c + i < cols) o[i] = e[i];
      }
    }
  }
}

// Rows over blockIdx.x, groups of chunks over blockIdx.y.  With many rows a warp takes as many chunks of a row as it
// can hold in flight; with few, every chunk gets a warp of its own.
constexpr int64_t kMaxGroups = 65535;                                    // blockIdx.y
constexpr int64_t kMaxCols = kMaxGroups * 512;                           // 33553920: two chunks of 256 fp32 columns a group
struct QuantShape {
  dim3 grid;
  int per_warp;
};
static QuantShape quant_shape(int64_t rows, int64_t cols, int chunk, int chunks_max, int per_sm, int matrices = 1) {
  const int64_t chunks = (cols + chunk - 1) / chunk;
  const int64_t blocks = (static_cast<int64_t>(device_info().sm_count) * per_sm + matrices - 1) / matrices;
  int per = chunks_max;
  while (per > 1 && rows * ((chunks + per - 1) / per) < blocks * (kQuantThreads / 32) &&
         (chunks + per / 2 - 1) / (per / 2) <= kMaxGroups)
    per /= 2;
  const int64_t groups = (chunks + per - 1) / per;
  int64_t x = (rows + kQuantThreads / 32 - 1) / (kQuantThreads / 32);
  const int64_t most = (blocks + groups - 1) / groups;
  if (x > most) x = most;
  return QuantShape{dim3(static_cast<unsigned>(x < 1 ? 1 : x), static_cast<unsigned>(groups)), per};
}
static int row_alignment(const void* x, int64_t row_bytes) {
  const uintptr_t v = reinterpret_cast<uintptr_t>(x) | static_cast<uintptr_t>(row_bytes);
  return v & 15 ? 1 : (v & 31 ? 16 : 32);
}

template <int T>
static int quantize_typed(const void* x_, int64_t row_stride, int64_t col_stride, int64_t rows, int64_t cols, void* codes,
                          void* scales, cudaStream_t s) {
  using E = typename MxType<T>::t;
  const E* x = static_cast<const E*>(x_);
  uint8_t* c = static_cast<uint8_t*>(codes);
  uint8_t* sc = static_cast<uint8_t*>(scales);
  if (col_stride == 1 || cols == 1) {
    const QuantShape q = quant_shape(rows, cols, MxLane<E>::chunk, kChunksMax, kQuantPerSm);
    mx_quantize_rows_kernel<E><<<q.grid, kQuantThreads, 0, s>>>(
        x, row_stride, static_cast<int>(rows), static_cast<int>(cols), nullptr, nullptr, c, sc,
        row_alignment(x, row_stride * static_cast<int64_t>(sizeof(E))), q.per_warp);
  } else {
    int64_t tiles = mx_row_atoms(rows) * (128 / MxCols<E>::rows) * mx_k_atoms(cols);
    if (tiles > (1 << 30)) tiles = 1 << 30;
    mx_quantize_cols_kernel<E><<<static_cast<unsigned>(tiles), kQuantThreads, 0, s>>>(
        x, col_stride, rows, cols, c, sc, ((reinterpret_cast<uintptr_t>(x) | static_cast<uintptr_t>(col_stride * sizeof(E))) & 3) == 0);
  }
  return cuda_status(cudaGetLastError());
}

// Few tokens: 2 KiB of shared memory, and the SM's memory divided as the products want it, so that their CTAs get their places while this
// kernel runs (an SM does not change the division while it is busy, and a cluster whose place is taken at first may wait
// until all others are done): linear 11008 -> 4096, 8 tokens of both modalities 20.0 -> 14.4 us, 4096 x 4096, 127
// tokens 13.0 -> 11.9.  Many tokens: CTAs that wait beside it only slow it down (4096 x 4096, 4000 tokens 38.3 -> 40.4).
int mx_route_quantize(const void* mask, int64_t M, const void* x, int64_t ldx, int64_t d, int32_t* perm, int32_t* counts,
                      void* scan, void* codes, void* scales, int32_t* status, void* stream) {
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const __nv_bfloat16* xb = static_cast<const __nv_bfloat16*>(x);
  uint8_t* c = static_cast<uint8_t*>(codes);
  uint8_t* sc = static_cast<uint8_t*>(scales);
  if (M <= kMxRouteTokens) {
    const QuantShape q = quant_shape(M, d, MxLane<__nv_bfloat16>::chunk, kChunksMax, kQuantPerSm);
    const bool beside = M <= kMxBesideTokens;
    if (beside) {
      static std::atomic<uint64_t> prepared{0};
      const int r = once_per_device(prepared, [] {
        return cudaFuncSetAttribute(mx_route_quantize_kernel<1>, cudaFuncAttributePreferredSharedMemoryCarveout,
                                    cudaSharedmemCarveoutMaxShared);
      });
      if (r) return r;
    }
    const auto kernel = beside ? mx_route_quantize_kernel<1> : mx_route_quantize_kernel<kMxRouteWords>;
    kernel<<<q.grid, kRouteThreads, 0, s>>>(static_cast<const uint8_t*>(mask), static_cast<int>(M),
                                            static_cast<int>(ffnk_route_capacity(M)), perm, counts, xb, ldx, static_cast<int>(d), c,
                                            sc, row_alignment(x, 2 * ldx), q.per_warp);
    return cuda_status(cudaGetLastError());
  }
  const int r = ffnk_route(mask, M, perm, counts, scan, status, stream);
  if (r) return r;
  const QuantShape q = quant_shape(M, d, MxLane<__nv_bfloat16>::chunk, kChunksMax, kQuantPerSm);
  mx_quantize_rows_kernel<__nv_bfloat16><<<q.grid, kQuantThreads, 0, s>>>(xb, ldx, static_cast<int>(M), static_cast<int>(d), perm,
                                                                          counts, c, sc, row_alignment(x, 2 * ldx), q.per_warp);
  return cuda_status(cudaGetLastError());
}

int mx_dequantize_weights(const void* const* codes, const void* const* scales, const int64_t* rows, const int64_t* cols,
                          const int* gate, int n, const int32_t* counts, void* const* out, void* stream) {
  MxDequantJob job{};
  int64_t most_rows = 0, most_cols = 0;
  for (int i = 0; i < n; ++i) {
    job.codes[i] = static_cast<const uint8_t*>(codes[i]);
    job.scales[i] = static_cast<const uint8_t*>(scales[i]);
    job.out[i] = out[i];
    job.rows[i] = rows[i];
    job.cols[i] = job.ldo[i] = cols[i];
    job.gate[i] = gate[i];
    most_rows = rows[i] > most_rows ? rows[i] : most_rows;
    most_cols = cols[i] > most_cols ? cols[i] : most_cols;
  }
  job.counts = counts;
  QuantShape q = quant_shape(most_rows, most_cols, MxLane<__nv_bfloat16>::chunk, kDequantChunks<__nv_bfloat16>, kQuantPerSm, n);
  q.grid = dim3(q.grid.x * q.grid.y, 1, n);
  mx_dequantize_kernel<__nv_bfloat16><<<q.grid, kQuantThreads, 0, static_cast<cudaStream_t>(stream)>>>(job, q.per_warp);
  return cuda_status(cudaGetLastError());
}

}  // namespace ffnk

using namespace ffnk;

static bool mx_bad_size(int64_t v) { return v < 0 || v >= (1ll << 30); }

extern "C" int64_t ffnk_mxfp4_code_bytes(int64_t rows, int64_t cols) {
  return mx_bad_size(rows) || mx_bad_size(cols) ? FFNK_ERR_SHAPE : rows * mx_code_ld(cols);
}
extern "C" int64_t ffnk_mxfp4_scale_bytes(int64_t rows, int64_t cols) {
  return mx_bad_size(rows) || mx_bad_size(cols) ? FFNK_ERR_SHAPE : mx_row_atoms(rows) * mx_k_atoms(cols) * kMxAtomBytes;
}

extern "C" int ffnk_mxfp4_quantize(const void* x, int dtype, int64_t row_stride, int64_t col_stride, int64_t rows,
                                   int64_t cols, void* codes, void* scales, void* stream) {
  if (mx_bad_size(rows) || mx_bad_size(cols) || cols > kMaxCols || dtype < FFNK_BF16 || dtype > FFNK_FP32) return FFNK_ERR_SHAPE;
  if (rows == 0 || cols == 0) return 0;
  if (!x || !codes || !scales) return FFNK_ERR_NULL;
  if (!(col_stride == 1 || cols == 1) && !(row_stride == 1 || rows == 1)) return FFNK_ERR_LAYOUT;
  if (row_stride < 0 || col_stride < 0) return FFNK_ERR_LAYOUT;
  if ((reinterpret_cast<uintptr_t>(codes) & 15) || (reinterpret_cast<uintptr_t>(scales) & 15) ||
      (reinterpret_cast<uintptr_t>(x) & (dtype == FFNK_FP32 ? 3 : 1)))
    return FFNK_ERR_ALIGN;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case FFNK_BF16: return quantize_typed<FFNK_BF16>(x, row_stride, col_stride, rows, cols, codes, scales, s);
    case FFNK_FP16: return quantize_typed<FFNK_FP16>(x, row_stride, col_stride, rows, cols, codes, scales, s);
    default: return quantize_typed<FFNK_FP32>(x, row_stride, col_stride, rows, cols, codes, scales, s);
  }
}

extern "C" int ffnk_mxfp4_dequantize(const void* codes, const void* scales, int64_t rows, int64_t cols, void* out, int dtype,
                                     int64_t ldo, void* stream) {
  if (mx_bad_size(rows) || mx_bad_size(cols) || cols > kMaxCols || dtype < FFNK_BF16 || dtype > FFNK_FP32) return FFNK_ERR_SHAPE;
  if (rows == 0 || cols == 0) return 0;
  if (!codes || !scales || !out) return FFNK_ERR_NULL;
  const int size = dtype == FFNK_FP32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(codes) & 15) || (reinterpret_cast<uintptr_t>(scales) & 15) ||
      (reinterpret_cast<uintptr_t>(out) & (size - 1)) || ldo < cols)
    return FFNK_ERR_ALIGN;
  QuantShape q = dtype == FFNK_FP32 ? quant_shape(rows, cols, MxLane<float>::chunk, kDequantChunks<float>, kQuantPerSm)
                                    : quant_shape(rows, cols, MxLane<__half>::chunk, kDequantChunks<__half>, kQuantPerSm);
  q.grid = dim3(q.grid.x * q.grid.y);
  MxDequantJob job{};
  job.codes[0] = static_cast<const uint8_t*>(codes);
  job.scales[0] = static_cast<const uint8_t*>(scales);
  job.out[0] = out;
  job.rows[0] = rows;
  job.cols[0] = cols;
  job.ldo[0] = ldo;
  job.gate[0] = -1;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case FFNK_BF16: mx_dequantize_kernel<__nv_bfloat16><<<q.grid, kQuantThreads, 0, s>>>(job, q.per_warp); break;
    case FFNK_FP16: mx_dequantize_kernel<__half><<<q.grid, kQuantThreads, 0, s>>>(job, q.per_warp); break;
    default: mx_dequantize_kernel<float><<<q.grid, kQuantThreads, 0, s>>>(job, q.per_warp);
  }
  return cuda_status(cudaGetLastError());
}
