// Quantisation to MXFP4 and back (the format: mxfp4.cuh).
//
//   mx_quantize_rows_kernel    x contiguous along the blocks: weights in nn.Linear storage, activations; with
//                              routing lists the rows come out in routed order
//   mx_route_quantize_kernel   routing, the copy into routed order and the quantisation of the activations in one
//                              launch, for masks of one routing tile
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

__device__ __forceinline__ float mx_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float mx_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float mx_float(float v) { return v; }

constexpr int kQuantThreads = 256;
constexpr int kChunk = 256;          // columns of one warp step: a lane holds 8 consecutive values, 4 lanes a block
constexpr int kChunksPerItem = 4;    // warp steps whose loads are in flight together

// Eight consecutive values of a row as floats; beyond `cols` zeros.  `vec`: the row is 16-byte aligned.
template <typename T>
__device__ __forceinline__ void load8(const T* row, int64_t c, int64_t cols, bool vec, float (&v)[8]) {
  if (vec && c + 8 <= cols) {
    if constexpr (sizeof(T) == 2) {
      const uint4 w = __ldg(reinterpret_cast<const uint4*>(row + c));
      __align__(16) T e[8];
      *reinterpret_cast<uint4*>(e) = w;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = mx_float(e[i]);
    } else {
      const float4 a = __ldg(reinterpret_cast<const float4*>(row + c)), b = __ldg(reinterpret_cast<const float4*>(row + c) + 1);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < cols ? mx_float(row[c + i]) : 0.0f;
  }
}

// One warp, one row, up to kChunksPerItem chunks of 256 columns from chunk `first` on.  Every lane of a block's
// four gets the block's maximum by two shuffles; the eight scale bytes of a chunk are two words of two atoms.
template <typename T>
__device__ __forceinline__ void quantize_row(const T* row, bool vec, int64_t cols, int first, int chunks, uint8_t* codes_row,
                                             uint8_t* scales, int64_t dst, int64_t k_atoms, int lane) {
  float v[kChunksPerItem][8];
#pragma unroll
  for (int u = 0; u < kChunksPerItem; ++u)
    if (first + u < chunks) load8(row, static_cast<int64_t>(first + u) * kChunk + lane * 8, cols, vec, v[u]);
#pragma unroll
  for (int u = 0; u < kChunksPerItem; ++u) {
    if (first + u >= chunks) break;                    // warp-uniform
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[u][i]) & 0x7FFFFFFFu);
    m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
    m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
    const uint32_t byte = mx_scale_byte(m);
    const float inv = mx_inverse_scale(byte);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[u][i] = mul_keep_subnormals(v[u][i], inv);
    uint32_t code = byte == 255u ? 0u : mx_pack8(v[u]);
    const int64_t c = static_cast<int64_t>(first + u) * kChunk + lane * 8;
    if (c < (cols + 31) / 32 * 32) *reinterpret_cast<uint32_t*>(codes_row + c / 2) = code;
    uint32_t word = byte << (8 * ((lane >> 2) & 3));
    word |= __shfl_xor_sync(0xFFFFFFFFu, word, 4);
    word |= __shfl_xor_sync(0xFFFFFFFFu, word, 8);
    const int64_t atom = static_cast<int64_t>(first + u) * 2 + (lane >> 4);
    if ((lane & 15) == 0 && atom < k_atoms) *reinterpret_cast<uint32_t*>(scales + mx_scale_word(dst, atom, k_atoms)) = word;
  }
}

// Plain (perm == nullptr): row r of x -> row r; the scale bytes of the rows that fill the last atom are zeroed.
// Routed: rows in routed order (visual rows first, text rows from the next multiple of 256), none beyond them.
template <typename T>
__global__ void __launch_bounds__(kQuantThreads) mx_quantize_rows_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows,
                                                                         int64_t cols, const int* __restrict__ perm,
                                                                         const int* __restrict__ counts,
                                                                         uint8_t* __restrict__ codes,
                                                                         uint8_t* __restrict__ scales, bool vec) {
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int chunks = static_cast<int>((cols + kChunk - 1) / kChunk);
  const int groups = (chunks + kChunksPerItem - 1) / kChunksPerItem;
  const int64_t ld = mx_code_ld(cols), k_atoms = mx_k_atoms(cols);
  const int64_t all_rows = perm ? rows : mx_row_atoms(rows) * 128;
  const int64_t items = all_rows * groups;
  int Mv = 0, cap = 0;
  if (perm) {
    Mv = counts[0];
    cap = counts[2];
  }
  const int64_t text_base = ((Mv + 255) >> 8) << 8;
  for (int64_t it = static_cast<int64_t>(blockIdx.x) * (kQuantThreads / 32) + (threadIdx.x >> 5); it < items;
       it += static_cast<int64_t>(gridDim.x) * (kQuantThreads / 32)) {
    const int64_t r = it / groups;
    const int first = static_cast<int>(it - r * groups) * kChunksPerItem;
    if (r >= rows) {
      for (int64_t a = first * 2 + lane; a < k_atoms && a < (first + kChunksPerItem) * 2; a += 32)
        *reinterpret_cast<uint32_t*>(scales + mx_scale_word(r, a, k_atoms)) = 0u;
      continue;
    }
    int64_t src = r, dst = r;
    if (perm) {
      src = r < Mv ? perm[r] : perm[cap + (r - Mv)];
      dst = r < Mv ? r : text_base + (r - Mv);
    }
    quantize_row(x + src * ldx, vec, cols, first, chunks, codes + dst * ld, scales, dst, k_atoms, lane);
  }
}

// Routing and quantisation of the activations in one launch (M <= 8192): every CTA routes the whole mask for
// itself in shared memory, CTA 0 also writes perm and counts, then every warp quantises its share of the rows.
__global__ void __launch_bounds__(kRouteThreads) mx_route_quantize_kernel(const uint8_t* __restrict__ mask, int M, int cap,
                                                                          int* __restrict__ perm, int* __restrict__ counts,
                                                                          const __nv_bfloat16* __restrict__ x, int64_t ldx,
                                                                          int64_t cols, uint8_t* __restrict__ codes,
                                                                          uint8_t* __restrict__ scales) {
  __shared__ int s_list[kRouteTile];   // visual tokens ascending, then text tokens ascending
  __shared__ int s_warp[kRouteThreads / 32];
  __shared__ int s_runs;
  const int tid = threadIdx.x, lane = tid & 31;
  griddep_launch_dependents();
  const ThreadTokens tt = load_thread_tokens(mask, M, tid * kRoutePerThread);
  if (tid == 0) s_runs = 0;
  int Mv = 0;
  const int ev = block_exclusive_scan(__popc(tt.bits), s_warp, &Mv);
  if (blockIdx.x == 0) {
    const int wr = __reduce_add_sync(0xFFFFFFFFu, tt.nruns);
    if (lane == 0 && wr) atomicAdd(&s_runs, wr);
  }
  compact_tile(s_list, s_list + Mv, 0, tt.bits, ev, tt.valid);
  __syncthreads();
  const int Mt = M - Mv;
  if (blockIdx.x == 0) {
    for (int i = tid; i < Mv; i += kRouteThreads) perm[i] = s_list[i];
    for (int i = tid; i < Mt; i += kRouteThreads) perm[cap + i] = s_list[Mv + i];
    if (tid == 0) {
      counts[0] = Mv;
      counts[1] = Mt;
      counts[2] = cap;
      counts[3] = M;
      counts[4] = s_runs;
    }
  }
  const int64_t text_base = ((Mv + 255) >> 8) << 8;
  const int chunks = static_cast<int>((cols + kChunk - 1) / kChunk);
  const int groups = (chunks + kChunksPerItem - 1) / kChunksPerItem;
  const int64_t ld = mx_code_ld(cols), k_atoms = mx_k_atoms(cols);
  const int64_t items = static_cast<int64_t>(M) * groups;
  for (int64_t it = static_cast<int64_t>(blockIdx.x) * (kRouteThreads / 32) + (tid >> 5); it < items;
       it += static_cast<int64_t>(gridDim.x) * (kRouteThreads / 32)) {
    const int i = static_cast<int>(it / groups);
    const int first = static_cast<int>(it - static_cast<int64_t>(i) * groups) * kChunksPerItem;
    const int64_t dst = i >= Mv ? text_base + (i - Mv) : i;
    quantize_row(x + static_cast<int64_t>(s_list[i]) * ldx, true, cols, first, chunks, codes + dst * ld, scales, dst,
                 k_atoms, lane);
  }
}

// x(r, c) at x[c * ldc + r]: blocks run across the contiguous dimension.  A CTA takes 64 rows x one atom of
// blocks; a thread reads the 32 values of one block (neighbouring lanes neighbouring rows), and the codes go
// through shared memory so that a row leaves as 64 contiguous bytes.
constexpr int kColRows = 64;
template <typename T>
__global__ void __launch_bounds__(kQuantThreads) mx_quantize_cols_kernel(const T* __restrict__ x, int64_t ldc, int64_t rows,
                                                                         int64_t cols, uint8_t* __restrict__ codes,
                                                                         uint8_t* __restrict__ scales) {
  __shared__ uint4 s_code[kColRows][5];      // four blocks a row, one piece of padding against bank conflicts
  __shared__ uint8_t s_scale[kColRows][4];
  const int tid = threadIdx.x;
  const int64_t ld = mx_code_ld(cols), k_atoms = mx_k_atoms(cols);
  const int64_t row_tiles = mx_row_atoms(rows) * 2;
  const int64_t tiles = row_tiles * k_atoms;
  const int lr = tid & (kColRows - 1), b = tid >> 6;
  for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int64_t atom = t / row_tiles, r0 = (t - atom * row_tiles) * kColRows;
    const int64_t r = r0 + lr, c0 = atom * 128 + b * 32;
    float v[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = r < rows && c0 + i < cols ? mx_float(x[(c0 + i) * ldc + r]) : 0.0f;
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    const uint32_t byte = mx_scale_byte(m);
    const float inv = mx_inverse_scale(byte);
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float a[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = mul_keep_subnormals(v[8 * j + i], inv);
      w[j] = byte == 255u ? 0u : mx_pack8(a);
    }
    s_code[lr][b] = make_uint4(w[0], w[1], w[2], w[3]);
    s_scale[lr][b] = static_cast<uint8_t>(byte);
    __syncthreads();
    const int64_t wr = r0 + (tid >> 2), block = atom * 4 + (tid & 3);
    if (wr < rows && block * 16 < ld) *reinterpret_cast<uint4*>(codes + wr * ld + block * 16) = s_code[tid >> 2][tid & 3];
    if (tid < kColRows)
      *reinterpret_cast<uint32_t*>(scales + mx_scale_word(r0 + tid, atom, k_atoms)) =
          *reinterpret_cast<const uint32_t*>(s_scale[tid]);
    __syncthreads();
  }
}

__device__ __forceinline__ void mx_put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void mx_put(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void mx_put(float* p, float v) { *p = v; }

// Up to six matrices in one launch (blockIdx.y).  gate[i] >= 0: matrix i belongs to a modality, and is left out when
// counts[gate] says that modality has no token.
struct MxDequantJob {
  const uint8_t* codes[6];
  const uint8_t* scales[6];
  void* out[6];
  int64_t rows[6], cols[6], ldo[6];
  int gate[6];
  const int* counts;
};

template <typename T>
__global__ void __launch_bounds__(kQuantThreads) mx_dequantize_kernel(const __grid_constant__ MxDequantJob job) {
  const int w = blockIdx.y;
  if (job.gate[w] >= 0 && job.counts[job.gate[w]] == 0) return;
  const uint8_t* __restrict__ codes = job.codes[w];
  const uint8_t* __restrict__ scales = job.scales[w];
  T* __restrict__ out = static_cast<T*>(job.out[w]);
  const int64_t rows = job.rows[w], cols = job.cols[w], ldo = job.ldo[w];
  const bool vec = ((reinterpret_cast<uintptr_t>(out) | static_cast<uintptr_t>(ldo * sizeof(T))) & 15) == 0;
  const int lane = threadIdx.x & 31;
  const int chunks = static_cast<int>((cols + kChunk - 1) / kChunk);
  const int groups = (chunks + kChunksPerItem - 1) / kChunksPerItem;
  const int64_t ld = mx_code_ld(cols), k_atoms = mx_k_atoms(cols);
  const int64_t items = rows * groups;
  for (int64_t it = static_cast<int64_t>(blockIdx.x) * (kQuantThreads / 32) + (threadIdx.x >> 5); it < items;
       it += static_cast<int64_t>(gridDim.x) * (kQuantThreads / 32)) {
    const int64_t r = it / groups;
    const int first = static_cast<int>(it - r * groups) * kChunksPerItem;
    uint32_t code[kChunksPerItem] = {}, word[kChunksPerItem] = {};
#pragma unroll
    for (int u = 0; u < kChunksPerItem; ++u) {
      const int64_t c = static_cast<int64_t>(first + u) * kChunk + lane * 8;
      if (c < cols) {
        code[u] = __ldg(reinterpret_cast<const uint32_t*>(codes + r * ld + c / 2));
        word[u] = __ldg(reinterpret_cast<const uint32_t*>(scales + mx_scale_word(r, c / 128, k_atoms)));
      }
    }
#pragma unroll
    for (int u = 0; u < kChunksPerItem; ++u) {
      const int64_t c = static_cast<int64_t>(first + u) * kChunk + lane * 8;
      if (c >= cols) break;
      const float s = mx_scale_value((word[u] >> (8 * ((lane >> 2) & 3))) & 255u);
      float v[8];
      mx_unpack8(code[u], v);
      __align__(16) T e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) mx_put(&e[i], mul_keep_subnormals(v[i], s));
      T* o = out + r * ldo + c;
      if (vec && c + 8 <= cols) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
          reinterpret_cast<uint4*>(o)[i] = reinterpret_cast<const uint4*>(e)[i];
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c + i < cols) o[i] = e[i];
      }
    }
  }
}

static unsigned quant_grid(int64_t warps_of_work, int per_sm) {
  int64_t blocks = (warps_of_work + kQuantThreads / 32 - 1) / (kQuantThreads / 32);
  const int64_t most = static_cast<int64_t>(device_info().sm_count) * per_sm;
  if (blocks > most) blocks = most;
  return static_cast<unsigned>(blocks < 1 ? 1 : blocks);
}
static int64_t row_groups(int64_t cols) { return (cols + kChunk * kChunksPerItem - 1) / (kChunk * kChunksPerItem); }

template <int T>
static int quantize_typed(const void* x_, int64_t row_stride, int64_t col_stride, int64_t rows, int64_t cols, void* codes,
                          void* scales, cudaStream_t s) {
  using E = typename MxType<T>::t;
  const E* x = static_cast<const E*>(x_);
  uint8_t* c = static_cast<uint8_t*>(codes);
  uint8_t* sc = static_cast<uint8_t*>(scales);
  if (col_stride == 1 || cols == 1) {
    const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (row_stride * static_cast<int64_t>(sizeof(E))) % 16 == 0;
    mx_quantize_rows_kernel<E><<<quant_grid(mx_row_atoms(rows) * 128 * row_groups(cols), 8), kQuantThreads, 0, s>>>(
        x, row_stride, rows, cols, nullptr, nullptr, c, sc, vec);
  } else {
    int64_t tiles = mx_row_atoms(rows) * 2 * mx_k_atoms(cols);
    const int64_t most = static_cast<int64_t>(device_info().sm_count) * 8;
    if (tiles > most) tiles = most;
    mx_quantize_cols_kernel<E><<<static_cast<unsigned>(tiles), kQuantThreads, 0, s>>>(x, col_stride, rows, cols, c, sc);
  }
  return cuda_status(cudaGetLastError());
}

int mx_route_quantize(const void* mask, int64_t M, const void* x, int64_t ldx, int64_t d, int32_t* perm, int32_t* counts,
                      void* scan, void* codes, void* scales, int32_t* status, void* stream) {
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const __nv_bfloat16* xb = static_cast<const __nv_bfloat16*>(x);
  uint8_t* c = static_cast<uint8_t*>(codes);
  uint8_t* sc = static_cast<uint8_t*>(scales);
  if (M <= kRouteTile) {
    mx_route_quantize_kernel<<<quant_grid(M * row_groups(d), 4), kRouteThreads, 0, s>>>(
        static_cast<const uint8_t*>(mask), static_cast<int>(M), static_cast<int>(ffnk_route_capacity(M)), perm, counts, xb,
        ldx, d, c, sc);
    return cuda_status(cudaGetLastError());
  }
  const int r = ffnk_route(mask, M, perm, counts, scan, status, stream);
  if (r) return r;
  mx_quantize_rows_kernel<__nv_bfloat16><<<quant_grid(M * row_groups(d), 8), kQuantThreads, 0, s>>>(
      xb, ldx, M, d, perm, counts, c, sc, true);
  return cuda_status(cudaGetLastError());
}

int mx_dequantize_weights(const void* const* codes, const void* const* scales, const int64_t* rows, const int64_t* cols,
                          const int* gate, int n, const int32_t* counts, void* const* out, void* stream) {
  MxDequantJob job{};
  int64_t items = 0;
  for (int i = 0; i < n; ++i) {
    job.codes[i] = static_cast<const uint8_t*>(codes[i]);
    job.scales[i] = static_cast<const uint8_t*>(scales[i]);
    job.out[i] = out[i];
    job.rows[i] = rows[i];
    job.cols[i] = job.ldo[i] = cols[i];
    job.gate[i] = gate[i];
    items = rows[i] * row_groups(cols[i]) > items ? rows[i] * row_groups(cols[i]) : items;
  }
  job.counts = counts;
  mx_dequantize_kernel<__nv_bfloat16><<<dim3(quant_grid(items, 8), n), kQuantThreads, 0, static_cast<cudaStream_t>(stream)>>>(job);
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
  if (mx_bad_size(rows) || mx_bad_size(cols) || dtype < FFNK_BF16 || dtype > FFNK_FP32) return FFNK_ERR_SHAPE;
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
  if (mx_bad_size(rows) || mx_bad_size(cols) || dtype < FFNK_BF16 || dtype > FFNK_FP32) return FFNK_ERR_SHAPE;
  if (rows == 0 || cols == 0) return 0;
  if (!codes || !scales || !out) return FFNK_ERR_NULL;
  const int size = dtype == FFNK_FP32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(codes) & 15) || (reinterpret_cast<uintptr_t>(scales) & 15) ||
      (reinterpret_cast<uintptr_t>(out) & (size - 1)) || ldo < cols)
    return FFNK_ERR_ALIGN;
  const unsigned grid = quant_grid(rows * row_groups(cols), 8);
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
    case FFNK_BF16: mx_dequantize_kernel<__nv_bfloat16><<<grid, kQuantThreads, 0, s>>>(job); break;
    case FFNK_FP16: mx_dequantize_kernel<__half><<<grid, kQuantThreads, 0, s>>>(job); break;
    default: mx_dequantize_kernel<float><<<grid, kQuantThreads, 0, s>>>(job);
  }
  return cuda_status(cudaGetLastError());
}
