// Routed GEMMs on MXFP4 operands (format: mxfp4.cuh) and the forward passes made of them.
//
// D[r, n] = sum over blocks b of 2^(Ea[r,b] + Ew[n,b]) * sum over the 32 values of block b of a * w, the rows r
// of one modality by that modality's weight.  tcgen05.mma.kind::mxf4.block_scale does both sums: codes come
// from shared memory (64 values of a row an instruction, four times the bf16 instruction's K for the same bytes),
// the scales from tensor memory, where tcgen05.cp puts each 512-byte scale atom (128 rows x 4 blocks).  Products
// of codes are exact, sums are fp32.
//
// Both operands are K-major: activations quantised into routed order (mxfp4.cu) and weights in nn.Linear order.
// Epilogues: bf16 rows scattered to token order; or silu(gate) * up, which leaves as MXFP4 again: the 32
// accumulator columns a lane reads at a time are one block of its row, so the maximum, the scale and the codes
// need no other lane.
#include "ffnk_internal.h"
#include "mxfp4.cuh"
#include "ptx.cuh"

namespace ffnk {

// ---------------------------------------------------------------------------------------------
// block-scaled tcgen05
// ---------------------------------------------------------------------------------------------
// Instruction descriptor of kind::mxf4: E2M1 operands, scales in powers of two (UE8M0).  sf: which half of
// the four scale bytes of a tensor-memory word this instruction's two blocks use (0: bytes 0,1; 2: bytes 2,3).
__host__ __device__ constexpr uint32_t mx_idesc(int m, int n, uint32_t sf) {
  return (sf << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (1u << 23) |
         (static_cast<uint32_t>(m >> 7) << 27) | (sf << 29);
}
// Descriptors are kept as their low word, (address >> 4) | leading offset << 16, and a constant high word, so that a
// step of the loop is one 32-bit addition; everything an instruction needs is computed outside the branch of the
// electing lane, where the compiler can use uniform registers.
constexpr uint32_t MX_DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);      // operands: 8-row groups 1 KiB apart, 128-byte swizzle
constexpr uint32_t MX_SCALE_DESC_HI = (128u >> 4) | (1u << 14);              // scale atoms: 8-row groups 128 bytes apart, no swizzle
__device__ __forceinline__ uint32_t mx_desc_lo(uint32_t smem) { return ((smem & 0x3FFFFu) >> 4) | (1u << 16); }

template <int CTAS>
__device__ __forceinline__ void umma_mxf4(uint32_t tmem_d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                          uint32_t accumulate) {
  if constexpr (CTAS == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
        "mov.b64 da, {%1, %7};\n\tmov.b64 db, {%2, %7};\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], da, db, %3, [%4], [%5], p;\n\t}" ::"r"(tmem_d),
        "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate), "r"(MX_DESC_HI)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
        "mov.b64 da, {%1, %7};\n\tmov.b64 db, {%2, %7};\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], da, db, %3, [%4], [%5], p;\n\t}" ::"r"(tmem_d),
        "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate), "r"(MX_DESC_HI)
        : "memory");
}
// One scale atom (512 consecutive bytes: 32 rows of 16 bytes) from shared memory to four tensor-memory columns,
// the same 32 lanes in all four lane quarters.  In issue order with the MMAs of the same thread.
template <int CTAS>
__device__ __forceinline__ void tmem_copy_scales(uint32_t tmem, uint32_t lo) {
  if constexpr (CTAS == 1)
    asm volatile("{\n\t.reg .b64 d;\n\tmov.b64 d, {%1, %2};\n\ttcgen05.cp.cta_group::1.32x128b.warpx4 [%0], d;\n\t}" ::"r"(tmem),
                 "r"(lo), "r"(MX_SCALE_DESC_HI)
                 : "memory");
  else
    asm volatile("{\n\t.reg .b64 d;\n\tmov.b64 d, {%1, %2};\n\ttcgen05.cp.cta_group::2.32x128b.warpx4 [%0], d;\n\t}" ::"r"(tmem),
                 "r"(lo), "r"(MX_SCALE_DESC_HI)
                 : "memory");
}

// ---------------------------------------------------------------------------------------------
// geometry
// ---------------------------------------------------------------------------------------------
constexpr int MX_BM = 128;                    // rows of a CTA's tile
constexpr int MX_BN = 256;                    // accumulator columns (gate/up tiles: 128 gate | 128 up)
constexpr int MX_A_BYTES = MX_BM * 128;       // 16 KiB of codes
constexpr int MX_SF_BYTES = 2 * kMxAtomBytes; // scales of 128 rows x one k-step

enum { MX_EPI_STORE = 0, MX_EPI_GLU = 1, MX_EPI_GLU_SAVE = 2 };
__host__ __device__ constexpr bool mx_glu(int e) { return e != MX_EPI_STORE; }

struct MxParams {
  const int* perm;
  const int* counts;
  int* status;
  int n_out;               // output columns: N, or h for the gate/up tiles
  int k_bytes;             // code bytes of a row along the contraction (a multiple of 16)
  int a_rows;              // rows of an A box (fewer than 128 when no tile has more)
  int group_m;
  // MX_EPI_STORE: out[token][n]; MX_EPI_GLU_SAVE: the backward pass's factors f1, f3 of kept_rows =
  // cap + 512 routed rows (kept_tile_offset)
  __nv_bfloat16* out;
  int64_t ldo;
  __half* f1;
  __half* f3;
  int64_t kept_rows;
  // MX_EPI_GLU*: codes [routed row][code_ld] and scales of the quantised product
  uint8_t* codes;
  uint8_t* scales;
  int64_t code_ld;
  int k_atoms_out;
  long long* prof;         // optional per-CTA wait-cycle counters (ffnk_debug_profile_buffer)
};

// Codes come through tensor maps; scales, whose atoms of a k-step are 1 KiB in a row, by plain bulk copies (each map
// saved is 0.2 us of host time, which counts where a call takes 10).  CTA pairs need tensor maps for the scales too: only
// a tensor copy may report to the barrier of another CTA than the one its data goes to.
struct MxMaps {
  CUtensorMap a;           // activation codes
  CUtensorMap b[4];        // weight codes: visual 0/1, text 0/1 (gate, up)
  CUtensorMap tsa, tsb[4]; // scales, CTA pairs only: [row atom][128 words a k atom], boxes of two k atoms
  const uint8_t* sa;       // activation scales
  const uint8_t* sb[4];    // weight scales
  int k_atoms;             // scale atoms of a row along the contraction
  int sb_atoms;            // row atoms of a weight
};

// 16-byte aligned bulk copy to this CTA's shared memory, completion on an mbarrier given by its shared::cluster address
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src),
               "r"(bytes), "r"(bar)
               : "memory");
}
// bytes of one row atom's scales in k-step ks: two atoms of 4 blocks, one where the contraction ends
__device__ __forceinline__ uint32_t mx_step_scale_bytes(int ks, int k_atoms) { return 2 * ks + 1 < k_atoms ? MX_SF_BYTES : kMxAtomBytes; }
__device__ __forceinline__ const uint8_t* mx_scale_at(const uint8_t* base, int row_atom, int ks, int k_atoms) {
  return base + (static_cast<int64_t>(row_atom) * k_atoms + 2 * ks) * kMxAtomBytes;
}

struct MxTile {
  int nt, row0, rows, list_off;
  int64_t routed0;         // first routed-order row of the tile
  bool text;
};

__device__ __forceinline__ int mx_text_base(int Mv) { return ((Mv + 255) >> 8) << 8; }

// Tile t: super-tiles of group_m row tiles x all column tiles, rows fastest.  bm: rows of the (pair) tile,
// half: this CTA's offset inside it.
__device__ __forceinline__ MxTile mx_tile(int t, int bm, int half, int tiles_v, int m_tiles, int n_tiles, int group_m, int Mv,
                                          int Mt, int cap) {
  MxTile c;
  const int per_super = group_m * n_tiles;
  const int st = t / per_super;
  const int r = t - st * per_super;
  const int m0 = st * group_m;
  const int gm = min(group_m, m_tiles - m0);
  c.nt = r / gm;
  const int mt = m0 + (r - c.nt * gm);
  c.text = mt >= tiles_v;
  c.row0 = (c.text ? mt - tiles_v : mt) * bm + half;
  c.rows = max(0, min(MX_BM, (c.text ? Mt : Mv) - c.row0));
  c.list_off = c.text ? cap : 0;
  c.routed0 = (c.text ? mx_text_base(Mv) : 0) + c.row0;
  return c;
}

__device__ __forceinline__ uint32_t mx_pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// 32 rows x 32 columns of one warp as bf16 through its 2 KiB of shared memory: 64 contiguous bytes a row, eight
// rows a store instruction.  `dst`: address of this lane's row (0: none).
__device__ __forceinline__ void mx_store_rows(const float (&v)[32], unsigned long long dst, int n0, int n_out, uint8_t* stg, int lane) {
  const int wsw = (lane >> 1) & 3, pc = lane & 3;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    *reinterpret_cast<uint4*>(stg + lane * 64 + ((j ^ wsw) << 4)) =
        make_uint4(mx_pack_bf16(v[8 * j], v[8 * j + 1]), mx_pack_bf16(v[8 * j + 2], v[8 * j + 3]),
                   mx_pack_bf16(v[8 * j + 4], v[8 * j + 5]), mx_pack_bf16(v[8 * j + 6], v[8 * j + 7]));
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = i * 8 + (lane >> 2);
    const unsigned long long rp = __shfl_sync(0xFFFFFFFFu, dst, r);
    const uint4 val = *reinterpret_cast<const uint4*>(stg + r * 64 + ((pc ^ ((r >> 1) & 3)) << 4));
    if (rp != 0ull && n0 + pc * 8 < n_out) *reinterpret_cast<uint4*>(rp + 2ull * (n0 + pc * 8)) = val;
  }
  __syncwarp();
}

// silu(t1) * t3 with an exponential and a reciprocal good to a few units in the last fp32 place: what is rounded
// to four bits next must not sit on the wrong side of a tie more often than fp32 sums put it there anyway
// (a hyperbolic tangent of 2^-11 would move one value in a thousand by a whole step).  The product with t3 keeps
// subnormals, as the rounding does; silu itself is 0 where it is below 2^-119 (t1 < -87.3: the reciprocal's range ends).
__device__ __forceinline__ float mx_silu_mul(float t1, float t3) {
  return mul_keep_subnormals(__fdividef(t1, 1.0f + __expf(-t1)), t3);
}
// The same value, and the two factors of the backward pass: f3 = dh/dt3 = silu(t1), f1 = dh/dt1 = t3 s (1 + t1 (1 - s)).
__device__ __forceinline__ float mx_silu_mul_keep(float& t1, float& t3) {
  const float d = 1.0f + __expf(-t1);
  const float f3 = __fdividef(t1, d), s = __fdividef(1.0f, d);
  const float h = mul_keep_subnormals(f3, t3);
  t1 = t3 * fmaf(f3, 1.0f - s, s);
  t3 = f3;
  return h;
}

// bits of the largest magnitude of 32 values (four chains, for their latency)
__device__ __forceinline__ uint32_t mx_block_top(const float (&v)[32]) {
  float t[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    t[k] = max_abs3(v[k], v[k + 4], v[k + 8]);
    t[k] = max_abs3(t[k], v[k + 12], v[k + 16]);
    t[k] = max_abs3(t[k], v[k + 20], v[k + 24]);
  }
  const float u = max_abs3(max_abs3(t[0], v[28], v[29]), max_abs3(t[1], v[30], v[31]), max_abs3(t[2], t[3], t[3]));
  return __float_as_uint(u) & 0x7FFFFFFFu;
}

// One block (32 values of one row): scale byte and 16 bytes of codes.
__device__ __forceinline__ uint32_t mx_quantize_block(const float (&v)[32], uint4& codes) {
  const uint32_t byte = mx_scale_byte(mx_block_top(v));
  const float inv = mx_inverse_scale(byte);
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float a[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = v[8 * j + i];
    w[j] = mx_round8(a, byte, inv);
  }
  codes = make_uint4(w[0], w[1], w[2], w[3]);
  return byte;
}

// One lane of a converged warp.  The producer and MMA warps run their loops with all lanes and let this one issue: the
// operands of TMA and tcgen05 instructions live in uniform registers, and in a branch that the compiler takes for
// divergent each of them is moved there one by one (about 20 cycles a register: an MMA cost 183 cycles to issue
// whatever its N, a scale copy 60).
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}
// Has the phase completed?  Never blocks (a try_wait may sleep for microseconds on a stage that is not coming).
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok)
               : "r"(smem_u32(bar)), "r"(parity)
               : "memory");
  return ok != 0;
}
// the same bounded wait for all lanes of a warp
__device__ __forceinline__ bool mbar_wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, abort_flag));
}

__device__ __forceinline__ void mx_report(int* status, int code) {
  if (status) atomicCAS(status, 0, code);
}

// Tensor memory.  Two accumulators of 256 columns and 24 columns of scales do not fit into 512, so the second
// accumulator starts 32 columns before the end of the first: the epilogue of a tile reads the shared 32 columns
// first, and from then on (the other accumulator's previous tile being drained) the next tile's MMAs may start.
constexpr uint32_t MX_ACC1 = 224;
constexpr uint32_t MX_SFA = 480;      // 2 atoms x 4 columns
constexpr uint32_t MX_SFB = 488;      // 2 atoms x 8 columns (256 weight rows)

// The instructions of one k-step: scales to tensor memory, four MMAs of 64 values.  lo words of the A and B codes, of
// the A scales [2 atoms] and the B scales [row atom][2 atoms].  `mmas` < 4: the contraction ends inside the step, and
// nothing is issued past its last scale atom.
constexpr uint32_t kAtomLo = kMxAtomBytes >> 4;
template <int CTAS, int TILE_M>
__device__ __forceinline__ void mx_issue_step(uint32_t d, uint32_t tmem, uint32_t a, uint32_t b, uint32_t sa, uint32_t sb, int mmas,
                                              uint32_t accumulate) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    if (2 * j < mmas) {
      tmem_copy_scales<CTAS>(tmem + MX_SFA + 4 * j, sa + j * kAtomLo);
      tmem_copy_scales<CTAS>(tmem + MX_SFB + 8 * j, sb + j * kAtomLo);
      tmem_copy_scales<CTAS>(tmem + MX_SFB + 8 * j + 4, sb + (2 + j) * kAtomLo);
    }
  }
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) {
    if (kk < mmas)
      umma_mxf4<CTAS>(d, a + kk * 2, b + kk * 2, mx_idesc(TILE_M, MX_BN, (kk & 1) * 2), tmem + MX_SFA + 4 * (kk >> 1),
                      tmem + MX_SFB + 8 * (kk >> 1), kk == 0 ? accumulate : 1u);
  }
}

// One row's 32 factors for the backward pass (kept_tile_offset: fp16 with a shared exponent).
__device__ __forceinline__ void mx_keep_block(const float (&v)[32], __half* base, int64_t kept_rows, int64_t row, int n0, int h) {
  const uint32_t byte = kept_scale_byte(mx_block_top(v));
  const float inv = kept_inverse_scale(byte);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (n0 + 8 * j < h) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __half2 t = __floats2half2_rn(v[8 * j + 2 * i] * inv, v[8 * j + 2 * i + 1] * inv);
        w[i] = *reinterpret_cast<const uint32_t*>(&t);
      }
      *reinterpret_cast<uint4*>(base + kept_tile_offset(row, n0 + 8 * j, h)) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  reinterpret_cast<uint8_t*>(base + kept_rows * h)[kept_scale_offset(row, n0, h)] = static_cast<uint8_t>(byte);
}

// Epilogue of one warp: TMEM lane quarter q, columns of `part` of PARTS.  `on_first` runs once after the first chunk has
// been read (the chunk holding the columns the two accumulators share, for the part that has it).
template <int EPI, int PARTS, class F>
__device__ __forceinline__ void mx_epilogue(uint32_t taddr, const MxParams& p, const MxTile& tc, int acc, int row, int part,
                                            unsigned long long dst, uint8_t* stg, int lane, F&& on_first) {
  const bool valid = row < tc.rows;
  if constexpr (!mx_glu(EPI)) {
    constexpr int CH = MX_BN / 32 / PARTS;    // 32-column chunks per part
#pragma unroll 1
    for (int i = 0; i < CH; ++i) {
      // accumulator 0 shares its last chunk, accumulator 1 its first
      const int c = acc == 0 ? (part + 1) * CH - 1 - i : part * CH + i;
      uint32_t v[32];
      tmem_ld_32x32(taddr + c * 32, v);
      tmem_ld_wait();
      if (i == 0) on_first();
      const int n0 = tc.nt * MX_BN + c * 32;
      if (n0 >= p.n_out) continue;            // warp-uniform
      float f[32];
#pragma unroll
      for (int e = 0; e < 32; ++e) f[e] = __uint_as_float(v[e]);
      mx_store_rows(f, dst, n0, p.n_out, stg, lane);
    }
  } else {
    constexpr int HALF = MX_BN / 2;            // gate columns | up columns
    constexpr int CH = HALF / 32 / PARTS;     // blocks of the product per part
    const int64_t drow = tc.routed0 + row;
#pragma unroll 1
    for (int i = 0; i < CH; ++i) {
      // shared columns: up block HALF/32 - 1 of accumulator 0 (the last part's last), gate block 0 of accumulator 1
      const int c = acc == 0 ? (part + 1) * CH - 1 - i : part * CH + i;
      uint32_t g[32], u[32];
      tmem_ld_32x32(taddr + c * 32, g);
      tmem_ld_32x32(taddr + HALF + c * 32, u);
      tmem_ld_wait();
      if (i == 0) on_first();
      const int n0 = tc.nt * HALF + c * 32;
      float a[32], b[32];
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        a[e] = __uint_as_float(g[e]);
        b[e] = __uint_as_float(u[e]);
      }
      float v[32];
      // columns past h are weight rows that do not exist: zeros, whatever their scales hold
      if constexpr (EPI == MX_EPI_GLU_SAVE) {
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = mx_silu_mul_keep(a[e], b[e]);
        if (n0 + 32 > p.n_out) {                // warp-uniform
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (n0 + e >= p.n_out) v[e] = a[e] = b[e] = 0.0f;
        }
        if (valid && n0 < p.n_out) {
          mx_keep_block(a, p.f1, p.kept_rows, drow, n0, p.n_out);
          mx_keep_block(b, p.f3, p.kept_rows, drow, n0, p.n_out);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = n0 + e < p.n_out ? mx_silu_mul(a[e], b[e]) : 0.0f;
      }
      uint4 codes;
      const uint32_t byte = mx_quantize_block(v, codes);
      const int block = tc.nt * (HALF / 32) + c;
      if (valid) {
        // every scale byte of an atom is written, also those of blocks past h (0): the next contraction reads them
        if (n0 < p.n_out) *reinterpret_cast<uint4*>(p.codes + drow * p.code_ld + block * 16) = codes;
        if ((block >> 2) < p.k_atoms_out) p.scales[mx_scale_word(drow, block >> 2, p.k_atoms_out) + (block & 3)] = static_cast<uint8_t>(byte);
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------
// CTAS = 1: one CTA per tile of 128 rows x 256 accumulator columns.  CTAS = 2: a cluster of two CTAs (one TPC) shares
// tcgen05.mma.cta_group::2 of 256 rows x 256 columns: each CTA fetches its own 128 rows of A and half of the weight
// rows (gate/up: the leader the gate rows, the partner the up rows), 35 KiB a k-step instead of 51; the scales of all
// 256 weight rows are needed in both.  The leader (rank 0) issues everything; its `full` barriers count both CTAs'
// bytes, its commits free the stage and publish the accumulator in both, both epilogues report to its `tempty`.
// Persistent, warp specialised: warp 0 producer (TMA), warp 1 scale copies and MMAs, the other warps epilogue.
// ---------------------------------------------------------------------------------------------
// Eight epilogue warps, two a lane quarter: sixteen are slower at every size (FFN 1024/2816, 4099 tokens 39.6 -> 42.6 us,
// 4096/11008, 16384 tokens 0.90 -> 0.94 ms).
template <int EPI, int CTAS> struct MxGeom {
  static constexpr int b_bytes = MX_BN / CTAS * 128;
  static constexpr int stage_bytes = MX_A_BYTES + b_bytes + 3 * MX_SF_BYTES;
  static constexpr int stages = CTAS == 2 ? 5 : 4;
  static constexpr int epi_warps = 8;
  static constexpr int threads = 64 + 32 * epi_warps;
  static constexpr int staging = mx_glu(EPI) ? 0 : epi_warps * 2048;     // a 32-row x 64-byte transposition buffer a warp
  static constexpr int smem = stages * stage_bytes + staging + 256 + 1024;
};

template <int CTAS>
__device__ __forceinline__ void mx_load(void* dst, const CUtensorMap* m, uint64_t* bar, uint32_t lead_bar, int x, int y) {
  if constexpr (CTAS == 1) tma_load_2d(dst, m, bar, x, y);
  else tma_load_2d_pair(dst, m, lead_bar, x, y);
}

template <int EPI, int CTAS>
__global__ void __launch_bounds__(MxGeom<EPI, CTAS>::threads, 1) mx_gemm_kernel(const __grid_constant__ MxMaps maps, const MxParams p) {
  using G = MxGeom<EPI, CTAS>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* staging = smem + G::stages * G::stage_bytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(staging + G::staging);
  uint64_t* empty = full + G::stages;
  uint64_t* tfull = empty + G::stages;     // accumulator ready for the epilogue [2]
  uint64_t* tempty = tfull + 2;            // the epilogue has read the first chunk of a tile
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0);   // warp-uniform for the compiler too
  const int lane = threadIdx.x & 31;
  const int rank = CTAS == 2 ? static_cast<int>(cluster_ctarank()) : 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < G::stages; ++s) {
      mbar_init(&full[s], CTAS);           // one arrive.expect_tx per CTA
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) mbar_init(&tfull[i], 1);
    mbar_init(tempty, G::epi_warps * CTAS);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&maps.a);
    for (int i = 0; i < 4; ++i) tma_prefetch_desc(&maps.b[i]);
    if constexpr (CTAS == 2) {
      tma_prefetch_desc(&maps.tsa);
      for (int i = 0; i < 4; ++i) tma_prefetch_desc(&maps.tsb[i]);
    }
  }
  if (warp == 1) {
    tmem_alloc<CTAS>(tmem_slot, 512);
    tmem_relinquish<CTAS>();
  }
  griddep_launch_dependents();
  tc_fence_before();
  __syncthreads();
  if constexpr (CTAS == 2) cluster_sync_all();   // both CTAs' barriers exist before anybody signals across
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  griddep_wait();

  const int Mv = p.counts[0], Mt = p.counts[1], cap = p.counts[2];
  constexpr int TILE_M = MX_BM * CTAS;
  const int tiles_v = (Mv + TILE_M - 1) / TILE_M;
  const int m_tiles = tiles_v + (Mt + TILE_M - 1) / TILE_M;
  constexpr int N_PER_TILE = mx_glu(EPI) ? MX_BN / 2 : MX_BN;
  const int n_tiles = (p.n_out + N_PER_TILE - 1) / N_PER_TILE;
  const int total = m_tiles * n_tiles;
  const int k_steps = (p.k_bytes + 127) / 128;
  const int first = blockIdx.x / CTAS, step = gridDim.x / CTAS;

  if (warp == 0) {
    int stage = 0, issued = 0;
    uint32_t phase = 0;
    bool ok = true;
    const bool lead = elect_one();
    const uint32_t code_bytes = p.a_rows * 128 + G::b_bytes;
    for (int t = first; t < total && ok; t += step) {
      const MxTile tc = mx_tile(t, TILE_M, rank * MX_BM, tiles_v, m_tiles, n_tiles, p.group_m, Mv, Mt, cap);
      const CUtensorMap* b0 = &maps.b[tc.text ? 2 : 0];
      const uint8_t* sb0 = maps.sb[tc.text ? 2 : 0];
      const uint8_t* sb1 = mx_glu(EPI) ? maps.sb[tc.text ? 3 : 1] : sb0;
      const CUtensorMap* ts0 = &maps.tsb[tc.text ? 2 : 0];
      const int n0 = tc.nt * N_PER_TILE;
      const int sb_row0 = n0 / 128, sb_row1 = mx_glu(EPI) ? sb_row0 : sb_row0 + 1;
      const bool second = sb_row1 < maps.sb_atoms;      // 256 columns may end in their first 128
      for (int ks = 0; ks < k_steps; ++ks) {
        if (!mbar_wait_warp(&empty[stage], phase ^ 1, abort_flag)) {
          if (lead) mx_report(p.status, ST_TIMEOUT_PRODUCER);
          ok = false;
          break;
        }
        if (lead) {
          uint8_t* a = smem + stage * G::stage_bytes;
          uint8_t* b = a + MX_A_BYTES;
          uint8_t* sa = b + G::b_bytes;
          uint8_t* sb = sa + MX_SF_BYTES;
          uint64_t* bar = &full[stage];
          uint32_t lead_bar = smem_u32(bar);
          const uint32_t sf = mx_step_scale_bytes(ks, maps.k_atoms);
          if constexpr (CTAS == 2) {
            lead_bar = mapa_shared(lead_bar, 0);
            mbar_arrive_expect_tx_cluster(lead_bar, code_bytes + 3 * MX_SF_BYTES);
          } else {
            mbar_arrive_expect_tx(bar, code_bytes + (second ? 3 : 2) * sf);
          }
          if constexpr (CTAS == 2) {
            if constexpr (mx_glu(EPI)) mx_load<CTAS>(b, b0 + rank, bar, lead_bar, ks * 128, n0);
            else mx_load<CTAS>(b, b0, bar, lead_bar, ks * 128, n0 + rank * (MX_BN / 2));
          } else {
            mx_load<CTAS>(b, b0, bar, lead_bar, ks * 128, n0);
            if constexpr (mx_glu(EPI)) mx_load<CTAS>(b + G::b_bytes / 2, b0 + 1, bar, lead_bar, ks * 128, n0);
          }
          mx_load<CTAS>(a, &maps.a, bar, lead_bar, ks * 128, static_cast<int>(tc.routed0));
          if constexpr (CTAS == 2) {
            mx_load<CTAS>(sb, ts0, bar, lead_bar, ks * 256, sb_row0);
            if constexpr (mx_glu(EPI)) mx_load<CTAS>(sb + MX_SF_BYTES, ts0 + 1, bar, lead_bar, ks * 256, sb_row0);
            mx_load<CTAS>(sa, &maps.tsa, bar, lead_bar, ks * 256, static_cast<int>(tc.routed0 >> 7));
          } else {
            bulk_load(sb, mx_scale_at(sb0, sb_row0, ks, maps.k_atoms), sf, lead_bar);
            if (second) bulk_load(sb + MX_SF_BYTES, mx_scale_at(sb1, sb_row1, ks, maps.k_atoms), sf, lead_bar);
            bulk_load(sa, mx_scale_at(maps.sa, static_cast<int>(tc.routed0 >> 7), ks, maps.k_atoms), sf, lead_bar);
          }
        }
        __syncwarp();
        ++issued;
        if (++stage == G::stages) { stage = 0; phase ^= 1; }
      }
    }
    if (rank == 0 && *abort_flag && lead) {
      // let the copies already issued land before the CTA gives its shared memory back (pairs: those of both, which the
      // partner waits for at the end)
      for (int i = 0; i < (issued < G::stages ? issued : G::stages); ++i) {
        if (--stage < 0) { stage = G::stages - 1; phase ^= 1; }
        int dummy = 0;
        mbar_wait(&full[stage], phase, &dummy, 1000000ull);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0) {
      int stage = 0, it = 0;
      uint32_t phase = 0;
      bool ok = true;
      const bool lead = elect_one();
      const long long t_begin = clock64();
      long long t_tmem = 0;
      const uint32_t lo0 = mx_desc_lo(smem_u32(smem));
      for (int t = first; t < total && ok; t += step, ++it) {
        const int acc = it & 1;
        const long long tw = clock64();
        if (it != 0 && !mbar_wait_warp(tempty, (it - 1) & 1, abort_flag)) {
          if (lead) mx_report(p.status, ST_TIMEOUT_MMA_TMEM);
          break;
        }
        t_tmem += clock64() - tw;
        tc_fence_after();
        const uint32_t d = tmem + (acc ? MX_ACC1 : 0);
        bool ready = mbar_test(&full[stage], phase);
        for (int ks = 0; ks < k_steps; ++ks) {
          if (!__all_sync(0xFFFFFFFFu, ready) && !mbar_wait_warp(&full[stage], phase, abort_flag)) {
            if (lead) mx_report(p.status, ST_TIMEOUT_MMA_FULL);
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a = lo0 + stage * (G::stage_bytes >> 4);
          const uint32_t b = a + (MX_A_BYTES >> 4), sa = b + (G::b_bytes >> 4), sb = sa + (MX_SF_BYTES >> 4);
          const int left = p.k_bytes - ks * 128;
          uint64_t* free_bar = &empty[stage];
          if (++stage == G::stages) { stage = 0; phase ^= 1; }
          ready = mbar_test(&full[stage], phase);          // asked before the step is issued, looked at after it
          if (lead) {
            if (left >= 128) mx_issue_step<CTAS, TILE_M>(d, tmem, a, b, sa, sb, 4, ks != 0);
            else mx_issue_step<CTAS, TILE_M>(d, tmem, a, b, sa, sb, (left + 31) / 32, ks != 0);
            if constexpr (CTAS == 2) umma_commit_pair(free_bar, 3);
            else umma_commit(free_bar);
          }
          __syncwarp();
        }
        if (ok && lead) {
          if constexpr (CTAS == 2) umma_commit_pair(&tfull[acc], 3);
          else umma_commit(&tfull[acc]);
        }
        __syncwarp();
      }
      if (p.prof && lead) {
        p.prof[blockIdx.x * 8 + 0] = clock64() - t_begin;
        p.prof[blockIdx.x * 8 + 2] = t_tmem;
        p.prof[blockIdx.x * 8 + 7] = it;
      }
    }
    __syncwarp();
  } else {
    const int q = warp & 3, part = (warp - 2) >> 2, row = q * 32 + lane;
    int it = 0;
    const long long t_begin = clock64();
    long long t_wait = 0;
    for (int t = first; t < total; t += step, ++it) {
      const MxTile tc = mx_tile(t, TILE_M, rank * MX_BM, tiles_v, m_tiles, n_tiles, p.group_m, Mv, Mt, cap);
      const int acc = it & 1;
      // where this lane's row goes, looked up while the tile is still being multiplied: the next tile's MMAs wait for
      // this epilogue's first chunk
      unsigned long long dst = 0;
      if (!mx_glu(EPI) && row < tc.rows)
        dst = reinterpret_cast<unsigned long long>(p.out + static_cast<int64_t>(p.perm[tc.list_off + tc.row0 + row]) * p.ldo);
      const long long tw = clock64();
      const bool filled = mbar_wait_warp(&tfull[acc], (it >> 1) & 1, abort_flag);
      t_wait += clock64() - tw;
      if (!filled) {
        if (lane == 0) mx_report(p.status, ST_TIMEOUT_EPILOGUE);
        break;
      }
      tc_fence_after();
      const uint32_t taddr = tmem + (static_cast<uint32_t>(q * 32) << 16) + (acc ? MX_ACC1 : 0);
      mx_epilogue<EPI, G::epi_warps / 4>(taddr, p, tc, acc, row, part, dst, staging + (warp - 2) * 2048, lane, [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (CTAS == 2) mbar_arrive_remote(mapa_shared(smem_u32(tempty), 0));
          else mbar_arrive(tempty);
        }
      });
    }
    if (p.prof && warp == 2 && lane == 0) {
      p.prof[blockIdx.x * 8 + 5] = t_wait;
      p.prof[blockIdx.x * 8 + 6] = clock64() - t_begin;
    }
  }

  tc_fence_before();
  __syncthreads();
  if constexpr (CTAS == 2) cluster_sync_all();   // the partner's shared memory and barriers stay alive until both are done
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<CTAS>(tmem, 512);
  }
}

// ---------------------------------------------------------------------------------------------
// Few row tiles: bound by the stream of weights, or by latency.  A cluster of up to four CTAs owns one tile of 128 rows
// x 128 weight rows of one matrix (gate/up: of both, a CTA takes one of them), the contraction cut into `splits` ranges.
// Every CTA leaves its fp32 partial tile in its own shared memory; after a cluster-wide barrier each CTA adds up a share
// of the rows out of its peers' shared memory, range by range in order (the same bits whichever CTA is last), and
// stores them: bf16 rows in token order, or silu(gate) * up in MXFP4 (a lane holds 4 columns, eight lanes a block).
// Two CTAs fit on an SM (about 100 KiB and 256 tensor-memory columns each), so that one loads while the other adds up.
//
// The weights do not depend on the kernel before this one: launched with programmatic stream serialization, a CTA
// counts the mask itself, asks for its first stages of weights, and only then waits for the activations.
//
// SELF (a handful of tokens): no kernel before this one at all.  Every CTA finds its rows in the mask, rounds their part
// of its contraction range to 4 bits straight into shared memory, in the layout TMA would have given it, while its
// weights are on their way, and the first CTA leaves the routing lists.  One launch less: one token, linear
// 4096 x 4096 7.5 -> 6.3 us, FFN 1024/2816 11.2 -> 10.0 us.
// ---------------------------------------------------------------------------------------------
constexpr int MXS_N = 128;
constexpr int MXS_CLUSTER = 4;                              // CTAs of a cluster at most (mx_small_splits)
constexpr int MXS_THREADS = 192;
constexpr int MXS_B_BYTES = MXS_N * 128;                    // 16 KiB
constexpr int MXS_STAGE_FIXED = MXS_B_BYTES + 2 * MX_SF_BYTES;
constexpr int MXS_MAX_STAGES = 6;
constexpr int MXS_SMEM_STAGES = 104 * 1024;                 // stages, later the partial tile (at most 64 KiB)
constexpr int MXS_SMEM = MXS_SMEM_STAGES + 256 + MX_BM * 4 + 1024;
constexpr int MXS_MASK_MAX = 4096;                          // tokens a CTA counts itself
constexpr uint32_t MXS_SFA = 128, MXS_SFB = 136;            // tensor-memory columns of the scales, behind the accumulator

__device__ __forceinline__ float4 ld_cluster(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

// Cluster-wide barrier that orders nothing: only for "no peer touches my shared memory any more" at the end of the
// kernel (a releasing arrival would wait a microsecond for the stores of the results).
__device__ __forceinline__ void cluster_sync_relaxed() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}

struct MxSmall {
  const uint8_t* mask;    // null: M is larger than a CTA counts
  int M;
  int splits;             // ranges of the contraction; the cluster has splits (gate/up: 2 x splits) CTAs
  int a_slot;             // bytes of a k-step's A rows (a multiple of 1 KiB; what the MMA reads past them is in rows nobody stores)
  int stages;
  // SELF: the activations, the lists to leave, and how many k-steps of A rows shared memory is laid out for
  const __nv_bfloat16* x;
  int64_t ldx;
  int K;
  int x_align;
  int a_steps;
  int* perm;
  int* counts;
  int cap;
};

// Rows `tok[0..rows)` of x, columns of k-steps ks0 ... ks1, to 4 bits in shared memory: codes of k-step i at
// a + i * a_slot as 128-byte rows with the 128-byte swizzle, scales at sa + i * 1 KiB as two atoms.  Four warps, units of
// (row, two k-steps), the loads of four units of a warp in flight together.
__device__ __forceinline__ void mx_self_quantize(const MxSmall& q, const int* tok, int rows, int ks0, int ks1, uint8_t* a, uint8_t* sa,
                                                 int warp, int lane) {
  using L = MxLane<__nv_bfloat16>;
  const int groups = (ks1 - ks0 + 1) / 2, units = rows * groups;
  for (int u0 = warp; u0 < units; u0 += 16) {
    MxRaw raw[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int u = u0 + 4 * i;
      if (u < units) {
        const int row = u / groups, c = (ks0 + 2 * (u - row * groups)) * 256 + lane * L::values;
        raw[i] = load_lane(q.x + static_cast<int64_t>(tok[row]) * q.ldx, c, q.K, q.x_align);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int u = u0 + 4 * i;
      if (u >= units) break;                             // warp-uniform
      const int row = u / groups, ks = 2 * (u - row * groups) + (lane >> 4);   // a k-step is 16 lanes
      uint32_t m = absmax_bits<__nv_bfloat16>(raw[i]);
      m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
      const uint32_t byte = mx_scale_byte(m);
      const float inv = mx_inverse_scale(byte);
      uint32_t code[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = raw_value<__nv_bfloat16>(raw[i], 8 * j + e);
        code[j] = mx_round8(v, byte, inv);
      }
      if (ks0 + ks < ks1) {
        const int piece = (lane & 15) >> 1;              // 16-byte piece of the row = block of the k-step
        *reinterpret_cast<uint2*>(a + ks * q.a_slot + row * 128 + ((piece ^ (row & 7)) << 4) + (lane & 1) * 8) = make_uint2(code[0], code[1]);
        if ((lane & 1) == 0)
          sa[ks * MX_SF_BYTES + (piece >> 2) * kMxAtomBytes + (row & 31) * 16 + (row >> 5) * 4 + (piece & 3)] = static_cast<uint8_t>(byte);
      }
    }
  }
}

template <bool GLU, bool SELF>
__global__ void __launch_bounds__(MXS_THREADS, 2) mx_small_kernel(const __grid_constant__ MxMaps maps, const MxParams p, const MxSmall q) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + MXS_SMEM_STAGES);
  uint64_t* empty = full + MXS_MAX_STAGES;
  uint64_t* done = empty + MXS_MAX_STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* s_count = reinterpret_cast<int*>(tmem_slot + 2);           // one word a warp
  int* s_tok = reinterpret_cast<int*>(smem + MXS_SMEM_STAGES + 256);   // SELF: tokens of this CTA's tile

  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0);
  const int lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const int csize = GLU ? 2 * q.splits : q.splits;
  const int split = GLU ? rank >> 1 : rank, up = GLU ? rank & 1 : 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < MXS_MAX_STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_mbar_init();
    if (!SELF) tma_prefetch_desc(&maps.a);
    tma_prefetch_desc(&maps.b[up]);
    tma_prefetch_desc(&maps.b[2 + up]);
  }
  if (warp == 1) {
    tmem_alloc<1>(tmem_slot, 256);
    tmem_relinquish<1>();
  }
  griddep_launch_dependents();

  // rows of each modality: counted here, or read from what the kernel before left
  int Mv;
  uint32_t vis = 0;                                       // SELF: the visual tokens among the 32 of this thread's warp
  if (SELF || q.mask) {
    int n = 0;
    if constexpr (SELF) {                                 // M <= 128: warp w < 4 holds tokens 32 w ... 32 w + 31
      const int i = threadIdx.x;
      vis = __ballot_sync(0xFFFFFFFFu, i < q.M && q.mask[i] != 0);
      n = __popc(vis);
    } else {
      for (int i = threadIdx.x; i < q.M; i += MXS_THREADS) n += q.mask[i] != 0 ? 1 : 0;
      n = __reduce_add_sync(0xFFFFFFFFu, n);
    }
    if (lane == 0) {
      s_count[warp] = n;
      if constexpr (SELF) s_count[MXS_THREADS / 32 + warp] = static_cast<int>(vis);
    }
    tc_fence_before();
    __syncthreads();
    Mv = 0;
    for (int i = 0; i < MXS_THREADS / 32; ++i) Mv += s_count[i];
  } else {
    tc_fence_before();
    __syncthreads();
    griddep_wait();
    Mv = p.counts[0];
  }
  tc_fence_after();
  const int Mt = q.M - Mv;
  const uint32_t tmem = *tmem_slot;
  const int tiles_v = (Mv + MX_BM - 1) / MX_BM;
  const int m_tiles = tiles_v + (Mt + MX_BM - 1) / MX_BM;
  const int n_tiles = (p.n_out + MXS_N - 1) / MXS_N;
  const int t = blockIdx.x / csize;                       // the same in the whole cluster
  const bool work = t < m_tiles * n_tiles;
  const int nt = work ? t / m_tiles : 0;
  const int mt = work ? t - nt * m_tiles : 0;
  const bool text = mt >= tiles_v;
  const int row0 = (text ? mt - tiles_v : mt) * MX_BM;
  const int rows = work ? min(MX_BM, (text ? Mt : Mv) - row0) : 0;
  const int routed0 = (text ? mx_text_base(Mv) : 0) + row0;
  const int k_steps = (p.k_bytes + 127) / 128;
  const int ks0 = split * k_steps / q.splits, ks1 = work ? (split + 1) * k_steps / q.splits : ks0;
  // SELF: [A of every k-step][A scales of every k-step][stages of B, B scales]; else stages of A, B, A scales, B scales
  const int stage_bytes = SELF ? MXS_B_BYTES + MX_SF_BYTES : q.a_slot + MXS_STAGE_FIXED;
  const int b_base = SELF ? q.a_steps * (q.a_slot + MX_SF_BYTES) : q.a_slot;
  constexpr int sb_off = SELF ? MXS_B_BYTES : MXS_B_BYTES + MX_SF_BYTES;   // of a stage's B scales behind its B codes

  if constexpr (SELF) {
    const int i = threadIdx.x;
    if (i < q.M) {
      int before = __popc(vis & ((1u << lane) - 1u));     // visual tokens before this one
      for (int w = 0; w < warp; ++w) before += s_count[w];
      const bool v = (vis >> lane) & 1u;
      const int pos = v ? before : i - before;
      if (v != text) s_tok[pos] = i;
      if (blockIdx.x == 0) q.perm[(v ? 0 : q.cap) + pos] = i;
    }
    if (blockIdx.x == 0 && i == 0) {
      int runs = 1;
      for (int k = 0; k < q.M; k += 32) {                 // changes of modality between neighbouring tokens
        const uint32_t v = static_cast<uint32_t>(s_count[MXS_THREADS / 32 + (k >> 5)]);
        const int n = min(32, q.M - k);
        runs += __popc((v ^ (v >> 1)) & ((1u << (n - 1)) - 1u));
        if (k + 32 < q.M) runs += ((v >> 31) ^ static_cast<uint32_t>(s_count[MXS_THREADS / 32 + (k >> 5) + 1])) & 1u;
      }
      q.counts[0] = Mv;
      q.counts[1] = Mt;
      q.counts[2] = q.cap;
      q.counts[3] = q.M;
      q.counts[4] = runs;
    }
    __syncthreads();
  }

  if (warp == 0) {
    const bool lead = elect_one();
    const CUtensorMap* mb = &maps.b[(text ? 2 : 0) + up];
    const uint8_t* sb = maps.sb[(text ? 2 : 0) + up];
    const uint32_t code_bytes = (SELF ? 0 : p.a_rows * 128) + MXS_B_BYTES;
    int issued = 0;
    auto load_b = [&](int ks, int stage) {
      uint8_t* b = smem + stage * stage_bytes + b_base;
      const uint32_t sf = mx_step_scale_bytes(ks, maps.k_atoms);
      mbar_arrive_expect_tx(&full[stage], code_bytes + (SELF ? 1 : 2) * sf);
      tma_load_2d(b, mb, &full[stage], ks * 128, nt * MXS_N);
      bulk_load(b + sb_off, mx_scale_at(sb, nt, ks, maps.k_atoms), sf, smem_u32(&full[stage]));
    };
    auto load_a = [&](int ks, int stage) {
      if constexpr (SELF) return;
      uint8_t* a = smem + stage * stage_bytes;
      tma_load_2d(a, &maps.a, &full[stage], ks * 128, routed0);
      bulk_load(a + q.a_slot + MXS_B_BYTES, mx_scale_at(maps.sa, routed0 >> 7, ks, maps.k_atoms),
                mx_step_scale_bytes(ks, maps.k_atoms), smem_u32(&full[stage]));
    };
    const int ahead = min(q.stages, ks1 - ks0);
    if (lead)
      for (int i = 0; i < ahead; ++i) load_b(ks0 + i, i);
    griddep_wait();                                       // the activations are there from here on
    if (lead)
      for (int i = 0; i < ahead; ++i) load_a(ks0 + i, i);
    __syncwarp();
    issued = ahead;
    int stage = 0;
    uint32_t phase = 0;
    if (ahead == q.stages) phase = 1;
    else stage = ahead;
    for (int ks = ks0 + ahead; ks < ks1; ++ks) {
      if (!mbar_wait_warp(&empty[stage], phase ^ 1, abort_flag)) {
        if (lead) mx_report(p.status, ST_TIMEOUT_PRODUCER);
        break;
      }
      if (lead) {
        load_b(ks, stage);
        load_a(ks, stage);
      }
      __syncwarp();
      ++issued;
      if (++stage == q.stages) { stage = 0; phase ^= 1; }
    }
    if (*abort_flag && lead) {
      for (int i = 0; i < (issued < q.stages ? issued : q.stages); ++i) {
        if (--stage < 0) { stage = q.stages - 1; phase ^= 1; }
        int dummy = 0;
        mbar_wait(&full[stage], phase, &dummy, 1000000ull);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    const bool lead = elect_one();
    const uint32_t lo0 = mx_desc_lo(smem_u32(smem));
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    if constexpr (SELF) asm volatile("bar.sync 1, 160;" ::: "memory");        // the activations are in shared memory
    auto issue = [&](uint32_t a, uint32_t b, uint32_t sa, uint32_t sb, int mmas, uint32_t accumulate) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (2 * j < mmas) {
          tmem_copy_scales<1>(tmem + MXS_SFA + 4 * j, sa + j * kAtomLo);
          tmem_copy_scales<1>(tmem + MXS_SFB + 4 * j, sb + j * kAtomLo);
        }
      }
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        if (kk < mmas)
          umma_mxf4<1>(tmem, a + kk * 2, b + kk * 2, mx_idesc(MX_BM, MXS_N, (kk & 1) * 2), tmem + MXS_SFA + 4 * (kk >> 1),
                       tmem + MXS_SFB + 4 * (kk >> 1), kk == 0 ? accumulate : 1u);
      }
    };
    bool ready = ks0 < ks1 && mbar_test(&full[0], 0);
    for (int ks = ks0; ks < ks1; ++ks) {
      if (!__all_sync(0xFFFFFFFFu, ready) && !mbar_wait_warp(&full[stage], phase, abort_flag)) {
        if (lead) mx_report(p.status, ST_TIMEOUT_MMA_FULL);
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t st = lo0 + stage * (stage_bytes >> 4);
      const uint32_t b = st + (b_base >> 4), sb = b + (sb_off >> 4);
      const uint32_t a = SELF ? lo0 + (ks - ks0) * (q.a_slot >> 4) : st;
      const uint32_t sa = SELF ? lo0 + ((q.a_steps * q.a_slot + (ks - ks0) * MX_SF_BYTES) >> 4) : b + (MXS_B_BYTES >> 4);
      const int left = p.k_bytes - ks * 128;
      uint64_t* free_bar = &empty[stage];
      if (++stage == q.stages) { stage = 0; phase ^= 1; }
      ready = mbar_test(&full[stage], phase);
      if (lead) {
        if (left >= 128) issue(a, b, sa, sb, 4, ks != ks0);
        else issue(a, b, sa, sb, (left + 31) / 32, ks != ks0);
        umma_commit(free_bar);
      }
      __syncwarp();
    }
    if (lead && ok) umma_commit(done);
    __syncwarp();
  } else {
    if constexpr (SELF) {
      mx_self_quantize(q, s_tok, rows, ks0, ks1, smem, smem + q.a_steps * q.a_slot, warp - 2, lane);
      fence_proxy_async_smem();
      asm volatile("bar.sync 1, 160;" ::: "memory");
    }
    // the partial tile to shared memory, [row][32 pieces of four columns], pieces XOR-swizzled by the row
    const int quarter = warp & 3, row = quarter * 32 + lane;
    if (quarter * 32 < rows) {
      if (!mbar_wait_warp(done, 0, abort_flag)) {
        if (lane == 0) mx_report(p.status, ST_TIMEOUT_EPILOGUE);
      } else {
        tc_fence_after();
        const uint32_t taddr = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t v[32];
          tmem_ld_32x32(taddr + c * 32, v);
          tmem_ld_wait();
          if (row < rows) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              *reinterpret_cast<uint4*>(smem + row * 512 + (((c * 8 + j) ^ (row & 31)) << 4)) =
                  make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          }
        }
      }
    }
  }
  griddep_wait();                                         // every thread: perm is read below
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                                     // every partial tile of the cluster is in place

  // This CTA's rows are rank, rank + csize, ...; a warp takes two of them at a time, so that twice the remote loads are
  // under way.
  for (int r0 = rank + csize * warp; r0 < rows; r0 += 2 * csize * (MXS_THREADS / 32)) {
    float4 sum[2][2] = {};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = r0 + h * csize * (MXS_THREADS / 32);
      if (row < rows) {
        const uint32_t mine = smem_u32(smem + row * 512 + ((lane ^ (row & 31)) << 4));
        float4 v[MXS_CLUSTER];
#pragma unroll
        for (int i = 0; i < MXS_CLUSTER; ++i)
          if (i < csize) v[i] = ld_cluster(mapa_shared(mine, i));
#pragma unroll
        for (int i = 0; i < MXS_CLUSTER; ++i) {
          if (i < csize) {
            float4& d = sum[h][GLU ? i & 1 : 0];
            d.x += v[i].x; d.y += v[i].y; d.z += v[i].z; d.w += v[i].w;
          }
        }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = r0 + h * csize * (MXS_THREADS / 32);
      if (row >= rows) break;                             // warp-uniform
      const float4 g = sum[h][0], u = sum[h][1];
      const int n0 = nt * MXS_N + lane * 4;
      if constexpr (!GLU) {
        if (n0 < p.n_out) {
          const int64_t token = SELF ? s_tok[row] : p.perm[(text ? p.counts[2] : 0) + row0 + row];
          *reinterpret_cast<uint2*>(p.out + token * p.ldo + n0) = make_uint2(mx_pack_bf16(g.x, g.y), mx_pack_bf16(g.z, g.w));
        }
      } else {
        const int64_t drow = routed0 + row;
        float v[8] = {};
        if (p.f1) {                                         // uniform: the factors of the backward pass are kept
          float t[4] = {g.x, g.y, g.z, g.w}, w[4] = {u.x, u.y, u.z, u.w};
          uint32_t m1 = 0, m3 = 0;
          if (n0 < p.n_out) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              v[i] = mx_silu_mul_keep(t[i], w[i]);
              m1 = max(m1, __float_as_uint(t[i]) & 0x7FFFFFFFu);
              m3 = max(m3, __float_as_uint(w[i]) & 0x7FFFFFFFu);
            }
          }
#pragma unroll
          for (int o = 1; o < 8; o <<= 1) {
            m1 = max(m1, __shfl_xor_sync(0xFFFFFFFFu, m1, o));
            m3 = max(m3, __shfl_xor_sync(0xFFFFFFFFu, m3, o));
          }
          const uint32_t k1 = kept_scale_byte(m1), k3 = kept_scale_byte(m3);
          if (n0 < p.n_out) {
            const float i1 = kept_inverse_scale(k1), i3 = kept_inverse_scale(k3);
            const int64_t o = kept_tile_offset(drow, n0, p.n_out);
            const __half2 h1[2] = {__floats2half2_rn(t[0] * i1, t[1] * i1), __floats2half2_rn(t[2] * i1, t[3] * i1)};
            const __half2 h3[2] = {__floats2half2_rn(w[0] * i3, w[1] * i3), __floats2half2_rn(w[2] * i3, w[3] * i3)};
            *reinterpret_cast<uint2*>(p.f1 + o) = make_uint2(*reinterpret_cast<const uint32_t*>(&h1[0]), *reinterpret_cast<const uint32_t*>(&h1[1]));
            *reinterpret_cast<uint2*>(p.f3 + o) = make_uint2(*reinterpret_cast<const uint32_t*>(&h3[0]), *reinterpret_cast<const uint32_t*>(&h3[1]));
            if ((lane & 7) == 0) {
              const int64_t so = kept_scale_offset(drow, n0, p.n_out);
              reinterpret_cast<uint8_t*>(p.f1 + p.kept_rows * p.n_out)[so] = static_cast<uint8_t>(k1);
              reinterpret_cast<uint8_t*>(p.f3 + p.kept_rows * p.n_out)[so] = static_cast<uint8_t>(k3);
            }
          }
        } else if (n0 < p.n_out) {
          v[0] = mx_silu_mul(g.x, u.x);
          v[1] = mx_silu_mul(g.y, u.y);
          v[2] = mx_silu_mul(g.z, u.z);
          v[3] = mx_silu_mul(g.w, u.w);
        }
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
        const uint32_t byte = mx_scale_byte(m);
        const uint32_t code = mx_round8(v, byte, mx_inverse_scale(byte));
        const int block = nt * 4 + (lane >> 3);
        if (block * 32 < p.n_out) *reinterpret_cast<uint16_t*>(p.codes + drow * p.code_ld + block * 16 + (lane & 7) * 2) = static_cast<uint16_t>(code);
        if ((lane & 7) == 0) p.scales[mx_scale_word(drow, nt, p.k_atoms_out) + (lane >> 3)] = static_cast<uint8_t>(byte);
      }
    }
  }
  cluster_sync_relaxed();                                 // nobody leaves while a peer still reads its shared memory
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<1>(tmem, 256);
  }
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
struct MxWeight {
  const void* codes;
  const void* scales;
};

// codes [rows, ld bytes], boxes of 128 bytes x box_rows; a box past the end reads zeros
static int mx_code_map(CUtensorMap* m, const void* codes, int64_t rows, int64_t cols, int box_rows) {
  return make_tensor_map_2d_of(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, codes, mx_code_ld(cols), rows, mx_code_ld(cols), 128, box_rows,
                               CU_TENSOR_MAP_SWIZZLE_128B);
}

static int mx_scale_map(CUtensorMap* m, const void* scales, int64_t rows, int64_t cols, int box_atoms) {
  return make_tensor_map_2d_of(m, CU_TENSOR_MAP_DATA_TYPE_UINT32, scales, mx_k_atoms(cols) * (kMxAtomBytes / 4), mx_row_atoms(rows),
                               mx_k_atoms(cols) * kMxAtomBytes, 256, box_atoms, CU_TENSOR_MAP_SWIZZLE_NONE);
}

// `n` weights [n_rows, k] (slot i of maps.b / maps.sb is weight slots[i]) and the routed activations of M tokens
static int mx_maps(MxMaps& m, const MxWeight& a, int64_t M, const MxWeight* w, const int* slots, int n, int64_t n_rows, int64_t k,
                   int a_box, int b_box, int pair_sb_box) {
  const int64_t a_rows = ffnk_route_capacity(M) + 512;
  int r = a.codes ? mx_code_map(&m.a, a.codes, a_rows, k, a_box) : 0;     // no codes yet: the kernel rounds the rows itself
  if (r) return r;
  if (pair_sb_box && (r = mx_scale_map(&m.tsa, a.scales, a_rows, k, 1))) return r;
  m.sa = static_cast<const uint8_t*>(a.scales);
  for (int i = 0; i < n; ++i) {
    if ((r = mx_code_map(&m.b[slots[i]], w[i].codes, n_rows, k, b_box))) return r;
    if (pair_sb_box && (r = mx_scale_map(&m.tsb[slots[i]], w[i].scales, n_rows, k, pair_sb_box))) return r;
    m.sb[slots[i]] = static_cast<const uint8_t*>(w[i].scales);
  }
  m.k_atoms = static_cast<int>(mx_k_atoms(k));
  m.sb_atoms = static_cast<int>(mx_row_atoms(n_rows));
  return 0;
}

// Row tiles of a super-tile: about 16 MiB of activation codes stay in L2 while the weights pass.
static int mx_group_m(int64_t k, int64_t rows_per_tile) {
  int64_t g = (16ll << 20) / (rows_per_tile * mx_code_ld(k) + 1);
  return static_cast<int>(g < 4 ? 4 : (g > 64 ? 64 : g));
}

static int mx_a_box_rows(int64_t M) { return M >= MX_BM || tune_overrides().pair > 0 ? MX_BM : static_cast<int>((M + 7) / 8 * 8); }

// CTA pairs or single CTAs.  Pairs halve the weight traffic of an SM but hand tiles out in twice the size and pay for
// signals between the two: worth it for long contractions, or for many rows; the gate/up tiles, with their longer epilogue,
// later.  Measured (single / pairs, us): linear 1024 -> 1024, 4096 tokens 14.4 / 14.9, 32768 tokens 50.4 / 48.8; 1024 -> 4096,
// 8192 tokens 34.0 / 32.8; 1536 -> 4096, 1500 tokens 18.1 / 16.2, 8192 tokens 39.6 / 37.4; 4096 x 4096, 1000 tokens 21.0 / 23.8,
// 8192 tokens 76.9 / 72.6; FFN with pairs for the second product, gate/up single / pairs: 2048/5504, 1500 tokens 38.2 / 40.3,
// 4096 tokens 69.3 / 70.4, with gradient 376 / 359; 4096/11008, 4096 tokens 219 / 217; 1024/2816, 16384 tokens 83.4 / 88.7.
static bool mx_pairs(int64_t M, int64_t k, bool glu) {
  const int forced = tune_overrides().pair;
  if (forced >= 0) return forced != 0;
  return glu ? M > 2048 && k >= 2048 : (M > 1024 && k >= 1536) || (M >= 8192 && k >= 1024);
}

// Dynamic shared memory of a kernel
template <class K>
static int mx_allow_smem(K kernel, int bytes, std::atomic<uint64_t>& allowed) {
  return once_per_device(allowed, [&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes); });
}

template <int EPI, int CTAS>
static int mx_launch_as(const MxMaps& maps, const MxParams& p, int64_t M, cudaStream_t stream) {
  const int n_per_tile = mx_glu(EPI) ? MX_BN / 2 : MX_BN;
  int64_t units = ((M + MX_BM * CTAS - 1) / (MX_BM * CTAS) + 1) * ((p.n_out + n_per_tile - 1) / n_per_tile);
  if (units > usable_sms() / CTAS) units = usable_sms() / CTAS;
  static std::atomic<uint64_t> allowed{0};
  if (const int r = mx_allow_smem(mx_gemm_kernel<EPI, CTAS>, MxGeom<EPI, CTAS>::smem, allowed)) return r;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(units * CTAS));
  cfg.blockDim = dim3(MxGeom<EPI, CTAS>::threads);
  cfg.dynamicSmemBytes = MxGeom<EPI, CTAS>::smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (CTAS == 2) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = CTAS;
    attr[n].val.clusterDim.y = 1;
    attr[n++].val.clusterDim.z = 1;
  }
  if (M < 4096 && tune_overrides().early_start != 0) {
    // few tiles leave SMs idle while the kernel before runs: set up beside it
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cuda_status(cudaLaunchKernelEx(&cfg, mx_gemm_kernel<EPI, CTAS>, maps, p));
}

template <int EPI>
static int mx_launch(const MxMaps& maps, const MxParams& p, int64_t M, bool pairs, cudaStream_t stream) {
  if (device_info().cc_major != 10) return FFNK_ERR_DEVICE;
  return pairs ? mx_launch_as<EPI, 2>(maps, p, M, stream) : mx_launch_as<EPI, 1>(maps, p, M, stream);
}

// Ranges of the contraction for the small kernel, 0: not the small kernel.
// Plain products: one row tile a modality, and more of them where 128 x 256 tiles would leave most SMs idle for a long
// contraction: one that can be cut into four ranges, or into two that are still long, while the rows do not outgrow it.
// Gate/up: up to 64 rows, whose longer tail (two matrices added up, rounded to 4 bits) still costs less than the few 128 x 256
// tiles; up to 16 where its CTAs, both modalities present, need a second wave.
// Measured (whole call by graph replay, small / 128 x 256 tiles, us): linear 4096 x 4096 1 token 6.6 / 11.0, 127 tokens 12.1 / 14.4,
// 200 tokens 14.8 / 14.8 (two ranges), 512 tokens 23.1 / 17.3 (one); 4096 -> 1024, 512 tokens (four) 13.2 / 14.8; 11008 -> 4096,
// 300 tokens (two) 24.7 / 27.6; 16384 -> 1024, 1024 tokens (four) 27.4 / 38.4, 2048 tokens (two) 40.3 / 40.8.
// Gate/up one way or the other, one modality, and both: FFN 1024/2816, 48 tokens 12.8 / 13.6, 12.8 / 13.6; 64 tokens
// 13.6 / 14.0, 13.2 / 13.6; 96 tokens 14.9 / 14.6, 14.5 / 14.2; FFN 4096/11008 (second wave), 16 tokens 23.7 / 26.2,
// 40.1 / 36.4; 32 tokens 25.2 / 26.7, 40.7 / 37.1.
// The number of ranges: as many as fill the places on the GPU once (two CTAs an SM), at most four, which always beat
// eight (linear 4096 x 4096, 64 tokens: 1 / 2 / 4 / 8 ranges 13.3 / 11.0 / 10.7 / 18.6 us).  Gate/up tiles take two ranges
// only where those CTAs nearly fit one an SM (FFN 512/1024, 64 tokens: 12.3 / 11.5 / 12.0 us with 1 / 2 / 4; FFN 4096/11008,
// 8 tokens 38.0 / 38.4 / 49.5 us).
static int mx_small_splits(int64_t M, int64_t n_out, int64_t k, bool glu) {
  const int forced = tune_overrides().narrow;
  const int64_t steps = (mx_code_ld(k) + 127) / 128, places = 2 * usable_sms();
  if (forced == 0) return 0;
  const int64_t m_tiles = (M + MX_BM - 1) / MX_BM + (M > 1 ? 1 : 0);
  const int64_t tiles = m_tiles * ((n_out + MXS_N - 1) / MXS_N) * (glu ? 2 : 1);
  const int64_t most = glu ? usable_sms() * 5 / 4 : places;
  int splits = 1;
  while (splits < (glu ? MXS_CLUSTER / 2 : MXS_CLUSTER) && tiles * splits * 2 <= most && steps >= splits * 2) splits *= 2;
  const bool fits = glu ? M <= (tiles <= places ? 64 : 16)
                        : M <= MX_BM || (M <= 32 * steps && splits > 1 && splits * steps >= 64);
  return fits || forced > 0 ? splits : 0;
}

// The activations of a call that a small kernel rounds itself (SELF), and where it leaves the routing lists.
struct MxSelf {
  const void* x;
  int64_t ldx;
  int32_t* perm;
  int32_t* counts;
};
// Does it?  At most 16 (row, two k-steps) units a CTA, whose loads its four warps have in flight at once; and room for all of
// A beside three stages of B.  Measured (itself / a kernel before it, whole call by graph replay, us): linear 2048 x 2048, 8 tokens
// 6.2 / 7.0, 16 tokens (16 units) 7.0 / 7.0, 24 tokens 7.9 / 7.0; 4096 x 4096, 4 tokens 7.5 / 7.4, 16 tokens (32 units)
// 9.1 / 7.5; FFN 4096/11008, 2 tokens (16 units) 23.6 / 22.7, 4 tokens (32) 25.4 / 22.6; the launch saved is 2 us of the host's time.
static bool mx_takes_self(int64_t M, int64_t k, int splits) {
  if (splits == 0 || M > MX_BM || tune_overrides().permute == 0) return false;
  const int64_t steps = ((mx_code_ld(k) + 127) / 128 + splits - 1) / splits;
  return M * ((steps + 1) / 2) <= 16 && steps * (((M + 7) / 8) * 1024 + MX_SF_BYTES) + 3 * (MXS_B_BYTES + MX_SF_BYTES) <= MXS_SMEM_STAGES;
}

template <bool GLU, bool SELF>
static int mx_launch_small(const MxMaps& maps, const MxParams& p, int64_t M, int64_t k, const void* mask, int splits, const MxSelf& self,
                           cudaStream_t stream) {
  if (device_info().cc_major != 10) return FFNK_ERR_DEVICE;
  MxSmall q{};
  q.mask = M <= MXS_MASK_MAX ? static_cast<const uint8_t*>(mask) : nullptr;
  q.M = static_cast<int>(M);
  q.splits = splits;
  q.a_slot = (p.a_rows * 128 + 1023) & ~1023;
  q.stages = MXS_SMEM_STAGES / (q.a_slot + MXS_STAGE_FIXED);
  if constexpr (SELF) {
    q.x = static_cast<const __nv_bfloat16*>(self.x);
    q.ldx = self.ldx;
    q.K = static_cast<int>(k);
    q.x_align = (reinterpret_cast<uintptr_t>(self.x) | static_cast<uintptr_t>(2 * self.ldx)) & 31 ? 16 : 32;
    q.perm = self.perm;
    q.counts = self.counts;
    q.cap = static_cast<int>(ffnk_route_capacity(M));
    q.a_steps = static_cast<int>(((mx_code_ld(k) + 127) / 128 + splits - 1) / splits);
    q.stages = (MXS_SMEM_STAGES - q.a_steps * (q.a_slot + MX_SF_BYTES)) / (MXS_B_BYTES + MX_SF_BYTES);
  }
  if (q.stages > MXS_MAX_STAGES) q.stages = MXS_MAX_STAGES;
  const int csize = GLU ? 2 * splits : splits;
  const int64_t tiles = ((M + MX_BM - 1) / MX_BM + (M > 1 ? 1 : 0)) * ((p.n_out + MXS_N - 1) / MXS_N);
  static std::atomic<uint64_t> allowed{0};
  if (const int r = mx_allow_smem(mx_small_kernel<GLU, SELF>, MXS_SMEM, allowed)) return r;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * csize));
  cfg.blockDim = dim3(MXS_THREADS);
  cfg.dynamicSmemBytes = MXS_SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = csize;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = !SELF && tune_overrides().early_start != 0 ? 2 : 1;    // SELF is a call's first kernel: it reads x at once
  return cuda_status(cudaLaunchKernelEx(&cfg, mx_small_kernel<GLU, SELF>, maps, p, q));
}

// y[token] = routed rows of (codes, scales) by the modality's weight [N, K].  `splits`: mx_small_splits, asked once by the
// caller, who decides by it what the kernel finds (overrides and the SM margin are process-wide and may change meanwhile)
static int mx_product(const MxWeight& a, const MxWeight& wv, const MxWeight& wt, const int32_t* perm, const int32_t* counts,
                      const void* mask, void* y, int64_t ldy, int64_t M, int64_t N, int64_t K, int splits, const MxSelf* self,
                      int32_t* status, cudaStream_t s) {
  const bool pairs = mx_pairs(M, K, false);
  const int a_box = mx_a_box_rows(M);
  const MxWeight w[2] = {wv, wt};
  const int slots[2] = {0, 2};
  MxMaps m{};
  const int r = mx_maps(m, a, M, w, slots, 2, N, K, a_box, splits ? MXS_N : pairs ? MX_BN / 2 : MX_BN,
                        pairs && !splits ? 2 : 0);
  if (r) return r;
  m.b[1] = m.b[0];
  m.b[3] = m.b[2];
  m.tsb[1] = m.tsb[0];
  m.tsb[3] = m.tsb[2];
  MxParams p{};
  p.perm = perm; p.counts = counts; p.status = status; p.prof = debug_profile_buffer();
  p.n_out = static_cast<int>(N);
  p.k_bytes = static_cast<int>(mx_code_ld(K));
  p.a_rows = a_box;
  p.group_m = mx_group_m(K, pairs ? 2 * MX_BM : MX_BM);
  p.out = static_cast<__nv_bfloat16*>(y);
  p.ldo = ldy;
  if (self) return mx_launch_small<false, true>(m, p, M, K, mask, splits, *self, s);
  return splits ? mx_launch_small<false, false>(m, p, M, K, mask, splits, MxSelf{}, s) : mx_launch<MX_EPI_STORE>(m, p, M, pairs, s);
}

// quantised silu(gate) * up of the routed rows, optionally with the factors of the backward pass kept (f1, f3 both or neither)
static int mx_gateup(const MxWeight& a, const MxWeight (&w)[4], const int32_t* perm, const int32_t* counts, void* codes,
                     void* scales, const void* mask, void* f1, void* f3, int64_t M, int64_t d, int64_t h, int splits,
                     const MxSelf* self, int32_t* status, cudaStream_t s) {
  const int slots[4] = {0, 1, 2, 3};
  const bool pairs = mx_pairs(M, d, true);
  const int a_box = mx_a_box_rows(M);
  MxMaps m{};
  const int r = mx_maps(m, a, M, w, slots, 4, h, d, a_box, MX_BN / 2, pairs && !splits ? 1 : 0);
  if (r) return r;
  MxParams p{};
  p.perm = perm; p.counts = counts; p.status = status; p.prof = debug_profile_buffer();
  p.n_out = static_cast<int>(h);
  p.k_bytes = static_cast<int>(mx_code_ld(d));
  p.a_rows = a_box;
  p.group_m = mx_group_m(d, pairs ? 2 * MX_BM : MX_BM);
  p.codes = static_cast<uint8_t*>(codes);
  p.scales = static_cast<uint8_t*>(scales);
  p.code_ld = mx_code_ld(h);
  p.k_atoms_out = static_cast<int>(mx_k_atoms(h));
  p.f1 = static_cast<__half*>(f1);
  p.f3 = static_cast<__half*>(f3);
  p.kept_rows = ffnk_route_capacity(M) + 512;
  if (self) return mx_launch_small<true, true>(m, p, M, d, mask, splits, *self, s);
  if (splits) return mx_launch_small<true, false>(m, p, M, d, mask, splits, MxSelf{}, s);
  return f1 ? mx_launch<MX_EPI_GLU_SAVE>(m, p, M, pairs, s) : mx_launch<MX_EPI_GLU>(m, p, M, pairs, s);
}

static int64_t mx_align(int64_t v) { return (v + 255) & ~int64_t(255); }

// Workspace of one call.  The routing lists come first and have a size of their own, because a backward pass needs
// them again; everything else is scratch.
struct MxWorkspace {
  int64_t scan, xc, xs, hc, hs, total;
};
static MxWorkspace mx_workspace(int64_t M, int64_t K, int64_t h) {
  MxWorkspace w{};
  const int64_t rows = ffnk_route_capacity(M) + 512;
  int64_t off = 0;
  w.scan = off; off += mx_align(ffnk_route_workspace_bytes(M));
  w.xc = off;   off += mx_align(rows * mx_code_ld(K));
  w.xs = off;   off += mx_align(mx_row_atoms(rows) * mx_k_atoms(K) * kMxAtomBytes);
  w.hc = off;   off += h ? mx_align(rows * mx_code_ld(h)) : 0;
  w.hs = off;   off += h ? mx_align(mx_row_atoms(rows) * mx_k_atoms(h) * kMxAtomBytes) : 0;
  w.total = off;
  return w;
}

static bool mx_bad_dim(int64_t v) { return v < 8 || (v & 7) || v >= (1ll << 30); }
static bool misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

}  // namespace ffnk

using namespace ffnk;

extern "C" int64_t ffnk_mxfp4_kept_bytes(int64_t M, int64_t h) {
  if (M <= 0 || h <= 0) return 256;
  const int64_t rows = ffnk_route_capacity(M) + 512;
  return rows * h * 2 + rows * ((h + 31) / 32);
}

extern "C" int64_t ffnk_mxfp4_workspace_bytes(int64_t M, int64_t K, int64_t h) {
  if (M <= 0 || K <= 0 || h < 0) return 256;
  return mx_workspace(M, K, h).total;
}

extern "C" int ffnk_mxfp4_linear_forward(const void* x, int64_t ldx, const void* b1_codes, const void* b1_scales,
                                         const void* b2_codes, const void* b2_scales, const void* mask, int32_t* perm,
                                         int32_t* counts, void* workspace, int64_t workspace_bytes, void* y, int64_t ldy,
                                         int64_t M, int64_t N, int64_t K, int32_t* status, void* stream) {
  if (M == 0) return 0;
  if (!x || !b1_codes || !b1_scales || !b2_codes || !b2_scales || !mask || !perm || !counts || !workspace || !y || !status)
    return FFNK_ERR_NULL;
  if (M < 0 || M >= (1ll << 30) || mx_bad_dim(N) || mx_bad_dim(K)) return FFNK_ERR_SHAPE;
  if ((ldx & 7) || (ldy & 7) || ldx < K || ldy < N || misaligned(x) || misaligned(y) || misaligned(b1_codes) ||
      misaligned(b1_scales) || misaligned(b2_codes) || misaligned(b2_scales) || misaligned(perm) ||
      (reinterpret_cast<uintptr_t>(workspace) & 255))
    return FFNK_ERR_ALIGN;
  const MxWorkspace w = mx_workspace(M, K, 0);
  if (workspace_bytes < w.total) return FFNK_ERR_CAPACITY;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const MxSelf self{x, ldx, perm, counts};
  const int splits = mx_small_splits(M, N, K, false);
  const bool takes = mx_takes_self(M, K, splits);
  int r = takes ? 0 : mx_route_quantize(mask, M, x, ldx, K, perm, counts, ws + w.scan, ws + w.xc, ws + w.xs, status, stream);
  if (r) return r;
  return mx_product(takes ? MxWeight{} : MxWeight{ws + w.xc, ws + w.xs}, MxWeight{b1_codes, b1_scales},
                    MxWeight{b2_codes, b2_scales}, perm, counts, mask, y, ldy, M, N, K, splits, takes ? &self : nullptr, status,
                    static_cast<cudaStream_t>(stream));
}

extern "C" int ffnk_mxfp4_ffn_forward(const void* x, int64_t ldx, const void* const* codes, const void* const* scales,
                                      const void* mask, int32_t* perm, int32_t* counts, void* workspace,
                                      int64_t workspace_bytes, void* f1, void* f3, void* y, int64_t ldy, int64_t M, int64_t d,
                                      int64_t h, int32_t* status, void* stream) {
  if (M == 0) return 0;
  if (!x || !codes || !scales || !mask || !perm || !counts || !workspace || !y || !status || !f1 != !f3) return FFNK_ERR_NULL;
  for (int i = 0; i < 6; ++i)
    if (!codes[i] || !scales[i]) return FFNK_ERR_NULL;
  if (M < 0 || M >= (1ll << 30) || mx_bad_dim(d) || mx_bad_dim(h)) return FFNK_ERR_SHAPE;
  if ((ldx & 7) || (ldy & 7) || ldx < d || ldy < d || misaligned(x) || misaligned(y) || misaligned(perm) || misaligned(f1) ||
      misaligned(f3) || (reinterpret_cast<uintptr_t>(workspace) & 255))
    return FFNK_ERR_ALIGN;
  for (int i = 0; i < 6; ++i)
    if (misaligned(codes[i]) || misaligned(scales[i])) return FFNK_ERR_ALIGN;
  const MxWorkspace w = mx_workspace(M, d, h);
  if (workspace_bytes < w.total) return FFNK_ERR_CAPACITY;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const MxSelf self{x, ldx, perm, counts};
  const int splits = mx_small_splits(M, h, d, true);
  const bool takes = mx_takes_self(M, d, splits);
  int r = takes ? 0 : mx_route_quantize(mask, M, x, ldx, d, perm, counts, ws + w.scan, ws + w.xc, ws + w.xs, status, stream);
  if (r) return r;
  const MxWeight gu[4] = {{codes[0], scales[0]}, {codes[2], scales[2]}, {codes[3], scales[3]}, {codes[5], scales[5]}};
  if ((r = mx_gateup(takes ? MxWeight{} : MxWeight{ws + w.xc, ws + w.xs}, gu, perm, counts, ws + w.hc, ws + w.hs, mask, f1, f3, M, d,
                     h, splits, takes ? &self : nullptr, status, s)))
    return r;
  return mx_product(MxWeight{ws + w.hc, ws + w.hs}, MxWeight{codes[1], scales[1]}, MxWeight{codes[4], scales[4]}, perm, counts, mask,
                    y, ldy, M, d, h, mx_small_splits(M, d, h, false), nullptr, status, s);
}

// ---------------------------------------------------------------------------------------------
// Backward passes: gradients of the activations, the weights being frozen.  The contraction runs over the other
// dimension of the weights than their blocks do, so the weights are read back to bf16 (exactly) and the bf16
// GEMMs of the framework do the rest; the rounding of activations to 4 bits counts as the identity.
// ---------------------------------------------------------------------------------------------
namespace ffnk {
struct MxBackwardSpace {
  int64_t gr, dt1, dt3, w[6], total;
};
static MxBackwardSpace mx_backward_space(int64_t M, int64_t K, int64_t N, int64_t h) {
  MxBackwardSpace w{};
  const int64_t rows = ffnk_route_capacity(M) + 512;
  int64_t off = 0;
  w.gr = off;
  off += mx_align(rows * N * 2);
  if (h) {
    w.dt1 = off; off += mx_align(rows * h * 2);
    w.dt3 = off; off += mx_align(rows * h * 2);
  }
  for (int i = 0; i < (h ? 6 : 2); ++i) {
    w.w[i] = off;
    off += mx_align((h ? h : N) * K * 2);
  }
  w.total = off;
  return w;
}
}  // namespace ffnk

extern "C" int64_t ffnk_mxfp4_backward_workspace_bytes(int64_t M, int64_t K, int64_t N, int64_t h) {
  if (M <= 0 || K <= 0 || N <= 0 || h < 0) return 256;
  return mx_backward_space(M, K, N, h).total;
}

extern "C" int ffnk_mxfp4_linear_backward(const void* g, int64_t ldg, const void* b1_codes, const void* b1_scales,
                                          const void* b2_codes, const void* b2_scales, const int32_t* perm,
                                          const int32_t* counts, void* workspace, int64_t workspace_bytes, void* dx,
                                          int64_t lddx, int64_t M, int64_t N, int64_t K, int32_t* status, void* stream) {
  if (M == 0) return 0;
  if (!g || !b1_codes || !b1_scales || !b2_codes || !b2_scales || !perm || !counts || !workspace || !dx || !status)
    return FFNK_ERR_NULL;
  if (M < 0 || M >= (1ll << 30) || mx_bad_dim(N) || mx_bad_dim(K)) return FFNK_ERR_SHAPE;
  if ((ldg & 7) || (lddx & 7) || ldg < N || lddx < K || misaligned(g) || misaligned(dx) || misaligned(b1_codes) ||
      misaligned(b1_scales) || misaligned(b2_codes) || misaligned(b2_scales) || (reinterpret_cast<uintptr_t>(workspace) & 255))
    return FFNK_ERR_ALIGN;
  const MxBackwardSpace w = mx_backward_space(M, K, N, 0);
  if (workspace_bytes < w.total) return FFNK_ERR_CAPACITY;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const void* codes[2] = {b1_codes, b2_codes};
  const void* scales[2] = {b1_scales, b2_scales};
  const int64_t rows[2] = {N, N}, cols[2] = {K, K};
  const int gate[2] = {0, 1};
  void* wd[2] = {ws + w.w[0], ws + w.w[1]};
  int r = mx_dequantize_weights(codes, scales, rows, cols, gate, 2, counts, wd, stream);
  if (r) return r;
  if ((r = ffnk_permute_rows(g, ldg, perm, counts, ws + w.gr, N, M, N, stream))) return r;
  return ffnk_ffn_down(ws + w.gr, N, wd[0], wd[1], K, 1, perm, counts, dx, lddx, M, K, N, status, stream);
}

extern "C" int ffnk_mxfp4_ffn_backward(const void* gy, int64_t ldg, const void* const* codes, const void* const* scales,
                                       const void* f1, const void* f3, const int32_t* perm, const int32_t* counts,
                                       void* workspace, int64_t workspace_bytes, void* dx, int64_t lddx, int64_t M, int64_t d,
                                       int64_t h, int32_t* status, void* stream) {
  if (M == 0) return 0;
  if (!gy || !codes || !scales || !f1 || !f3 || !perm || !counts || !workspace || !dx || !status) return FFNK_ERR_NULL;
  for (int i = 0; i < 6; ++i)
    if (!codes[i] || !scales[i]) return FFNK_ERR_NULL;
  if (M < 0 || M >= (1ll << 30) || mx_bad_dim(d) || mx_bad_dim(h)) return FFNK_ERR_SHAPE;
  if ((ldg & 7) || (lddx & 7) || ldg < d || lddx < d || misaligned(gy) || misaligned(dx) || misaligned(f1) || misaligned(f3) ||
      (reinterpret_cast<uintptr_t>(workspace) & 255))
    return FFNK_ERR_ALIGN;
  for (int i = 0; i < 6; ++i)
    if (misaligned(codes[i]) || misaligned(scales[i])) return FFNK_ERR_ALIGN;
  const MxBackwardSpace w = mx_backward_space(M, d, d, h);
  if (workspace_bytes < w.total) return FFNK_ERR_CAPACITY;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  int64_t rows[6], cols[6];
  const int gate[6] = {0, 0, 0, 1, 1, 1};
  void* wd[6];
  for (int i = 0; i < 6; ++i) {
    rows[i] = i % 3 == 1 ? d : h;
    cols[i] = i % 3 == 1 ? h : d;
    wd[i] = ws + w.w[i];
  }
  const int r = mx_dequantize_weights(codes, scales, rows, cols, gate, 6, counts, wd, stream);
  if (r) return r;
  return ffn_backward_dx(gy, ldg, f1, f3, wd[0], wd[1], wd[2], wd[3], wd[4], wd[5], perm, counts, ws + w.gr, ws + w.dt1,
                         ws + w.dt3, dx, lddx, M, d, h, status, stream);
}
