// f8_gemm.hip -- C = alpha * A * B^T + beta * C for matrices in 8 bits with a power-of-two scale for each block of 128
// along the contracted dimension (bof_f8.h).
//
//   C[i][j] = alpha * sum_b 2^(sa[i][b] + sb[j][b]) * sum_{k in block b} a[i][k] b[j][k] + beta * C[i][j]
//
// One v_mfma_scale_f32_16x16x128_f8f6f4 contracts exactly one block and applies both scales, so the sums stay in the
// matrix unit's accumulators (fp32) over the whole of k and a block costs no vector instruction.  The B rows are the
// instruction's first operand, the A rows its second: a lane then holds FOUR NEIGHBOURS of a row of C (rows of C are A
// rows), j = 4 * (lane / 16) + 0..3, i = lane % 16.  Lane l feeds 32 bytes of row l % 16, the same bytes of the block
// on both sides; which 32 is free (the sum does not depend on the order of k).
//
// That instruction adds eight neighbouring products at a time, aligned to the largest and cut at 2^-13 of it (measured:
// a product of 2^16 next to one of 2^2 leaves nothing of the smaller; across groups of eight nothing is cut).  Under
// a 16-bit C (a half step of 2^-9 or 2^-11 of the value) that does not show; a 32-bit C, what gradients of weights are
// added into, is computed WIDE: both operands are widened to bf16, exactly and with their scales applied
// (v_cvt_scalef32_pk_bf16_*), and multiplied by v_mfma_f32_16x16x32_bf16, whose sums are exact to fp32 (measured
// 2.4e-9 relative on 32 products) at half the rate.
#include "f8_common.h"

namespace bof {

namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

struct F8Product {
  const uint8_t *a, *b, *sa, *sb;
  int64_t lda, ldb, ldsa, ldsb, ldc;
  int a_shift, b_shift;   // log2 of the rows that share a scale
  int m, n, k;
  float alpha, beta;
  void *c;
  int c_type;
  float *part;            // split along k: part z of the sums goes to part + z * m * n
  int blocks_per_part;    // blocks of 128 along k in one part
};

// ---- fragments ----------------------------------------------------------------------
// The 32 bytes a lane feeds into one block, as they are (the scale goes along as a byte) or widened to four operands of
// the bf16 instruction.
template <bool WIDE>
struct Frag;
template <>
struct Frag<false> {
  i32x8 q;
  int s;
};
template <>
struct Frag<true> {
  bf16x8 q[4];
};

// 2^(code - 127) as a float: code 0 is below the normal floats, 255 is NaN
__device__ __forceinline__ float scale_value(uint32_t code) {
  return __uint_as_float(code == 0u ? 0x00400000u : code == 255u ? 0x7fc00000u : code << 23);
}

template <int T>
__device__ __forceinline__ bf16x8 widen8(int lo, int hi, float s) {
  bf16x2 p[4];
  if constexpr (T == BOF_E4M3) {
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, false);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, true);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, false);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, true);
  } else {
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(lo, s, false);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(lo, s, true);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(hi, s, false);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(hi, s, true);
  }
  return __builtin_shufflevector(__builtin_shufflevector(p[0], p[1], 0, 1, 2, 3), __builtin_shufflevector(p[2], p[3], 0, 1, 2, 3),
                                 0, 1, 2, 3, 4, 5, 6, 7);
}

template <int T, bool WIDE>
__device__ __forceinline__ Frag<WIDE> make_frag(u32x4 lo, u32x4 hi, uint32_t code) {
  Frag<WIDE> f;
  if constexpr (WIDE) {
    const float s = scale_value(code);
    f.q[0] = widen8<T>((int) lo[0], (int) lo[1], s);
    f.q[1] = widen8<T>((int) lo[2], (int) lo[3], s);
    f.q[2] = widen8<T>((int) hi[0], (int) hi[1], s);
    f.q[3] = widen8<T>((int) hi[2], (int) hi[3], s);
  } else {
    f.q = i32x8{(int) lo[0], (int) lo[1], (int) lo[2], (int) lo[3], (int) hi[0], (int) hi[1], (int) hi[2], (int) hi[3]};
    f.s = (int) code;
  }
  return f;
}

// acc += (B rows) x (A rows) over one block
template <int TA, int TB, bool WIDE>
__device__ __forceinline__ f32x4 mma(const Frag<WIDE> &b, const Frag<WIDE> &a, f32x4 acc) {
  if constexpr (WIDE) {
#pragma unroll
    for (int j = 0; j < 4; j++) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b.q[j], a.q[j], acc, 0, 0, 0);
    return acc;
  } else {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b.q, a.q, acc, TB == BOF_E4M3 ? 0 : 1, TA == BOF_E4M3 ? 0 : 1,
                                                            0, b.s, 0, a.s);
  }
}

// ---- output -------------------------------------------------------------------------
__device__ __forceinline__ float dense_at(const void *p, int64_t i, int type) {
  return type == BOF_F32 ? load_dense<BOF_F32>(p, i) : type == BOF_BF16 ? load_dense<BOF_BF16>(p, i) : load_dense<BOF_F16>(p, i);
}
__device__ __forceinline__ void dense_put(void *p, int64_t i, int type, float v) {
  if (type == BOF_F32) store_dense<BOF_F32>(p, i, v);
  else if (type == BOF_BF16) store_dense<BOF_BF16>(p, i, v);
  else store_dense<BOF_F16>(p, i, v);
}
// alpha * sum + beta * C, rounded once to the type of C; beta == 0 does not read C
__device__ __forceinline__ void finish(const F8Product &p, int64_t i, int64_t j, float sum) {
  const int64_t at = i * p.ldc + j;
  float v = p.alpha * sum;
  if (p.beta != 0.f) v = fmaf(p.beta, dense_at(p.c, at, p.c_type), v);
  dense_put(p.c, at, p.c_type, v);
}

// ---- tiles of any shape and alignment -----------------------------------------------
// 16 bytes of a row from byte k0 on, zeros from byte k on.  Only a row's last chunk is short: it is read as the row's
// last 16 bytes and shifted (or byte by byte, in rows shorter than that).
__device__ __forceinline__ u32x4 load_chunk(const uint8_t *row, int k0, int k) {
  u32x4 v = {0u, 0u, 0u, 0u};
  if (k0 + 16 <= k) {
    __builtin_memcpy(&v, row + k0, 16);
  } else if (k0 < k) {
    if (k >= 16) {
      unsigned __int128 w;
      __builtin_memcpy(&w, row + k - 16, 16);
      w >>= 8 * (k0 + 16 - k);
      __builtin_memcpy(&v, &w, 16);
    } else {
      uint8_t tmp[16];
#pragma unroll
      for (int i = 0; i < 16; i++) tmp[i] = k0 + i < k ? row[k0 + i] : 0;
      __builtin_memcpy(&v, tmp, 16);
    }
  }
  return v;
}

// One workgroup of four waves, 128 x 128 of C, one block of k at a time through LDS (rows of 128 bytes, their 16-byte
// chunks XOR-ed with the row so that the fragment reads meet no bank twice).  Rows outside the matrices read the last
// row and are not stored.
template <int TA, int TB, bool WIDE>
__global__ void __launch_bounds__(256) f8_tile_any_kernel(F8Product p) {
  __shared__ u32x4 lds[2][128 * 8];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int tiles_n = (p.n + 127) >> 7;
  const int i0 = (int) (blockIdx.x / tiles_n) * 128, j0 = (int) (blockIdx.x % tiles_n) * 128;
  const int wi = (wave >> 1) * 64, wj = (wave & 1) * 64;
  const int l16 = lane & 15, g = lane >> 4;
  const int nb = (p.k + 127) >> 7;
  const int b0 = blockIdx.y * p.blocks_per_part, b1 = min(nb, b0 + p.blocks_per_part);
  f32x4 acc[4][4];
#pragma unroll
  for (int x = 0; x < 16; x++) acc[x >> 2][x & 3] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int blk = b0; blk < b1; blk++) {
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const int at = t + 256 * u, r = at >> 3, c = at & 7;
      lds[0][r * 8 + (c ^ (r & 7))] = load_chunk(p.a + (int64_t) min(i0 + r, p.m - 1) * p.lda, blk * 128 + c * 16, p.k);
      lds[1][r * 8 + (c ^ (r & 7))] = load_chunk(p.b + (int64_t) min(j0 + r, p.n - 1) * p.ldb, blk * 128 + c * 16, p.k);
    }
    __syncthreads();
    Frag<WIDE> fa[4];
#pragma unroll
    for (int x = 0; x < 4; x++) {
      const int r = wi + x * 16 + l16, i = min(i0 + r, p.m - 1);
      fa[x] = make_frag<TA, WIDE>(lds[0][r * 8 + (g ^ (r & 7))], lds[0][r * 8 + ((g + 4) ^ (r & 7))],
                                  p.sa[(int64_t) (i >> p.a_shift) * p.ldsa + blk]);
    }
#pragma unroll
    for (int y = 0; y < 4; y++) {
      const int r = wj + y * 16 + l16, j = min(j0 + r, p.n - 1);
      const Frag<WIDE> fb = make_frag<TB, WIDE>(lds[1][r * 8 + (g ^ (r & 7))], lds[1][r * 8 + ((g + 4) ^ (r & 7))],
                                                p.sb[(int64_t) (j >> p.b_shift) * p.ldsb + blk]);
#pragma unroll
      for (int x = 0; x < 4; x++) acc[x][y] = mma<TA, TB, WIDE>(fb, fa[x], acc[x][y]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int x = 0; x < 4; x++)
#pragma unroll
    for (int y = 0; y < 4; y++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int i = i0 + wi + x * 16 + l16, j = j0 + wj + y * 16 + g * 4 + e;
        if (i < p.m && j < p.n) {
          if (p.part) p.part[((int64_t) blockIdx.y * p.m + i) * p.n + j] = acc[x][y][e];
          else finish(p, i, j, acc[x][y][e]);
        }
      }
}

// ---- 256 x 256 tiles ----------------------------------------------------------------
// Four waves, one on each SIMD, 128 x 128 of C each: 64 accumulators of four floats = 256 registers (the accumulator
// half of the file), the other half holds the fragments.  A slab is one block of k, 256 rows x 128 bytes of each operand;
// both lie in LDS twice (128 KB).  Rows reach LDS without touching registers: one global_load_lds_dwordx4 moves 8 rows,
// lane l fetching chunk (l & 7) ^ (l >> 3) of row l >> 3, so that the image is [row][chunk ^ (row & 7)] and a fragment
// read (16 rows x 16 bytes) meets every bank once.  Per slab and wave: 64 MFMAs of 32 cycles, 32 ds_read_b128, 16 DMA
// pieces.
//
// The A fragments of a slab are read into registers during the slab BEFORE (8 x 8 registers, twice), the B fragments one
// tile ahead.  The barrier of a slab stands in front of its last B tile: by then every wave has read all it wants from
// this slab's B image and the next slab's A image, and the pieces of the next B and the next but one A image, issued at the
// slab's start, have landed.
//
// Scales: thread t fetches the word with four blocks' scales of A row t and of B row t, once in four slabs, into LDS
// (twice 2 KB); a fragment's scale byte is read from there along with it.  No vector instruction is left in a slab but a few
// for the whole of it.
//
// A tile at the lower or right edge starts earlier (at m - 256, n - 256), so that every row it fetches exists; what lies
// in the tile before is not stored again.
__device__ __forceinline__ uint32_t lds_address(const void *p) {
  return (uint32_t) (uintptr_t) (const __attribute__((address_space(3))) void *) p;
}
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// 64 lanes x 16 bytes from base + voff to LDS, contiguous from `to` on (M0 carries the destination)
__device__ __forceinline__ void dma16(uint32_t voff, uint64_t base, uint32_t to) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" :: "v"(voff), "s"(base), "s"(to) : "memory", "m0");
}
#pragma clang diagnostic pop

// workgroups go round the 8 XCDs; tiles of one XCD are neighbours (each XCD has its own L2), GROUP rows of tiles deep
__device__ __forceinline__ void tile_of(int bid, int tiles_m, int tiles_n, int group, int &tm, int &tn) {
  const int nwg = tiles_m * tiles_n, q = nwg >> 3, r = nwg & 7, xcd = bid & 7, idx = bid >> 3;
  bid = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + idx;
  const int per = group * tiles_n, first = bid / per * group, deep = min(tiles_m - first, group);
  tm = first + bid % per % deep;
  tn = bid % per / deep;
}

// The four scale bytes of blocks b .. b + 3 of a row (nb >= 4 blocks in all, b < nb) as one word, read inside the row:
// the word that is read begins up to three bytes early, scale_shift bits of it are left out.
__device__ __forceinline__ uint32_t scale_word(const uint8_t *row, int b, int nb) {
  uint32_t w;
  __builtin_memcpy(&w, row + min(b, nb - 4), 4);
  return w;
}
__device__ __forceinline__ int scale_shift(int b, int nb) { return 8 * max(0, b - (nb - 4)); }

__device__ __forceinline__ i32x8 both(u32x4 lo, u32x4 hi) {
  return i32x8{(int) lo[0], (int) lo[1], (int) lo[2], (int) lo[3], (int) hi[0], (int) hi[1], (int) hi[2], (int) hi[3]};
}

// A wave's 128 x 128 sums to C, from row i, column j on: 64 rows at a time through the wave's own 32 KB of LDS (rows of
// 32 chunks of four floats, XOR-ed with the row), so that a row of C leaves in whole lines.  Rows before i_from and
// columns before j_from are left out.
__device__ __forceinline__ void store_wave_128(const F8Product &p, f32x4 (&acc)[8][8], f32x4 *own, int i, int j, int i_from, int j_from) {
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const bool wide = p.c_type != BOF_F32 && p.beta == 0.f && p.ldc % 8 == 0 && j_from == j && j + 128 <= p.n && j % 8 == 0 && reinterpret_cast<uintptr_t>(p.c) % 16 == 0;
#pragma unroll
  for (int half = 0; half < 2; half++) {
#pragma unroll
    for (int x = 0; x < 4; x++)
#pragma unroll
      for (int y = 0; y < 8; y++) own[(x * 16 + l16) * 32 + ((y * 4 + g) ^ (l16 & 7))] = acc[half * 4 + x][y];
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (wide) {
#pragma unroll 4
      for (int it = 0; it < 16; it++) {
        const int r = it * 4 + g, row = i + half * 64 + r;
        const f32x4 v0 = own[r * 32 + ((l16 * 2) ^ (r & 7))], v1 = own[r * 32 + ((l16 * 2 + 1) ^ (r & 7))];
        if (row < i_from || row >= p.m) continue;
        if (p.c_type == BOF_BF16) {
          typedef __bf16 b8 __attribute__((ext_vector_type(8)));
          b8 o;
#pragma unroll
          for (int e = 0; e < 4; e++) { o[e] = (__bf16) (p.alpha * v0[e]); o[e + 4] = (__bf16) (p.alpha * v1[e]); }
          *(b8 *) ((__bf16 *) p.c + (int64_t) row * p.ldc + j + l16 * 8) = o;
        } else {
          typedef _Float16 h8 __attribute__((ext_vector_type(8)));
          h8 o;
#pragma unroll
          for (int e = 0; e < 4; e++) { o[e] = (_Float16) (p.alpha * v0[e]); o[e + 4] = (_Float16) (p.alpha * v1[e]); }
          *(h8 *) ((_Float16 *) p.c + (int64_t) row * p.ldc + j + l16 * 8) = o;
        }
      }
    } else {
#pragma unroll 1
      for (int it = 0; it < 128; it++) {
        const int r = it >> 1, c = (it & 1) * 64 + lane, row = i + half * 64 + r;
        const float v = ((const float *) own)[(r * 32 + ((c >> 2) ^ (r & 7))) * 4 + (c & 3)];
        if (row >= i_from && row < p.m && j + c >= j_from && j + c < p.n) finish(p, row, j + c, v);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

// The slab's product, its accumulators pinned to the accumulator registers (left to itself the compiler moves them through
// both halves of the file: 200 copies a slab).  Hazards: the same accumulator comes round after 64 of these, the fragments
// come from LDS; whoever reads acc afterwards calls settle() first.
template <int TA, int TB>
__device__ __forceinline__ void mma_pinned(const Frag<false> &b, const Frag<false> &a, f32x4 &acc) {
  asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0] cbsz:%5 blgp:%6"
               : "+a"(acc) : "v"(b.q), "v"(a.q), "v"(b.s), "v"(a.s), "n"(TB == BOF_E4M3 ? 0 : 1), "n"(TA == BOF_E4M3 ? 0 : 1));
}
__device__ __forceinline__ void settle() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); }

// LDS, in chunks of 16 bytes: A twice, B twice, scale words twice (A rows, B rows)
constexpr int kImage = 2048, kScales = 4 * kImage, kLds256 = kScales + 2 * 128;

struct Slab256 {
  u32x4 *lds;
  uint32_t a_voff, b_voff;       // of this lane's row in a piece
  uint64_t a_step, b_step;       // bytes from piece to piece (32 rows)
  uint32_t a_to, b_to;           // LDS addresses of this wave's pieces in image 0
  int a_lo, a_hi, b_lo, b_hi;    // this lane's chunks in the image, of tile 0
  const uint8_t *sa, *sb;        // this lane's scale bytes of tile 0, block 0 of four
};

template <int TA, int TB, int P>
__device__ __forceinline__ void slab256(const Slab256 &s, uint64_t b_next, uint64_t a_next, int sc_b, int sc_a, Frag<false> (&fa)[2][8],
                                        Frag<false> (&fb)[2], f32x4 (&acc)[8][8]) {
#pragma unroll
  for (int y = 0; y < 8; y++) {
    if (y == 7) {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    }
#pragma unroll
    for (int x = 0; x < 8; x++) {
      mma_pinned<TA, TB>(fb[y & 1], fa[P][x], acc[x][y]);
      if (x == 1) {   // the next B tile: of this slab, or the next one's first
        const int at = (y < 7 ? P : P ^ 1) * kImage + (y < 7 ? y + 1 : 0) * 128;
        fb[(y + 1) & 1].q = both(s.lds[s.b_lo + at], s.lds[s.b_hi + at]);
        fb[(y + 1) & 1].s = s.sb[(y < 7 ? sc_b : sc_a) + (y < 7 ? y + 1 : 0) * 64];
      }
      if (y < 4 && (x & 1)) {   // pieces: B first
        const int piece = y * 4 + (x >> 1);
        if (piece < 8) dma16(s.b_voff, b_next + piece * s.b_step, s.b_to + (P ^ 1) * kImage * 16 + piece * 4096);
        else dma16(s.a_voff, a_next + (piece - 8) * s.a_step, s.a_to + P * kImage * 16 + (piece - 8) * 4096);
      }
      if (y >= 2 && y < 6 && (x == 3 || x == 6)) {   // the next slab's A fragments
        const int f = (y - 2) * 2 + (x == 6), at = (P ^ 1) * kImage + f * 128;
        fa[P ^ 1][f].q = both(s.lds[s.a_lo + at], s.lds[s.a_hi + at]);
        fa[P ^ 1][f].s = s.sa[sc_a + f * 64];
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

template <int TA, int TB>
__global__ void __launch_bounds__(256, 1) f8_tile256_kernel(F8Product p, int tiles_m, int tiles_n) {
  __shared__ u32x4 lds[kLds256];
  int tm, tn;
  tile_of(blockIdx.x, tiles_m, tiles_n, 4, tm, tn);
  const int i0 = min(tm * 256, p.m - 256), j0 = min(tn * 256, p.n - 256);
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wi = (wave >> 1) * 128, wj = (wave & 1) * 128;
  const int l16 = lane & 15, g = lane >> 4;
  const int nb = (p.k + 127) >> 7, full = p.k >> 7;
  Slab256 s;
  s.lds = lds;
  const int r8 = lane >> 3, chunk = ((lane & 7) ^ r8) << 4;
  s.a_voff = (uint32_t) (8 * wave + r8) * (uint32_t) p.lda + chunk;
  s.b_voff = (uint32_t) (8 * wave + r8) * (uint32_t) p.ldb + chunk;
  s.a_step = (uint64_t) p.lda * 32;
  s.b_step = (uint64_t) p.ldb * 32;
  s.a_to = lds_address(lds) + wave * 1024;
  s.b_to = s.a_to + 2 * kImage * 16;
  s.a_lo = (wi + l16) * 8 + (g ^ (l16 & 7)); s.a_hi = (wi + l16) * 8 + ((g + 4) ^ (l16 & 7));
  s.b_lo = 2 * kImage + (wj + l16) * 8 + (g ^ (l16 & 7)); s.b_hi = 2 * kImage + (wj + l16) * 8 + ((g + 4) ^ (l16 & 7));
  s.sa = (const uint8_t *) (lds + kScales) + (wi + l16) * 4;
  s.sb = (const uint8_t *) (lds + kScales + 64) + (wj + l16) * 4;
  uint32_t *const sw = (uint32_t *) (lds + kScales) + t;
  const uint8_t *const sa_row = p.sa + (int64_t) ((i0 + t) >> p.a_shift) * p.ldsa, *const sb_row = p.sb + (int64_t) ((j0 + t) >> p.b_shift) * p.ldsb;
  const uint64_t a_org = reinterpret_cast<uint64_t>(p.a + (int64_t) i0 * p.lda), b_org = reinterpret_cast<uint64_t>(p.b + (int64_t) j0 * p.ldb);
  // A of slabs 0 and 1, B of slab 0, the scales of the first four
#pragma unroll
  for (int q = 0; q < 8; q++) {
    dma16(s.a_voff, a_org + q * s.a_step, s.a_to + q * 4096);
    dma16(s.b_voff, b_org + q * s.b_step, s.b_to + q * 4096);
    dma16(s.a_voff, a_org + 128 + q * s.a_step, s.a_to + kImage * 16 + q * 4096);
  }
  f32x4 acc[8][8];
#pragma unroll
  for (int x = 0; x < 64; x++) acc[x >> 3][x & 7] = f32x4{0.f, 0.f, 0.f, 0.f};
  uint32_t wa = scale_word(sa_row, 0, nb), wb = scale_word(sb_row, 0, nb);
  sw[0] = wa;
  sw[256] = wb;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  Frag<false> fa[2][8], fb[2];
#pragma unroll
  for (int x = 0; x < 8; x++) {
    fa[0][x].q = both(lds[s.a_lo + x * 128], lds[s.a_hi + x * 128]);
    fa[0][x].s = s.sa[x * 64];
  }
  fb[0].q = both(lds[s.b_lo], lds[s.b_hi]);
  fb[0].s = s.sb[0];
  __syncthreads();
  // (the pieces behind the last slab fetch the last slab again, into images nobody reads)
  auto words = [&](int kb) {   // in front of slab kb: the next four blocks' scales, fetched at 0, in LDS before 2's barrier
    if ((kb & 3) == 0 && kb + 4 < nb) { wa = scale_word(sa_row, kb + 4, nb); wb = scale_word(sb_row, kb + 4, nb); }
    if ((kb & 3) == 2 && kb + 2 < nb) { uint32_t *to = sw + (~kb & 4) * 128; to[0] = wa >> scale_shift(kb + 2, nb); to[256] = wb >> scale_shift(kb + 2, nb); }
  };
  auto byte_of = [](int kb) { return (kb & 4) * 512 + (kb & 3); };
  int kb = 0;
  for (; kb + 2 <= full; kb += 2) {
    words(kb);
    slab256<TA, TB, 0>(s, b_org + (uint64_t) min(kb + 1, full - 1) * 128, a_org + (uint64_t) min(kb + 2, full - 1) * 128, byte_of(kb), byte_of(kb + 1), fa, fb, acc);
    slab256<TA, TB, 1>(s, b_org + (uint64_t) min(kb + 2, full - 1) * 128, a_org + (uint64_t) min(kb + 3, full - 1) * 128, byte_of(kb + 1), byte_of(kb + 2), fa, fb, acc);
  }
  if (kb < full) {
    words(kb);
    slab256<TA, TB, 0>(s, b_org + (uint64_t) (full - 1) * 128, a_org + (uint64_t) (full - 1) * 128, byte_of(kb), byte_of(kb + 1), fa, fb, acc);
    kb++;
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __syncthreads();
  if (nb > full) {   // the short block: through registers, zeros behind k
#pragma unroll 1
    for (int u = 0; u < 8; u++) {
      const int at = t + 256 * u, r = at >> 3, c = at & 7;
      lds[r * 8 + (c ^ (r & 7))] = load_chunk(p.a + (int64_t) (i0 + r) * p.lda, full * 128 + c * 16, p.k);
      lds[2 * kImage + r * 8 + (c ^ (r & 7))] = load_chunk(p.b + (int64_t) (j0 + r) * p.ldb, full * 128 + c * 16, p.k);
    }
    sw[0] = sa_row[full];
    sw[256] = sb_row[full];
    __syncthreads();
#pragma unroll
    for (int x = 0; x < 8; x++) {
      fa[0][x].q = both(lds[s.a_lo + x * 128], lds[s.a_hi + x * 128]);
      fa[0][x].s = s.sa[x * 64];
    }
#pragma unroll
    for (int y = 0; y < 8; y++) {
      Frag<false> b;
      b.q = both(lds[s.b_lo + y * 128], lds[s.b_hi + y * 128]);
      b.s = s.sb[y * 64];
#pragma unroll
      for (int x = 0; x < 8; x++) mma_pinned<TA, TB>(b, fa[0][x], acc[x][y]);
    }
    __syncthreads();
  }
  settle();
  store_wave_128(p, acc, (f32x4 *) lds + wave * kImage, i0 + wi, j0 + wj, max(tm * 256, i0 + wi), max(tn * 256, j0 + wj));
}

// C from the parts of the sums, added in their order (no parts: C = beta * C)
__global__ void __launch_bounds__(256) f8_join_kernel(F8Product p, int parts) {
  const int64_t mn = (int64_t) p.m * p.n;
  for (int64_t at = (int64_t) blockIdx.x * 256 + threadIdx.x; at < mn; at += (int64_t) gridDim.x * 256) {
    float sum = 0.f;
    for (int z = 0; z < parts; z++) sum += p.part[z * mn + at];
    finish(p, at / p.n, at % p.n, sum);
  }
}

constexpr int kMaxParts = 32;

// parts along k: enough workgroups to fill the card's 256 compute units twice, each with four blocks at least
int wanted_parts(int64_t m, int64_t n, int64_t k) {
  const int64_t tiles = ((m + 127) / 128) * ((n + 127) / 128), nb = (k + 127) / 128;
  int64_t parts = tiles > 0 ? 512 / tiles : 1;
  if (parts > nb / 4) parts = nb / 4;
  return (int) (parts < 1 ? 1 : parts > kMaxParts ? kMaxParts : parts);
}

template <int TA, int TB>
hipError_t launch_product(F8Product p, int parts, hipStream_t st) {
  const int nb = (p.k + 127) / 128;
  p.blocks_per_part = (nb + parts - 1) / parts;
  parts = (nb + p.blocks_per_part - 1) / p.blocks_per_part;
  if (parts == 1) p.part = nullptr;
  const int tiles_m = (p.m + 255) / 256, tiles_n = (p.n + 255) / 256;
  if (p.c_type != BOF_F32 && p.m >= 256 && p.n >= 256 && (int64_t) tiles_m * tiles_n >= 64 && p.k >= 512 && p.lda % 16 == 0 && p.ldb % 16 == 0 &&
      p.lda <= (1 << 23) && p.ldb <= (1 << 23) && reinterpret_cast<uintptr_t>(p.a) % 16 == 0 && reinterpret_cast<uintptr_t>(p.b) % 16 == 0) {
    drop_stale_error();
    f8_tile256_kernel<TA, TB><<<(unsigned) (tiles_m * tiles_n), 256, 0, st>>>(p, tiles_m, tiles_n);
    return hipGetLastError();
  }
  const dim3 grid((unsigned) (((p.n + 127) / 128) * (int64_t) ((p.m + 127) / 128)), (unsigned) parts);
  drop_stale_error();
  if (p.c_type == BOF_F32) f8_tile_any_kernel<TA, TB, true><<<grid, 256, 0, st>>>(p);
  else f8_tile_any_kernel<TA, TB, false><<<grid, 256, 0, st>>>(p);
  if (parts > 1) {
    const int64_t wg = ((int64_t) p.m * p.n + 255) / 256;
    f8_join_kernel<<<(unsigned) (wg < 2048 ? wg : 2048), 256, 0, st>>>(p, parts);
  }
  return hipGetLastError();
}

}  // namespace

}  // namespace bof

using namespace bof;

extern "C" {

uint64_t bof_f8_gemm_workspace_bytes(int64_t m, int64_t n, int64_t k) {
  if (m <= 0 || n <= 0 || k <= 0 || m > INT32_MAX || n > INT32_MAX || k > INT32_MAX) return 0;
  const int parts = wanted_parts(m, n, k);
  return parts > 1 ? (uint64_t) parts * (uint64_t) m * (uint64_t) n * 4u : 0;
}

int bof_f8_gemm(int64_t m, int64_t n, int64_t k, float alpha, const void *a, int64_t lda, int a_type, const uint8_t *sa,
                int64_t ldsa, int ga, const void *b, int64_t ldb, int b_type, const uint8_t *sb, int64_t ldsb, int gb,
                float beta, void *c, int64_t ldc, int c_type, void *work, uint64_t work_bytes, void *stream) {
  static const char kCall[] = "bof_f8_gemm";
  if (m < 0 || n < 0 || k < 0 || m > INT32_MAX - 255 || n > INT32_MAX - 255 || k > INT32_MAX - 255) return refuse(kCall, "bad size");
  if ((a_type != BOF_E4M3 && a_type != BOF_E5M2) || (b_type != BOF_E4M3 && b_type != BOF_E5M2)) return refuse(kCall, "A and B are of BOF_E4M3 or BOF_E5M2");
  if (c_type < BOF_F32 || c_type > BOF_F16) return refuse(kCall, "C is of BOF_F32, BOF_BF16 or BOF_F16");
  if ((ga != 1 && ga != 128) || (gb != 1 && gb != 128)) return refuse(kCall, "1 or 128 rows share a scale");
  if (m == 0 || n == 0) return BOF_OK;
  const bool product = k > 0 && alpha != 0.f;
  const int64_t nb = (k + 127) / 128;
  if (!c || ldc < n) return refuse(kCall, "C is missing or its rows overlap");
  if (reinterpret_cast<uintptr_t>(c) % dense_bytes(c_type)) return refuse(kCall, "C is not aligned to its type");
  if (product && (!a || !b || !sa || !sb)) return refuse(kCall, "an operand is missing");
  if (product && (lda < k || ldb < k || ldsa < nb || ldsb < nb)) return refuse(kCall, "rows of an operand overlap");
  if (work && reinterpret_cast<uintptr_t>(work) % 16) return refuse(kCall, "work is not aligned to 16 bytes");
  LaunchDevice dev((hipStream_t) stream);
  if (dev.status()) return dev.status();
  if (int rc = dev.reaches(c, kCall, "C")) return rc;
  F8Product p{};
  p.ldc = ldc; p.m = (int) m; p.n = (int) n; p.k = product ? (int) k : 0;
  p.alpha = alpha; p.beta = beta; p.c = c; p.c_type = c_type;
  if (!product) {
    if (beta == 1.f) return BOF_OK;
    const int64_t wg = (m * n + 255) / 256;
    drop_stale_error();
    f8_join_kernel<<<(unsigned) (wg < 2048 ? wg : 2048), 256, 0, (hipStream_t) stream>>>(p, 0);
    BOF_HIP_TRY(hipGetLastError());
    return BOF_OK;
  }
  for (auto [q, name] : {std::pair<const void *, const char *>{a, "A"}, {b, "B"}, {sa, "sa"}, {sb, "sb"}})
    if (int rc = dev.reaches(q, kCall, name)) return rc;
  int parts = wanted_parts(m, n, k);
  const uint64_t one = (uint64_t) m * (uint64_t) n * 4u;
  if (!work || work_bytes / one < (uint64_t) parts) parts = work ? (int) (work_bytes / one) : 1;
  if (parts < 2) parts = 1;
  else if (int rc = dev.reaches(work, kCall, "work")) return rc;
  p.a = (const uint8_t *) a; p.b = (const uint8_t *) b; p.sa = sa; p.sb = sb;
  p.lda = lda; p.ldb = ldb; p.ldsa = ldsa; p.ldsb = ldsb;
  p.a_shift = ga == 128 ? 7 : 0; p.b_shift = gb == 128 ? 7 : 0;
  p.part = (float *) work;
  hipError_t e;
  if (a_type == BOF_E4M3) e = b_type == BOF_E4M3 ? launch_product<BOF_E4M3, BOF_E4M3>(p, parts, (hipStream_t) stream) : launch_product<BOF_E4M3, BOF_E5M2>(p, parts, (hipStream_t) stream);
  else e = b_type == BOF_E4M3 ? launch_product<BOF_E5M2, BOF_E4M3>(p, parts, (hipStream_t) stream) : launch_product<BOF_E5M2, BOF_E5M2>(p, parts, (hipStream_t) stream);
  BOF_HIP_TRY(e);
  return BOF_OK;
}

}  // extern "C"
