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
// a product of 2^16 next to one of 2^2 leaves nothing of the smaller; across groups of eight nothing is cut): 1.5e-5 of the
// result, relative, on random data.  The rounding of a 16-bit C is larger (relative error against 64 bits of 1021 x 2000 x 4096: bf16
// 1.66e-3 with the cut and without, f16 2.11e-4 and 2.08e-4), though one element in forty of bf16, one in eight of f16,
// rounds to the other neighbour for it.  A 32-bit C, what gradients of weights are added into, is computed WIDE: both operands are widened to bf16, exactly and with their scales applied
// (v_cvt_scalef32_pk_bf16_*), and multiplied by v_mfma_f32_16x16x32_bf16, whose sums are exact to fp32 (measured
// 2.4e-9 relative on 32 products) at half the rate.
#include "f8_common.h"

#include <type_traits>
#include <utility>

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

// a scale as the widening instructions take it: they read the exponent field of a float, as E8M0 (0 is 2^-127, 255 is NaN)
__device__ __forceinline__ float scale_value(uint32_t code) { return __uint_as_float(code << 23); }

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

// alpha * v + beta * C of eight neighbours that all lie inside C
template <int T>
__device__ __forceinline__ void finish_eight(const F8Product &p, int64_t at, f32x4 lo, f32x4 hi) {
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; e++) v[e] = p.alpha * (e < 4 ? lo[e] : hi[e - 4]);
  if (p.beta != 0.f) {
    const Eight<T> c = load_eight<T>(p.c, at, 8);
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = fmaf(p.beta, c.at(e), v[e]);
  }
  store_eight<T>(p.c, at, v, 8);
}

// A wave's sums to C, from row i, column j on: 64 rows at a time through the wave's own part of LDS (rows of 4 Y chunks of four
// floats, XOR-ed with the row), so that a row of C leaves in whole lines.  Rows before i_from and columns before j_from are left
// out.
template <int X, int Y>
__device__ __forceinline__ void store_wave(const F8Product &p, f32x4 (&acc)[X][Y], f32x4 *own, int i, int j, int i_from, int j_from) {
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  constexpr int W = 4 * Y, LANES = 2 * Y;   // chunks in a row, lanes a row
  constexpr int XP = X < 4 ? X : 4;         // tiles at a time
  constexpr int SWZ = W % 8 ? 3 : 7;
#pragma unroll
  for (int part = 0; part < X / XP; part++) {
#pragma unroll
    for (int x = 0; x < XP; x++)
#pragma unroll
      for (int y = 0; y < Y; y++) own[(x * 16 + l16) * W + ((y * 4 + g) ^ (l16 & SWZ))] = acc[part * XP + x][y];
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll 2
    for (int it = 0; it < XP * 16 * LANES / 64; it++) {
      const int r = (it * 64 + lane) / LANES, c2 = (it * 64 + lane) % LANES * 2, row = i + part * XP * 16 + r, col = j + c2 * 4;
      const f32x4 lo = own[r * W + (c2 ^ (r & SWZ))], hi = own[r * W + ((c2 + 1) ^ (r & SWZ))];
      if (row < i_from || row >= p.m) continue;
      if (col >= j_from && col + 8 <= p.n) {
        const int64_t at = (int64_t) row * p.ldc + col;
        if (p.c_type == BOF_BF16) finish_eight<BOF_BF16>(p, at, lo, hi);
        else if (p.c_type == BOF_F16) finish_eight<BOF_F16>(p, at, lo, hi);
        else finish_eight<BOF_F32>(p, at, lo, hi);
      } else {
#pragma unroll
        for (int e = 0; e < 8; e++)
          if (col + e >= j_from && col + e < p.n) finish(p, row, col + e, e < 4 ? lo[e] : hi[e - 4]);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

// ---- tiles of any shape and alignment -----------------------------------------------
// 16 bytes of a row from byte k0 on, zeros from byte k on.  A chunk that ends behind the row is read as the row's last 16 bytes
// and shifted: no branch, so that several may be in flight.
__device__ __forceinline__ u32x4 load_chunk_of_16(const uint8_t *row, int k0, int k) {   // k >= 16
  const int at = min(k0, k - 16), over = k0 - at;
  unsigned __int128 w;
  __builtin_memcpy(&w, row + at, 16);
  w = over < 16 ? w >> (8 * over) : 0;
  u32x4 v;
  __builtin_memcpy(&v, &w, 16);
  return v;
}
__device__ __forceinline__ u32x4 load_chunk(const uint8_t *row, int k0, int k) {
  if (k >= 16) return load_chunk_of_16(row, k0, k);
  u32x4 v;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    v[e] = 0;
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (k0 + 4 * e + i < k) v[e] |= (uint32_t) row[k0 + 4 * e + i] << (8 * i);
  }
  return v;
}

// One workgroup of four waves, 128 x 128 of C, one block of k at a time through LDS (rows of 128 bytes, their 16-byte
// chunks XOR-ed with the row so that the fragment reads meet no bank twice).  Rows outside the matrices read the last
// row and are not stored.  For k < 128 and for rows so far apart that offsets inside a tile need 64 bits.  Nothing is in flight
// while it multiplies: latency bounds it, 8192 x 8192 x 96 in 61 us (2.2 TB/s of C); with C stored element by element 135 us.
template <int TA, int TB, bool WIDE>
__global__ void __launch_bounds__(256) f8_tile_any_kernel(F8Product p) {
  __shared__ u32x4 lds[4][128 * 8];   // rows of A, of B; the waves' sums in the end
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int tiles_n = (p.n + 127) >> 7;
  const int i0 = (int) (blockIdx.x / tiles_n) * 128, j0 = (int) (blockIdx.x % tiles_n) * 128;
  const int wi = (wave >> 1) * 64, wj = (wave & 1) * 64;
  const int l16 = lane & 15, g = lane >> 4;
  const int nb = (p.k + 127) >> 7;
  f32x4 acc[4][4];
#pragma unroll
  for (int x = 0; x < 16; x++) acc[x >> 2][x & 3] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int blk = 0; blk < nb; blk++) {
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
  store_wave<4, 4>(p, acc, (f32x4 *) lds[wave], i0 + wi, j0 + wj, 0, 0);
}

// ---- tiles ---------------------------------------------------------------------------
// Four waves, X x Y tiles of 16 x 16 each, 2 x 2 waves: a workgroup owns 32 X rows and 32 Y columns of C.  8 x 8 (256 x 256):
// one wave on each SIMD, 64 accumulators of four floats = 256 registers (the accumulator half of the file), the other half
// holds the fragments.
//
// A slab is one block of k: rows of 128 bytes; both operands lie in LDS twice.  DMA: rows reach LDS without touching
// registers -- one global_load_lds_dwordx4 moves 8 rows, lane l fetching chunk (l & 7) ^ (l >> 3) of row l >> 3, so that the
// image is [row][chunk ^ (row & 7)] and a fragment read (16 rows x 16 bytes) meets every bank once.  It needs rows aligned to
// four bytes; for others (DMA = false) a thread loads its 16-byte chunks of the same rows, unaligned, and writes them to the
// same places one slab later.  Per slab and wave of 8 x 8: 64 MFMAs of 32 cycles, 32 ds_read_b128, 16 pieces.
//
// The A fragments of a slab are read into registers during the slab BEFORE (twice X x 8 registers), the B fragments one tile
// ahead.  The barrier of a slab stands in front of its last row of tiles: by then every wave has read all it wants from this
// slab's B image and the next slab's A image, and the pieces of the next B and the next but one A image, issued at the slab's
// start, have landed.  That is time enough from the L2, not from memory, and a CU has only so many misses in flight: so
// every lane also touches one line of the slab but three or four, a quarter of the tile's rows a workgroup -- those of an
// XCD that share the rows touch the other quarters (8192 cubed, zeros for data: 410 us without, 329 us with).
//
// Bound by the card's power at 8192 cubed: 329 us (3.3 PFLOP/s) on zeros, 396 to 418 us (2.8 to 2.6) on random bytes, card by card.
//
// A fragment's scale byte is read from LDS along with it.  No vector instruction is left in a slab but a few for the whole of it.
//
// A tile at the lower or right edge starts earlier (at m - 32 X, n - 32 Y), so that every row it fetches exists; what lies in
// the tile before is not stored again.
__device__ __forceinline__ uint32_t lds_address(const void *p) {
  return (uint32_t) (uintptr_t) (const __attribute__((address_space(3))) void *) p;
}
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// 64 lanes x 16 bytes from base + voff to LDS, contiguous from `to` on (M0 carries the destination)
__device__ __forceinline__ void dma16(uint32_t voff, uint64_t base, uint32_t to) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" :: "v"(voff), "s"(base), "s"(to) : "memory", "m0");
}
// one word a lane from `from` to LDS at `to`, which nobody reads: brings the line into the L2
__device__ __forceinline__ void touch(const uint8_t *from, uint32_t to) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" :: "v"(from), "s"(to) : "memory", "m0");
}
#pragma clang diagnostic pop

// 16 bytes of memory (not of LDS or scratch, which the type says: a load through an address of any kind also counts as one of LDS,
// and the wait for fragments in front of a barrier would wait for memory)
__device__ __forceinline__ u32x4 load16(uint64_t from, uint32_t off) {
  u32x4 v;
  __builtin_memcpy(&v, (const uint8_t *) ((const __attribute__((address_space(1))) uint8_t *) from + off), 16);
  return v;
}

// workgroups go round the 8 XCDs; tiles of one XCD are neighbours (each XCD has its own L2), GROUP rows of tiles deep
__device__ __forceinline__ void tile_of(int bid, int tiles_m, int tiles_n, int group, int &tm, int &tn) {
  const int nwg = tiles_m * tiles_n, q = nwg >> 3, r = nwg & 7, xcd = bid & 7, idx = bid >> 3;
  bid = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + idx;
  const int per = group * tiles_n, first = bid / per * group, deep = min(tiles_m - first, group);
  tm = first + bid % per % deep;
  tn = bid % per / deep;
}

// Scales in LDS: for every row of a tile the bytes of 32 blocks, in two halves of 16, 20 bytes from row to row (no bank twice).
// Both halves are filled in front of the loop over k; later on, when the loop enters a half, the other one is filled with the
// bytes behind it.  (That waits for all that is in flight, once in 16 blocks: rows of up to 4096 never do.)
constexpr int scale_chunks(int rows) { return (rows * 40 + 15) / 16; }   // of 16 bytes, both halves
__device__ __forceinline__ int scale_byte(int kb, int rows) { return ((kb >> 4) & 1) * rows * 20 + (kb & 15); }
// (in the loop: rows are longer than 16 there.  The wait is one that the compiler sees: else it puts its own, for a register that
// may still be loading, in front of every step's reads, and with it waits for the pieces in flight)
__device__ __forceinline__ u32x4 next_scales(const uint8_t *row, int b, int nb) {
  const u32x4 v = load_chunk_of_16(row, b, nb);
  __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0)
  return v;
}
__device__ __forceinline__ void put_scales(uint8_t *half, int row, u32x4 v) {
  uint32_t *to = (uint32_t *) (half + row * 20);
#pragma unroll
  for (int e = 0; e < 4; e++) to[e] = v[e];
}

__device__ __forceinline__ i32x8 both(u32x4 lo, u32x4 hi) {
  return i32x8{(int) lo[0], (int) lo[1], (int) lo[2], (int) lo[3], (int) hi[0], (int) hi[1], (int) hi[2], (int) hi[3]};
}

// The slab's product, its accumulators pinned to the accumulator half of the register file (left to itself the compiler moves
// them through both: 200 copies a slab).  The compiler puts no wait states around inline assembly, so they are part of it: two
// in front of the instruction, for an operand or a scale that a vector instruction may have written last (8192 cubed in 418 us,
// 413 without them on the same card); 32 behind the last one, in settle(), which hands the accumulators on.  What comes
// between -- nothing but these instructions touches an accumulator -- the compiler decides: tests/test_f8_assembly.py looks at it.
template <int TA, int TB>
__device__ __forceinline__ void mma_pinned(const Frag<false> &b, const Frag<false> &a, f32x4 &acc) {
  asm volatile("s_nop 1\n\tv_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0] cbsz:%5 blgp:%6"
               : "+a"(acc) : "v"(b.q), "v"(a.q), "v"(b.s), "v"(a.s), "n"(TB == BOF_E4M3 ? 0 : 1), "n"(TA == BOF_E4M3 ? 0 : 1));
}
template <int X, int Y>
__device__ __forceinline__ void settle(f32x4 (&acc)[X][Y]) {
  asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
  for (int x = 0; x < X * Y; x++) asm volatile("" : "+a"(acc[x / Y][x % Y]));
}

template <int X, int Y, bool DMA>
struct Slab {
  static constexpr int A_IMAGE = 256 * X, B_IMAGE = 256 * Y;       // chunks of 16 bytes in an image
  static constexpr int B0 = 2 * A_IMAGE, S0 = B0 + 2 * B_IMAGE;    // where the B images and the scales begin
  static constexpr int J0 = S0 + scale_chunks(32 * (X + Y)), CHUNKS = J0 + 64;   // scales, and where touches go
  static constexpr int PIECES = X + Y;                             // of 32 rows (8 a wave)
  static constexpr bool TOUCH = DMA;
  u32x4 *lds;
  uint32_t a_voff, b_voff;       // of this thread's row and chunk in a piece
  uint64_t a_step, b_step;       // bytes from piece to piece
  uint32_t a_to, b_to;           // LDS addresses of this wave's pieces in image 0 (DMA)
  int put;                       // this thread's chunk in a piece (staged)
  int a_lo, a_hi, b_lo, b_hi;    // this lane's chunks in the image, of tile 0
  const uint8_t *sa, *sb;        // this lane's scale bytes of tile 0
  const uint8_t *ahead;          // the line this lane touches
  uint32_t junk;
  u32x4 staged[DMA ? 1 : PIECES];
};

template <int TA, int TB, int X, int Y, bool DMA, int P>
__device__ __forceinline__ void slab(Slab<X, Y, DMA> &s, uint64_t b_next, uint64_t a_next, uint32_t ahead, int sc_b, int sc_a,
                                     Frag<false> (&fa)[2][X], Frag<false> (&fb)[2], f32x4 (&acc)[X][Y]) {
  using S = Slab<X, Y, DMA>;
  // piece p: B first, into the other B image; then A, into the image whose fragments are in registers
  auto piece = [&](int q) {
    const bool b = q < Y;
    const int r = b ? q : q - Y;
    const uint64_t from = b ? b_next + r * s.b_step : a_next + r * s.a_step;
    if constexpr (DMA) {
      dma16(b ? s.b_voff : s.a_voff, from, (b ? s.b_to + (P ^ 1) * S::B_IMAGE * 16 : s.a_to + P * S::A_IMAGE * 16) + r * 4096);
    } else {
      s.lds[s.put + (b ? S::B0 + (P ^ 1) * S::B_IMAGE : P * S::A_IMAGE) + r * 256] = s.staged[q];
      asm volatile("" ::: "memory");   // (the load into the same registers stays behind)
      s.staged[q] = load16(from, b ? s.b_voff : s.a_voff);
    }
  };
  constexpr int N = X * Y, LAST = N - X;   // MFMAs, those in front of the barrier
#pragma unroll
  for (int y = 0; y < Y; y++) {
    if (y == Y - 1) {
      if constexpr (DMA) asm volatile("s_waitcnt vmcnt(%0)" :: "n"(S::TOUCH ? 1 : 0) : "memory");
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    }
#pragma unroll
    for (int x = 0; x < X; x++) {
      const int at = y * X + x;
      mma_pinned<TA, TB>(fb[y & 1], fa[P][x], acc[x][y]);
      if (x == 1) {   // the next B tile: of this slab, or the next one's first
        const int from = (y < Y - 1 ? P : P ^ 1) * S::B_IMAGE + (y < Y - 1 ? y + 1 : 0) * 128;
        fb[(y + 1) & 1].q = both(s.lds[s.b_lo + from], s.lds[s.b_hi + from]);
        fb[(y + 1) & 1].s = s.sb[(y < Y - 1 ? sc_b : sc_a) + (y < Y - 1 ? y + 1 : 0) * 320];
      }
      // the pieces: behind two MFMAs of three from the start on, then the touch, which is waited for
      // at the barrier of the next slab.  (One piece for every MFMA is more than the texture unit takes, one for every second or
      // third gives them less time to land: 8192 cubed 329 us, 349, 334 and 365 for zeros.)
      const int q = at / 3 * 2 + at % 3;
      if (at % 3 != 2 && q < S::PIECES) piece(q);
      if (S::TOUCH && at == S::PIECES / 2 * 3) touch(s.ahead + ahead, s.junk);
      // the next slab's A fragments: X of them between a quarter and three quarters of the slab
      constexpr int F0 = N / 4, STEP = (LAST - F0 - 2) / X > 4 ? 4 : (LAST - F0 - 2) / X;
      if (at >= F0 && (at - F0) % STEP == 0 && (at - F0) / STEP < X) {
        const int f = (at - F0) / STEP, from = (P ^ 1) * S::A_IMAGE + f * 128;
        fa[P ^ 1][f].q = both(s.lds[s.a_lo + from], s.lds[s.a_hi + from]);
        fa[P ^ 1][f].s = s.sa[sc_a + f * 320];
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  static_assert(S::PIECES <= LAST, "every piece finds its place in front of the barrier");
}

template <int TA, int TB, int X, int Y, bool DMA>
__global__ void __launch_bounds__(256, 1) f8_tile_kernel(F8Product p, int tiles_m, int tiles_n) {
  using S = Slab<X, Y, DMA>;
  __shared__ u32x4 lds[S::CHUNKS];
  constexpr int TM = 32 * X, TN = 32 * Y;
  int tm, tn;
  tile_of(blockIdx.x, tiles_m, tiles_n, 4, tm, tn);
  const int i0 = min(tm * TM, p.m - TM), j0 = min(tn * TN, p.n - TN);
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wi = (wave >> 1) * 16 * X, wj = (wave & 1) * 16 * Y;
  const int l16 = lane & 15, g = lane >> 4;
  const int nb = (p.k + 127) >> 7, full = p.k >> 7;   // whole slabs, one at least
  S s;
  s.lds = lds;
  const int r8 = lane >> 3, chunk = (DMA ? (lane & 7) ^ r8 : lane & 7) << 4;
  s.a_voff = (uint32_t) (8 * wave + r8) * (uint32_t) p.lda + chunk;
  s.b_voff = (uint32_t) (8 * wave + r8) * (uint32_t) p.ldb + chunk;
  s.a_step = (uint64_t) p.lda * 32;
  s.b_step = (uint64_t) p.ldb * 32;
  s.a_to = lds_address(lds) + wave * 1024;
  s.b_to = s.a_to + S::B0 * 16;
  s.put = (8 * wave + r8) * 8 + ((lane & 7) ^ r8);
  s.a_lo = (wi + l16) * 8 + (g ^ (l16 & 7)); s.a_hi = (wi + l16) * 8 + ((g + 4) ^ (l16 & 7));
  s.b_lo = S::B0 + (wj + l16) * 8 + (g ^ (l16 & 7)); s.b_hi = S::B0 + (wj + l16) * 8 + ((g + 4) ^ (l16 & 7));
  uint8_t *const scales = (uint8_t *) (lds + S::S0);
  s.sa = scales + (wi + l16) * 20;
  s.sb = scales + (TM + wj + l16) * 20;
  // thread t has the scales of row t of A and of row t of B
  const uint8_t *const sa_row = p.sa + (int64_t) ((i0 + t) >> p.a_shift) * p.ldsa, *const sb_row = p.sb + (int64_t) ((j0 + t) >> p.b_shift) * p.ldsb;
  auto half_of = [&](int seg) { return scales + (seg & 1) * (TM + TN) * 20; };
  const uint64_t a_org = reinterpret_cast<uint64_t>(p.a + (int64_t) i0 * p.lda), b_org = reinterpret_cast<uint64_t>(p.b + (int64_t) j0 * p.ldb);
  auto a_at = [&](int kb) { return a_org + (uint64_t) min(kb, full - 1) * 128; };   // (behind the last slab: the last one again)
  auto b_at = [&](int kb) { return b_org + (uint64_t) min(kb, full - 1) * 128; };
  auto ahead_at = [&](int kb) { return (uint32_t) min(kb + 4, full - 1) * 128u; };
  {
    const int r = wave * 16 + l16, half = (lane & 32) * 2;
    s.ahead = (lane & 16 ? p.b + (int64_t) (j0 + (tm & 3) * (TN / 4) + r % (TN / 4)) * p.ldb : p.a + (int64_t) (i0 + (tn & 3) * (TM / 4) + r % (TM / 4)) * p.lda) + half;
    s.junk = lds_address(lds) + S::J0 * 16 + wave * 256;
  }
  f32x4 acc[X][Y];
#pragma unroll
  for (int x = 0; x < X * Y; x++) acc[x / Y][x % Y] = f32x4{0.f, 0.f, 0.f, 0.f};
  Frag<false> fa[2][X], fb[2];
  // A of the first two slabs, B of the first (staged: and what the first slab is to write), the scales of its four
#pragma unroll
  for (int r = 0; r < X; r++) {
    if constexpr (DMA) {
      dma16(s.a_voff, a_at(0) + r * s.a_step, s.a_to + r * 4096);
      dma16(s.a_voff, a_at(1) + r * s.a_step, s.a_to + S::A_IMAGE * 16 + r * 4096);
    } else {
      u32x4 v[2];
      v[0] = load16(a_at(0) + r * s.a_step, s.a_voff);
      v[1] = load16(a_at(1) + r * s.a_step, s.a_voff);
      s.staged[Y + r] = load16(a_at(2) + r * s.a_step, s.a_voff);
      lds[s.put + r * 256] = v[0];
      lds[s.put + S::A_IMAGE + r * 256] = v[1];
    }
  }
#pragma unroll
  for (int r = 0; r < Y; r++) {
    if constexpr (DMA) {
      dma16(s.b_voff, b_at(0) + r * s.b_step, s.b_to + r * 4096);
    } else {
      u32x4 v;
      v = load16(b_at(0) + r * s.b_step, s.b_voff);
      s.staged[r] = load16(b_at(1) + r * s.b_step, s.b_voff);
      lds[s.put + S::B0 + r * 256] = v;
    }
  }
  {
    const u32x4 v[4] = {load_chunk(sa_row, 0, nb), load_chunk(sb_row, 0, nb), load_chunk(sa_row, 16, nb), load_chunk(sb_row, 16, nb)};
    put_scales(half_of(0), t, v[0]);
    put_scales(half_of(0), TM + t, v[1]);
    put_scales(half_of(1), t, v[2]);
    put_scales(half_of(1), TM + t, v[3]);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  auto byte_of = [](int kb) { return scale_byte(kb, TM + TN); };
#pragma unroll
  for (int x = 0; x < X; x++) {
    fa[0][x].q = both(lds[s.a_lo + x * 128], lds[s.a_hi + x * 128]);
    fa[0][x].s = s.sa[byte_of(0) + x * 320];
  }
  fb[0].q = both(lds[s.b_lo], lds[s.b_hi]);
  fb[0].s = s.sb[byte_of(0)];
  __syncthreads();
  int kb = 0;
  for (; kb + 2 <= full; kb += 2) {
    if ((kb & 15) == 0 && kb > 0) {
      const u32x4 v[2] = {next_scales(sa_row, kb + 16, nb), next_scales(sb_row, kb + 16, nb)};
      put_scales(half_of((kb >> 4) + 1), t, v[0]);
      put_scales(half_of((kb >> 4) + 1), TM + t, v[1]);
    }
    slab<TA, TB, X, Y, DMA, 0>(s, DMA ? b_at(kb + 1) : b_at(kb + 2), DMA ? a_at(kb + 2) : a_at(kb + 3), ahead_at(kb), byte_of(kb), byte_of(kb + 1), fa, fb, acc);
    slab<TA, TB, X, Y, DMA, 1>(s, DMA ? b_at(kb + 2) : b_at(kb + 3), DMA ? a_at(kb + 3) : a_at(kb + 4), ahead_at(kb + 1), byte_of(kb + 1), byte_of(kb + 2), fa, fb, acc);
  }
  if (kb < full) slab<TA, TB, X, Y, DMA, 0>(s, b_at(kb), a_at(kb), ahead_at(kb), byte_of(kb), byte_of(kb), fa, fb, acc);
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __syncthreads();
  if (nb > full) {   // the short block: through registers, zeros behind k
    u32x4 v[X + Y];
#pragma unroll
    for (int u = 0; u < X + Y; u++)
      v[u] = load_chunk_of_16(u < X ? p.a + (int64_t) (i0 + 32 * u + 8 * wave + r8) * p.lda : p.b + (int64_t) (j0 + 32 * (u - X) + 8 * wave + r8) * p.ldb,
                        full * 128 + (lane & 7) * 16, p.k);
    const uint8_t sa_last = sa_row[full], sb_last = sb_row[full];
#pragma unroll
    for (int u = 0; u < X + Y; u++) lds[s.put + (u < X ? u * 256 : S::B0 + (u - X) * 256)] = v[u];
    scales[t * 20] = sa_last;
    scales[(TM + t) * 20] = sb_last;
    __syncthreads();
#pragma unroll
    for (int x = 0; x < X; x++) {
      fa[0][x].q = both(lds[s.a_lo + x * 128], lds[s.a_hi + x * 128]);
      fa[0][x].s = s.sa[x * 320];
    }
#pragma unroll
    for (int y = 0; y < Y; y++) {
      Frag<false> b;
      b.q = both(lds[s.b_lo + y * 128], lds[s.b_hi + y * 128]);
      b.s = s.sb[y * 320];
#pragma unroll
      for (int x = 0; x < X; x++) mma_pinned<TA, TB>(b, fa[0][x], acc[x][y]);
    }
    __syncthreads();
  }
  settle(acc);
  store_wave<X, Y>(p, acc, (f32x4 *) lds + wave * (S::S0 / 4), i0 + wi, j0 + wj, max(tm * TM, i0 + wi), max(tn * TN, j0 + wj));
}

// A part of a product that is split along k writes its sums instead of C.
__device__ __forceinline__ F8Product part_of(F8Product p, int z) {
  if (p.part) {
    p.c = p.part + (int64_t) z * p.m * p.n;
    p.c_type = BOF_F32;
    p.ldc = p.n;
    p.alpha = 1.f;
    p.beta = 0.f;
  }
  return p;
}

// ---- outputs of few tiles ------------------------------------------------------------
// Four waves, X x Y tiles of 16 x 16 each: what counts here is not the matrix unit but the way to memory, so LDS is a ring of ST
// blocks of k.  Step t multiplies block t out of registers, reads the fragments of block t + 1 into the other set of them, and
// fetches block t + ST into the place that block t has left: a piece has ST - 1 steps to land, a fragment one.  The barrier of a
// step stands in front of its last MFMAs: by then every wave has read what it wants from LDS, and block t + 2 has landed.  Rows,
// chunks, scales and the staged form are those of the tiles above (staged: written three blocks ahead, loaded two steps before
// that); rows behind the last one are read as the last one and not stored.
//
// 128 x 128, four blocks, one workgroup a CU: a block takes 0.5 us of it, two thirds of that LDS (64 KB of fragments are read
// for 32 KB of rows, at 128 bytes a cycle); two images of LDS and two workgroups a CU took 0.8 us on an idle card:
// 1024 x 4096 x 4096 in 21 us for 28.
// Two of 128 x 128 a CU with two blocks each: slower in its steps, which wait for their fetches, but one loads and stores
// while the other multiplies: for many tiles and few blocks.
// 128 x 160: the same as the first, for outputs that it covers in fewer rounds of 256 workgroups: 1021 x 5000 x 4100 without padding in 34.9 us for 53
// (rows of 4100 bytes lie across the L2's lines and cost 5 of them, the short block 4).
// 256 x 128, three blocks: for one round of what takes 128 x 128 two: 2048 x 4096 x 4096 in 34 us for 38.
// 64 x 32, six blocks, two workgroups a CU, for few rows and few columns: bound by the bytes of B, 48 x 8192 x 4096 in 9.1 us
// (3.7 TB/s), 4.7 TB/s at 8 x 8192 x 8192; with eight blocks and one workgroup a CU 128 x 8192 x 4096 took 15.5 us for 13.
// Rows through registers: 48 x 8192 x 4099 in 15.5 us, 1024 x 4096 x 4099 in 38.5, 1021 x 5000 x 4099 in 47.0 (128 x 160).
template <int X_, int Y_, int WM_, int ST_, bool DMA>
struct Ring {
  static constexpr int X = X_, Y = Y_, WM = WM_, WN = 4 / WM, ST = ST_;          // tiles a wave, waves along m and n, blocks in the ring
  static constexpr int TM = 16 * X * WM, TN = 16 * Y * WN;                       // rows and columns of C
  static constexpr int B0 = 8 * TM, BLOCK = B0 + 8 * TN, S0 = ST * BLOCK;        // chunks of 16 bytes: B rows, a block, where the scales begin
  static constexpr int ROWS = TM + TN, CHUNKS = S0 + scale_chunks(ROWS);
  static constexpr int PA = TM / 32, PIECES = PA + TN / 32;                      // of 32 rows (8 a wave), A's, then B's
  static constexpr int STEPS = ST % 2 ? 2 * ST : ST;                             // until place in the ring and set of fragments come round
  u32x4 *lds;
  uint32_t voff[PIECES];         // of this thread's row and chunk
  uint32_t to;                   // LDS address of this wave's part of a piece in block 0 (DMA)
  int put;                       // this thread's chunk in a piece (staged)
  int a_lo, a_hi, b_lo, b_hi;    // this lane's chunks in a block, of tile 0
  const uint8_t *sa, *sb;        // this lane's scale bytes of tile 0
  u32x4 staged[2][DMA ? 1 : PIECES];
};

// Step t, U = t mod STEPS; a, b: where the block to fetch begins; sc: the scale byte of block t + 1.
template <int TA, int TB, bool DMA, int U, class S, int X, int Y>
__device__ __forceinline__ void ring_step(S &s, uint64_t a, uint64_t b, int sc, Frag<false> (&fa)[2][X], Frag<false> (&fb)[2][Y], f32x4 (&acc)[X][Y]) {
  constexpr int P = U & 1, AT = U % S::ST, N = X * Y, LAST = N - N / 5, WORK = 2 * S::PIECES;   // MFMAs, those in front of the barrier, work beside them
  static_assert(X + Y == S::PIECES, "a fragment to read for every piece");
  auto piece = [&](int q) {
    const uint64_t from = q < S::PA ? a : b;
    if constexpr (DMA) {
      dma16(s.voff[q], from, s.to + AT * S::BLOCK * 16 + q * 4096);
    } else {
      u32x4 &v = s.staged[P][q];
      s.lds[s.put + (AT + 3) % S::ST * S::BLOCK + q * 256] = v;
      asm volatile("" ::: "memory");   // (the load into the same registers stays behind)
      v = load16(from, s.voff[q]);
    }
  };
  auto read = [&](int f) {   // fragment f of the next block
    const u32x4 *block = s.lds + (AT + 1) % S::ST * S::BLOCK;
    if (f < Y) {
      fb[P ^ 1][f].q = both(block[s.b_lo + f * 128], block[s.b_hi + f * 128]);
      fb[P ^ 1][f].s = s.sb[sc + f * 320];
    } else {
      fa[P ^ 1][f - Y].q = both(block[s.a_lo + (f - Y) * 128], block[s.a_hi + (f - Y) * 128]);
      fa[P ^ 1][f - Y].s = s.sa[sc + (f - Y) * 320];
    }
  };
#pragma unroll
  for (int at = 0; at <= N; at++) {
    if (at == LAST) {
      if constexpr (DMA) asm volatile("s_waitcnt vmcnt(%0)" :: "n"((S::ST - 2) * S::PIECES) : "memory");   // block t + 2 has landed
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    }
    if (at == N) break;
    acc[at % X][at / X] = mma<TA, TB, false>(fb[P][at / X], fa[P][at % X], acc[at % X][at / X]);
    if (at < LAST) {
#pragma unroll
      for (int w = at * WORK / LAST; w < (at + 1) * WORK / LAST; w++) {
        if (w & 1) read(w >> 1);
        else piece(w >> 1);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

template <class F, int... U>
__device__ __forceinline__ void each_place(F &&f, std::integer_sequence<int, U...>) { (f(std::integral_constant<int, U>()), ...); }

template <int TA, int TB, int X, int Y, int WM, int ST, bool DMA>
__global__ void __launch_bounds__(256, X >= 4 && ST > 2 ? 1 : 2) f8_ring_kernel(F8Product q, int tiles_m, int tiles_n) {
  using S = Ring<X, Y, WM, ST, DMA>;
  __shared__ u32x4 lds[S::CHUNKS];
  const F8Product p = part_of(q, blockIdx.y);
  int tm, tn;
  tile_of(blockIdx.x, tiles_m, tiles_n, 4, tm, tn);
  const int i0 = tm * S::TM, j0 = tn * S::TN;
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wi = wave / S::WN * 16 * X, wj = wave % S::WN * 16 * Y;
  const int l16 = lane & 15, g = lane >> 4;
  const int nb = (p.k + 127) >> 7, all = p.k >> 7;
  const int b0 = blockIdx.y * p.blocks_per_part, full = min(all, b0 + p.blocks_per_part);   // blocks b0 .. full - 1, one at least
  const bool tail = nb > all && blockIdx.y == gridDim.y - 1;
  S s;
  s.lds = lds;
  const int r8 = lane >> 3, chunk = (DMA ? (lane & 7) ^ r8 : lane & 7) << 4;
#pragma unroll
  for (int r = 0; r < S::PIECES; r++)
    s.voff[r] = (r < S::PA ? (uint32_t) min(32 * r + 8 * wave + r8, p.m - 1 - i0) * (uint32_t) p.lda
                           : (uint32_t) min(32 * (r - S::PA) + 8 * wave + r8, p.n - 1 - j0) * (uint32_t) p.ldb) + chunk;
  s.to = lds_address(lds) + wave * 1024;
  s.put = (8 * wave + r8) * 8 + ((lane & 7) ^ r8);
  s.a_lo = (wi + l16) * 8 + (g ^ (l16 & 7)); s.a_hi = (wi + l16) * 8 + ((g + 4) ^ (l16 & 7));
  s.b_lo = S::B0 + (wj + l16) * 8 + (g ^ (l16 & 7)); s.b_hi = S::B0 + (wj + l16) * 8 + ((g + 4) ^ (l16 & 7));
  uint8_t *const scales = (uint8_t *) (lds + S::S0);
  s.sa = scales + (wi + l16) * 20;
  s.sb = scales + (S::TM + wj + l16) * 20;
  // thread t has the scales of row t of A and then B, and those of row 256 + t
  auto scales_of = [&](int row) {
    return row < S::TM ? p.sa + (int64_t) (min(i0 + row, p.m - 1) >> p.a_shift) * p.ldsa
                       : p.sb + (int64_t) (min(j0 + min(row - S::TM, S::TN - 1), p.n - 1) >> p.b_shift) * p.ldsb;
  };
  const uint8_t *const s_row = scales_of(t), *const s_row2 = S::ROWS > 256 ? scales_of(t + 256) : s_row;
  auto put_half = [&](int seg, u32x4 v, u32x4 v2) {
    if (S::ROWS >= 256 || t < S::ROWS) put_scales(scales + (seg & 1) * S::ROWS * 20, t, v);
    if (S::ROWS > 256 && t < S::ROWS - 256) put_scales(scales + (seg & 1) * S::ROWS * 20, t + 256, v2);
  };
  const uint64_t a_org = reinterpret_cast<uint64_t>(p.a + (int64_t) i0 * p.lda), b_org = reinterpret_cast<uint64_t>(p.b + (int64_t) j0 * p.ldb);
  auto a_at = [&](int kb) { return a_org + (uint64_t) min(kb, full - 1) * 128; };   // (behind the last block: the last one again)
  auto b_at = [&](int kb) { return b_org + (uint64_t) min(kb, full - 1) * 128; };
  f32x4 acc[X][Y];
#pragma unroll
  for (int x = 0; x < X * Y; x++) acc[x / Y][x % Y] = f32x4{0.f, 0.f, 0.f, 0.f};
  Frag<false> fa[2][X], fb[2][Y];
  // the first blocks: as many as fit on their way to LDS; staged: three, and two in registers
#pragma unroll
  for (int u = 0; u < (DMA ? S::ST : 3); u++)
#pragma unroll
    for (int r = 0; r < S::PIECES; r++) {
      const uint64_t from = r < S::PA ? a_at(b0 + u) : b_at(b0 + u);
      if constexpr (DMA) {
        dma16(s.voff[r], from, s.to + u * S::BLOCK * 16 + r * 4096);
      } else {
        u32x4 v;
        v = load16(from, s.voff[r]);
        lds[s.put + u * S::BLOCK + r * 256] = v;
      }
    }
  if constexpr (!DMA) {
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
      for (int r = 0; r < S::PIECES; r++)
        s.staged[u][r] = load16(r < S::PA ? a_at(b0 + 3 + u) : b_at(b0 + 3 + u), s.voff[r]);
  }
  int seg = b0 >> 4;   // LDS has the scales of blocks 16 seg .. 16 seg + 31
  {
    const u32x4 v0 = load_chunk(s_row, seg * 16, nb), v1 = load_chunk(s_row, seg * 16 + 16, nb);
    u32x4 w0 = v0, w1 = v1;
    if constexpr (S::ROWS > 256) { w0 = load_chunk(s_row2, seg * 16, nb); w1 = load_chunk(s_row2, seg * 16 + 16, nb); }
    put_half(seg, v0, w0);
    put_half(seg + 1, v1, w1);
  }
  if constexpr (DMA) asm volatile("s_waitcnt vmcnt(%0)" :: "n"((S::ST - 2) * S::PIECES) : "memory");   // the first two blocks (and the scales)
  __syncthreads();
  auto byte_of = [](int kb) { return scale_byte(kb, S::ROWS); };
  auto fragments = [&](int sc) {
#pragma unroll
    for (int x = 0; x < X; x++) {
      fa[0][x].q = both(lds[s.a_lo + x * 128], lds[s.a_hi + x * 128]);
      fa[0][x].s = s.sa[sc + x * 320];
    }
#pragma unroll
    for (int y = 0; y < Y; y++) {
      fb[0][y].q = both(lds[s.b_lo + y * 128], lds[s.b_hi + y * 128]);
      fb[0][y].s = s.sb[sc + y * 320];
    }
  };
  fragments(byte_of(b0));
  __syncthreads();
  int kb = b0;
  auto next = [&](auto place) {   // one step, at its place in the ring
    constexpr int U = decltype(place)::value, AHEAD = DMA ? ST : 5;
    ring_step<TA, TB, DMA, U>(s, a_at(kb + AHEAD), b_at(kb + AHEAD), byte_of(kb + 1), fa, fb, acc);
    kb++;
  };
  auto more_scales = [&] {        // the half that is read for the first time ten steps later at the earliest
    if (kb >> 4 == seg) return;
    seg++;
    const u32x4 v = next_scales(s_row, seg * 16 + 16, nb);
    u32x4 w = v;
    if constexpr (S::ROWS > 256) w = next_scales(s_row2, seg * 16 + 16, nb);
    put_half(seg + 1, v, w);
  };
  while (kb + S::STEPS <= full) {
    more_scales();
    each_place(next, std::make_integer_sequence<int, S::STEPS>());
  }
  more_scales();
  each_place([&](auto place) { if (kb < full) next(place); }, std::make_integer_sequence<int, S::STEPS - 1>());
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __syncthreads();
  if (tail) {   // the short block: through registers, zeros behind k
    u32x4 v[S::PIECES];
#pragma unroll
    for (int r = 0; r < S::PIECES; r++) {
      const int row = (r < S::PA ? r : r - S::PA) * 32 + 8 * wave + r8;
      v[r] = load_chunk_of_16(r < S::PA ? p.a + (int64_t) min(i0 + row, p.m - 1) * p.lda : p.b + (int64_t) min(j0 + row, p.n - 1) * p.ldb,
                              all * 128 + (lane & 7) * 16, p.k);
    }
    const uint8_t s_last = s_row[all], s_last2 = s_row2[all];
#pragma unroll
    for (int r = 0; r < S::PIECES; r++) lds[s.put + r * 256] = v[r];
    if (t < S::ROWS) scales[t * 20] = s_last;
    if (S::ROWS > 256 && t < S::ROWS - 256) scales[(t + 256) * 20] = s_last2;
    __syncthreads();
    fragments(0);
#pragma unroll
    for (int at = 0; at < X * Y; at++) acc[at % X][at / X] = mma<TA, TB, false>(fb[0][at / X], fa[0][at % X], acc[at % X][at / X]);
    __syncthreads();
  }
  store_wave<X, Y>(p, acc, (f32x4 *) lds + wave * (S::S0 / 4), i0 + wi, j0 + wj, 0, 0);
}

// ---- tiles, wide ---------------------------------------------------------------------
// A 32-bit C: fragments are widened to bf16 in registers, 8 conversions for 16 bytes a lane, and multiplied by 2
// instructions of 16 cycles.  A SIMD holds TWO waves, so that one converts while the other multiplies: a workgroup of eight
// owns 32 X rows and 128 columns of C, waves 0-3 work on the first half of every block of k, waves 4-7 on the second, each
// with sums of its own that are added in the end.
//
// LDS: three slots of one block (A and B rows of 128 bytes, swizzled as above) and the scales.  Step t multiplies block t
// out of registers, reads block t + 1 into them -- every fragment as soon as its predecessor is widened -- and fetches block
// t + 3 into the slot that block t has left: a piece has two steps to land, a fragment one.  A barrier ends each step.
//
// 256 x 128, X = 8: 4096 x 2048 x 16384 in 218 to 227 us (1.24 PFLOP/s), card by card: the matrix unit, at the clock that the card's power leaves it, and
// the conversions that do not fit beside it.  128 x 128, X = 4, for outputs of few tiles: 128 x 4096 x 4096 in 19.6 us.
template <int X>
struct WideSlab {
  static constexpr int A_IMAGE = 256 * X, SLOT = A_IMAGE + 1024;   // chunks of 16 bytes
  static constexpr int S0 = 3 * SLOT, ROWS = 32 * X + 128, CHUNKS = S0 + scale_chunks(ROWS);
  static constexpr int PIECES = (X + 4) / 2;                       // of 64 rows (8 a wave)
};

template <int TA, int TB, int X, bool DMA>
__global__ void __launch_bounds__(512, 1) f8_wide_kernel(F8Product q, int tiles_m, int tiles_n) {
  using S = WideSlab<X>;
  __shared__ u32x4 lds[S::CHUNKS];
  const F8Product p = part_of(q, blockIdx.y);
  constexpr int TM = 32 * X, TN = 128, Y = 4;
  int tm, tn;
  tile_of(blockIdx.x, tiles_m, tiles_n, 4, tm, tn);
  // (X = 8 has a whole tile at least; with X = 4 rows behind the last one are read as the last one and not stored)
  constexpr bool CLAMP = X == 4;
  const int i0 = CLAMP ? tm * TM : min(tm * TM, p.m - TM), j0 = CLAMP ? tn * TN : min(tn * TN, p.n - TN);
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), group = wave >> 2;
  const int wi = ((wave >> 1) & 1) * 16 * X, wj = (wave & 1) * 64;
  const int l16 = lane & 15, g = lane >> 4;
  const int nb = (p.k + 127) >> 7, all = p.k >> 7;
  const int b0 = blockIdx.y * p.blocks_per_part, full = min(all, b0 + p.blocks_per_part);   // blocks b0 .. full - 1, one at least
  const bool tail = nb > all && blockIdx.y == gridDim.y - 1;
  // piece r: rows 64 r + 8 wave + lane / 8 of A and then B
  const int r8 = lane >> 3, chunk = (DMA ? (lane & 7) ^ r8 : lane & 7) << 4;
  const uint32_t a_voff = (uint32_t) (8 * wave + r8) * (uint32_t) p.lda + chunk, b_voff = (uint32_t) (8 * wave + r8) * (uint32_t) p.ldb + chunk;
  uint32_t voff[CLAMP ? S::PIECES : 1];
#pragma unroll
  for (int r = 0; CLAMP && r < S::PIECES; r++)
    voff[r] = (r < X / 2 ? (uint32_t) min(64 * r + 8 * wave + r8, p.m - 1 - i0) * (uint32_t) p.lda
                         : (uint32_t) min(64 * (r - X / 2) + 8 * wave + r8, p.n - 1 - j0) * (uint32_t) p.ldb) + chunk;
  const uint64_t a_step = CLAMP ? 0 : (uint64_t) p.lda * 64, b_step = CLAMP ? 0 : (uint64_t) p.ldb * 64;
  const uint64_t a_org = reinterpret_cast<uint64_t>(p.a + (int64_t) i0 * p.lda), b_org = reinterpret_cast<uint64_t>(p.b + (int64_t) j0 * p.ldb);
  const uint32_t to = lds_address(lds) + wave * 1024;
  const int put = (8 * wave + r8) * 8 + ((lane & 7) ^ r8);
  u32x4 staged[DMA ? 1 : S::PIECES];
  auto fetch = [&](int blk, int slot) {   // a block (behind the last one: the last one again) on its way: DMA to LDS, or to registers
#pragma unroll
    for (int r = 0; r < S::PIECES; r++) {
      const bool a = r < X / 2;
      const uint64_t from = (a ? a_org + r * a_step : b_org + (r - X / 2) * b_step) + (uint64_t) min(blk, full - 1) * 128;
      const uint32_t off = CLAMP ? voff[CLAMP ? r : 0] : a ? a_voff : b_voff;
      if constexpr (DMA) dma16(off, from, to + slot * S::SLOT * 16 + r * 8192);
      else staged[r] = load16(from, off);
    }
  };
  auto land = [&](int slot) {             // ... and there (staged)
    if constexpr (!DMA) {
#pragma unroll
      for (int r = 0; r < S::PIECES; r++) lds[slot * S::SLOT + put + r * 512] = staged[r];
    }
  };
  // thread t has the scales of row t of A and then B
  uint8_t *const scales = (uint8_t *) (lds + S::S0);
  const uint8_t *const s_row = t < TM ? p.sa + (int64_t) (min(i0 + t, p.m - 1) >> p.a_shift) * p.ldsa
                                      : p.sb + (int64_t) (min(j0 + min(t - TM, TN - 1), p.n - 1) >> p.b_shift) * p.ldsb;
  auto put_half = [&](int seg, u32x4 v) { if (t < S::ROWS) put_scales(scales + (seg & 1) * S::ROWS * 20, t, v); };
  // this lane's chunk in an image, of tile 0: its half of the block
  const int a_at = (wi + l16) * 8 + ((4 * group + g) ^ (l16 & 7)), b_at = S::A_IMAGE + (wj + l16) * 8 + ((4 * group + g) ^ (l16 & 7));
  const uint8_t *const sa = scales + (wi + l16) * 20, *const sb = scales + (TM + wj + l16) * 20;
  auto byte_of = [](int kb) { return scale_byte(kb, S::ROWS); };
  f32x4 acc[X][Y];
#pragma unroll
  for (int x = 0; x < X * Y; x++) acc[x / Y][x % Y] = f32x4{0.f, 0.f, 0.f, 0.f};
  u32x4 ra[X], rb[Y];   // the block that is multiplied next, as it lies in memory
  bf16x8 b[Y][2];
  // one block out of registers; its successor is read from `next`
  auto multiply = [&](int next, int byte) {
    const u32x4 *const img = lds + next * S::SLOT;
#pragma unroll
    for (int y = 0; y < Y; y++) {
      const float sc = scale_value(sb[byte + y * 320]);
      b[y][0] = widen8<TB>((int) rb[y][0], (int) rb[y][1], sc);
      b[y][1] = widen8<TB>((int) rb[y][2], (int) rb[y][3], sc);
      rb[y] = img[b_at + y * 128];
    }
#pragma unroll
    for (int x = 0; x < X; x++) {
      const float sc = scale_value(sa[byte + x * 320]);
      const bf16x8 a0 = widen8<TA>((int) ra[x][0], (int) ra[x][1], sc), a1 = widen8<TA>((int) ra[x][2], (int) ra[x][3], sc);
      ra[x] = img[a_at + x * 128];
#pragma unroll
      for (int y = 0; y < Y; y++) acc[x][y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[y][0], a0, acc[x][y], 0, 0, 0);
#pragma unroll
      for (int y = 0; y < Y; y++) acc[x][y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[y][1], a1, acc[x][y], 0, 0, 0);
    }
  };
  auto read_first = [&](int slot) {
#pragma unroll
    for (int x = 0; x < X; x++) ra[x] = lds[slot * S::SLOT + a_at + x * 128];
#pragma unroll
    for (int y = 0; y < Y; y++) rb[y] = lds[slot * S::SLOT + b_at + y * 128];
    __syncthreads();
  };
  fetch(b0, 0); land(0);
  fetch(b0 + 1, 1); land(1);
  fetch(b0 + 2, 2);
  {
    const int seg = b0 >> 4;
    const u32x4 v0 = load_chunk(s_row, seg * 16, nb), v1 = load_chunk(s_row, seg * 16 + 16, nb);
    put_half(seg, v0);
    put_half(seg + 1, v1);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  read_first(0);
  int slot = 0;   // of block kb
  for (int kb = b0; kb < full; kb++) {
    if ((kb & 15) == 0 && kb > b0) put_half((kb >> 4) + 1, next_scales(s_row, kb + 16, nb));
    const int next = slot == 2 ? 0 : slot + 1;
    if constexpr (!DMA) land(next == 2 ? 0 : next + 1);   // (block kb + 2, fetched in the step before)
    fetch(kb + 3, slot);
    multiply(next, byte_of(kb));
    if constexpr (DMA) asm volatile("s_waitcnt vmcnt(%0)" :: "n"(S::PIECES) : "memory");   // block kb + 2 has landed
    __syncthreads();
    slot = next;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tail) {   // the short block: through registers, zeros behind k
    u32x4 v[S::PIECES];
#pragma unroll
    for (int u = 0; u < S::PIECES; u++) {
      const int r = 64 * u + 8 * wave + r8;
      v[u] = load_chunk_of_16(u < X / 2 ? p.a + (int64_t) min(i0 + r, p.m - 1) * p.lda : p.b + (int64_t) min(j0 + r - TM, p.n - 1) * p.ldb,
                              all * 128 + (lane & 7) * 16, p.k);
    }
    const uint8_t s_last = s_row[all];
#pragma unroll
    for (int u = 0; u < S::PIECES; u++) lds[put + u * 512] = v[u];
    if (t < S::ROWS) scales[t * 20] = s_last;
    __syncthreads();
    read_first(0);
    multiply(0, 0);
    __syncthreads();
  }
  // each group stores one half of the rows: it gets the other's sums for them
  f32x4 *const mine = (f32x4 *) lds + wave * (X / 2 * Y * 64), *const theirs = (f32x4 *) lds + (wave ^ 4) * (X / 2 * Y * 64);
  f32x4 sum[X / 2][Y];
#pragma unroll
  for (int x = 0; x < X / 2; x++)
#pragma unroll
    for (int y = 0; y < Y; y++) mine[(x * Y + y) * 64 + lane] = group ? acc[x][y] : acc[x + X / 2][y];
  __syncthreads();
#pragma unroll
  for (int x = 0; x < X / 2; x++)
#pragma unroll
    for (int y = 0; y < Y; y++) {
      const f32x4 v = theirs[(x * Y + y) * 64 + lane];
      sum[x][y] = group ? v + acc[x + X / 2][y] : acc[x][y] + v;
    }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  const int i = i0 + wi + group * X / 2 * 16;
  store_wave<X / 2, Y>(p, sum, theirs, i, j0 + wj, max(tm * TM, i), max(tn * TN, j0 + wj));
}

// ---- few rows of A -------------------------------------------------------------------
// Up to 16 rows of A, 32 of a wide product: the bytes of B bound it.  A workgroup owns 16 NT columns of C and all of k; its waves
// take the blocks of k in turn, so that every wave streams B straight into registers, four blocks in flight (and A, from the
// caches, two), and nobody waits for anybody until the waves' sums are added, in their order, through LDS.  1 x 4096 x 4096 in
// 5.9 us (2.8 TB/s, 2.5 us of it the launch), wide 32 x 4096 x 4096 in 11.9.
template <int TA, int TB, bool WIDE, int MT, int NT>
__global__ void __launch_bounds__(512) f8_rows_kernel(F8Product p) {
  extern __shared__ f32x4 sums[];   // [wave][tile][lane]
  constexpr int DEEP = 4;           // blocks of B in flight a wave
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), waves = blockDim.x >> 6;
  const int l16 = lane & 15, g = lane >> 4, j0 = blockIdx.x * 16 * NT;
  const int full = p.k >> 7;
  // (offsets of 32 bits from where the workgroup's rows begin: half the registers that pointers would take)
  const uint8_t *const b0 = p.b + (int64_t) j0 * p.ldb, *const sb0 = p.sb + (int64_t) (j0 >> p.b_shift) * p.ldsb;
  uint32_t a_off[MT], b_off[NT], sa_off[MT], sb_off[NT];
#pragma unroll
  for (int x = 0; x < MT; x++) {
    const int i = min(x * 16 + l16, p.m - 1);
    a_off[x] = (uint32_t) i * (uint32_t) p.lda + g * 16;
    sa_off[x] = (uint32_t) (i >> p.a_shift) * (uint32_t) p.ldsa;
  }
#pragma unroll
  for (int y = 0; y < NT; y++) {
    const int j = min(j0 + y * 16 + l16, p.n - 1);
    b_off[y] = (uint32_t) (j - j0) * (uint32_t) p.ldb + g * 16;
    sb_off[y] = (uint32_t) ((j >> p.b_shift) - (j0 >> p.b_shift)) * (uint32_t) p.ldsb;
  }
  f32x4 acc[MT][NT];
#pragma unroll
  for (int x = 0; x < MT * NT; x++) acc[x / NT][x % NT] = f32x4{0.f, 0.f, 0.f, 0.f};
  struct BlockA { u32x4 q[MT][2]; uint8_t s[MT]; };
  struct BlockB { u32x4 q[NT][2]; uint8_t s[NT]; };
  auto fetch_a = [&](BlockA &v, int blk) {
#pragma unroll
    for (int x = 0; x < MT; x++) {
      const uint8_t *from = p.a + (int64_t) blk * 128 + a_off[x];
      __builtin_memcpy(&v.q[x][0], from, 16);
      __builtin_memcpy(&v.q[x][1], from + 64, 16);
      v.s[x] = (p.sa + blk)[sa_off[x]];
    }
  };
  auto fetch_b = [&](BlockB &v, int blk) {
#pragma unroll
    for (int y = 0; y < NT; y++) {
      const uint8_t *from = b0 + (int64_t) blk * 128 + b_off[y];
      __builtin_memcpy(&v.q[y][0], from, 16);
      __builtin_memcpy(&v.q[y][1], from + 64, 16);
      v.s[y] = (sb0 + blk)[sb_off[y]];
    }
  };
  auto multiply = [&](const BlockA &a, const BlockB &b) {
    Frag<WIDE> fa[MT];
#pragma unroll
    for (int x = 0; x < MT; x++) fa[x] = make_frag<TA, WIDE>(a.q[x][0], a.q[x][1], a.s[x]);
#pragma unroll
    for (int y = 0; y < NT; y++) {
      const Frag<WIDE> fb = make_frag<TB, WIDE>(b.q[y][0], b.q[y][1], b.s[y]);
#pragma unroll
      for (int x = 0; x < MT; x++) acc[x][y] = mma<TA, TB, WIDE>(fb, fa[x], acc[x][y]);
    }
  };
  // (blocks behind the last one: the last one again, not multiplied)
  for (int blk = wave; blk < full; blk += DEEP * waves) {
    BlockB b[DEEP];
    BlockA a[2];
#pragma unroll
    for (int u = 0; u < DEEP; u++) fetch_b(b[u], min(blk + u * waves, full - 1));
    fetch_a(a[0], blk);
#pragma unroll
    for (int u = 0; u < DEEP; u++) {
      if (u + 1 < DEEP) fetch_a(a[(u + 1) & 1], min(blk + (u + 1) * waves, full - 1));
      __builtin_amdgcn_sched_barrier(0);
      if (blk + u * waves < full) multiply(a[u & 1], b[u]);
    }
  }
  if ((p.k & 127) && wave == full % waves) {   // the short block
    BlockA a;
    BlockB b;
#pragma unroll
    for (int x = 0; x < MT; x++) {
      a.q[x][0] = load_chunk(p.a + a_off[x] - g * 16, full * 128 + g * 16, p.k);
      a.q[x][1] = load_chunk(p.a + a_off[x] - g * 16, full * 128 + g * 16 + 64, p.k);
      a.s[x] = (p.sa + full)[sa_off[x]];
    }
#pragma unroll
    for (int y = 0; y < NT; y++) {
      b.q[y][0] = load_chunk(b0 + b_off[y] - g * 16, full * 128 + g * 16, p.k);
      b.q[y][1] = load_chunk(b0 + b_off[y] - g * 16, full * 128 + g * 16 + 64, p.k);
      b.s[y] = (sb0 + full)[sb_off[y]];
    }
    multiply(a, b);
  }
#pragma unroll
  for (int x = 0; x < MT * NT; x++) sums[(wave * MT * NT + x) * 64 + lane] = acc[x / NT][x % NT];
  __syncthreads();
  for (int at = t; at < MT * NT * 64; at += blockDim.x) {
    f32x4 v = sums[at];
    for (int w = 1; w < waves; w++) v += sums[w * MT * NT * 64 + at];
    const int x = (at >> 6) / NT, y = (at >> 6) % NT;
    const int i = x * 16 + l16, j = j0 + y * 16 + g * 4;
    if (i < p.m) {
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (j + e < p.n) finish(p, i, j + e, v[e]);
    }
  }
}

// C from the parts of the sums, added in their order (no parts: C = beta * C).  Bound by its launch, 2.6 us, and the parts' bytes.
__global__ void __launch_bounds__(256) f8_join_kernel(F8Product p, int parts) {
  const int64_t mn = (int64_t) p.m * p.n;
  if (p.n % 8 == 0) {   // eight neighbours a thread
    for (int64_t at = ((int64_t) blockIdx.x * 256 + threadIdx.x) * 8; at < mn; at += (int64_t) gridDim.x * 2048) {
      f32x4 lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
#pragma unroll 4
      for (int z = 0; z < parts; z++) {
        lo += *(const f32x4 *) (p.part + z * mn + at);
        hi += *(const f32x4 *) (p.part + z * mn + at + 4);
      }
      const int64_t c = at / p.n * p.ldc + at % p.n;
      if (p.c_type == BOF_BF16) finish_eight<BOF_BF16>(p, c, lo, hi);
      else if (p.c_type == BOF_F16) finish_eight<BOF_F16>(p, c, lo, hi);
      else finish_eight<BOF_F32>(p, c, lo, hi);
    }
    return;
  }
  for (int64_t at = (int64_t) blockIdx.x * 256 + threadIdx.x; at < mn; at += (int64_t) gridDim.x * 256) {
    float sum = 0.f;
    for (int z = 0; z < parts; z++) sum += p.part[z * mn + at];
    finish(p, at / p.n, at % p.n, sum);
  }
}

// ---- which kernel --------------------------------------------------------------------
enum Kind { kAny, kRows, kRing64, kRing128, kTwo128, kRing160, kRing256, kTile256, kWide128, kWide256 };
struct Plan {
  Kind kind;
  int parts;   // along k
};
constexpr int kMaxParts = 32;

// The kernel, and the parts along k, of least time by this estimate, in us: 1, and for every round of workgroups what it takes to
// begin and to store, and what a block of k takes; a round is one workgroup a CU, or two where two numbers stand (the second
// is for two).  For parts a join of 2.3 us and 4 TB/s for what they write and it reads.  The constants are fitted to every kernel's
// times over k from 256 to 16384, one round and several: of 171 other outputs (17 to 8192 rows, 128 to 16384 columns, k up to 28672) the
// kernel that it names takes 1.3 % longer than the fastest of them on average, and more than 6 % longer for 15.  Measured, the
// kernel named against its neighbours:
//                 round      block
//   64 x 32       2.9, 3.1   0.15, 0.35   512 x 2048 x 1024 6.8 us, 256 x 2048 x 4096 8.8 (128 x 128: 8.7, and 13.8 in four parts)
//   128 x 128     6.1        0.47         2048 x 2048 x 1024 11.2 us, x 4096 21.7, 1024 x 4096 x 14336 58 (128 x 160: 15.6, 24.8, 64)
//     two a CU    5.0, 6.6   0.71, 0.93   8192 x 8192 x 256 62 us (256 x 256: 66), 4096 x 2048 x 1024 16.3 (256 x 128: 18.2); only by DMA
//   128 x 160     9.9        0.53         2048 x 2560 x 1024 15.0 us, x 4096 26.0, x 14336 67 (128 x 128: 18.6, 35, 96)
//   256 x 128     10.4       0.70         4096 x 2048 x 4096 35 us, x 14336 108 (128 x 128: 42, 135); only by DMA: staged it spills
//   256 x 256     14.9       1.24         4096 x 4096 x 1024 27 us, x 4096 58, x 14336 170 (two of 128 x 128: 30, 69, 239)
//   wide          4.3        0.96 (128 x 128), 6.0, 1.73 (256 x 128)   2048 x 2048 x 4096 41 us (256 x 128: 58), 4096 x 4096 x 4096 134 (154)
// One to sixteen rows of A and a workgroup a CU at most go to the kernel for few rows: 1 x 4096 x 4096 in 5.9 us, in 7.5 by tiles
// of 64 x 32; 8 x 4096 x 8192 in 10.8 and 11.1; 1 x 8192 x 4096 in 8.8 and 8.4, 1 x 512 x 16384 in 11.9 and 9.0.  Wide: all up to
// 32 rows, 32 x 4096 x 4096 in 12.0 us (33 rows by tiles: 15.6).
Plan plan_product(int64_t m, int64_t n, int64_t k, bool wide, bool near, bool dma, int max_parts) {
  if (m <= 16 && n <= 4096 && k <= 8192 && near) return {kRows, 1};
  if (wide && m <= 32 && n <= (1 << 26) && near) return {kRows, 1};
  if (k < 128 || !near) return {kAny, 1};
  const int64_t nb = k / 128;
  Plan best{kAny, 1};
  double least = 1e30;
  struct Cost { double round, block; };
  auto consider = [&](Kind kind, int tm, int tn, Cost one, Cost two) {   // two.round 0: a CU holds one workgroup
    const int64_t tiles = ((m + tm - 1) / tm) * ((n + tn - 1) / tn);
    if (tiles >= (1 << 23)) return;   // (512 threads each: a launch holds less than 2^32)
    const int64_t full = two.round > 0 ? 512 : 256;
    for (int64_t parts = 1; parts <= max_parts && (parts == 1 || (parts * tiles <= full && parts * 8 <= nb + 7)); parts++) {
      const int64_t all = tiles * parts, rest = all % full;
      const double blocks = (double) ((nb + parts - 1) / parts);
      auto round = [&](Cost c) { return c.round + blocks * c.block; };
      const double us = 1 + (double) (all / full) * round(full == 512 ? two : one) + (rest == 0 ? 0 : rest <= 256 ? round(one) : round(two)) +
                        (parts > 1 ? 2.3 + (double) parts * (double) m * (double) n * 8 / 4e6 : 0);
      if (us < least) { least = us; best = {kind, (int) parts}; }
    }
  };
  if (wide) {
    consider(kWide128, 128, 128, {4.3, 0.96}, {0, 0});
    if (m >= 256 && n >= 128) consider(kWide256, 256, 128, {6, 1.73}, {0, 0});
  } else {
    consider(kRing64, 64, 32, {2.9, 0.15}, {3.1, 0.35});
    consider(kRing128, 128, 128, {6.1, 0.47}, {0, 0});
    consider(kRing160, 128, 160, {9.9, 0.53}, {0, 0});
    if (dma) {
      consider(kTwo128, 128, 128, {5, 0.71}, {6.6, 0.93});
      consider(kRing256, 256, 128, {10.4, 0.7}, {0, 0});
    }
    if (m >= 256 && n >= 256) max_parts = 1, consider(kTile256, 256, 256, {14.9, 1.24}, {0, 0});
  }
  return best;
}

// what the DMA to LDS needs of a row: 16-byte chunks at multiples of four bytes (at no loss: reads from the L2 run at 20 TB/s at any
// such address, at 10 at odd ones)
bool rows_aligned(const void *a, int64_t lda, const void *b, int64_t ldb) {
  return lda % 4 == 0 && ldb % 4 == 0 && reinterpret_cast<uintptr_t>(a) % 4 == 0 && reinterpret_cast<uintptr_t>(b) % 4 == 0;
}

template <int TA, int TB>
void start_tiles(const F8Product &p, hipStream_t st) {
  const int tiles_m = (p.m + 255) / 256, tiles_n = (p.n + 255) / 256;
  if (rows_aligned(p.a, p.lda, p.b, p.ldb)) f8_tile_kernel<TA, TB, 8, 8, true><<<(unsigned) (tiles_m * tiles_n), 256, 0, st>>>(p, tiles_m, tiles_n);
  else f8_tile_kernel<TA, TB, 8, 8, false><<<(unsigned) (tiles_m * tiles_n), 256, 0, st>>>(p, tiles_m, tiles_n);
}
template <int TA, int TB, int X, int Y, int WM, int ST, bool ANY = true>   // (ANY: also for rows that the DMA does not take)
void start_ring(const F8Product &p, int parts, hipStream_t st) {
  using S = Ring<X, Y, WM, ST, true>;
  const int tiles_m = (p.m + S::TM - 1) / S::TM, tiles_n = (p.n + S::TN - 1) / S::TN;
  const dim3 grid((unsigned) (tiles_m * tiles_n), (unsigned) parts);
  if (!ANY || rows_aligned(p.a, p.lda, p.b, p.ldb)) f8_ring_kernel<TA, TB, X, Y, WM, ST, true><<<grid, 256, 0, st>>>(p, tiles_m, tiles_n);
  else if constexpr (ANY) f8_ring_kernel<TA, TB, X, Y, WM, ST, false><<<grid, 256, 0, st>>>(p, tiles_m, tiles_n);
}

template <int TA, int TB, int X>
void start_wide(const F8Product &p, int parts, hipStream_t st) {
  const int tiles_m = (p.m + 32 * X - 1) / (32 * X), tiles_n = (p.n + 127) / 128;
  const dim3 grid((unsigned) (tiles_m * tiles_n), (unsigned) parts);
  if (rows_aligned(p.a, p.lda, p.b, p.ldb)) f8_wide_kernel<TA, TB, X, true><<<grid, 512, 0, st>>>(p, tiles_m, tiles_n);
  else f8_wide_kernel<TA, TB, X, false><<<grid, 512, 0, st>>>(p, tiles_m, tiles_n);
}

template <int TA, int TB, bool WIDE, int MT, int NT>
void start_rows(const F8Product &p, hipStream_t st) {
  const int waves = 8;
  const unsigned wg = (unsigned) ((p.n + 16 * NT - 1) / (16 * NT)), bytes = waves * MT * NT * 1024;
  f8_rows_kernel<TA, TB, WIDE, MT, NT><<<wg, 64 * waves, bytes, st>>>(p);
}

// the plan for a call's arguments; work_bytes: of the workspace, 0 without one
Plan plan_call(int64_t m, int64_t n, int64_t k, const void *a, int64_t lda, int64_t ldsa, const void *b, int64_t ldb, int64_t ldsb, int c_type, uint64_t work_bytes) {
  const uint64_t room = work_bytes / ((uint64_t) m * (uint64_t) n * 4u);
  const bool near = lda <= (1 << 24) && ldb <= (1 << 24) && ldsa <= (1 << 24) && ldsb <= (1 << 24);   // a tile of 256 rows: offsets of 32 bits
  return plan_product(m, n, k, c_type == BOF_F32, near, rows_aligned(a, lda, b, ldb), room < 2 ? 1 : room < kMaxParts ? (int) room : kMaxParts);
}
// parts of whole blocks, as even as they come: blocks in one, and how many there are (the short block is the last one's)
int whole_parts(int64_t k, int parts, int &blocks) {
  const int all = k / 128 ? (int) (k / 128) : 1;
  blocks = (all + parts - 1) / parts;
  return (all + blocks - 1) / blocks;
}

template <int TA, int TB>
hipError_t launch_product(F8Product p, Plan plan, hipStream_t st) {
  const int parts = whole_parts(p.k, plan.parts, p.blocks_per_part);
  if (parts == 1) p.part = nullptr;
  drop_stale_error();
  switch (plan.kind) {
    case kAny: {
      const unsigned tiles = (unsigned) (((p.m + 127) / 128) * (int64_t) ((p.n + 127) / 128));
      if (p.c_type == BOF_F32) f8_tile_any_kernel<TA, TB, true><<<tiles, 256, 0, st>>>(p);
      else f8_tile_any_kernel<TA, TB, false><<<tiles, 256, 0, st>>>(p);
      break;
    }
    case kRows:
      if (p.c_type != BOF_F32) start_rows<TA, TB, false, 1, 1>(p, st);
      else if (p.m <= 16) start_rows<TA, TB, true, 1, 1>(p, st);
      else start_rows<TA, TB, true, 2, 2>(p, st);
      break;
    case kRing64: start_ring<TA, TB, 2, 1, 2, 6>(p, parts, st); break;
    case kRing128: start_ring<TA, TB, 4, 4, 2, 4>(p, parts, st); break;
    case kTwo128: start_ring<TA, TB, 4, 4, 2, 2, false>(p, parts, st); break;
    case kRing256: start_ring<TA, TB, 8, 4, 2, 3, false>(p, parts, st); break;
    case kRing160: start_ring<TA, TB, 4, 5, 2, 4>(p, parts, st); break;
    case kTile256: start_tiles<TA, TB>(p, st); break;
    case kWide128: start_wide<TA, TB, 4>(p, parts, st); break;
    case kWide256: start_wide<TA, TB, 8>(p, parts, st); break;
  }
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
  int parts = plan_product(m, n, k, true, true, true, kMaxParts).parts;
  for (bool dma : {false, true}) parts = std::max(parts, plan_product(m, n, k, false, true, dma, kMaxParts).parts);
  return parts > 1 ? (uint64_t) parts * (uint64_t) m * (uint64_t) n * 4u : 0;
}

int bof_f8_gemm_plan(int64_t m, int64_t n, int64_t k, const void *a, int64_t lda, int64_t ldsa, const void *b, int64_t ldb, int64_t ldsb, int c_type,
                     uint64_t work_bytes, int *parts) {
  if (m <= 0 || n <= 0 || k <= 0 || m > INT32_MAX - 255 || n > INT32_MAX - 255 || k > INT32_MAX - 255 || c_type < BOF_F32 || c_type > BOF_F16 || !parts)
    return refuse("bof_f8_gemm_plan", "bad size or type, or parts is missing");
  const Plan plan = plan_call(m, n, k, a, lda, ldsa, b, ldb, ldsb, c_type, work_bytes);
  int blocks;
  *parts = whole_parts(k, plan.parts, blocks);
  return plan.kind;
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
  p.alpha = product ? alpha : 0.f; p.beta = beta;   // (no product: beta * C whatever alpha is)
  p.c = c; p.c_type = c_type;
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
  const Plan plan = plan_call(m, n, k, a, lda, ldsa, b, ldb, ldsb, c_type, work ? work_bytes : 0);
  if (plan.parts > 1)
    if (int rc = dev.reaches(work, kCall, "work")) return rc;
  p.a = (const uint8_t *) a; p.b = (const uint8_t *) b; p.sa = sa; p.sb = sb;
  p.lda = lda; p.ldb = ldb; p.ldsa = ldsa; p.ldsb = ldsb;
  p.a_shift = ga == 128 ? 7 : 0; p.b_shift = gb == 128 ? 7 : 0;
  p.part = (float *) work;
  hipError_t e;
  if (a_type == BOF_E4M3) e = b_type == BOF_E4M3 ? launch_product<BOF_E4M3, BOF_E4M3>(p, plan, (hipStream_t) stream) : launch_product<BOF_E4M3, BOF_E5M2>(p, plan, (hipStream_t) stream);
  else e = b_type == BOF_E4M3 ? launch_product<BOF_E5M2, BOF_E4M3>(p, plan, (hipStream_t) stream) : launch_product<BOF_E5M2, BOF_E5M2>(p, plan, (hipStream_t) stream);
  BOF_HIP_TRY(e);
  return BOF_OK;
}

}  // extern "C"
