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
