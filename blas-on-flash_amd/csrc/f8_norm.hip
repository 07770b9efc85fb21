// f8_norm.hip -- the quantiser of matrices into 8 bits with power-of-two block scales, and the root-mean-square norm
// with its gradient (bof_f8.h).  All of it is bound by memory: each array is to be read or written once.
#include "f8_common.h"

namespace bof {

namespace {

// ---- quantiser ----------------------------------------------------------------------
struct Quant {
  const void *x;
  int64_t ldx, rows, cols;
  uint8_t *q, *s, *qt, *st;
  int64_t ldq, lds, ldqt, ldst;
};

// One workgroup, one 128 x 128 block of X through LDS.  A thread pair owns a row (64 elements each), and in the second
// half a column.
template <int X, int F8, int GROUP>
__global__ void __launch_bounds__(256) quant_tile_kernel(Quant p) {
  __shared__ float tile[128][129];
  __shared__ uint32_t top[256];
  const int t = threadIdx.x;
  const int64_t tiles_c = (p.cols + 127) >> 7;
  const int64_t bi = blockIdx.x / tiles_c, bj = blockIdx.x % tiles_c;
  const int64_t r0 = bi * 128, c0 = bj * 128;
  const int nr = (int) min((int64_t) 128, p.rows - r0), nc = (int) min((int64_t) 128, p.cols - c0);
  for (int at = t; at < 128 * 128; at += 256) {
    const int r = at >> 7, c = at & 127;
    tile[r][c] = r < nr && c < nc ? load_dense<X>(p.x, (r0 + r) * p.ldx + c0 + c) : 0.f;
  }
  __syncthreads();
  const int line = t >> 1, h = (t & 1) * 64;
  uint32_t whole = 0;
  if (GROUP == 128) {
    uint32_t m = 0;
    for (int e = 0; e < 64; e++) m = max(m, finite_magnitude(tile[line][h + e]));
    top[t] = m;
    __syncthreads();
    for (int e = 0; e < 256; e++) whole = max(whole, top[e]);
    __syncthreads();
  }
  for (int pass = 0; pass < 2; pass++) {   // 0: rows of X, 1: its columns
    uint8_t *q = pass ? p.qt : p.q, *s = pass ? p.st : p.s;
    if (!q) continue;
    const int64_t ld = pass ? p.ldqt : p.ldq, lds = pass ? p.ldst : p.lds;
    const int64_t line0 = pass ? c0 : r0, along0 = pass ? r0 : c0, block = pass ? bi : bj;
    const int lines = pass ? nc : nr, along = pass ? nr : nc;
    uint32_t m = whole;
    if (GROUP == 1) {
      m = 0;
      for (int e = 0; e < 64; e++) m = max(m, finite_magnitude(pass ? tile[h + e][line] : tile[line][h + e]));
      m = max(m, (uint32_t) __shfl_xor((int) m, 1));
    }
    const uint32_t code = scale_code<F8>(m);
    const float inv = scale_inverse(code);
    if (line < lines) {
      if (h == 0 && (GROUP == 1 || line == 0)) s[(line0 + line) / GROUP * lds + block] = (uint8_t) code;
      for (int e = 0; e < 64 && h + e < along; e++) {
        const float v = pass ? tile[h + e][line] : tile[line][h + e];
        q[(line0 + line) * ld + along0 + h + e] = (uint8_t) f8_pair<F8, false>(v * inv, 0.f, 0u);
      }
    }
  }
}

template <int X, int F8>
hipError_t launch_quant(const Quant &p, int group, hipStream_t st) {
  const unsigned tiles = (unsigned) (((p.rows + 127) >> 7) * ((p.cols + 127) >> 7));
  drop_stale_error();
  if (group == 1) quant_tile_kernel<X, F8, 1><<<tiles, 256, 0, st>>>(p);
  else quant_tile_kernel<X, F8, 128><<<tiles, 256, 0, st>>>(p);
  return hipGetLastError();
}

// ---- norm ---------------------------------------------------------------------------
struct Norm {
  const void *x, *r, *w;
  int64_t ldx, ldr, ldh, ldq, lds, ldy, n;
  float eps;
  void *h, *y;
  uint8_t *q, *s;
  float *rstd;
};

// sum over the workgroup's 256 threads, in a fixed order, for all of them
__device__ __forceinline__ float group_sum(float v, float *part) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = (part[0] + part[1]) + (part[2] + part[3]);
  __syncthreads();
  return v;
}

// One workgroup a row, which is read twice.
template <int T, int F8>
__global__ void __launch_bounds__(256) norm_row_kernel(Norm p) {
  __shared__ float part[4];
  const int64_t row = blockIdx.x;
  const int t = threadIdx.x;
  float sq = 0.f;
  for (int64_t c = t; c < p.n; c += 256) {
    float v = load_dense<T>(p.x, row * p.ldx + c);
    if (p.r) v += load_dense<T>(p.r, row * p.ldr + c);
    sq = fmaf(v, v, sq);
  }
  const float rstd = 1.f / sqrtf(group_sum(sq, part) / (float) p.n + p.eps);
  if (t == 0 && p.rstd) p.rstd[row] = rstd;
  for (int64_t c0 = 0; c0 < p.n; c0 += 512) {   // a wave: one block of 128, two neighbours a lane
    const int64_t c = c0 + 2 * t;
    float y[2] = {0.f, 0.f};
    uint32_t m = 0;
    for (int e = 0; e < 2; e++)
      if (c + e < p.n) {
        float v = load_dense<T>(p.x, row * p.ldx + c + e);
        if (p.r) v += load_dense<T>(p.r, row * p.ldr + c + e);
        if (p.h) store_dense<T>(p.h, row * p.ldh + c + e, v);
        y[e] = v * rstd * load_dense<T>(p.w, c + e);
        if (p.y) store_dense<T>(p.y, row * p.ldy + c + e, y[e]);
        m = max(m, finite_magnitude(y[e]));
      }
    if (!p.q) continue;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) m = max(m, (uint32_t) __shfl_xor((int) m, d));
    const uint32_t code = scale_code<F8>(m), two = f8_pair<F8, false>(y[0] * scale_inverse(code), y[1] * scale_inverse(code), 0u);
    for (int e = 0; e < 2; e++)
      if (c + e < p.n) p.q[row * p.ldq + c + e] = (uint8_t) (two >> (8 * e));
    if ((t & 63) == 0 && c < p.n) p.s[row * p.lds + (c >> 7)] = (uint8_t) code;
  }
}

// ---- gradient of the norm -----------------------------------------------------------
struct NormGrad {
  const void *dy, *h, *w, *dh;
  const float *rstd;
  void *dx;
  int64_t lddy, ldh, lddh, lddx, rows, n;
  float *part, *dw;   // part: gridDim.x rows of n
  float beta;
};

// Workgroup g of G takes rows g, g + G, ...: dx row by row, and the sums over its rows into part[g].
template <int T>
__global__ void __launch_bounds__(256) norm_grad_kernel(NormGrad p) {
  __shared__ float red[4];
  float *part = p.part ? p.part + (int64_t) blockIdx.x * p.n : nullptr;
  const int t = threadIdx.x;
  bool first = true;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const float rstd = p.rstd[row];
    float dot = 0.f;
    for (int64_t c = t; c < p.n; c += 256)
      dot = fmaf(load_dense<T>(p.dy, row * p.lddy + c) * load_dense<T>(p.w, c), load_dense<T>(p.h, row * p.ldh + c) * rstd, dot);
    const float mean = group_sum(dot, red) / (float) p.n;
    for (int64_t c = t; c < p.n; c += 256) {
      const float dy = load_dense<T>(p.dy, row * p.lddy + c), xhat = load_dense<T>(p.h, row * p.ldh + c) * rstd;
      float v = rstd * (dy * load_dense<T>(p.w, c) - xhat * mean);
      if (p.dh) v += load_dense<T>(p.dh, row * p.lddh + c);
      store_dense<T>(p.dx, row * p.lddx + c, v);
      if (part) part[c] = first ? dy * xhat : part[c] + dy * xhat;
    }
    first = false;
  }
}

// dw = beta * dw + the partial sums, in their order
__global__ void __launch_bounds__(256) norm_grad_join_kernel(const float *part, int parts, int64_t n, float beta, float *dw) {
  const int64_t c = (int64_t) blockIdx.x * 256 + threadIdx.x;
  if (c >= n) return;
  float sum = 0.f;
  for (int g = 0; g < parts; g++) sum += part[g * n + c];
  dw[c] = beta == 0.f ? sum : fmaf(beta, dw[c], sum);
}

constexpr int64_t kGradGroups = 256;

template <int T>
hipError_t launch_norm(const Norm &p, int64_t rows, int f8_type, hipStream_t st) {
  drop_stale_error();
  if (f8_type == BOF_E5M2) norm_row_kernel<T, BOF_E5M2><<<(unsigned) rows, 256, 0, st>>>(p);
  else norm_row_kernel<T, BOF_E4M3><<<(unsigned) rows, 256, 0, st>>>(p);
  return hipGetLastError();
}

template <int T>
hipError_t launch_norm_grad(const NormGrad &p, hipStream_t st) {
  const int64_t groups = p.rows < kGradGroups ? p.rows : kGradGroups;
  drop_stale_error();
  norm_grad_kernel<T><<<(unsigned) groups, 256, 0, st>>>(p);
  if (p.dw) norm_grad_join_kernel<<<(unsigned) ((p.n + 255) / 256), 256, 0, st>>>(p.part, (int) groups, p.n, p.beta, p.dw);
  return hipGetLastError();
}

bool dense_type(int t) { return t == BOF_F32 || t == BOF_BF16 || t == BOF_F16; }
bool aligned_to(const void *p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

}  // namespace

}  // namespace bof

using namespace bof;

extern "C" {

int bof_f8_quant(int64_t rows, int64_t cols, const void *x, int64_t ldx, int x_type, int f8_type, int group, void *q,
                 int64_t ldq, uint8_t *s, int64_t lds, void *qt, int64_t ldqt, uint8_t *st, int64_t ldst, void *stream) {
  static const char kCall[] = "bof_f8_quant";
  if (rows < 0 || cols < 0 || rows > INT32_MAX - 255 || cols > INT32_MAX - 255) return refuse(kCall, "bad size");
  if (!dense_type(x_type)) return refuse(kCall, "X is of BOF_F32, BOF_BF16 or BOF_F16");
  if (f8_type != BOF_E4M3 && f8_type != BOF_E5M2) return refuse(kCall, "the outputs are of BOF_E4M3 or BOF_E5M2");
  if (group != 1 && group != 128) return refuse(kCall, "1 or 128 rows share a scale");
  if (!q != !s || !qt != !st || (!q && !qt)) return refuse(kCall, "an output is missing");
  if (rows == 0 || cols == 0) return BOF_OK;
  if (!x || ldx < cols || !aligned_to(x, dense_bytes(x_type))) return refuse(kCall, "X is missing, its rows overlap or it is not aligned to its type");
  if ((q && (ldq < cols || lds < (cols + 127) / 128)) || (qt && (ldqt < rows || ldst < (rows + 127) / 128)))
    return refuse(kCall, "rows of an output overlap");
  if (((rows + 127) >> 7) * ((cols + 127) >> 7) >= (1 << 24)) return refuse(kCall, "bad size");
  LaunchDevice dev((hipStream_t) stream);
  if (dev.status()) return dev.status();
  for (auto [p, name] : {std::pair<const void *, const char *>{x, "X"}, {q, "q"}, {s, "s"}, {qt, "qt"}, {st, "st"}})
    if (int rc = p ? dev.reaches(p, kCall, name) : 0) return rc;
  Quant p{x, ldx, rows, cols, (uint8_t *) q, s, (uint8_t *) qt, st, ldq, lds, ldqt, ldst};
  hipStream_t hs = (hipStream_t) stream;
  hipError_t e;
  if (f8_type == BOF_E4M3)
    e = x_type == BOF_F32 ? launch_quant<BOF_F32, BOF_E4M3>(p, group, hs) : x_type == BOF_BF16 ? launch_quant<BOF_BF16, BOF_E4M3>(p, group, hs) : launch_quant<BOF_F16, BOF_E4M3>(p, group, hs);
  else
    e = x_type == BOF_F32 ? launch_quant<BOF_F32, BOF_E5M2>(p, group, hs) : x_type == BOF_BF16 ? launch_quant<BOF_BF16, BOF_E5M2>(p, group, hs) : launch_quant<BOF_F16, BOF_E5M2>(p, group, hs);
  BOF_HIP_TRY(e);
  return BOF_OK;
}

int bof_rmsnorm_f8(int64_t rows, int64_t n, int type, const void *x, int64_t ldx, const void *r, int64_t ldr, const void *w,
                   float eps, void *h, int64_t ldh, int f8_type, void *q, int64_t ldq, uint8_t *s, int64_t lds, void *y,
                   int64_t ldy, float *rstd, void *stream) {
  static const char kCall[] = "bof_rmsnorm_f8";
  if (rows < 0 || n < 0 || rows > (1 << 24) - 1 || n > INT32_MAX - 255) return refuse(kCall, "bad size (at most 2^24 - 1 rows)");
  if (!dense_type(type)) return refuse(kCall, "X is of BOF_F32, BOF_BF16 or BOF_F16");
  if (q && f8_type != BOF_E4M3 && f8_type != BOF_E5M2) return refuse(kCall, "q is of BOF_E4M3 or BOF_E5M2");
  if (!q != !s) return refuse(kCall, "q and s come together");
  if (!h && !q && !y && !rstd) return refuse(kCall, "no output");
  if (h && ((h == x && ldh != ldx) || (h == r && ldh != ldr))) return refuse(kCall, "h lies over an input with other rows");
  if (!(eps >= 0.f)) return refuse(kCall, "eps is negative");
  if (rows == 0 || n == 0) return BOF_OK;
  const size_t z = dense_bytes(type);
  if (!x || !w) return refuse(kCall, "X or w is missing");
  if (ldx < n || (r && ldr < n) || (h && ldh < n) || (q && (ldq < n || lds < (n + 127) / 128)) || (y && ldy < n)) return refuse(kCall, "rows of an array overlap");
  if (!aligned_to(x, z) || !aligned_to(r, z) || !aligned_to(w, z) || !aligned_to(h, z) || !aligned_to(y, z) || !aligned_to(rstd, 4)) return refuse(kCall, "an array is not aligned to its type");
  LaunchDevice dev((hipStream_t) stream);
  if (dev.status()) return dev.status();
  for (auto [p, name] : {std::pair<const void *, const char *>{x, "X"}, {r, "R"}, {w, "w"}, {h, "h"}, {q, "q"}, {s, "s"}, {y, "y"}, {rstd, "rstd"}})
    if (int rc = p ? dev.reaches(p, kCall, name) : 0) return rc;
  Norm p{x, r, w, ldx, ldr, ldh, ldq, lds, ldy, n, eps, h, y, (uint8_t *) q, s, rstd};
  hipStream_t hs = (hipStream_t) stream;
  BOF_HIP_TRY(type == BOF_F32 ? launch_norm<BOF_F32>(p, rows, f8_type, hs) : type == BOF_BF16 ? launch_norm<BOF_BF16>(p, rows, f8_type, hs) : launch_norm<BOF_F16>(p, rows, f8_type, hs));
  return BOF_OK;
}

uint64_t bof_rmsnorm_grad_workspace_bytes(int64_t rows, int64_t n) {
  if (rows <= 0 || n <= 0 || rows > (1 << 24) - 1 || n > INT32_MAX - 255) return 0;
  return (uint64_t) (rows < kGradGroups ? rows : kGradGroups) * (uint64_t) n * 4u;
}

int bof_rmsnorm_grad(int64_t rows, int64_t n, int type, const void *dy, int64_t lddy, const void *h, int64_t ldh, const void *w,
                     const float *rstd, const void *dh, int64_t lddh, void *dx, int64_t lddx, float beta, float *dw, void *work,
                     uint64_t work_bytes, void *stream) {
  static const char kCall[] = "bof_rmsnorm_grad";
  if (rows < 0 || n < 0 || rows > (1 << 24) - 1 || n > INT32_MAX - 255) return refuse(kCall, "bad size (at most 2^24 - 1 rows)");
  if (!dense_type(type)) return refuse(kCall, "dy is of BOF_F32, BOF_BF16 or BOF_F16");
  if (n == 0) return BOF_OK;
  const size_t z = dense_bytes(type);
  if (!aligned_to(dw, 4)) return refuse(kCall, "an array is not aligned to its type");
  if (rows > 0) {
    if (!dy || !h || !w || !rstd || !dx) return refuse(kCall, "an array is missing");
    if (lddy < n || ldh < n || (dh && lddh < n) || lddx < n) return refuse(kCall, "rows of an array overlap");
    if (!aligned_to(dy, z) || !aligned_to(h, z) || !aligned_to(w, z) || !aligned_to(dh, z) || !aligned_to(dx, z) || !aligned_to(rstd, 4)) return refuse(kCall, "an array is not aligned to its type");
    if ((dx == dy && lddx != lddy) || (dx == dh && lddx != lddh) || dx == h) return refuse(kCall, "dx lies over an input with other rows, or over h");
    if (dw && (!work || reinterpret_cast<uintptr_t>(work) % 16 || work_bytes < bof_rmsnorm_grad_workspace_bytes(rows, n)))
      return refuse(kCall, "work is missing, not aligned to 16 bytes or smaller than bof_rmsnorm_grad_workspace_bytes says");
  } else if (!dw || beta == 1.f) {
    return BOF_OK;
  }
  LaunchDevice dev((hipStream_t) stream);
  if (dev.status()) return dev.status();
  hipStream_t hs = (hipStream_t) stream;
  if (int rc = dw ? dev.reaches(dw, kCall, "dw") : 0) return rc;
  if (rows == 0) {   // no rows: dw = beta * dw
    drop_stale_error();
    norm_grad_join_kernel<<<(unsigned) ((n + 255) / 256), 256, 0, hs>>>(nullptr, 0, n, beta, dw);
    BOF_HIP_TRY(hipGetLastError());
    return BOF_OK;
  }
  for (auto [p, name] : {std::pair<const void *, const char *>{dy, "dy"}, {h, "h"}, {w, "w"}, {rstd, "rstd"}, {dh, "dh"}, {dx, "dx"}, {dw ? work : nullptr, "work"}})
    if (int rc = p ? dev.reaches(p, kCall, name) : 0) return rc;
  NormGrad p{dy, h, w, dh, rstd, dx, lddy, ldh, lddh, lddx, rows, n, dw ? (float *) work : nullptr, dw, beta};
  BOF_HIP_TRY(type == BOF_F32 ? launch_norm_grad<BOF_F32>(p, hs) : type == BOF_BF16 ? launch_norm_grad<BOF_BF16>(p, hs) : launch_norm_grad<BOF_F16>(p, hs));
  return BOF_OK;
}

}  // extern "C"
