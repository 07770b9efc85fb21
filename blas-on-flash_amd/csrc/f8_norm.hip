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
  int top;
};

// One workgroup, one 128 x 128 block of X, which is read once and stays in registers: thread t holds an 8 x 8 block, columns
// 8 * (t & 15), rows 8 * (t >> 4).  The largest magnitude of a row of the block is then that of 16 neighbouring lanes, that
// of a column is joined through LDS.  Transposed elements pass through LDS: a thread's eight rows of a column are eight
// neighbouring bytes there, a unit; column c keeps its 16 units XOR-ed with c / 8, so that neither the writes (16 lanes,
// 16 columns) nor the reads meet a bank twice.
//
// q = X / s with s = 2^e the smallest that brings the block's largest finite magnitude into range: the quotient is exact (s is a
// power of two, and q's type rounds it once) unless it falls below fp32's normal numbers.  Bound by bytes: both layouts of
// 4096 x 4096 fp32 in 21 us (4.8 TB/s), of 16384 x 4096 bf16 in 60 us (4.5 TB/s; a large copy: 4.9); with the
// block as floats in LDS and a pair of threads to a row and then a column it took 212 and 827 us.
template <int X, int GROUP, bool T>
__global__ void __launch_bounds__(256) quant_kernel(Quant p) {
  __shared__ uint64_t turned[T ? 128 * 16 : 1];
  __shared__ uint32_t top[4][128];
  const int t = threadIdx.x, c8 = (t & 15) * 8, r8 = (t >> 4) * 8;
  const int64_t tiles_c = (p.cols + 127) >> 7, bi = blockIdx.x / tiles_c, bj = blockIdx.x % tiles_c;
  const int64_t r0 = bi * 128, c0 = bj * 128;
  const int nr = (int) min((int64_t) 128, p.rows - r0), nc = (int) min((int64_t) 128, p.cols - c0);
  Eight<X> x[8];
#pragma unroll
  for (int u = 0; u < 8; u++) x[u] = load_eight<X>(p.x, (r0 + r8 + u) * p.ldx + c0 + c8, r8 + u < nr ? nc - c8 : 0);
  uint32_t row_top[8], col_top[8] = {};
#pragma unroll
  for (int u = 0; u < 8; u++) {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const uint32_t v = finite_magnitude(x[u].at(e));
      m = max(m, v);
      if (T && GROUP == 1) col_top[e] = max(col_top[e], v);
    }
    row_top[u] = max_of_16(m);
  }
  if (GROUP == 128) {   // one scale for all of it
    uint32_t m = row_top[0];
#pragma unroll
    for (int u = 1; u < 8; u++) m = max(m, row_top[u]);
    m = max(m, (uint32_t) __shfl_xor((int) m, 16));
    m = max(m, (uint32_t) __shfl_xor((int) m, 32));
    if ((t & 63) == 0) top[t >> 6][0] = m;
    __syncthreads();
    m = max(max(top[0][0], top[1][0]), max(top[2][0], top[3][0]));
#pragma unroll
    for (int u = 0; u < 8; u++) { row_top[u] = m; col_top[u] = m; }
  } else if (T) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
      col_top[e] = max(col_top[e], (uint32_t) __shfl_xor((int) col_top[e], 16));
      col_top[e] = max(col_top[e], (uint32_t) __shfl_xor((int) col_top[e], 32));
    }
    if ((t & 48) == 0) {
#pragma unroll
      for (int e = 0; e < 8; e++) top[t >> 6][c8 + e] = col_top[e];
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; e++) col_top[e] = max(max(top[0][c8 + e], top[1][c8 + e]), max(top[2][c8 + e], top[3][c8 + e]));
  }
  if (!T || p.q) {
#pragma unroll
    for (int u = 0; u < 8; u++) {
      const uint32_t code = scale_code(row_top[u], p.top);
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] = x[u].at(e);
      if (r8 + u < nr) {
        store_bytes(p.q + (r0 + r8 + u) * p.ldq + c0 + c8, f8_eight(v, scale_inverse(code), p.top), nc - c8);
        if ((t & 15) == 0 && (GROUP == 1 || r8 + u == 0)) p.s[(GROUP == 1 ? r0 + r8 + u : bi) * p.lds + bj] = (uint8_t) code;
      }
    }
  }
  if (!T) return;
#pragma unroll
  for (int e = 0; e < 8; e++) {
    const uint32_t code = scale_code(col_top[e], p.top);
    float v[8];
#pragma unroll
    for (int u = 0; u < 8; u++) v[u] = x[u].at(e);
    turned[(c8 + e) * 16 + ((t >> 4) ^ (t & 15))] = f8_eight(v, scale_inverse(code), p.top);
    if (t < 16 && c8 + e < nc && (GROUP == 1 || c8 + e == 0)) p.st[(GROUP == 1 ? c0 + c8 + e : bj) * p.ldst + bi] = (uint8_t) code;
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < 4; u++) {   // 8 threads a column: two units each
    const int c = u * 32 + (t >> 3), k = c >> 3, pair = t & 7;
    if (c >= nc) continue;
    uint8_t *to = p.qt + (c0 + c) * p.ldqt + r0 + pair * 16;
    const uint64_t lo = turned[c * 16 + ((2 * pair) ^ k)], hi = turned[c * 16 + ((2 * pair + 1) ^ k)];
    if (pair * 16 + 16 <= nr) {
      const uint64_t both[2] = {lo, hi};
      __builtin_memcpy(to, both, 16);
    } else {
      store_bytes(to, lo, nr - pair * 16);
      store_bytes(to + 8, hi, nr - pair * 16 - 8);
    }
  }
}

template <int X>
hipError_t launch_quant(const Quant &p, int group, hipStream_t st) {
  const unsigned tiles = (unsigned) (((p.rows + 127) >> 7) * ((p.cols + 127) >> 7));
  drop_stale_error();
  if (p.qt) {
    if (group == 1) quant_kernel<X, 1, true><<<tiles, 256, 0, st>>>(p);
    else quant_kernel<X, 128, true><<<tiles, 256, 0, st>>>(p);
  } else {
    if (group == 1) quant_kernel<X, 1, false><<<tiles, 256, 0, st>>>(p);
    else quant_kernel<X, 128, false><<<tiles, 256, 0, st>>>(p);
  }
  return hipGetLastError();
}

// A launch holds less than 2^32 threads along a dimension of its grid: workgroups go on along the second one.
__device__ __forceinline__ int64_t workgroup() { return (int64_t) blockIdx.y * gridDim.x + blockIdx.x; }
dim3 grid_of(int64_t workgroups) {
  const int64_t x = workgroups < (1 << 21) ? workgroups : 1 << 21;
  return dim3((unsigned) x, (unsigned) ((workgroups + x - 1) / x));
}

// ---- a row and its team -------------------------------------------------------------
// TEAM threads (a wave, or a workgroup of several) work on one row; thread t of the team holds CH chunks of eight
// neighbours, chunk i at column (i * TEAM + t) * 8: 16 neighbouring lanes hold one block of 128.  Rows of up to
// TEAM * CH * 8 columns stay in registers (KEEP); longer ones are read again for the second half of the work.
constexpr int team_width(int team, int ch) { return team * ch * 8; }

// sum over the team, in a fixed order, for all of it; `part`: a float for each wave of the workgroup
template <int TEAM>
__device__ __forceinline__ float team_sum(float v, float *part) {
  v = sum_of_wave(v);
  if constexpr (TEAM > 64) {
    __syncthreads();   // (the last sum's parts have been read)
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int i = 1; i < TEAM / 64; i++) v += part[i];
  }
  return v;
}

// ---- norm ---------------------------------------------------------------------------
struct Norm {
  const void *x, *r, *w;
  int64_t ldx, ldr, ldh, ldq, lds, ldy, n, rows;
  float eps;
  void *h, *y;
  uint8_t *q, *s;
  float *rstd;
  int top;
};

// One pass: the row lies in registers between its sum of squares and its outputs (the team is the smallest whose registers hold it:
// a wave for 512 columns, 256 threads for 8192, 1024 beyond that), so every array is read or written once and bytes bound it:
// 8192 x 8192 bf16 with residual, h, 8-bit output and rstd in 114 us (5.3 TB/s; read twice and element by element, 352 us).  One row is bound by its
// launch and one latency of memory, 3 us; its call by the host.
template <int T, int TEAM, int CH, bool KEEP>
__global__ void __launch_bounds__(TEAM < 256 ? 256 : TEAM) norm_kernel(Norm p) {
  constexpr int TEAMS = TEAM < 256 ? 256 / TEAM : 1;
  __shared__ float part[TEAM < 256 ? 1 : TEAM / 64];
  const int t = threadIdx.x % TEAM;
  const int64_t row = workgroup() * TEAMS + threadIdx.x / TEAM;
  if (row >= p.rows) return;
  float h[CH][8];
  auto fetch = [&](int64_t c0) {
    Eight<T> x[CH], r[CH];
#pragma unroll
    for (int i = 0; i < CH; i++) {
      const int64_t c = c0 + (i * TEAM + t) * 8;
      x[i] = load_eight<T>(p.x, row * p.ldx + c, p.n - c);
      if (p.r) r[i] = load_eight<T>(p.r, row * p.ldr + c, p.n - c);
    }
#pragma unroll
    for (int i = 0; i < CH; i++)
#pragma unroll
      for (int e = 0; e < 8; e++) h[i][e] = p.r ? x[i].at(e) + r[i].at(e) : x[i].at(e);
  };
  float sq = 0.f;
  for (int64_t c0 = 0; c0 < (KEEP ? 1 : p.n); c0 += team_width(TEAM, CH)) {
    fetch(c0);
#pragma unroll
    for (int i = 0; i < CH; i++)
#pragma unroll
      for (int e = 0; e < 8; e++) sq = fmaf(h[i][e], h[i][e], sq);
  }
  const float rstd = 1.f / sqrtf(team_sum<TEAM>(sq, part) / (float) p.n + p.eps);
  if (t == 0 && p.rstd) p.rstd[row] = rstd;
  for (int64_t c0 = 0; c0 < (KEEP ? 1 : p.n); c0 += team_width(TEAM, CH)) {
    if (!KEEP) fetch(c0);
#pragma unroll
    for (int i = 0; i < CH; i++) {
      const int64_t c = c0 + (i * TEAM + t) * 8, valid = p.n - c;
      if (p.h) store_eight<T>(p.h, row * p.ldh + c, h[i], valid);
      if (!p.y && !p.q) continue;
      const Eight<T> w = load_eight<T>(p.w, c, valid);
      float y[8];
      uint32_t m = 0;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        y[e] = e < valid ? h[i][e] * rstd * w.at(e) : 0.f;   // (rstd may be infinite: nothing beyond the row counts)
        m = max(m, finite_magnitude(y[e]));
      }
      if (p.y) store_eight<T>(p.y, row * p.ldy + c, y, valid);
      if (p.q) {
        const uint32_t code = scale_code(max_of_16(m), p.top);
        store_bytes(p.q + row * p.ldq + c, f8_eight(y, scale_inverse(code), p.top), valid);
        if ((t & 15) == 0 && valid > 0) p.s[row * p.lds + (c >> 7)] = (uint8_t) code;
      }
    }
  }
}

template <int T, int TEAM, int CH, bool KEEP = true>
void start_norm(const Norm &p, hipStream_t st) {
  constexpr int TEAMS = TEAM < 256 ? 256 / TEAM : 1;
  norm_kernel<T, TEAM, CH, KEEP><<<grid_of((p.rows + TEAMS - 1) / TEAMS), TEAM < 256 ? 256 : TEAM, 0, st>>>(p);
}
template <int T>
hipError_t launch_norm(const Norm &p, hipStream_t st) {
  drop_stale_error();
  if (p.n <= team_width(64, 1)) start_norm<T, 64, 1>(p, st);
  else if (p.n <= team_width(64, 2)) start_norm<T, 64, 2>(p, st);
  else if (p.n <= team_width(256, 1)) start_norm<T, 256, 1>(p, st);
  else if (p.n <= team_width(256, 2)) start_norm<T, 256, 2>(p, st);
  else if (p.n <= team_width(256, 4)) start_norm<T, 256, 4>(p, st);
  else if (p.n <= team_width(1024, 2)) start_norm<T, 1024, 2>(p, st);
  else if (p.n <= team_width(1024, 4)) start_norm<T, 1024, 4>(p, st);
  else start_norm<T, 1024, 4, false>(p, st);
  return hipGetLastError();
}

// ---- gradient of the norm -----------------------------------------------------------
struct NormGrad {
  const void *dy, *h, *w, *dh;
  const float *rstd;
  void *dx;
  int64_t lddy, ldh, lddh, lddx, rows, n;
  float *part;   // a row of part_columns(n) sums for each team
  float *dw;
  float beta;
  int teams;
};

// rows of `part` begin at multiples of 16 bytes; what lies behind n is read and not used
__host__ __device__ inline int64_t part_columns(int64_t n) { return (n + 3) & ~(int64_t) 3; }

// Team g of `teams` takes rows g, g + teams, ...: every thread keeps its columns' part of dw in registers over all of them
// (rows too long for that: in the team's row of `part`).  Bound by bytes: 8192 x 8192 bf16 with dh in 101 us, and 4 for the join
// (5.1 TB/s together).  Few rows are bound by the two launches: 129 x 5001 fp32 in 12 us.
template <int T, int TEAM, int CH, bool KEEP>
__global__ void __launch_bounds__(TEAM < 256 ? 256 : TEAM) norm_grad_kernel(NormGrad p) {
  constexpr int TEAMS = TEAM < 256 ? 256 / TEAM : 1;
  __shared__ float red[TEAM < 256 ? 1 : TEAM / 64];
  const int t = threadIdx.x % TEAM, team = blockIdx.x * TEAMS + threadIdx.x / TEAM;
  if (TEAMS > 1 && team >= p.teams) return;
  float *part = p.part ? p.part + (int64_t) team * part_columns(p.n) : nullptr;
  const int64_t span = KEEP ? 1 : p.n;
  float dw[CH][8] = {};
  Eight<T> w[CH], dy[CH], h[CH], dh[CH];
  auto fetch = [&](int64_t row, int64_t c0) {
#pragma unroll
    for (int i = 0; i < CH; i++) {
      const int64_t c = c0 + (i * TEAM + t) * 8;
      dy[i] = load_eight<T>(p.dy, row * p.lddy + c, p.n - c);
      h[i] = load_eight<T>(p.h, row * p.ldh + c, p.n - c);
      if (p.dh && KEEP) dh[i] = load_eight<T>(p.dh, row * p.lddh + c, p.n - c);
      if (!KEEP) w[i] = load_eight<T>(p.w, c, p.n - c);
    }
  };
  if (KEEP) {
#pragma unroll
    for (int i = 0; i < CH; i++) w[i] = load_eight<T>(p.w, (i * TEAM + t) * 8, p.n - (i * TEAM + t) * 8);
  }
  for (int64_t row = team; row < p.rows; row += p.teams) {
    const float rstd = p.rstd[row];
    float dot = 0.f;
    for (int64_t c0 = 0; c0 < span; c0 += team_width(TEAM, CH)) {
      fetch(row, c0);
#pragma unroll
      for (int i = 0; i < CH; i++)
#pragma unroll
        for (int e = 0; e < 8; e++) dot = fmaf(dy[i].at(e) * w[i].at(e), h[i].at(e) * rstd, dot);
    }
    const float mean = team_sum<TEAM>(dot, red) / (float) p.n;
    for (int64_t c0 = 0; c0 < span; c0 += team_width(TEAM, CH)) {
      if (!KEEP) fetch(row, c0);
#pragma unroll
      for (int i = 0; i < CH; i++) {
        const int64_t c = c0 + (i * TEAM + t) * 8, valid = p.n - c;
        if (!KEEP && p.dh) dh[i] = load_eight<T>(p.dh, row * p.lddh + c, valid);
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const float g = dy[i].at(e), xhat = h[i].at(e) * rstd;
          v[e] = rstd * (g * w[i].at(e) - xhat * mean);
          if (p.dh) v[e] += dh[i].at(e);
          if (KEEP) dw[i][e] = fmaf(g, xhat, dw[i][e]);
        }
        store_eight<T>(p.dx, row * p.lddx + c, v, valid);
        if (!KEEP && part) {
          const bool first = row == team;
#pragma unroll
          for (int e = 0; e < 8; e++)
            if (e < valid) {
              const float xhat = h[i].at(e) * rstd;
              part[c + e] = first ? dy[i].at(e) * xhat : fmaf(dy[i].at(e), xhat, part[c + e]);
            }
        }
      }
    }
  }
  if (KEEP && part) {
#pragma unroll
    for (int i = 0; i < CH; i++) store_eight<BOF_F32>(part, (i * TEAM + t) * 8, dw[i], p.n - (i * TEAM + t) * 8);
  }
}

// dw = beta * dw + the teams' sums.  A workgroup: 32 columns, four a thread; 32 slices of the teams, each summed in its order, then
// the slices in theirs, 16 a thread.  (The gradient of 16384 rows of 512 in 19.5 us, with 64 columns and 16 slices in 22.4.)
__global__ void __launch_bounds__(256) norm_grad_join_kernel(const float *part, int teams, int64_t n, float beta, float *dw) {
  __shared__ f32x4 sums[32][8];
  const int t = threadIdx.x, col = t & 7, slice = t >> 3;
  const int64_t np = part_columns(n), c = workgroup() * 32 + col * 4;
  const int per = (teams + 31) / 32, g0 = slice * per, g1 = min(teams, g0 + per);
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  if (c < n) {
#pragma unroll 8
    for (int g = g0; g < g1; g++) sum += *(const f32x4 *) (part + g * np + c);
  }
  sums[slice][col] = sum;
  __syncthreads();
  if (t >= 64) return;
  const int64_t to = workgroup() * 32 + (t & 31);
  float v = 0.f;
#pragma unroll
  for (int i = 0; i < 16; i++) v += sums[(t >> 5) * 16 + i][(t & 31) >> 2][t & 3];
  v += __shfl_xor(v, 32);
  if (t < 32 && to < n) dw[to] = beta == 0.f ? v : fmaf(beta, dw[to], v);
}

// enough teams to fill the card; each writes a row of n sums, which the join reads: 3 % of the rows' own bytes at 8192 rows
int64_t grad_teams(int64_t rows, int64_t n) {
  const int64_t most = n <= team_width(64, 2) ? 2048 : n <= team_width(256, 4) ? 512 : 256;
  return rows < most ? rows : most;
}

template <int T, int TEAM, int CH, bool KEEP = true>
void start_norm_grad(const NormGrad &p, hipStream_t st) {
  constexpr int TEAMS = TEAM < 256 ? 256 / TEAM : 1;
  norm_grad_kernel<T, TEAM, CH, KEEP><<<(unsigned) ((p.teams + TEAMS - 1) / TEAMS), TEAM < 256 ? 256 : TEAM, 0, st>>>(p);
}
template <int T>
hipError_t launch_norm_grad(const NormGrad &p, hipStream_t st) {
  drop_stale_error();
  if (p.n <= team_width(64, 1)) start_norm_grad<T, 64, 1>(p, st);
  else if (p.n <= team_width(64, 2)) start_norm_grad<T, 64, 2>(p, st);
  else if (p.n <= team_width(256, 1)) start_norm_grad<T, 256, 1>(p, st);
  else if (p.n <= team_width(256, 2)) start_norm_grad<T, 256, 2>(p, st);
  else if (p.n <= team_width(256, 4)) start_norm_grad<T, 256, 4>(p, st);
  else if (p.n <= team_width(1024, 2)) start_norm_grad<T, 1024, 2>(p, st);
  else start_norm_grad<T, 1024, 1, false>(p, st);
  if (p.dw) norm_grad_join_kernel<<<grid_of((p.n + 31) / 32), 256, 0, st>>>(p.part, p.teams, p.n, p.beta, p.dw);
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
  Quant p{x, ldx, rows, cols, (uint8_t *) q, s, (uint8_t *) qt, st, ldq, lds, ldqt, ldst, f8_top(f8_type)};
  hipStream_t hs = (hipStream_t) stream;
  BOF_HIP_TRY(x_type == BOF_F32 ? launch_quant<BOF_F32>(p, group, hs) : x_type == BOF_BF16 ? launch_quant<BOF_BF16>(p, group, hs) : launch_quant<BOF_F16>(p, group, hs));
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
  Norm p{x, r, w, ldx, ldr, ldh, ldq, lds, ldy, n, rows, eps, h, y, (uint8_t *) q, s, rstd, f8_top(f8_type)};
  hipStream_t hs = (hipStream_t) stream;
  BOF_HIP_TRY(type == BOF_F32 ? launch_norm<BOF_F32>(p, hs) : type == BOF_BF16 ? launch_norm<BOF_BF16>(p, hs) : launch_norm<BOF_F16>(p, hs));
  return BOF_OK;
}

uint64_t bof_rmsnorm_grad_workspace_bytes(int64_t rows, int64_t n) {
  if (rows <= 0 || n <= 0 || rows > (1 << 24) - 1 || n > INT32_MAX - 255) return 0;
  return (uint64_t) grad_teams(rows, n) * (uint64_t) part_columns(n) * 4u;
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
    norm_grad_join_kernel<<<grid_of((n + 31) / 32), 256, 0, hs>>>(nullptr, 0, n, beta, dw);
    BOF_HIP_TRY(hipGetLastError());
    return BOF_OK;
  }
  for (auto [p, name] : {std::pair<const void *, const char *>{dy, "dy"}, {h, "h"}, {w, "w"}, {rstd, "rstd"}, {dh, "dh"}, {dx, "dx"}, {dw ? work : nullptr, "work"}})
    if (int rc = p ? dev.reaches(p, kCall, name) : 0) return rc;
  NormGrad p{dy, h, w, dh, rstd, dx, lddy, ldh, lddh, lddx, rows, n, dw ? (float *) work : nullptr, dw, beta, (int) grad_teams(rows, n)};
  BOF_HIP_TRY(type == BOF_F32 ? launch_norm_grad<BOF_F32>(p, hs) : type == BOF_BF16 ? launch_norm_grad<BOF_BF16>(p, hs) : launch_norm_grad<BOF_F16>(p, hs));
  return BOF_OK;
}

}  // extern "C"
