// LayerNorm over the last axis of token tensors, forward and backward, for fp32 / bf16 / fp16 activations of any width:
//   mean = sum x / D,  rstd = 1 / sqrt(sum (x - mean)^2 / D + eps),  y = (x - mean) rstd w + b
//   xhat = (x - mean) rstd,  a = dy w,  dx = rstd (a - mean(a) - xhat mean(a xhat)),  dw = sum_rows dy xhat,  db = sum_rows dy
// (train/models.py:90, :116, :214 apply it in fp32 to packed tokens of one model width).
//
// Bound: HBM (8 and 14 flop per value).  A row is read once and stays in registers between its statistics and its output,
// so the variance is the two-pass one at no cost.  LANES lanes share a row, each holding NV pieces of 16 bytes: as many
// lanes as the row has pieces up to a wave, then NV up to 4, then a whole workgroup.  Rows of more than 256 x 8 pieces are
// read again for each pass (they come back from the caches).  Statistics, sums and products are fp32.
#include "token.h"

namespace {

// Sum of one value per lane over a whole 256-thread workgroup (LANES == 256) or a group inside a wave.  `red` is 8 floats of
// LDS; the two halves alternate between consecutive calls so that one barrier per call is enough.
template <int LANES>
__device__ __forceinline__ float row_sum(float v, float* red, int& phase) {
  if constexpr (LANES <= 64) {
    return lanes_sum<LANES>(v);
  } else {
    v = lanes_sum<64>(v);
    float* r = red + 4 * phase;
    phase ^= 1;
    if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = v;
    __syncthreads();
    return (r[0] + r[1]) + (r[2] + r[3]);
  }
}

// A lane group works on `per` rows one after the other, RPB apart, with the parameters in registers and the next row
// requested ahead: at one row each, 16 KB of weights and biases come from L2 for every 4 KB row of 2048 bf16 values.
template <typename T, typename W, int VEC, int LANES, int NV, bool NT>
__global__ __launch_bounds__(256) void ln_fwd_kernel(const T* __restrict__ x, long ldx, const W* __restrict__ w,
                                                     const W* __restrict__ b, float eps, T* __restrict__ y,
                                                     float* __restrict__ mean, float* __restrict__ rstd, long rows, int D,
                                                     int per) {
  constexpr int RPB = 256 / LANES;
  __shared__ float red[8];
  int phase = 0;
  const int lane = threadIdx.x % LANES;
  long row = (long)blockIdx.x * RPB * per + threadIdx.x / LANES;
  if (row >= rows) return;                                    // LANES == 256: the whole workgroup
  const long end = min(rows, row + (long)RPB * per);
  using Piece = typename VecOf<T, VEC>::type;
  Piece next[NV];
  auto request = [&](long r) {
    const T* xr = x + (size_t)r * ldx;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * LANES + lane) * VEC;
      if (c < D) next[k] = *reinterpret_cast<const Piece*>(xr + c);
    }
  };
  request(row);
  float ww[NV][VEC], bb[NV][VEC];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (k * LANES + lane) * VEC;
#pragma unroll
    for (int i = 0; i < VEC; ++i) ww[k][i] = 1.f, bb[k][i] = 0.f;
    if (w && c < D) load_vec<W, VEC>(w + c, ww[k]);
    if (b && c < D) load_vec<W, VEC>(b + c, bb[k]);
  }
  const float inv = 1.f / (float)D;
  for (; row < end; row += RPB) {
    float v[NV][VEC];
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const bool in = (k * LANES + lane) * VEC < D;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        if constexpr (VEC == 1) v[k][i] = in ? (float)next[k] : 0.f;
        else v[k][i] = in ? (float)next[k][i] : 0.f;
        s += v[k][i];
      }
    }
    if (row + RPB < end) request(row + RPB);
    const float m = row_sum<LANES>(s, red, phase) * inv;
    float q = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const bool in = (k * LANES + lane) * VEC < D;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        v[k][i] = v[k][i] - m;
        q += in ? v[k][i] * v[k][i] : 0.f;
      }
    }
    const float r = 1.f / sqrtf(row_sum<LANES>(q, red, phase) * inv + eps);
    T* yr = y + (size_t)row * D;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * LANES + lane) * VEC;
      if (c >= D) continue;
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[k][i] = v[k][i] * r * ww[k][i] + bb[k][i];
      store_vec_nt<NT, T, VEC>(yr + c, v[k]);
    }
    if (lane == 0) {
      if (mean) mean[row] = m;
      if (rstd) rstd[row] = r;
    }
  }
}

// Rows too wide for registers: one workgroup per row, three passes.
template <typename T, typename W>
__global__ __launch_bounds__(256) void ln_fwd_wide_kernel(const T* __restrict__ x, long ldx, const W* __restrict__ w,
                                                          const W* __restrict__ b, float eps, T* __restrict__ y,
                                                          float* __restrict__ mean, float* __restrict__ rstd, int D) {
  __shared__ float red[8];
  int phase = 0;
  const long row = blockIdx.x;
  const T* xr = x + (size_t)row * ldx;
  float s = 0.f;
  for (int c = threadIdx.x; c < D; c += 256) s += (float)xr[c];
  const float m = row_sum<256>(s, red, phase) / (float)D;
  float q = 0.f;
  for (int c = threadIdx.x; c < D; c += 256) {
    const float d = (float)xr[c] - m;
    q += d * d;
  }
  const float r = 1.f / sqrtf(row_sum<256>(q, red, phase) / (float)D + eps);
  T* yr = y + (size_t)row * D;
  for (int c = threadIdx.x; c < D; c += 256) {
    float o = ((float)xr[c] - m) * r;
    if (w) o *= (float)w[c];
    if (b) o += (float)b[c];
    yr[c] = (T)o;
  }
  if (threadIdx.x == 0) {
    if (mean) mean[row] = m;
    if (rstd) rstd[row] = r;
  }
}

// A workgroup walks its rows; a lane keeps the sums of dw and db of its columns in registers, the row groups of a workgroup
// are added in LDS in a fixed order, and each workgroup leaves one slab row [dw | db] for ln_fold_kernel: no atomics, the
// same result on every run.  A row's sums are fp32 over rows / (grid x groups) terms, the fold is in double.
template <typename T, typename W, int VEC, int LANES, int NV, bool NT>
__global__ __launch_bounds__(256) void ln_bwd_kernel(const T* __restrict__ dy, long lddy, const T* __restrict__ x, long ldx,
                                                     const float* __restrict__ mean, const float* __restrict__ rstd,
                                                     const W* __restrict__ w, T* __restrict__ dx, float* __restrict__ slab,
                                                     long rows, int D) {
  constexpr int RPB = 256 / LANES;
  __shared__ float red[8];
  __shared__ float part[LANES < 256 ? 256 * VEC : 1];
  int phase = 0;
  const int lane = threadIdx.x % LANES, grp = threadIdx.x / LANES;
  float ww[NV][VEC], dw[NV][VEC], db[NV][VEC];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (k * LANES + lane) * VEC;
#pragma unroll
    for (int i = 0; i < VEC; ++i) ww[k][i] = 1.f, dw[k][i] = 0.f, db[k][i] = 0.f;
    if (w && c < D) load_vec<W, VEC>(w + c, ww[k]);
  }
  const float inv = 1.f / (float)D;
  // the next row is requested before the current one is worked on
  using Piece = typename VecOf<T, VEC>::type;
  Piece nx[NV], ng[NV];
  float nm = 0.f, nr = 0.f;
  auto request = [&](long row) {
    const T *xr = x + (size_t)row * ldx, *gr = dy + (size_t)row * lddy;
    nm = mean[row];
    nr = rstd[row];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * LANES + lane) * VEC;
      if (c < D) {
        nx[k] = *reinterpret_cast<const Piece*>(xr + c);
        ng[k] = *reinterpret_cast<const Piece*>(gr + c);
      }
    }
  };
  const long step = (long)gridDim.x * RPB;
  long row = (long)blockIdx.x * RPB + grp;
  if (row < rows) request(row);
  for (; row < rows; row += step) {
    const float m = nm, r = nr;
    float h[NV][VEC], g[NV][VEC];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const bool in = (k * LANES + lane) * VEC < D;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        if constexpr (VEC == 1) {
          h[k][i] = in ? (float)nx[k] : m;
          g[k][i] = in ? (float)ng[k] : 0.f;
        } else {
          h[k][i] = in ? (float)nx[k][i] : m;
          g[k][i] = in ? (float)ng[k][i] : 0.f;
        }
      }
    }
    if (row + step < rows) request(row + step);
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        h[k][i] = (h[k][i] - m) * r;
        dw[k][i] += g[k][i] * h[k][i];
        db[k][i] += g[k][i];
        g[k][i] *= ww[k][i];
        s1 += g[k][i];
        s2 += g[k][i] * h[k][i];
      }
    s1 = row_sum<LANES>(s1, red, phase) * inv;
    s2 = row_sum<LANES>(s2, red, phase) * inv;
    T* o = dx + (size_t)row * D;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * LANES + lane) * VEC;
      if (c >= D) continue;
#pragma unroll
      for (int i = 0; i < VEC; ++i) g[k][i] = r * (g[k][i] - s1 - h[k][i] * s2);
      store_vec_nt<NT, T, VEC>(o + c, g[k]);
    }
  }
  if (!slab) return;
  float* out = slab + (size_t)blockIdx.x * 2 * D;
#pragma unroll
  for (int which = 0; which < 2; ++which)
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float* acc = which ? db[k] : dw[k];
      const int c = (k * LANES + lane) * VEC;
      if constexpr (LANES < 256) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < VEC; ++i) part[i * 256 + threadIdx.x] = acc[i];
        __syncthreads();
        if (grp == 0 && c < D) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            float t = 0.f;
            for (int j = 0; j < RPB; ++j) t += part[i * 256 + j * LANES + lane];
            out[(size_t)which * D + c + i] = t;
          }
        }
      } else if (c < D) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) out[(size_t)which * D + c + i] = acc[i];
      }
    }
}

// Rows too wide for registers, first half: dx with the row read twice.
template <typename T, typename W>
__global__ __launch_bounds__(256) void ln_bwd_wide_kernel(const T* __restrict__ dy, long lddy, const T* __restrict__ x,
                                                          long ldx, const float* __restrict__ mean,
                                                          const float* __restrict__ rstd, const W* __restrict__ w,
                                                          T* __restrict__ dx, int D) {
  __shared__ float red[8];
  int phase = 0;
  const long row = blockIdx.x;
  const T *xr = x + (size_t)row * ldx, *gr = dy + (size_t)row * lddy;
  const float m = mean[row], r = rstd[row], inv = 1.f / (float)D;
  float s1 = 0.f, s2 = 0.f;
  for (int c = threadIdx.x; c < D; c += 256) {
    const float a = (float)gr[c] * (w ? (float)w[c] : 1.f);
    s1 += a;
    s2 += a * (((float)xr[c] - m) * r);
  }
  s1 = row_sum<256>(s1, red, phase) * inv;
  s2 = row_sum<256>(s2, red, phase) * inv;
  T* o = dx + (size_t)row * D;
  for (int c = threadIdx.x; c < D; c += 256) {
    const float a = (float)gr[c] * (w ? (float)w[c] : 1.f);
    o[c] = (T)(r * (a - s1 - ((float)xr[c] - m) * r * s2));
  }
}
// second half: column sums, a workgroup covers 256 columns of a share of the rows
template <typename T>
__global__ __launch_bounds__(256) void ln_bwd_cols_kernel(const T* __restrict__ dy, long lddy, const T* __restrict__ x,
                                                          long ldx, const float* __restrict__ mean,
                                                          const float* __restrict__ rstd, float* __restrict__ slab, long rows,
                                                          int D) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= D) return;
  float a = 0.f, b = 0.f;
  for (long row = blockIdx.y; row < rows; row += gridDim.y) {
    const float g = (float)dy[(size_t)row * lddy + c];
    a += g * (((float)x[(size_t)row * ldx + c] - mean[row]) * rstd[row]);
    b += g;
  }
  float* out = slab + (size_t)blockIdx.y * 2 * D;
  out[c] = a;
  out[D + c] = b;
}

// dw, db = column sums of the slab, COLS columns x 256 / COLS row lanes per workgroup, eight rows in flight per lane.
template <typename W, int COLS>
__global__ __launch_bounds__(256) void ln_fold_kernel(const float* __restrict__ slab, int nrows, W* __restrict__ dw,
                                                      W* __restrict__ db, int D) {
  constexpr int RL = 256 / COLS;
  __shared__ double red[256];
  const long col = (long)blockIdx.x * COLS + threadIdx.x % COLS;
  const int rl = threadIdx.x / COLS;
  const long ncols = 2L * D;
  double s = 0.0;
  if (col < ncols)
    for (int r0 = rl; r0 < nrows; r0 += 8 * RL) {
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int r = r0 + u * RL;
        v[u] = slab[(size_t)(r < nrows ? r : nrows - 1) * ncols + col];
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) s += r0 + u * RL < nrows ? (double)v[u] : 0.0;
    }
  red[threadIdx.x] = s;
  __syncthreads();
  if (rl == 0 && col < ncols) {
    double t = 0.0;
    for (int j = 0; j < RL; ++j) t += red[j * COLS + threadIdx.x];
    if (col < D) {
      if (dw) dw[col] = (W)(float)t;
    } else {
      if (db) db[col - D] = (W)(float)t;
    }
  }
}

// Slab rows of a backward call.  More workgroups than fit the GPU at once gain nothing here, and the slab (8 D bytes a row,
// written and read again) has to stay small beside the rows themselves.
constexpr int LN_BWD_GRID = 1024, LN_WIDE_SLAB = 64;

struct LnGeom {
  int vec, lanes, nv;   // lanes == 0: the wide kernels
};

// The narrowest group of lanes that holds the row, a wave with at most `most` pieces per lane (forward 4; backward 2, since each
// piece brings two gradient sums along: 65536 rows of 2048 bf16 values take 179 us with 64 lanes x 4 and 156 with 256 x 1).
// `vec` is the 16-byte piece when every row of every tensor starts on a 16-byte boundary and the width is a whole number of
// pieces, else single values, whatever the width.
LnGeom ln_geom(int D, int vec, int most) {
  static const int shapes[][2] = {{16, 1}, {32, 1}, {64, 1}, {64, 2}, {64, 4}, {256, 1}, {256, 2}, {256, 4}, {256, 8}};
  for (auto& s : shapes)
    if ((s[0] == 256 || s[1] <= most) && (long)s[0] * s[1] * vec >= D) return {vec, s[0], s[1]};
  return {vec, 0, 0};
}

// Results of 128 MB and more are stored past the caches: their reader would not find them there, and the inputs keep the room
// (65536 rows of 2048 bf16 values: 116 -> 91 us; no difference at 134 MB, nothing lost below).
bool ln_past_caches(long rows, int D, int esize) { return rows * D * esize >= (1L << 27); }

bool aligned16(const void* p) { return p == nullptr || ((uintptr_t)p & 15) == 0; }

template <typename T>
int ln_vec(int D, long ld0, long ld1, std::initializer_list<const void*> ptrs) {
  constexpr int V = 16 / sizeof(T);
  if (D % V || ld0 % V || ld1 % V) return 1;
  for (const void* p : ptrs)
    if (!aligned16(p)) return 1;
  return V;
}

// A grid holds at most 2^32 threads, so one launch of a workgroup per row covers at most this many rows.
constexpr long LN_LAUNCH_ROWS = 1L << 23;

// Rows per lane group of a forward call, where 2048 workgroups remain: more of them amortise the parameters, fewer keep the
// accesses in flight close together.  1 / 2 / 4 / 8 rows: 65536 x 2048 bf16 107 / 93 / 99 / 109 us, 16384 x 8192 bf16 - / 96 / 98 /
// 109, 524288 x 128 fp32 - / 93 / 97 / 97.
constexpr int LN_FWD_PER = 2, LN_FWD_FULL = 2048;

// M(vec, lanes, nv, nt) for the chosen shape; rows of 129 to 256 pieces take L lanes with N pieces each.  Only whole pieces are
// stored past the caches; single values go through them and are merged into lines there.
#define LN_SHAPES(M, V, NT, L, N)                                           \
  if (g.lanes == 16) M(V, 16, 1, NT)                                        \
  else if (g.lanes == 32) M(V, 32, 1, NT)                                   \
  else if (g.lanes == 64 && g.nv == 1) M(V, 64, 1, NT)                      \
  else if (g.lanes == 64 && g.nv == 2) M(V, 64, 2, NT)                      \
  else if (g.lanes == L && g.nv == N) M(V, L, N, NT)                        \
  else if (g.nv == 2) M(V, 256, 2, NT)                                      \
  else if (g.nv == 4) M(V, 256, 4, NT)                                      \
  else M(V, 256, 8, NT)
#define LN_PICK(M, L, N)                                       \
  if (g.vec == V && nt) { LN_SHAPES(M, V, true, L, N) }        \
  else if (g.vec == V) { LN_SHAPES(M, V, false, L, N) }        \
  else { LN_SHAPES(M, 1, false, L, N) }

template <typename T, typename W>
void ln_fwd_rows(const LnGeom& g, const T* x, long ldx, const W* w, const W* b, float eps, T* y, float* mean, float* rstd,
                 long rows, int D, bool nt, hipStream_t st) {
  constexpr int V = 16 / sizeof(T);
  if (g.lanes == 0) {
    hipLaunchKernelGGL((ln_fwd_wide_kernel<T, W>), dim3((unsigned)rows), dim3(256), 0, st, x, ldx, w, b, eps, y, mean, rstd, D);
    return;
  }
  const long rpb = 256 / g.lanes, groups = (rows + rpb - 1) / rpb;
  const int per = groups >= (long)LN_FWD_FULL * LN_FWD_PER ? LN_FWD_PER : 1;
  const dim3 grid((unsigned)((groups + per - 1) / per));
#define LN_FWD(VV, L, N, NT) hipLaunchKernelGGL((ln_fwd_kernel<T, W, VV, L, N, NT>), grid, dim3(256), 0, st, x, ldx, w, b, eps, y, mean, rstd, rows, D, per);
  LN_PICK(LN_FWD, 64, 4)
#undef LN_FWD
}

template <typename T, typename W>
void ln_fwd(const void* x, long ldx, const void* w, const void* b, float eps, void* y, float* mean, float* rstd, long rows,
            int D, hipStream_t st) {
  const LnGeom g = ln_geom(D, ln_vec<T>(D, ldx, D, {x, w, b, y}), 4);
  const bool nt = ln_past_caches(rows, D, sizeof(T));
  const W *wp = (const W*)w, *bp = (const W*)b;
  for (const long all = rows; rows > 0; rows -= LN_LAUNCH_ROWS) {
    const long first = all - rows, n = rows < LN_LAUNCH_ROWS ? rows : LN_LAUNCH_ROWS;
    const T* xp = (const T*)x + first * ldx;
    T* yp = (T*)y + first * D;
    float *mp = mean ? mean + first : nullptr, *rp = rstd ? rstd + first : nullptr;
    ln_fwd_rows<T, W>(g, xp, ldx, wp, bp, eps, yp, mp, rp, n, D, nt, st);
  }
}

template <typename T, typename W>
void ln_bwd(const void* dy, long lddy, const void* x, long ldx, const float* mean, const float* rstd, const void* w, void* dx,
            void* dw, void* db, float* slab, long rows, int D, hipStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const LnGeom g = ln_geom(D, ln_vec<T>(D, ldx, lddy, {dy, x, w, dx}), 2);
  const bool nt = ln_past_caches(rows, D, sizeof(T));
  const T *xp = (const T*)x, *gp = (const T*)dy;
  const W* wp = (const W*)w;
  T* dp = (T*)dx;
  float* sl = dw || db ? slab : nullptr;
  int nslab;
  if (g.lanes == 0) {
    for (long r = 0; r < rows; r += LN_LAUNCH_ROWS)
      hipLaunchKernelGGL((ln_bwd_wide_kernel<T, W>), dim3((unsigned)(rows - r < LN_LAUNCH_ROWS ? rows - r : LN_LAUNCH_ROWS)), dim3(256), 0,
                         st, gp + r * lddy, lddy, xp + r * ldx, ldx, mean + r, rstd + r, wp, dp + r * D, D);
    nslab = (int)(rows < LN_WIDE_SLAB ? rows : LN_WIDE_SLAB);
    if (sl)
      hipLaunchKernelGGL((ln_bwd_cols_kernel<T>), dim3(noise_cdiv(D, 256), nslab), dim3(256), 0, st, gp, lddy, xp, ldx, mean, rstd, sl, rows, D);
  } else {
    // Measured with 256 / 512 / 1024 / 2048 workgroups: 65536 x 1024 bf16 (64 lanes x 2) 107 / 67 / 78 / 83 us, 65536 x 2048 bf16
    // (256 x 1) - / 159 / 153 / 173, 16384 x 8192 bf16 (256 x 4) 145 / 153 / - / 167
    nslab = noise_grid(rows, 256 / g.lanes, g.lanes < 256 ? LN_BWD_GRID / 2 : g.nv == 1 ? LN_BWD_GRID : LN_BWD_GRID / 4);
    const dim3 grid(nslab);
#define LN_BWD(VV, L, N, NT) hipLaunchKernelGGL((ln_bwd_kernel<T, W, VV, L, N, NT>), grid, dim3(256), 0, st, gp, lddy, xp, ldx, mean, rstd, wp, dp, sl, rows, D);
    LN_PICK(LN_BWD, 256, 1)
#undef LN_BWD
  }
  if (sl) {
    // narrow rows: 8 columns and 32 row lanes per workgroup shorten the chain of dependent reads; wide rows: whole cache lines
    if (D <= 512)
      hipLaunchKernelGGL((ln_fold_kernel<W, 8>), dim3(noise_cdiv(2L * D, 8)), dim3(256), 0, st, sl, nslab, (W*)dw, (W*)db, D);
    else
      hipLaunchKernelGGL((ln_fold_kernel<W, 32>), dim3(noise_cdiv(2L * D, 32)), dim3(256), 0, st, sl, nslab, (W*)dw, (W*)db, D);
  }
}

// activation type x parameter type (fp32, or the activations' own)
#define LN_TYPES(CALL)                                                                              \
  if (dtype == NOISE_F32) CALL(float, float)                                                        \
  else if (dtype == NOISE_BF16 && wdtype == NOISE_F32) CALL(bf16_t, float)                          \
  else if (dtype == NOISE_BF16) CALL(bf16_t, bf16_t)                                                \
  else if (wdtype == NOISE_F32) CALL(f16_t, float)                                                  \
  else CALL(f16_t, f16_t)

bool ln_types_ok(int dtype, int wdtype) {
  return dtype >= NOISE_F32 && dtype <= NOISE_F16 && (wdtype == NOISE_F32 || wdtype == dtype);
}

}  // namespace

// Slab rows a backward call needs at most (rows wider than 256 x 8 pieces always take the wide kernels).
NOISE_EXPORT int noise_layer_norm_bwd_rows(long rows, int D) {
  const long cap = D <= 256 * 8 * 8 ? LN_BWD_GRID : LN_WIDE_SLAB;
  return (int)(rows < 1 ? 1 : rows < cap ? rows : cap);
}

NOISE_EXPORT int noise_layer_norm_fwd(const void* x, long ldx, const void* w, const void* b, float eps, void* y, float* mean,
                                      float* rstd, long rows, int D, int dtype, int wdtype, void* stream) {
  NOISE_REQUIRE(x && y, "noise_layer_norm_fwd: null pointer");
  NOISE_REQUIRE(rows > 0 && rows <= 0x7fffffffL && D > 0 && D <= (1 << 24), "noise_layer_norm_fwd: 1 <= rows < 2^31 and 1 <= D <= 2^24 (got %ld x %d)", rows, D);
  NOISE_REQUIRE(ldx >= 0, "noise_layer_norm_fwd: negative row stride");
  NOISE_REQUIRE(ln_types_ok(dtype, wdtype), "noise_layer_norm_fwd: parameters are fp32 or of the activations' type");
  hipStream_t st = (hipStream_t)stream;
#define CALL(T, W) ln_fwd<T, W>(x, ldx, w, b, eps, y, mean, rstd, rows, D, st);
  LN_TYPES(CALL)
#undef CALL
  NOISE_CHECK_LAUNCH("noise_layer_norm_fwd");
  return 0;
}

NOISE_EXPORT int noise_layer_norm_bwd(const void* dy, long lddy, const void* x, long ldx, const float* mean, const float* rstd,
                                      const void* w, void* dx, void* dw, void* db, float* slab, long rows, int D, int dtype,
                                      int wdtype, void* stream) {
  NOISE_REQUIRE(dy && x && mean && rstd && dx, "noise_layer_norm_bwd: null pointer");
  NOISE_REQUIRE((!dw && !db) || slab, "noise_layer_norm_bwd: parameter gradients need the slab");
  NOISE_REQUIRE(rows > 0 && rows <= 0x7fffffffL && D > 0 && D <= (1 << 24), "noise_layer_norm_bwd: 1 <= rows < 2^31 and 1 <= D <= 2^24 (got %ld x %d)", rows, D);
  NOISE_REQUIRE(ldx >= 0 && lddy >= 0, "noise_layer_norm_bwd: negative row stride");
  NOISE_REQUIRE(ln_types_ok(dtype, wdtype), "noise_layer_norm_bwd: parameters are fp32 or of the activations' type");
  hipStream_t st = (hipStream_t)stream;
#define CALL(T, W) ln_bwd<T, W>(dy, lddy, x, ldx, mean, rstd, w, dx, dw, db, slab, rows, D, st);
  LN_TYPES(CALL)
#undef CALL
  NOISE_CHECK_LAUNCH("noise_layer_norm_bwd");
  return 0;
}
