// Layer norm over the last axis, forward and backward, with the 8-bit checkpoint of its input (act8.h) as one way to keep x.
//
//   forward    mean, rstd = 1 / sqrt(var + eps) (biased, from centred values in registers: no difference of large sums)
//              y = (x - mean) rstd w + b                       [act8: x also leaves as e4m3 blocks, from the same registers]
//   backward   h = (x - mean) rstd, x as it came or from the checkpoint;  g = dy w
//              dx = rstd (g - mean(g) - h mean(g h))           dw = sum over rows of dy h        db = sum over rows of dy
//
// Bound by HBM: one read of x and one write of y; one read of x (or a byte a value) and dy and one write of dx.  A row is held in
// the registers of TPR lanes, NCH chunks of eight values each (the smallest pair that covers the row, tables below), so nothing is read
// twice up to 16384 columns; longer rows walk memory (norm_long_*).  Workgroups stay and take row after row: the parameters are read once,
// and the column sums of dw and db grow in registers.  They leave as one partial row per workgroup, summed by norm_reduce_kernel in
// a fixed order (no atomics: the same bits on every run).
#include <algorithm>
#include "act8.h"
#include "../../include/hcmoco_hip.h"

namespace {

using namespace hcm;

struct Params { const void *w, *b; int wdt, bdt; };

// Sum over the TPR lanes that hold one row; `red`: LDS for TPR > 64 (two float per wave and call parity, so that one barrier a call is enough).
template <int TPR, int N>
__device__ __forceinline__ void row_sum(float (&s)[N], float (*red)[TPR > 64 ? TPR / 64 : 1][2], int& parity) {
#pragma unroll
  for (int n = 0; n < N; ++n) s[n] = TPR == 16 ? row16_sum(s[n]) : wave_sum(s[n]);
  if constexpr (TPR > 64) {
    constexpr int W = TPR / 64;
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int n = 0; n < N; ++n) red[parity][w][n] = s[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {
      s[n] = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) s[n] += red[parity][i][n];
    }
    parity ^= 1;      // the next call writes the other half: a wave cannot be two barriers ahead
  }
}

template <typename T, int TPR, int NCH, int NT>
__global__ __launch_bounds__(NT) void norm_fwd_kernel(const T* __restrict__ x, int64_t ldx, uint32_t rows, int cols, Params P, float eps, T* __restrict__ y,
                                                      float* __restrict__ mean_out, float* __restrict__ rstd_out, uint8_t* __restrict__ q,
                                                      int64_t ldq, uint8_t* __restrict__ scale, int64_t lds) {
  __shared__ float red[2][TPR > 64 ? TPR / 64 : 1][2];
  constexpr int RPB = NT / TPR;
  const int t = threadIdx.x % TPR;
  int parity = 0;
  float w[NCH][8], b[NCH][8];
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    const int col = (j * TPR + t) * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) w[j][i] = 1.f, b[j][i] = 0.f;
    if (col < cols) {
      if (P.w) load8_dt(P.w, P.wdt, col, cols - col, w[j]);
      if (P.b) load8_dt(P.b, P.bdt, col, cols - col, b[j]);
    }
  }
  const float inv_n = 1.f / (float)cols;
  // The next row's values are loaded while this one's are worked on (32768 x 2000 in bf16: 80 -> 66 us).  Eight at a time whatever is left
  // of the row: what lies behind it is the next row's and is masked; only at the very end of the tensor is there nothing behind.
  typedef typename Vec8<T>::type Raw;
  const int64_t end = (int64_t)(rows - 1) * ldx + cols;
  const bool room = cols >= 8;
  auto load = [&](Raw (&r)[NCH], uint32_t row) {
#pragma unroll
    for (int j = 0; j < NCH; ++j)
      if (room) __builtin_memcpy(&r[j], x + min((int64_t)row * ldx + min((j * TPR + t) * 8, cols - 1), end - 8), 8 * sizeof(T));
  };
  Raw next[NCH];
  load(next, min(blockIdx.x * RPB + threadIdx.x / TPR, rows - 1));
  // every lane of a workgroup makes the same number of trips (the barriers of row_sum), rows past the end are clamped and not stored
  for (uint32_t base = blockIdx.x * RPB; base < rows; base += gridDim.x * RPB) {
    const uint32_t want = base + threadIdx.x / TPR, row = min(want, rows - 1);
    float v[NCH][8];
    float s[1] = {0.f};
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int col = (j * TPR + t) * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[j][i] = col + i < cols ? (float)next[j][i] : 0.f;
      if (col < cols && (!room || (int64_t)row * ldx + col > end - 8)) load8(x + (int64_t)row * ldx + col, cols - col, v[j]);
    }
    load(next, min(want + gridDim.x * RPB, rows - 1));
#pragma unroll
    for (int j = 0; j < NCH; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) s[0] += v[j][i];
    row_sum<TPR, 1>(s, red, parity);
    const float mean = s[0] * inv_n;
    if (q) {
#pragma unroll
      for (int j = 0; j < NCH; ++j) {
        const int c8 = j * TPR + t, col = c8 * 8;
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = fmaxf(m, finite_abs(v[j][i]));
        const int byte = act8_byte(row16_max(m));
        if (want < rows) {
          if (col < ldq) *(v2i*)(q + (int64_t)row * ldq + col) = act8_bytes(v[j], inv_pow2_of_byte(byte));
          if ((c8 & 15) == 0 && (c8 >> 4) < lds) scale[(int64_t)row * lds + (c8 >> 4)] = (uint8_t)(col < cols ? byte : 127);
        }
      }
      if (want < rows)      // scale pads that no chunk covers
        for (int k = NCH * TPR / 16 + t; k < lds; k += TPR) scale[(int64_t)row * lds + k] = 127;
    }
    float s2[1] = {0.f};
#pragma unroll
    for (int j = 0; j < NCH; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = (j * TPR + t) * 8 + i < cols ? v[j][i] - mean : 0.f;
        v[j][i] = d;
        s2[0] = fmaf(d, d, s2[0]);
      }
    row_sum<TPR, 1>(s2, red, parity);
    const float rstd = 1.f / sqrtf(s2[0] * inv_n + eps);
    if (want < rows) {
#pragma unroll
      for (int j = 0; j < NCH; ++j) {
        const int col = (j * TPR + t) * 8;
        if (col >= cols) continue;
        float o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = fmaf(v[j][i] * rstd, w[j][i], b[j][i]);
        store8(y + (int64_t)row * cols + col, cols - col, o);
      }
      if (t == 0 && mean_out) mean_out[row] = mean, rstd_out[row] = rstd;
    }
  }
}

// x (ACT8: q, scale) and dy [rows, cols] -> dx, and this workgroup's column sums: part[block][0] = sum dy h, part[block][1] = sum dy
template <typename T, bool ACT8, int TPR, int NCH, int NT>
__global__ __launch_bounds__(NT) void norm_bwd_kernel(const T* __restrict__ x, int64_t ldx, const uint8_t* __restrict__ q, int64_t ldq,
                                                      const uint8_t* __restrict__ scale, int64_t lds, const T* __restrict__ dy, uint32_t rows, int cols,
                                                      Params P, const float* __restrict__ mean_in, const float* __restrict__ rstd_in, T* __restrict__ dx,
                                                      float* __restrict__ part) {
  __shared__ float red[2][TPR > 64 ? TPR / 64 : 1][2];
  constexpr int RPB = NT / TPR;
  const int t = threadIdx.x % TPR;
  int parity = 0;
  float w[NCH][8], aw[NCH][8], ab[NCH][8];
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    const int col = (j * TPR + t) * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) w[j][i] = 1.f, aw[j][i] = 0.f, ab[j][i] = 0.f;
    if (P.w && col < cols) load8_dt(P.w, P.wdt, col, cols - col, w[j]);
  }
  const float inv_n = 1.f / (float)cols;
  // The next row's values are loaded while this one's are worked on.  Eight at a time whatever is left of the row: what lies behind it is
  // the next row's and is masked; only at the very end of the tensor is there nothing behind.
  struct Raw {
    typename Vec8<T>::type d[NCH], x[ACT8 ? 1 : NCH];
    v2i q[ACT8 ? NCH : 1];
    int e[ACT8 ? NCH : 1];
    float mean, rstd;
  };
  const int64_t d_end = (int64_t)rows * cols, x_end = (int64_t)(rows - 1) * ldx + cols;
  const bool room = cols >= 8;
  auto load = [&](Raw& R, uint32_t row) {
    R.mean = mean_in[row];
    R.rstd = rstd_in[row];
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int c8 = j * TPR + t, col = min(c8 * 8, cols - 1);
      if (room) __builtin_memcpy(&R.d[j], dy + min((int64_t)row * cols + col, d_end - 8), 8 * sizeof(T));
      if constexpr (ACT8) {
        R.q[j] = *(const v2i*)(q + (int64_t)row * ldq + min(c8 * 8, (int)ldq - 8));
        R.e[j] = scale[(int64_t)row * lds + min(c8 >> 4, (int)lds - 1)];
      } else {
        if (room) __builtin_memcpy(&R.x[j], x + min((int64_t)row * ldx + col, x_end - 8), 8 * sizeof(T));
      }
    }
  };
  Raw next;
  load(next, min(blockIdx.x * RPB + threadIdx.x / TPR, rows - 1));
  for (uint32_t base = blockIdx.x * RPB; base < rows; base += gridDim.x * RPB) {
    const uint32_t want = base + threadIdx.x / TPR, row = min(want, rows - 1);
    const float mean = next.mean, rstd = next.rstd;
    float h[NCH][8], d[NCH][8];
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int c8 = j * TPR + t, col = c8 * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) d[j][i] = col + i < cols ? (float)next.d[j][i] : 0.f;
      if constexpr (ACT8) {
        act8_values(next.q[j], pow2_of_byte(next.e[j]), h[j]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) h[j][i] = (float)next.x[j][i];
        // the last values of x: load() read others, so as not to pass its end
        if (col < cols && (!room || (int64_t)row * ldx + col > x_end - 8)) load8(x + (int64_t)row * ldx + col, cols - col, h[j]);
      }
      if (col < cols && (!room || (int64_t)row * cols + col > d_end - 8)) load8(dy + (int64_t)row * cols + col, cols - col, d[j]);
#pragma unroll
      for (int i = 0; i < 8; ++i) h[j][i] = col + i < cols ? h[j][i] : mean;
    }
    load(next, min(want + gridDim.x * RPB, rows - 1));
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NCH; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        // columns past the end: dy is zero, and h is not used
        h[j][i] = (h[j][i] - mean) * rstd;
        const float g = d[j][i] * w[j][i];
        s[0] += g;
        s[1] = fmaf(g, h[j][i], s[1]);
      }
    row_sum<TPR, 2>(s, red, parity);
    if (want < rows) {
      const float mg = s[0] * inv_n, mgh = s[1] * inv_n;
#pragma unroll
      for (int j = 0; j < NCH; ++j) {
        const int col = (j * TPR + t) * 8;
        if (col >= cols) continue;
        float o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          aw[j][i] = fmaf(d[j][i], h[j][i], aw[j][i]);
          ab[j][i] += d[j][i];
          o[i] = rstd * (d[j][i] * w[j][i] - mg - h[j][i] * mgh);
        }
        store8(dx + (int64_t)row * cols + col, cols - col, o);
      }
    }
  }
  // the rows of a workgroup that were held side by side: added up through LDS, one of the two sums at a time
  if constexpr (RPB > 1) {
    constexpr int C = TPR * NCH * 8;
    __shared__ float col_sum[RPB][C];
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < NCH; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) col_sum[threadIdx.x / TPR][(j * TPR + t) * 8 + i] = which ? ab[j][i] : aw[j][i];
      __syncthreads();
      for (int c = threadIdx.x; c < cols; c += NT) {
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < RPB; ++r) sum += col_sum[r][c];
        part[((int64_t)blockIdx.x * 2 + which) * cols + c] = sum;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int col = (j * TPR + t) * 8;
      if (col >= cols) continue;
      store8(part + (int64_t)blockIdx.x * 2 * cols + col, cols - col, aw[j]);
      store8(part + ((int64_t)blockIdx.x * 2 + 1) * cols + col, cols - col, ab[j]);
    }
  }
}

// No fp32 sum here is a chain of more than 2 kChain additions, whatever the size (each can lose half a unit of a sum that has grown that
// long): what is longer is added up in runs of kChain, and a batch of many rows gets more launches or slices, each of at most kChain trips.
constexpr int kChain = 256;

// out[c] = sum over `parts` rows of part[][c], c < 2 cols: 64 columns a workgroup, 16 slices of the rows, every load of a slice in flight
constexpr int kRedSlices = 16;
__global__ __launch_bounds__(1024) void norm_reduce_kernel(const float* __restrict__ part, int parts, int cols, void* __restrict__ dw, int wdt,
                                                           void* __restrict__ db, int bdt) {
  __shared__ float s[kRedSlices][64];
  const int lane = threadIdx.x & 63, slice = threadIdx.x >> 6;
  const int64_t c = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 64 + lane, n = 2ll * cols;
  float a[4] = {0.f, 0.f, 0.f, 0.f};
  if (c < n) {
    int p = slice;
    while (p + 3 * kRedSlices < parts) {
      float run[4] = {0.f, 0.f, 0.f, 0.f};
      for (int k = 0; k < kChain && p + 3 * kRedSlices < parts; ++k, p += 4 * kRedSlices)
#pragma unroll
        for (int u = 0; u < 4; ++u) run[u] += part[(int64_t)(p + u * kRedSlices) * n + c];
#pragma unroll
      for (int u = 0; u < 4; ++u) a[u] += run[u];
    }
    for (; p < parts; p += kRedSlices) a[0] += part[(int64_t)p * n + c];
  }
  s[slice][lane] = (a[0] + a[1]) + (a[2] + a[3]);
  __syncthreads();
  if (slice == 0 && c < n) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < kRedSlices; ++i) sum += s[i][lane];
    if (c < cols) { if (dw) store_dt(dw, wdt, c, sum); }
    else if (db) store_dt(db, bdt, c - cols, sum);
  }
}

// ---- rows too long for registers: one workgroup a row, memory is walked again for every pass (it lies in L2 by then) ----
constexpr int kLong = 1024;
__device__ __forceinline__ float block_sum(float v, float* red) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kLong / 64; ++i) s += red[i];
  return s;
}

// sum of term(c) over this thread's columns, in runs (term adds to what it is given)
template <int N, typename Term>
__device__ __forceinline__ void lane_sums(int cols, float (&s)[N], Term term) {
#pragma unroll
  for (int n = 0; n < N; ++n) s[n] = 0.f;
  for (int64_t c0 = threadIdx.x; c0 < cols; c0 += (int64_t)kChain * kLong) {
    const int64_t end = min((int64_t)cols, c0 + (int64_t)kChain * kLong);
    float run[N] = {};
    for (int64_t c = c0; c < end; c += kLong) term(c, run);
#pragma unroll
    for (int n = 0; n < N; ++n) s[n] += run[n];
  }
}

template <typename T>
__global__ __launch_bounds__(kLong) void norm_long_fwd_kernel(const T* __restrict__ x, int64_t ldx, int cols, Params P, float eps, T* __restrict__ y,
                                                              float* __restrict__ mean_out, float* __restrict__ rstd_out, uint8_t* __restrict__ q,
                                                              int64_t ldq, uint8_t* __restrict__ scale, int64_t lds) {
  __shared__ float red[kLong / 64];
  const int64_t row = blockIdx.x;
  const T* xr = x + row * ldx;
  float s[1];
  lane_sums(cols, s, [&](int64_t c, float (&run)[1]) { run[0] += (float)xr[c]; });
  const float mean = block_sum(s[0], red) / (float)cols;
  lane_sums(cols, s, [&](int64_t c, float (&run)[1]) {
    const float d = (float)xr[c] - mean;
    run[0] = fmaf(d, d, run[0]);
  });
  const float rstd = 1.f / sqrtf(block_sum(s[0], red) / (float)cols + eps);
  for (int64_t c = threadIdx.x; c < cols; c += kLong) {
    const float w = P.w ? load_dt(P.w, P.wdt, c) : 1.f, b = P.b ? load_dt(P.b, P.bdt, c) : 0.f;
    y[row * cols + c] = (T)fmaf(((float)xr[c] - mean) * rstd, w, b);
  }
  if (threadIdx.x == 0 && mean_out) mean_out[row] = mean, rstd_out[row] = rstd;
  if (q) {
    // whole groups of sixteen lanes stay together: the bound is the pitch of the scale row, in blocks
    for (int64_t kb = threadIdx.x >> 4; kb < lds; kb += kLong / 16) {
      const int64_t col = kb * 128 + (threadIdx.x & 15) * 8;
      float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (col < cols) load8(xr + col, (int)min((int64_t)8, cols - col), v);
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = fmaxf(m, finite_abs(v[i]));
      const int byte = act8_byte(row16_max(m));
      if (col < ldq) *(v2i*)(q + row * ldq + col) = act8_bytes(v, inv_pow2_of_byte(byte));
      if ((threadIdx.x & 15) == 0) scale[row * lds + kb] = (uint8_t)byte;
    }
  }
}

template <typename T, bool ACT8>
__device__ __forceinline__ float long_x(const T* xr, const uint8_t* qr, const uint8_t* sr, int64_t c) {
  if constexpr (ACT8) return __builtin_amdgcn_cvt_f32_fp8(qr[c], 0) * pow2_of_byte(sr[c >> 7]);
  else return (float)xr[c];
}

template <typename T, bool ACT8>
__global__ __launch_bounds__(kLong) void norm_long_bwd_kernel(const T* __restrict__ x, int64_t ldx, const uint8_t* __restrict__ q, int64_t ldq,
                                                              const uint8_t* __restrict__ scale, int64_t lds, const T* __restrict__ dy, int cols, Params P,
                                                              const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
                                                              T* __restrict__ dx) {
  __shared__ float red[kLong / 64];
  const int64_t row = blockIdx.x;
  const T *xr = ACT8 ? nullptr : x + row * ldx, *dr = dy + row * cols;
  const uint8_t *qr = ACT8 ? q + row * ldq : nullptr, *sr = ACT8 ? scale + row * lds : nullptr;
  const float mean = mean_in[row], rstd = rstd_in[row];
  float s[2];
  lane_sums(cols, s, [&](int64_t c, float (&run)[2]) {
    const float g = (float)dr[c] * (P.w ? load_dt(P.w, P.wdt, c) : 1.f);
    run[0] += g;
    run[1] = fmaf(g, (long_x<T, ACT8>(xr, qr, sr, c) - mean) * rstd, run[1]);
  });
  const float mg = block_sum(s[0], red) / (float)cols, mgh = block_sum(s[1], red) / (float)cols;
  for (int64_t c = threadIdx.x; c < cols; c += kLong) {
    const float g = (float)dr[c] * (P.w ? load_dt(P.w, P.wdt, c) : 1.f);
    dx[row * cols + c] = (T)(rstd * (g - mg - (long_x<T, ACT8>(xr, qr, sr, c) - mean) * rstd * mgh));
  }
}

// the column sums of long rows: 256 columns and every gridDim.y-th row a workgroup
template <typename T, bool ACT8>
__global__ __launch_bounds__(256) void norm_long_cols_kernel(const T* __restrict__ x, int64_t ldx, const uint8_t* __restrict__ q, int64_t ldq,
                                                             const uint8_t* __restrict__ scale, int64_t lds, const T* __restrict__ dy, int64_t rows,
                                                             int cols, const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
                                                             float* __restrict__ part) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= cols) return;
  float aw = 0.f, ab = 0.f;
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
    const float d = (float)dy[r * cols + c];
    aw = fmaf(d, (long_x<T, ACT8>(ACT8 ? nullptr : x + r * ldx, q + r * ldq, scale + r * lds, c) - mean_in[r]) * rstd_in[r], aw);
    ab += d;
  }
  part[((int64_t)blockIdx.y * 2) * cols + c] = aw;
  part[((int64_t)blockIdx.y * 2 + 1) * cols + c] = ab;
}

// Lanes a row and chunks a lane: the smallest product that covers the row.  (TPR, NCH, threads of a workgroup)
#define HCM_NORM_SHAPES(X)                                                                                   \
  X(16, 1, 256) X(16, 3, 256) X(64, 1, 256) X(64, 2, 256) X(64, 4, 256) X(256, 2, 256) X(256, 4, 256) X(512, 4, 512)

// what the widest shape holds; rows of 16385 walk memory (4096 rows of bf16, forward: 54 us at 16384 columns, 130 at 16385)
constexpr int kRegCols = 16384;

// slices of the rows in norm_long_cols_kernel
int long_slices(int64_t rows) { return (int)std::max(std::min(rows, (int64_t)32), (rows + kChain - 1) / kChain); }

// Workgroups of the backward pass: as many as run at once; each costs a partial row of 2 * cols floats, so wide rows get fewer (8192 x 8000 in
// fp32: 116 us with 256, 126 with 512).  Rows that would make over kChain trips are further launches, one behind the other: as more workgroups
// in one launch they would be walked in strides that memory likes less (300000 x 4096 in bf16: 2310 -> 2630 us).
struct BwdPlan { int cap, per; };        // workgroups of a launch at most, rows side by side in one
BwdPlan bwd_plan(int cols) {
  int per = 1;
#define X(TPR, NCH, NT) if (cols <= TPR * NCH * 8 && per == 1 && NT / TPR > 1) per = NT / TPR;
  HCM_NORM_SHAPES(X)
#undef X
  return {cols <= 384 ? 1024 : cols <= 4096 ? 512 : 256, per};
}
int64_t bwd_launch_rows(const BwdPlan& p) { return (int64_t)p.cap * p.per * kChain; }
int bwd_groups(const BwdPlan& p, int64_t rows) { return (int)std::min((rows + p.per - 1) / p.per, (int64_t)p.cap); }
// partial rows of all launches
int bwd_parts(int64_t rows, int cols) {
  const BwdPlan p = bwd_plan(cols);
  const int64_t chunk = bwd_launch_rows(p);
  return (int)(rows / chunk * p.cap + bwd_groups(p, rows % chunk));
}

template <typename T>
int fwd(const void* x, int64_t ldx, int64_t rows, int cols, Params P, float eps, void* y, float* mean, float* rstd, uint8_t* q, int64_t ldq,
        uint8_t* scale, int64_t lds, hipStream_t st) {
#define X(TPR, NCH, NT)                                                                                                                          \
  if (cols <= TPR * NCH * 8) {                                                                                                                   \
    const int64_t need = (rows + NT / TPR - 1) / (NT / TPR), cap = 256 * ((cols <= 384 ? 2048 : 1024) / NT);                                                            \
    norm_fwd_kernel<T, TPR, NCH, NT><<<(uint32_t)(need < cap ? need : cap), NT, 0, st>>>((const T*)x, ldx, (uint32_t)rows, cols, P, eps, (T*)y, mean, \
                                                                                        rstd, q, ldq, scale, lds);                               \
    HCM_CHECK_LAUNCH();                                                                                                                          \
    return 0;                                                                                                                                    \
  }
  HCM_NORM_SHAPES(X)
#undef X
  norm_long_fwd_kernel<T><<<(uint32_t)rows, kLong, 0, st>>>((const T*)x, ldx, cols, P, eps, (T*)y, mean, rstd, q, ldq, scale, lds);
  HCM_CHECK_LAUNCH();
  return 0;
}

template <typename T, bool ACT8>
int bwd(const void* x, int64_t ldx, const uint8_t* q, int64_t ldq, const uint8_t* scale, int64_t lds, const void* dy, int64_t rows, int cols, Params P,
        const float* mean, const float* rstd, void* dx, float* part, int& parts, hipStream_t st) {
#define X(TPR, NCH, NT)                                                                                                                            \
  if (cols <= TPR * NCH * 8) {                                                                                                                     \
    const BwdPlan p = bwd_plan(cols);                                                                                                              \
    parts = 0;                                                                                                                                     \
    for (int64_t r = 0; r < rows; r += bwd_launch_rows(p)) {                                                                                       \
      const int64_t n = std::min(rows - r, bwd_launch_rows(p));                                                                                    \
      const int groups = bwd_groups(p, n);                                                                                                         \
      norm_bwd_kernel<T, ACT8, TPR, NCH, NT><<<groups, NT, 0, st>>>(ACT8 ? nullptr : (const T*)x + r * ldx, ldx, ACT8 ? q + r * ldq : nullptr, ldq,\
                                                                    ACT8 ? scale + r * lds : nullptr, lds, (const T*)dy + r * cols, (uint32_t)n, cols,\
                                                                    P, mean + r, rstd + r, (T*)dx + r * cols, part + (int64_t)parts * 2 * cols);   \
      HCM_CHECK_LAUNCH();                                                                                                                          \
      parts += groups;                                                                                                                             \
    }                                                                                                                                              \
    return 0;                                                                                                                                      \
  }
  HCM_NORM_SHAPES(X)
#undef X
  norm_long_bwd_kernel<T, ACT8><<<(uint32_t)rows, kLong, 0, st>>>((const T*)x, ldx, q, ldq, scale, lds, (const T*)dy, cols, P, mean, rstd, (T*)dx);
  HCM_CHECK_LAUNCH();
  parts = long_slices(rows);
  norm_long_cols_kernel<T, ACT8><<<dim3((cols + 255) / 256, parts), 256, 0, st>>>((const T*)x, ldx, q, ldq, scale, lds, (const T*)dy, rows, cols, mean, rstd,
                                                                                  part);
  HCM_CHECK_LAUNCH();
  return 0;
}

// what launches of fewer than 2^32 threads an axis cover: kLong threads a row that is too long for registers
bool size_ok(int64_t rows, int cols) {
  return rows > 0 && rows < (1ll << 31) - 8192 && cols > 0 && cols < (1 << 27) && (cols <= kRegCols || rows < (1ll << 32) / kLong);
}
bool dt_ok(int d) { return d == kF32 || d == kBF16 || d == kF16; }
bool pitches_ok(int cols, int64_t ldq, int64_t lds) { return ldq == hcm_act8_pitch(cols) && lds == hcm_act8_scale_pitch(cols); }

}  // namespace

extern "C" {

int hcm_layer_norm_forward(const void* x, int dtype, int64_t rows, int cols, int64_t ldx, const void* w, int w_dtype, const void* b, int b_dtype,
                           float eps, void* y, float* mean, float* rstd, uint8_t* q, int64_t ldq, uint8_t* scale, int64_t lds, hcm_stream_t stream) {
  if (!x || !y || !size_ok(rows, cols) || ldx < cols || !dt_ok(dtype) || !dt_ok(w_dtype) ||
      !dt_ok(b_dtype) || (!mean != !rstd) || (!q != !scale) || (q && (!pitches_ok(cols, ldq, lds) || ((uintptr_t)q & 15))))
    return (int)hipErrorInvalidValue;
  const Params P = {w, b, w_dtype, b_dtype};
  hipStream_t st = (hipStream_t)stream;
  if (dtype == kF32) return fwd<float>(x, ldx, rows, cols, P, eps, y, mean, rstd, q, ldq, scale, lds, st);
  if (dtype == kBF16) return fwd<__bf16>(x, ldx, rows, cols, P, eps, y, mean, rstd, q, ldq, scale, lds, st);
  return fwd<_Float16>(x, ldx, rows, cols, P, eps, y, mean, rstd, q, ldq, scale, lds, st);
}

size_t hcm_layer_norm_backward_workspace_bytes(int64_t rows, int cols) {
  if (rows <= 0 || cols <= 0) return 0;
  const int64_t parts = cols > kRegCols ? long_slices(rows) : bwd_parts(rows, cols);
  return (size_t)parts * 2 * cols * sizeof(float);
}

int hcm_layer_norm_backward(const void* x, int64_t ldx, const uint8_t* q, int64_t ldq, const uint8_t* scale, int64_t lds, const void* dy, int dtype,
                            int64_t rows, int cols, const void* w, int w_dtype, const float* mean, const float* rstd, void* dx, void* dw, void* db,
                            int b_dtype, void* workspace, size_t workspace_bytes, hcm_stream_t stream) {
  if ((!x == !q) || (!q != !scale) || !dy || !mean || !rstd || !dx || !workspace || !size_ok(rows, cols) ||
      (x && ldx < cols) || !dt_ok(dtype) || !dt_ok(w_dtype) || !dt_ok(b_dtype) ||
      (q && (!pitches_ok(cols, ldq, lds) || ((uintptr_t)q & 15))) || workspace_bytes < hcm_layer_norm_backward_workspace_bytes(rows, cols))
    return (int)hipErrorInvalidValue;
  const Params P = {w, nullptr, w_dtype, b_dtype};
  hipStream_t st = (hipStream_t)stream;
  float* part = (float*)workspace;
  int parts = 0, rc;
  if (dtype == kF32)
    rc = q ? bwd<float, true>(x, ldx, q, ldq, scale, lds, dy, rows, cols, P, mean, rstd, dx, part, parts, st)
           : bwd<float, false>(x, ldx, q, ldq, scale, lds, dy, rows, cols, P, mean, rstd, dx, part, parts, st);
  else if (dtype == kBF16)
    rc = q ? bwd<__bf16, true>(x, ldx, q, ldq, scale, lds, dy, rows, cols, P, mean, rstd, dx, part, parts, st)
           : bwd<__bf16, false>(x, ldx, q, ldq, scale, lds, dy, rows, cols, P, mean, rstd, dx, part, parts, st);
  else
    rc = q ? bwd<_Float16, true>(x, ldx, q, ldq, scale, lds, dy, rows, cols, P, mean, rstd, dx, part, parts, st)
           : bwd<_Float16, false>(x, ldx, q, ldq, scale, lds, dy, rows, cols, P, mean, rstd, dx, part, parts, st);
  if (rc || (!dw && !db)) return rc;
  // in two axes: the 32 threads a column would be 2^32 in one for the longest rows
  const int64_t groups = (2ll * cols + 63) / 64;
  norm_reduce_kernel<<<dim3((uint32_t)std::min(groups, (int64_t)1 << 16), (uint32_t)((groups + 65535) >> 16)), 64 * kRedSlices, 0, st>>>(part, parts, cols, dw,
                                                                                                                                     w_dtype, db, b_dtype);
  HCM_CHECK_LAUNCH();
  return 0;
}

}  // extern "C"
