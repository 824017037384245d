// 8-bit activation checkpoints (act8.h has the format): pack, unpack, and the two-way packing of a weight.
//
// Bound by HBM: a pack reads x and writes a byte a value and a byte a block, an unpack the reverse; the arithmetic (a maximum
// over 128 values, a multiply and a conversion each) hides under the loads.  One block of 128 = sixteen lanes of eight values:
// the maximum is four DPP steps inside a row of lanes, a 16-bit input is read in 16-byte pieces.
#include "act8.h"
#include "../../include/hcmoco_hip.h"

namespace {

using namespace hcm;

constexpr int kThreads = 256, kGroups = kThreads / 16, kUnroll = 4;

// Sixteen-lane group `g` of the grid takes blocks g, g + G, ... (kUnroll of them, all loaded before the first is used): block
// numbers run along the rows, so neighbouring groups touch neighbouring memory.
struct Cell { uint32_t row, kb; };
__device__ __forceinline__ Cell cell_of(uint32_t id, uint32_t kblocks) { return {id / kblocks, id % kblocks}; }

template <typename T>
__global__ __launch_bounds__(kThreads) void act8_pack_kernel(const T* __restrict__ x, int64_t ldx, int cols, uint32_t kblocks, uint32_t cells,
                                                             uint8_t* __restrict__ q, int64_t ldq, uint8_t* __restrict__ scale, int64_t lds) {
  const int lane = threadIdx.x & 15;
  const uint32_t first = blockIdx.x * (kGroups * kUnroll) + (threadIdx.x >> 4);
  float v[kUnroll][8];
  Cell c[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const uint32_t id = first + u * kGroups;
    c[u] = cell_of(min(id, cells - 1), kblocks);
    const int col = (int)c[u].kb * 128 + lane * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[u][i] = 0.f;
    if (id < cells && col < cols) load8(x + (int64_t)c[u].row * ldx + col, cols - col, v[u]);
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const uint32_t id = first + u * kGroups;
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, finite_abs(v[u][i]));
    m = row16_max(m);
    const int byte = act8_byte(m);
    const v2i out = act8_bytes(v[u], inv_pow2_of_byte(byte));
    const int col = (int)c[u].kb * 128 + lane * 8;
    if (id < cells) {
      if (col < ldq) *(v2i*)(q + (int64_t)c[u].row * ldq + col) = out;     // ldq: a multiple of 16, the pad is zero
      if (lane == 0) scale[(int64_t)c[u].row * lds + c[u].kb] = (uint8_t)byte;
      // the pad of the scale row (its pitch is a multiple of four: read as dwords by the products): 1.0
      else if (c[u].kb == kblocks - 1 && lane < (int)(lds - kblocks) + 1) scale[(int64_t)c[u].row * lds + c[u].kb + lane] = 127;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void act8_unpack_kernel(const uint8_t* __restrict__ q, int64_t ldq, const uint8_t* __restrict__ scale,
                                                               int64_t lds, int cols, uint32_t kblocks, uint32_t cells, T* __restrict__ x,
                                                               float top) {
  const int lane = threadIdx.x & 15;
  const uint32_t first = blockIdx.x * (kGroups * kUnroll) + (threadIdx.x >> 4);
  v2i v[kUnroll];
  int byte[kUnroll];
  Cell c[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const uint32_t id = first + u * kGroups;
    c[u] = cell_of(min(id, cells - 1), kblocks);
    const int col = min((int)c[u].kb * 128 + lane * 8, (int)ldq - 8);
    v[u] = *(const v2i*)(q + (int64_t)c[u].row * ldq + col);
    byte[u] = scale[(int64_t)c[u].row * lds + c[u].kb];
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const uint32_t id = first + u * kGroups;
    const int col = (int)c[u].kb * 128 + lane * 8;
    if (id >= cells || col >= cols) continue;
    float f[8];
    act8_values(v[u], pow2_of_byte(byte[u]), f);
    // the block's largest value may round up past the type's own largest (65504 -> 65536): it stays finite
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = f[i] > top ? top : f[i] < -top ? -top : f[i];
    store8(x + (int64_t)c[u].row * cols + col, cols - col, f);
  }
}

// A weight block of 128 x 128: the maximum over the block, then q as it lies [rows, cols] and transposed [cols, rows] (the
// product of the backward pass contracts over the rows).  The transposed copy goes through LDS so that both are written in
// 16-byte pieces.  One workgroup a block: a weight has hundreds of them, and a small one is latency anyway.
template <typename T>
__global__ __launch_bounds__(256) void fp8_weight_kernel(const T* __restrict__ w, int64_t ldw, int rows, int cols, uint8_t* __restrict__ q, int64_t ldq,
                                                         uint8_t* __restrict__ scale, int64_t lds, uint8_t* __restrict__ qt, int64_t ldqt,
                                                         uint8_t* __restrict__ scale_t, int64_t ldst) {
  __shared__ float part[4];
  __shared__ __attribute__((aligned(16))) uint8_t tile[128][128 + 16];
  const int t = threadIdx.x, lane = t & 15, r0 = blockIdx.y * 128, c0 = blockIdx.x * 128;
  float v[8][8];
  float m = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int row = r0 + j * 16 + (t >> 4), col = c0 + lane * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[j][i] = 0.f;
    if (row < rows && col < cols) load8(w + (int64_t)row * ldw + col, cols - col, v[j]);
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, finite_abs(v[j][i]));
  }
  m = wave_max(m);
  if ((t & 63) == 0) part[t >> 6] = m;
  __syncthreads();
  const int byte = act8_byte(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])));
  const float inv = inv_pow2_of_byte(byte);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int lr = j * 16 + (t >> 4), row = r0 + lr, col = c0 + lane * 8;
    const v2i out = act8_bytes(v[j], inv);
    if (row < rows && col < ldq) *(v2i*)(q + (int64_t)row * ldq + col) = out;
    *(v2i*)&tile[lr][lane * 8] = out;
  }
  if (t == 0) {
    scale[(int64_t)blockIdx.y * lds + blockIdx.x] = (uint8_t)byte;
    scale_t[(int64_t)blockIdx.x * ldst + blockIdx.y] = (uint8_t)byte;
  }
  // the pads of the scale rows (pitch a multiple of four): 1.0
  if (t < 3 && blockIdx.x == gridDim.x - 1 && blockIdx.x + 1 + t < lds) scale[(int64_t)blockIdx.y * lds + blockIdx.x + 1 + t] = 127;
  if (t < 3 && blockIdx.y == gridDim.y - 1 && blockIdx.y + 1 + t < ldst) scale_t[(int64_t)blockIdx.x * ldst + blockIdx.y + 1 + t] = 127;
  __syncthreads();
  // thread -> column c of the block and half of its rows, sixteen rows a store
  const int c = t & 127, half = t >> 7, col = c0 + c;
  if (col < cols) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int lr = half * 64 + j * 16;
      v4i o;
#pragma unroll
      for (int d = 0; d < 4; ++d)
        o[d] = tile[lr + 4 * d][c] | tile[lr + 4 * d + 1][c] << 8 | tile[lr + 4 * d + 2][c] << 16 | (int)((uint32_t)tile[lr + 4 * d + 3][c] << 24);
      if (r0 + lr < ldqt) *(v4i*)(qt + (int64_t)col * ldqt + r0 + lr) = o;
    }
  }
}

// rows * kb < 2^30: four threads a block of 128, and a launch has fewer than 2^32
bool shape_ok(int64_t rows, int cols, int64_t ldq, int64_t lds) {
  const int64_t kb = ((int64_t)cols + 127) / 128;
  return rows > 0 && cols > 0 && cols <= INT32_MAX - 128 && rows <= INT32_MAX && rows * kb < (1ll << 30) && ldq == ((int64_t)cols + 15) / 16 * 16 && lds == (kb + 3) / 4 * 4;
}
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

extern "C" {

int64_t hcm_act8_pitch(int64_t cols) { return (cols + 15) / 16 * 16; }
int64_t hcm_act8_scale_pitch(int64_t cols) { return ((cols + 127) / 128 + 3) / 4 * 4; }

int hcm_act8_pack(const void* x, int dtype, int64_t rows, int cols, int64_t ldx, uint8_t* q, int64_t ldq, uint8_t* scale, int64_t lds,
                  hcm_stream_t stream) {
  if (!x || !q || !scale || !shape_ok(rows, cols, ldq, lds) || ldx < cols || !aligned16(q)) return (int)hipErrorInvalidValue;
  const uint32_t kb = (cols + 127) / 128, cells = (uint32_t)(rows * kb), grid = (cells + kGroups * kUnroll - 1) / (kGroups * kUnroll);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == kF32) act8_pack_kernel<float><<<grid, kThreads, 0, st>>>((const float*)x, ldx, cols, kb, cells, q, ldq, scale, lds);
  else if (dtype == kBF16) act8_pack_kernel<__bf16><<<grid, kThreads, 0, st>>>((const __bf16*)x, ldx, cols, kb, cells, q, ldq, scale, lds);
  else if (dtype == kF16) act8_pack_kernel<_Float16><<<grid, kThreads, 0, st>>>((const _Float16*)x, ldx, cols, kb, cells, q, ldq, scale, lds);
  else return (int)hipErrorInvalidValue;
  HCM_CHECK_LAUNCH();
  return 0;
}

int hcm_act8_unpack(const uint8_t* q, int64_t ldq, const uint8_t* scale, int64_t lds, int64_t rows, int cols, void* x, int dtype,
                    hcm_stream_t stream) {
  if (!x || !q || !scale || !shape_ok(rows, cols, ldq, lds) || !aligned16(q)) return (int)hipErrorInvalidValue;
  const uint32_t kb = (cols + 127) / 128, cells = (uint32_t)(rows * kb), grid = (cells + kGroups * kUnroll - 1) / (kGroups * kUnroll);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == kF32) act8_unpack_kernel<float><<<grid, kThreads, 0, st>>>(q, ldq, scale, lds, cols, kb, cells, (float*)x, 3.4028234663852886e38f);
  else if (dtype == kBF16) act8_unpack_kernel<__bf16><<<grid, kThreads, 0, st>>>(q, ldq, scale, lds, cols, kb, cells, (__bf16*)x, 3.3895313892515355e38f);
  else if (dtype == kF16) act8_unpack_kernel<_Float16><<<grid, kThreads, 0, st>>>(q, ldq, scale, lds, cols, kb, cells, (_Float16*)x, 65504.f);
  else return (int)hipErrorInvalidValue;
  HCM_CHECK_LAUNCH();
  return 0;
}

int hcm_fp8_weight_pack(const void* w, int dtype, int rows, int cols, int64_t ldw, uint8_t* q, int64_t ldq, uint8_t* scale, int64_t lds,
                        uint8_t* qt, int64_t ldqt, uint8_t* scale_t, int64_t ldst, hcm_stream_t stream) {
  if (!w || !q || !scale || !qt || !scale_t || ldw < cols || !shape_ok(rows, cols, ldq, lds) || !shape_ok(cols, rows, ldqt, ldst) || !aligned16(q) ||
      !aligned16(qt) || rows > 65535 * 128)
    return (int)hipErrorInvalidValue;
  const dim3 grid((cols + 127) / 128, (rows + 127) / 128);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == kF32) fp8_weight_kernel<float><<<grid, 256, 0, st>>>((const float*)w, ldw, rows, cols, q, ldq, scale, lds, qt, ldqt, scale_t, ldst);
  else if (dtype == kBF16) fp8_weight_kernel<__bf16><<<grid, 256, 0, st>>>((const __bf16*)w, ldw, rows, cols, q, ldq, scale, lds, qt, ldqt, scale_t, ldst);
  else if (dtype == kF16) fp8_weight_kernel<_Float16><<<grid, 256, 0, st>>>((const _Float16*)w, ldw, rows, cols, q, ldq, scale, lds, qt, ldqt, scale_t, ldst);
  else return (int)hipErrorInvalidValue;
  HCM_CHECK_LAUNCH();
  return 0;
}

}  // extern "C"
