// Products of 8-bit blocks (act8.h has the format):  y[m][n] = sum_k X[m][k] W[n][k] (+ bias[n]),  X [M, K] with a scale for 128
// values of a row, W [N, K] with a scale for each block of 128 x 128.  Forward: X = Q(x), W = Q(weight); data gradient:
// X = Q(dy), W = the transposed copy of Q(weight).
//
// A block of 128 along k is ONE scaled matrix instruction (v_mfma_scale_f32_16x16x128_f8f6f4), and the format's scale byte is
// its scale operand: the scales cost no arithmetic.  Its two operands only have to agree on the order of k, so a lane takes
// the 16-byte pieces g and g + 4 of its row (g = lane / 16).  W is the A operand, so that a lane ends up with neighbouring
// columns of y: four, a 16-byte piece of fp32 (WIDE); for a 16-bit y the A rows of two instructions are interleaved so that they are eight.
//
// Precision.  Every 8-bit matrix instruction of this chip adds its products in groups of eight neighbouring k, aligned to the
// group's largest product, and drops what lies below 2^-13 of it (measured on single products, the same for the scaled form and for
// 16x16x32; the sums of groups are full fp32): 2e-5 .. 7e-5 of the result's norm on random data.  That is under the rounding of
// a 16-bit y (2^-9, 2^-12), and it is over that of an fp32 one, so y in fp32 takes the WIDE form: the 8-bit values are widened to bf16
// on their way from LDS -- exact in the range of scales that act8.h states, the scales included, by v_cvt_scalef32_pk_bf16_fp8 -- and multiplied
// by v_mfma_f32_16x16x32_bf16, whose sums are fp32 (1e-8 .. 3e-7 on the same data), at half the rate (8192 x 4096 x 4096: 1.33 PFLOP/s; 2.4 in 8 bits).
#include <cmath>
#include "act8.h"
#include "../../include/hcmoco_hip.h"

namespace {

using namespace hcm;

struct Mm {
  const uint8_t *x, *sx, *w, *sw;
  int64_t ldx, ldsx, ldw, ldsw;
  int M, N, kblocks, ldk;          // ldk: bytes of a row that hold values (the pitch of both operands)
  const void* bias;
  int bias_dt, out_dt;
  void* y;
  float* part;                     // split > 1: [split][M][N] partial sums instead of y
  int split;
};

// Direct loads from memory to LDS, 16 or 4 bytes a lane: lane l's piece lands at lds + l * BYTES, a piece outside the buffer reads as
// zero.  In assembly because the compiler, which cannot tell the two stages apart, would wait for the loads of the next stage before
// every LDS read of this one.  Nothing is written but LDS; whoever reads it waits for vmcnt(0) and a barrier first, and a kernel
// waits for vmcnt(0) before it ends.  (s_nop 4: the wait states between a vector instruction that writes a scalar register, which may stand
// right before, and a load that takes its buffer from it; the compiler does not look for them in here.)
typedef v4i rsrc_t;
__device__ __forceinline__ rsrc_t make_rsrc(const void* p, int bytes) {
  const uint64_t a = (uint64_t)p;
  return rsrc_t{(int)(uint32_t)a, (int)((uint32_t)(a >> 32) & 0xffffu), bytes, 0x00020000};
}
template <int BYTES>
__device__ __forceinline__ void load_lds(rsrc_t r, uint32_t lds, int off) {
  if constexpr (BYTES == 16)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(off), "s"(r) : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(lds), "v"(off), "s"(r) : "memory", "m0");
}
__device__ __forceinline__ uint32_t lds_addr(const void* p) { return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p; }
// All but the newest N loads of this wave are done, and all of its LDS reads: before a barrier behind which others overwrite what it read.
template <int N = 0>
__device__ __forceinline__ void wait_loads() {
  static_assert(N < 64, "vmcnt");
  __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | (N >> 4) << 14);      // vmcnt(N) lgkmcnt(0)
}
constexpr int kOutside = (int)0x80000000;       // an offset past every buffer used here (they are under 2^31 bytes)

// Workgroups go to the eight XCDs in turn; each XCD gets a run of neighbouring tiles (columns of four row tiles, so
// that 32 workgroups side by side share 4 + 8 row and column panels in its L2; eight by four: 428 against 421 us at 8192^3).
__device__ __forceinline__ void tile_of(int id, int tm, int tn, int& im, int& in) {
  const int total = tm * tn, xcd = id & 7, k = id >> 3, base = total >> 3, rem = total & 7;
  const int t = xcd * base + min(xcd, rem) + k;
  const int band = 4 * tn, b = t / band, in_band = t - b * band, h = min(4, tm - 4 * b);
  in = in_band / h;
  im = 4 * b + (in_band - in * h);
}

// thirty-two 8-bit values (the pieces g and g + 4 of a row) -> four operands of the bf16 instruction, times a power of two
__device__ __forceinline__ void widen(const v8i& q, float scale, v8bf (&out)[4]) {
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const v2bf a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[2 * s], scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[2 * s], scale, true);
    const v2bf c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[2 * s + 1], scale, false),
               d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[2 * s + 1], scale, true);
    out[s] = v8bf{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  }
}
__device__ __forceinline__ v8i join16(const v4i& lo, const v4i& hi) { return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7); }

// eight neighbouring columns of one row
__device__ __forceinline__ void out8(const Mm& P, int m, int n, float (&v)[8]) {
  const int left = P.N - n;
  if (m >= P.M || left <= 0) return;
  if (P.part) {
    store8(P.part + ((int64_t)blockIdx.z * P.M + m) * P.N + n, left, v);
    return;
  }
  if (P.bias) {
    float b[8];
    load8_dt(P.bias, P.bias_dt, n, left, b);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += b[i];
  }
  const int64_t at = (int64_t)m * P.N + n;
  if (P.out_dt == kF32) store8((float*)P.y + at, left, v);
  else if (P.out_dt == kBF16) store8((__bf16*)P.y + at, left, v);
  else store8((_Float16*)P.y + at, left, v);
}

// four neighbouring columns of one row, fp32
__device__ __forceinline__ void out4(const Mm& P, int m, int n, v4f v) {
  const int left = P.N - n;
  if (m >= P.M || left <= 0) return;
  float* y = P.part ? P.part + ((int64_t)blockIdx.z * P.M + m) * P.N + n : (float*)P.y + (int64_t)m * P.N + n;
  if (left >= 4) {
    if (P.bias && !P.part)
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] += load_dt(P.bias, P.bias_dt, n + r);
    __builtin_memcpy(y, &v, 16);
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (r < left) y[r] = v[r] + (P.bias && !P.part ? load_dt(P.bias, P.bias_dt, n + r) : 0.f);
  }
}

// BN columns x BM rows of y a workgroup, WN x WM waves of TN x TM tiles of 16 x 16.  S LDS stages of (BN + BM) x 128 bytes in a ring;
// one barrier a block of k, behind which the loads of the stage S - 1 blocks ahead go out between the matrix instructions (all at once
// they block the waves' LDS reads: 480 -> 431 us at 8192^3).  Small tiles run where few workgroups do and a block of k is latency: four
// stages.  The 256 x 256 tile was bound by these loads: 64 KB a block of k a CU take 1.4 us when an XCD's workgroups, in step, all wait for
// the same lines from behind L2, against 1.25 us of matrix instructions and LDS reads.  So each workgroup also touches, two blocks
// ahead, its share of the lines that the XCD's workgroups will want (431 -> 421 us; the loads alone then take 1.15 us a block).  What is
// left is the two together, 1.5 us a block: the matrix pipes are busy 0.93 us of it.  Measured and not kept: four waves of 128 x 128 (spills,
// 632 us), the barrier before the last of the eight tiles with the next block's first fragments read behind it (417 us for twice the code).
template <int BN, int BM, int WN, int WM, int S, bool WIDE>
__global__ __launch_bounds__(WN * WM * 64) void fp8_tile_kernel(const Mm P) {
  constexpr int NT = WN * WM * 64, TN = BN / WN / 16, TM = BM / WM / 16;
  constexpr int LW = BN * 8 / NT, LX = BM * 8 / NT;        // load instructions of a wave a stage
  constexpr int PER = (2 * (LW + LX) + TN - 1) / TN;       // of them behind each of the first tiles: all are out at half time
  constexpr bool TOUCH = BN == 256 && BM == 256;
  static_assert(TN % 2 == 0 && LW >= 1 && LX >= 1 && BN * 8 % NT == 0 && BM * 8 % NT == 0, "tile");
  __shared__ __attribute__((aligned(128))) uint8_t stage[S][(BN + BM) * 128];
  __shared__ uint32_t sx_stage[2][BM], sw_stage[2][64];    // the scales of four blocks of k, one dword a row of X, one a block of W
  __shared__ uint32_t touched[TOUCH ? 128 : 1];            // never read
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), wn = wave % WN, wm = wave / WN;
  int im, in;
  tile_of(blockIdx.x, (P.M + BM - 1) / BM, (P.N + BN - 1) / BN, im, in);
  const int m0 = im * BM, n0 = in * BN;
  const int per = ((P.kblocks + P.split - 1) / P.split + 3) & ~3;      // whole dwords of scales
  const int k_from = blockIdx.z * per, k_to = min(P.kblocks, k_from + per);

  const uint8_t* wbase = P.w + (int64_t)n0 * P.ldw;
  const uint8_t* xbase = P.x + (int64_t)m0 * P.ldx;
  const int wbytes = (int)(min(P.N - n0, BN) * P.ldw), xbytes = (int)(min(P.M - m0, BM) * P.ldx);

  // Row r of a stage lies at r * 128, its piece c in slot c ^ key(r): eight lanes that read the same piece of eight rows hit eight
  // different slots.  A load instruction of a wave fills eight rows; which piece a lane fetches is what places it.
  const int r8 = lane >> 3, slot = lane & 7;
  rsrc_t rw, rx;
  int left = 0;
  auto aim = [&](int kb) {
    const int64_t ko = (int64_t)kb * 128;
    rw = make_rsrc(wbase + ko, wbytes - (int)ko);
    rx = make_rsrc(xbase + ko, xbytes - (int)ko);
    left = P.ldk - kb * 128;       // pieces past the row's end would be the next row's: sent outside, they read as zero
  };
  auto issue = [&](int buf, int j) {
    if (j < LW) {
      const int rg = wave + j * (NT / 64), r = rg * 8 + r8;                     // W rows: key (r & 3) | (r >> 3 & 1) << 2, WIDE r & 7
      const int c = slot ^ (WIDE ? r8 : (r8 & 3) | ((rg & 1) << 2));
      load_lds<16>(rw, lds_addr(&stage[buf][rg * 1024]), c * 16 < left ? r * (int)P.ldw + c * 16 : kOutside);
    } else {
      const int rg = wave + (j - LW) * (NT / 64), r = rg * 8 + r8;              // X rows: key r & 7
      const int c = slot ^ r8;
      load_lds<16>(rx, lds_addr(&stage[buf][(BN + rg * 8) * 128]), c * 16 < left ? r * (int)P.ldx + c * 16 : kOutside);
    }
  };
  const rsrc_t rs = make_rsrc(P.sx + (int64_t)m0 * P.ldsx, (int)(min(P.M - m0, BM) * P.ldsx));
  const int wblocks = (min(P.N - n0, BN) + 127) / 128;
  const rsrc_t rsw = make_rsrc(P.sw + (int64_t)(n0 / 128) * P.ldsw, wblocks * (int)P.ldsw);
  auto issue_scales = [&](int kq) {          // blocks 4 kq .. 4 kq + 3; rows past the end read as zero, their sums are not stored
#pragma unroll
    for (int j = 0; j < (BM + NT - 1) / NT; ++j) {
      const int r0 = (wave + j * (NT / 64)) * 64;
      if (r0 < BM) load_lds<4>(rs, lds_addr(&sx_stage[kq & 1][r0]), (r0 + lane) * (int)P.ldsx + kq * 4);
    }
    if (wave == NT / 64 - 1) load_lds<4>(rsw, lds_addr(sw_stage[kq & 1]), lane < wblocks ? lane * (int)P.ldsw + kq * 4 : kOutside);
  };

  const int i = lane & 15, g = lane >> 4;
  const int frag = (g ^ (i & 7)) << 4;
  int wrow[TN], xrow[TM];
#pragma unroll
  for (int a = 0; a < TN; ++a) wrow[a] = (wn * TN * 16 + (WIDE ? a * 16 + i : 32 * (a >> 1) + (i >> 2) * 8 + (a & 1) * 4 + (i & 3))) * 128 + frag;
#pragma unroll
  for (int b = 0; b < TM; ++b) xrow[b] = (BN + (wm * TM + b) * 16 + i) * 128 + frag;
  v4f acc[TN][TM];
#pragma unroll
  for (int a = 0; a < TN; ++a)
#pragma unroll
    for (int b = 0; b < TM; ++b) acc[a][b] = v4f{0.f, 0.f, 0.f, 0.f};

  uint32_t sx4[TM], sw4 = 0;
  auto begin = [&](int kb) {       // what comes before the loads of block kb's stage; past the end they go outside
    if (kb < k_to && (kb & 3) == 0) issue_scales(kb >> 2);
    aim(min(kb, k_to - 1));
    if (kb >= k_to) left = 0;
  };
  if (k_from < k_to)
    for (int p = 0; p < S - 1; ++p) {
      begin(k_from + p);
#pragma unroll
      for (int j = 0; j < LW + LX; ++j) issue(p, j);
    }
  int buf = 0;
  for (int kb = k_from; kb < k_to; ++kb, buf = buf + 1 == S ? 0 : buf + 1) {
    wait_loads<(S - 2) * (LW + LX)>();       // this wave's pieces of the stage have landed (its scales went out before them)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();            // everybody's have, and nobody reads the stage before it any more
    asm volatile("" ::: "memory");
    if ((kb & 3) == 0) {
#pragma unroll
      for (int b = 0; b < TM; ++b) sx4[b] = sx_stage[(kb >> 2) & 1][(wm * TM + b) * 16 + i];
      sw4 = __builtin_amdgcn_readfirstlane(sw_stage[(kb >> 2) & 1][wn * TN * 16 / 128]);
    }
    begin(kb + S - 1);
    const int next = buf == 0 ? S - 1 : buf - 1;
    if constexpr (TOUCH) {
      // of the four row tiles and eight column tiles that run side by side on an XCD: a quarter of this tile's W rows, an eighth of its X rows
      if (wave < 2 && kb + 2 < k_to) {
        const int r = wave ? (im & 3) * (BN / 4) + (lane & (BN / 4 - 1)) : (in & 7) * (BM / 8) + (lane & (BM / 8 - 1));
        if (wave) load_lds<4>(make_rsrc(wbase, wbytes), lds_addr(touched + 64), r * (int)P.ldw + (kb + 2) * 128);
        else load_lds<4>(make_rsrc(xbase, xbytes), lds_addr(touched), r * (int)P.ldx + (kb + 2) * 128);
      }
    }
    const int sh = (kb & 3) * 8, sw = (sw4 >> sh) & 255;
    int sx[TM];
#pragma unroll
    for (int b = 0; b < TM; ++b) sx[b] = (sx4[b] >> sh) & 255;
    const uint8_t* s = stage[buf];
    v8i xf[TM];
    v8bf xw[WIDE ? TM : 1][4];
#pragma unroll
    for (int b = 0; b < TM; ++b) {
      xf[b] = join16(*(const v4i*)(s + xrow[b]), *(const v4i*)(s + (xrow[b] ^ 64)));
      if constexpr (WIDE) widen(xf[b], pow2_of_byte(sx[b]), xw[b]);
    }
#pragma unroll
    for (int a = 0; a < TN; ++a) {
      const v8i wf = join16(*(const v4i*)(s + wrow[a]), *(const v4i*)(s + (wrow[a] ^ 64)));
      if constexpr (WIDE) {
        v8bf ww[4];
        widen(wf, pow2_of_byte(sw), ww);
#pragma unroll
        for (int b = 0; b < TM; ++b)
#pragma unroll
          for (int q = 0; q < 4; ++q) acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ww[q], xw[b][q], acc[a][b], 0, 0, 0);
      } else {
#pragma unroll
        for (int b = 0; b < TM; ++b)
          acc[a][b] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf, xf[b], acc[a][b], 0, 0, 0, sw, 0, sx[b]);
      }
#pragma unroll
      for (int j = a * PER; j < (a + 1) * PER && j < LW + LX; ++j) issue(next, j);
    }
  }
  wait_loads();
  if constexpr (WIDE) {
#pragma unroll
    for (int b = 0; b < TM; ++b)
#pragma unroll
      for (int a = 0; a < TN; ++a) out4(P, m0 + (wm * TM + b) * 16 + i, n0 + (wn * TN + a) * 16 + 4 * g, acc[a][b]);
    return;
  }
#pragma unroll
  for (int b = 0; b < TM; ++b)
#pragma unroll
    for (int a = 0; a < TN; a += 2) {
      float v[8];
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = acc[a][b][r], v[4 + r] = acc[a + 1][b][r];
      out8(P, m0 + (wm * TM + b) * 16 + i, n0 + wn * TN * 16 + 16 * a + 8 * g, v);
    }
}

// A few rows (at most 32): bound by reading W once, and by latency.  Sixteen columns of y a workgroup, the blocks of k dealt to its
// eight waves, each straight from memory to registers (a W row is read in whole lines: eight waves x 128 bytes); the waves' sums
// meet in LDS.  X comes packed (T = uint8_t), or as it is and is packed here by every workgroup (at most kFewBlocks blocks of 128: a
// launch costs more than that); the first workgroup then also writes the packed copy where one is wanted.
constexpr int kFewRows = 32, kFewBlocks = 256, kFewWaves = 8, kFewAhead = 4;

template <typename T, bool WIDE, int MT>
__global__ __launch_bounds__(kFewWaves * 64) void fp8_few_kernel(const Mm P, const T* __restrict__ xraw, int64_t ld_raw, int K, uint8_t* __restrict__ q_out,
                                                                 uint8_t* __restrict__ s_out) {
  constexpr bool PACK = sizeof(T) > 1;
  extern __shared__ __attribute__((aligned(16))) uint8_t dyn[];      // PACK: M rows of (kblocks * 128 + 16) bytes, then M rows of kblocks scales
  __shared__ float red[kFewWaves][MT * 16][17];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), i = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const uint8_t* wr = P.w + (int64_t)min(n0 + i, P.N - 1) * P.ldw;
  const uint8_t* swr = P.sw + (int64_t)(n0 / 128) * P.ldsw;
  const v4i zero = {0, 0, 0, 0};
  auto piece = [&](const uint8_t* row, int at) { return at < P.ldk ? *(const v4i*)(row + at) : zero; };

  v4i wlo[kFewAhead], whi[kFewAhead];
  int sw[kFewAhead];
  auto fetch = [&](int u, int kb) {
    kb = min(kb, P.kblocks - 1);       // past the end: read again, not used
    wlo[u] = piece(wr, kb * 128 + g * 16);
    whi[u] = piece(wr, kb * 128 + 64 + g * 16);
    sw[u] = swr[kb];
  };
#pragma unroll
  for (int u = 0; u < kFewAhead; ++u) fetch(u, wave + u * kFewWaves);

  const int pitch = P.kblocks * 128 + 16;
  uint8_t* xs = dyn + P.M * pitch;
  if constexpr (PACK) {
    const int cells = P.M * P.kblocks;
    for (int c = t >> 4; c < cells; c += kFewWaves * 4) {
      const int row = c / P.kblocks, kb = c - row * P.kblocks, col = kb * 128 + (lane & 15) * 8;
      float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (col < K) load8(xraw + (int64_t)row * ld_raw + col, K - col, v);
      float m = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) m = fmaxf(m, finite_abs(v[e]));
      const int byte = act8_byte(row16_max(m));
      const v2i b = act8_bytes(v, inv_pow2_of_byte(byte));
      *(v2i*)(dyn + row * pitch + col) = b;
      if ((lane & 15) == 0) xs[c] = (uint8_t)byte;
      if (q_out && blockIdx.x == 0) {
        if (col < P.ldx) *(v2i*)(q_out + (int64_t)row * P.ldx + col) = b;
        if ((lane & 15) == 0) s_out[(int64_t)row * P.ldsx + kb] = (uint8_t)byte;
        else if (kb == P.kblocks - 1 && kb + (lane & 15) < P.ldsx) s_out[(int64_t)row * P.ldsx + kb + (lane & 15)] = 127;
      }
    }
    __syncthreads();
  }
  v4f acc[MT];
#pragma unroll
  for (int b = 0; b < MT; ++b) acc[b] = v4f{0.f, 0.f, 0.f, 0.f};
  for (int base = wave; base < P.kblocks; base += kFewAhead * kFewWaves) {
#pragma unroll
    for (int u = 0; u < kFewAhead; ++u) {
      const int kb = base + u * kFewWaves;
      if (kb < P.kblocks) {
        const v8i wf = join16(wlo[u], whi[u]);
        v8bf ww[4];
        if constexpr (WIDE) widen(wf, pow2_of_byte(sw[u]), ww);
#pragma unroll
        for (int b = 0; b < MT; ++b) {
          const int row = min(b * 16 + i, P.M - 1);        // rows past the end repeat the last one and are not stored
          v8i xf;
          int sx;
          if constexpr (PACK) {
            xf = join16(*(const v4i*)(dyn + row * pitch + kb * 128 + g * 16), *(const v4i*)(dyn + row * pitch + kb * 128 + 64 + g * 16));
            sx = xs[row * P.kblocks + kb];
          } else {
            const uint8_t* xr = P.x + (int64_t)row * P.ldx;
            xf = join16(piece(xr, kb * 128 + g * 16), piece(xr, kb * 128 + 64 + g * 16));
            sx = P.sx[(int64_t)row * P.ldsx + kb];
          }
          if constexpr (WIDE) {
            v8bf xw[4];
            widen(xf, pow2_of_byte(sx), xw);
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ww[q], xw[q], acc[b], 0, 0, 0);
          } else {
            acc[b] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf, xf, acc[b], 0, 0, 0, sw[u], 0, sx);
          }
        }
      }
      fetch(u, kb + kFewAhead * kFewWaves);
    }
  }
#pragma unroll
  for (int b = 0; b < MT; ++b)
#pragma unroll
    for (int r = 0; r < 4; ++r) red[wave][b * 16 + i][4 * g + r] = acc[b][r];
  __syncthreads();
  for (int e = t; e < MT * 256; e += kFewWaves * 64) {
    const int m = e >> 4, n = e & 15;
    if (m >= P.M || n0 + n >= P.N) continue;
    float s = 0.f;
#pragma unroll
    for (int z = 0; z < kFewWaves; ++z) s += red[z][m][n];
    if (P.bias) s += load_dt(P.bias, P.bias_dt, n0 + n);
    store_dt(P.y, P.out_dt, (int64_t)m * P.N + n0 + n, s);
  }
}

template <typename T, bool WIDE>
int few(const Mm& P, const T* xraw, int64_t ld_raw, int K, uint8_t* q_out, uint8_t* s_out, hipStream_t st) {
  const size_t lds = sizeof(T) > 1 ? (size_t)P.M * (P.kblocks * 128 + 16) + (size_t)P.M * P.kblocks : 0;
  const uint32_t grid = (P.N + 15) / 16;
  if (P.M <= 16) fp8_few_kernel<T, WIDE, 1><<<grid, kFewWaves * 64, lds, st>>>(P, xraw, ld_raw, K, q_out, s_out);
  else fp8_few_kernel<T, WIDE, 2><<<grid, kFewWaves * 64, lds, st>>>(P, xraw, ld_raw, K, q_out, s_out);
  HCM_CHECK_LAUNCH();
  return 0;
}

// y (or dW and behind it db) = sum over the split of part[z][e], + bias for y.  SL slices of the split side by side, their sums through LDS:
// a small output with a deep split would otherwise be a few waves that wait for one load after the other.
struct Join { const float* part; int split; int64_t stride, n, n2; int N; const void* bias; int bias_dt; void* out; int dt; void* out2; int dt2; };

template <int SL>
__global__ __launch_bounds__(256) void join_kernel(const Join J) {
  constexpr int E = 256 / SL;
  __shared__ float s[SL][E];
  const int lane = threadIdx.x % E, slice = threadIdx.x / E;
  const int64_t e = (int64_t)blockIdx.x * E + lane;
  float a[4] = {0.f, 0.f, 0.f, 0.f};
  if (e < J.n + J.n2) {
    int z = slice;
    for (; z + 3 * SL < J.split; z += 4 * SL)
#pragma unroll
      for (int u = 0; u < 4; ++u) a[u] += J.part[(z + u * SL) * J.stride + e];
    for (; z < J.split; z += SL) a[0] += J.part[z * J.stride + e];
  }
  float sum = (a[0] + a[1]) + (a[2] + a[3]);
  if constexpr (SL > 1) {
    s[slice][lane] = sum;
    __syncthreads();
    if (slice) return;
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < SL; ++i) sum += s[i][lane];
  }
  if (e < J.n) {
    if (J.bias) sum += load_dt(J.bias, J.bias_dt, e % J.N);
    if (J.out) store_dt(J.out, J.dt, e, sum);
  } else if (e < J.n + J.n2 && J.out2) {
    store_dt(J.out2, J.dt2, e - J.n, sum);
  }
}

int join(const Join& J, hipStream_t st) {
  const int64_t n = J.n + J.n2;
  if (J.split >= 16) join_kernel<16><<<(uint32_t)((n + 15) / 16), 256, 0, st>>>(J);
  else join_kernel<1><<<(uint32_t)((n + 255) / 256), 256, 0, st>>>(J);
  HCM_CHECK_LAUNCH();
  return 0;
}

// ---------------------------------------------------------------------------------------------------------------------------------
// Weight gradient from the 8-bit checkpoint:  dW[n][k] = sum_m dy[m][n] X[m][k],  db[n] = sum_m dy[m][n].
//
// q * 2^E is exact in bf16 (act8.h: over nearly all of the range), so X enters v_mfma_f32_16x16x32_bf16 without a rounding; dy enters as the bf16 pieces that hold its type
// exactly (bf16: 1, fp16: 2, fp32: 3), one instruction a piece: only the fp32 sums round.  Both operands lie row by row (m),
// and the instruction wants eight m of one column in a lane: the LDS transpose read (lane p of sixteen points at row p / 4, columns
// 4 (p % 4) .. + 3, and receives column p of the four rows).  128 columns k (one scale a row) x 128 columns n a workgroup.
struct Wg {
  const uint8_t *q, *scale;
  int64_t ldq, lds;
  const void* dy;
  int64_t M;
  int N, K;
  int64_t rows_per_split;         // a multiple of every kernel's ROWS
  float* part;                    // split > 1: [split][stride] partial sums, N * K of dW and N of db; else dw, db
  int64_t stride;
  void *dw, *db;
  int dw_dt, db_dt;
};
constexpr int kWgRows = 64;

typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s* lds_v4s;

// Eight floats -> the bf16 pieces that hold their type exactly (down to bf16's smallest step, 2^-133: values under 2^-110 keep fewer
// bits).  The first piece is cut off, not rounded: the remainder is as exact, and the largest finite values do not round up to infinity.  An
// infinity has no remainder (inf - inf would make its products NaN).
template <int P>
__device__ __forceinline__ void pieces(const float (&v)[8], v8bf (&out)[P]) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t cut = __float_as_uint(v[i]) & 0xffff0000u;
    out[0][i] = __builtin_bit_cast(__bf16, (uint16_t)(cut >> 16));
    r[i] = __builtin_isinf(v[i]) ? 0.f : v[i] - __uint_as_float(cut);
  }
#pragma unroll
  for (int p = 1; p < P; ++p)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      out[p][i] = (__bf16)r[i];
      r[i] -= (float)out[p][i];
    }
}

// TK columns k x TN columns n of dW a workgroup of WK x WN = 8 waves; ROWS rows m a stage, two stages.  What a stage needs is on its
// way in registers AHEAD stages before it goes to LDS (one stage of a small tile computes in 0.3 us, and a load takes 1 - 2 us; a second
// set does not fit the registers of the 384-wide tile: 75.6 against 65.6 us for 131072 x 128 x 270).  With
// DIRECT, dy (bf16, rows of 16-byte pieces) goes from memory to LDS by itself, and only X, which is widened on the way, through registers.
template <typename T, int P, int TK, int TN, int ROWS, int WK, int WN, bool DIRECT>
__global__ __launch_bounds__(512) void fp8_wgrad_kernel(const Wg G) {
  constexpr int FA = TK / WK / 16, FB = TN / WN / 16, AHEAD = DIRECT || TK == 384 || TN == 256 ? 1 : 2;
  constexpr int RG = ROWS / 32, CX = TK / 128 * RG, CD = DIRECT ? 4 : TN / 128 * RG;      // pieces a thread moves: eight values, sixteen threads a row of 128
  constexpr int XBYTES = ROWS * TK * 2, DBYTES = ROWS * TN * 2;
  static_assert(WK * WN == 8 && TK % 128 == 0 && kWgRows % ROWS == 0 && (DIRECT ? P == 1 && TN == 256 && ROWS == 64 && FB == CD : TN % 128 == 0), "shape");
  // X as bf16 [ROWS][TK], then the P pieces of dy [ROWS][TN]; 16-byte piece c of row r in slot c ^ swz(r): the four rows that
  // sixteen lanes of a transpose read touch lie in different banks
  __shared__ __attribute__((aligned(16))) uint8_t stage[2][XBYTES + P * DBYTES];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), wk = wave % WK, wn = wave / WK;
  int ik, in;
  tile_of(blockIdx.x, (G.K + TK - 1) / TK, (G.N + TN - 1) / TN, ik, in);
  const int k0 = ik * TK, n0 = in * TN;
  const int64_t m_from = (int64_t)blockIdx.z * G.rows_per_split, m_to = min(G.M, m_from + G.rows_per_split);
  auto swz = [](int r) { return ((r & 3) << 1) | (((r >> 3) & 1) << 3); };

  const int tr = t >> 4, tc = t & 15;
  const int x_off = tr * (int)G.ldq + k0 + tc * 8, x_left = (int)G.ldq - k0 - tc * 8, s_off = tr * (int)G.lds + k0 / 128;
  struct Set { v2i xq[CX]; int xs[CX]; typename Vec8<T>::type d[DIRECT ? 1 : CD]; };
  Set set[AHEAD];
  float cs[DIRECT ? 1 : TN / 128][8] = {};       // of the columns tc * 8 .. + 7 of each 128 of dy, this thread's rows
  auto d_at = [&](int64_t m, int j) { return (m + tr + j % RG * 32) * G.N + n0 + j / RG * 128 + tc * 8; };
  // The stage that begins at m.  Rows of X past the split's end read as zero; of dy they are made zero in put().
  auto fetch = [&](Set& S, int64_t m) {
    const int rows = (int)max((int64_t)0, min(m_to - m, (int64_t)ROWS));
    const auto rq = __builtin_amdgcn_make_buffer_rsrc((void*)(G.q + m * G.ldq), 0, rows * (int)G.ldq, 0x00020000);
    const auto rs = __builtin_amdgcn_make_buffer_rsrc((void*)(G.scale + m * G.lds), 0, rows * (int)G.lds, 0x00020000);
#pragma unroll
    for (int j = 0; j < CX; ++j) {
      const int panel = j / RG, row = j % RG * 32;
      S.xq[j] = __builtin_bit_cast(v2i, __builtin_amdgcn_raw_buffer_load_b64(
                                            rq, panel * 128 < x_left ? x_off + row * (int)G.ldq + panel * 128 : kOutside, 0, 0));
      S.xs[j] = __builtin_amdgcn_raw_buffer_load_b8(rs, s_off + row * (int)G.lds + panel, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < (DIRECT ? 0 : CD) && G.M * G.N >= 8; ++j)        // unconditional: a load in a branch would be waited for at the branch's end
      __builtin_memcpy(&S.d[j], (const T*)G.dy + max((int64_t)0, min(d_at(m, j), G.M * G.N - 8)), 8 * sizeof(T));
  };
  auto put = [&](Set& S, int buf, int64_t m) {
#pragma unroll
    for (int j = 0; j < CX; ++j) {
      const float f = pow2_of_byte(S.xs[j]);
      const v2bf a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(S.xq[j][0], f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(S.xq[j][0], f, true);
      const v2bf c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(S.xq[j][1], f, false), e = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(S.xq[j][1], f, true);
      const int row = tr + j % RG * 32, chunk = j / RG * 16 + tc;
      *(v8bf*)(stage[buf] + row * TK * 2 + ((chunk ^ swz(row)) << 4)) = v8bf{a[0], a[1], b[0], b[1], c[0], c[1], e[0], e[1]};
    }
#pragma unroll
    for (int j = 0; j < (DIRECT ? 0 : CD); ++j) {
      const int row = tr + j % RG * 32, at = XBYTES + row * TN * 2 + (((j / RG * 16 + tc) ^ swz(row)) << 4);
      // columns past N are whatever lies there: their sums are not stored
      const int64_t from = d_at(m, j);
      if (m + row >= m_to) {
#pragma unroll
        for (int q = 0; q < 8; ++q) S.d[j][q] = (T)0.f;
      } else if (from + 8 > G.M * G.N) {                 // the last values of dy: fetch() read others, so as not to pass its end
#pragma unroll
        for (int q = 0; q < 8; ++q) S.d[j][q] = from + q < G.M * G.N ? ((const T*)G.dy)[from + q] : (T)0.f;
      }
      if (!DIRECT && ik == 0) {
#pragma unroll
        for (int q = 0; q < 8; ++q) cs[DIRECT ? 0 : j / RG][q] += (float)S.d[j][q];
      }
      if constexpr (P == 1) {
        *(v8bf*)(stage[buf] + at) = __builtin_bit_cast(v8bf, S.d[j]);
      } else {
        float v[8];
        v8bf e[P];
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = (float)S.d[j][q];
        pieces<P>(v, e);
#pragma unroll
        for (int p = 0; p < P; ++p) *(v8bf*)(stage[buf] + at + p * DBYTES) = e[p];
      }
    }
  };
  // DIRECT: rows 2 (wave + 8 j), + 1 of the stage that begins at m, one load instruction; columns past the row's end are another row's, in sums that are not stored
  auto direct = [&](int64_t m, int buf, int j) {
    const rsrc_t rd = make_rsrc((const T*)G.dy + m * G.N + n0, (int)(min(m_to - m, (int64_t)ROWS) * G.N - n0) * 2);
    const int row = 2 * (wave + 8 * j) + (lane >> 5);
    load_lds<16>(rd, lds_addr(stage[buf] + XBYTES + 2 * (wave + 8 * j) * TN * 2), row * G.N * 2 + (((lane & 31) ^ swz(row)) << 4));
  };
  const int p16 = lane & 15, g = lane >> 4;
  // rows 32 s + 8 g .. + 7 of sixteen columns from c0 (a multiple of 16), lane p16 the column; `plane`: LDS, rows of `width` values
  auto frag = [&](const uint8_t* plane, int width, int s, int c0) {
    v4s h[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int r = 32 * s + 8 * g + 4 * u + (p16 >> 2), c = c0 + 4 * (p16 & 3);
      h[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(plane + r * width * 2 + (((c >> 3) ^ swz(r)) << 4) + (c & 7) * 2));
    }
    return __builtin_bit_cast(v8bf, __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7));
  };

  v4f acc[FA][FB], accb[DIRECT ? FB : 1];
#pragma unroll
  for (int b = 0; b < FB; ++b) {
    accb[DIRECT ? b : 0] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int a = 0; a < FA; ++a) acc[a][b] = v4f{0.f, 0.f, 0.f, 0.f};
  }
  // the first column of tiles also sums dy's columns: as a product with ones where a thread never sees dy
  const bool sums = DIRECT && ik == 0 && wk == 0;
  v8bf ones;
#pragma unroll
  for (int e = 0; e < 8; ++e) ones[e] = (__bf16)1.f;

  // the stage at m is in `buf`, the next ones in `S` and (AHEAD = 2) the other set
  auto step = [&](Set& S, int buf, int64_t m) {
    if (m + ROWS < m_to) {
      put(S, buf ^ 1, m + ROWS);
      fetch(S, m + (1 + AHEAD) * ROWS);
    }
#pragma unroll
    for (int s = 0; s < ROWS / 32; ++s) {
      v8bf xf[FA];
#pragma unroll
      for (int a = 0; a < FA; ++a) xf[a] = frag(stage[buf], TK, s, (wk * FA + a) * 16);
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int b = 0; b < FB; ++b) {
          const v8bf df = frag(stage[buf] + XBYTES + p * DBYTES, TN, s, (wn * FB + b) * 16);
#pragma unroll
          for (int a = 0; a < FA; ++a) acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf[a], df, acc[a][b], 0, 0, 0);
          if (sums) accb[DIRECT ? b : 0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, df, accb[DIRECT ? b : 0], 0, 0, 0);
          // between the instructions: all at once they hold up the LDS reads (8192 x 4096 x 4096: 273 -> 246 us)
          if constexpr (DIRECT)
            if (s == 0 && m + ROWS < m_to) direct(m + ROWS, buf ^ 1, b);
        }
    }
    if constexpr (DIRECT) wait_loads();
    __syncthreads();
  };
  if (m_from < m_to) {
    if constexpr (DIRECT)
#pragma unroll
      for (int j = 0; j < CD; ++j) direct(m_from, 0, j);
    fetch(set[0], m_from);
    if constexpr (AHEAD == 2) fetch(set[1], m_from + ROWS);
    put(set[0], 0, m_from);
    fetch(set[0], m_from + AHEAD * ROWS);
  }
  if constexpr (DIRECT) wait_loads();
  __syncthreads();
  for (int64_t m = m_from; m < m_to; m += 2 * ROWS) {
    step(set[AHEAD - 1], 0, m);
    if (m + ROWS < m_to) step(set[0], 1, m + ROWS);
  }
  float* part = G.part ? G.part + blockIdx.z * G.stride : nullptr;
#pragma unroll
  for (int b = 0; b < FB; ++b) {
    const int n = n0 + (wn * FB + b) * 16 + p16;
    if (n >= G.N) continue;
#pragma unroll
    for (int a = 0; a < FA; ++a) {
      const int k = k0 + (wk * FA + a) * 16 + 4 * g;
      const int64_t at = (int64_t)n * G.K + k;
      if (part && k + 4 <= G.K) {
        __builtin_memcpy(part + at, &acc[a][b], 16);
      } else if (!part && G.dw && G.dw_dt == kF32 && k + 4 <= G.K) {
        __builtin_memcpy((float*)G.dw + at, &acc[a][b], 16);
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (k + r < G.K) {
            if (part) part[at + r] = acc[a][b][r];
            else if (G.dw) store_dt(G.dw, G.dw_dt, at + r, acc[a][b][r]);
          }
      }
    }
    if (sums && g == 0) {
      if (part) part[(int64_t)G.N * G.K + n] = accb[DIRECT ? b : 0][0];
      else if (G.db) store_dt(G.db, G.db_dt, n, accb[DIRECT ? b : 0][0]);
    }
  }
  if (!DIRECT && ik == 0) {
    float* red = (float*)stage;        // [8][TN]; the last step ended with a barrier
#pragma unroll
    for (int c = 0; c < (DIRECT ? 1 : TN / 128); ++c)
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        float v = cs[c][q];
        v += __shfl_xor(v, 16, 64);
        v += __shfl_xor(v, 32, 64);
        if (lane < 16) red[wave * TN + c * 128 + tc * 8 + q] = v;
      }
    __syncthreads();
    if (t < TN && n0 + t < G.N) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) v += red[w * TN + t];
      if (part) part[(int64_t)G.N * G.K + n0 + t] = v;
      else if (G.db) store_dt(G.db, G.db_dt, n0 + t, v);
    }
  }
}

// dy that goes to LDS directly: bf16, rows of 16-byte pieces
static bool wgrad_direct(int N, int dy_dt) { return dy_dt == kBF16 && N % 8 == 0; }

// The tile of dW: 256 x 256 where that leaves enough workgroups, and where dy goes through registers, stages of half the rows, enough rows
// (fp16 dy, 128 wide against 256: 8192 x 4096 x 4096: 768 / 571 us, 4000 x 2000 x 2000: 102 / 92 us, 1000 x 2001 x 2001: 44 / 57 us; bf16,
// 8192 x 4097 x 4096: 689 / 479 us).  Three pieces of fp32 spill there (874 / 1015 us).  Else 128 columns n, and of 384, 256 or 128
// columns k those that pad K least (K = 270: 384; 131072 rows of fp32, N = 128).
struct WgPlan { int tk, tn, split; };
WgPlan wgrad_plan(int64_t M, int N, int K, int dy_dt) {
  auto tiles = [&](int tk, int tn) { return (int64_t)((K + tk - 1) / tk) * ((N + tn - 1) / tn); };
  auto padded = [&](int tk) { return (int64_t)(K + tk - 1) / tk * tk; };
  WgPlan p = {384, 128, 1};
  if (tiles(256, 256) >= 64 && (wgrad_direct(N, dy_dt) || (dy_dt != kF32 && M >= 2048))) p = {256, 256, 1};
  else if (padded(256) < padded(384) || padded(128) < padded(384)) p.tk = padded(256) <= padded(128) ? 256 : 128;
  // A stage of 64 rows costs about 2 us where few workgroups run, a split's partial sums N K 8 bytes at 4 TB/s: sqrt of the ratio,
  // as long as the workgroups it makes find a free CU.
  const int64_t have = tiles(p.tk, p.tn), want = p.tk == 128 ? 512 : 256, steps = (M + kWgRows - 1) / kWgRows;
  int64_t split = (int64_t)ceil(sqrt((double)steps * 1e6 / ((double)N * K)));
  if (split > want / have) split = want / have;
  if (split > steps) split = steps;
  if (split < 1) split = 1;
  p.split = (int)split;
  return p;
}

template <typename T, int P, int ROWS>
void wgrad(const WgPlan& p, const dim3& grid, const Wg& G, hipStream_t st) {
  if constexpr (P < 3)
    if (p.tn == 256) { fp8_wgrad_kernel<T, P, 256, 256, 32, 2, 4, false><<<grid, 512, 0, st>>>(G); return; }
  if (p.tk == 384) fp8_wgrad_kernel<T, P, 384, 128, ROWS, 4, 2, false><<<grid, 512, 0, st>>>(G);
  else if (p.tk == 256) fp8_wgrad_kernel<T, P, 256, 128, ROWS, 4, 2, false><<<grid, 512, 0, st>>>(G);
  else fp8_wgrad_kernel<T, P, 128, 128, ROWS, 4, 2, false><<<grid, 512, 0, st>>>(G);
}

template <int TILE, int S>
void tile_launch(bool wide, const dim3& grid, const Mm& P, hipStream_t st) {
  if (wide) fp8_tile_kernel<TILE, TILE, 2, 2, S, true><<<grid, 256, 0, st>>>(P);
  else fp8_tile_kernel<TILE, TILE, 2, 2, S, false><<<grid, 256, 0, st>>>(P);
}

struct Plan { int tile, split; };      // tile: columns = rows of a workgroup's tile

// The largest tile that leaves enough workgroups and is not padded away; a contraction is split where they do not fill the CUs.
//   256: from 128 tiles up (3000 x 3000 x 4000 in bf16, 144 tiles on 256 CUs: 53 us, 128-wide tiles 71; 2500 x 2500 x 5000, 100 tiles: 65
//   against 50), unsplit, unless it computes over 1.3 times what 128-wide tiles would (131072 x 128 x 270 in bf16: 26 against 21 us)
Plan plan(int M, int N, int kblocks) {
  auto tiles = [&](int t) { return (int64_t)((M + t - 1) / t) * ((N + t - 1) / t); };
  const int tile = tiles(256) >= 128 && tiles(256) * 40 <= tiles(128) * 13 ? 256 : tiles(128) >= 192 ? 128 : 64;
  int split = 1;
  const int64_t have = tiles(tile);
  if (have < 256 && tile < 256) split = (int)((512 + have - 1) / have);
  if (split > kblocks / 4) split = kblocks / 4;
  if (split > 16) split = 16;
  if (split < 1) split = 1;
  return {tile, split};
}

}  // namespace

extern "C" {

size_t hcm_fp8_matmul_workspace_bytes(int M, int N, int K) {
  if (M <= kFewRows || N <= 0 || K <= 0) return 0;
  const Plan p = plan(M, N, (K + 127) / 128);
  return p.split > 1 ? (size_t)p.split * M * N * sizeof(float) : 0;
}

int hcm_fp8_matmul(const uint8_t* x, int64_t ldx, const uint8_t* x_scale, int64_t ldsx, const uint8_t* w, int64_t ldw, const uint8_t* w_scale,
                   int64_t ldsw, const void* bias, int bias_dtype, int M, int N, int K, void* y, int out_dtype, void* workspace,
                   size_t workspace_bytes, hcm_stream_t stream) {
  if (!x || !x_scale || !w || !w_scale || !y || M <= 0 || M > INT32_MAX - 512 || N <= 0 || N > (1 << 22) || K <= 0 || K > (1 << 22) || ldx != hcm_act8_pitch(K) || ldw != ldx ||
      ldsx != hcm_act8_scale_pitch(K) || ldsw != ldsx || out_dtype < 0 || out_dtype > 2 || (bias && (bias_dtype < 0 || bias_dtype > 2)) ||
      ((uintptr_t)x & 15) || ((uintptr_t)w & 15) || ((uintptr_t)x_scale & 3) || ((uintptr_t)w_scale & 3))
    return (int)hipErrorInvalidValue;
  Mm P = {x, x_scale, w, w_scale, ldx, ldsx, ldw, ldsw, M, N, (K + 127) / 128, (int)ldx, bias, bias_dtype, out_dtype, y, nullptr, 1};
  const bool wide = out_dtype == kF32;
  hipStream_t st = (hipStream_t)stream;
  if (M <= kFewRows)
    return wide ? few<uint8_t, true>(P, nullptr, 0, K, nullptr, nullptr, st) : few<uint8_t, false>(P, nullptr, 0, K, nullptr, nullptr, st);
  const Plan p = plan(M, N, P.kblocks);
  if (workspace_bytes < hcm_fp8_matmul_workspace_bytes(M, N, K) || (p.split > 1 && !workspace)) return (int)hipErrorInvalidValue;
  P.split = p.split;
  if (p.split > 1) P.part = (float*)workspace;
  const int64_t tiles = (int64_t)((M + p.tile - 1) / p.tile) * ((N + p.tile - 1) / p.tile);
  if (tiles * (p.tile == 256 ? 512 : 256) >= (1ll << 32)) return (int)hipErrorInvalidValue;       // threads of a launch
  const dim3 grid((uint32_t)tiles, 1, p.split);
  // Four stages keep a long contraction fed where each CU has no more workgroups than fit beside each other with them (one of 128-wide
  // tiles, two of 64: 500 x 4096 x 4096 in bf16 21.8 -> 17.4 us); where it has more, two stages and twice the workgroups at once are
  // faster (1000 x 5000 x 1000 in bf16: 20.6 -> 14.1 us; 131072 x 128 x 270 in fp32: 41.7 -> 30.6 us).
  const bool deep = P.kblocks > 4 && tiles * p.split <= (p.tile == 128 ? 256 : 512);
  if (p.tile == 256 && wide) fp8_tile_kernel<256, 256, 2, 4, 2, true><<<grid, 512, 0, st>>>(P);
  else if (p.tile == 256) fp8_tile_kernel<256, 256, 2, 4, 2, false><<<grid, 512, 0, st>>>(P);
  else if (p.tile == 128) deep ? tile_launch<128, 4>(wide, grid, P, st) : tile_launch<128, 2>(wide, grid, P, st);
  else deep ? tile_launch<64, 4>(wide, grid, P, st) : tile_launch<64, 2>(wide, grid, P, st);
  HCM_CHECK_LAUNCH();
  if (p.split > 1) {
    const int64_t n = (int64_t)M * N;
    return join({P.part, p.split, n, n, 0, N, bias, bias_dtype, y, out_dtype, nullptr, 0}, st);
  }
  return 0;
}

int hcm_fp8_rows_supported(int64_t M, int K) { return M > 0 && M <= kFewRows && K > 0 && K <= (1 << 22) && M * ((K + 127) / 128) <= kFewBlocks; }

int hcm_fp8_rows(const void* x, int dtype, int64_t ldx, const uint8_t* w, int64_t ldw, const uint8_t* w_scale, int64_t ldsw, const void* bias,
                 int bias_dtype, int M, int N, int K, void* y, uint8_t* q, uint8_t* q_scale, hcm_stream_t stream) {
  if (!x || !w || !w_scale || !y || !hcm_fp8_rows_supported(M, K) || N <= 0 || N > (1 << 22) || ldx < K || ldw != hcm_act8_pitch(K) ||
      ldsw != hcm_act8_scale_pitch(K) || dtype < 0 || dtype > 2 || (bias && (bias_dtype < 0 || bias_dtype > 2)) || (!q != !q_scale) ||
      ((uintptr_t)w & 15) || ((uintptr_t)q & 15))
    return (int)hipErrorInvalidValue;
  const Mm P = {nullptr, nullptr, w, w_scale, ldw, ldsw, ldw, ldsw, M, N, (K + 127) / 128, (int)ldw, bias, bias_dtype, dtype, y, nullptr, 1};
  hipStream_t st = (hipStream_t)stream;
  if (dtype == kF32) return few<float, true>(P, (const float*)x, ldx, K, q, q_scale, st);
  if (dtype == kBF16) return few<__bf16, false>(P, (const __bf16*)x, ldx, K, q, q_scale, st);
  return few<_Float16, false>(P, (const _Float16*)x, ldx, K, q, q_scale, st);
}

// partial sums of dW and db, a multiple of four floats apart
static int64_t wgrad_stride(int N, int K) { return ((int64_t)N * K + N + 3) / 4 * 4; }

size_t hcm_fp8_wgrad_workspace_bytes(int64_t M, int N, int K, int dy_dtype, int with_dw) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  if (!with_dw) K = 1;
  const WgPlan p = wgrad_plan(M, N, K, dy_dtype);
  return p.split > 1 ? (size_t)p.split * wgrad_stride(N, K) * sizeof(float) : 0;
}

int hcm_fp8_wgrad(const uint8_t* x, int64_t ldx, const uint8_t* x_scale, int64_t ldsx, const void* dy, int dy_dtype, int64_t M, int N, int K, void* dw,
                  int dw_dtype, void* db, int db_dtype, void* workspace, size_t workspace_bytes, hcm_stream_t stream) {
  if ((dw && (!x || !x_scale)) || !dy || (!dw && !db) || M <= 0 || M >= (1ll << 31) || N <= 0 || K <= 0 || K > (1 << 22) || N > (1 << 22) ||
      ldx != hcm_act8_pitch(K) || ldsx != hcm_act8_scale_pitch(K) || dy_dtype < 0 || dy_dtype > 2 || dw_dtype < 0 || dw_dtype > 2 || db_dtype < 0 ||
      db_dtype > 2 || ((uintptr_t)x & 15) || ((uintptr_t)dy & 15))
    return (int)hipErrorInvalidValue;
  if (!dw) x = x_scale = nullptr, ldx = ldsx = 0, K = 1;       // the sums of dy's columns alone: one column of tiles, an X of no bytes
  const WgPlan p = wgrad_plan(M, N, K, dy_dtype);
  if (p.split > 1 && (!workspace || workspace_bytes < hcm_fp8_wgrad_workspace_bytes(M, N, K, dy_dtype, dw != nullptr))) return (int)hipErrorInvalidValue;
  const int64_t tiles = (int64_t)((K + p.tk - 1) / p.tk) * ((N + p.tn - 1) / p.tn), steps = (M + kWgRows - 1) / kWgRows;
  if (tiles * 512 >= (1ll << 32)) return (int)hipErrorInvalidValue;       // threads of a launch
  const Wg G = {x,  x_scale, ldx, ldsx, dy, M, N, K, (steps + p.split - 1) / p.split * kWgRows, p.split > 1 ? (float*)workspace : nullptr, wgrad_stride(N, K),
                dw, db,      dw_dtype, db_dtype};
  const dim3 grid((uint32_t)tiles, 1, p.split);
  hipStream_t st = (hipStream_t)stream;
  if (dy_dtype == kF32) wgrad<float, 3, 32>(p, grid, G, st);
  else if (dy_dtype == kF16) wgrad<_Float16, 2, 32>(p, grid, G, st);
  else if (p.tn == 256 && wgrad_direct(N, dy_dtype)) fp8_wgrad_kernel<__bf16, 1, 256, 256, 64, 2, 4, true><<<grid, 512, 0, st>>>(G);
  else wgrad<__bf16, 1, 64>(p, grid, G, st);
  HCM_CHECK_LAUNCH();
  if (p.split > 1) return join({G.part, p.split, G.stride, (int64_t)N * K, N, N, nullptr, 0, dw, dw_dtype, db, db_dtype}, st);
  return 0;
}

}  // extern "C"
