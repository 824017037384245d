// Products of 8-bit blocks (act8.h has the format):  y[m][n] = sum_k X[m][k] W[n][k] (+ bias[n]),  X [M, K] with a scale for 128
// values of a row, W [N, K] with a scale for each block of 128 x 128.  Forward: X = Q(x), W = Q(weight); data gradient:
// X = Q(dy), W = the transposed copy of Q(weight).
//
// A block of 128 along k is ONE scaled matrix instruction (v_mfma_scale_f32_16x16x128_f8f6f4), and the format's scale byte is
// its scale operand: the scales cost no arithmetic.  Its two operands only have to agree on the order of k, so a lane takes
// the 16-byte pieces g and g + 4 of its row (g = lane / 16).  W is the A operand, so that a lane ends up with neighbouring
// columns of y; the sixteen A rows of two instructions are interleaved so that they are eight neighbours.
//
// Precision.  Every 8-bit matrix instruction of this chip adds its products in groups of eight neighbouring k, aligned to the
// group's largest product, and drops what lies below 2^-13 of it (measured on single products, the same for the scaled form and for
// 16x16x32; the sums of groups are full fp32): 2e-5 .. 7e-5 of the result's norm on random data.  That is under the rounding of
// a 16-bit y (2^-9, 2^-12), and it is over that of an fp32 one, so y in fp32 takes the WIDE form: the 8-bit values are widened to bf16
// on their way from LDS -- exact, the scales included, by v_cvt_scalef32_pk_bf16_fp8 -- and multiplied by v_mfma_f32_16x16x32_bf16,
// whose sums are fp32 (1e-8 .. 3e-7 on the same data), at half the rate.
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

typedef __attribute__((address_space(3))) void lds_void;
typedef __amdgpu_buffer_rsrc_t rsrc_t;

// Workgroups go to the eight XCDs in turn; each XCD gets a run of neighbouring tiles (whole columns of eight row tiles), so that
// its L2 serves the rows they share.
__device__ __forceinline__ void tile_of(int id, int tm, int tn, int& im, int& in) {
  const int total = tm * tn, xcd = id & 7, k = id >> 3, base = total >> 3, rem = total & 7;
  const int t = xcd * base + min(xcd, rem) + k;
  const int band = 8 * tn, b = t / band, in_band = t - b * band, h = min(8, tm - 8 * b);
  in = in_band / h;
  im = 8 * b + (in_band - in * h);
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

// BN columns x BM rows of y a workgroup, WN x WM waves of TN x TM tiles of 16 x 16.  Two LDS stages of (BN + BM) x 128 bytes,
// filled by direct loads; one barrier a block of k.
template <int BN, int BM, int WN, int WM, bool WIDE>
__global__ __launch_bounds__(WN * WM * 64) void fp8_tile_kernel(const Mm P) {
  constexpr int NT = WN * WM * 64, TN = BN / WN / 16, TM = BM / WM / 16;
  constexpr int LW = BN * 8 / NT, LX = BM * 8 / NT;        // 16-byte pieces a thread moves
  static_assert(TN % 2 == 0 && LW >= 1 && LX >= 1 && BN * 8 % NT == 0 && BM * 8 % NT == 0, "tile");
  __shared__ __attribute__((aligned(128))) uint8_t stage[2][(BN + BM) * 128];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, wn = wave % WN, wm = wave / WN;
  int im, in;
  tile_of(blockIdx.x, (P.M + BM - 1) / BM, (P.N + BN - 1) / BN, im, in);
  const int m0 = im * BM, n0 = in * BN;
  const int per = (P.kblocks + P.split - 1) / P.split, k_from = blockIdx.z * per, k_to = min(P.kblocks, k_from + per);

  const uint8_t* wbase = P.w + (int64_t)n0 * P.ldw;
  const uint8_t* xbase = P.x + (int64_t)m0 * P.ldx;
  const int wbytes = (int)(min(P.N - n0, BN) * P.ldw), xbytes = (int)(min(P.M - m0, BM) * P.ldx);

  // Row r of a stage lies at r * 128, its piece c in slot c ^ key(r): eight lanes that read the same piece of eight rows hit eight
  // different slots.  A load instruction of a wave fills eight rows; which piece a lane fetches is what places it.
  const int r8 = lane >> 3, slot = lane & 7;
  auto issue = [&](int kb, int buf) {
    const int64_t ko = (int64_t)kb * 128;
    const rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc((void*)(wbase + ko), 0, wbytes - (int)ko, 0x00020000);
    const rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc((void*)(xbase + ko), 0, xbytes - (int)ko, 0x00020000);
    const int left = P.ldk - kb * 128;       // pieces past the row's end would be the next row's: sent out of range, they read as zero
#pragma unroll
    for (int j = 0; j < LW; ++j) {
      const int rg = wave + j * (NT / 64), r = rg * 8 + r8;                     // W rows: key (r & 3) | (r >> 3 & 1) << 2
      const int c = slot ^ ((r8 & 3) | ((rg & 1) << 2));
      const int off = c * 16 < left ? r * (int)P.ldw + c * 16 : (int)0x80000000;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rw, (lds_void*)&stage[buf][rg * 1024], 16, off, 0, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < LX; ++j) {
      const int rg = wave + j * (NT / 64), r = rg * 8 + r8;                     // X rows: key r & 7
      const int c = slot ^ r8;
      const int off = c * 16 < left ? r * (int)P.ldx + c * 16 : (int)0x80000000;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rx, (lds_void*)&stage[buf][(BN + rg * 8) * 128], 16, off, 0, 0, 0);
    }
  };

  const int i = lane & 15, g = lane >> 4;
  const int frag = (g ^ (i & 7)) << 4;
  int wrow[TN], xrow[TM];
#pragma unroll
  for (int a = 0; a < TN; ++a) wrow[a] = (wn * TN * 16 + 32 * (a >> 1) + (i >> 2) * 8 + (a & 1) * 4 + (i & 3)) * 128 + frag;
#pragma unroll
  for (int b = 0; b < TM; ++b) xrow[b] = (BN + (wm * TM + b) * 16 + i) * 128 + frag;
  const uint8_t* sxp[TM];
#pragma unroll
  for (int b = 0; b < TM; ++b) sxp[b] = P.sx + (int64_t)min(m0 + (wm * TM + b) * 16 + i, P.M - 1) * P.ldsx;
  const uint8_t* swp = P.sw + (int64_t)(min(n0 + wn * TN * 16, P.N - 1) / 128) * P.ldsw;

  v4f acc[TN][TM];
#pragma unroll
  for (int a = 0; a < TN; ++a)
#pragma unroll
    for (int b = 0; b < TM; ++b) acc[a][b] = v4f{0.f, 0.f, 0.f, 0.f};

  int sx_next[TM], sw_next = 0;
  auto scales = [&](int kb) {
#pragma unroll
    for (int b = 0; b < TM; ++b) sx_next[b] = sxp[b][kb];
    sw_next = swp[kb];
  };
  if (k_from < k_to) scales(k_from), issue(k_from, 0);
  for (int kb = k_from; kb < k_to; ++kb) {
    const int buf = (kb - k_from) & 1;
    __builtin_amdgcn_s_waitcnt(0x0f70);          // vmcnt(0): this wave's pieces of the stage have landed
    __syncthreads();
    int sx[TM];
#pragma unroll
    for (int b = 0; b < TM; ++b) sx[b] = sx_next[b];
    const int sw = sw_next;
    if (kb + 1 < k_to) scales(kb + 1), issue(kb + 1, buf ^ 1);
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
    }
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

// y = sum of the split's partial sums (in order) + bias
__global__ __launch_bounds__(256) void fp8_join_kernel(const float* __restrict__ part, int split, int64_t n, int N, const void* __restrict__ bias, int bias_dt,
                                                       void* __restrict__ y, int out_dt) {
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < n; e += (int64_t)gridDim.x * 256) {
    float s = 0.f;
    for (int z = 0; z < split; ++z) s += part[z * n + e];
    if (bias) s += load_dt(bias, bias_dt, e % N);
    store_dt(y, out_dt, e, s);
  }
}

// ---------------------------------------------------------------------------------------------------------------------------------
// Weight gradient from the 8-bit checkpoint:  dW[n][k] = sum_m dy[m][n] X[m][k],  db[n] = sum_m dy[m][n].
//
// q * 2^E is exact in bf16, so X enters v_mfma_f32_16x16x32_bf16 without a rounding; dy enters as the bf16 pieces that hold its type
// exactly (bf16: 1, fp16: 2, fp32: 3), one instruction a piece: only the fp32 sums round.  Both operands lie row by row (m),
// and the instruction wants eight m of one column in a lane: the LDS transpose read (lane p of sixteen points at row p / 4, columns
// 4 (p % 4) .. + 3, and receives column p of the four rows).  128 columns k (one scale a row) x 128 columns n a workgroup.
struct Wg {
  const uint8_t *q, *scale;
  int64_t ldq, lds;
  const void* dy;
  int64_t M;
  int N, K;
  int rows_per_split;             // a multiple of kWgRows
  float* part;                    // [split][N * K + N]
};
constexpr int kWgRows = 64;

typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s* lds_v4s;

template <int P>
__device__ __forceinline__ void pieces(const float (&v)[8], v8bf (&out)[P]) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = v[i];
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      out[p][i] = (__bf16)r[i];
      r[i] -= (float)out[p][i];
    }
}

template <typename T, int P>
__global__ __launch_bounds__(256) void fp8_wgrad_kernel(const Wg G) {
  // plane 0: X, planes 1 .. P: the pieces of dy; [kWgRows][128] bf16, 16-byte piece c of row r in slot c ^ swz(r)
  __shared__ __attribute__((aligned(16))) uint8_t stage[(1 + P) * kWgRows * 256];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, wk = wave & 1, wn = wave >> 1;
  const int k0 = blockIdx.x * 128, n0 = blockIdx.y * 128;
  const int64_t m_from = (int64_t)blockIdx.z * G.rows_per_split, m_to = min(G.M, m_from + G.rows_per_split);
  auto swz = [](int r) { return ((r & 3) << 1) | (((r >> 3) & 1) << 3); };
  // a thread stages a quarter row: 32 values of X and of dy
  const int sr = t >> 2, sc = (t & 3) * 32;
  v8i xq;
  int xs;
  float d[4][8];
  auto fetch = [&](int64_t m) {
    const int64_t row = m + sr;
    const bool in = row < m_to;
    xq = v8i{0, 0, 0, 0, 0, 0, 0, 0};
    xs = 127;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) d[j][i] = 0.f;
    if (!in) return;
    const uint8_t* qr = G.q + row * G.ldq + k0 + sc;
    if (k0 + sc < G.ldq) { const v4i a = *(const v4i*)qr; xq[0] = a[0]; xq[1] = a[1]; xq[2] = a[2]; xq[3] = a[3]; }
    if (k0 + sc + 16 < G.ldq) { const v4i a = *(const v4i*)(qr + 16); xq[4] = a[0]; xq[5] = a[1]; xq[6] = a[2]; xq[7] = a[3]; }
    xs = G.scale[row * G.lds + blockIdx.x];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + sc + 8 * j;
      if (n < G.N) load8((const T*)G.dy + row * G.N + n, G.N - n, d[j]);
    }
  };
  auto put = [&]() {
    const float sf = pow2_of_byte(xs);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float f[8];
      act8_values(v2i{xq[2 * j], xq[2 * j + 1]}, sf, f);
      v8bf o[1], e[P];
      pieces<1>(f, o);
      const int at = sr * 256 + (((sc >> 3) + j) ^ swz(sr)) * 16;
      *(v8bf*)(stage + at) = o[0];
      pieces<P>(d[j], e);
#pragma unroll
      for (int p = 0; p < P; ++p) *(v8bf*)(stage + (1 + p) * kWgRows * 256 + at) = e[p];
    }
  };
  v4f acc[4][4], accb[4];
#pragma unroll
  for (int a = 0; a < 4; ++a) {
    accb[a] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int b = 0; b < 4; ++b) acc[a][b] = v4f{0.f, 0.f, 0.f, 0.f};
  }
  const int p16 = lane & 15, g = lane >> 4;
  // eight rows 32 s + 8 g .. + 7 of sixteen columns from c0 (a multiple of 16), lane p16 the column
  auto frag = [&](int plane, int s, int c0) {
    v4s h[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int r = 32 * s + 8 * g + 4 * u + (p16 >> 2), c = c0 + 4 * (p16 & 3);
      h[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(stage + plane * kWgRows * 256 + r * 256 + (((c >> 3) ^ swz(r)) << 4) + (c & 7) * 2));
    }
    return __builtin_bit_cast(v8bf, __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7));
  };
  const bool sums = blockIdx.x == 0 && wk == 0;
  v8bf ones;
#pragma unroll
  for (int i = 0; i < 8; ++i) ones[i] = (__bf16)1.f;
  if (m_from < m_to) fetch(m_from);
  for (int64_t m = m_from; m < m_to; m += kWgRows) {
    put();
    __syncthreads();
    if (m + kWgRows < m_to) fetch(m + kWgRows);
#pragma unroll
    for (int s = 0; s < kWgRows / 32; ++s) {
      v8bf xf[4];
#pragma unroll
      for (int a = 0; a < 4; ++a) xf[a] = frag(0, s, wk * 64 + a * 16);
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const v8bf df = frag(1 + p, s, wn * 64 + b * 16);
#pragma unroll
          for (int a = 0; a < 4; ++a) acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf[a], df, acc[a][b], 0, 0, 0);
          if (sums) accb[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, df, accb[b], 0, 0, 0);
        }
    }
    __syncthreads();
  }
  float* out = G.part + (int64_t)blockIdx.z * ((int64_t)G.N * G.K + G.N);
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const int n = n0 + wn * 64 + b * 16 + p16;
    if (n >= G.N) continue;
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const int k = k0 + wk * 64 + a * 16 + 4 * g;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (k + r < G.K) out[(int64_t)n * G.K + k + r] = acc[a][b][r];
    }
    if (sums && g == 0) out[(int64_t)G.N * G.K + n] = accb[b][0];
  }
}

// dW = sum of the split's partial sums, db likewise behind them
__global__ __launch_bounds__(256) void fp8_wgrad_join_kernel(const float* __restrict__ part, int split, int64_t n, int N, void* __restrict__ dw, int dw_dt,
                                                             void* __restrict__ db, int db_dt) {
  const int64_t all = n + N;
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < all; e += (int64_t)gridDim.x * 256) {
    float s = 0.f;
    for (int z = 0; z < split; ++z) s += part[z * all + e];
    if (e < n) { if (dw) store_dt(dw, dw_dt, e, s); }
    else if (db) store_dt(db, db_dt, e - n, s);
  }
}

int wgrad_split(int64_t M, int N, int K) {
  const int64_t tiles = (int64_t)((N + 127) / 128) * ((K + 127) / 128), steps = (M + kWgRows - 1) / kWgRows;
  int64_t split = (512 + tiles - 1) / tiles;
  if (split > (steps + 7) / 8) split = (steps + 7) / 8;      // at least 512 rows each
  return (int)(split < 1 ? 1 : split);
}

struct Plan { int tile, split; };      // tile: columns = rows of a workgroup's tile

// `wide`: the bf16 operands of a 256 x 256 tile do not fit the registers
Plan plan(int M, int N, int kblocks, bool wide) {
  auto tiles = [&](int t) { return (int64_t)((M + t - 1) / t) * ((N + t - 1) / t); };
  const int tile = tiles(256) >= 192 && !wide ? 256 : tiles(128) >= 192 ? 128 : 64;
  int split = 1;
  const int64_t have = tiles(tile);
  if (have < 256) split = (int)((512 + have - 1) / have);
  if (split > kblocks / 4) split = kblocks / 4;
  if (split > 16) split = 16;
  if (split < 1) split = 1;
  return {tile, split};
}

}  // namespace

extern "C" {

size_t hcm_fp8_matmul_workspace_bytes(int M, int N, int K, int out_dtype) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const Plan p = plan(M, N, (K + 127) / 128, out_dtype == kF32);
  return p.split > 1 ? (size_t)p.split * M * N * sizeof(float) : 0;
}

int hcm_fp8_matmul(const uint8_t* x, int64_t ldx, const uint8_t* x_scale, int64_t ldsx, const uint8_t* w, int64_t ldw, const uint8_t* w_scale,
                   int64_t ldsw, const void* bias, int bias_dtype, int M, int N, int K, void* y, int out_dtype, void* workspace,
                   size_t workspace_bytes, hcm_stream_t stream) {
  if (!x || !x_scale || !w || !w_scale || !y || M <= 0 || M > INT32_MAX - 512 || N <= 0 || N > (1 << 22) || K <= 0 || K > (1 << 22) || ldx != hcm_act8_pitch(K) || ldw != ldx ||
      ldsx != hcm_act8_scale_pitch(K) || ldsw != ldsx || out_dtype < 0 || out_dtype > 2 || (bias && (bias_dtype < 0 || bias_dtype > 2)) ||
      ((uintptr_t)x & 15) || ((uintptr_t)w & 15))
    return (int)hipErrorInvalidValue;
  Mm P = {x, x_scale, w, w_scale, ldx, ldsx, ldw, ldsw, M, N, (K + 127) / 128, (int)ldx, bias, bias_dtype, out_dtype, y, nullptr, 1};
  const bool wide = out_dtype == kF32;
  const Plan p = plan(M, N, P.kblocks, wide);
  if (workspace_bytes < hcm_fp8_matmul_workspace_bytes(M, N, K, out_dtype) || (p.split > 1 && !workspace)) return (int)hipErrorInvalidValue;
  P.split = p.split;
  if (p.split > 1) P.part = (float*)workspace;
  hipStream_t st = (hipStream_t)stream;
  const int64_t tiles = (int64_t)((M + p.tile - 1) / p.tile) * ((N + p.tile - 1) / p.tile);
  if (tiles >= (1ll << 31)) return (int)hipErrorInvalidValue;
  const dim3 grid((uint32_t)tiles, 1, p.split);
  if (p.tile == 256) fp8_tile_kernel<256, 256, 2, 4, false><<<grid, 512, 0, st>>>(P);
  else if (p.tile == 128 && wide) fp8_tile_kernel<128, 128, 2, 2, true><<<grid, 256, 0, st>>>(P);
  else if (p.tile == 128) fp8_tile_kernel<128, 128, 2, 2, false><<<grid, 256, 0, st>>>(P);
  else if (wide) fp8_tile_kernel<64, 64, 2, 2, true><<<grid, 256, 0, st>>>(P);
  else fp8_tile_kernel<64, 64, 2, 2, false><<<grid, 256, 0, st>>>(P);
  HCM_CHECK_LAUNCH();
  if (p.split > 1) {
    const int64_t n = (int64_t)M * N, blocks = (n + 255) / 256;
    fp8_join_kernel<<<(uint32_t)(blocks < 4096 ? blocks : 4096), 256, 0, st>>>(P.part, p.split, n, N, bias, bias_dtype, y, out_dtype);
    HCM_CHECK_LAUNCH();
  }
  return 0;
}

size_t hcm_fp8_wgrad_workspace_bytes(int64_t M, int N, int K) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  return (size_t)wgrad_split(M, N, K) * ((size_t)N * K + N) * sizeof(float);
}

int hcm_fp8_wgrad(const uint8_t* x, int64_t ldx, const uint8_t* x_scale, int64_t ldsx, const void* dy, int dy_dtype, int64_t M, int N, int K, void* dw,
                  int dw_dtype, void* db, int db_dtype, void* workspace, size_t workspace_bytes, hcm_stream_t stream) {
  if (!x || !x_scale || !dy || (!dw && !db) || !workspace || M <= 0 || M >= (1ll << 31) || N <= 0 || K <= 0 || K > (1 << 22) || N > (1 << 22) ||
      ldx != hcm_act8_pitch(K) || ldsx != hcm_act8_scale_pitch(K) || dy_dtype < 0 || dy_dtype > 2 || dw_dtype < 0 || dw_dtype > 2 || db_dtype < 0 ||
      db_dtype > 2 || ((uintptr_t)x & 15) || workspace_bytes < hcm_fp8_wgrad_workspace_bytes(M, N, K))
    return (int)hipErrorInvalidValue;
  const int split = wgrad_split(M, N, K);
  const int64_t steps = (M + kWgRows - 1) / kWgRows;
  const Wg G = {x, x_scale, ldx, ldsx, dy, M, N, K, (int)((steps + split - 1) / split * kWgRows), (float*)workspace};
  const dim3 grid((K + 127) / 128, (N + 127) / 128, split);
  hipStream_t st = (hipStream_t)stream;
  if (dy_dtype == kF32) fp8_wgrad_kernel<float, 3><<<grid, 256, 0, st>>>(G);
  else if (dy_dtype == kBF16) fp8_wgrad_kernel<__bf16, 1><<<grid, 256, 0, st>>>(G);
  else fp8_wgrad_kernel<_Float16, 2><<<grid, 256, 0, st>>>(G);
  HCM_CHECK_LAUNCH();
  const int64_t n = (int64_t)N * K, blocks = (n + N + 255) / 256;
  fp8_wgrad_join_kernel<<<(uint32_t)(blocks < 4096 ? blocks : 4096), 256, 0, st>>>(G.part, split, n, N, dw, dw_dtype, db, db_dtype);
  HCM_CHECK_LAUNCH();
  return 0;
}

}  // extern "C"
