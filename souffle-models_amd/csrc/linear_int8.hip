// Linear layers in 8-bit integers: rows quantised as they come (one scale per row), weights quantised once (one scale per
// output channel), products on the integer matrix cores, scales, bias and activation in the epilogue.
//
//   q[m][k] = round_half_even(x[m][k] / s[m]),   y[m][n] = act(s[m] t[n] sum_k q[m][k] w[k][n] + b[n])
//
// The sums are 32-bit integers and exact (K <= 131071 keeps them in range), so neither the order of K nor a split of
// it changes a result.
//
// Weights are kept in one packed copy [N/64][K/64][4 operands][64 lanes][16 bytes] (zeros up to multiples of 64): an
// operand of v_mfma_i32_16x16x64_i8 is one contiguous KB that a wave loads straight into registers with one
// 16-byte load per lane, and the four operands of 64 columns x 64 of K are 4 KB in a row.  Lane 16 c + 4 g + v of operand t holds
// k = 16 c .. 16 c + 15 of column 16 g + 4 t + v.  With the weights as the instruction's first operand a lane's four
// results are the columns 16 g + 4 t .. + 3 of one row (g = lane / 16), so over the four operands a lane owns 16 adjacent columns of a row: 32
// bytes of an fp16 result.
#include <algorithm>
#include "typed.hpp"
#include "host_util.hpp"

namespace souffle {
namespace linear_int8 {

typedef int i4 __attribute__((ext_vector_type(4)));

// v_mfma_i32_16x16x64_i8: D[i][j] += sum_k A[i][k] B[k][j]; lane l holds row i (column j) = l % 16, k = 16 (l / 16) .. + 15
// of A (of B), and rows 4 (l / 16) .. + 3 of column l % 16 of D.
__device__ __forceinline__ i4 mfma_i8(i4 a, i4 b, i4 c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }

// The 4-byte form of load_lds16: lane L's word lands at lds_addr + 4 L.
__device__ __forceinline__ void load_lds4(const void *src, unsigned lds_addr) {
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dword %1, off" ::"s"(__builtin_amdgcn_readfirstlane(lds_addr)), "v"(src) : "memory", "m0");
#pragma clang diagnostic pop
}

__device__ __forceinline__ i4 ldg16(const int8_t *p) { return *(const __attribute__((address_space(1))) i4 *)p; }

// ---------------------------------------------------------------------------------------- quantisation ----
// Rows: TPR threads per row, NV vectors of 8 per thread kept in registers between the largest value and the rounding
// (NV = 0: any length, the row is read again for the rounding).  Bound by memory, 3 bytes per fp16 element: 8192 x 4096 bf16 takes 20 us,
// 101 MB at 5.0 TB/s.  The thread count per row keeps one or two vectors a thread, so that small inputs spread over many waves, and
// that rows of up to 128 elements share a wave (262144 x 64 fp16: 19 us with 16 threads a row, 58 with 64).
template <class T, int TPR, int NV, RowForm FORM>
__global__ void __launch_bounds__(256) k_quantize_rows(const T *x, long long ldx, int8_t *q, long long ldq, float *scale, int rows, int cols) {
  constexpr int kSlots = 256 / TPR;
  __shared__ unsigned lds_max[2][4];
  const int slot = threadIdx.x / TPR, t = threadIdx.x % TPR;
  int turn = 0;      // (rows of 256 threads: every thread takes the same turns)
  for (long long row = (long long)blockIdx.x * kSlots + slot; row < rows; row += (long long)gridDim.x * kSlots, turn ^= 1) {
    const T *xr = x + row * ldx;
    int8_t *qr = q + row * ldq;
    typename Vec8<T>::type v[NV ? NV : 1];
    unsigned m = 0u;
    auto widen = [&](float (&f)[8], typename Vec8<T>::type w, int c) { to_f32(f, settle_row<FORM, T>(w, c, cols)); };
    auto largest = [&](const float (&f)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) m = max(m, abs_bits(f[e]));
    };
    float f[NV ? NV : 1][8];
    if constexpr (NV > 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i) v[i] = load_row<FORM>(xr, (i * TPR + t) * 8, cols);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        widen(f[i], v[i], (i * TPR + t) * 8);
        largest(f[i]);
      }
    } else {
      for (int c = t * 8; c < cols; c += TPR * 8) {
        widen(f[0], load_row<FORM>(xr, c, cols), c);
        largest(f[0]);
      }
    }
    m = TPR == 16 ? row16_umax_dpp(m) : wave_umax_dpp(m);
    if constexpr (TPR > 64) {
      unsigned *r = lds_max[turn];
      if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = m;
      __syncthreads();
      m = max(max(r[0], r[1]), max(r[2], r[3]));
    }
    const RowScale rs = row_scale(m);
    if constexpr (NV > 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + t) * 8;
        const u2 p = quantize8(f[i], rs);
        if (c < cols) *reinterpret_cast<u2 *>(qr + c) = p;
      }
    } else {
      for (int c = t * 8; c < cols; c += TPR * 8) {
        widen(f[0], load_row<FORM>(xr, c, cols), c);
        *reinterpret_cast<u2 *>(qr + c) = quantize8(f[0], rs);
      }
    }
    if (t == 0) scale[row] = rs.scale;
  }
}

// Byte offset of weight (k, n) in the packed copy.
__device__ __forceinline__ size_t packed_at(int k, int n, int kblocks) {
  const int kk = k & 63, nn = n & 63;
  const int lane = 16 * (kk >> 4) + 4 * (nn >> 4) + (nn & 3), t = (nn >> 2) & 3;
  return (((size_t)(n >> 6) * kblocks + (k >> 6)) * 4 + t) * 1024 + lane * 16 + (kk & 15);
}

// Weights, once per model: a workgroup takes 64 columns, its waves parts of K; scale and rounding per column.  W = int8_t: packing alone.
// 16 loads of a thread are under way at once (none behind a branch; what lies outside is read at the border and counts as 0).
// 4096 x 4096 fp16: 65 us, of int8: 27 us; the bytes alone would take 10 (64 workgroups on 256 CUs that read every weight twice).
constexpr int kPackParts = 16;
template <class W>
__global__ void __launch_bounds__(kPackParts * 64) k_pack_weight(const W *w, long long ldw, int8_t *packed, float *scale, int K, int N) {
  __shared__ unsigned lds_max[kPackParts][64];
  const int lane = threadIdx.x & 63, part = threadIdx.x >> 6, n = blockIdx.x * 64 + lane, kblocks = (K + 63) / 64;
  const W *column = w + min(n, N - 1);
  W v[16];
  RowScale rs = {1.f, 1.f, true};
  if constexpr (sizeof(W) > 1) {
    unsigned m = 0u;
    for (int k = part * 16; k < K; k += kPackParts * 16) {
#pragma unroll
      for (int b = 0; b < 16; ++b) v[b] = column[min(k + b, K - 1) * ldw];
#pragma unroll
      for (int b = 0; b < 16; ++b) m = max(m, abs_bits((float)v[b]));
    }
    lds_max[part][lane] = m;
    __syncthreads();
    m = 0u;
#pragma unroll
    for (int i = 0; i < kPackParts; ++i) m = max(m, lds_max[i][lane]);
    rs = row_scale(m);
    if (part == 0 && n < N) scale[n] = rs.scale;
  }
  for (int k = part * 16; k < kblocks * 64; k += kPackParts * 16) {      // 16 of K: one lane's 16 bytes
#pragma unroll
    for (int b = 0; b < 16; ++b) v[b] = column[min(k + b, K - 1) * ldw];
    unsigned d[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int b = 0; b < 16; ++b) {
      int q;
      if constexpr (sizeof(W) > 1) q = quantize((float)v[b], rs);
      else q = v[b];
      d[b >> 2] |= (k + b < K && n < N ? (unsigned)q & 255u : 0u) << (8 * (b & 3));
    }
    *reinterpret_cast<u4 *>(packed + packed_at(k, n, kblocks)) = u4{d[0], d[1], d[2], d[3]};
  }
}

// -------------------------------------------------------------------------------------------- products ----
struct Args {
  const int8_t *q;               // rows and their scales, or
  long long ldq;
  const float *row_scale;
  const void *x;                 // activations that the kernel quantises itself
  long long ldx;
  const int8_t *packed;
  const float *col_scale;
  const void *bias;              // of the output's type, nullable
  void *y;
  long long ldy;
  int M, N, K, act;
  int kblocks;                   // K / 64, rounded up
  int col_tiles;                 // workgroups along N
  int num_cus;
};

// 0.5 v (1 + erf(v / sqrt 2)) as max(v, 0) - 0.5 z erfc(z / sqrt 2), z = |v|: no digits are lost in the negative tail.  erfc(z / sqrt 2) =
// exp(-z^2 / 2) times a function that is smooth in t = 1 / (1 + p z) (the substitution of Abramowitz and Stegun 7.1.25 to 7.1.28, with p = 0.35
// here), half of it divided by t as a polynomial of degree 8 fitted for z in 0..20 for the least largest relative error: 5.2e-8 with
// the constants as they are rounded to fp32.  In all within 3 roundings of |v|, and 1e-6 of the result for z <= 4.  17 instructions and two at
// quarter rate, no branch: 8192 x 4096 -> 4096 takes 130 us with it and 114 without an activation (each call alone); the library's erf,
// whose two ranges a wave both runs through, was 10 us slower than it in a build that differed in nothing else.
__device__ __forceinline__ float gelu_exact(float v) {
  const float z = __builtin_fminf(__builtin_fabsf(v), 20.0f), t = __builtin_amdgcn_rcpf(__builtin_fmaf(z, 0.35f, 1.0f));
  constexpr float c[9] = {0.13962258398f, 0.13983604312f, 0.12006171793f, 0.10442747176f, -0.02011764981f, 0.15416617692f, -0.25073748827f, 0.14127224684f,
                          -0.02853108943f};
  float g = c[8];
#pragma unroll
  for (int i = 7; i >= 0; --i) g = __builtin_fmaf(g, t, c[i]);
  return (v < 0.f ? 0.f : v) - z * t * g * __builtin_amdgcn_exp2f(z * -0.72134752044f * z);
}
// NaN stays NaN in all of them.  The tanh GELU in its logistic form v / (1 + exp(-2 u)), u = 0.79788456 (v + 0.044715 v^3): exact
// in both tails (1 - 1 / (1 + exp 2u) would lose the negative one's digits); -infinity gives NaN, as the formula's own product does.
template <int ACT>
__device__ __forceinline__ float activate(float v) {
  if constexpr (ACT == SOUFFLE_ACT_RELU) return v < 0.f ? 0.f : v;
  if constexpr (ACT == SOUFFLE_ACT_GELU_TANH) {
    constexpr float K1 = -2.0f * 0.7978845608028654f * 1.4426950408889634f, K2 = K1 * 0.044715f;
    return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * __builtin_fmaf(v * v, K2, K1)));
  }
  if constexpr (ACT == SOUFFLE_ACT_GELU_ERF) return gelu_exact(v);
  return v;
}
template <int ACT>
struct ActTag {
  static constexpr int value = ACT;
};
// `f(tag)` with the activation as a constant: one branch per epilogue, not one per value.
template <class F>
__device__ __forceinline__ void with_activation(int act, F f) {
  if (act == SOUFFLE_ACT_NONE) f(ActTag<SOUFFLE_ACT_NONE>());
  else if (act == SOUFFLE_ACT_RELU) f(ActTag<SOUFFLE_ACT_RELU>());
  else if (act == SOUFFLE_ACT_GELU_TANH) f(ActTag<SOUFFLE_ACT_GELU_TANH>());
  else f(ActTag<SOUFFLE_ACT_GELU_ERF>());
}

// Scales and bias of four columns from n.
template <class T>
struct Columns4 {
  float scale[4], bias[4];
  __device__ __forceinline__ void load(const Args &a, int n) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int c = min(n + e, a.N - 1);
      scale[e] = a.col_scale[c];
      bias[e] = a.bias ? (float)static_cast<const T *>(a.bias)[c] : 0.f;
    }
  }
};
template <class T, int ACT>
__device__ __forceinline__ void finish4(const Args &a, int m, int n, i4 s, float rs, const Columns4<T> &col) {
  T *y = static_cast<T *>(a.y) + m * a.ldy + n;
  typedef T V4 __attribute__((ext_vector_type(4)));
  typedef T V4u __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  V4 out;
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e] = (T)activate<ACT>(((float)s[e] * col.scale[e]) * rs + col.bias[e]);
  if (n + 4 <= a.N) {
    *reinterpret_cast<V4u *>(y) = out;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < a.N) y[e] = out[e];
  }
}

// Few rows: a workgroup of W waves computes 16 MF rows x 16 NF columns, each wave a part of K with both operands straight from
// memory into registers (nothing is shared between waves, so nothing goes through LDS and the loop has no
// barrier), and the W partial sums meet in LDS at the end.  A wave's part is contiguous: two steps share the 128-byte
// lines of the rows.  Bound by the arrival of the weights: 24 x 4096 -> 8192 takes 9.4 us, 34 MB at 3.6 TB/s (U = 2; with 3 or 4
// steps asked for ahead 16 x 4096 -> 8192 takes 11.7 and 11.0 us instead of 10.3).
//
// ROWS: the rows come as activations, and every workgroup quantises its own into LDS itself while its first weights are under
// way: that repeats the work for each tile of columns, but costs a call less than a launch of its own in front of this one.
constexpr int kRowsK = 1024, kRowsPitch = kRowsK + 16;      // of tiles of 32 rows
template <RowForm FORM>
struct FormTag {
  static constexpr RowForm value = FORM;
};
template <class T, int MF, int NF, int W, int U, bool ROWS>
__global__ void __launch_bounds__(W * 64) k_gemm_split(const Args a) {
  static_assert(4 % NF == 0, "operands of the four that 64 columns have");
  static_assert(MF * NF <= W, "four results per thread");
  constexpr int kParts = 4 / NF;
  __shared__ i4 lds[W][MF * NF][64];
  __shared__ float lds_scale[16 * MF];
  extern __shared__ __attribute__((aligned(16))) unsigned char lds_dynamic[];      // ROWS: [M][64 kblocks + 16]
  __shared__ __attribute__((aligned(16))) unsigned char lds_static[ROWS && MF > 1 ? 16 * MF * kRowsPitch : 16];      // (more than 64 KB in all)
  unsigned char *lds_rows = MF > 1 ? lds_static : lds_dynamic;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = blockIdx.x % a.col_tiles, group = col / kParts, t0 = col % kParts * NF, m0 = blockIdx.x / a.col_tiles * 16 * MF;
  const int pitch = a.kblocks * 64 + 16, rows_here = min(16 * MF, a.M - m0);
  i4 acc[MF][NF] = {};
  const int8_t *wp = a.packed + ((size_t)group * a.kblocks * 4 + t0) * 1024 + lane * 16;
  const int8_t *xp[MF];
  const unsigned char *xrow[MF];
#pragma unroll
  for (int i = 0; i < MF; ++i) xrow[i] = lds_rows + min(16 * i + (lane & 15), rows_here - 1) * pitch + 16 * (lane >> 4);
#pragma unroll
  for (int i = 0; i < MF; ++i) xp[i] = a.q + min(m0 + 16 * i + (lane & 15), a.M - 1) * a.ldq + 16 * (lane >> 4);
  // U steps at a time, the next U loaded while the present ones are multiplied.  (A step behind the part's end reads its
  // last operands again, with the weights replaced by zeros.)
  const int part = (a.kblocks + W - 1) / W, k_first = wave * part, k_end = min(k_first + part, a.kblocks);
  i4 wv[U][NF], xv[U][MF];
  auto fetch = [&](int kb) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = min(kb + u, k_end - 1);
#pragma unroll
      for (int j = 0; j < NF; ++j) wv[u][j] = ldg16(wp + (size_t)k * 4096 + j * 1024);
      if constexpr (!ROWS)
#pragma unroll
        for (int i = 0; i < MF; ++i) xv[u][i] = ldg16(xp[i] + k * 64);
    }
  };
  if (k_first < k_end) fetch(k_first);
  // The thread's four results and what their epilogue needs, asked for now.
  const int out_tile = threadIdx.x >> 6, out_m = m0 + 16 * (out_tile / NF) + (lane & 15), out_n = group * 64 + 16 * (lane >> 4) + 4 * (t0 + out_tile % NF);
  const bool has_out = out_tile < MF * NF && out_m < a.M && out_n < a.N;
  Columns4<T> columns;
  float rs = 0.f;
  if (has_out) {
    columns.load(a, out_n);
    if constexpr (!ROWS) rs = a.row_scale[out_m];
  }
  if constexpr (ROWS && MF > 1) {
    // every wave has its share of the rows (at most 1024 elements each), all asked for at once
    constexpr int R = 16 * MF / W;
    auto quantise = [&](auto form) {
      constexpr RowForm FORM = decltype(form)::value;
      typename Vec8<T>::type v[R][2];
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          v[r][i] = load_row<FORM>(static_cast<const T *>(a.x) + (m0 + min(wave * R + r, rows_here - 1)) * a.ldx, (i * 64 + lane) * 8, a.K);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int row = wave * R + r;
        float f[2][8];
        unsigned m = 0u;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          to_f32(f[i], settle_row<FORM, T>(v[r][i], (i * 64 + lane) * 8, a.K));
#pragma unroll
          for (int e = 0; e < 8; ++e) m = max(m, abs_bits(f[i][e]));
        }
        const RowScale rs = row_scale(wave_umax_dpp(m));
        if (row < rows_here) {
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if ((i * 64 + lane) * 8 < a.K) *reinterpret_cast<u2 *>(lds_rows + row * pitch + (i * 64 + lane) * 8) = quantize8(f[i], rs);
          if (lane == 0) lds_scale[row] = rs.scale;
        }
      }
    };
    if (a.K % 8 == 0) quantise(FormTag<kWhole>());
    else if (a.K > 8) quantise(FormTag<kRagged>());
    else quantise(FormTag<kShort>());
    __syncthreads();
  } else if constexpr (ROWS) {
    // as many waves per row as there are for M rows at a time
    __shared__ unsigned lds_max[2][W];
    const int per_row = a.M == 1 ? W : a.M == 2 ? W / 2 : a.M <= 4 ? W / 4 : W / 8, slots = W / per_row;
    const int c0 = (wave % per_row * 64 + lane) * 8, stride = per_row * 512;
    for (int base = 0, turn = 0; base < a.M; base += slots, turn ^= 1) {
      const int row = base + wave / per_row;
      const T *x = static_cast<const T *>(a.x) + min(row, a.M - 1) * a.ldx;
      auto values = [&](float (&f)[8], int c) {
        if (a.K % 8 == 0) to_f32(f, settle_row<kWhole, T>(load_row<kWhole>(x, c, a.K), c, a.K));
        else if (a.K > 8) to_f32(f, settle_row<kRagged, T>(load_row<kRagged>(x, c, a.K), c, a.K));
        else to_f32(f, settle_row<kShort, T>(load_row<kShort>(x, c, a.K), c, a.K));
      };
      float first[8], f[8];
      values(first, c0);
      unsigned m = 0u;
#pragma unroll
      for (int e = 0; e < 8; ++e) m = max(m, abs_bits(first[e]));
      for (int c = c0 + stride; c < a.K; c += stride) {
        values(f, c);
#pragma unroll
        for (int e = 0; e < 8; ++e) m = max(m, abs_bits(f[e]));
      }
      m = wave_umax_dpp(m);
      if (per_row > 1) {
        if (lane == 0) lds_max[turn][wave] = m;
        __syncthreads();
        for (int w = 0; w < per_row; ++w) m = max(m, lds_max[turn][wave / per_row * per_row + w]);
      }
      const RowScale rs = row_scale(m);
      if (row < a.M) {
        if (c0 < a.K) *reinterpret_cast<u2 *>(lds_rows + row * pitch + c0) = quantize8(first, rs);
        for (int c = c0 + stride; c < a.K; c += stride) {
          values(f, c);
          *reinterpret_cast<u2 *>(lds_rows + row * pitch + c) = quantize8(f, rs);
        }
        if (lane == 0) lds_scale[row] = rs.scale;
      }
    }
    __syncthreads();
  }
  for (int kb = k_first; kb < k_end; kb += U) {
    i4 wn[U][NF], xn[U][MF];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int j = 0; j < NF; ++j) wn[u][j] = kb + u < k_end ? wv[u][j] : i4{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < MF; ++i) {
        if constexpr (ROWS) xn[u][i] = __builtin_bit_cast(i4, lds_load16(xrow[i] + min(kb + u, k_end - 1) * 64));
        else xn[u][i] = xv[u][i];
      }
    }
    if (kb + U < k_end) fetch(kb + U);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int j = 0; j < NF; ++j) acc[i][j] = mfma_i8(wn[u][j], xn[u][i], acc[i][j]);
  }
#pragma unroll
  for (int i = 0; i < MF; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j) lds[wave][i * NF + j][lane] = acc[i][j];
  __syncthreads();
  if (!has_out) return;
  if constexpr (ROWS) rs = lds_scale[out_m - m0];
  i4 sum = lds[0][out_tile][lane];
#pragma unroll
  for (int w = 1; w < W; ++w) sum += lds[w][out_tile][lane];
  with_activation(a.act, [&](auto act) { finish4<T, decltype(act)::value>(a, out_m, out_n, sum, rs, columns); });
}

// Rows of 16 lanes: the odd ones of a change places with the even ones of b (permlane16), the upper two of a with the lower two of b (permlane32).
template <class V>
__device__ __forceinline__ void swap16(V &a, V &b) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const auto p = __builtin_amdgcn_permlane16_swap(a[e], b[e], false, false);
    a[e] = p[0];
    b[e] = p[1];
  }
}
template <class V>
__device__ __forceinline__ void swap32(V &a, V &b) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const auto p = __builtin_amdgcn_permlane32_swap(a[e], b[e], false, false);
    a[e] = p[0];
    b[e] = p[1];
  }
}
// The 64 columns from n0 of row m, 16 of them (from 16 g, g = lane / 16) in this lane, with their scales and bias in registers.  The
// 16-byte pieces change places between the four lanes of a row, so that these store 64 bytes in a row each time.
template <class T, int ACT>
__device__ __forceinline__ void finish16(const Args &a, int m, int n0, const i4 (&s)[4], float rs, const float (&cs)[16], const float (&bias)[16]) {
  const int g = (threadIdx.x & 63) >> 4;
  constexpr int kPer = 16 / sizeof(T), kPieces = 16 / kPer;      // elements of a piece; pieces of a lane
  u4 piece[kPieces];
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    typedef T V __attribute__((ext_vector_type(kPer)));
    V v;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int c = kPer * k + e;
      v[e] = (T)activate<ACT>(((float)s[c >> 2][c & 3] * cs[c]) * rs + bias[c]);
    }
    piece[k] = __builtin_bit_cast(u4, v);
  }
  swap16(piece[0], piece[1]);
  if constexpr (kPieces == 2) {
    swap32(piece[0], piece[1]);
  } else {
    swap16(piece[2], piece[3]);
    swap32(piece[0], piece[2]);
    swap32(piece[1], piece[3]);
  }
  if (m >= a.M) return;
  T *y = static_cast<T *>(a.y) + m * a.ldy;
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    const int n = n0 + (4 * k + g) * kPer;
    typedef T V __attribute__((ext_vector_type(kPer)));
    typedef T Vu __attribute__((ext_vector_type(kPer), aligned(sizeof(T))));
    const V v = __builtin_bit_cast(V, piece[k]);
    if (n + kPer <= a.N) {
      *(__attribute__((address_space(1))) Vu *)(y + n) = v;
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        if (n + e < a.N) y[n + e] = v[e];
    }
  }
}

__device__ const int8_t zero_bytes[16] __attribute__((aligned(16))) = {};

// Many rows: a workgroup of WM x WN waves computes 16 MI WM rows x 64 WN columns, 128 of K at a time.  A wave holds MI x 4 accumulator
// tiles.  The rows go through LDS (every wave of a row of waves needs them) in a ring of three stages filled by
// direct loads, two steps ahead; the packed weights go straight into registers one step ahead, a wave's 64 columns being 4 KB in a
// row per 64 of K: through LDS as well they would double its traffic, which at 128 bytes a cycle is
// what runs out first (a 256 x 256 tile then asks for 64 + 32 + 32 bytes per cycle of matrix instructions).  8192 x 4096 x 4096 takes
// 114 us alone (median; 2410 TOP/s) and 122 to 129 in a row of calls, where the clock sinks (the library's product of these sizes 131 and 137):
// the matrix cores are busy in 73 % of the cycles, LDS has no conflicts, 202 MB are read; without any load in the loop it would be 87 us.
//
// LDS stage [BM rows][8 slots of 16 bytes]: slot p of row r holds bytes 16 (p ^ (r / 2 % 8)) .. + 15 of the row's 128, so that the 16
// rows of an operand read lie in different banks (64 banks are two rows); a direct load of 8 rows x 128 bytes fills 1 KB.
template <class T, int MI, int WM, int WN>
__global__ void __launch_bounds__(WM * WN * 64) k_gemm_tile(const Args a) {
  constexpr int kWaves = WM * WN, kBM = 16 * MI * WM, kStage = kBM * 128, kLoads = kBM / 8 / kWaves, kWLoads = 8;
  static_assert(kLoads * kWaves * 8 == kBM && kLoads <= MI && kWLoads % MI == 0, "every wave fills the same number of KB of a stage, in half a step");
  __shared__ __attribute__((aligned(16))) unsigned char lds[3 * kStage + (kBM + 64 * WN) * 4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
  // Workgroup b runs on XCD b % 8: each XCD takes a run of tiles, eight rows of tiles deep, so that what its L2 holds is shared.
  const int row_tiles = (a.M + kBM - 1) / kBM, tiles = row_tiles * a.col_tiles;
  const int per_xcd = tiles / 8, left = tiles % 8, xcd = blockIdx.x % 8;
  const int tile = xcd * per_xcd + min(xcd, left) + blockIdx.x / 8;
  const int band = tile / (8 * a.col_tiles), deep = min(8, row_tiles - 8 * band), in_band = tile - band * 8 * a.col_tiles;
  const int m0 = (band * 8 + in_band % deep) * kBM, group = in_band / deep * WN + wn, last_group = (a.N + 63) / 64 - 1;

  const unsigned lds0 = lds_address(lds);
  const int k_end = a.kblocks * 64;
  const int8_t *src[kLoads];
  int chunk[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int row = (wave * kLoads + i) * 8 + (lane >> 3);
    src[i] = a.q + min(m0 + row, a.M - 1) * a.ldq;
    chunk[i] = ((lane & 7) ^ (row >> 1 & 7)) * 16;
  }
  // (behind K's end: zeros, so that steps come in pairs, always with the same loads, and the loop has no branch)
  auto stage_in = [&](int s, int slot, int i) {
    const int off = s * 128 + chunk[i];
    load_lds16(off < k_end ? src[i] + off : zero_bytes, lds0 + slot * kStage + (wave * kLoads + i) * 1024);
  };
  const int8_t *wp = a.packed + (size_t)min(group, last_group) * a.kblocks * 4096 + lane * 16;
  auto fetch_w = [&](i4 (&w)[2][4], int s, int i) { w[i / 4][i % 4] = ldg16(wp + (size_t)min(2 * s + i / 4, a.kblocks - 1) * 4096 + i % 4 * 1024); };
  i4 acc[MI][4];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = i4{0, 0, 0, 0};
  const int r = lane & 15, g = lane >> 4;
  const unsigned char *rows = lds + (wm * 16 * MI + r) * 128;
  auto row16 = [&](int slot, int i, int h) {
    return __builtin_bit_cast(i4, lds_load16(rows + slot * kStage + i * 2048 + (((h * 4 + g) ^ (r >> 1 & 7)) * 16)));
  };
  // Stage s of the ring with its weights in w; those of s + 1 go to wnext.  The 2 MI operands of rows are read two ahead of their use, across
  // the step's end, so the one barrier of a step stands in its middle: it says that the rows of s + 1 are there and that nobody reads
  // those of s - 1 any more.  A wave's loads are queued one by one between the matrix instructions (in a burst, all waves at once, each
  // stands still until the texture unit takes its next one), in the order weights of s + 1, rows of s + 2 | ...  The
  // compiler waits for weights at their first use and does not count the direct loads, so these are queued behind
  // the step's last first use: its count, too small by that many, then only asks for loads that are a step old.
  i4 x0, x1;
  auto step = [&](int s, int slot, i4 (&w)[2][4], i4 (&wnext)[2][4]) {
    const int slot1 = slot == 2 ? 0 : slot + 1, slot2 = slot == 0 ? 2 : slot - 1;
#pragma unroll
    for (int u = 0; u < 2 * MI; ++u) {
      const i4 x2 = u + 2 < 2 * MI ? row16(slot, (u + 2) % MI, (u + 2) / MI) : row16(slot1, u + 2 - 2 * MI, 0);
      if (u < MI)
#pragma unroll
        for (int i = u * kWLoads / MI; i < (u + 1) * kWLoads / MI; ++i) fetch_w(wnext, s + 1, i);
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[u % MI][j] = mfma_i8(w[u / MI][j], x0, acc[u % MI][j]);
      x0 = x1;
      x1 = x2;
      if (u == MI - 1) {
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kWLoads) : "memory");
        __builtin_amdgcn_s_barrier();
        compiler_fence();
      }
      __builtin_amdgcn_sched_barrier(0);      // (otherwise the reads sink to their uses)
      if (u >= MI && u - MI < kLoads) stage_in(s + 2, slot2, u - MI);
    }
  };
  // The scales of the tile's rows and columns wait for the epilogue in LDS, behind the stages.
  float *row_scale = reinterpret_cast<float *>(lds + 3 * kStage), *col_scale = row_scale + kBM;
#pragma unroll
  for (int i = 0; i < (kBM / 64 + WN + kWaves - 1) / kWaves; ++i) {
    const int part = wave + i * kWaves, c = (in_band / deep * WN + part - kBM / 64) * 64 + lane;
    const float *from = part < kBM / 64 ? a.row_scale + min(m0 + part * 64 + lane, a.M - 1) : a.col_scale + min(c, a.N - 1);
    if (part < kBM / 64 + WN) load_lds4(from, lds0 + 3 * kStage + part * 256);
  }
  i4 w0[2][4], w1[2][4];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) stage_in(0, 0, i);
#pragma unroll
  for (int i = 0; i < kLoads; ++i) stage_in(1, 1, i);
#pragma unroll
  for (int i = 0; i < kWLoads; ++i) fetch_w(w0, 0, i);
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kWLoads + kLoads) : "memory");
  __builtin_amdgcn_s_barrier();
  compiler_fence();
  x0 = row16(0, 0, 0);
  x1 = row16(0, 1, 0);
  for (int s = 0, slot = 0; 2 * s < a.kblocks; s += 2) {
    step(s, slot, w0, w1);
    slot = slot == 2 ? 0 : slot + 1;
    step(s + 1, slot, w1, w0);
    slot = slot == 2 ? 0 : slot + 1;
  }
  wait_vmcnt<0>();      // no direct load is under way when the workgroup gives its LDS back
  const int n = group * 64 + 16 * g;
  float cs[16], bias[16];
#pragma unroll
  for (int c = 0; c < 16; ++c) {
    cs[c] = col_scale[wn * 64 + 16 * g + c];
    bias[c] = 0.f;
  }
  if (a.bias) {
    float b[2][8];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      to_f32(b[half], load8(static_cast<const T *>(a.bias), n + 8 * half, a.N));
#pragma unroll
      for (int e = 0; e < 8; ++e) bias[8 * half + e] = b[half][e];
    }
  }
  // One row tile at a time through one copy of the code: unrolled, the epilogue is 64 lines of instructions that every launch
  // fetches once and runs once.
  with_activation(a.act, [&](auto act) {
#pragma unroll 1
    for (int i = 0; i < MI; ++i) {
      i4 v[4];
#pragma unroll
      for (int k = 0; k < MI; ++k)
        if (i == k)
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = acc[k][j];
      finish16<T, decltype(act)::value>(a, m0 + (wm * MI + i) * 16 + r, group * 64, v, row_scale[(wm * MI + i) * 16 + r], cs, bias);
    }
  });
}

// ------------------------------------------------------------------------------------------- host side ----
constexpr int kMaxK = 131071;      // 128 * 128 * K stays below 2^31
constexpr int kMaxRows = 1 << 30;

static bool known_dtype(int t) { return t == SOUFFLE_F16 || t == SOUFFLE_BF16 || t == SOUFFLE_F32; }
static unsigned size_of(int t) { return t == SOUFFLE_F32 ? 4 : 2; }

static int check_kn(int K, int N) {
  if (K < 1 || K > kMaxK) return fail(SOUFFLE_ERR_SHAPE, "K must be in 1..%d (got %d)", kMaxK, K);
  if (N < 1 || N > (1 << 24)) return fail(SOUFFLE_ERR_SHAPE, "N must be in 1..2^24 (got %d)", N);
  return SOUFFLE_OK;
}
static int check_q(const void *q, long long ldq, int K) {
  if (!aligned16(q) || ldq % 16) return fail(SOUFFLE_ERR_ALIGN, "the rows of q must be 16-byte aligned");
  if (ldq < (long long)round_up(K, 64)) return fail(SOUFFLE_ERR_SHAPE, "ldq must be at least K rounded up to 64 (got %lld)", ldq);
  return SOUFFLE_OK;
}
static int check_x(const char *name, const void *x, int dtype, long long ld, int cols) {
  if (reinterpret_cast<uintptr_t>(x) % size_of(dtype)) return fail(SOUFFLE_ERR_ALIGN, "%s is not aligned to its elements", name);
  if (ld < cols) return fail(SOUFFLE_ERR_SHAPE, "the rows of %s overlap: stride %lld, %d columns", name, ld, cols);
  return SOUFFLE_OK;
}

constexpr int kMostRowGroups = 1 << 22;      // (a launch holds fewer than 2^32 threads; beyond that a workgroup takes several rows)
template <RowForm FORM, class T>
static void launch_quantize(const T *x, long long ldx, int8_t *q, long long ldq, float *scale, int M, int K, hipStream_t st) {
  const dim3 wide(std::min(M, kMostRowGroups)), narrow(std::min((M + 3) / 4, kMostRowGroups)), block(256);
  if (K <= 128) hipLaunchKernelGGL((k_quantize_rows<T, 16, 1, FORM>), dim3(std::min((M + 15) / 16, kMostRowGroups)), block, 0, st, x, ldx, q, ldq, scale, M, K);
  else if (K <= 512) hipLaunchKernelGGL((k_quantize_rows<T, 64, 1, FORM>), narrow, block, 0, st, x, ldx, q, ldq, scale, M, K);
  else if (K <= 1024) hipLaunchKernelGGL((k_quantize_rows<T, 64, 2, FORM>), narrow, block, 0, st, x, ldx, q, ldq, scale, M, K);
  else if (K <= 2048) hipLaunchKernelGGL((k_quantize_rows<T, 256, 1, FORM>), wide, block, 0, st, x, ldx, q, ldq, scale, M, K);
  else if (K <= 4096) hipLaunchKernelGGL((k_quantize_rows<T, 256, 2, FORM>), wide, block, 0, st, x, ldx, q, ldq, scale, M, K);
  else if (K <= 8192) hipLaunchKernelGGL((k_quantize_rows<T, 256, 4, FORM>), wide, block, 0, st, x, ldx, q, ldq, scale, M, K);
  else hipLaunchKernelGGL((k_quantize_rows<T, 256, 0, FORM>), wide, block, 0, st, x, ldx, q, ldq, scale, M, K);
}
template <class T>
static int quantize_rows(const void *xv, long long ldx, int8_t *q, long long ldq, float *scale, int M, int K, hipStream_t st) {
  const T *x = static_cast<const T *>(xv);
  if (K < 8) hipLaunchKernelGGL((k_quantize_rows<T, 16, 1, kShort>), dim3(std::min((M + 15) / 16, kMostRowGroups)), dim3(256), 0, st, x, ldx, q, ldq, scale, M, K);
  else if (K % 8) launch_quantize<kRagged>(x, ldx, q, ldq, scale, M, K, st);
  else launch_quantize<kWhole>(x, ldx, q, ldq, scale, M, K, st);
  SOUFFLE_HIP_TRY(hipGetLastError());
  return SOUFFLE_OK;
}
static int quantize_rows(const void *x, int dtype, long long ldx, int8_t *q, long long ldq, float *scale, int M, int K, hipStream_t st) {
  if (dtype == SOUFFLE_F16) return quantize_rows<half_t>(x, ldx, q, ldq, scale, M, K, st);
  if (dtype == SOUFFLE_BF16) return quantize_rows<bf16_t>(x, ldx, q, ldq, scale, M, K, st);
  return quantize_rows<float>(x, ldx, q, ldq, scale, M, K, st);
}

// One workgroup per tile.  (Tiles narrower than 64 columns interleave: there are 64 / cols of them for any part of 64.)
static int grid_of(const Args &a, int rows, int cols, int threads, unsigned *grid, int *col_tiles) {
  *col_tiles = cols < 64 ? (a.N + 63) / 64 * (64 / cols) : (a.N + cols - 1) / cols;
  const long long n = (long long)*col_tiles * ((a.M + rows - 1) / rows);
  if (n * threads > 0xffffffffll) return fail(SOUFFLE_ERR_SHAPE, "M = %d rows of N = %d are more tiles than one launch holds", a.M, a.N);
  *grid = (unsigned)n;
  return SOUFFLE_OK;
}
template <class T, int MF, int NF, int W, int U>
static int launch_split(Args a, hipStream_t st) {
  unsigned grid;
  if (int rc = grid_of(a, 16 * MF, 16 * NF, W * 64, &grid, &a.col_tiles)) return rc;
  hipLaunchKernelGGL((k_gemm_split<T, MF, NF, W, U, false>), dim3(grid), dim3(W * 64), 0, st, a);
  SOUFFLE_HIP_TRY(hipGetLastError());
  return SOUFFLE_OK;
}
template <class T, int MF, int NF, int U>
static int launch_rows(Args a, hipStream_t st) {
  unsigned grid;
  if (int rc = grid_of(a, 16 * MF, 16 * NF, 512, &grid, &a.col_tiles)) return rc;
  hipLaunchKernelGGL((k_gemm_split<T, MF, NF, 8, U, true>), dim3(grid), dim3(512), MF > 1 ? 0 : a.M * (a.kblocks * 64 + 16), st, a);
  SOUFFLE_HIP_TRY(hipGetLastError());
  return SOUFFLE_OK;
}
template <class T, int MI, int WM, int WN>
static int launch_tile(Args a, hipStream_t st) {
  unsigned grid;
  if (int rc = grid_of(a, 16 * MI * WM, 64 * WN, WM * WN * 64, &grid, &a.col_tiles)) return rc;
  hipLaunchKernelGGL((k_gemm_tile<T, MI, WM, WN>), dim3(grid), dim3(WM * WN * 64), 0, st, a);
  SOUFFLE_HIP_TRY(hipGetLastError());
  return SOUFFLE_OK;
}
static long long tiles(int M, int rows, int N, int cols) { return (long long)((M + rows - 1) / rows) * ((N + cols - 1) / cols); }

// Which kernel: the one with the most work per workgroup that still gives the CUs enough workgroups.  Measured on the GPU (bf16
// out, us, the best of several runs; split = 32 x 32 / 32 x 64 with the waves along K, tiles of 64 x 128 with four waves | with two | 128 x 128 | 256 x 256):
//   64 x 4096 x 4096      7.5 /  8.3   15.3 | 17.4 | 21.0 | 44.7       512 x 4096 x 4096    39 / 25   16.3 | 18.3 | 21.8 | 48.2
//   384 x 768 x 768       4.3 /  3.7    5.7 |  6.6 |  7.8 | 15.2       1024 x 768 x 2304    15 / 10    8.4 |  8.2 |  7.8 | 14.5
//   8192 x 768 x 2304      99 /   62   30.1 | 26.5 | 26.7 | 30.2       5760 x 1600 x 1925   85 / 63   43.5 | 37.3 | 33.6 | 32.7
//   8192 x 4096 x 4096    315 (per 64 x 64)  184 | 149 | 142 | 112      600 x 2048 x 8192   -  / 35   21.3 | 17.4 | 19.1 | 24.0
//   4096 x 768 x 768       - / 12.6   8.5 |  8.4 |  7.5 | 13.4       5000 x 8192 x 800    - / 112  68.8 | 48.7 | 55.2 | 72.0
// Between the smallest and the largest products these stay at two to four times the floor: output tiles are whole, so the last round of
// workgroups is part empty, and with few steps of K nothing hides a workgroup's first loads and its epilogue.
// (8192 x 768 x 2304: 288 tiles of 256 x 256 on 256 CUs: the second round is an eighth full; 600 x 2048 x 8192: 320 tiles of
// 128 x 128, so some CUs get two where tiles of 64 rows give them three halves.)
template <class T>
static int gemm(const Args &a, hipStream_t st) {
  const long long cus = a.num_cus, big = tiles(a.M, 256, a.N, 256), rounds = (big + cus - 1) / cus;
  if (a.M <= 16) return tiles(a.M, 16, a.N, 16) <= cus ? launch_split<T, 1, 1, 8, 4>(a, st) : launch_split<T, 1, 4, 8, 2>(a, st);
  if (tiles(a.M, 32, a.N, 32) <= cus) return launch_split<T, 2, 2, 8, 2>(a, st);
  if (tiles(a.M, 32, a.N, 64) <= 2 * cus) return launch_split<T, 2, 4, 8, 1>(a, st);
  if (tiles(a.M, 64, a.N, 128) <= cus) return launch_tile<T, 2, 2, 2>(a, st);
  if (rounds == 1 ? big * 16 >= cus * 9 : big * 10 >= rounds * cus * 7) return launch_tile<T, 8, 2, 4>(a, st);
  // the most 64 rows that one CU gets, as tiles of 128 and of 64 rows
  const long long pairs = 2 * ((tiles(a.M, 128, a.N, 128) + cus - 1) / cus), singles = (tiles(a.M, 64, a.N, 128) + cus - 1) / cus;
  return pairs * 9 <= singles * 10 ? launch_tile<T, 4, 2, 2>(a, st) : launch_tile<T, 4, 1, 2>(a, st);
}
static int gemm(const Args &a, int dtype, hipStream_t st) {
  if (dtype == SOUFFLE_F16) return gemm<half_t>(a, st);
  if (dtype == SOUFFLE_BF16) return gemm<bf16_t>(a, st);
  return gemm<float>(a, st);
}
// Whether the product's workgroups quantise the rows themselves (one launch, no workspace).  Measured on the GPU in one launch and in
// two, us: 1 x 768 -> 2304 3.7 and 5.0, 2 x 4096 -> 8192 9.1 and 10.1, 4 x 4096 -> 4096 9.0 and 8.9, 8 x 4096 -> 4096 11.5 and 9.2, 16 x 1024 ->
// 4096 6.0 and 6.0; tiles of 32 rows: 32 x 512 -> 512 5.7 and 6.4, 384 x 768 -> 768 7.8 and 7.3, 128 x 1024 -> 4096 8.1 and 7.6, 333 x 1000 ->
// 1111 fp32 8.4 and 7.7, 640 x 768 -> 768 7.7 and 7.7 (captured in a graph: 384 rows 7.7 and 7.1, 128 rows 8.1 and 7.3, 32 rows 6.1 and 6.5).
// One call after another, which the host bounds, takes 8.8 and 12.9 in all of these.
constexpr int kOneRound = 256;      // workgroups, one per CU: 98 KB of LDS each
static bool rows_in_kernel(int M, int N, int K) {
  return M <= 16 ? (long long)M * K <= 16384 : K <= kRowsK && tiles(M, 32, N, 64) <= kOneRound;
}
template <class T>
static int linear_rows(const Args &a, hipStream_t st) {
  if (a.M > 16) return tiles(a.M, 32, a.N, 32) <= a.num_cus ? launch_rows<T, 2, 2, 2>(a, st) : launch_rows<T, 2, 4, 1>(a, st);
  return tiles(a.M, 16, a.N, 16) <= a.num_cus ? launch_rows<T, 1, 1, 4>(a, st) : launch_rows<T, 1, 4, 2>(a, st);
}

static int check_product(const void *packed, const float *col_scale, const void *bias, int act, const void *y, int dtype, long long ldy, int M,
                         int N, int K) {
  if (M < 0 || M > kMaxRows) return fail(SOUFFLE_ERR_SHAPE, "M must be in 0..2^30 (got %d)", M);
  if (int rc = check_kn(K, N)) return rc;
  if (!known_dtype(dtype)) return fail(SOUFFLE_ERR_SHAPE, "unknown dtype %d", dtype);
  if (act != SOUFFLE_ACT_NONE && act != SOUFFLE_ACT_RELU && act != SOUFFLE_ACT_GELU_TANH && act != SOUFFLE_ACT_GELU_ERF)
    return fail(SOUFFLE_ERR_SHAPE, "unknown activation %d", act);
  if (M == 0) return SOUFFLE_OK;
  if (!packed || !col_scale || !y) return fail(SOUFFLE_ERR_NULL, "packed, col_scale and y must not be NULL");
  if (!aligned16(packed)) return fail(SOUFFLE_ERR_ALIGN, "packed must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(col_scale) % 4 || reinterpret_cast<uintptr_t>(bias) % size_of(dtype))
    return fail(SOUFFLE_ERR_ALIGN, "col_scale or bias is not aligned to its elements");
  return check_x("y", y, dtype, ldy, N);
}

}  // namespace linear_int8
}  // namespace souffle

using namespace souffle;
using namespace souffle::linear_int8;

extern "C" size_t souffle_int8_packed_bytes(int K, int N) {
  if (check_kn(K, N)) return 0;
  return round_up(K, 64) * round_up(N, 64);
}

extern "C" int souffle_int8_pack_weight(const int8_t *w, long long ldw, void *packed, int K, int N, souffle_stream_t stream) {
  if (int rc = check_kn(K, N)) return rc;
  if (!w || !packed) return fail(SOUFFLE_ERR_NULL, "w and packed must not be NULL");
  if (!aligned16(packed)) return fail(SOUFFLE_ERR_ALIGN, "packed must be 16-byte aligned");
  if (ldw < N) return fail(SOUFFLE_ERR_SHAPE, "the rows of w overlap: stride %lld, %d columns", ldw, N);
  DeviceFacts df;
  if (int rc = device_facts(&df)) return rc;
  hipLaunchKernelGGL(k_pack_weight<int8_t>, dim3((N + 63) / 64), dim3(kPackParts * 64), 0, static_cast<hipStream_t>(stream), w, ldw, static_cast<int8_t *>(packed),
                     static_cast<float *>(nullptr), K, N);
  SOUFFLE_HIP_TRY(hipGetLastError());
  return SOUFFLE_OK;
}

extern "C" int souffle_int8_quantize_weight(const void *w, int dtype, long long ldw, void *packed, float *col_scale, int K, int N, souffle_stream_t stream) {
  if (int rc = check_kn(K, N)) return rc;
  if (!known_dtype(dtype)) return fail(SOUFFLE_ERR_SHAPE, "unknown dtype %d", dtype);
  if (!w || !packed || !col_scale) return fail(SOUFFLE_ERR_NULL, "w, packed and col_scale must not be NULL");
  if (!aligned16(packed) || reinterpret_cast<uintptr_t>(col_scale) % 4) return fail(SOUFFLE_ERR_ALIGN, "packed must be 16-byte aligned, col_scale to its elements");
  if (int rc = check_x("w", w, dtype, ldw, N)) return rc;
  DeviceFacts df;
  if (int rc = device_facts(&df)) return rc;
  const dim3 grid((N + 63) / 64), block(kPackParts * 64);
  hipStream_t st = static_cast<hipStream_t>(stream);
  int8_t *p = static_cast<int8_t *>(packed);
  if (dtype == SOUFFLE_F16) hipLaunchKernelGGL(k_pack_weight<half_t>, grid, block, 0, st, static_cast<const half_t *>(w), ldw, p, col_scale, K, N);
  else if (dtype == SOUFFLE_BF16) hipLaunchKernelGGL(k_pack_weight<bf16_t>, grid, block, 0, st, static_cast<const bf16_t *>(w), ldw, p, col_scale, K, N);
  else hipLaunchKernelGGL(k_pack_weight<float>, grid, block, 0, st, static_cast<const float *>(w), ldw, p, col_scale, K, N);
  SOUFFLE_HIP_TRY(hipGetLastError());
  return SOUFFLE_OK;
}

extern "C" int souffle_quantize_rows(const void *x, int dtype, long long ldx, int8_t *q, long long ldq, float *row_scale, int M, int K,
                                     souffle_stream_t stream) {
  if (M < 0 || M > kMaxRows) return fail(SOUFFLE_ERR_SHAPE, "M must be in 0..2^30 (got %d)", M);
  if (int rc = check_kn(K, 1)) return rc;
  if (!known_dtype(dtype)) return fail(SOUFFLE_ERR_SHAPE, "unknown dtype %d", dtype);
  if (M == 0) return SOUFFLE_OK;
  if (!x || !q || !row_scale) return fail(SOUFFLE_ERR_NULL, "x, q and row_scale must not be NULL");
  if (int rc = check_x("x", x, dtype, ldx, K)) return rc;
  if (int rc = check_q(q, ldq, K)) return rc;
  if (reinterpret_cast<uintptr_t>(row_scale) % 4) return fail(SOUFFLE_ERR_ALIGN, "row_scale is not aligned to its elements");
  DeviceFacts df;
  if (int rc = device_facts(&df)) return rc;
  return quantize_rows(x, dtype, ldx, q, ldq, row_scale, M, K, static_cast<hipStream_t>(stream));
}

extern "C" int souffle_gemm_int8(const int8_t *q, long long ldq, const float *row_scale, const void *packed, const float *col_scale,
                                 const void *bias, int act, void *y, int dtype, long long ldy, int M, int N, int K, souffle_stream_t stream) {
  if (int rc = check_product(packed, col_scale, bias, act, y, dtype, ldy, M, N, K)) return rc;
  if (M == 0) return SOUFFLE_OK;
  if (!q || !row_scale) return fail(SOUFFLE_ERR_NULL, "q and row_scale must not be NULL");
  if (int rc = check_q(q, ldq, K)) return rc;
  if (reinterpret_cast<uintptr_t>(row_scale) % 4) return fail(SOUFFLE_ERR_ALIGN, "row_scale is not aligned to its elements");
  DeviceFacts df;
  if (int rc = device_facts(&df)) return rc;
  const Args a = {q, ldq, row_scale, nullptr, 0, static_cast<const int8_t *>(packed), col_scale, bias, y, ldy, M, N, K, act, (K + 63) / 64, 0, df.num_cus};
  return gemm(a, dtype, static_cast<hipStream_t>(stream));
}

extern "C" size_t souffle_linear_int8_workspace_bytes(int M, int N, int K) {
  if (M < 0 || M > kMaxRows || check_kn(K, N) || rows_in_kernel(M, N, K)) return 0;
  return round_up((size_t)M * round_up(K, 64) + (size_t)M * 4, 256);
}

extern "C" int souffle_linear_int8(const void *x, long long ldx, const void *packed, const float *col_scale, const void *bias, int act, void *y,
                                   int dtype, long long ldy, int M, int N, int K, void *ws, size_t ws_bytes, souffle_stream_t stream) {
  if (int rc = check_product(packed, col_scale, bias, act, y, dtype, ldy, M, N, K)) return rc;
  if (M == 0) return SOUFFLE_OK;
  if (!x) return fail(SOUFFLE_ERR_NULL, "x must not be NULL");
  if (int rc = check_x("x", x, dtype, ldx, K)) return rc;
  const size_t need = souffle_linear_int8_workspace_bytes(M, N, K);
  if (need && (!ws || ws_bytes < need)) return fail(SOUFFLE_ERR_WORKSPACE, "workspace too small: need %zu bytes", need);
  if (need && !aligned16(ws)) return fail(SOUFFLE_ERR_ALIGN, "workspace must be 16-byte aligned");
  DeviceFacts df;
  if (int rc = device_facts(&df)) return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  Args a = {nullptr, 0, nullptr, x, ldx, static_cast<const int8_t *>(packed), col_scale, bias, y, ldy, M, N, K, act, (K + 63) / 64, 0, df.num_cus};
  if (need == 0) {
    if (dtype == SOUFFLE_F16) return linear_rows<half_t>(a, st);
    if (dtype == SOUFFLE_BF16) return linear_rows<bf16_t>(a, st);
    return linear_rows<float>(a, st);
  }
  const long long ldq = (long long)round_up(K, 64);
  int8_t *q = static_cast<int8_t *>(ws);
  float *row_scale = reinterpret_cast<float *>(q + (size_t)M * ldq);
  if (int rc = quantize_rows(x, dtype, ldx, q, ldq, row_scale, M, K, st)) return rc;
  a.q = q;
  a.ldq = ldq;
  a.row_scale = row_scale;
  return gemm(a, dtype, st);
}
