// The norms on both sides of a block, its gate and the residual scale as one pass over the rows, and their gradients.
//
//   forward    p = N_post(f), y = a x + g * p, h = N_pre(y)       per row of D elements, statistics in fp32
//   backward   dh -> dyt = dy + N_pre'(dh), dx = a dyt, dg = sum dyt p, df = N_post'(dyt g), and the vectors' gradients
//
// Both are bound by memory: 2 + 2 row arrays of traffic forward, 4 + 2 backward, against some 20 and 50 operations an
// element.  A row lives in the registers of TPR threads (8 NV elements each) between its one load and its one store; the
// vectors (gamma, beta, gate) stay in registers over the rows a workgroup walks, as they would otherwise be read from
// the L2 once per row, as often as the rows themselves.  h is computed from y before y is rounded.
#include <algorithm>
#include "typed.hpp"
#include "host_util.hpp"

namespace souffle {
namespace gated_norm {

struct FwdArgs {
  const void *x, *f, *post_gamma, *post_beta, *gate, *pre_gamma, *pre_beta;
  void *y, *h;                      // y nullable
  int8_t *q;                        // instead of h: the row in 8-bit integers
  float *q_scale;
  long long ldx, ldf, ldy, ldh, ldq;
  int rows, cols, post, pre, rows_per_gate, rows_per_slot;
  float a, post_eps, pre_eps;
};

// Sum over the TPR threads of a row.  `red` has two halves that are used in turn, so one barrier per sum is enough: a
// wave that writes half i again has passed the barrier of the sum in between, behind which nobody reads half i any more.
template <int TPR>
struct RowReduce {
  static constexpr int kWaves = TPR < 64 ? 1 : TPR / 64;
  unsigned *red;                    // [2][2 kWaves] of this row slot
  int turn;
  __device__ __forceinline__ float sum(float v) {
    if constexpr (TPR == 16) return row16_sum_dpp(v);
    v = wave_sum_dpp(v);
    if constexpr (kWaves == 1) return v;
    float *r = reinterpret_cast<float *>(red) + turn * 2 * kWaves;
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) r[(threadIdx.x / 64) % kWaves] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) s += r[w];
    return s;
  }
  // Two sums for one barrier.
  __device__ __forceinline__ void sum2(float &v0, float &v1) {
    if constexpr (TPR == 16) v0 = row16_sum_dpp(v0), v1 = row16_sum_dpp(v1);
    else wave_sum2_dpp(v0, v1);
    if constexpr (kWaves > 1) {
      float *r = reinterpret_cast<float *>(red) + turn * 2 * kWaves;
      turn ^= 1;
      if ((threadIdx.x & 63) == 0) {
        r[(threadIdx.x / 64) % kWaves] = v0;
        r[kWaves + (threadIdx.x / 64) % kWaves] = v1;
      }
      __syncthreads();
      v0 = v1 = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) v0 += r[w], v1 += r[kWaves + w];
    }
  }
  __device__ __forceinline__ unsigned umax(unsigned v) {
    if constexpr (TPR == 16) return row16_umax_dpp(v);
    v = wave_umax_dpp(v);
    if constexpr (kWaves == 1) return v;
    unsigned *r = red + turn * 2 * kWaves;
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) r[(threadIdx.x / 64) % kWaves] = v;
    __syncthreads();
    unsigned s = 0u;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) s = max(s, r[w]);
    return s;
  }
};

// A vector's elements c .. c+7, or `missing` where the caller has none; zeros behind the row's end, which keep what is computed
// there zero.  In two steps, so that the loads of all vectors are under way before the first is waited for: a missing
// vector's are made from `any`, a row of n, as a branch around them would wait at its end.
template <RowForm FORM, class T>
__device__ __forceinline__ typename Vec8<T>::type param_load(const void *p, const void *any, int c, int n) {
  return load_row<FORM>(static_cast<const T *>(p ? p : any), c, n);
}
template <RowForm FORM, class T>
__device__ __forceinline__ typename Vec8<T>::type param_settle(typename Vec8<T>::type v, const void *p, int c, int n, float missing) {
  v = settle_row<FORM, T>(v, c, n);
  if (!p) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (T)(c + e < n ? missing : 0.f);
  }
  return v;
}

// (v - mean) / deviation or v / rms of a row in place, elements behind the row's end 0; returns 1 / deviation.  Two
// passes over the registers: the mean first, then the squares around it, so that a large mean costs no digits.
template <RowForm FORM, int TPR, int NV>
__device__ __forceinline__ float normalize(float (&v)[NV][8], int kind, float eps, int cols, int c0, RowReduce<TPR> &red) {
  const float inv_n = 1.0f / (float)cols;
  if (kind == SOUFFLE_NORM_LAYER) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) s += v[i][e];
    const float mean = red.sum(s) * inv_n;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const float m = c0 + i * TPR * 8 < cols ? mean : 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] -= m;
      if constexpr (FORM != kWhole) {
        int left = cols - c0 - i * TPR * 8;
        asm volatile("" : "+v"(left));      // (eight comparisons per row, not eight masks that are kept)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = e < left ? v[i][e] : 0.f;
      }
    }
  }
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) s = __builtin_fmaf(v[i][e], v[i][e], s);
  const float r = 1.0f / sqrtf(red.sum(s) * inv_n + eps);
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) v[i][e] *= r;
  return r;
}

// Where a slot has several rows, the next one is asked for while the present one is reduced.  16384 x 4096 bf16
// takes 108 us (median; 105 at best), 537 MB at 5.0 TB/s (a large copy: 5.05).  4096 x 768 fp16 takes 8.4 to 9.0 us, of which some 3 are the start and
// the end: one row per slot there, so nothing overlaps.  With fp32 rows of more than 8192 elements (two vectors a thread, 1024 threads, 128 registers) 114 to 160
// registers a lane do not fit: 1024 x 16384 takes 166 us, three times its bytes.
template <class T, int TPR, int NV, int WG, bool OUT8, RowForm FORM>
__global__ void __launch_bounds__(WG) k_gated_norm(const FwdArgs a) {
  typedef typename Vec8<T>::type V;
  constexpr int kSlots = WG / TPR;
  __shared__ __attribute__((aligned(16))) unsigned lds_red[WG / 64 * 4];
  const int slot = TPR < 64 ? threadIdx.x / TPR : __builtin_amdgcn_readfirstlane(threadIdx.x / TPR), t = threadIdx.x % TPR, c0 = t * 8, n = a.cols;
  RowReduce<TPR> red{lds_red + (TPR < 64 ? 0 : slot) * 4 * RowReduce<TPR>::kWaves, 0};

  const int first = (blockIdx.x * kSlots + slot) * a.rows_per_slot, end = min(first + a.rows_per_slot, a.rows);
  if (TPR <= 64 && first >= end) return;      // (rows of several waves: every workgroup has one)
  V xv[NV], fv[NV];
  auto fetch = [&](int row) {
    const T *x = static_cast<const T *>(a.x) + row * a.ldx, *f = static_cast<const T *>(a.f) + row * a.ldf;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      xv[i] = load_row<FORM>(x, c0 + i * TPR * 8, n);
      fv[i] = load_row<FORM>(f, c0 + i * TPR * 8, n);
    }
  };
  fetch(first);
  int gate_row = first / a.rows_per_gate;
  auto gate_at = [&](int row) { return a.gate ? static_cast<const T *>(a.gate) + (long long)row * n : nullptr; };
  V pg[NV], pb[NV], gt[NV], ng[NV], nb[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = c0 + i * TPR * 8;
    pg[i] = param_load<FORM, T>(a.post_gamma, a.x, c, n);
    pb[i] = param_load<FORM, T>(a.post_beta, a.x, c, n);
    gt[i] = param_load<FORM, T>(gate_at(gate_row), a.x, c, n);
    ng[i] = param_load<FORM, T>(a.pre_gamma, a.x, c, n);
    nb[i] = param_load<FORM, T>(a.pre_beta, a.x, c, n);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = c0 + i * TPR * 8;
    pg[i] = param_settle<FORM, T>(pg[i], a.post_gamma, c, n, 1.f);
    pb[i] = param_settle<FORM, T>(pb[i], a.post_beta, c, n, 0.f);
    gt[i] = param_settle<FORM, T>(gt[i], a.gate, c, n, 1.f);
    ng[i] = param_settle<FORM, T>(ng[i], a.pre_gamma, c, n, 1.f);
    nb[i] = param_settle<FORM, T>(nb[i], a.pre_beta, c, n, 0.f);
  }
  // (rows of several waves: one row per workgroup at a time, so every thread takes the same turns through the barriers)
  for (int row = first; row < end; ++row) {
    if (a.gate) {
      const int gr = row / a.rows_per_gate;
      if (gr != gate_row) {
        gate_row = gr;
#pragma unroll
        for (int i = 0; i < NV; ++i) gt[i] = param_load<FORM, T>(gate_at(gr), nullptr, c0 + i * TPR * 8, n);
#pragma unroll
        for (int i = 0; i < NV; ++i) gt[i] = settle_row<FORM, T>(gt[i], c0 + i * TPR * 8, n);
      }
    }
    float x[NV][8], p[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if constexpr (NV > 1) pg[i] = opaque(pg[i]), pb[i] = opaque(pb[i]), gt[i] = opaque(gt[i]), ng[i] = opaque(ng[i]), nb[i] = opaque(nb[i]);
      to_f32(x[i], settle_row<FORM, T>(xv[i], c0 + i * TPR * 8, n));
      to_f32(p[i], settle_row<FORM, T>(fv[i], c0 + i * TPR * 8, n));
    }
    if (row + 1 < end) fetch(row + 1);
    if (a.post != SOUFFLE_NORM_NONE) (void)normalize<FORM, TPR, NV>(p, a.post, a.post_eps, n, c0, red);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = __builtin_fmaf(p[i][e], (float)pg[i][e], (float)pb[i][e]);
        x[i][e] = __builtin_fmaf((float)gt[i][e], v, a.a * x[i][e]);
      }
    if (a.y) {
      T *y = static_cast<T *>(a.y) + row * a.ldy;
#pragma unroll
      for (int i = 0; i < NV; ++i) store_row<FORM>(y, c0 + i * TPR * 8, n, from_f32<T>(x[i]));
    }
    (void)normalize<FORM, TPR, NV>(x, a.pre, a.pre_eps, n, c0, red);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) x[i][e] = __builtin_fmaf(x[i][e], (float)ng[i][e], (float)nb[i][e]);
    if constexpr (!OUT8) {
      T *h = static_cast<T *>(a.h) + row * a.ldh;
#pragma unroll
      for (int i = 0; i < NV; ++i) store_row<FORM>(h, c0 + i * TPR * 8, n, from_f32<T>(x[i]));
    } else {
      unsigned m = 0u;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c0 + i * TPR * 8 + e < n) m = max(m, abs_bits(x[i][e]));
      const RowScale rs = row_scale(red.umax(m));
      int8_t *q = a.q + row * a.ldq;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = c0 + i * TPR * 8;      // (a q row has room up to a multiple of 64)
        if (c < n) *reinterpret_cast<u2 *>(q + c) = quantize8(x[i], rs);
      }
      if (t == 0) a.q_scale[row] = rs.scale;
    }
  }
}

// ------------------------------------------------------------------------------------------ backward ----
enum { kPreGamma = 0, kPreBeta, kGate, kPostGamma, kPostBeta, kVectors };

struct BwdArgs {
  const void *x, *f, *dy, *dh, *post_gamma, *post_beta, *gate, *pre_gamma;
  void *dx, *df;                    // nullable
  void *dgate;                      // written here where a group of rows is one workgroup's own
  float *partial;                   // [chunks][wanted vectors][cols]
  long long ldx, ldf, ld_dy, ld_dh, ld_dx, ld_df;
  int rows, cols, post, pre;
  int rows_per_gate;                // rows that share a gate row (all rows: one gate row, or no gate)
  int chunk_rows;                   // rows of a workgroup; a multiple of rows_per_gate, or within one gate row's rows
  int chunks_per_gate;              // > 0: that many chunks per gate row; 0: chunks hold whole gate rows
  int vectors, wanted;              // wanted: bit v set = the gradient of vector v goes to `partial`
  int wanted_gate;                  // the gate's gradient goes there or to dgate
  int row_gates;                    // chunks hold whole gate rows of few rows each
  float a, post_eps, pre_eps;
};

// Several rows at a time (one per slot of TPR threads), slots in step, so that a barrier of the workgroup serves them all.
// Rows that share a gate row are taken in one go by all slots, or, where there are few of them (ROW_GATES), by one
// slot each, which loads the gate with its row and writes the gate's gradient itself.
// 8192 x 4096 bf16 takes 85 us (median, alone), 403 MB at 4.7 TB/s.  With few rows per workgroup the arithmetic and the barriers of a
// turn count instead, some 4 us for eight waves: 1182 x 1001 fp32, two turns, 16.8 us.
// Two vectors a thread hold five sums of 16 elements beside four rows and four vectors of parameters.  Registers a lane that do not fit: rows of
// 4097 to 8192 elements 158 in fp32 (2048 x 8192: 128 us, bytes 80), 4 to 26 in 16 bits (55 us, bytes 40); beyond 8192 349 to 525
// (1024 x 16384: 561 us in fp32, 335 in fp16, bytes 80 and 40); with ROW_GATES 0 to 7 and 295 to 386.
template <class T, int TPR, int NV, int WG, RowForm FORM, bool KEEP, bool ROW_GATES>
__global__ void __launch_bounds__(WG) k_gated_norm_grad(const BwdArgs a) {
  typedef typename Vec8<T>::type V;
  constexpr int kSlots = WG / TPR;
  __shared__ __attribute__((aligned(16))) unsigned lds_red[WG / 64 * 4];
  constexpr int kSlotCols = TPR * NV * 8;
  __shared__ __attribute__((aligned(16))) float lds_sum[kSlots > 1 ? kVectors * kSlots * kSlotCols : 1];
  const int slot = TPR < 64 ? threadIdx.x / TPR : __builtin_amdgcn_readfirstlane(threadIdx.x / TPR), t = threadIdx.x % TPR, c0 = t * 8, n = a.cols;
  const float inv_n = 1.0f / (float)n;
  RowReduce<TPR> red{lds_red + (TPR < 64 ? 0 : slot) * 4 * RowReduce<TPR>::kWaves, 0};

  float sums[kVectors][NV][8] = {};
  // The sums of the vectors in `mask`, over the slots in their order: whole(v, c, eight of them) or one(v, c, sum).
  auto collect = [&](int mask, auto whole, auto one) {
    if constexpr (kSlots == 1) {
#pragma unroll
      for (int v = 0; v < kVectors; ++v)
        if (mask >> v & 1)
#pragma unroll
          for (int i = 0; i < NV; ++i) whole(v, c0 + i * TPR * 8, sums[v][i]);
    } else {
#pragma unroll
      for (int v = 0; v < kVectors; ++v)
        if (mask >> v & 1)
#pragma unroll
          for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) lds_sum[(v * kSlots + slot) * kSlotCols + c0 + i * TPR * 8 + e] = sums[v][i][e];
      __syncthreads();
#pragma unroll 1
      for (int v = 0; v < kVectors; ++v)
        if (mask >> v & 1)
          for (int c = threadIdx.x; c < n; c += WG) {
            float s = 0.f;
#pragma unroll
            for (int k = 0; k < kSlots; ++k) s += lds_sum[(v * kSlots + k) * kSlotCols + c];
            one(v, c, s);
          }
      __syncthreads();
    }
  };

  // a gradient that is not there: x instead, taken as zeros
  const T *dy = static_cast<const T *>(a.dy ? a.dy : a.x), *dh = static_cast<const T *>(a.dh ? a.dh : a.x);
  const long long ld_dy = a.dy ? a.ld_dy : a.ldx, ld_dh = a.dh ? a.ld_dh : a.ldx;
  int first, end;
  if (a.chunks_per_gate > 0) {
    const int g = blockIdx.x / a.chunks_per_gate, k = blockIdx.x % a.chunks_per_gate, g_end = min((g + 1) * a.rows_per_gate, a.rows);
    first = min(g * a.rows_per_gate + k * a.chunk_rows, g_end);
    end = min(first + a.chunk_rows, g_end);
  } else {
    first = min((long long)blockIdx.x * a.chunk_rows, (long long)a.rows);
    end = min(first + a.chunk_rows, a.rows);
  }
  // rows first .. end in runs that share a gate row
  for (int run = first; run < end;) {
    const int gr = run / a.rows_per_gate, run_end = ROW_GATES ? end : min((gr + 1) * a.rows_per_gate, end);
    V gt[NV], pg[NV], pb[NV], ng[NV];
    const void *gate = a.gate ? static_cast<const T *>(a.gate) + (long long)gr * n : nullptr;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = c0 + i * TPR * 8;
      if constexpr (!ROW_GATES) gt[i] = param_load<FORM, T>(gate, a.x, c, n);
      pg[i] = param_load<FORM, T>(a.post_gamma, a.x, c, n);
      pb[i] = param_load<FORM, T>(a.post_beta, a.x, c, n);
      ng[i] = param_load<FORM, T>(a.pre_gamma, a.x, c, n);
    }
    V xv[NV], fv[NV], yv[NV], hv[NV], gv[NV];
    auto fetch = [&](int row) {      // (a slot without a row takes the run's first one, with gradients of zero)
      const bool valid = row < run_end;
      const long long r = valid ? row : run;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = c0 + i * TPR * 8;
        xv[i] = load_row<FORM>(static_cast<const T *>(a.x) + r * a.ldx, c, n);
        fv[i] = load_row<FORM>(static_cast<const T *>(a.f) + r * a.ldf, c, n);
        yv[i] = load_row<FORM>(dy + r * ld_dy, c, n);
        hv[i] = load_row<FORM>(dh + r * ld_dh, c, n);
        if constexpr (ROW_GATES) gv[i] = load_row<FORM>(static_cast<const T *>(a.gate) + r / a.rows_per_gate * n, c, n);
      }
    };
    const int few = a.rows_per_gate, turns = ROW_GATES ? ((run_end - run) / few + kSlots - 1) / kSlots * few : (run_end - run + kSlots - 1) / kSlots;
    auto row_of = [&](int turn) { return run + (ROW_GATES ? (turn / few * kSlots + slot) * few + turn % few : turn * kSlots + slot); };
    if constexpr (KEEP) fetch(row_of(0));
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = c0 + i * TPR * 8;
      if constexpr (!ROW_GATES) gt[i] = param_settle<FORM, T>(gt[i], gate, c, n, 1.f);
      pg[i] = param_settle<FORM, T>(pg[i], a.post_gamma, c, n, 1.f);
      pb[i] = param_settle<FORM, T>(pb[i], a.post_beta, c, n, 0.f);
      ng[i] = param_settle<FORM, T>(ng[i], a.pre_gamma, c, n, 1.f);
    }
    for (int turn = 0; turn < turns; ++turn) {
      const int row = row_of(turn);
      const bool valid = row < run_end;
      float y[NV][8], fh[NV][8], d[NV][8], h[NV][8];
      if constexpr (!KEEP) {
        fetch(row);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          pg[i] = opaque(pg[i]), pb[i] = opaque(pb[i]);
          if constexpr (!ROW_GATES) gt[i] = opaque(gt[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = c0 + i * TPR * 8;
        if constexpr (ROW_GATES) gt[i] = settle_row<FORM, T>(gv[i], c, n);
        to_f32(y[i], settle_row<FORM, T>(xv[i], c, n));
        to_f32(fh[i], settle_row<FORM, T>(fv[i], c, n));
        to_f32(d[i], settle_row<FORM, T>(yv[i], valid && a.dy ? c : n, n));
        to_f32(h[i], settle_row<FORM, T>(hv[i], valid && a.dh ? c : n, n));
      }
      if constexpr (KEEP)
        if (turn + 1 < turns) fetch(row_of(turn + 1));
      float fr = 1.f;
      if (a.post != SOUFFLE_NORM_NONE) fr = normalize<FORM, TPR, NV>(fh, a.post, a.post_eps, n, c0, red);
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          y[i][e] = __builtin_fmaf((float)gt[i][e], __builtin_fmaf(fh[i][e], (float)pg[i][e], (float)pb[i][e]), a.a * y[i][e]);
      const float yr = normalize<FORM, TPR, NV>(y, a.pre, a.pre_eps, n, c0, red);
      float s0 = 0.f, s1 = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if constexpr (!KEEP) ng[i] = opaque(ng[i]);
        if (a.wanted >> kPreBeta & 1)
#pragma unroll
          for (int e = 0; e < 8; ++e) sums[kPreBeta][i][e] += h[i][e];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          sums[kPreGamma][i][e] = __builtin_fmaf(h[i][e], y[i][e], sums[kPreGamma][i][e]);
          h[i][e] *= (float)ng[i][e];
          s1 = __builtin_fmaf(h[i][e], y[i][e], s1);
        }
        if (a.pre == SOUFFLE_NORM_LAYER)
#pragma unroll
          for (int e = 0; e < 8; ++e) s0 += h[i][e];
      }
      red.sum2(s0, s1);
      s0 *= yr * inv_n, s1 *= yr * inv_n;
      float s2 = 0.f, s3 = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if constexpr (!KEEP) pg[i] = opaque(pg[i]), pb[i] = opaque(pb[i]), gt[i] = opaque(gt[i]);
        if (a.pre == SOUFFLE_NORM_LAYER)
#pragma unroll
          for (int e = 0; e < 8; ++e) d[i][e] -= s0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {      // gradient of y
          d[i][e] = __builtin_fmaf(-s1, y[i][e], __builtin_fmaf(yr, h[i][e], d[i][e]));
          y[i][e] = a.a * d[i][e];
        }
        if (a.wanted_gate)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            sums[kGate][i][e] = __builtin_fmaf(d[i][e], __builtin_fmaf(fh[i][e], (float)pg[i][e], (float)pb[i][e]), sums[kGate][i][e]);
#pragma unroll
        for (int e = 0; e < 8; ++e) d[i][e] *= (float)gt[i][e];      // gradient of N_post(f); the vectors are 0 behind the row's end
        if (a.wanted >> kPostBeta & 1)
#pragma unroll
          for (int e = 0; e < 8; ++e) sums[kPostBeta][i][e] += d[i][e];
        if (a.post != SOUFFLE_NORM_NONE)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            sums[kPostGamma][i][e] = __builtin_fmaf(d[i][e], fh[i][e], sums[kPostGamma][i][e]);
            d[i][e] *= (float)pg[i][e];
            s3 = __builtin_fmaf(d[i][e], fh[i][e], s3);
          }
        if (a.post == SOUFFLE_NORM_LAYER)
#pragma unroll
          for (int e = 0; e < 8; ++e) s2 += d[i][e];
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) store_row<FORM>(static_cast<T *>(a.dx) + row * a.ld_dx, c0 + i * TPR * 8, a.dx && valid ? n : 0, from_f32<T>(y[i]));
      if (a.post != SOUFFLE_NORM_NONE) {
        red.sum2(s2, s3);
        s2 *= fr * inv_n, s3 *= fr * inv_n;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
          for (int e = 0; e < 8; ++e) d[i][e] = __builtin_fmaf(-s3, fh[i][e], fr * d[i][e]);
          if (a.post == SOUFFLE_NORM_LAYER)
#pragma unroll
            for (int e = 0; e < 8; ++e) d[i][e] -= s2;
        }
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) store_row<FORM>(static_cast<T *>(a.df) + row * a.ld_df, c0 + i * TPR * 8, a.df && valid ? n : 0, from_f32<T>(d[i]));
      if constexpr (ROW_GATES)
        if (a.dgate && turn % few == few - 1) {      // the slot's rows of this gate row are done
          T *dg = static_cast<T *>(a.dgate) + (long long)(row / few) * n;
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            store_row<FORM>(dg, c0 + i * TPR * 8, valid ? n : 0, from_f32<T>(sums[kGate][i]));
#pragma unroll
            for (int e = 0; e < 8; ++e) sums[kGate][i][e] = 0.f;
          }
        }
    }
    if (!ROW_GATES && a.dgate && a.chunks_per_gate == 0) {      // the gate row's rows were all this workgroup's
      T *dg = static_cast<T *>(a.dgate) + (long long)gr * n;
      collect(1 << kGate, [&](int, int c, const float (&s)[8]) { store_row<FORM>(dg, c, n, from_f32<T>(s)); }, [&](int, int c, float s) { dg[c] = (T)s; });
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) sums[kGate][i][e] = 0.f;
    }
    run = run_end;
  }
  float *out = a.partial + (long long)blockIdx.x * a.vectors * n;
  auto at = [&](int v) { return out + (long long)__popc(a.wanted & ((1 << v) - 1)) * n; };
  collect(a.wanted, [&](int v, int c, const float (&s)[8]) { store_row<FORM>(at(v), c, n, from_f32<float>(s)); }, [&](int v, int c, float s) { at(v)[c] = s; });
}

struct FinishArgs {
  const float *partial;
  void *out[kVectors];
  int cols, vectors, wanted, chunks;
  int chunks_per_gate;              // of each of the gate's rows
  int others;                       // vectors except the gate
  int vector_blocks;                // their workgroups
  int gate_width;                   // columns of a workgroup of the gate's rows: 32, 128 or 1024
};
// Column sums over the chunks, W columns x 1024 / W slices of the chunks per workgroup, slices added in order.  W is about the
// largest that leaves a thread up to eight loads, all under way at once: 32 for the vectors' 256 chunks, more for a row of the
// gate, which may have two chunks only (a workgroup per 32 columns of 128 gate rows x 4096 takes 27 us longer).
template <class T, int W>
__device__ __forceinline__ void finish_columns(const FinishArgs &a, float *lds, int v, int first, int count, int c0, long long row) {
  constexpr int kSlices = 1024 / W;
  const int lane = threadIdx.x % W, slice = threadIdx.x / W, c = c0 + lane;
  float s = 0.f;
  if (c < a.cols) {
    const float *p = a.partial + ((long long)first * a.vectors + __popc(a.wanted & ((1 << v) - 1))) * a.cols + c;
#pragma unroll 8
    for (int k = slice; k < count; k += kSlices) s += p[(long long)k * a.vectors * a.cols];
  }
  if constexpr (kSlices > 1) {
    lds[slice * (W + 1) + lane] = s;
    __syncthreads();
    s = 0.f;
    if (slice == 0)
#pragma unroll
      for (int k = 0; k < kSlices; ++k) s += lds[k * (W + 1) + lane];
  }
  if (slice == 0 && c < a.cols) static_cast<T *>(a.out[v])[row * a.cols + c] = (T)s;
}
template <class T>
__global__ void __launch_bounds__(1024) k_gated_norm_grad_finish(const FinishArgs a) {
  __shared__ float lds[1024 + 32];
  int b = blockIdx.x;
  if (b < a.vector_blocks) {      // the vectors take turns
    int left = a.wanted & ~(1 << kGate);
    for (int i = b % a.others; i > 0; --i) left &= left - 1;
    finish_columns<T, 32>(a, lds, __ffs(left) - 1, 0, a.chunks, b / a.others * 32, 0);
    return;
  }
  b -= a.vector_blocks;
  const int blocks = (a.cols + a.gate_width - 1) / a.gate_width, row = b / blocks, c0 = b % blocks * a.gate_width, first = row * a.chunks_per_gate;
  if (a.gate_width == 32) finish_columns<T, 32>(a, lds, kGate, first, a.chunks_per_gate, c0, row);
  else if (a.gate_width == 128) finish_columns<T, 128>(a, lds, kGate, first, a.chunks_per_gate, c0, row);
  else finish_columns<T, 1024>(a, lds, kGate, first, a.chunks_per_gate, c0, row);
}

// ------------------------------------------------------------------------------------------ host side ----
constexpr int kMaxCols = 16384;

static int check_cfg(const souffle_gated_norm_cfg *c) {
  if (!c) return fail(SOUFFLE_ERR_NULL, "cfg is NULL");
  if (c->rows < 0 || c->rows > (1 << 30)) return fail(SOUFFLE_ERR_SHAPE, "rows must be in 0..2^30 (got %d)", c->rows);
  if (c->cols < 1 || c->cols > kMaxCols) return fail(SOUFFLE_ERR_SHAPE, "cols must be in 1..%d (got %d)", kMaxCols, c->cols);
  if (c->dtype != SOUFFLE_F16 && c->dtype != SOUFFLE_BF16 && c->dtype != SOUFFLE_F32) return fail(SOUFFLE_ERR_SHAPE, "unknown dtype %d", c->dtype);
  if (c->post_norm < SOUFFLE_NORM_NONE || c->post_norm > SOUFFLE_NORM_RMS) return fail(SOUFFLE_ERR_SHAPE, "unknown post_norm %d", c->post_norm);
  if (c->pre_norm != SOUFFLE_NORM_LAYER && c->pre_norm != SOUFFLE_NORM_RMS) return fail(SOUFFLE_ERR_SHAPE, "pre_norm must be LAYER or RMS (got %d)", c->pre_norm);
  if (c->rows_per_gate < 0 || (c->rows_per_gate > 0 && c->rows % c->rows_per_gate))
    return fail(SOUFFLE_ERR_SHAPE, "rows_per_gate must divide the %d rows (got %d)", c->rows, c->rows_per_gate);
  if (!(c->post_eps >= 0.f) || !(c->pre_eps >= 0.f)) return fail(SOUFFLE_ERR_SHAPE, "the norms' eps must not be negative");
  return SOUFFLE_OK;
}
static int check_row(const char *name, const void *p, long long ld, const souffle_gated_norm_cfg *c) {
  const unsigned size = c->dtype == SOUFFLE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(p) % size) return fail(SOUFFLE_ERR_ALIGN, "%s is not aligned to its elements", name);
  if (ld < c->cols) return fail(SOUFFLE_ERR_SHAPE, "the rows of %s overlap: stride %lld, %d columns", name, ld, c->cols);
  return SOUFFLE_OK;
}
static int check_vectors(const souffle_gated_norm_cfg *c, const souffle_gated_norm_w *w) {
  if (!w) return fail(SOUFFLE_ERR_NULL, "the vectors' struct is NULL");
  if (c->post_norm == SOUFFLE_NORM_NONE && (w->post_gamma || w->post_beta)) return fail(SOUFFLE_ERR_SHAPE, "post_gamma and post_beta need a post_norm");
  const void *p[5] = {w->post_gamma, w->post_beta, w->gate, w->pre_gamma, w->pre_beta};
  for (int i = 0; i < 5; ++i)
    if (reinterpret_cast<uintptr_t>(p[i]) % (c->dtype == SOUFFLE_F32 ? 4 : 2)) return fail(SOUFFLE_ERR_ALIGN, "a vector is not aligned to its elements");
  return SOUFFLE_OK;
}

template <RowForm FORM, class T, int TPR, int NV, int WG>
static int launch_fwd(FwdArgs a, int num_cus, hipStream_t st) {
  constexpr int kSlots = WG / TPR;
  // Row slots, counted as if 2048 threads of a CU were resident.  The kernels' registers let 512 to 1536 stand (2 to 6 waves a SIMD), so just below
  // this many rows the slots of one row each run in two to four rounds.
  const long long slots = (long long)num_cus * (2048 / WG) * kSlots;
  a.rows_per_slot = (int)std::max<long long>(1, (a.rows + slots - 1) / slots);
  const int grid = (int)(((long long)a.rows + (long long)a.rows_per_slot * kSlots - 1) / ((long long)a.rows_per_slot * kSlots));
  if (a.q) hipLaunchKernelGGL((k_gated_norm<T, TPR, NV, WG, true, FORM>), dim3(grid), dim3(WG), 0, st, a);
  else hipLaunchKernelGGL((k_gated_norm<T, TPR, NV, WG, false, FORM>), dim3(grid), dim3(WG), 0, st, a);
  SOUFFLE_HIP_TRY(hipGetLastError());
  return SOUFFLE_OK;
}
template <RowForm FORM, class T>
static int forward(const FwdArgs &a, int num_cus, hipStream_t st) {
  // One vector of 8 per thread in fp32, two in the 16-bit types from 513 elements on except 1025 to 2048 (measured: 4096 x 4096 fp32 48.6 us with one
  // and 55.5 with two, which leave two waves per SIMD; 8192 x 4096 bf16 49.3 and 45.3, where two halve the waves of a sum; fp32 4096 x 768 12.0 with
  // 128 threads and 13.5 with 64, 4096 x 2048 23.6 with 256 and 26.2 with 128; fp16 4096 x 2048 15.8 with 256 and 15.2 with 128).  Rows of up to
  // 256 elements share a wave, 16 threads each: 262144 x 64 fp16 32 us (106 with 64 threads), 131072 x 256 fp16 45 (60), fp32 117 (114).
  if constexpr (sizeof(T) == 4) {
    if (a.cols <= 128) return launch_fwd<FORM, T, 16, 1, 256>(a, num_cus, st);
    if (a.cols <= 256) return launch_fwd<FORM, T, 16, 2, 256>(a, num_cus, st);
    if (a.cols <= 512) return launch_fwd<FORM, T, 64, 1, 256>(a, num_cus, st);
    if (a.cols <= 1024) return launch_fwd<FORM, T, 128, 1, 128>(a, num_cus, st);
    if (a.cols <= 2048) return launch_fwd<FORM, T, 256, 1, 256>(a, num_cus, st);
    if (a.cols <= 4096) return launch_fwd<FORM, T, 512, 1, 512>(a, num_cus, st);
    if (a.cols <= 8192) return launch_fwd<FORM, T, 1024, 1, 1024>(a, num_cus, st);
    return launch_fwd<FORM, T, 1024, 2, 1024>(a, num_cus, st);
  } else {
    if (a.cols <= 128) return launch_fwd<FORM, T, 16, 1, 256>(a, num_cus, st);
    if (a.cols <= 256) return launch_fwd<FORM, T, 16, 2, 256>(a, num_cus, st);
    if (a.cols <= 512) return launch_fwd<FORM, T, 64, 1, 256>(a, num_cus, st);
    if (a.cols <= 1024) return launch_fwd<FORM, T, 64, 2, 256>(a, num_cus, st);
    if (a.cols <= 2048) return launch_fwd<FORM, T, 256, 1, 256>(a, num_cus, st);
    if (a.cols <= 4096) return launch_fwd<FORM, T, 256, 2, 256>(a, num_cus, st);
    if (a.cols <= 8192) return launch_fwd<FORM, T, 512, 2, 512>(a, num_cus, st);
    return launch_fwd<FORM, T, 1024, 2, 1024>(a, num_cus, st);
  }
}
template <class T>
static int forward(const FwdArgs &a, int num_cus, hipStream_t st) {
  if (a.cols < 8) return launch_fwd<kShort, T, 16, 1, 256>(a, num_cus, st);
  return a.cols % 8 ? forward<kRagged, T>(a, num_cus, st) : forward<kWhole, T>(a, num_cus, st);
}

// How the rows are cut into chunks, one workgroup each: at most `want` of them, none across gate rows unless it holds
// whole gate rows.  (With a gradient of the gate, 129 to 255 gate rows are that many chunks and 257 are 129: 130 | 256 | 257 gate rows of 200 x 768
// fp16 take 137 | 146 | 269 us.)
struct Chunks {
  int count, rows, per_gate;
};
static Chunks plan_chunks(int rows, int rows_per_gate, int gate_grad, int want) {
  Chunks c;
  if (!gate_grad) {
    c.rows = std::max(1, (rows + want - 1) / want);
    c.per_gate = 0;
    c.count = (rows + c.rows - 1) / c.rows;
    return c;
  }
  const int gates = rows / rows_per_gate;
  if (gates >= want) {
    const int per_chunk = (gates + want - 1) / want;
    c.rows = per_chunk * rows_per_gate;
    c.per_gate = 0;
    c.count = (gates + per_chunk - 1) / per_chunk;
  } else {
    c.per_gate = std::max(1, std::min(rows_per_gate, want / gates));
    c.rows = (rows_per_gate + c.per_gate - 1) / c.per_gate;
    c.per_gate = (rows_per_gate + c.rows - 1) / c.rows;
    c.count = c.per_gate * gates;
  }
  return c;
}
constexpr int kChunks = 256;      // one per CU
// Gate rows of fewer rows than this are taken by one slot each.  Measured, us for 1 | 2 | 4 rows a gate row: 4096 x 512 fp16 15.9 | 14.9 | 18.2, by
// all slots 53.2 | 30.7 | 20.1 (14.1 with 16 rows); 8192 x 4096 bf16 124 | 115 | 113 and 163 | 136 | 121 (105).
constexpr int kFewRows = 8;

static int wanted_vectors(const souffle_gated_norm_grad *g) {
  return (g->pre_gamma ? 1 << kPreGamma : 0) | (g->pre_beta ? 1 << kPreBeta : 0) | (g->gate ? 1 << kGate : 0) |
         (g->post_gamma ? 1 << kPostGamma : 0) | (g->post_beta ? 1 << kPostBeta : 0);
}

template <RowForm FORM, class T, int TPR, int NV, int WG, bool KEEP = true>
static int launch_bwd(const BwdArgs &a, int chunks, hipStream_t st) {
  if (a.row_gates) hipLaunchKernelGGL((k_gated_norm_grad<T, TPR, NV, WG, FORM, KEEP, true>), dim3(chunks), dim3(WG), 0, st, a);
  else hipLaunchKernelGGL((k_gated_norm_grad<T, TPR, NV, WG, FORM, KEEP, false>), dim3(chunks), dim3(WG), 0, st, a);
  SOUFFLE_HIP_TRY(hipGetLastError());
  return SOUFFLE_OK;
}
// (16 threads a row as in the forward pass: 262144 x 64 fp16 65 us, 235 with 64 threads; 131072 x 256 fp16 94 and 131, fp32 171 and 172)
template <RowForm FORM, class T>
static int rows_backward(const BwdArgs &a, int chunks, hipStream_t st) {
  if (a.cols <= 128) return launch_bwd<FORM, T, 16, 1, 512>(a, chunks, st);
  if (a.cols <= 256) return launch_bwd<FORM, T, 16, 2, 256>(a, chunks, st);
  if (a.cols <= 512) return launch_bwd<FORM, T, 64, 1, 512>(a, chunks, st);
  if (a.cols <= 1024) return launch_bwd<FORM, T, 128, 1, 512>(a, chunks, st);
  if (a.cols <= 2048) return launch_bwd<FORM, T, 256, 1, 512>(a, chunks, st);
  if (a.cols <= 4096) return launch_bwd<FORM, T, 512, 1, 512>(a, chunks, st);
  if (a.cols <= 8192) return launch_bwd<FORM, T, 512, 2, 512, false>(a, chunks, st);
  return launch_bwd<FORM, T, 1024, 2, 1024, false>(a, chunks, st);
}
template <class T>
static int backward(const BwdArgs &a, const FinishArgs &f, int gate_rows, hipStream_t st) {
  const int rc = a.cols < 8 ? launch_bwd<kShort, T, 16, 1, 512>(a, f.chunks, st)
                            : a.cols % 8 ? rows_backward<kRagged, T>(a, f.chunks, st) : rows_backward<kWhole, T>(a, f.chunks, st);
  if (rc || f.vectors == 0) return rc;
  const bool gate = f.wanted >> kGate & 1;
  const int gate_blocks = gate ? gate_rows * ((f.cols + f.gate_width - 1) / f.gate_width) : 0;
  hipLaunchKernelGGL(k_gated_norm_grad_finish<T>, dim3(f.vector_blocks + gate_blocks), dim3(1024), 0, st, f);
  SOUFFLE_HIP_TRY(hipGetLastError());
  return SOUFFLE_OK;
}

static int run_forward(const souffle_gated_norm_cfg *c, const souffle_gated_norm_w *w, const void *x, const void *f, void *y, void *h,
                       int8_t *q, long long ldq, float *q_scale, souffle_stream_t stream) {
  if (int rc = check_cfg(c)) return rc;
  if (int rc = check_vectors(c, w)) return rc;
  if (c->rows == 0) return SOUFFLE_OK;
  if (!x || !f) return fail(SOUFFLE_ERR_NULL, "x and f must not be NULL");
  if (int rc = check_row("x", x, c->ldx, c)) return rc;
  if (int rc = check_row("f", f, c->ldf, c)) return rc;
  if (y)
    if (int rc = check_row("y", y, c->ldy, c)) return rc;
  if (h)
    if (int rc = check_row("h", h, c->ldh, c)) return rc;
  DeviceFacts df;
  if (int rc = device_facts(&df)) return rc;
  FwdArgs a = {x, f, w->post_gamma, w->post_beta, w->gate, w->pre_gamma, w->pre_beta, y, h, q, q_scale, c->ldx, c->ldf, c->ldy, c->ldh, ldq,
               c->rows, c->cols, c->post_norm, c->pre_norm, c->rows_per_gate ? c->rows_per_gate : c->rows, 1, c->residual_scale, c->post_eps, c->pre_eps};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (c->dtype == SOUFFLE_F16) return forward<half_t>(a, df.num_cus, st);
  if (c->dtype == SOUFFLE_BF16) return forward<bf16_t>(a, df.num_cus, st);
  return forward<float>(a, df.num_cus, st);
}

}  // namespace gated_norm
}  // namespace souffle

using namespace souffle;
using namespace souffle::gated_norm;

extern "C" int souffle_gated_norm_forward(const souffle_gated_norm_cfg *cfg, const souffle_gated_norm_w *w, const void *x, const void *f,
                                          void *y, void *h, souffle_stream_t stream) {
  if (cfg && cfg->rows > 0 && !h) return fail(SOUFFLE_ERR_NULL, "h must not be NULL");
  return run_forward(cfg, w, x, f, y, h, nullptr, 0, nullptr, stream);
}

extern "C" int souffle_gated_norm_forward_int8(const souffle_gated_norm_cfg *cfg, const souffle_gated_norm_w *w, const void *x, const void *f,
                                               void *y, int8_t *q, long long ldq, float *row_scale, souffle_stream_t stream) {
  if (cfg && cfg->rows > 0) {
    if (!q || !row_scale) return fail(SOUFFLE_ERR_NULL, "q and row_scale must not be NULL");
    if (!aligned16(q) || ldq % 16) return fail(SOUFFLE_ERR_ALIGN, "the rows of q must be 16-byte aligned");
    if (reinterpret_cast<uintptr_t>(row_scale) % 4) return fail(SOUFFLE_ERR_ALIGN, "row_scale is not aligned to its elements");
    if (ldq < (long long)round_up((size_t)std::max(cfg->cols, 0), 64)) return fail(SOUFFLE_ERR_SHAPE, "ldq must be at least cols rounded up to 64 (got %lld)", ldq);
  }
  return run_forward(cfg, w, x, f, y, nullptr, q, ldq, row_scale, stream);
}

extern "C" size_t souffle_gated_norm_backward_workspace_bytes(const souffle_gated_norm_cfg *cfg) {
  if (check_cfg(cfg)) return 0;
  // the most chunks that any set of wanted gradients makes, each with all five vectors
  const int rpg = cfg->rows_per_gate ? cfg->rows_per_gate : std::max(cfg->rows, 1);
  const int chunks = std::max(plan_chunks(cfg->rows, rpg, 0, kChunks).count, cfg->rows ? plan_chunks(cfg->rows, rpg, 1, kChunks).count : 0);
  return round_up((size_t)std::max(chunks, 1) * kVectors * cfg->cols * 4, 256);
}

extern "C" int souffle_gated_norm_backward(const souffle_gated_norm_cfg *c, const souffle_gated_norm_w *w, const void *dy, const void *dh,
                                           const void *x, const void *f, const souffle_gated_norm_grad *g, void *ws, size_t ws_bytes,
                                           souffle_stream_t stream) {
  if (int rc = check_cfg(c)) return rc;
  if (int rc = check_vectors(c, w)) return rc;
  if (!g) return fail(SOUFFLE_ERR_NULL, "the gradients' struct is NULL");
  if (c->rows == 0) return fail(SOUFFLE_ERR_SHAPE, "there are no rows to take gradients of");
  if (!x || !f || (!dy && !dh)) return fail(SOUFFLE_ERR_NULL, "x, f and one of dy and dh must not be NULL");
  if (c->post_norm == SOUFFLE_NORM_NONE && (g->post_gamma || g->post_beta)) return fail(SOUFFLE_ERR_SHAPE, "gradients of post_gamma and post_beta need a post_norm");
  if (g->gate && !w->gate) return fail(SOUFFLE_ERR_NULL, "the gate's gradient needs the gate");
  const struct { const char *name; const void *p; long long ld; } rows[6] = {{"x", x, c->ldx}, {"f", f, c->ldf}, {"dy", dy, g->ld_dy}, {"dh", dh, g->ld_dh},
                                                                            {"dx", g->dx, g->ld_dx}, {"df", g->df, g->ld_df}};
  for (const auto &r : rows)
    if (r.p)
      if (int rc = check_row(r.name, r.p, r.ld, c)) return rc;
  const void *vec[5] = {g->pre_gamma, g->pre_beta, g->gate, g->post_gamma, g->post_beta};
  for (const void *p : vec)
    if (reinterpret_cast<uintptr_t>(p) % (c->dtype == SOUFFLE_F32 ? 4 : 2)) return fail(SOUFFLE_ERR_ALIGN, "a gradient vector is not aligned to its elements");
  const int rpg = w->gate && c->rows_per_gate ? c->rows_per_gate : c->rows, wanted = wanted_vectors(g);
  if (wanted) {
    if (!ws || ws_bytes < souffle_gated_norm_backward_workspace_bytes(c))
      return fail(SOUFFLE_ERR_WORKSPACE, "workspace too small: need %zu bytes", souffle_gated_norm_backward_workspace_bytes(c));
    if (!aligned16(ws)) return fail(SOUFFLE_ERR_ALIGN, "workspace must be 16-byte aligned");
  }
  DeviceFacts df;
  if (int rc = device_facts(&df)) return rc;
  // (whole gate rows to a chunk also where their gradient is not wanted, if a gate row's rows are few)
  const bool few = w->gate && rpg < kFewRows;
  const Chunks ch = plan_chunks(c->rows, rpg, g->gate || few, kChunks);
  const bool gate_direct = g->gate && ch.per_gate == 0;
  BwdArgs a = {};
  a.x = x; a.f = f; a.dy = dy; a.dh = dh;
  a.post_gamma = w->post_gamma; a.post_beta = w->post_beta; a.gate = w->gate; a.pre_gamma = w->pre_gamma;
  a.dx = g->dx; a.df = g->df; a.dgate = gate_direct ? g->gate : nullptr;
  a.partial = static_cast<float *>(ws);
  a.ldx = c->ldx; a.ldf = c->ldf; a.ld_dy = g->ld_dy; a.ld_dh = g->ld_dh; a.ld_dx = g->ld_dx; a.ld_df = g->ld_df;
  a.rows = c->rows; a.cols = c->cols; a.post = c->post_norm; a.pre = c->pre_norm;
  a.rows_per_gate = rpg; a.chunk_rows = ch.rows; a.chunks_per_gate = ch.per_gate;
  a.wanted = gate_direct ? wanted & ~(1 << kGate) : wanted;
  a.vectors = __builtin_popcount(a.wanted);
  a.wanted_gate = g->gate != nullptr;
  a.row_gates = few && ch.per_gate == 0;
  a.a = c->residual_scale; a.post_eps = c->post_eps; a.pre_eps = c->pre_eps;
  FinishArgs fin = {static_cast<const float *>(ws), {g->pre_gamma, g->pre_beta, g->gate, g->post_gamma, g->post_beta}, c->cols, a.vectors, a.wanted, ch.count, ch.per_gate, 0, 0, 0};
  fin.others = __builtin_popcount(a.wanted & ~(1 << kGate));
  fin.vector_blocks = fin.others * ((c->cols + 31) / 32);
  fin.gate_width = ch.per_gate > 32 ? 32 : ch.per_gate > 8 ? 128 : 1024;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int gate_rows = c->rows / rpg;
  if (c->dtype == SOUFFLE_F16) return backward<half_t>(a, fin, gate_rows, st);
  if (c->dtype == SOUFFLE_BF16) return backward<bf16_t>(a, fin, gate_rows, st);
  return backward<float>(a, fin, gate_rows, st);
}
