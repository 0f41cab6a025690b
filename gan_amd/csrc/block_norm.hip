// The norms before and after a transformer block, fused with the block's gate and the residual scale:
//
//   y = rho x + gate * (fh * wo + bo)           fh = (f - mu_f) r_f      (mu = 0 for a root-mean-square norm)
//   h = (yh * wi + bi) * (1 + s) + t            yh = (y - mu_y) r_y      r = 1 / sqrt(mean((. - mu)^2) + eps)
//
// f is what the block in front computed, x the residual stream, h what the next block reads.  Parts: only h (the norm in
// front of the first block), only y (behind the last), or both (a boundary between two blocks) in one sweep over the row.
// With A = gate wo, B = gate bo, C = wi (1 + s), D = bi (1 + s) + t:   y = rho x + A fh + B,   h = C yh + D.
//
// Backward, row by row with q = C dh:
//   g  = dy + r_y (q - yh mean(q yh) - [layer] mean(q))            dx = rho g
//   p  = A g,  df = r_f (p - fh mean(p fh) - [layer] mean(p))
// and per channel, over the rows of a sample, S = sums of (g fh, g, dh yh, dh, g x), from which every parameter's gradient
// follows: d wo = gate S0, d bo = gate S1, d gate = wo S0 + bo S1, d wi = (1 + s) S2, d bi = (1 + s) S3, ds = wi S2 + bi S3,
// dt = S3, d rho = S4.
//
// Bound by HBM: a row is read once (8 consecutive channels per thread, kept in registers between its two reductions) and
// written once.  Rows of up to 512 channels belong to 2^k lanes of one wave (sums by lane exchange, no LDS); wider rows to a
// workgroup.  A thread keeps its channels for all its rows, so the parameters are read once per workgroup and the sums S
// live in registers; they leave as one partial row per workgroup and are added in a fixed order (no atomics).  Statistics
// and sums are fp32; y enters the second norm before it is rounded to its storage type.
#include "common.h"

namespace gc {
namespace {

constexpr int kE = 8;              // channels per thread
constexpr int kSums = 5;
constexpr int kMaxThreads = 1024;

enum Part { kIn = 0, kOut = 1, kBoth = 2 };

struct NormParams {
  gc_block_norm a;
  int tpr;                        // threads per row (a power of two; more than 64: the workgroup)
  int vec;                        // 16-byte loads and stores are possible
  int slabs;                      // workgroups per sample
  float* part;                    // backward: [batch][slabs][kSums][cols]
};

template <typename T>
__device__ __forceinline__ void load8(const void* base, int64_t off, int c0, int C, bool vec, float (&v)[kE]) {
  if (vec) {
    const f32x4 a = load4<T>(base, (size_t)(off + c0)), b = load4<T>(base, (size_t)(off + c0 + 4));
#pragma unroll
    for (int e = 0; e < 4; e++) { v[e] = a[e]; v[4 + e] = b[e]; }
  } else {
#pragma unroll
    for (int e = 0; e < kE; e++) {
      v[e] = 0.f;
      if (c0 + e < C) {
        if constexpr (sizeof(T) == 4) v[e] = static_cast<const float*>(base)[off + c0 + e];
        else v[e] = bf16_bits_to_float(static_cast<const uint16_t*>(base)[off + c0 + e]);
      }
    }
  }
}
template <>
__device__ __forceinline__ void load8<uint16_t>(const void* base, int64_t off, int c0, int C, bool vec, float (&v)[kE]) {
  const uint16_t* p = static_cast<const uint16_t*>(base) + off + c0;
  if (vec) {
    const u32x4 q = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
    for (int e = 0; e < 4; e++) {
      v[2 * e] = __builtin_bit_cast(float, q[e] << 16);
      v[2 * e + 1] = __builtin_bit_cast(float, q[e] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int e = 0; e < kE; e++) v[e] = c0 + e < C ? bf16_bits_to_float(p[e]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store8(void* base, int64_t off, int c0, int C, bool vec, const float (&v)[kE]) {
  if (vec) {
    const f32x4 a = {v[0], v[1], v[2], v[3]}, b = {v[4], v[5], v[6], v[7]};
    if constexpr (sizeof(T) == 4) {
      float* p = static_cast<float*>(base) + off + c0;
      *reinterpret_cast<f32x4*>(p) = a;
      *reinterpret_cast<f32x4*>(p + 4) = b;
    } else {
      const u32x2 lo = cvt_bf16x4(a), hi = cvt_bf16x4(b);
      *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(base) + off + c0) = u32x4{lo[0], lo[1], hi[0], hi[1]};
    }
  } else {
#pragma unroll
    for (int e = 0; e < kE; e++)
      if (c0 + e < C) {
        if constexpr (sizeof(T) == 4) static_cast<float*>(base)[off + c0 + e] = v[e];
        else static_cast<uint16_t*>(base)[off + c0 + e] = float_to_bf16_bits(v[e]);
      }
  }
}

// fp32 parameter: null -> `neutral`; one value per channel, or per (sample, channel)
__device__ __forceinline__ void load_param(const float* p, int per_sample, int64_t sample, int c0, int C, float neutral, float (&v)[kE]) {
#pragma unroll
  for (int e = 0; e < kE; e++) v[e] = neutral;
  if (p == nullptr) return;
  p += (per_sample ? sample * C : 0) + c0;
#pragma unroll
  for (int e = 0; e < kE; e++)
    if (c0 + e < C) v[e] = p[e];
}

// Sums of N values over a row's threads, in all of them.  WIDE: the workgroup is the row; `red` holds two sets of
// N * (kMaxThreads / 64) floats used in turn, so one barrier per call is enough (a set is written again only two calls
// later, behind the barrier of the call between).
template <bool WIDE, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], int tpr, float* red, int& turn) {
#pragma unroll
  for (int n = 0; n < N; n++)
    for (int o = (WIDE ? 32 : tpr >> 1); o > 0; o >>= 1) v[n] += __shfl_xor(v[n], o, 64);
  if (WIDE) {
    const int nw = blockDim.x >> 6;
    float* r = red + turn * (2 * (kMaxThreads / 64));
    turn ^= 1;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int n = 0; n < N; n++) r[n * (kMaxThreads / 64) + (threadIdx.x >> 6)] = v[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; n++) {
      float s = 0.f;
      for (int w = 0; w < nw; w++) s += r[n * (kMaxThreads / 64) + w];
      v[n] = s;
    }
  }
}

// mean (0 for the root-mean-square norm) and 1 / standard deviation of a row held as 8 values per thread
template <bool WIDE>
__device__ __forceinline__ void row_stats(const float (&v)[kE], int c0, int C, bool layer, float eps, int tpr, float* red, int& turn, float& mu,
                                          float& r) {
  const float inv = 1.f / (float)C;
  mu = 0.f;
  if (layer) {
    float s[1] = {0.f};
#pragma unroll
    for (int e = 0; e < kE; e++) s[0] += v[e];
    row_sum<WIDE, 1>(s, tpr, red, turn);
    mu = s[0] * inv;
  }
  float q[1] = {0.f};
#pragma unroll
  for (int e = 0; e < kE; e++) {
    const float t = c0 + e < C ? v[e] - mu : 0.f;
    q[0] += t * t;
  }
  row_sum<WIDE, 1>(q, tpr, red, turn);
  r = 1.f / sqrtf(q[0] * inv + eps);
}

template <typename T, bool WIDE, int PART>
__global__ __launch_bounds__(WIDE ? kMaxThreads : kThreads) void block_norm_fwd_kernel(const NormParams P) {
  __shared__ float red[WIDE ? 4 * (kMaxThreads / 64) : 1];
  const gc_block_norm& a = P.a;
  const int C = a.cols, tpr = P.tpr, rpw = WIDE ? 1 : kThreads / tpr;
  const int c0 = (WIDE ? (int)threadIdx.x : (int)threadIdx.x & (tpr - 1)) * kE, sub = WIDE ? 0 : (int)threadIdx.x / tpr;
  const bool mine = c0 < C, layer = a.layer != 0;
  const int64_t sample = blockIdx.y, nstat = a.batch * a.rows;
  int turn = 0;
  float A[kE], B[kE], Cw[kE], D[kE], rho[kE];
  if (PART != kIn) {
    float g[kE];
    load_param(a.gate, a.gate_per_sample, sample, c0, C, 1.f, g);
    load_param(a.out_weight, 0, 0, c0, C, 1.f, A);
    load_param(a.out_bias, 0, 0, c0, C, 0.f, B);
    load_param(a.residual_scale, 0, 0, a.residual_per_channel ? c0 : 0, a.residual_per_channel ? C : 1, a.residual_constant, rho);
#pragma unroll
    for (int e = 0; e < kE; e++) {
      A[e] *= g[e];
      B[e] *= g[e];
      if (a.residual_scale != nullptr && !a.residual_per_channel) rho[e] = rho[0];
    }
  }
  if (PART != kOut) {
    float s[kE], t[kE];
    load_param(a.in_weight, 0, 0, c0, C, 1.f, Cw);
    load_param(a.in_bias, 0, 0, c0, C, 0.f, D);
    load_param(a.scale, a.mod_per_sample, sample, c0, C, 0.f, s);
    load_param(a.shift, a.mod_per_sample, sample, c0, C, 0.f, t);
#pragma unroll
    for (int e = 0; e < kE; e++) {
      Cw[e] *= 1.f + s[e];
      D[e] = D[e] * (1.f + s[e]) + t[e];
    }
  }
  for (int64_t row0 = (int64_t)blockIdx.x * rpw; row0 < a.rows; row0 += (int64_t)gridDim.x * rpw) {
    const int64_t row = row0 + sub;
    const bool live = mine && row < a.rows;
    float y[kE], f[kE];
    // a dead thread (past the last channel or row) takes part in the sums with zeros
    const bool vec = P.vec != 0;
#pragma unroll
    for (int e = 0; e < kE; e++) { y[e] = 0.f; f[e] = 0.f; }
    if (live) {
      load8<T>(a.x, sample * a.x_batch_stride + row * a.x_row_stride, c0, C, vec, y);
      if (PART != kIn) load8<T>(a.f, sample * a.f_batch_stride + row * a.f_row_stride, c0, C, vec, f);
    }
    const int64_t out = (sample * a.rows + row) * C;
    float mu_f = 0.f, r_f = 0.f, mu_y = 0.f, r_y = 0.f;
    if (PART != kIn) {
      row_stats<WIDE>(f, c0, C, layer, a.eps, tpr, red, turn, mu_f, r_f);
#pragma unroll
      for (int e = 0; e < kE; e++) y[e] = c0 + e < C ? rho[e] * y[e] + (A[e] * ((f[e] - mu_f) * r_f) + B[e]) : 0.f;
      if (live) store8<T>(a.y, out, c0, C, vec, y);
    }
    if (PART != kOut) {
      row_stats<WIDE>(y, c0, C, layer, a.eps, tpr, red, turn, mu_y, r_y);
      float h[kE];
#pragma unroll
      for (int e = 0; e < kE; e++) h[e] = Cw[e] * ((y[e] - mu_y) * r_y) + D[e];
      if (live) store8<T>(a.h, out, c0, C, vec, h);
    }
    if (a.stats != nullptr && c0 == 0 && live) {       // [4][batch * rows]: r_f, r_y, mu_f, mu_y (those the parts have)
      const int64_t i = sample * a.rows + row;
      if (PART != kIn) { a.stats[i] = r_f; if (layer) a.stats[2 * nstat + i] = mu_f; }
      if (PART != kOut) { a.stats[nstat + i] = r_y; if (layer) a.stats[3 * nstat + i] = mu_y; }
    }
  }
}

template <typename T, bool WIDE, int PART>
__global__ __launch_bounds__(WIDE ? kMaxThreads : kThreads) void block_norm_bwd_kernel(const NormParams P) {
  __shared__ float red[WIDE ? 4 * (kMaxThreads / 64) : 1];
  __shared__ float fold[WIDE ? 1 : kThreads * kE];
  const gc_block_norm& a = P.a;
  const int C = a.cols, tpr = P.tpr, rpw = WIDE ? 1 : kThreads / tpr;
  const int lane_in_row = WIDE ? (int)threadIdx.x : (int)threadIdx.x & (tpr - 1);
  const int c0 = lane_in_row * kE, sub = WIDE ? 0 : (int)threadIdx.x / tpr;
  const bool mine = c0 < C, layer = a.layer != 0, vec = P.vec != 0;
  const int64_t sample = blockIdx.y, nstat = a.batch * a.rows;
  const float inv = 1.f / (float)C;
  int turn = 0;
  float A[kE], B[kE], Cw[kE], rho[kE];
  if (PART != kIn) {
    float g[kE];
    load_param(a.gate, a.gate_per_sample, sample, c0, C, 1.f, g);
    load_param(a.out_weight, 0, 0, c0, C, 1.f, A);
    load_param(a.out_bias, 0, 0, c0, C, 0.f, B);
    load_param(a.residual_scale, 0, 0, a.residual_per_channel ? c0 : 0, a.residual_per_channel ? C : 1, a.residual_constant, rho);
#pragma unroll
    for (int e = 0; e < kE; e++) {
      A[e] *= g[e];
      B[e] *= g[e];
      if (a.residual_scale != nullptr && !a.residual_per_channel) rho[e] = rho[0];
    }
  }
  if (PART != kOut) {
    float s[kE];
    load_param(a.in_weight, 0, 0, c0, C, 1.f, Cw);
    load_param(a.scale, a.mod_per_sample, sample, c0, C, 0.f, s);
#pragma unroll
    for (int e = 0; e < kE; e++) Cw[e] *= 1.f + s[e];
  }
  float S[kSums][kE];
#pragma unroll
  for (int k = 0; k < kSums; k++)
#pragma unroll
    for (int e = 0; e < kE; e++) S[k][e] = 0.f;

  for (int64_t row0 = (int64_t)blockIdx.x * rpw; row0 < a.rows; row0 += (int64_t)gridDim.x * rpw) {
    const int64_t row = row0 + sub;
    const bool live = mine && row < a.rows;
    float x[kE], f[kE], g[kE], dh[kE];
#pragma unroll
    for (int e = 0; e < kE; e++) { x[e] = 0.f; f[e] = 0.f; g[e] = 0.f; dh[e] = 0.f; }
    const int64_t out = (sample * a.rows + row) * C;
    float r_f = 0.f, r_y = 0.f, mu_f = 0.f, mu_y = 0.f;
    if (live) {
      load8<T>(a.x, sample * a.x_batch_stride + row * a.x_row_stride, c0, C, vec, x);
      if (PART != kIn) load8<T>(a.f, sample * a.f_batch_stride + row * a.f_row_stride, c0, C, vec, f);
      if (PART != kIn && a.dy != nullptr) load8<T>(a.dy, out, c0, C, vec, g);
      if (PART != kOut && a.dh != nullptr) load8<T>(a.dh, out, c0, C, vec, dh);
      const int64_t i = sample * a.rows + row;
      if (PART != kIn) { r_f = a.stats[i]; if (layer) mu_f = a.stats[2 * nstat + i]; }
      if (PART != kOut) { r_y = a.stats[nstat + i]; if (layer) mu_y = a.stats[3 * nstat + i]; }
    }
    if (PART != kIn)
#pragma unroll
      for (int e = 0; e < kE; e++) f[e] = c0 + e < C ? (f[e] - mu_f) * r_f : 0.f;          // fh from here on
    if (PART != kOut) {
      float yh[kE], m[2] = {0.f, 0.f};
#pragma unroll
      for (int e = 0; e < kE; e++) {
        const float y = PART == kIn ? x[e] : rho[e] * x[e] + (A[e] * f[e] + B[e]);
        yh[e] = c0 + e < C ? (y - mu_y) * r_y : 0.f;
        S[2][e] += dh[e] * yh[e];
        S[3][e] += dh[e];
        const float q = Cw[e] * dh[e];
        m[0] += q * yh[e];
        m[1] += q;
      }
      row_sum<WIDE, 2>(m, tpr, red, turn);
      const float mq = m[0] * inv, m1 = layer ? m[1] * inv : 0.f;
#pragma unroll
      for (int e = 0; e < kE; e++) g[e] += r_y * (Cw[e] * dh[e] - yh[e] * mq - m1);
    }
    if (PART == kIn) {
      if (live) store8<T>(a.dx, out, c0, C, vec, g);
    } else {
      float p[kE], m[2] = {0.f, 0.f};
#pragma unroll
      for (int e = 0; e < kE; e++) {
        if (c0 + e >= C) g[e] = 0.f;
        S[0][e] += g[e] * f[e];
        S[1][e] += g[e];
        S[4][e] += g[e] * x[e];
        p[e] = A[e] * g[e];
        m[0] += p[e] * f[e];
        m[1] += p[e];
        x[e] = rho[e] * g[e];
      }
      if (live) store8<T>(a.dx, out, c0, C, vec, x);
      row_sum<WIDE, 2>(m, tpr, red, turn);
      const float mp = m[0] * inv, m1 = layer ? m[1] * inv : 0.f;
#pragma unroll
      for (int e = 0; e < kE; e++) p[e] = r_f * (p[e] - f[e] * mp - m1);
      if (live) store8<T>(a.df, out, c0, C, vec, p);
    }
  }

  // the workgroup's sums: rows handled side by side are folded in a fixed order, one sum at a time
  float* dst = P.part + ((size_t)sample * gridDim.x + blockIdx.x) * kSums * C;
#pragma unroll
  for (int k = 0; k < kSums; k++) {
    if ((PART == kIn && k != 2 && k != 3) || (PART == kOut && (k == 2 || k == 3))) continue;
    if (!WIDE) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < kE; e++) fold[threadIdx.x * kE + e] = S[k][e];
      __syncthreads();
      for (int i = threadIdx.x; i < tpr * kE; i += kThreads) {
        float s = 0.f;
        for (int r = 0; r < rpw; r++) s += fold[r * tpr * kE + i];
        if (i < C) dst[(size_t)k * C + i] = s;
      }
    } else {
#pragma unroll
      for (int e = 0; e < kE; e++)
        if (c0 + e < C) dst[(size_t)k * C + c0 + e] = S[k][e];
    }
  }
}

// part [batch][slabs][kSums][C] -> sums [batch][kSums][C].  grid (C / 16, kSums, batch), 1024 threads: 16 channels x 64 rows
__global__ __launch_bounds__(1024) void block_norm_sums_kernel(const float* part, float* sums, int slabs, int C, int parts) {
  const int k = blockIdx.y;
  if (((parts == kIn) && k != 2 && k != 3) || (parts == kOut && (k == 2 || k == 3))) return;
  __shared__ float red[64][17];
  const int c = blockIdx.x * 16 + (threadIdx.x & 15), r0 = threadIdx.x >> 4;
  const int64_t sample = blockIdx.z;
  float s = 0.f;
  if (c < C)
    for (int r = r0; r < slabs; r += 64) s += part[((sample * slabs + r) * kSums + k) * C + c];
  red[r0][threadIdx.x & 15] = s;
  __syncthreads();
  if (threadIdx.x < 16 && c < C) {
    float t = 0.f;
#pragma unroll
    for (int r = 0; r < 64; r++) t += red[r][threadIdx.x];
    sums[(sample * kSums + k) * C + c] = t;
  }
}

// Parameter gradients from the samples' sums.  Blocks 0 .. n - 1: 64 channels x 4 threads each; block n: the gradient of a
// scalar residual scale.
__global__ __launch_bounds__(kThreads) void block_norm_params_kernel(const gc_block_norm a, const float* sums, int parts) {
  __shared__ float red[5][4][64];
  const int C = a.cols;
  if (blockIdx.x == gridDim.x - 1) {
    if (a.d_residual_scale == nullptr || a.residual_per_channel || parts == kIn) return;
    float s = 0.f;
    for (int64_t b = 0; b < a.batch; b++)
      for (int c = threadIdx.x; c < C; c += kThreads) s += sums[(b * kSums + 4) * C + c];
    float* r = &red[0][0][0];
    r[threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
      float t = 0.f;
      for (int i = 0; i < kThreads; i++) t += r[i];
      a.d_residual_scale[0] = t;
    }
    return;
  }
  const int lc = threadIdx.x & 63, q = threadIdx.x >> 6, c = blockIdx.x * 64 + lc;
  float acc[5] = {0.f, 0.f, 0.f, 0.f, 0.f};      // out_weight, out_bias, in_weight, in_bias, residual scale
  float gsum = 0.f, ssum = 0.f, tsum = 0.f;       // gate, scale, shift where all samples share them (those have batch 1 or are summed)
  const float wo = c < C && a.out_weight ? a.out_weight[c] : 1.f, bo = c < C && a.out_bias ? a.out_bias[c] : 0.f;
  const float wi = c < C && a.in_weight ? a.in_weight[c] : 1.f, bi = c < C && a.in_bias ? a.in_bias[c] : 0.f;
  if (c < C)
    for (int64_t b = q; b < a.batch; b += 4) {
      const float* S = sums + b * kSums * C + c;
      if (parts != kIn) {
        const float g = a.gate ? a.gate[(a.gate_per_sample ? b * C : 0) + c] : 1.f, s0 = S[0], s1 = S[C];
        acc[0] += g * s0;
        acc[1] += g * s1;
        acc[4] += S[4 * C];
        const float dg = wo * s0 + bo * s1;
        if (a.gate_per_sample) { if (a.d_gate) a.d_gate[b * C + c] = dg; }
        else gsum += dg;
      }
      if (parts != kOut) {
        const float m = 1.f + (a.scale ? a.scale[(a.mod_per_sample ? b * C : 0) + c] : 0.f), s2 = S[2 * C], s3 = S[3 * C];
        acc[2] += m * s2;
        acc[3] += m * s3;
        const float ds = wi * s2 + bi * s3;
        if (a.mod_per_sample) {
          if (a.d_scale) a.d_scale[b * C + c] = ds;
          if (a.d_shift) a.d_shift[b * C + c] = s3;
        } else { ssum += ds; tsum += s3; }
      }
    }
#pragma unroll
  for (int k = 0; k < 5; k++) red[k][q][lc] = acc[k];
  __syncthreads();
  if (q == 0 && c < C) {
    float* dst[5] = {a.d_out_weight, a.d_out_bias, a.d_in_weight, a.d_in_bias, a.residual_per_channel ? a.d_residual_scale : nullptr};
#pragma unroll
    for (int k = 0; k < 5; k++)
      if (dst[k]) dst[k][c] = ((red[k][0][lc] + red[k][1][lc]) + red[k][2][lc]) + red[k][3][lc];
  }
  __syncthreads();
  red[0][q][lc] = gsum;
  red[1][q][lc] = ssum;
  red[2][q][lc] = tsum;
  __syncthreads();
  if (q == 0 && c < C) {
    float* dst[3] = {a.gate_per_sample ? nullptr : a.d_gate, a.mod_per_sample ? nullptr : a.d_scale, a.mod_per_sample ? nullptr : a.d_shift};
#pragma unroll
    for (int k = 0; k < 3; k++)
      if (dst[k]) dst[k][c] = ((red[k][0][lc] + red[k][1][lc]) + red[k][2][lc]) + red[k][3][lc];
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Checks the descriptor; parts: which of the two norms it asks for.
int check_desc(const gc_block_norm* d, bool bwd, int& parts) {
  if (d == nullptr || d->x == nullptr) { set_error("block norm: descriptor and x must not be null"); return GC_BAD_ARGUMENT; }
  if (d->dtype != GC_F32 && d->dtype != GC_BF16) { set_error("block norm: dtype must be GC_F32 or GC_BF16"); return GC_BAD_ARGUMENT; }
  if (d->batch < 0 || d->rows < 0 || d->cols <= 0 || d->cols > kMaxThreads * kE || d->batch > 65535) {
    set_error("block norm: 1 <= cols <= %d, 0 <= batch <= 65535, rows >= 0 are supported (got batch=%lld rows=%lld cols=%d)", kMaxThreads * kE,
              (long long)d->batch, (long long)d->rows, d->cols);
    return GC_UNSUPPORTED_GEOMETRY;
  }
  const bool out = d->f != nullptr, in = d->with_input_norm != 0;
  if (!out && !in) { set_error("block norm: neither f (norm behind a block) nor with_input_norm (norm in front of one) is given"); return GC_BAD_ARGUMENT; }
  if (!(d->eps > 0.f)) { set_error("block norm: eps must be positive"); return GC_BAD_ARGUMENT; }
  parts = out && in ? kBoth : (out ? kOut : kIn);
  if (!bwd) {
    if ((out && d->y == nullptr) || (in && d->h == nullptr)) { set_error("block norm: an output pointer is null"); return GC_BAD_ARGUMENT; }
  } else {
    if (d->stats == nullptr || d->dx == nullptr || (out && d->df == nullptr) || (d->dy == nullptr && d->dh == nullptr)) {
      set_error("block norm backward: stats, dx, df and one of dy, dh must not be null");
      return GC_BAD_ARGUMENT;
    }
  }
  return GC_OK;
}

int slab_count(const gc_block_norm* d, int tpr, bool bwd) {
  const int64_t rpw = tpr > 64 ? 1 : kThreads / tpr, passes = (d->rows + rpw - 1) / rpw;
  // enough workgroups to fill the chip; the backward pass writes (and its second launch reads) one row of sums per workgroup
  const int64_t fill = (int64_t)device_cu_count() * (bwd ? 4 : 8) * (tpr > kThreads ? 1 : 1);
  int64_t s = (fill + d->batch - 1) / d->batch;
  if (s > passes) s = passes;
  return (int)(s < 1 ? 1 : s);
}

NormParams make_params(const gc_block_norm* d, bool bwd) {
  NormParams P{};
  P.a = *d;
  int tpr = 1;
  while (tpr * kE < d->cols) tpr *= 2;
  P.tpr = tpr;
  const int unit = kE;
  P.vec = d->cols % unit == 0 && d->x_row_stride % unit == 0 && d->x_batch_stride % unit == 0 && d->f_row_stride % unit == 0 &&
          d->f_batch_stride % unit == 0 && aligned16(d->x) && aligned16(d->f) && aligned16(d->y) && aligned16(d->h) && aligned16(d->dy) &&
          aligned16(d->dh) && aligned16(d->dx) && aligned16(d->df);
  P.slabs = slab_count(d, tpr, bwd);
  return P;
}

template <typename T, bool WIDE>
void launch_fwd(const NormParams& P, int parts, hipStream_t s) {
  const dim3 grid(P.slabs, (unsigned)P.a.batch), block(WIDE ? P.tpr : kThreads);
  if (parts == kIn) hipLaunchKernelGGL((block_norm_fwd_kernel<T, WIDE, kIn>), grid, block, 0, s, P);
  else if (parts == kOut) hipLaunchKernelGGL((block_norm_fwd_kernel<T, WIDE, kOut>), grid, block, 0, s, P);
  else hipLaunchKernelGGL((block_norm_fwd_kernel<T, WIDE, kBoth>), grid, block, 0, s, P);
}
template <typename T, bool WIDE>
void launch_bwd(const NormParams& P, int parts, hipStream_t s) {
  const dim3 grid(P.slabs, (unsigned)P.a.batch), block(WIDE ? P.tpr : kThreads);
  if (parts == kIn) hipLaunchKernelGGL((block_norm_bwd_kernel<T, WIDE, kIn>), grid, block, 0, s, P);
  else if (parts == kOut) hipLaunchKernelGGL((block_norm_bwd_kernel<T, WIDE, kOut>), grid, block, 0, s, P);
  else hipLaunchKernelGGL((block_norm_bwd_kernel<T, WIDE, kBoth>), grid, block, 0, s, P);
}

}  // namespace
}  // namespace gc

using namespace gc;

extern "C" int gc_block_norm_fwd(const gc_block_norm* desc, void* stream) {
  int parts = 0;
  if (int e = check_desc(desc, false, parts)) return e;
  if (desc->batch == 0 || desc->rows == 0) return GC_OK;
  const NormParams P = make_params(desc, false);
  hipStream_t s = (hipStream_t)stream;
  ProfScope ps("gc::block_norm_fwd_kernel", 0.0, s);
  const bool wide = P.tpr > 64;
  if (desc->dtype == GC_F32) { if (wide) launch_fwd<float, true>(P, parts, s); else launch_fwd<float, false>(P, parts, s); }
  else { if (wide) launch_fwd<uint16_t, true>(P, parts, s); else launch_fwd<uint16_t, false>(P, parts, s); }
  return check_hip(hipGetLastError(), "block_norm fwd launch");
}

extern "C" size_t gc_block_norm_workspace_bytes(int64_t batch, int64_t rows, int32_t cols) {
  if (batch <= 0 || rows <= 0 || cols <= 0) return 0;
  int tpr = 1;
  while (tpr * kE < cols) tpr *= 2;
  gc_block_norm d{};
  d.batch = batch; d.rows = rows; d.cols = cols;
  return ((size_t)batch * slab_count(&d, tpr, true) + batch) * kSums * (size_t)cols * sizeof(float);
}

extern "C" int gc_block_norm_bwd(const gc_block_norm* desc, void* workspace, size_t workspace_bytes, void* stream) {
  int parts = 0;
  if (int e = check_desc(desc, true, parts)) return e;
  if (desc->batch == 0 || desc->rows == 0) {
    set_error("block norm backward: an empty tensor has no gradient to compute");
    return GC_BAD_ARGUMENT;
  }
  const size_t need = gc_block_norm_workspace_bytes(desc->batch, desc->rows, desc->cols);
  if (workspace == nullptr || !aligned16(workspace) || workspace_bytes < need) {
    set_error("block norm backward: a 16-byte aligned workspace of %zu bytes is needed", need);
    return GC_WORKSPACE_TOO_SMALL;
  }
  NormParams P = make_params(desc, true);
  float* sums = static_cast<float*>(workspace);
  P.part = sums + (size_t)desc->batch * kSums * desc->cols;
  hipStream_t s = (hipStream_t)stream;
  {
    ProfScope ps("gc::block_norm_bwd_kernel", 0.0, s);
    const bool wide = P.tpr > 64;
    if (desc->dtype == GC_F32) { if (wide) launch_bwd<float, true>(P, parts, s); else launch_bwd<float, false>(P, parts, s); }
    else { if (wide) launch_bwd<uint16_t, true>(P, parts, s); else launch_bwd<uint16_t, false>(P, parts, s); }
    if (check_hip(hipGetLastError(), "block_norm bwd launch")) return GC_HIP_ERROR;
  }
  const float* totals = P.part;
  if (P.slabs > 1) {
    hipLaunchKernelGGL(block_norm_sums_kernel, dim3((desc->cols + 15) / 16, kSums, (unsigned)desc->batch), dim3(1024), 0, s, (const float*)P.part,
                       sums, P.slabs, desc->cols, parts);
    if (check_hip(hipGetLastError(), "block_norm sums launch")) return GC_HIP_ERROR;
    totals = sums;
  }
  hipLaunchKernelGGL(block_norm_params_kernel, dim3((desc->cols + 63) / 64 + 1), dim3(kThreads), 0, s, *desc, totals, parts);
  return check_hip(hipGetLastError(), "block_norm params launch");
}
