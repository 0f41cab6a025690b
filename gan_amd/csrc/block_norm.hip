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
// and sums are fp32; y enters the second norm before it is rounded to its storage type.  64 x 4096 rows of 128 bf16, both parts: forward
// 61 us, backward 92 (4.4 TB/s both; a large copy reaches 4.9) and 11 for the parameters; 16384 rows of 4096 forward 113 (4.7 TB/s).
#include <mutex>

#include "common.h"

namespace gc {
namespace {

constexpr int kSums = 5;
constexpr int kMaxThreads = 512, kMaxCols = 16 * kMaxThreads;

enum Part { kIn = 0, kOut = 1, kBoth = 2 };

struct NormParams {
  gc_block_norm a;
  int tpr;                        // threads per row (a power of two; more than 64: the workgroup)
  int width;                      // neighbouring elements per access
  int slabs;                      // workgroups per sample
  float* part;                    // backward: [batch][slabs][kSums][cols]
  float* rho_part;                // [batch][slabs], or null (no scalar residual scale asked for)
};

// A thread's E channels (8, or 16 in rows of more than 4096) lie in E / W runs of W neighbours, a run of all threads of the row behind the other, so that every load
// instruction of a wave covers one contiguous stretch: W = 8 (bf16) or 4 (fp32) for 16-byte accesses; where the row length, a stride or
// an address does not allow them 4 bytes, W = 2 or 1, at any address that an element may have (the memory takes unaligned ones; a row's
// last element goes alone if the row is odd).  262144 rows of 128 bf16, forward and backward: 164 us in 16-byte, 172 in 4-byte accesses,
// 411 element by element.
typedef uint32_t __attribute__((aligned(2))) u32_any;
template <int W>
struct Lane {
  int first, step, C;
  __device__ __forceinline__ Lane(int t, int tpr, int C_) : first(t * W), step(tpr * W), C(C_) {}
  __device__ __forceinline__ int ch(int e) const { return (e / W) * step + first + e % W; }
  __device__ __forceinline__ bool has(int e) const { return ch(e) < C; }
};

template <typename T, int E> struct Raw { uint32_t w[E * sizeof(T) / 4]; };    // E values as stored

template <typename T, int W, int E>
__device__ __forceinline__ Raw<T, E> load_raw(const void* base, int64_t off, const Lane<W>& L, bool live) {
  Raw<T, E> r;
#pragma unroll
  for (int i = 0; i < (int)(E * sizeof(T) / 4); i++) r.w[i] = 0u;
  if (!live) return r;
  const T* p = static_cast<const T*>(base) + off;
  if constexpr (W > 1) {
    constexpr int words = W * sizeof(T) / 4;                                    // one access of 4 or 16 bytes per run
#pragma unroll
    for (int k = 0; k < E / W; k++)
      if (L.has(k * W)) {
        if constexpr (words == 1) {
          if (L.has(k * W + 1)) r.w[k] = *reinterpret_cast<const u32_any*>(p + L.ch(k * W));
          else r.w[k] = p[L.ch(k * W)];
        } else {
          const u32x4 q = *reinterpret_cast<const u32x4*>(p + L.ch(k * W));
#pragma unroll
          for (int i = 0; i < words; i++) r.w[k * words + i] = q[i];
        }
      }
  } else {
#pragma unroll
    for (int e = 0; e < E; e++)
      if (L.has(e)) r.w[e] = __builtin_bit_cast(uint32_t, p[L.ch(e)]);
  }
  return r;
}
template <typename T, int E>
__device__ __forceinline__ void widen(const Raw<T, E>& r, float (&v)[E]) {
#pragma unroll
  for (int e = 0; e < E; e++) {
    if constexpr (sizeof(T) == 4) { const uint32_t u = r.w[e]; v[e] = __builtin_bit_cast(float, u); }
    else v[e] = __builtin_bit_cast(float, (e & 1) ? (r.w[e / 2] & 0xffff0000u) : (r.w[e / 2] << 16));
  }
}
template <typename T, int W, int E>
__device__ __forceinline__ void store_row(void* base, int64_t off, const Lane<W>& L, const float (&v)[E]) {
  T* p = static_cast<T*>(base) + off;
  if constexpr (W > 1) {
#pragma unroll
    for (int k = 0; k < E / W; k++)
      if (L.has(k * W)) {
        if constexpr (sizeof(T) == 4) {
          *reinterpret_cast<f32x4*>(p + L.ch(k * W)) = f32x4{v[k * W], v[k * W + 1], v[k * W + 2], v[k * W + 3]};
        } else if constexpr (W == 2) {
          const uint32_t u = cvt_bf16x4(f32x4{v[2 * k], v[2 * k + 1], 0.f, 0.f})[0];
          if (L.has(k * W + 1)) *reinterpret_cast<u32_any*>(p + L.ch(k * W)) = u;
          else p[L.ch(k * W)] = (uint16_t)u;
        } else {
          const float* u = v + k * W;
          const u32x2 lo = cvt_bf16x4(f32x4{u[0], u[1], u[2], u[3]}), hi = cvt_bf16x4(f32x4{u[4], u[5], u[6], u[7]});
          *reinterpret_cast<u32x4*>(p + L.ch(k * W)) = u32x4{lo[0], lo[1], hi[0], hi[1]};
        }
      }
  } else {
#pragma unroll
    for (int e = 0; e < E; e++)
      if (L.has(e)) p[L.ch(e)] = v[e];
  }
}

// fp32 parameter: null -> `neutral`; one value per channel, or per (sample, channel)
template <int W, int E>
__device__ __forceinline__ void load_param(const float* p, int per_sample, int64_t sample, const Lane<W>& L, float neutral, float (&v)[E]) {
#pragma unroll
  for (int e = 0; e < E; e++) v[e] = neutral;
  if (p == nullptr) return;
  p += per_sample ? sample * L.C : 0;
#pragma unroll
  for (int e = 0; e < E; e++)
    if (L.has(e)) v[e] = p[L.ch(e)];
}
template <int W, int E>
__device__ __forceinline__ void load_rho(const gc_block_norm& a, const Lane<W>& L, float (&v)[E]) {
  if (a.residual_per_channel) { load_param<W, E>(a.residual_scale, 0, 0, L, 1.f, v); return; }
  const float r = a.residual_scale != nullptr ? a.residual_scale[0] : a.residual_constant;
#pragma unroll
  for (int e = 0; e < E; e++) v[e] = r;
}

// v + the value of the lane whose number differs in one bit, in the vector unit: within 16 lanes by data-parallel-primitive moves (the
// sums of a quad / of 8 lanes are already equal when lanes are mirrored within 8 / 16), beyond by the row and half-wave swaps.
template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
template <bool HALVES>
__device__ __forceinline__ float swap_add(float v) {
  typedef unsigned int u32pair __attribute__((ext_vector_type(2)));
  const unsigned int u = __builtin_bit_cast(unsigned int, v);
  const u32pair r = HALVES ? __builtin_amdgcn_permlane32_swap(u, u, false, false) : __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const unsigned int x = r[0], y = r[1];                   // (scalars first: a bit cast of a vector's element itself reads element 0)
  return __builtin_bit_cast(float, x) + __builtin_bit_cast(float, y);
}
// Sum over groups of n (a power of two up to 64) neighbouring lanes, in all of them
__device__ __forceinline__ float lanes_sum(float v, int n) {
  if (n >= 2) v = dpp_add<0xb1>(v);                        // quad_perm 1 0 3 2
  if (n >= 4) v = dpp_add<0x4e>(v);                        // quad_perm 2 3 0 1
  if (n >= 8) v = dpp_add<0x141>(v);                       // mirrored within 8
  if (n >= 16) v = dpp_add<0x140>(v);                      // mirrored within 16
  if (n >= 32) v = swap_add<false>(v);
  if (n >= 64) v = swap_add<true>(v);
  return v;
}

// Sums of N values over a row's threads, in all of them.  WIDE: the workgroup is the row; `red` holds two sets of
// N * (kMaxThreads / 64) floats used in turn, so one barrier per call is enough (a set is written again only two calls
// later, behind the barrier of the call between).
template <bool WIDE, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], int tpr, float* red, int& turn) {
#pragma unroll
  for (int n = 0; n < N; n++) v[n] = lanes_sum(v[n], WIDE ? 64 : tpr);
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

// mean (0 for the root-mean-square norm) and 1 / standard deviation of a row held as E values per thread
template <bool WIDE, int W, int E>
__device__ __forceinline__ void row_stats(const float (&v)[E], const Lane<W>& L, bool layer, float eps, int tpr, float* red, int& turn, float& mu, float& r) {
  const float inv = 1.f / (float)L.C;
  mu = 0.f;
  if (layer) {
    float s[1] = {0.f};
#pragma unroll
    for (int e = 0; e < E; e++) s[0] += v[e];
    row_sum<WIDE, 1>(s, tpr, red, turn);
    mu = s[0] * inv;
  }
  float q[1] = {0.f};
#pragma unroll
  for (int e = 0; e < E; e++) {
    const float t = L.has(e) ? v[e] - mu : 0.f;
    q[0] += t * t;
  }
  row_sum<WIDE, 1>(q, tpr, red, turn);
  r = 1.f / sqrtf(q[0] * inv + eps);
}

// The rows of a workgroup: side by side (narrow rows) and one after the other.  The next rows are asked for before the current ones are
// worked on: the two reductions of a row leave no other work to hide the loads behind.
// MAXT: 256 (narrow rows) or the most threads a wide row takes, 512: that leaves the backward pass the registers it needs, also for 16
// channels per thread, and 1024 threads do not (16384 rows of 2048 bf16, forward and backward: 193 against 338 us; of 8192: 1260 against 624).
template <typename T, int MAXT, int PART, int W, int E>
__global__ __launch_bounds__(MAXT) void block_norm_fwd_kernel(const NormParams P) {
  constexpr bool WIDE = MAXT > kThreads;
  __shared__ float red[WIDE ? 4 * (kMaxThreads / 64) : 1];
  const gc_block_norm& a = P.a;
  const int C = a.cols, tpr = P.tpr, rpw = WIDE ? 1 : kThreads / tpr;
  const int t = WIDE ? (int)threadIdx.x : (int)threadIdx.x & (tpr - 1), sub = WIDE ? 0 : (int)threadIdx.x / tpr;
  const Lane<W> L(t, tpr, C);
  const bool layer = a.layer != 0;
  const int64_t sample = blockIdx.y, nstat = a.batch * a.rows, hop = (int64_t)gridDim.x * rpw;
  int turn = 0;
  // a thread past the last row takes part in the sums with zeros
  int64_t row = (int64_t)blockIdx.x * rpw + sub;
  Raw<T, E> rx = load_raw<T, W, E>(a.x, sample * a.x_batch_stride + row * a.x_row_stride, L, row < a.rows), rf;
  if (PART != kIn) rf = load_raw<T, W, E>(a.f, sample * a.f_batch_stride + row * a.f_row_stride, L, row < a.rows);
  float A[E], B[E], Cw[E], D[E], rho[E];
  if (PART != kIn) {
    float g[E];
    load_param<W, E>(a.gate, a.gate_per_sample, sample, L, 1.f, g);
    load_param<W, E>(a.out_weight, 0, 0, L, 1.f, A);
    load_param<W, E>(a.out_bias, 0, 0, L, 0.f, B);
    load_rho<W, E>(a, L, rho);
#pragma unroll
    for (int e = 0; e < E; e++) {
      A[e] *= g[e];
      B[e] *= g[e];
    }
  }
  if (PART != kOut) {
    float s[E], sh[E];
    load_param<W, E>(a.in_weight, 0, 0, L, 1.f, Cw);
    load_param<W, E>(a.in_bias, 0, 0, L, 0.f, D);
    load_param<W, E>(a.scale, a.mod_per_sample, sample, L, 0.f, s);
    load_param<W, E>(a.shift, a.mod_per_sample, sample, L, 0.f, sh);
#pragma unroll
    for (int e = 0; e < E; e++) {
      Cw[e] *= 1.f + s[e];
      D[e] = D[e] * (1.f + s[e]) + sh[e];
    }
  }
  for (int64_t row0 = (int64_t)blockIdx.x * rpw; row0 < a.rows; row0 += hop, row += hop) {
    const bool live = row < a.rows;
    float y[E], f[E];
    widen<T, E>(rx, y);
    if (PART != kIn) widen<T, E>(rf, f);
    if (row0 + hop < a.rows) {
      const int64_t next = row + hop;
      rx = load_raw<T, W, E>(a.x, sample * a.x_batch_stride + next * a.x_row_stride, L, next < a.rows);
      if (PART != kIn) rf = load_raw<T, W, E>(a.f, sample * a.f_batch_stride + next * a.f_row_stride, L, next < a.rows);
    }
    const int64_t out = (sample * a.rows + row) * C;
    float mu_f = 0.f, r_f = 0.f, mu_y = 0.f, r_y = 0.f;
    if (PART != kIn) {
      row_stats<WIDE, W, E>(f, L, layer, a.eps, tpr, red, turn, mu_f, r_f);
#pragma unroll
      for (int e = 0; e < E; e++) y[e] = L.has(e) ? rho[e] * y[e] + (A[e] * ((f[e] - mu_f) * r_f) + B[e]) : 0.f;
      if (live) store_row<T, W, E>(a.y, out, L, y);
    }
    if (PART != kOut) {
      row_stats<WIDE, W, E>(y, L, layer, a.eps, tpr, red, turn, mu_y, r_y);
      float h[E];
#pragma unroll
      for (int e = 0; e < E; e++) h[e] = Cw[e] * ((y[e] - mu_y) * r_y) + D[e];
      if (live) store_row<T, W, E>(a.h, out, L, h);
    }
    if (a.stats != nullptr && t == 0 && live) {            // [4][batch * rows]: r_f, r_y, mu_f, mu_y (those the parts have)
      const int64_t i = sample * a.rows + row;
      if (PART != kIn) { a.stats[i] = r_f; if (layer) a.stats[2 * nstat + i] = mu_f; }
      if (PART != kOut) { a.stats[nstat + i] = r_y; if (layer) a.stats[3 * nstat + i] = mu_y; }
    }
  }
}

template <typename T, int MAXT, int PART, int W, int E>
__global__ __launch_bounds__(MAXT) void block_norm_bwd_kernel(const NormParams P) {
  constexpr bool WIDE = MAXT > kThreads;
  __shared__ float red[WIDE ? 4 * (kMaxThreads / 64) : 1];
  __shared__ float fold[WIDE ? 1 : kThreads * E], scalar[MAXT / 64];
  const gc_block_norm& a = P.a;
  const int C = a.cols, tpr = P.tpr, rpw = WIDE ? 1 : kThreads / tpr;
  const int t = WIDE ? (int)threadIdx.x : (int)threadIdx.x & (tpr - 1), sub = WIDE ? 0 : (int)threadIdx.x / tpr;
  const Lane<W> L(t, tpr, C);
  const bool layer = a.layer != 0;
  const int64_t sample = blockIdx.y, nstat = a.batch * a.rows, hop = (int64_t)gridDim.x * rpw;
  const float inv = 1.f / (float)C;
  int turn = 0;
  struct Row { Raw<T, E> x, f, dy, dh; float st[4]; } next;
  auto ask = [&](int64_t row) {
    const bool live = row < a.rows;
    const int64_t out = (sample * a.rows + row) * C, i = sample * a.rows + row;
    next.x = load_raw<T, W, E>(a.x, sample * a.x_batch_stride + row * a.x_row_stride, L, live);
    if (PART != kIn) next.f = load_raw<T, W, E>(a.f, sample * a.f_batch_stride + row * a.f_row_stride, L, live);
    if (PART != kIn) next.dy = load_raw<T, W, E>(a.dy, out, L, live && a.dy != nullptr);
    if (PART != kOut) next.dh = load_raw<T, W, E>(a.dh, out, L, live && a.dh != nullptr);
#pragma unroll
    for (int k = 0; k < 4; k++) next.st[k] = 0.f;
    if (live) {
      if (PART != kIn) { next.st[0] = a.stats[i]; if (layer) next.st[2] = a.stats[2 * nstat + i]; }
      if (PART != kOut) { next.st[1] = a.stats[nstat + i]; if (layer) next.st[3] = a.stats[3 * nstat + i]; }
    }
  };
  constexpr bool AHEAD = E == 8 || PART != kBoth;          // (16 channels of everything leave no registers for the next row)
  int64_t row = (int64_t)blockIdx.x * rpw + sub;
  if (AHEAD) ask(row);
  float A[E], B[E], Cw[E], rho[E];
  if (PART != kIn) {
    float g[E];
    load_param<W, E>(a.gate, a.gate_per_sample, sample, L, 1.f, g);
    load_param<W, E>(a.out_weight, 0, 0, L, 1.f, A);
    load_param<W, E>(a.out_bias, 0, 0, L, 0.f, B);
    load_rho<W, E>(a, L, rho);
#pragma unroll
    for (int e = 0; e < E; e++) {
      A[e] *= g[e];
      B[e] *= g[e];
    }
  }
  if (PART != kOut) {
    float s[E];
    load_param<W, E>(a.in_weight, 0, 0, L, 1.f, Cw);
    load_param<W, E>(a.scale, a.mod_per_sample, sample, L, 0.f, s);
#pragma unroll
    for (int e = 0; e < E; e++) Cw[e] *= 1.f + s[e];
  }
  float S[kSums][E];
#pragma unroll
  for (int k = 0; k < kSums; k++)
#pragma unroll
    for (int e = 0; e < E; e++) S[k][e] = 0.f;

  for (int64_t row0 = (int64_t)blockIdx.x * rpw; row0 < a.rows; row0 += hop, row += hop) {
    const bool live = row < a.rows;
    float x[E], f[E], g[E], dh[E];
    if (!AHEAD) ask(row);
    widen<T, E>(next.x, x);
    if (PART != kIn) { widen<T, E>(next.f, f); widen<T, E>(next.dy, g); }
    else
#pragma unroll
      for (int e = 0; e < E; e++) g[e] = 0.f;
    if (PART != kOut) widen<T, E>(next.dh, dh);
    const float r_f = next.st[0], r_y = next.st[1], mu_f = next.st[2], mu_y = next.st[3];
    if (AHEAD && row0 + hop < a.rows) ask(row + hop);
    const int64_t out = (sample * a.rows + row) * C;
    if (PART != kIn)
#pragma unroll
      for (int e = 0; e < E; e++) f[e] = L.has(e) ? (f[e] - mu_f) * r_f : 0.f;            // fh from here on
    if (PART != kOut) {
      float yh[E], m[2] = {0.f, 0.f};
#pragma unroll
      for (int e = 0; e < E; e++) {
        const float y = PART == kIn ? x[e] : rho[e] * x[e] + (A[e] * f[e] + B[e]);
        yh[e] = L.has(e) ? (y - mu_y) * r_y : 0.f;
        S[2][e] += dh[e] * yh[e];
        S[3][e] += dh[e];
        const float q = Cw[e] * dh[e];
        m[0] += q * yh[e];
        m[1] += q;
      }
      row_sum<WIDE, 2>(m, tpr, red, turn);
      const float mq = m[0] * inv, m1 = layer ? m[1] * inv : 0.f;
#pragma unroll
      for (int e = 0; e < E; e++) g[e] += r_y * (Cw[e] * dh[e] - yh[e] * mq - m1);
    }
    if (PART == kIn) {
      if (live) store_row<T, W, E>(a.dx, out, L, g);
    } else {
      float p[E], m[2] = {0.f, 0.f};
#pragma unroll
      for (int e = 0; e < E; e++) {
        if (!L.has(e)) g[e] = 0.f;
        S[0][e] += g[e] * f[e];
        S[1][e] += g[e];
        S[4][e] += g[e] * x[e];
        p[e] = A[e] * g[e];
        m[0] += p[e] * f[e];
        m[1] += p[e];
        x[e] = rho[e] * g[e];
      }
      if (live) store_row<T, W, E>(a.dx, out, L, x);
      row_sum<WIDE, 2>(m, tpr, red, turn);
      const float mp = m[0] * inv, m1 = layer ? m[1] * inv : 0.f;
#pragma unroll
      for (int e = 0; e < E; e++) p[e] = r_f * (p[e] - f[e] * mp - m1);
      if (live) store_row<T, W, E>(a.df, out, L, p);
    }
  }

  // the workgroup's sums: rows handled side by side are folded in a fixed order, one sum at a time
  float* dst = P.part + ((size_t)sample * gridDim.x + blockIdx.x) * kSums * C;
  if (PART != kIn && P.rho_part != nullptr) {              // a scalar residual scale: its sum runs over the channels too
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; e++) s += S[4][e];
    s = lanes_sum(s, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) scalar[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < (int)(blockDim.x >> 6); w++) s += scalar[w];
      P.rho_part[sample * gridDim.x + blockIdx.x] = s;
    }
  }
#pragma unroll
  for (int k = 0; k < kSums; k++) {
    if ((PART == kIn && k != 2 && k != 3) || (PART == kOut && (k == 2 || k == 3))) continue;
    if (k == 4 && !a.residual_per_channel) continue;
    if (!WIDE) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < E; e++) fold[e * kThreads + threadIdx.x] = S[k][e];
      __syncthreads();
      for (int i = threadIdx.x; i < tpr * E; i += kThreads) {
        const int e = i / tpr, l = i - e * tpr, c = (e / W) * (tpr * W) + l * W + e % W;
        float s = 0.f;
        for (int r = 0; r < rpw; r++) s += fold[e * kThreads + r * tpr + l];
        if (c < C) dst[(size_t)k * C + c] = s;
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; e++)
        if (L.has(e)) dst[(size_t)k * C + L.ch(e)] = S[k][e];
    }
  }
}

__device__ __forceinline__ bool sum_used(int k, int parts, const gc_block_norm& a) {
  return (k < 2 && parts != kIn) || ((k == 2 || k == 3) && parts != kOut) || (k == 4 && parts != kIn && a.residual_per_channel);
}
// N sums' column c of a sample's partials over its rows: 128 threads per column (8 columns a workgroup: one CU takes 16 cycles for every
// wave's load, so the work has to be spread), every load independent (also of the sums that the parts
// do not have, whose memory is there but was not written: nothing uses those totals)
template <int N>
__device__ __forceinline__ void column_sums(const float* part, int slabs, int C, int c, float (&total)[N], float (*red)[16][8]) {
  const int r0 = threadIdx.x >> 3, lc = threadIdx.x & 7;
  float s[N];
#pragma unroll
  for (int k = 0; k < N; k++) s[k] = 0.f;
  if (c < C) {
#pragma unroll 8
    for (int r = r0; r < slabs; r += 128)
#pragma unroll
      for (int k = 0; k < N; k++) s[k] += part[((size_t)r * kSums + k) * C + c];
  }
#pragma unroll
  for (int k = 0; k < N; k++) {
    s[k] = dpp_add<0x128>(s[k]);                           // the other 8 lanes of 16, the other 16 of 32, the other half
    s[k] = swap_add<true>(swap_add<false>(s[k]));
    if ((threadIdx.x & 63) < 8) red[k][threadIdx.x >> 6][lc] = s[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; k++) {
    total[k] = 0.f;
#pragma unroll
    for (int w = 0; w < 16; w++) total[k] += red[k][w][lc];
  }
}
// the gradient of a scalar residual scale: the workgroups' shares in order
__device__ __forceinline__ void scalar_rho(const gc_block_norm& a, const float* rho_part, int64_t n, float* red, int threads) {
  float s = 0.f;
  for (int64_t i = threadIdx.x; i < n; i += threads) s += rho_part[i];
  s = lanes_sum(s, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < threads / 64; w++) s += red[w];
    a.d_residual_scale[0] = s;
  }
}

// part [batch][slabs][kSums][C] -> sums [batch][kSums][C].  grid (C / 8, kSums, batch), 1024 threads: 8 channels x 128 rows
__global__ __launch_bounds__(1024) void block_norm_sums_kernel(const gc_block_norm a, const float* part, float* sums, int slabs, int parts) {
  const int k = blockIdx.y, C = a.cols;
  if (!sum_used(k, parts, a)) return;
  __shared__ float red[1][16][8];
  const int c = blockIdx.x * 8 + (threadIdx.x & 7);
  const int64_t sample = blockIdx.z;
  float t[1];
  column_sums<1>(part + (sample * slabs * kSums + k) * C, slabs, C, c, t, red);
  if (threadIdx.x < 8 && c < C) sums[(sample * kSums + k) * C + c] = t[0];
}

// One sample (or one run of rows): the sums and the parameters' gradients in one launch.  Blocks of 8 channels x 128 rows; the last
// block: a scalar residual scale.
__global__ __launch_bounds__(1024) void block_norm_finish_kernel(const gc_block_norm a, const float* part, const float* rho_part, int slabs, int parts) {
  __shared__ float red[kSums][16][8];
  const int C = a.cols, c = blockIdx.x * 8 + (threadIdx.x & 7);
  if (blockIdx.x == gridDim.x - 1) {
    if (rho_part != nullptr) scalar_rho(a, rho_part, slabs, &red[0][0][0], 1024);
    return;
  }
  float S[kSums];
  column_sums<kSums>(part, slabs, C, c, S, red);
  if (threadIdx.x >= 8 || c >= C) return;
  if (parts != kIn) {
    const float wo = a.out_weight ? a.out_weight[c] : 1.f, bo = a.out_bias ? a.out_bias[c] : 0.f, g = a.gate ? a.gate[c] : 1.f;
    if (a.d_out_weight) a.d_out_weight[c] = g * S[0];
    if (a.d_out_bias) a.d_out_bias[c] = g * S[1];
    if (a.d_gate) a.d_gate[c] = wo * S[0] + bo * S[1];
    if (a.residual_per_channel && a.d_residual_scale) a.d_residual_scale[c] = S[4];
  }
  if (parts != kOut) {
    const float wi = a.in_weight ? a.in_weight[c] : 1.f, bi = a.in_bias ? a.in_bias[c] : 0.f, m = 1.f + (a.scale ? a.scale[c] : 0.f);
    if (a.d_in_weight) a.d_in_weight[c] = m * S[2];
    if (a.d_in_bias) a.d_in_bias[c] = m * S[3];
    if (a.d_scale) a.d_scale[c] = wi * S[2] + bi * S[3];
    if (a.d_shift) a.d_shift[c] = S[3];
  }
}

// Parameter gradients from the samples' sums.  Blocks 0 .. n - 1: 64 channels x 4 threads each; block n: the gradient of a
// scalar residual scale.
__global__ __launch_bounds__(kThreads) void block_norm_params_kernel(const gc_block_norm a, const float* sums, const float* rho_part, int slabs, int parts) {
  __shared__ float red[5][4][64];
  const int C = a.cols;
  if (blockIdx.x == gridDim.x - 1) {
    if (rho_part != nullptr) scalar_rho(a, rho_part, a.batch * slabs, &red[0][0][0], kThreads);
    return;
  }
  const int lc = threadIdx.x & 63, q = threadIdx.x >> 6, c = blockIdx.x * 64 + lc;
  float acc[5] = {0.f, 0.f, 0.f, 0.f, 0.f};      // out_weight, out_bias, in_weight, in_bias, residual scale
  float shared[3] = {0.f, 0.f, 0.f};              // gate, scale, shift that all samples share
  const float wo = c < C && a.out_weight ? a.out_weight[c] : 1.f, bo = c < C && a.out_bias ? a.out_bias[c] : 0.f;
  const float wi = c < C && a.in_weight ? a.in_weight[c] : 1.f, bi = c < C && a.in_bias ? a.in_bias[c] : 0.f;
  if (c < C)
#pragma unroll 2
    for (int64_t b = q; b < a.batch; b += 4) {
      const float* S = sums + b * kSums * C + c;
      if (parts != kIn) {
        const float g = a.gate ? a.gate[(a.gate_per_sample ? b * C : 0) + c] : 1.f, s0 = S[0], s1 = S[C];
        acc[0] += g * s0;
        acc[1] += g * s1;
        if (a.residual_per_channel) acc[4] += S[4 * C];
        const float dg = wo * s0 + bo * s1;
        if (a.gate_per_sample) { if (a.d_gate) a.d_gate[b * C + c] = dg; }
        else shared[0] += dg;
      }
      if (parts != kOut) {
        const float m = 1.f + (a.scale ? a.scale[(a.mod_per_sample ? b * C : 0) + c] : 0.f), s2 = S[2 * C], s3 = S[3 * C];
        acc[2] += m * s2;
        acc[3] += m * s3;
        const float ds = wi * s2 + bi * s3;
        if (a.mod_per_sample) {
          if (a.d_scale) a.d_scale[b * C + c] = ds;
          if (a.d_shift) a.d_shift[b * C + c] = s3;
        } else { shared[1] += ds; shared[2] += s3; }
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
#pragma unroll
  for (int k = 0; k < 3; k++) red[k][q][lc] = shared[k];
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
  if (d->batch < 0 || d->rows < 0 || d->cols <= 0 || d->cols > kMaxCols || d->batch > 65535) {
    set_error("block norm: 1 <= cols <= %d, 0 <= batch <= 65535, rows >= 0 are supported (got batch=%lld rows=%lld cols=%d)", kMaxCols,
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

// Workgroups per sample: at most `per_cu` per CU in all, so that every workgroup works on several rows (it reads the parameters once,
// and its next rows are under way while it works).
constexpr int kMostPerCu = 8;
int slab_count(int64_t batch, int64_t rows, int tpr, int per_cu) {
  const int64_t rpw = tpr > 64 ? 1 : kThreads / tpr, passes = (rows + rpw - 1) / rpw;
  int64_t s = ((int64_t)device_cu_count() * per_cu + batch - 1) / batch;
  if (s > passes) s = passes;
  return (int)(s < 1 ? 1 : s);
}
int row_threads(int cols) {
  int tpr = 1;
  while (tpr * 8 < cols && tpr < kMaxThreads) tpr *= 2;
  return tpr;
}
// Workgroups of a kernel that a CU holds (asked once per kernel; 72 of them)
int held_per_cu(const void* kernel, int threads) {
  struct Entry { const void* kernel; int threads, n; };
  static std::mutex mu;
  static Entry known[128];
  static int count = 0;
  std::lock_guard<std::mutex> lock(mu);
  for (int i = 0; i < count; i++)
    if (known[i].kernel == kernel && known[i].threads == threads) return known[i].n;
  int n = 0;
  if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, 0) != hipSuccess || n < 1) n = 2;
  if (n > kMostPerCu) n = kMostPerCu;
  if (count < 128) known[count++] = Entry{kernel, threads, n};
  return n;
}

NormParams make_params(const gc_block_norm* d) {
  NormParams P{};
  P.a = *d;
  P.tpr = row_threads(d->cols);
  auto fits = [&](int unit) {                              // accesses of `unit` elements
    const uintptr_t mask = (d->dtype == GC_F32 ? 4 : 2) * unit - 1;
    const void* all[] = {d->x, d->f, d->y, d->h, d->dy, d->dh, d->dx, d->df};
    for (const void* p : all)
      if (reinterpret_cast<uintptr_t>(p) & mask) return false;
    return d->cols % unit == 0 && d->x_row_stride % unit == 0 && d->x_batch_stride % unit == 0 && d->f_row_stride % unit == 0 && d->f_batch_stride % unit == 0;
  };
  P.width = d->dtype == GC_F32 ? (fits(4) ? 4 : 1) : (fits(8) ? 8 : 2);
  return P;
}

typedef void (*NormKernel)(const NormParams);
template <typename T, int MAXT, int W, int E>
NormKernel kernel_for(int parts, bool bwd) {
  if (bwd)
    return parts == kIn ? block_norm_bwd_kernel<T, MAXT, kIn, W, E>
                        : (parts == kOut ? block_norm_bwd_kernel<T, MAXT, kOut, W, E> : block_norm_bwd_kernel<T, MAXT, kBoth, W, E>);
  return parts == kIn ? block_norm_fwd_kernel<T, MAXT, kIn, W, E>
                      : (parts == kOut ? block_norm_fwd_kernel<T, MAXT, kOut, W, E> : block_norm_fwd_kernel<T, MAXT, kBoth, W, E>);
}
template <typename T, int W>
NormKernel kernel_width(int cols, int tpr, int parts, bool bwd) {
  if (tpr <= 64) return kernel_for<T, kThreads, W, 8>(parts, bwd);
  return cols <= 8 * kMaxThreads ? kernel_for<T, kMaxThreads, W, 8>(parts, bwd) : kernel_for<T, kMaxThreads, W, 16>(parts, bwd);
}
// Launches the kernel for P (whose slabs it sets)
int launch(NormParams& P, int parts, bool bwd, hipStream_t s) {
  NormKernel k;
  const int C = P.a.cols;
  if (P.a.dtype == GC_F32) k = P.width == 4 ? kernel_width<float, 4>(C, P.tpr, parts, bwd) : kernel_width<float, 1>(C, P.tpr, parts, bwd);
  else k = P.width == 8 ? kernel_width<uint16_t, 8>(C, P.tpr, parts, bwd) : kernel_width<uint16_t, 2>(C, P.tpr, parts, bwd);
  const int threads = P.tpr > 64 ? P.tpr : kThreads;
  P.slabs = slab_count(P.a.batch, P.a.rows, P.tpr, held_per_cu(reinterpret_cast<const void*>(k), threads));
  hipLaunchKernelGGL(k, dim3(P.slabs, (unsigned)P.a.batch), dim3(threads), 0, s, P);
  return check_hip(hipGetLastError(), bwd ? "block_norm bwd launch" : "block_norm fwd launch");
}

}  // namespace
}  // namespace gc

using namespace gc;

extern "C" int gc_block_norm_fwd(const gc_block_norm* desc, void* stream) {
  int parts = 0;
  if (int e = check_desc(desc, false, parts)) return e;
  if (desc->batch == 0 || desc->rows == 0) return GC_OK;
  NormParams P = make_params(desc);
  hipStream_t s = (hipStream_t)stream;
  ProfScope ps("gc::block_norm_fwd_kernel", 0.0, s);
  return launch(P, parts, false, s);
}

// floats: the samples' sums, the scalar residual scale's shares, the workgroups' sums
extern "C" size_t gc_block_norm_workspace_bytes(int64_t batch, int64_t rows, int32_t cols) {
  if (batch <= 0 || rows <= 0 || cols <= 0) return 0;
  const size_t wgs = (size_t)batch * slab_count(batch, rows, row_threads(cols), kMostPerCu);
  return ((size_t)batch * kSums * cols + (wgs + 3) / 4 * 4 + wgs * kSums * cols) * sizeof(float);
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
  NormParams P = make_params(desc);
  const size_t wgs = (size_t)desc->batch * slab_count(desc->batch, desc->rows, P.tpr, kMostPerCu);
  float* sums = static_cast<float*>(workspace);
  const bool scalar = parts != kIn && desc->d_residual_scale != nullptr && !desc->residual_per_channel;
  P.rho_part = scalar ? sums + (size_t)desc->batch * kSums * desc->cols : nullptr;
  P.part = sums + (size_t)desc->batch * kSums * desc->cols + (wgs + 3) / 4 * 4;
  hipStream_t s = (hipStream_t)stream;
  {
    ProfScope ps("gc::block_norm_bwd_kernel", 0.0, s);
    if (int e = launch(P, parts, true, s)) return e;
  }
  if (desc->batch == 1) {
    hipLaunchKernelGGL(block_norm_finish_kernel, dim3((desc->cols + 7) / 8 + 1), dim3(1024), 0, s, *desc, (const float*)P.part, (const float*)P.rho_part,
                       P.slabs, parts);
    return check_hip(hipGetLastError(), "block_norm finish launch");
  }
  const float* totals = P.part;
  if (P.slabs > 1) {
    hipLaunchKernelGGL(block_norm_sums_kernel, dim3((desc->cols + 7) / 8, kSums, (unsigned)desc->batch), dim3(1024), 0, s, *desc, (const float*)P.part,
                       sums, P.slabs, parts);
    if (check_hip(hipGetLastError(), "block_norm sums launch")) return GC_HIP_ERROR;
    totals = sums;
  }
  hipLaunchKernelGGL(block_norm_params_kernel, dim3((desc->cols + 63) / 64 + 1), dim3(kThreads), 0, s, *desc, totals, (const float*)P.rho_part, P.slabs, parts);
  return check_hip(hipGetLastError(), "block_norm params launch");
}
