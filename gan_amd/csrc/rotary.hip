// Rotary positions with several axes (time, height, width): pair p of a head, which belongs to axis a(p) with frequency
// w(p), turns by the angle position_a * w(p):
//
//   (u, v) -> (u cos - v sin, u sin + v cos)        backward: the same with the angle negated (a rotation's adjoint)
//
// Pairs are neighbours (2p, 2p + 1) or halves (p, P + p); elements behind the P pairs pass through.  q and k of a layer go
// in one launch, since they share positions.
//
// Bound by HBM (each tensor read and written once) as long as the angles are cheap: a workgroup owns a run of tokens, works
// out cos and sin of their P pairs once into LDS and then streams all heads (and, where the samples share positions, several
// samples) of those tokens with 16-byte accesses.  An angle is formed in turns (w / 2 pi per unit of position, fp64), its
// whole turns dropped in fp64, and only the fraction is rounded to fp32: a position of a million in the fastest pair would
// otherwise lose 17 of 24 bits.  64 x 4096 tokens, 8 heads of 32 fp32: 114 us (4.7 TB/s; a large copy reaches 4.9), of bf16 44; 2 x 16384
// tokens, 40 heads of 128 bf16, positions of their own: 141 (4.75 TB/s).  Element by element, where 16-byte accesses do not fit: 159 and 62.
#include "common.h"

namespace gc {
namespace {

constexpr int kMaxPairs = 256;
constexpr int kTableBytes = 32768;         // cos / sin of tokens x pairs, at most

struct RotaryParams {
  gc_rotary a;
  int tokens;                              // per workgroup
  int samples;                             // per workgroup (1 unless the samples share positions)
  FastDiv units_row, units_head;           // work items per token (all heads) and per head
  int q_units;                             // work items of a token that belong to q
};

template <typename T> __device__ __forceinline__ float get1(const void* p, int64_t i) {
  if constexpr (sizeof(T) == 4) return static_cast<const float*>(p)[i];
  else return bf16_bits_to_float(static_cast<const uint16_t*>(p)[i]);
}
template <typename T> __device__ __forceinline__ void put1(void* p, int64_t i, float v) {
  if constexpr (sizeof(T) == 4) static_cast<float*>(p)[i] = v;
  else static_cast<uint16_t*>(p)[i] = float_to_bf16_bits(v);
}
// 16 bytes: W = 4 (fp32) or 8 (bf16) elements
template <typename T> struct Vec { static constexpr int W = 16 / sizeof(T); u32x4 q; };
template <typename T> __device__ __forceinline__ Vec<T> get(const void* p, int64_t i) {
  return Vec<T>{*reinterpret_cast<const u32x4*>(static_cast<const T*>(p) + i)};
}
template <typename T> __device__ __forceinline__ void widen(const Vec<T>& v, float (&f)[Vec<T>::W]) {
#pragma unroll
  for (int e = 0; e < Vec<T>::W; e++) {
    if constexpr (sizeof(T) == 4) { const uint32_t u = v.q[e]; f[e] = __builtin_bit_cast(float, u); }
    else f[e] = __builtin_bit_cast(float, (e & 1) ? (v.q[e / 2] & 0xffff0000u) : (v.q[e / 2] << 16));
  }
}
template <typename T> __device__ __forceinline__ void put(void* p, int64_t i, const float (&v)[Vec<T>::W]) {
  T* d = static_cast<T*>(p) + i;
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<f32x4*>(d) = f32x4{v[0], v[1], v[2], v[3]};
  } else {
    const u32x2 lo = cvt_bf16x4(f32x4{v[0], v[1], v[2], v[3]}), hi = cvt_bf16x4(f32x4{v[4], v[5], v[6], v[7]});
    *reinterpret_cast<u32x4*>(d) = u32x4{lo[0], lo[1], hi[0], hi[1]};
  }
}

__device__ __forceinline__ double position_at(const gc_rotary& a, int64_t i) {
  switch (a.position_dtype) {
    case GC_POS_I32: return (double)static_cast<const int32_t*>(a.positions)[i];
    case GC_POS_I64: return (double)static_cast<const int64_t*>(a.positions)[i];
    case GC_POS_F32: return (double)static_cast<const float*>(a.positions)[i];
    default: return static_cast<const double*>(a.positions)[i];
  }
}

// A work item of a head: VEC: 16 bytes of neighbouring elements (NEIGHBOURS), or 16 bytes of the first half and their partners, then
// 16-byte runs that pass through; otherwise one pair, then single elements that pass through.
template <typename T, bool VEC, bool NEIGHBOURS>
__global__ __launch_bounds__(kThreads) void rotary_kernel(const RotaryParams P) {
  extern __shared__ float2 table[];                        // [token][pair]: cos, sin
  constexpr int W = Vec<T>::W;
  const gc_rotary& a = P.a;
  const int np = a.pairs;
  const int64_t n0 = (int64_t)blockIdx.x * P.tokens;
  const int nt = (int)(a.tokens - n0 < P.tokens ? a.tokens - n0 : P.tokens);
  const int64_t b0 = (int64_t)blockIdx.y * P.samples;
  const int nb = (int)(a.batch - b0 < P.samples ? a.batch - b0 : P.samples);
  const float sign = a.inverse ? -1.f : 1.f;
  for (int i = threadIdx.x; i < nt * np; i += kThreads) {
    const int t = i / np, p = i - t * np;
    const int64_t row = (a.positions_per_sample ? b0 * a.tokens : 0) + n0 + t;
    const double turns = position_at(a, row * a.axes + a.pair_axis[p]) * a.pair_turns[p];
    float s, c;
    sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
    table[i] = make_float2(c, sign * s);
  }
  __syncthreads();

  const int units = (int)P.units_row.d, per_head = (int)P.units_head.d;
  const int turn_units = VEC ? np * (NEIGHBOURS ? 2 : 1) / W : np;
  const int items = nt * units;
  for (int i = threadIdx.x; i < items; i += kThreads) {
    const int t = (int)fd_div((uint32_t)i, P.units_row);
    int u = i - t * units;
    const bool is_q = u < P.q_units;
    if (!is_q) u -= P.q_units;
    const int head = (int)fd_div((uint32_t)u, P.units_head), c = u - head * per_head;
    const int64_t n = n0 + t;
    const void* src = is_q ? a.q : a.k;
    void* dst = is_q ? a.q_out : a.k_out;
    const int64_t* st = is_q ? a.q_stride : a.k_stride;
    const int heads = is_q ? a.q_heads : a.k_heads;
    const int64_t out_step = a.tokens * heads * a.dim, in_step = st[0];
    int64_t in = b0 * in_step + n * st[1] + head * st[2], out = b0 * out_step + (n * heads + head) * a.dim;
    const float2* cs = table + t * np;
    if (VEC) {
      const bool turned = c < turn_units;
      const int x0 = turned ? c * W : 2 * np + (c - turn_units) * W, y0 = NEIGHBOURS || !turned ? x0 : np + x0;
      // all samples of this item: the next sample's elements are asked for before this one's are turned
      Vec<T> vx = get<T>(src, in + x0), vy;
      if (!NEIGHBOURS) vy = get<T>(src, in + y0);
      for (int b = 0; b < nb; b++, in += in_step, out += out_step) {
        float x[W], y[W];
        widen<T>(vx, x);
        widen<T>(NEIGHBOURS ? vx : vy, y);
        if (b + 1 < nb) {
          vx = get<T>(src, in + in_step + x0);
          if (!NEIGHBOURS) vy = get<T>(src, in + in_step + y0);
        }
        if (turned) {
          if (NEIGHBOURS) {
#pragma unroll
            for (int e = 0; e < W / 2; e++) {
              const float2 z = cs[c * (W / 2) + e];
              y[2 * e] = x[2 * e] * z.x - x[2 * e + 1] * z.y;
              y[2 * e + 1] = x[2 * e] * z.y + x[2 * e + 1] * z.x;
            }
          } else {
#pragma unroll
            for (int e = 0; e < W; e++) {
              const float2 z = cs[c * W + e];
              const float r = x[e] * z.x - y[e] * z.y;
              y[e] = x[e] * z.y + y[e] * z.x;
              x[e] = r;
            }
            put<T>(dst, out + x0, x);
          }
        }
        put<T>(dst, out + y0, y);
      }
    } else {
      for (int b = 0; b < nb; b++, in += in_step, out += out_step) {
        if (c < turn_units) {
          const int i0 = NEIGHBOURS ? 2 * c : c, i1 = NEIGHBOURS ? 2 * c + 1 : np + c;
          const float x = get1<T>(src, in + i0), y = get1<T>(src, in + i1);
          const float2 z = cs[c];
          put1<T>(dst, out + i0, x * z.x - y * z.y);
          put1<T>(dst, out + i1, x * z.y + y * z.x);
        } else {
          const int64_t o = 2 * np + (c - turn_units);
          put1<T>(dst, out + o, get1<T>(src, in + o));
        }
      }
    }
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace gc

using namespace gc;

extern "C" int gc_axial_rotary(const gc_rotary* d, void* stream) {
  if (d == nullptr || d->q == nullptr || d->q_out == nullptr || d->positions == nullptr || d->pair_turns == nullptr || d->pair_axis == nullptr ||
      (d->k_heads > 0 && (d->k == nullptr || d->k_out == nullptr))) {
    set_error("axial rotary: a pointer is null");
    return GC_BAD_ARGUMENT;
  }
  if (d->dtype != GC_F32 && d->dtype != GC_BF16) { set_error("axial rotary: dtype must be GC_F32 or GC_BF16"); return GC_BAD_ARGUMENT; }
  if (d->position_dtype < GC_POS_I32 || d->position_dtype > GC_POS_F64) { set_error("axial rotary: unknown position type %d", d->position_dtype); return GC_BAD_ARGUMENT; }
  if (d->batch < 0 || d->tokens < 0 || d->q_heads <= 0 || d->k_heads < 0 || d->axes <= 0 || d->pairs <= 0 || d->pairs > kMaxPairs ||
      2 * d->pairs > d->dim || d->dim > 4096 || (int64_t)d->q_heads + d->k_heads > 4096 || d->batch > 65535) {
    set_error("axial rotary: supported are 1 to %d pairs with 2 * pairs <= dim <= 4096, up to 4096 heads, batch <= 65535 (got pairs=%d dim=%d heads=%d+%d batch=%lld)",
              kMaxPairs, d->pairs, d->dim, d->q_heads, d->k_heads, (long long)d->batch);
    return GC_UNSUPPORTED_GEOMETRY;
  }
  if (d->batch == 0 || d->tokens == 0) return GC_OK;
  const int W = d->dtype == GC_F32 ? 4 : 8;
  bool vec = d->dim % W == 0 && d->pairs % (d->halves ? W : W / 2) == 0 && aligned16(d->q) && aligned16(d->k) && aligned16(d->q_out) && aligned16(d->k_out);
  for (int i = 0; i < 3; i++) vec = vec && d->q_stride[i] % W == 0 && (d->k_heads == 0 || d->k_stride[i] % W == 0);
  RotaryParams P{};
  P.a = *d;
  const int rest = d->dim - 2 * d->pairs;
  const int per_head = vec ? (d->halves ? d->pairs : 2 * d->pairs) / W + rest / W : d->pairs + rest;
  const int heads = d->q_heads + d->k_heads;
  P.units_head = make_fastdiv((uint32_t)per_head);
  P.units_row = make_fastdiv((uint32_t)(per_head * heads));
  P.q_units = per_head * d->q_heads;
  // tokens per workgroup: what the LDS table holds, but no more than leaves 8 workgroups per CU, and enough for every thread
  const int64_t cus = device_cu_count();
  int64_t most = kTableBytes / (8 * d->pairs);
  const int64_t fill = (d->tokens * d->batch + cus * 8 - 1) / (cus * 8);
  int64_t tok = most < 16 ? most : 16;
  if (d->positions_per_sample == 0) {
    // shared positions: one table serves several samples, as far as the grid still fills the chip
    while (tok > 1 && ((d->tokens + tok - 1) / tok) * d->batch < cus * 8) tok >>= 1;
    int64_t s = ((d->tokens + tok - 1) / tok) * d->batch / (cus * 8);
    P.samples = (int)(s < 1 ? 1 : (s > d->batch ? d->batch : (s > 8 ? 8 : s)));
  } else {
    if (tok > fill) tok = fill < 1 ? 1 : fill;
    P.samples = 1;
  }
  P.tokens = (int)tok;
  const int64_t gx = (d->tokens + tok - 1) / tok;
  if (gx >= (1ll << 31)) { set_error("axial rotary: too many tokens (%lld)", (long long)d->tokens); return GC_UNSUPPORTED_GEOMETRY; }
  const dim3 grid((unsigned)gx, (unsigned)((d->batch + P.samples - 1) / P.samples));
  const size_t lds = (size_t)P.tokens * d->pairs * sizeof(float2);
  hipStream_t s = (hipStream_t)stream;
  ProfScope ps("gc::rotary_kernel", 0.0, s);
#define GC_ROTARY(T)                                                                                                          \
  do {                                                                                                                        \
    if (vec) {                                                                                                                \
      if (d->halves) hipLaunchKernelGGL((rotary_kernel<T, true, false>), grid, dim3(kThreads), lds, s, P);                    \
      else hipLaunchKernelGGL((rotary_kernel<T, true, true>), grid, dim3(kThreads), lds, s, P);                               \
    } else {                                                                                                                  \
      if (d->halves) hipLaunchKernelGGL((rotary_kernel<T, false, false>), grid, dim3(kThreads), lds, s, P);                   \
      else hipLaunchKernelGGL((rotary_kernel<T, false, true>), grid, dim3(kThreads), lds, s, P);                              \
    }                                                                                                                         \
  } while (0)
  if (d->dtype == GC_F32) GC_ROTARY(float);
  else GC_ROTARY(uint16_t);
#undef GC_ROTARY
  return check_hip(hipGetLastError(), "rotary launch");
}
