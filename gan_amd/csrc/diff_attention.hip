// Differential attention: the difference of two softmax maps over the same values,
//
//   out_i = sum_j (p1_ij - lam p2_ij) v_j,      pm_ij = exp(scale <q_m,i , k_m,j>) / sum_j' exp(..)      (visible keys j)
//
// with one lam per head.  Nothing of size rows x keys is stored.
//
// Forward: one pass over the keys with a running maximum and sum per map and two accumulators (the maps' denominators are known
// only at the end), which share every value fragment read from LDS: per pair of positions 4 d + 4 dv multiply-adds of which the
// definition needs 4 d + 2 dv.  Scores are computed TRANSPOSED, S^T = K Q^T on 32x32x16 matrix instructions, so that a lane holds
// one softmax row i = lane % 32 at keys j = 8 (r / 4) + 4 h + r % 4 (h = lane / 32).  Taking the reduction index of the second
// product in the order in which those accumulators lie (slot (h, e) of k-step t  <->  j = 16 t + 8 (e / 4) + 4 h + e % 4), the
// exponentiated scores are its B operand P^T without a trip through LDS, and V^T in that order is what two transposing LDS reads
// return.  The running maximum moves only when an exponential would exceed 2^8 (the sums are fp32 and keep their precision).
//
// Backward from the saved log2-sums L_m (P recomputed, dP = dO V^T shared by both maps, delta_m,i = dO_i . O_m,i):
//   dV_j = sum_i (p1 - lam p2)_ij dO_i     dS1 = P1 (dP - delta1)     dS2 = -lam P2 (dP - delta2)     dQm = dSm Km, dKm = dSm^T Qm
//   dlam = -sum_i (delta2_i + sum_j p2_ij (dP_ij - delta2_i)):  the second term vanishes but for the rounding of the stored O, which
//   it takes out of the sum (an fp32 gradient that is not held to the bf16 rounding of O)
// in two kernels that own the rows of their outputs (dkv: 128 keys of a key head, summed over the query heads that share them;
// dq: 128 queries of a head): no atomics, results reproduce.
//
// Tiles of 64 rows go from HBM to LDS directly (16 bytes per lane), two stages in turn; the 16-byte chunks of a row are permuted on
// the SOURCE side so that both the row-wise and the transposing reads spread over the banks.  Rows past the end, and the columns
// between d and its padded width, are answered with zeros by the buffer's range check, so nothing behind a sample's length is read.
// Probabilities and score gradients are rounded to bf16 for the second products (the operands' own type; 2^-9 each, independent),
// everything else is fp32.
#include <algorithm>

#include "common.h"

namespace gc {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4_ptr;

constexpr int kRows = 128;                       // rows of a workgroup: 32 per wave
constexpr int kBlk = 64;                         // rows staged per step
constexpr uint32_t kOutOfRange = 0x80000000u;
constexpr float kLazy = 8.f;                     // log2 units by which a score may exceed the running maximum
constexpr float kLazyExp = 256.f;                // 2^kLazy
constexpr float kLargeScore = 1048576.f;         // log2 units

struct DiffParams {
  gc_diff_attention a;
  int G, tiles, nsplit, blocks_per_split, few;     // few: at most 32 rows per key head (diff_few_rows_kernel; shares in tiles of 32 keys)
  FastDiv div_nq;
  float c2, lazy;                                // scale * log2(e); kLazy in units of a score
  float *part, *ml, *delta, *rows4, *lampart;
};

__device__ __forceinline__ bf16x8 zero8() { return __builtin_bit_cast(bf16x8, u32x4{0u, 0u, 0u, 0u}); }
__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int r = 0; r < 16; r++) z[r] = 0.f;
  return z;
}
__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ bf16x8 pack8(const f32x16& v, int r0) {
  const u32x2 lo = cvt_bf16x4(f32x4{v[r0], v[r0 + 1], v[r0 + 2], v[r0 + 3]}), hi = cvt_bf16x4(f32x4{v[r0 + 4], v[r0 + 5], v[r0 + 6], v[r0 + 7]});
  return __builtin_bit_cast(bf16x8, u32x4{lo[0], lo[1], hi[0], hi[1]});
}
__device__ __forceinline__ bf16x8 pack8_sum(const f32x16& u, const f32x16& v, float f, int r0) {
  f32x4 a, b;
#pragma unroll
  for (int x = 0; x < 4; x++) {
    a[x] = u[r0 + x] + f * v[r0 + x];
    b[x] = u[r0 + 4 + x] + f * v[r0 + 4 + x];
  }
  const u32x2 lo = cvt_bf16x4(a), hi = cvt_bf16x4(b);
  return __builtin_bit_cast(bf16x8, u32x4{lo[0], lo[1], hi[0], hi[1]});
}
// The two half-waves' values of a row, in both (v_permlane32_swap: one result holds the lower half's value, the other the upper's).
// The results are copied to scalars first: a bit cast of a vector's element itself reads element 0.
__device__ __forceinline__ void both_halves(float v, float& lo, float& hi) {
  typedef unsigned int u32pair __attribute__((ext_vector_type(2)));
  const unsigned int u = __builtin_bit_cast(unsigned int, v);
  const u32pair r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const unsigned int a = r[0], b = r[1];
  lo = __builtin_bit_cast(float, a);
  hi = __builtin_bit_cast(float, b);
}
__device__ __forceinline__ float half_max(float v) {
  float a, b;
  both_halves(v, a, b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float half_sum(float v) {
  float a, b;
  both_halves(v, a, b);
  return a + b;
}

// Chunk permutations of a tile row of ROWB bytes (64 banks of 4 bytes: rows closer than 256 / ROWB apart never collide), by how the
// tile is read: row-wise (16 rows at one chunk), transposed (4 rows x 4 chunks), or both ways.  Transposed reads of a tile that is
// only read so depend on two bits of the row, which leaves their addresses to immediate offsets.
enum Use { kRowWise, kTransposed, kBothWays };
template <int ROWB, Use U>
__device__ __forceinline__ int swz(int row) {
  if (U == kRowWise) return ROWB == 64 ? (row >> 2) & 3 : (ROWB == 128 ? (row >> 1) & 7 : row & 15);
  if (U == kTransposed) return ROWB == 64 ? 0 : (ROWB == 128 ? ((row >> 1) & 1) << 2 : (row & 3) << 2);
  return ROWB == 64 ? (row >> 2) & 3 : (ROWB == 128 ? (((row >> 1) & 1) << 2) | ((row >> 2) & 3) : ((row & 3) << 2) | ((row >> 2) & 3));
}

// Every load into LDS that this wave issued has landed, then the workgroup meets: the staged tile is complete and the other stage
// is no longer read.  (A workgroup barrier alone does not wait for loads that are counted as vector memory.)
__device__ __forceinline__ void tile_ready() {
  __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8));        // vmcnt(0)
  __syncthreads();
}

// 16 (or 4) bytes per lane from a buffer straight into LDS at `lds` + 16 (4) * lane.  Written in assembly because the compiler, which
// cannot tell the stages apart, would wait for every such load in front of the next transposing LDS read.  No register receives
// data; tile_ready() waits for the loads.
typedef uint32_t u32x4s __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void load_to_lds16(u32x4s rsrc, uint32_t voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(voff), "s"(rsrc) : "memory", "m0");
}
__device__ __forceinline__ void load_to_lds4(u32x4s rsrc, uint32_t voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(lds), "v"(voff), "s"(rsrc) : "memory", "m0");
}
// Raw buffer of `bytes` bytes at p (uniform): loads at or past its end return zeros
__device__ __forceinline__ u32x4s buffer_at(const void* p, uint32_t bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(p);
  return u32x4s{(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a), (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(a >> 32) & 0xffffu)),
                (uint32_t)__builtin_amdgcn_readfirstlane((int)bytes), 0x00020000u};
}

template <int N>
__device__ __forceinline__ void wait_loads() {             // all but the N youngest loads of this wave have landed
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}

// One tile of ROWS rows of `width` elements (padded to ROWB / 2 columns), from a tensor with row stride `stride` bytes.
template <int ROWB, Use U, int ROWS = kBlk, int NW = kThreads / 64>
struct Loader {
  // a wave's instructions repeat their chunk permutation every 16 rows: BASES of them differ
  static constexpr int CPR = ROWB / 16, RPI = 64 / CPR, NI = ROWS * ROWB / (1024 * NW), BASES = RPI * NW >= 16 ? 1 : 16 / (RPI * NW);
  static_assert(NI >= 1 && NI % BASES == 0, "every wave loads whole periods of a tile");
  uint32_t voff[BASES];
  uint32_t step;
  int wave;
  __device__ __forceinline__ void init(int wave_, int lane, uint32_t stride, int width) {
    wave = wave_;
#pragma unroll
    for (int b = 0; b < BASES; b++) {
      const int row = (wave + NW * b) * RPI + lane / CPR, chunk = (lane % CPR) ^ swz<ROWB, U>(row);
      voff[b] = chunk * 8 < width ? (uint32_t)row * stride + chunk * 16 : kOutOfRange;
    }
    step = NW * RPI * stride;                              // bytes between a wave's consecutive instructions
  }
  // ROWS rows at p, of which the first `left` (possibly none or fewer) exist, to LDS at `lds`.  The instructions' row offsets go into the
  // (scalar) buffer base, so that one offset register serves all of them.
  __device__ __forceinline__ void load(const char* p, int left, uint32_t stride, int width, uint32_t lds) const {
    const int n_rows = left < ROWS ? left : ROWS;
    const uint32_t bytes = n_rows > 0 ? (uint32_t)(n_rows - 1) * stride + width * 2 : 0u;
#pragma unroll
    for (int n = 0; n < NI; n += BASES) {
      const uint32_t skip = (uint32_t)n * step;
      const u32x4s rs = buffer_at(p + skip, (uint32_t)max((int)bytes - (int)skip, 0));
#pragma unroll
      for (int b = 0; b < BASES; b++) load_to_lds16(rs, voff[b], lds + (wave + NW * (n + b)) * 1024);
    }
  }
};
// The same for tiles of kBlk rows that follow each other, fetched piece by piece in few scalar instructions: one descriptor, moved on by
// a tile, and an offset register for every piece.
template <int ROWB, Use U, int NW>
struct TileStream {
  static constexpr int CPR = ROWB / 16, RPI = 64 / CPR, NI = kBlk * ROWB / (1024 * NW);
  static_assert(NI >= 1, "every wave loads a part of a tile");
  uint32_t voff[NI], stride, full, last, bytes;            // bytes of a whole tile, of a row, of what is there of this tile
  const char* p;
  int left;
  __device__ __forceinline__ void init(int wave, int lane, const char* first, int rows, uint32_t stride_, int width) {
    stride = stride_;
    last = width * 2;
    full = (kBlk - 1) * stride + last;
    p = first;
    left = rows;
    measure();
#pragma unroll
    for (int n = 0; n < NI; n++) {
      const int row = (wave + NW * n) * RPI + lane / CPR, chunk = (lane % CPR) ^ swz<ROWB, U>(row);
      voff[n] = chunk * 8 < width ? (uint32_t)row * stride + chunk * 16 : kOutOfRange;
    }
  }
  // piece n of the tile to LDS at `lds`; rows that do not exist (possibly all) are answered with zeros
  __device__ __forceinline__ void piece(int n, int wave, uint32_t lds) const {
    load_to_lds16(buffer_at(p, bytes), voff[n], lds + (wave + NW * n) * 1024);
  }
  __device__ __forceinline__ void next() {
    p += kBlk * stride;
    left -= kBlk;
    measure();
  }
  __device__ __forceinline__ void measure() {
    bytes = full;
    if (left < kBlk) bytes = left > 0 ? (uint32_t)(left - 1) * stride + last : 0u;
  }
};
// Keys and values of one key head, staged tile after tile: running (scalar) addresses instead of products per tile.
template <int KROW, int VROW, Use KU, Use VU, int ROWS, int NW>
struct KeyTiles {
  Loader<KROW, KU, ROWS, NW> lk;
  Loader<VROW, VU, ROWS, NW> lv;
  const char *k0, *k1, *v;
  uint32_t kst, vst;
  int left, d, dv;
  __device__ __forceinline__ void init(const gc_diff_attention& a, int b, int hk, int row, int len, int wave, int lane) {
    kst = (uint32_t)(a.k_stride[1] * 2);
    vst = (uint32_t)(a.v_stride[1] * 2);
    d = a.d;
    dv = a.dv;
    lk.init(wave, lane, kst, d);
    lv.init(wave, lane, vst, dv);
    k0 = reinterpret_cast<const char*>(static_cast<const uint16_t*>(a.k) + b * a.k_stride[0] + hk * a.k_stride[2]) + row * (int64_t)kst;
    k1 = k0 + a.k_stride[3] * 2;
    v = reinterpret_cast<const char*>(static_cast<const uint16_t*>(a.v) + b * a.v_stride[0] + hk * a.v_stride[2]) + row * (int64_t)vst;
    left = len - row;
  }
  // the next tile's two maps of keys and its values, one behind the other
  __device__ __forceinline__ void next(uint32_t lds) {
    lk.load(k0, left, kst, d, lds);
    lk.load(k1, left, kst, d, lds + ROWS * KROW);
    lv.load(v, left, vst, dv, lds + 2 * ROWS * KROW);
    k0 += ROWS * kst;
    k1 += ROWS * kst;
    v += ROWS * vst;
    left -= ROWS;
  }
};

typedef __attribute__((address_space(3))) const bf16x8* lds_bf16x8_ptr;
__device__ __forceinline__ uint32_t lds_offset(const char* p) { return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p; }
__device__ __forceinline__ bf16x8 read_row(uint32_t addr) { return *(lds_bf16x8_ptr)(uintptr_t)addr; }
__device__ __forceinline__ bf16x8 read_col(uint32_t lo_addr, uint32_t hi_addr) {
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(uintptr_t)lo_addr);
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(uintptr_t)hi_addr);
  typedef short s16x8 __attribute__((ext_vector_type(8)));
  const s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  return __builtin_bit_cast(bf16x8, v);
}
// Address of this lane's chunk in row lane % 32 of a tile for k-step 0; k-step ks is at address ^ (ks << 5)
template <int ROWB, Use U>
__device__ __forceinline__ uint32_t row_addr(int lane) {
  const int row = lane & 31, h = lane >> 5;
  return row * ROWB + ((h ^ swz<ROWB, U>(row)) << 4);
}
// Address of this lane's 8 bytes of a transposing read of rows row0 .. row0 + 7 (4 per half-wave), columns 0 .. 31; column block cb is
// at address ^ (cb << 6), the rows 8 further on at the same offset + 8 rows (read both ways: at that, with bit 5 flipped)
template <int ROWB, Use U>
__device__ __forceinline__ uint32_t col_addr(int lane, int row0) {
  const int h = lane >> 5, rr = row0 + 4 * h + ((lane >> 2) & 3), chunk = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
  return rr * ROWB + ((chunk ^ swz<ROWB, U>(rr)) << 4) + (lane & 1) * 8;
}
template <int ROWB>
__device__ __forceinline__ bf16x8 read_col_both(uint32_t lo_addr) { return read_col(lo_addr, (lo_addr ^ 32) + 8 * ROWB); }
// 8 elements of a global row as a B operand; zero past the row's width
__device__ __forceinline__ bf16x8 global_frag(const uint16_t* row, bool valid, int col, int width) {
  if (!valid || col >= width) return zero8();
  return __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(row + col));
}

// Makes the compiler have operands ready here.  Otherwise it waits for them where they are first used, in every round of a loop,
// and for all loads, among them those into LDS that are meant to stay in flight.
template <int M, int N>
__device__ __forceinline__ void arrived(bf16x8 (&v)[M][N]) {
#pragma unroll
  for (int m = 0; m < M; m++)
#pragma unroll
    for (int n = 0; n < N; n++) {
      u32x4 u = __builtin_bit_cast(u32x4, v[m][n]);
      asm volatile("" : "+v"(u));
      v[m][n] = __builtin_bit_cast(bf16x8, u);
    }
}

__device__ __forceinline__ int sample_length(const gc_diff_attention& a, int b) {
  if (a.key_lengths == nullptr) return a.NK;
  const int n = a.key_lengths[b];
  return n < 0 ? 0 : (n > a.NK ? a.NK : n);
}
// number of visible keys of query i (possibly <= 0)
__device__ __forceinline__ int visible(const gc_diff_attention& a, int i, int len) {
  const int n = i + 1 + len - a.NQ;
  return a.causal ? (n < 0 ? 0 : (n < len ? n : len)) : len;
}

// Which (sample and head, tile, share) a workgroup owns.  Workgroup n runs on XCD n % 8, each with an L2 of its own: an XCD gets a
// contiguous run of the work, so that the workgroups that walk one head's keys (queries) at the same time meet in one L2.  Causal
// tiles differ in length.  `runs` runs of tiles from short to long (the heads of a group) follow each other in a head's tiles, or, with
// runs = 0, one run from long to short.  Where every XCD gets whole runs, they go one after the other, long tiles first; otherwise the
// longest tiles of all heads start first on all XCDs (16 heads, 4 key heads, N 8192: 455 against 508 us forward).
struct WorkId { int bh, tile, share; };
__device__ __forceinline__ WorkId work_id(const DiffParams& P, uint32_t heads, uint32_t runs) {
  const uint32_t n = P.nsplit, T = P.tiles;
  if (!P.a.causal) {
    const uint32_t lid = xcd_remap(blockIdx.x, gridDim.x);
    return WorkId{(int)(lid / n / T), (int)(lid / n % T), (int)(lid % n)};
  }
  if (runs == 0) return WorkId{(int)(blockIdx.x % (heads * n) / n), (int)(blockIdx.x / (heads * n)), (int)(blockIdx.x % n)};
  if (T % runs != 0) runs = 1;
  const uint32_t per = T / runs;
  if (heads * runs % 8 == 0) {
    const uint32_t lid = xcd_remap(blockIdx.x, gridDim.x), t = lid / n % T;
    return WorkId{(int)(lid / n / T), (int)(t - t % per + per - 1 - t % per), (int)(lid % n)};
  }
  const uint32_t in = blockIdx.x % (heads * n), t = blockIdx.x / (heads * n);
  return WorkId{(int)(in / n), (int)((t % runs) * per + per - 1 - t / runs), (int)(in % n)};
}

template <int DK, int DV>
struct Cfg {
  static constexpr int KROW = DK * 2, VROW = DV * 2, KB = kBlk * KROW, VB = kBlk * VROW;
  static constexpr int KS = DK / 16, VS = DV / 16, KC = DK / 32, VC = DV / 32;
  static constexpr int WAVES = DV > 128 ? 1 : 2;      // per SIMD: the accumulators of the widest form take the registers of two
};

// Scores of hidden keys (from `room` on, counted from this lane's first) of both maps
__device__ __forceinline__ void hide(f32x16 (&s)[2], int room) {
#pragma unroll
  for (int e = 0; e < 16; e++) {
    s[0][e] = 8 * (e >> 2) + (e & 3) >= room ? -INFINITY : s[0][e];
    s[1][e] = 8 * (e >> 2) + (e & 3) >= room ? -INFINITY : s[1][e];
  }
}
// The careful way of the running softmax of both maps over 32 keys: moves the running maxima where a score exceeds them by kLazy, and
// leaves s[m] and base[m] so that the exponential of a score is exp2(s c2 - base).
template <int VC>
__device__ __forceinline__ void softmax_step(f32x16 (&s)[2], f32x16 (&acc)[2][VC], float (&mrun)[2], float (&lsum)[2], float (&base)[2], float c2,
                                             float lazy) {
  float mx[2], top[2];
#pragma unroll
  for (int m = 0; m < 2; m++) {
    mx[m] = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16; e += 2) mx[m] = fmaxf(fmaxf(s[m][e], s[m][e + 1]), mx[m]);
    mx[m] = half_max(mx[m]);
  }
  if (__builtin_amdgcn_ballot_w64(mx[0] > mrun[0] + lazy || mx[1] > mrun[1] + lazy) != 0) {
#pragma unroll
    for (int m = 0; m < 2; m++) {
      const float mn = fmaxf(mrun[m], mx[m]);
      const float alpha = __builtin_amdgcn_exp2f((mrun[m] - (mn == -INFINITY ? 0.f : mn)) * c2);
      mrun[m] = mn;
      lsum[m] *= alpha;
#pragma unroll
      for (int cb = 0; cb < VC; cb++) acc[m][cb] *= alpha;
    }
  }
#pragma unroll
  for (int m = 0; m < 2; m++) {
    top[m] = mrun[m] == -INFINITY ? 0.f : mrun[m];
    base[m] = top[m] * c2;
  }
  // one multiply-add per score; its constant residue (2^-24 of base, the same for a whole row) cancels in the quotient unless it is
  // itself an exponent to speak of, as with scores that stand for a mask's lowest value
  if (__builtin_amdgcn_ballot_w64(fmaxf(fabsf(base[0]), fabsf(base[1])) > kLargeScore) != 0) {
#pragma unroll
    for (int m = 0; m < 2; m++) {
#pragma unroll
      for (int e = 0; e < 16; e++) s[m][e] -= top[m];
      base[m] = 0.f;
    }
  }
}

// A row's share of the keys, for the joining kernel: running maxima, sums and unnormalised accumulators
template <int VC>
__device__ __forceinline__ void store_share(const DiffParams& P, size_t row, int h, const f32x16 (&acc)[2][VC], const float (&mrun)[2], const float (&lsum)[2]) {
  if (h == 0) *reinterpret_cast<f32x4*>(P.ml + row * 4) = f32x4{mrun[0], lsum[0], mrun[1], lsum[1]};
#pragma unroll
  for (int m = 0; m < 2; m++)
#pragma unroll
    for (int cb = 0; cb < VC; cb++)
#pragma unroll
      for (int e = 0; e < 4; e++)
        *reinterpret_cast<f32x4*>(P.part + (row * 2 + m) * (VC * 32) + cb * 32 + 8 * e + 4 * h) =
            f32x4{acc[m][cb][4 * e], acc[m][cb][4 * e + 1], acc[m][cb][4 * e + 2], acc[m][cb][4 * e + 3]};
}

// The same between the waves of a workgroup, through LDS (p: this lane's first of kShareItems rows of 64 items)
template <int VC> constexpr int kShareItems = 8 * VC + 1;
template <int VC>
__device__ __forceinline__ void lend_share(f32x4* p, const f32x16 (&acc)[2][VC], const float (&mrun)[2], const float (&lsum)[2]) {
#pragma unroll
  for (int m = 0; m < 2; m++)
#pragma unroll
    for (int cb = 0; cb < VC; cb++)
#pragma unroll
      for (int e = 0; e < 4; e++)
        p[((m * VC + cb) * 4 + e) * 64] = f32x4{acc[m][cb][4 * e], acc[m][cb][4 * e + 1], acc[m][cb][4 * e + 2], acc[m][cb][4 * e + 3]};
  p[8 * VC * 64] = f32x4{mrun[0], lsum[0], mrun[1], lsum[1]};
}
template <int VC>
__device__ __forceinline__ void take_share(const f32x4* p, f32x16 (&acc)[2][VC], float (&mrun)[2], float (&lsum)[2], float c2) {
  const f32x4 ml = p[8 * VC * 64];
#pragma unroll
  for (int m = 0; m < 2; m++) {
    const float mn = fmaxf(mrun[m], ml[2 * m]), top = mn == -INFINITY ? 0.f : mn;
    const float own = __builtin_amdgcn_exp2f((mrun[m] - top) * c2), other = __builtin_amdgcn_exp2f((ml[2 * m] - top) * c2);
    mrun[m] = mn;
    lsum[m] = lsum[m] * own + ml[2 * m + 1] * other;
#pragma unroll
    for (int cb = 0; cb < VC; cb++) {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const f32x4 v = p[((m * VC + cb) * 4 + e) * 64];
#pragma unroll
        for (int x = 0; x < 4; x++) acc[m][cb][4 * e + x] = acc[m][cb][4 * e + x] * own + v[x] * other;
      }
      if (VC > 4) __builtin_amdgcn_sched_barrier(0);       // (few values at once: the accumulators fill the registers)
    }
  }
}

// A finished row: out = O1 - lam O2, and for a backward pass O2 and the log2-sums
template <int VC>
__device__ __forceinline__ void store_row(const DiffParams& P, const f32x16 (&acc)[2][VC], const float (&mrun)[2], const float (&lsum)[2], int b, int i,
                                          int head, int h) {
  const gc_diff_attention& a = P.a;
  const float inv0 = lsum[0] != 0.f ? 1.f / lsum[0] : 0.f, inv1 = lsum[1] != 0.f ? 1.f / lsum[1] : 0.f, lam = a.lam[head];
  const size_t orow = (((size_t)b * a.NQ + i) * a.H + head) * a.dv;
#pragma unroll
  for (int cb = 0; cb < VC; cb++)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int c = cb * 32 + 8 * e + 4 * h;
      if (c >= a.dv) continue;
      f32x4 o2, o;
#pragma unroll
      for (int x = 0; x < 4; x++) {
        o2[x] = acc[1][cb][4 * e + x] * inv1;
        o[x] = acc[0][cb][4 * e + x] * inv0 - lam * o2[x];
      }
      *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(a.out) + orow + c) = cvt_bf16x4(o);
      if (a.out2 != nullptr) *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(a.out2) + orow + c) = cvt_bf16x4(o2);
    }
  if (a.lse != nullptr && h == 0) {
    float* l = a.lse + ((size_t)b * a.H + head) * 2 * a.NQ + i;
    l[0] = lsum[0] != 0.f ? mrun[0] * P.c2 + __log2f(lsum[0]) : INFINITY;
    l[a.NQ] = lsum[1] != 0.f ? mrun[1] * P.c2 + __log2f(lsum[1]) : INFINITY;
  }
}

// ---------------------------------------------------------------------------------------------------------------------------
// Rows of a workgroup: 128 of the G * NQ rows (head of the group, query) that share a key head.
template <int DK, int DV>
__global__ __launch_bounds__(kThreads, (Cfg<DK, DV>::WAVES)) void diff_fwd_kernel(const DiffParams P) {
  typedef Cfg<DK, DV> F;
  constexpr int STAGE = 2 * F::KB + F::VB;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const gc_diff_attention& a = P.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const WorkId id = work_id(P, (uint32_t)a.B * a.HK, (uint32_t)P.G);
  const int split = id.share, tile = id.tile, bh = id.bh, b = bh / a.HK, hk = bh - b * a.HK;
  const int R = P.G * a.NQ, len = sample_length(a, b);
  const int r0 = tile * kRows, w0 = r0 + wave * 32, r = w0 + (lane & 31);
  const bool valid = r < R;
  const int rc = valid ? r : R - 1, g = (int)fd_div((uint32_t)rc, P.div_nq), i = rc - g * a.NQ, head = hk * P.G + g;
  const int lim = visible(a, i, len);
  // most and fewest visible keys of this wave's rows, most of the workgroup's
  int kend = len, wmin = len, wmax = len;
  if (a.causal) {
    const int e = (r0 + kRows < R ? r0 + kRows : R) - 1, ge = (int)fd_div((uint32_t)e, P.div_nq), gs = (int)fd_div((uint32_t)r0, P.div_nq);
    kend = gs == ge ? visible(a, e - ge * a.NQ, len) : len;
    const int first = w0 < R ? w0 : R - 1, last = w0 + 31 < R ? w0 + 31 : R - 1;
    const int gf = (int)fd_div((uint32_t)first, P.div_nq), gl = (int)fd_div((uint32_t)last, P.div_nq);
    wmin = gf == gl ? visible(a, first - gf * a.NQ, len) : visible(a, 0, len);
    wmax = gf == gl ? visible(a, last - gl * a.NQ, len) : len;
  }
  wmin = __builtin_amdgcn_readfirstlane(wmin);
  wmax = __builtin_amdgcn_readfirstlane(wmax);

  const uint16_t* qrow = static_cast<const uint16_t*>(a.q) + b * a.q_stride[0] + i * a.q_stride[1] + head * a.q_stride[2];
  bf16x8 qf[2][F::KS];
#pragma unroll
  for (int m = 0; m < 2; m++)
#pragma unroll
    for (int ks = 0; ks < F::KS; ks++) qf[m][ks] = global_frag(qrow + m * a.q_stride[3], valid, ks * 16 + 8 * h, a.d);

  f32x16 acc[2][F::VC];
  float mrun[2] = {-INFINITY, -INFINITY}, lsum[2] = {0.f, 0.f}, base[2] = {0.f, 0.f};
  bool careful = true;                                     // (of the whole wave) no maximum yet, or scores too large for the short way
#pragma unroll
  for (int m = 0; m < 2; m++)
#pragma unroll
    for (int cb = 0; cb < F::VC; cb++) acc[m][cb] = zero16();

  const uint32_t base0 = lds_offset(smem);
  const uint32_t kaddr = base0 + row_addr<F::KROW, kRowWise>(lane), vaddr = base0 + 2 * F::KB + col_addr<F::VROW, kTransposed>(lane, 0);
  const int nblk = (kend + kBlk - 1) / kBlk;
  const int blk0 = split * P.blocks_per_split, blk1 = min(nblk, blk0 + P.blocks_per_split);
  KeyTiles<F::KROW, F::VROW, kRowWise, kTransposed, kBlk, kThreads / 64> tiles;
  tiles.init(a, b, hk, blk0 * kBlk, len, wave, lane);
  if (blk0 < blk1) tiles.next(base0);
  for (int blk = blk0; blk < blk1; blk++) {
    tile_ready();
    if (blk + 1 < blk1) tiles.next(base0 + ((blk + 1 - blk0) & 1) * STAGE);
    const uint32_t stage = ((blk - blk0) & 1) * STAGE;
    // (the whole wave; the barrier above is met by every wave in every step)
    if (blk * kBlk >= wmax) continue;
#pragma unroll 1
    for (int jb = 0; jb < 2; jb++) {
      const int j0 = blk * kBlk + jb * 32;
      const uint32_t ka = kaddr + stage + jb * 32 * F::KROW, va = vaddr + stage + jb * 32 * F::VROW;
      // LDS reads are issued well in front of the matrix instructions that use them, all K fragments first, the V fragments in two
      // halves; the fences keep the compiler from moving them back down
      f32x16 s[2];
      {
        bf16x8 kf[2][F::KS];
#pragma unroll
        for (int ks = 0; ks < F::KS; ks++)
#pragma unroll
          for (int m = 0; m < 2; m++) kf[m][ks] = read_row((ka ^ (ks << 5)) + m * F::KB);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int ks = 0; ks < F::KS; ks++)
#pragma unroll
          for (int m = 0; m < 2; m++) s[m] = mfma(kf[m][ks], qf[m][ks], ks == 0 ? zero16() : s[m]);
      }
      if (j0 + 32 > wmin) hide(s, lim - j0 - 4 * h);
      // Exponentials against the maxima so far, without looking for new ones: the sum of a lane's 16 exponentials, wanted anyway,
      // tells whether one of them passed 2^8 (it is then above 2^8 ... 2^12, or infinite).  Then, and while a row has no maximum
      // yet, the scores are formed again and take the careful way.
      float sum[2];
      auto exponentials = [&]() {
#pragma unroll
        for (int m = 0; m < 2; m++) {
          sum[m] = 0.f;
#pragma unroll
          for (int e = 0; e < 16; e++) {
            s[m][e] = __builtin_amdgcn_exp2f(s[m][e] * P.c2 - base[m]);
            sum[m] += s[m][e];
          }
        }
      };
      bool again = careful;
      if (!again) {
        exponentials();
        again = __builtin_amdgcn_ballot_w64(fmaxf(sum[0], sum[1]) > 16.f * kLazyExp) != 0;
      }
      if (again) {
        if (!careful) {
#pragma unroll
          for (int m = 0; m < 2; m++)
#pragma unroll
            for (int ks = 0; ks < F::KS; ks++) {
              s[m] = mfma(read_row((ka ^ (ks << 5)) + m * F::KB), qf[m][ks], ks == 0 ? zero16() : s[m]);
              __builtin_amdgcn_sched_barrier(0);           // (one operand at a time: rare, and the registers are taken)
            }
          if (j0 + 32 > wmin) hide(s, lim - j0 - 4 * h);
        }
        softmax_step<F::VC>(s, acc, mrun, lsum, base, P.c2, P.lazy);
        exponentials();
        careful = __builtin_amdgcn_ballot_w64(mrun[0] == -INFINITY || mrun[1] == -INFINITY ||
                                              fmaxf(fabsf(mrun[0]), fabsf(mrun[1])) * P.c2 > kLargeScore) != 0;
      }
      bf16x8 vf[F::VC], pb[2][2];
#pragma unroll
      for (int cb = 0; cb < F::VC; cb++) vf[cb] = read_col(va ^ (cb << 6), (va ^ (cb << 6)) + 8 * F::VROW);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int m = 0; m < 2; m++) {
        lsum[m] += sum[m];
        pb[m][0] = pack8(s[m], 0);
        pb[m][1] = pack8(s[m], 8);
      }
      __builtin_amdgcn_sched_barrier(0);
      bf16x8 vg[F::VC];
#pragma unroll
      for (int cb = 0; cb < F::VC; cb++) vg[cb] = read_col((va ^ (cb << 6)) + 16 * F::VROW, (va ^ (cb << 6)) + 24 * F::VROW);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int cb = 0; cb < F::VC; cb++) {
        acc[0][cb] = mfma(vf[cb], pb[0][0], acc[0][cb]);
        acc[1][cb] = mfma(vf[cb], pb[1][0], acc[1][cb]);
      }
#pragma unroll
      for (int cb = 0; cb < F::VC; cb++) {
        acc[0][cb] = mfma(vg[cb], pb[0][1], acc[0][cb]);
        acc[1][cb] = mfma(vg[cb], pb[1][1], acc[1][cb]);
      }
    }
  }

  lsum[0] = half_sum(lsum[0]);
  lsum[1] = half_sum(lsum[1]);
  if (!valid) return;
  if (P.nsplit > 1) {
    store_share<F::VC>(P, ((size_t)split * a.B * a.HK + bh) * R + r, h, acc, mrun, lsum);
    return;
  }
  store_row<F::VC>(P, acc, mrun, lsum, b, i, head, h);
}

// The forms whose registers hold two waves per SIMD: 8 waves, of which four and four take turns on the matrix units.  Two waves of a SIMD
// left alone fall into step, and the matrix unit waits while both form exponentials: its share of the cycles and the vector unit's added
// up to the whole.  Here waves 0-3 work on the first 32 keys of every tile, waves 4-7 on the second, for the same 128 rows, and a barrier
// after every phase keeps one half multiplying (a block's probabilities with its values, then the next block's scores) while the other
// half forms exponentials; the multiplying waves go first where both could issue.  The two shares are joined at the end.  Tiles go through
// a ring of five: two are in use, the others have landed or are on their way.  N 4096, batch 32, one head of 64/128: 436 us with two
// independent workgroups of 4 waves per CU, 411 so (752 TFLOP/s, matrix unit busy 55 % of the cycles at the 1.84 GHz that power leaves);
// N 4096, 8 heads of one sample, where every CU has one workgroup: 126 and 97; 2048, 16 heads: 68 and 55.  It starts later and ends with the
// joining of the halves, so that short walks are left to the four waves (takes_turns).
template <int DK, int DV>
struct TurnsCfg {
  static constexpr int NW = 8, KB = kBlk * DK * 2, VB = kBlk * DV * 2, STAGE = 2 * KB + VB, LOADS = STAGE / 1024 / NW;
  static constexpr int RING = 5 * STAGE;
  static constexpr int SHARES = 4 * 64 * 16 * kShareItems<DV / 32>, LDS = RING > SHARES ? RING : SHARES;
};
template <int DK, int DV>
__global__ __launch_bounds__(512, 2) void diff_fwd_turns_kernel(const DiffParams P) {
  typedef Cfg<DK, DV> F;
  typedef TurnsCfg<DK, DV> X;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const gc_diff_attention& a = P.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), late = wave >> 2, h = lane >> 5;
  const WorkId id = work_id(P, (uint32_t)a.B * a.HK, (uint32_t)P.G);
  const int split = id.share, tile = id.tile, bh = id.bh, b = bh / a.HK, hk = bh - b * a.HK;
  const int R = P.G * a.NQ, len = sample_length(a, b);
  const int r0 = tile * kRows, w0 = r0 + (wave & 3) * 32, r = w0 + (lane & 31);
  const bool valid = r < R;
  const int rc = valid ? r : R - 1, g = (int)fd_div((uint32_t)rc, P.div_nq), i = rc - g * a.NQ, head = hk * P.G + g;
  const int lim = visible(a, i, len);
  // most and fewest visible keys of this wave's rows, most of the workgroup's
  int kend = len, wmin = len, wmax = len;
  if (a.causal) {
    const int e = (r0 + kRows < R ? r0 + kRows : R) - 1, ge = (int)fd_div((uint32_t)e, P.div_nq), gs = (int)fd_div((uint32_t)r0, P.div_nq);
    kend = gs == ge ? visible(a, e - ge * a.NQ, len) : len;
    const int first = w0 < R ? w0 : R - 1, last = w0 + 31 < R ? w0 + 31 : R - 1;
    const int gf = (int)fd_div((uint32_t)first, P.div_nq), gl = (int)fd_div((uint32_t)last, P.div_nq);
    wmin = gf == gl ? visible(a, first - gf * a.NQ, len) : visible(a, 0, len);
    wmax = gf == gl ? visible(a, last - gl * a.NQ, len) : len;
  }
  wmin = __builtin_amdgcn_readfirstlane(wmin);
  wmax = __builtin_amdgcn_readfirstlane(wmax);

  const uint16_t* qrow = static_cast<const uint16_t*>(a.q) + b * a.q_stride[0] + i * a.q_stride[1] + head * a.q_stride[2];
  bf16x8 qf[2][F::KS];
#pragma unroll
  for (int m = 0; m < 2; m++)
#pragma unroll
    for (int ks = 0; ks < F::KS; ks++) qf[m][ks] = global_frag(qrow + m * a.q_stride[3], valid, ks * 16 + 8 * h, a.d);

  f32x16 acc[2][F::VC];
  float mrun[2] = {-INFINITY, -INFINITY}, lsum[2] = {0.f, 0.f}, base[2] = {0.f, 0.f};
  bool careful = true;                                     // (of the whole wave) no maximum yet, or scores too large for the short way
#pragma unroll
  for (int m = 0; m < 2; m++)
#pragma unroll
    for (int cb = 0; cb < F::VC; cb++) acc[m][cb] = zero16();

  const uint32_t base0 = lds_offset(smem);
  const uint32_t kaddr = base0 + late * 32 * F::KROW + row_addr<F::KROW, kRowWise>(lane);
  const uint32_t vaddr = base0 + 2 * F::KB + late * 32 * F::VROW + col_addr<F::VROW, kTransposed>(lane, 0);
  const int nblk = (kend + kBlk - 1) / kBlk;
  const int blk0 = split * P.blocks_per_split, T = max(0, min(nblk, blk0 + P.blocks_per_split) - blk0);
  // a wave fetches rows of one map of the keys and of the values; behind the last row: loads of no rows, which read nothing
  TileStream<F::KROW, kRowWise, 4> tk;
  TileStream<F::VROW, kTransposed, 8> tv;
  const uint32_t kst = (uint32_t)(a.k_stride[1] * 2), vst = (uint32_t)(a.v_stride[1] * 2);
  const int first = blk0 * kBlk;
  tk.init(wave & 3, lane, reinterpret_cast<const char*>(static_cast<const uint16_t*>(a.k) + b * a.k_stride[0] + hk * a.k_stride[2] + late * a.k_stride[3]) + first * (int64_t)kst,
          len - first, kst, a.d);
  tv.init(wave, lane, reinterpret_cast<const char*>(static_cast<const uint16_t*>(a.v) + b * a.v_stride[0] + hk * a.v_stride[2]) + first * (int64_t)vst, len - first, vst, a.dv);
  auto after = [](uint32_t st) { return st + X::STAGE == X::RING ? 0u : st + X::STAGE; };
  uint32_t ask = 0;
  constexpr int PIECES = tk.NI + tv.NI;
  auto fetch = [&](int n) {                                // pieces of the next tile, in order
    if (n < tk.NI) tk.piece(n < tk.NI ? n : 0, wave & 3, base0 + ask + late * F::KB);
    else if (n < PIECES) tv.piece(n < PIECES && n >= tk.NI ? n - tk.NI : 0, wave, base0 + ask + 2 * F::KB);
    if (n == PIECES - 1) {
      ask = after(ask);
      tk.next();
      tv.next();
    }
  };
  auto turn = [&]() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  float sum[2];
  auto exponentials = [&](f32x16 (&s)[2]) {
#pragma unroll
    for (int m = 0; m < 2; m++) {
      sum[m] = 0.f;
#pragma unroll
      for (int e = 0; e < 16; e++) {
        s[m][e] = __builtin_amdgcn_exp2f(s[m][e] * P.c2 - base[m]);
        sum[m] += s[m][e];
      }
    }
  };

  auto scores = [&](f32x16 (&s)[2], const bf16x8 (&k)[2], int ks) {
#pragma unroll
    for (int m = 0; m < 2; m++) s[m] = mfma(k[m], qf[m][ks], ks == 0 ? zero16() : s[m]);
  };
  auto keys = [&](bf16x8 (&k)[2], uint32_t ka, int ks) {
#pragma unroll
    for (int m = 0; m < 2; m++) k[m] = read_row((ka ^ (ks << 5)) + m * F::KB);
  };
  auto value = [&](bf16x8& v, uint32_t va, int n) {
    const uint32_t x = (va ^ ((n % F::VC) << 6)) + (n / F::VC) * 16 * F::VROW;
    v = read_col(x, x + 8 * F::VROW);
  };
  arrived(qf);
#pragma unroll
  for (int x = 0; x < 4; x++)
#pragma unroll
    for (int n = 0; n < PIECES; n++) fetch(n);
  wait_loads<3 * X::LOADS>();
  turn();
  if (late) turn();
  f32x16 s[2];
  {
    bf16x8 k[F::KS][2];
#pragma unroll
    for (int ks = 0; ks < F::KS; ks++) keys(k[ks], kaddr, ks);
#pragma unroll
    for (int ks = 0; ks < F::KS; ks++) scores(s, k[ks], ks);
  }
  wait_loads<2 * X::LOADS>();
  turn();
  // In every step everyone asks for the tile four on; letting the youngest two stay in flight puts the tile that the other half reads
  // in two phases in place.
  const int own = min(T, max(0, (wmax - blk0 * kBlk - late * 32 + kBlk - 1) / kBlk));      // steps in which this wave sees keys
  uint32_t here = 0;                                       // stage of this step's tile
  int t = 0;
  for (; t < own; t++) {
    const int j0 = (blk0 + t) * kBlk + late * 32;
    if (j0 + 32 > wmin) hide(s, lim - j0 - 4 * h);
    // Exponentials against the maxima so far, without looking for new ones: the sum of a lane's 16 exponentials, wanted anyway,
    // tells whether one of them passed 2^8 (it is then above 2^8 ... 2^12, or infinite).  Then, and while a row has no maximum
    // yet, the scores are formed again and take the careful way.
    bool again = careful;
    if (!again) {
      exponentials(s);
      again = __builtin_amdgcn_ballot_w64(fmaxf(sum[0], sum[1]) > 16.f * kLazyExp) != 0;
    }
    if (again) {
      if (!careful) {
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
          for (int ks = 0; ks < F::KS; ks++) {
            s[m] = mfma(read_row(((kaddr + here) ^ (ks << 5)) + m * F::KB), qf[m][ks], ks == 0 ? zero16() : s[m]);
            __builtin_amdgcn_sched_barrier(0);             // (one operand at a time: rare, and the registers are taken)
          }
        if (j0 + 32 > wmin) hide(s, lim - j0 - 4 * h);
      }
      softmax_step<F::VC>(s, acc, mrun, lsum, base, P.c2, P.lazy);
      exponentials(s);
      careful = __builtin_amdgcn_ballot_w64(mrun[0] == -INFINITY || mrun[1] == -INFINITY ||
                                            fmaxf(fabsf(mrun[0]), fabsf(mrun[1])) * P.c2 > kLargeScore) != 0;
    }
      bf16x8 pb[2][2];
#pragma unroll
    for (int m = 0; m < 2; m++) {
      lsum[m] += sum[m];
      pb[m][0] = pack8(s[m], 0);
      pb[m][1] = pack8(s[m], 8);
    }
    // This block's products, then the next block's scores (of whatever lies there behind the last block: nobody looks at them), two matrix
    // instructions at a time.  An operand is read from LDS three of these steps before its turn, the first ones in this phase already;
    // the loads are asked for in between.
    constexpr int NV = 2 * F::VC, AHEAD = 3;
    const uint32_t va = vaddr + here, ka = kaddr + after(here);
    bf16x8 v[NV], k[F::KS][2];
#pragma unroll
    for (int n = 0; n < AHEAD; n++) value(v[n], va, n);
    arrived(pb);                                           // (and not put off into the other phase)
    turn();
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int q = 0; q < NV + F::KS; q++) {
      if (q < NV) {
        acc[0][q % F::VC] = mfma(v[q], pb[0][q / F::VC], acc[0][q % F::VC]);
        acc[1][q % F::VC] = mfma(v[q], pb[1][q / F::VC], acc[1][q % F::VC]);
      } else {
        scores(s, k[q - NV], q - NV);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (q + AHEAD < NV) value(v[q + AHEAD < NV ? q + AHEAD : 0], va, q + AHEAD);
      else if (q + AHEAD < NV + F::KS) keys(k[q + AHEAD < NV + F::KS ? q + AHEAD - NV : 0], ka, q + AHEAD - NV);
      if (q & 1) fetch(q / 2);
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
    wait_loads<2 * X::LOADS>();
    turn();
    here = after(here);
  }
  for (; t < T; t++) {
    turn();
#pragma unroll
    for (int n = 0; n < PIECES; n++) fetch(n);
    wait_loads<2 * X::LOADS>();
    turn();
  }
  if (!late) turn();

  wait_loads<0>();                                         // (nothing is still writing LDS)
  lsum[0] = half_sum(lsum[0]);
  lsum[1] = half_sum(lsum[1]);
  f32x4* const lds = reinterpret_cast<f32x4*>(smem) + (wave & 3) * kShareItems<F::VC> * 64 + lane;
  __syncthreads();
  if (late) lend_share<F::VC>(lds, acc, mrun, lsum);
  __syncthreads();
  if (late || !valid) return;
  take_share<F::VC>(lds, acc, mrun, lsum, P.c2);
  if (P.nsplit > 1) store_share<F::VC>(P, ((size_t)split * a.B * a.HK + bh) * R + r, h, acc, mrun, lsum);
  else store_row<F::VC>(P, acc, mrun, lsum, b, i, head, h);
}

// At most 32 rows per key head (single queries and short runs of them against long keys): bound by reading the keys and values once.
// Every wave walks a share of the keys of its own in tiles of 32, staged privately (no barriers; the loads of the next tile are in
// flight while one is worked on), so that a CU keeps 64 KiB of loads under way; the waves' shares become one in LDS (4 x 65536 keys, 16
// heads on 4: 117 us either way; 16384 keys, one head: 32 us with every wave's share left to the joining kernel, 20 so), the
// workgroups' are joined by a second launch, or the row is finished where there is one.  The matrix
// instructions are idle most of the time here, which pays for probabilities held to 16 bits: their bf16 rounding and its remainder
// are multiplied with the values separately.  One query of 16 heads on 4 against 4 x 65536 keys: 95 us, 4.9 TB/s, what a large copy reaches.
template <int DK, int DV>
struct FewCfg {
  static constexpr int NW = DV > 128 ? 2 : 4;              // waves
  static constexpr int KB = 32 * DK * 2, VB = 32 * DV * 2, STAGE = 2 * KB + VB, LOADS = STAGE / 1024;
};
__device__ __forceinline__ bf16x8 pack8_rest(const f32x16& v, int r0, bf16x8 hi) {
  const u32x4 b = __builtin_bit_cast(u32x4, hi);
  f32x16 d;
#pragma unroll
  for (int x = 0; x < 4; x++) {
    d[2 * x] = v[r0 + 2 * x] - __builtin_bit_cast(float, b[x] << 16);
    d[2 * x + 1] = v[r0 + 2 * x + 1] - __builtin_bit_cast(float, b[x] & 0xffff0000u);
  }
  return pack8(d, 0);
}
template <int DK, int DV>
__global__ __launch_bounds__((FewCfg<DK, DV>::NW * 64), 1) void diff_few_rows_kernel(const DiffParams P) {
  typedef Cfg<DK, DV> F;
  typedef FewCfg<DK, DV> X;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const gc_diff_attention& a = P.a;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), h = lane >> 5;
  const int bh = (int)(blockIdx.x / (uint32_t)P.nsplit), share = (int)(blockIdx.x % (uint32_t)P.nsplit);
  const int b = bh / a.HK, hk = bh - b * a.HK, R = P.G * a.NQ, len = sample_length(a, b), r = lane & 31;
  const bool valid = r < R;
  const int rc = valid ? r : R - 1, g = (int)fd_div((uint32_t)rc, P.div_nq), i = rc - g * a.NQ, head = hk * P.G + g;
  const int lim = visible(a, i, len), wmin = visible(a, 0, len), wmax = visible(a, a.NQ - 1, len);

  const uint16_t* qrow = static_cast<const uint16_t*>(a.q) + b * a.q_stride[0] + i * a.q_stride[1] + head * a.q_stride[2];
  bf16x8 qf[2][F::KS];
#pragma unroll
  for (int m = 0; m < 2; m++)
#pragma unroll
    for (int ks = 0; ks < F::KS; ks++) qf[m][ks] = global_frag(qrow + m * a.q_stride[3], valid, ks * 16 + 8 * h, a.d);
  f32x16 acc[2][F::VC];
  float mrun[2] = {-INFINITY, -INFINITY}, lsum[2] = {0.f, 0.f};
#pragma unroll
  for (int m = 0; m < 2; m++)
#pragma unroll
    for (int cb = 0; cb < F::VC; cb++) acc[m][cb] = zero16();

  const uint32_t base0 = lds_offset(smem) + wave * 2 * X::STAGE;
  const uint32_t kaddr = base0 + row_addr<F::KROW, kRowWise>(lane), vaddr = base0 + 2 * X::KB + col_addr<F::VROW, kTransposed>(lane, 0);
  const int t0 = (share * X::NW + wave) * P.blocks_per_split, t1 = min((wmax + 31) / 32, t0 + P.blocks_per_split);
  KeyTiles<F::KROW, F::VROW, kRowWise, kTransposed, 32, 1> tiles;
  tiles.init(a, b, hk, t0 * 32, len, 0, lane);
  arrived(qf);
  if (t0 < t1) tiles.next(base0);
  for (int t = t0; t < t1; t++) {
    // (behind the last tile: loads of no rows, which read nothing; the count of loads in flight stays the same)
    if (t + 1 == t1) tiles.left = 0;
    tiles.next(base0 + ((t + 1 - t0) & 1) * X::STAGE);
    wait_loads<X::LOADS>();
    const int j0 = t * 32;
    const uint32_t ka = kaddr + ((t - t0) & 1) * X::STAGE, va = vaddr + ((t - t0) & 1) * X::STAGE;
    f32x16 s[2];
#pragma unroll
    for (int ks = 0; ks < F::KS; ks++)
#pragma unroll
      for (int m = 0; m < 2; m++) s[m] = mfma(read_row((ka ^ (ks << 5)) + m * X::KB), qf[m][ks], ks == 0 ? zero16() : s[m]);
    float base[2];
    if (j0 + 32 > wmin) hide(s, lim - j0 - 4 * h);
    softmax_step<F::VC>(s, acc, mrun, lsum, base, P.c2, P.lazy);
    bf16x8 hi[2][2], lo[2][2];
#pragma unroll
    for (int m = 0; m < 2; m++) {
#pragma unroll
      for (int e = 0; e < 16; e++) {
        s[m][e] = __builtin_amdgcn_exp2f(s[m][e] * P.c2 - base[m]);
        lsum[m] += s[m][e];
      }
#pragma unroll
      for (int x = 0; x < 2; x++) {
        hi[m][x] = pack8(s[m], 8 * x);
        lo[m][x] = pack8_rest(s[m], 8 * x, hi[m][x]);
      }
    }
#pragma unroll
    for (int x = 0; x < 2; x++)
#pragma unroll
      for (int cb = 0; cb < F::VC; cb++) {
        const uint32_t y = (va ^ (cb << 6)) + x * 16 * F::VROW;
        const bf16x8 vf = read_col(y, y + 8 * F::VROW);
#pragma unroll
        for (int m = 0; m < 2; m++) {
          acc[m][cb] = mfma(vf, hi[m][x], acc[m][cb]);
          acc[m][cb] = mfma(vf, lo[m][x], acc[m][cb]);
        }
      }
  }
  wait_loads<0>();                                         // (nothing of this wave is still writing LDS)
  lsum[0] = half_sum(lsum[0]);
  lsum[1] = half_sum(lsum[1]);
  // The waves' shares become one, by halves, through the LDS that held the tiles
  f32x4* const lds = reinterpret_cast<f32x4*>(smem) + lane;
#pragma unroll
  for (int n = X::NW / 2; n > 0; n /= 2) {
    __syncthreads();
    if (wave >= n && wave < 2 * n && valid) lend_share<F::VC>(lds + (wave - n) * kShareItems<F::VC> * 64, acc, mrun, lsum);
    __syncthreads();
    if (wave < n && valid) take_share<F::VC>(lds + wave * kShareItems<F::VC> * 64, acc, mrun, lsum, P.c2);
  }
  if (wave > 0 || !valid) return;
  if (P.nsplit > 1) store_share<F::VC>(P, ((size_t)share * a.B * a.HK + bh) * R + r, h, acc, mrun, lsum);
  else store_row<F::VC>(P, acc, mrun, lsum, b, i, head, h);
}

// Joins up to 32 shares: DV / 4 lanes per row, four columns of both maps each; a lane forms the weights of all shares for itself.  (A
// workgroup per row, as for more shares, took eight times the attention's own time with many rows: N 1024, 16 heads of 64/128 in 4
// shares 315 us in all, against 41.)
constexpr int kFewShares = 32;
template <int DV>
__global__ __launch_bounds__(kThreads) void diff_join_rows_kernel(const DiffParams P) {
  constexpr int LANES = DV / 4;
  const gc_diff_attention& a = P.a;
  const int64_t R = (int64_t)P.G * a.NQ, rows = R * a.B * a.HK, idx = (int64_t)blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
  if (idx >= rows) return;
  const int c = threadIdx.x % LANES * 4, bh = (int)(idx / R), r = (int)(idx - bh * R), b = bh / a.HK, hk = bh - b * a.HK;
  const int g = (int)fd_div((uint32_t)r, P.div_nq), i = r - g * a.NQ, head = hk * P.G + g;
  const float *ml = P.ml + idx * 4, *part = P.part + idx * 2 * DV + c;
  float top[2] = {-INFINITY, -INFINITY}, L[2] = {0.f, 0.f};
  f32x4 o[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
  // eight shares at a time, all their loads under way together: latency is what this kernel is made of
  for (int s0 = 0; s0 < P.nsplit; s0 += 8) {
    f32x4 v[8], p[8][2];
#pragma unroll
    for (int x = 0; x < 8; x++) {
      const int64_t at = (s0 + x < P.nsplit ? s0 + x : P.nsplit - 1) * rows;
      v[x] = *reinterpret_cast<const f32x4*>(ml + at * 4);
#pragma unroll
      for (int m = 0; m < 2; m++) p[x][m] = *reinterpret_cast<const f32x4*>(part + (at * 2 + m) * DV);
    }
#pragma unroll
    for (int m = 0; m < 2; m++) {
      float now = top[m];
#pragma unroll
      for (int x = 0; x < 8; x++) now = v[x][2 * m + 1] != 0.f ? fmaxf(now, v[x][2 * m]) : now;
      const float ref = now == -INFINITY ? 0.f : now, before = __builtin_amdgcn_exp2f((top[m] - ref) * P.c2);
      top[m] = now;
      L[m] *= before;
      o[m] *= before;
#pragma unroll
      for (int x = 0; x < 8; x++) {
        // an empty share has no weight; a sum that is not a number has to reach the result
        const float l = v[x][2 * m + 1];
        const float w = s0 + x >= P.nsplit || l == 0.f ? 0.f : (l != l ? l : __builtin_amdgcn_exp2f((v[x][2 * m] - ref) * P.c2));
        L[m] += w == 0.f ? 0.f : w * l;
        o[m] += w * p[x][m];
      }
    }
  }
  const float inv0 = L[0] != 0.f ? 1.f / L[0] : 0.f, inv1 = L[1] != 0.f ? 1.f / L[1] : 0.f, lam = a.lam[head];
  const f32x4 o2 = o[1] * inv1, o1 = o[0] * inv0 - lam * o2;
  if (c < a.dv) {
    const int64_t at = (((int64_t)b * a.NQ + i) * a.H + head) * a.dv + c;
    *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(a.out) + at) = cvt_bf16x4(o1);
    if (a.out2 != nullptr) *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(a.out2) + at) = cvt_bf16x4(o2);
  }
  if (a.lse != nullptr && c == 0) {
    float* l = a.lse + ((int64_t)b * a.H + head) * 2 * a.NQ + i;
    l[0] = L[0] != 0.f ? top[0] * P.c2 + __log2f(L[0]) : INFINITY;
    l[a.NQ] = L[1] != 0.f ? top[1] * P.c2 + __log2f(L[1]) : INFINITY;
  }
}

// Joins the shares of a row that was split over the keys: one workgroup per row.  The shares' weights are worked out first (a thread
// per share), then every thread adds one value column of one map over every 4th or 8th share, all its loads independent: latency is
// what this kernel is made of.
constexpr int kMaxShares = 512, kJoinThreads = 1024;
__global__ __launch_bounds__(kJoinThreads) void diff_join_kernel(const DiffParams P, int DV) {
  __shared__ float wt[2][kMaxShares], red[4][kMaxShares / 64], cols[kJoinThreads];
  const gc_diff_attention& a = P.a;
  const int R = P.G * a.NQ, tid = threadIdx.x;
  const int64_t idx = blockIdx.x;
  const size_t rows = (size_t)a.B * a.HK * R;
  const int bh = (int)(idx / R), r = (int)(idx - (int64_t)bh * R), b = bh / a.HK, hk = bh - b * a.HK;
  const int g = r / a.NQ, i = r - g * a.NQ, head = hk * P.G + g;
  float top[2] = {-INFINITY, -INFINITY}, own[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  if (tid < P.nsplit) {
    const f32x4 ml = *reinterpret_cast<const f32x4*>(P.ml + ((size_t)tid * rows + idx) * 4);
#pragma unroll
    for (int m = 0; m < 2; m++) {
      own[m] = ml[2 * m];
      l[m] = ml[2 * m + 1];
      if (l[m] != 0.f) top[m] = own[m];
    }
  }
#pragma unroll
  for (int m = 0; m < 2; m++) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top[m] = fmaxf(top[m], __shfl_xor(top[m], o, 64));
    if (tid < kMaxShares && (tid & 63) == 0) red[m][tid >> 6] = top[m];
  }
  __syncthreads();
#pragma unroll
  for (int m = 0; m < 2; m++) {
#pragma unroll
    for (int w = 0; w < kMaxShares / 64; w++) top[m] = fmaxf(top[m], red[m][w]);
    // an empty share has no weight; a sum that is not a number has to reach the result
    const float w = l[m] == 0.f ? 0.f : (l[m] != l[m] ? l[m] : __builtin_amdgcn_exp2f((own[m] - top[m]) * P.c2));
    if (tid < P.nsplit) wt[m][tid] = w;
    float t = l[m] == 0.f ? 0.f : w * l[m];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) t += __shfl_xor(t, o, 64);
    if (tid < kMaxShares && (tid & 63) == 0) red[2 + m][tid >> 6] = t;
  }
  __syncthreads();
  float L[2] = {0.f, 0.f};
#pragma unroll
  for (int m = 0; m < 2; m++)
#pragma unroll
    for (int w = 0; w < kMaxShares / 64; w++) L[m] += red[2 + m][w];
  const float inv0 = L[0] != 0.f ? 1.f / L[0] : 0.f, inv1 = L[1] != 0.f ? 1.f / L[1] : 0.f, lam = a.lam[head];
  const size_t orow = (((size_t)b * a.NQ + i) * a.H + head) * a.dv;
  const int width = DV < 128 ? DV : 128, per = 2 * width, groups = kJoinThreads / per, grp = tid / per, m = (tid % per) / width;
  for (int c0 = 0; c0 < a.dv; c0 += width) {
    const float* src = P.part + ((size_t)idx * 2 + m) * DV + c0 + tid % width;
    float acc = 0.f;
#pragma unroll 16
    for (int s = grp; s < P.nsplit; s += groups) acc += wt[m][s] * src[(size_t)s * rows * 2 * DV];
    cols[tid] = acc;
    __syncthreads();
    const int c = c0 + tid;
    if (tid < width && c < a.dv) {
      float t[2] = {0.f, 0.f};
      for (int q = 0; q < groups; q++)
#pragma unroll
        for (int x = 0; x < 2; x++) t[x] += cols[q * per + x * width + tid];
      const float o2 = t[1] * inv1;
      static_cast<uint16_t*>(a.out)[orow + c] = float_to_bf16_bits(t[0] * inv0 - lam * o2);
      if (a.out2 != nullptr) static_cast<uint16_t*>(a.out2)[orow + c] = float_to_bf16_bits(o2);
    }
    __syncthreads();
  }
  if (a.lse != nullptr && tid < 2)
    a.lse[((size_t)b * a.H + head) * 2 * a.NQ + (size_t)tid * a.NQ + i] = (tid == 0 ? L[0] : L[1]) != 0.f ? (tid == 0 ? top[0] : top[1]) * P.c2 + __log2f(tid == 0 ? L[0] : L[1]) : INFINITY;
}

// delta [B][H][2][NQ]: dO . O1 = dO . out + lam dO . O2, and dO . O2; 16 lanes per row.  rows4 [B][H][4][NQ]: what the key gradients' kernel
// stages of a query: L1, L2 - log2|lam|, -delta1, sgn (delta1 - delta2) with sgn = -sign(lam): with p2' = |lam| p2 the mixed
// probability is p1 + sgn p2', dP - delta1 comes out of the matrix instructions, and dS2 = p2' (sgn (dP - delta1) + sgn (delta1 - delta2)).
// Bound by HBM and short: 131072 rows of 128 in 19 us (5.3 TB/s).
__global__ __launch_bounds__(kThreads) void diff_delta_kernel(const DiffParams P) {
  const gc_diff_attention& a = P.a;
  const size_t rows = (size_t)a.B * a.NQ * a.H, row = ((size_t)blockIdx.x * kThreads + threadIdx.x) >> 4;
  const int sub = threadIdx.x & 15;
  float s[2] = {0.f, 0.f};
  if (row < rows)
    for (int c = sub * 8; c < a.dv; c += 128) {
      const size_t o = row * a.dv + c;
      const u32x4 w = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.dout) + o);
      const u32x4 x = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.out) + o);
      const u32x4 y = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.out2) + o);
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float wl = __builtin_bit_cast(float, w[e] << 16), wh = __builtin_bit_cast(float, w[e] & 0xffff0000u);
        s[0] += wl * __builtin_bit_cast(float, x[e] << 16) + wh * __builtin_bit_cast(float, x[e] & 0xffff0000u);
        s[1] += wl * __builtin_bit_cast(float, y[e] << 16) + wh * __builtin_bit_cast(float, y[e] & 0xffff0000u);
      }
    }
#pragma unroll
  for (int m = 0; m < 2; m++)
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) s[m] += __shfl_xor(s[m], o);
  if (row < rows && sub == 0) {
    const int head = (int)(row % a.H);
    const size_t bi = row / a.H, b = bi / a.NQ, i = bi - b * a.NQ;
    float* d = P.delta + (b * a.H + head) * 2 * a.NQ + i;
    const float lam = a.lam[head], d0 = s[0] + lam * s[1], d1 = s[1];
    d[0] = d0;
    d[a.NQ] = d1;
    const float* l = a.lse + (b * a.H + head) * 2 * a.NQ + i;
    float* q = P.rows4 + (b * a.H + head) * 4 * a.NQ + i;
    q[0] = l[0];
    q[a.NQ] = l[a.NQ] - __log2f(fabsf(lam));
    q[2 * a.NQ] = -d0;
    q[3 * a.NQ] = lam > 0.f ? d1 - d0 : d0 - d1;
  }
}

// ---------------------------------------------------------------------------------------------------------------------------
// Owner: 128 queries of a head; walks the keys.  Produces dQ and the workgroup's share of dlam.  N 4096, batch 32, one head of 64/128: 440 us
// (702 TFLOP/s), bound as the key gradients' kernel.
template <int DK, int DV>
__global__ __launch_bounds__(kThreads, (Cfg<DK, DV>::WAVES)) void diff_bwd_dq_kernel(const DiffParams P) {
  typedef Cfg<DK, DV> F;
  constexpr int STAGE = 2 * F::KB + F::VB;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  __shared__ float red[kThreads / 64];
  const gc_diff_attention& a = P.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const WorkId id = work_id(P, (uint32_t)a.B * a.H, 1);
  const int share = id.share, tile = id.tile, bh = id.bh, b = bh / a.H, head = bh - b * a.H, hk = head / P.G;
  const int len = sample_length(a, b), r0 = tile * kRows, w0 = r0 + wave * 32, r = w0 + (lane & 31);
  const bool valid = r < a.NQ;
  const int i = valid ? r : a.NQ - 1, lim = visible(a, i, len);
  const int kend = visible(a, min(r0 + kRows, a.NQ) - 1, len);
  const int wmin = visible(a, min(w0, a.NQ - 1), len), wmax = visible(a, min(w0 + 31, a.NQ - 1), len);

  const uint16_t* qrow = static_cast<const uint16_t*>(a.q) + b * a.q_stride[0] + i * a.q_stride[1] + head * a.q_stride[2];
  const size_t orow = (((size_t)b * a.NQ + i) * a.H + head) * a.dv;
  const uint16_t* grow = static_cast<const uint16_t*>(a.dout) + orow;
  bf16x8 qf[2][F::KS], gf[F::VS];
#pragma unroll
  for (int m = 0; m < 2; m++)
#pragma unroll
    for (int ks = 0; ks < F::KS; ks++) qf[m][ks] = global_frag(qrow + m * a.q_stride[3], valid, ks * 16 + 8 * h, a.d);
#pragma unroll
  for (int ks = 0; ks < F::VS; ks++) gf[ks] = global_frag(grow, valid, ks * 16 + 8 * h, a.dv);
  // The matrix unit rounds its sums down by a small part of their last bit, whatever their sign.  The sum of 1e5 rows that makes dlam
  // showed it (1e-7 of the terms' sizes, 3e-5 of what is left of them); with dP of every other row formed with its sign turned the
  // bias cancels (4096 queries, batch 32: off by 3.5e-3 for every input, and by 1e-4 either way).
  const float turn = (r & 1) ? -1.f : 1.f;
  if (r & 1)
#pragma unroll
    for (int ks = 0; ks < F::VS; ks++) gf[ks] = __builtin_bit_cast(bf16x8, __builtin_bit_cast(u32x4, gf[ks]) ^ 0x80008000u);
  float L[2], D[2];
#pragma unroll
  for (int m = 0; m < 2; m++) {
    const size_t o = ((size_t)(b * a.H + head) * 2 + m) * a.NQ + i;
    L[m] = a.lse[o];
    D[m] = P.delta[o];
  }

  f32x16 acc[2][F::KC];
#pragma unroll
  for (int m = 0; m < 2; m++)
#pragma unroll
    for (int cb = 0; cb < F::KC; cb++) acc[m][cb] = zero16();
  float left = 0.f;                                        // sum_j p2 (dP - delta2), its sign turned in odd rows
  const float gap = turn * (D[0] - D[1]);
  f32x16 start;
#pragma unroll
  for (int e = 0; e < 16; e++) start[e] = -turn * D[0];

  const uint32_t base0 = lds_offset(smem);
  const uint32_t kra = base0 + row_addr<F::KROW, kBothWays>(lane), kca = base0 + col_addr<F::KROW, kBothWays>(lane, 0);
  const uint32_t vra = base0 + 2 * F::KB + row_addr<F::VROW, kRowWise>(lane);
  const int blk0 = share * P.blocks_per_split, blk1 = min((kend + kBlk - 1) / kBlk, blk0 + P.blocks_per_split);
  KeyTiles<F::KROW, F::VROW, kBothWays, kRowWise, kBlk, kThreads / 64> tiles;
  tiles.init(a, b, hk, blk0 * kBlk, len, wave, lane);
  if (blk0 < blk1) tiles.next(base0);
  for (int blk = blk0; blk < blk1; blk++) {
    tile_ready();
    if (blk + 1 < blk1) tiles.next(base0 + ((blk + 1 - blk0) & 1) * STAGE);
    const uint32_t stage = ((blk - blk0) & 1) * STAGE;
    if (blk * kBlk >= wmax) continue;
#pragma unroll 1
    for (int jb = 0; jb < 2; jb++) {
      const int j0 = blk * kBlk + jb * 32;
      const uint32_t ka = kra + stage + jb * 32 * F::KROW, va = vra + stage + jb * 32 * F::VROW, kc = kca + stage + jb * 32 * F::KROW;
      // (LDS reads ahead of their matrix instructions, as in the forward kernel)
      f32x16 s[2], dp;
      {
        bf16x8 kf[2][F::KS];
#pragma unroll
        for (int ks = 0; ks < F::KS; ks++)
#pragma unroll
          for (int m = 0; m < 2; m++) kf[m][ks] = read_row((ka ^ (ks << 5)) + m * F::KB);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int ks = 0; ks < F::KS; ks++)
#pragma unroll
          for (int m = 0; m < 2; m++) s[m] = mfma(kf[m][ks], qf[m][ks], ks == 0 ? zero16() : s[m]);
      }
      {
        constexpr int HALF = F::VS / 2;
        bf16x8 vf[HALF];
#pragma unroll
        for (int x = 0; x < 2; x++) {
#pragma unroll
          for (int ks = 0; ks < HALF; ks++) vf[ks] = read_row(va ^ ((x * HALF + ks) << 5));
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int ks = 0; ks < HALF; ks++) dp = mfma(vf[ks], gf[x * HALF + ks], x + ks == 0 ? start : dp);      // dP - delta1
        }
      }
      // The wave whose matrix instructions come next goes first: two waves of a SIMD then take turns, one on the matrix unit, the other on
      // the exponentials (N 4096, batch 32: 476 against 438 us; in the forward kernel the same gained nothing, 433 against 437)
      __builtin_amdgcn_s_setprio(0);
      if (j0 + 32 > wmin) hide(s, lim - j0 - 4 * h);
      float here_left = 0.f;                               // (16 of its addends at a time: fewer roundings at its full size)
#pragma unroll
      for (int e = 0; e < 16; e++) {
        s[0][e] = __builtin_amdgcn_exp2f(s[0][e] * P.c2 - L[0]) * dp[e];
        s[1][e] = __builtin_amdgcn_exp2f(s[1][e] * P.c2 - L[1]) * (dp[e] + gap);
        here_left += s[1][e];
      }
      left += here_left;
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int t = 0; t < 2; t++) {
        bf16x8 kt[2][F::KC], d[2];
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
          for (int cb = 0; cb < F::KC; cb++) kt[m][cb] = read_col_both<F::KROW>((kc ^ (cb << 6)) + m * F::KB + t * 16 * F::KROW);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int m = 0; m < 2; m++) d[m] = pack8(s[m], 8 * t);
#pragma unroll
        for (int cb = 0; cb < F::KC; cb++)
#pragma unroll
          for (int m = 0; m < 2; m++) acc[m][cb] = mfma(kt[m][cb], d[m], acc[m][cb]);
      }
    }
  }
  const float lam = a.lam[head];
  if (valid) {
    const float f[2] = {turn * a.scale, -turn * lam * a.scale};
    const size_t row = (((size_t)b * a.NQ + i) * a.H + head) * 2 * a.d;
    uint16_t* dst = static_cast<uint16_t*>(a.dq) + row;
    float* part = P.part + (size_t)share * a.B * a.NQ * a.H * 2 * a.d + row;
#pragma unroll
    for (int m = 0; m < 2; m++)
#pragma unroll
      for (int cb = 0; cb < F::KC; cb++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int c = cb * 32 + 8 * e + 4 * h;
          if (c >= a.d) continue;
          const f32x4 v = {acc[m][cb][4 * e] * f[m], acc[m][cb][4 * e + 1] * f[m], acc[m][cb][4 * e + 2] * f[m], acc[m][cb][4 * e + 3] * f[m]};
          if (P.nsplit > 1) *reinterpret_cast<f32x4*>(part + m * a.d + c) = v;
          else *reinterpret_cast<u32x2*>(dst + m * a.d + c) = cvt_bf16x4(v);
        }
  }
  float t = valid ? turn * left + (h == 0 && share == 0 ? D[1] : 0.f) : 0.f;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) t += __shfl_xor(t, o, 64);
  if (lane == 0) red[wave] = t;
  __syncthreads();
  if (tid == 0) P.lampart[((size_t)bh * P.tiles + tile) * P.nsplit + share] = ((red[0] + red[1]) + red[2]) + red[3];
}

// dlam[head] = -(the workgroups' shares, added in a fixed order); one workgroup per head
__global__ __launch_bounds__(kThreads) void diff_dlam_kernel(const DiffParams P) {
  __shared__ double red[kThreads];
  const int head = blockIdx.x;
  const int64_t per = (int64_t)P.tiles * P.nsplit, n = P.a.B * per;
  double s = 0.0;                                          // (sums of either sign, of which little may be left)
  for (int64_t i = threadIdx.x; i < n; i += kThreads) {
    const int64_t b = i / per, t = i - b * per;
    s += P.lampart[(b * P.a.H + head) * per + t];
  }
  red[threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (int i = 0; i < kThreads; i++) t += red[i];
    P.a.dlam[head] = (float)-t;
  }
}

// out = the sum of `shares` fp32 partial results, added in order; two tensors back to back in part: [shares][n0], [shares][n1]
__global__ __launch_bounds__(kThreads) void diff_sum_kernel(const float* part, int shares, uint16_t* out0, size_t n0, uint16_t* out1, size_t n1) {
  size_t i = ((size_t)blockIdx.x * kThreads + threadIdx.x) * 4, n = n0;
  const float* src = part;
  uint16_t* out = out0;
  if (i >= n0) {
    src += (size_t)shares * n0;
    i -= n0;
    n = n1;
    out = out1;
  }
  if (i >= n) return;
  f32x4 t = *reinterpret_cast<const f32x4*>(src + i);
#pragma unroll 4
  for (int s = 1; s < shares; s++) t += *reinterpret_cast<const f32x4*>(src + (size_t)s * n + i);
  *reinterpret_cast<u32x2*>(out + i) = cvt_bf16x4(t);
}

// The dQ kernel with the halves of a workgroup taking turns, as in the forward kernel: in one phase a block's dQ products, the next block's
// scores and its dP, in the other the exponentials and score gradients between them.  Three matrix instructions at a time, so that the one
// chain that dP is does not wait for itself.  For grids of up to a workgroup per CU, which it fills with two waves per SIMD (dQ and the rest
// of both passes, N 2048, 16 heads on 4: 259 us with the kernel above, 247 with this one; 1500, 16 heads 173 and 163; 4 x 1024, 8 heads,
// causal 133 and 127).  Larger grids it does no good (batch 32, N 4096: 442 and 459 us), small ones that are split further neither (1024,
// 4 heads: 85 and 87), nor walks of fewer than 12 blocks (both passes, 8 heads of 64/128, us with the kernel above and with this one: 32 x 128
// rows of 128 keys 58 and 63, of 320 88 and 94, of 704 153 and 152; 1536 x 1536, two shares of 12, 132 and 128).
template <int DK, int DV>
__global__ __launch_bounds__(512, 2) void diff_bwd_dq_turns_kernel(const DiffParams P) {
  typedef Cfg<DK, DV> F;
  typedef TurnsCfg<DK, DV> X;
  static_assert(2 * F::KC + F::KS == F::VS, "dP's steps go beside the others");
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const gc_diff_attention& a = P.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), late = wave >> 2, h = lane >> 5;
  const WorkId id = work_id(P, (uint32_t)a.B * a.H, 1);
  const int share = id.share, tile = id.tile, bh = id.bh, b = bh / a.H, head = bh - b * a.H, hk = head / P.G;
  const int len = sample_length(a, b), r0 = tile * kRows, w0 = r0 + (wave & 3) * 32, r = w0 + (lane & 31);
  const bool valid = r < a.NQ;
  const int i = valid ? r : a.NQ - 1, lim = visible(a, i, len);
  const int kend = visible(a, min(r0 + kRows, a.NQ) - 1, len);
  const int wmin = __builtin_amdgcn_readfirstlane(visible(a, min(w0, a.NQ - 1), len));
  const int wmax = __builtin_amdgcn_readfirstlane(visible(a, min(w0 + 31, a.NQ - 1), len));

  const uint16_t* qrow = static_cast<const uint16_t*>(a.q) + b * a.q_stride[0] + i * a.q_stride[1] + head * a.q_stride[2];
  const uint16_t* grow = static_cast<const uint16_t*>(a.dout) + (((size_t)b * a.NQ + i) * a.H + head) * a.dv;
  bf16x8 qf[2][F::KS], gf[1][F::VS];
#pragma unroll
  for (int m = 0; m < 2; m++)
#pragma unroll
    for (int ks = 0; ks < F::KS; ks++) qf[m][ks] = global_frag(qrow + m * a.q_stride[3], valid, ks * 16 + 8 * h, a.d);
#pragma unroll
  for (int ks = 0; ks < F::VS; ks++) gf[0][ks] = global_frag(grow, valid, ks * 16 + 8 * h, a.dv);
  // (every other row's dP with its sign turned, as in the kernel above)
  const float turned = (r & 1) ? -1.f : 1.f;
  if (r & 1)
#pragma unroll
    for (int ks = 0; ks < F::VS; ks++) gf[0][ks] = __builtin_bit_cast(bf16x8, __builtin_bit_cast(u32x4, gf[0][ks]) ^ 0x80008000u);
  float L[2], D[2];
#pragma unroll
  for (int m = 0; m < 2; m++) {
    const size_t o = ((size_t)(b * a.H + head) * 2 + m) * a.NQ + i;
    L[m] = a.lse[o];
    D[m] = P.delta[o];
  }
  asm volatile("" : "+v"(L[0]), "+v"(L[1]), "+v"(D[0]), "+v"(D[1]));      // (as arrived() does)
  arrived(qf);
  arrived(gf);

  f32x16 acc[2][F::KC];
#pragma unroll
  for (int m = 0; m < 2; m++)
#pragma unroll
    for (int cb = 0; cb < F::KC; cb++) acc[m][cb] = zero16();
  float left = 0.f;                                        // sum_j p2 (dP - delta2), its sign turned in odd rows
  const float gap = turned * (D[0] - D[1]);
  f32x16 start;
#pragma unroll
  for (int e = 0; e < 16; e++) start[e] = -turned * D[0];

  const uint32_t base0 = lds_offset(smem);
  const uint32_t kra = base0 + late * 32 * F::KROW + row_addr<F::KROW, kBothWays>(lane);
  const uint32_t kca = base0 + late * 32 * F::KROW + col_addr<F::KROW, kBothWays>(lane, 0);
  const uint32_t vra = base0 + 2 * F::KB + late * 32 * F::VROW + row_addr<F::VROW, kRowWise>(lane);
  const int blk0 = share * P.blocks_per_split, T = max(0, min((kend + kBlk - 1) / kBlk, blk0 + P.blocks_per_split) - blk0);
  TileStream<F::KROW, kBothWays, 4> tk;
  TileStream<F::VROW, kRowWise, 8> tv;
  const uint32_t kst = (uint32_t)(a.k_stride[1] * 2), vst = (uint32_t)(a.v_stride[1] * 2);
  const int first = blk0 * kBlk;
  tk.init(wave & 3, lane, reinterpret_cast<const char*>(static_cast<const uint16_t*>(a.k) + b * a.k_stride[0] + hk * a.k_stride[2] + late * a.k_stride[3]) + first * (int64_t)kst,
          len - first, kst, a.d);
  tv.init(wave, lane, reinterpret_cast<const char*>(static_cast<const uint16_t*>(a.v) + b * a.v_stride[0] + hk * a.v_stride[2]) + first * (int64_t)vst, len - first, vst, a.dv);
  auto after = [](uint32_t st) { return st + X::STAGE == X::RING ? 0u : st + X::STAGE; };
  uint32_t ask = 0;
  constexpr int PIECES = tk.NI + tv.NI;
  auto fetch = [&](int n) {                                // pieces of the next tile, in order
    if (n < tk.NI) tk.piece(n < tk.NI ? n : 0, wave & 3, base0 + ask + late * F::KB);
    else if (n < PIECES) tv.piece(n < PIECES && n >= tk.NI ? n - tk.NI : 0, wave, base0 + ask + 2 * F::KB);
    if (n == PIECES - 1) {
      ask = after(ask);
      tk.next();
      tv.next();
    }
  };
  auto turn = [&]() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  // operands of step n: 2 KC steps of dQ (half a block, a column block), then KS of the scores; one of dP's beside each
  struct Operands { bf16x8 k[2], v; };
  auto operands = [&](Operands& o, uint32_t here, uint32_t next, int n) {
#pragma unroll
    for (int m = 0; m < 2; m++)
      o.k[m] = n < 2 * F::KC ? read_col_both<F::KROW>(((kca + here) ^ ((n % F::KC) << 6)) + m * F::KB + (n / F::KC) * 16 * F::KROW)
                             : read_row(((kra + next) ^ ((n - 2 * F::KC) << 5)) + m * F::KB);
    o.v = read_row((vra + next) ^ (n << 5));
  };

#pragma unroll
  for (int x = 0; x < 4; x++)
#pragma unroll
    for (int n = 0; n < PIECES; n++) fetch(n);
  wait_loads<2 * X::LOADS>();
  turn();
  if (late) turn();
  f32x16 s[2], dp = start;                                 // dP - delta1
#pragma unroll
  for (int n = 0; n < F::VS; n++) {
    Operands o;
    operands(o, 0, 0, n);
    if (n >= 2 * F::KC)
#pragma unroll
      for (int m = 0; m < 2; m++) s[m] = mfma(o.k[m], qf[m][n < 2 * F::KC ? 0 : n - 2 * F::KC], n == 2 * F::KC ? zero16() : s[m]);
    dp = mfma(o.v, gf[0][n], dp);
  }
  wait_loads<X::LOADS>();
  turn();
  // In every step everyone asks for the tile four on; letting only this youngest one stay in flight puts the tile whose first operands
  // the other half reads in the next phase in place.
  const int own = min(T, max(0, (wmax - blk0 * kBlk - late * 32 + kBlk - 1) / kBlk));      // steps in which this wave sees keys
  uint32_t here = 0;                                       // stage of this step's tile
  int t = 0;
  for (; t < own; t++) {
    const int j0 = (blk0 + t) * kBlk + late * 32;
    if (j0 + 32 > wmin) hide(s, lim - j0 - 4 * h);
    float here_left = 0.f;                                 // (16 of its addends at a time: fewer roundings at its full size)
#pragma unroll
    for (int e = 0; e < 16; e++) {
      s[0][e] = __builtin_amdgcn_exp2f(s[0][e] * P.c2 - L[0]) * dp[e];
      s[1][e] = __builtin_amdgcn_exp2f(s[1][e] * P.c2 - L[1]) * (dp[e] + gap);
      here_left += s[1][e];
    }
    left += here_left;
    bf16x8 d[2][2];
#pragma unroll
    for (int m = 0; m < 2; m++) {
      d[m][0] = pack8(s[m], 0);
      d[m][1] = pack8(s[m], 8);
    }
    constexpr int AHEAD = 2;
    const uint32_t next = after(here);
    Operands o[F::VS];
#pragma unroll
    for (int n = 0; n < AHEAD; n++) operands(o[n], here, next, n);
    arrived(d);                                            // (and not put off into the other phase)
    turn();
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int n = 0; n < F::VS; n++) {
      if (n < 2 * F::KC) {
#pragma unroll
        for (int m = 0; m < 2; m++) acc[m][n % F::KC] = mfma(o[n].k[m], d[m][n / F::KC], acc[m][n % F::KC]);
      } else {
#pragma unroll
        for (int m = 0; m < 2; m++) s[m] = mfma(o[n].k[m], qf[m][n - 2 * F::KC], n == 2 * F::KC ? zero16() : s[m]);
      }
      dp = mfma(o[n].v, gf[0][n], n == 0 ? start : dp);
      __builtin_amdgcn_sched_barrier(0);
      if (n + AHEAD < F::VS) operands(o[n + AHEAD < F::VS ? n + AHEAD : 0], here, next, n + AHEAD);
      if (n >= 2) fetch(n - 2);
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
    wait_loads<X::LOADS>();
    turn();
    here = next;
  }
  for (; t < T; t++) {
    turn();
#pragma unroll
    for (int n = 0; n < PIECES; n++) fetch(n);
    wait_loads<X::LOADS>();
    turn();
  }
  if (!late) turn();

  wait_loads<0>();                                         // (nothing is still writing LDS)
  __syncthreads();
  f32x4* const lent = reinterpret_cast<f32x4*>(smem) + (wave & 3) * (8 * F::KC) * 64 + lane;
  float* const red = reinterpret_cast<float*>(smem + 4 * 8 * F::KC * 64 * 16);
  if (late)
#pragma unroll
    for (int x = 0; x < 8 * F::KC; x++) {
      const f32x16& v = acc[x / (4 * F::KC)][x / 4 % F::KC];
      lent[x * 64] = f32x4{v[4 * (x % 4)], v[4 * (x % 4) + 1], v[4 * (x % 4) + 2], v[4 * (x % 4) + 3]};
    }
  float tl = valid ? turned * left + (h == 0 && share == 0 && !late ? D[1] : 0.f) : 0.f;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) tl += __shfl_xor(tl, o, 64);
  if (lane == 0) red[wave] = tl;
  __syncthreads();
  if (tid == 0) {
    float sum = red[0];
    for (int w = 1; w < 8; w++) sum += red[w];
    P.lampart[((size_t)bh * P.tiles + tile) * P.nsplit + share] = sum;
  }
  if (late || !valid) return;
  const float lam = a.lam[head], f[2] = {turned * a.scale, -turned * lam * a.scale};
  const size_t row = (((size_t)b * a.NQ + i) * a.H + head) * 2 * a.d;
  uint16_t* dst = static_cast<uint16_t*>(a.dq) + row;
  float* part = P.part + (size_t)share * a.B * a.NQ * a.H * 2 * a.d + row;
#pragma unroll
  for (int m = 0; m < 2; m++)
#pragma unroll
    for (int cb = 0; cb < F::KC; cb++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int c = cb * 32 + 8 * e + 4 * h;
        if (c >= a.d) continue;
        f32x4 v = lent[((m * F::KC + cb) * 4 + e) * 64];
#pragma unroll
        for (int x = 0; x < 4; x++) v[x] = (acc[m][cb][4 * e + x] + v[x]) * f[m];
        if (P.nsplit > 1) *reinterpret_cast<f32x4*>(part + m * a.d + c) = v;
        else *reinterpret_cast<u32x2*>(dst + m * a.d + c) = cvt_bf16x4(v);
      }
}

// Owner: 128 keys of a key head; walks the queries of every head that shares them.  Produces dK and dV.  OUT: 1 dK, 2 dV, 3 both
// (both accumulators of the widest form do not fit the register file: it runs as two launches).  VLDS: the owned values, an operand of
// dP, stay in LDS instead of registers, and the queries are staged 32 rows at a time to make room: with 64 keys' worth of accumulators
// per wave that is what lets two waves share a SIMD without spilling (N 4096, batch 32, one head of 64/128: 626 us, 658 TFLOP/s, of which the
// power left after 47 % of the cycles on the matrix and 50 % on the vector unit is the bound; with the values in registers, 691 us at the
// time against 908 with what spilled, 925 in two launches and 1007 with one wave per SIMD).
template <int DK, int DV, int OUT>
struct DkvCfg {
  static constexpr bool VLDS = DV == 128 && (OUT & 1);
  static constexpr int ROWS = VLDS ? 32 : kBlk, KB = ROWS * DK * 2, VB = ROWS * DV * 2;
  static constexpr int STAGE = 2 * KB + VB + 4 * kBlk * 4;                  // with L1, L2, delta1, delta2 of the staged queries
  static constexpr int LDS = 2 * STAGE + (VLDS ? kRows * DV * 2 : 0);
};
template <int DK, int DV, int OUT>
__global__ __launch_bounds__(kThreads, (Cfg<DK, DV>::WAVES)) void diff_bwd_dkv_kernel(const DiffParams P) {
  typedef Cfg<DK, DV> F;
  typedef DkvCfg<DK, DV, OUT> X;
  constexpr int ROWS = X::ROWS, STAGE = X::STAGE;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const gc_diff_attention& a = P.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const WorkId id = work_id(P, (uint32_t)a.B * a.HK, 0);
  const int share = id.share, tile = id.tile, bh = id.bh, b = bh / a.HK, hk = bh - b * a.HK;
  const int len = sample_length(a, b), j0 = tile * kRows, w0 = j0 + wave * 32, j = w0 + (lane & 31);
  const bool valid = j < len;

  const int jc = valid ? j : 0;
  const uint16_t* kbase = static_cast<const uint16_t*>(a.k) + b * a.k_stride[0] + hk * a.k_stride[2];
  const uint16_t* vbase = static_cast<const uint16_t*>(a.v) + b * a.v_stride[0] + hk * a.v_stride[2];
  const uint32_t base0 = lds_offset(smem);
  bf16x8 kf[2][F::KS], vf[X::VLDS ? 1 : F::VS];
#pragma unroll
  for (int m = 0; m < 2; m++)
#pragma unroll
    for (int ks = 0; ks < F::KS; ks++) kf[m][ks] = global_frag(kbase + jc * a.k_stride[1] + m * a.k_stride[3], valid, ks * 16 + 8 * h, a.d);
  if (X::VLDS) {
    Loader<F::VROW, kRowWise> lv;
    const uint32_t vst = (uint32_t)(a.v_stride[1] * 2);
    lv.init(wave, lane, vst, a.dv);
#pragma unroll
    for (int x = 0; x < kRows / kBlk; x++)
      lv.load(reinterpret_cast<const char*>(vbase) + (j0 + x * kBlk) * (int64_t)vst, len - j0 - x * kBlk, vst, a.dv, base0 + 2 * STAGE + x * kBlk * F::VROW);
  } else if (OUT & 1) {
#pragma unroll
    for (int ks = 0; ks < F::VS; ks++) vf[ks] = global_frag(vbase + jc * a.v_stride[1], valid, ks * 16 + 8 * h, a.dv);
  }

  f32x16 adk[2][F::KC], adv[F::VC];
#pragma unroll
  for (int cb = 0; cb < F::KC; cb++) { adk[0][cb] = zero16(); adk[1][cb] = zero16(); }
#pragma unroll
  for (int cb = 0; cb < F::VC; cb++) adv[cb] = zero16();

  const uint32_t qst = (uint32_t)(a.q_stride[1] * 2), gst = (uint32_t)a.H * a.dv * 2;
  Loader<F::KROW, kBothWays, ROWS> lq;
  Loader<F::VROW, kBothWays, ROWS> lg;
  lq.init(wave, lane, qst, a.d);
  lg.init(wave, lane, gst, a.dv);
  // first query that sees key j: i >= j + NQ - len
  const int shift = a.causal ? a.NQ - len : -a.NK - 1;
  const int first = max(0, (j0 + shift) / ROWS), nblk = j0 < len ? (a.NQ + ROWS - 1) / ROWS : 0;
  // the staged queries: running (scalar) addresses, set anew for every head of the group
  const char *q0 = nullptr, *q1 = nullptr, *go = nullptr;
  const float* four = nullptr;
  float weight = 0.f;
  int left = 0;
  auto seek = [&](int g, int blk) {
    const int head = hk * P.G + g;
    const int64_t row = (int64_t)blk * ROWS;
    q0 = reinterpret_cast<const char*>(static_cast<const uint16_t*>(a.q) + b * a.q_stride[0] + head * a.q_stride[2]) + row * qst;
    q1 = q0 + a.q_stride[3] * 2;
    go = reinterpret_cast<const char*>(static_cast<const uint16_t*>(a.dout) + ((size_t)b * a.NQ * a.H + head) * a.dv) + row * gst;
    four = P.rows4 + ((size_t)(b * a.H + head) * 4 + wave) * a.NQ + row;
    left = a.NQ - (int)row;
    weight = a.lam[head];
  };
  auto fetch = [&](uint32_t st) {
    lq.load(q0, left, qst, a.d, st);
    lq.load(q1, left, qst, a.d, st + X::KB);
    lg.load(go, left, gst, a.dv, st + 2 * X::KB);
    // a wave each: the four floats of a query.  ROWS floats, then zeros (also past the last query), 64 in all
    load_to_lds4(buffer_at(four, min(ROWS, left) * 4), lane * 4, st + 2 * X::KB + X::VB + wave * kBlk * 4);
    q0 += ROWS * qst;
    q1 += ROWS * qst;
    go += ROWS * gst;
    four += ROWS;
    left -= ROWS;
  };
  const uint32_t qra = base0 + row_addr<F::KROW, kBothWays>(lane), qca = base0 + col_addr<F::KROW, kBothWays>(lane, 0);
  const uint32_t gra = base0 + 2 * X::KB + row_addr<F::VROW, kBothWays>(lane), gca = base0 + 2 * X::KB + col_addr<F::VROW, kBothWays>(lane, 0);
  const uint32_t vra = base0 + 2 * STAGE + wave * 32 * F::VROW + row_addr<F::VROW, kRowWise>(lane);
  // this workgroup's share of the (head, block) steps
  const int per_head = nblk > first ? nblk - first : 0, steps = per_head * P.G;
  const int step0 = (int)((int64_t)steps * share / P.nsplit), step1 = (int)((int64_t)steps * (share + 1) / P.nsplit);
  int g = per_head > 0 ? step0 / per_head : 0, blk = first + step0 - g * per_head, odd = 0;
  if (step0 < step1) {
    seek(g, blk);
    fetch(base0);
  }
  for (int step = step0; step < step1; step++) {
    tile_ready();                                          // (and a new head's weight with it)
    const float sgn = weight > 0.f ? -1.f : 1.f;
    const int i_blk = blk * ROWS;
    const bool more = step + 1 < step1;
    if (++blk == nblk) {
      blk = first;
      g++;
      if (more) seek(g, blk);
    }
    if (more) fetch(base0 + (odd ^ 1) * STAGE);
    const uint32_t stage = odd * STAGE;
    odd ^= 1;
    if (i_blk + ROWS - 1 < w0 + shift) continue;           // no query of the block sees a key of this wave
#pragma unroll 1
    for (int ib = 0; ib < ROWS / 32; ib++) {
      const int i0 = i_blk + ib * 32;
      const uint32_t qr = qra + stage + ib * 32 * F::KROW, qc = qca + stage + ib * 32 * F::KROW;
      const uint32_t gr = gra + stage + ib * 32 * F::VROW, gc = gca + stage + ib * 32 * F::VROW;
      const float* vec = reinterpret_cast<const float*>(smem + stage + 2 * X::KB + X::VB) + ib * 32 + 4 * h;
      // the order keeps few values alive at once: scores and probabilities, their mix and dV, then dP, the score gradients and dK
      f32x16 s[2];
#pragma unroll
      for (int x = 0; x < F::KS; x += 2) {                 // (four LDS reads ahead of the matrix instructions: what the registers hold)
        bf16x8 q[2][2];
#pragma unroll
        for (int y = 0; y < 2; y++)
#pragma unroll
          for (int m = 0; m < 2; m++) q[m][y] = read_row((qr ^ ((x + y) << 5)) + m * X::KB);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int y = 0; y < 2; y++)
#pragma unroll
          for (int m = 0; m < 2; m++) s[m] = mfma(q[m][y], kf[m][x + y], x + y == 0 ? zero16() : s[m]);
      }
      // (priorities as in the dQ kernel; to the end of dP here: 656 against 617 us, with dV and dP in front of the others 638)
      __builtin_amdgcn_s_setprio(0);
      if (i0 < w0 + 31 + shift) {
        const int hidden = w0 + (lane & 31) + shift - i0 - 4 * h;      // this lane's key is seen from there on
#pragma unroll
        for (int e = 0; e < 16; e++) {
          s[0][e] = 8 * (e >> 2) + (e & 3) < hidden ? -INFINITY : s[0][e];
          s[1][e] = 8 * (e >> 2) + (e & 3) < hidden ? -INFINITY : s[1][e];
        }
      }
#pragma unroll
      for (int e4 = 0; e4 < 4; e4++) {
        const f32x4 L0 = *reinterpret_cast<const f32x4*>(vec + 8 * e4), L1 = *reinterpret_cast<const f32x4*>(vec + kBlk + 8 * e4);
#pragma unroll
        for (int x = 0; x < 4; x++) {
          s[0][4 * e4 + x] = __builtin_amdgcn_exp2f(s[0][4 * e4 + x] * P.c2 - L0[x]);
          s[1][4 * e4 + x] = __builtin_amdgcn_exp2f(s[1][4 * e4 + x] * P.c2 - L1[x]);
        }
      }
      if (OUT & 2) {
#pragma unroll
        for (int t = 0; t < 2; t++) {
          bf16x8 gt[F::VC];
#pragma unroll
          for (int cb = 0; cb < F::VC; cb++) gt[cb] = read_col_both<F::VROW>((gc ^ (cb << 6)) + t * 16 * F::VROW);
          __builtin_amdgcn_sched_barrier(0);
          const bf16x8 d = pack8_sum(s[0], s[1], sgn, 8 * t);
#pragma unroll
          for (int cb = 0; cb < F::VC; cb++) adv[cb] = mfma(gt[cb], d, adv[cb]);
        }
      }
      if (OUT & 1) {
        f32x16 dp;                                         // dP - delta1
#pragma unroll
        for (int e4 = 0; e4 < 4; e4++) {
          const f32x4 D = *reinterpret_cast<const f32x4*>(vec + 2 * kBlk + 8 * e4);
#pragma unroll
          for (int x = 0; x < 4; x++) dp[4 * e4 + x] = D[x];
        }
#pragma unroll
        for (int x = 0; x < F::VS; x += 2) {
          bf16x8 gg[2], vv[2];
#pragma unroll
          for (int y = 0; y < 2; y++) {
            gg[y] = read_row(gr ^ ((x + y) << 5));
            vv[y] = X::VLDS ? read_row(vra ^ ((x + y) << 5)) : vf[X::VLDS ? 0 : x + y];
          }
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int y = 0; y < 2; y++) dp = mfma(gg[y], vv[y], dp);
        }
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int e4 = 0; e4 < 4; e4++) {
          const f32x4 E = *reinterpret_cast<const f32x4*>(vec + 3 * kBlk + 8 * e4);
#pragma unroll
          for (int x = 0; x < 4; x++) {
            s[0][4 * e4 + x] *= dp[4 * e4 + x];
            s[1][4 * e4 + x] *= dp[4 * e4 + x] * sgn + E[x];
          }
        }
#pragma unroll
        for (int t = 0; t < 2; t++) {
          bf16x8 qt[2][F::KC];
#pragma unroll
          for (int m = 0; m < 2; m++)
#pragma unroll
            for (int cb = 0; cb < F::KC; cb++) qt[m][cb] = read_col_both<F::KROW>((qc ^ (cb << 6)) + m * X::KB + t * 16 * F::KROW);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int m = 0; m < 2; m++) {
            const bf16x8 d = pack8(s[m], 8 * t);
#pragma unroll
            for (int cb = 0; cb < F::KC; cb++) adk[m][cb] = mfma(qt[m][cb], d, adk[m][cb]);
          }
        }
      }
    }
  }
  if (j >= a.NK) return;
  // keys behind the sample's length: zeros (their columns hold whatever the zero-filled operands gave)
  const size_t key = ((size_t)b * a.NK + j) * a.HK + hk, keys = (size_t)a.B * a.NK * a.HK;
  auto put = [&](void* out, float* part, int c, const f32x16& v, int e, float f) {
    f32x4 x = {v[4 * e] * f, v[4 * e + 1] * f, v[4 * e + 2] * f, v[4 * e + 3] * f};
    if (!valid) x = f32x4{0.f, 0.f, 0.f, 0.f};
    if (P.nsplit > 1) *reinterpret_cast<f32x4*>(part + c) = x;
    else *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(out) + c) = cvt_bf16x4(x);
  };
  uint16_t* dk = static_cast<uint16_t*>(a.dk) + key * 2 * a.d;
  uint16_t* dv = static_cast<uint16_t*>(a.dv_out) + key * a.dv;
  float* pk = P.part + ((size_t)share * keys + key) * 2 * a.d;
  float* pv = P.part + (size_t)P.nsplit * keys * 2 * a.d + ((size_t)share * keys + key) * a.dv;
#pragma unroll
  for (int e = 0; e < 4; e++) {
#pragma unroll
    for (int m = 0; m < ((OUT & 1) ? 2 : 0); m++)
#pragma unroll
      for (int cb = 0; cb < F::KC; cb++)
        if (cb * 32 + 8 * e + 4 * h < a.d) put(dk + m * a.d, pk + m * a.d, cb * 32 + 8 * e + 4 * h, adk[m][cb], e, a.scale);
#pragma unroll
    for (int cb = 0; cb < ((OUT & 2) ? F::VC : 0); cb++)
      if (cb * 32 + 8 * e + 4 * h < a.dv) put(dv, pv, cb * 32 + 8 * e + 4 * h, adv[cb], e, 1.f);
  }
}

// ---------------------------------------------------------------------------------------------------------------------------
bool misaligned(const void* p) { return p == nullptr || (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

int form_of(const gc_diff_attention* a) { return a->d <= 32 && a->dv <= 64 ? 0 : (a->d <= 64 && a->dv <= 128 ? 1 : 2); }
constexpr int kDV[3] = {64, 128, 256};

int check_desc(const gc_diff_attention* a, bool backward) {
  if (a == nullptr) { set_error("differential attention: null descriptor"); return GC_BAD_ARGUMENT; }
  if (a->B < 0 || a->NQ < 0 || a->NK < 0 || a->H <= 0 || a->HK <= 0 || a->H % a->HK != 0 || a->d <= 0 || a->d > 128 || a->d % 8 != 0 || a->dv <= 0 ||
      a->dv > 256 || a->dv % 8 != 0) {
    set_error("differential attention: supported are d %% 8 == 0 up to 128, dv %% 8 == 0 up to 256, H a multiple of HK (got B=%d NQ=%d NK=%d H=%d HK=%d d=%d dv=%d)",
              a->B, a->NQ, a->NK, a->H, a->HK, a->d, a->dv);
    return GC_UNSUPPORTED_GEOMETRY;
  }
  const int64_t G = a->H / a->HK;
  const int64_t tiles = (int64_t)a->B * a->H * (((int64_t)(a->NQ > a->NK ? a->NQ : a->NK) + kRows - 1) / kRows);
  if (G * a->NQ >= (1ll << 30) || a->NK >= (1 << 30) || tiles * 64 >= (1ll << 31)) {
    set_error("differential attention: too many rows (B=%d NQ=%d NK=%d H=%d)", a->B, a->NQ, a->NK, a->H);
    return GC_UNSUPPORTED_GEOMETRY;
  }
  if (!(a->scale >= 1e-30f) || a->scale > 1e30f) { set_error("differential attention: scale must be positive and finite (1e-30 to 1e30)"); return GC_BAD_ARGUMENT; }
  for (int i = 0; i < 4; i++)
    if (a->q_stride[i] % 8 != 0 || a->k_stride[i] % 8 != 0 || (i < 3 && a->v_stride[i] % 8 != 0)) {
      set_error("differential attention: strides must be multiples of 8 elements");
      return GC_BAD_ARGUMENT;
    }
  const int64_t widest = 1ll << 23;       // elements: 64 rows stay below 2^30 bytes
  if (a->q_stride[1] < a->d || a->k_stride[1] < a->d || a->v_stride[1] < a->dv || a->q_stride[1] >= widest || a->k_stride[1] >= widest || a->v_stride[1] >= widest ||
      (int64_t)a->H * a->dv >= widest) {
    set_error("differential attention: rows must not overlap and row strides must be below 2^23 elements");
    return GC_UNSUPPORTED_GEOMETRY;
  }
  const void* base[] = {a->q, a->k, a->v, a->out};
  for (const void* p : base)
    if (misaligned(p)) { set_error("differential attention: q, k, v and out must be non-null and 16-byte aligned"); return GC_BAD_ARGUMENT; }
  if (a->lam == nullptr || (a->out2 != nullptr && misaligned(a->out2))) { set_error("differential attention: lam is null or out2 misaligned"); return GC_BAD_ARGUMENT; }
  if (backward) {
    const void* more[] = {a->out2, a->dout, a->dq, a->dk, a->dv_out};
    for (const void* p : more)
      if (misaligned(p)) { set_error("differential attention backward: out2, dout, dq, dk, dv must be non-null and 16-byte aligned"); return GC_BAD_ARGUMENT; }
    if (a->lse == nullptr || a->dlam == nullptr) { set_error("differential attention backward: lse and dlam must not be null"); return GC_BAD_ARGUMENT; }
  }
  return GC_OK;
}

// Whether and how far the keys of a row are split.
// Shares of a backward walk of `steps` blocks by `groups` workgroups: as many as give every CU one workgroup, at least 4 blocks each, or two
// workgroups per CU where these still have `least` blocks each and the registers hold two.  Two at a time walk only 1.2 times as fast as
// one, and their results are twice the work to add.  With the forward pass, us: N 3000, 8 heads 335 in one share, 307 in two; N 4096, one
// head 142 in 16 shares of 4, 124 in 8; 4 x 1024, 8 heads 170 in two shares of 8, 146 in one.
int64_t shares_of(const gc_diff_attention* a, int64_t groups, int64_t steps, int64_t least) {
  if (groups <= 0) return 1;
  const int64_t cus = device_cu_count();
  int64_t n = std::min(cus / groups, steps / 4);
  if (form_of(a) < 2) n = std::max(n, std::min(2 * cus / groups, steps / least));
  return std::max<int64_t>(n, 1);
}
void plan_forward(const gc_diff_attention* a, DiffParams& P) {
  P.a = *a;
  P.G = a->H / a->HK;
  const int64_t R = (int64_t)P.G * a->NQ, cus = device_cu_count(), heads = (int64_t)a->B * a->HK;
  P.tiles = (int)((R + kRows - 1) / kRows);
  P.div_nq = make_fastdiv((uint32_t)a->NQ);
  P.c2 = a->scale * 1.44269504088896340736f;
  P.lazy = kLazy / P.c2;
  const int form = form_of(a);
  // Up to 32 rows: the kernel for few rows, measured beside the general one with its shares (one query, us).  64 wide it is ahead from 64
  // keys on (1 head x 256 keys 8 and 10, 512 x 64 10 and 13, 64 x 16384 52 and 69), 128 wide ahead or level (1 x 256 12 and 13, 64 x 1024
  // 18 and 26, 512 x 256 29 and 33, 64 x 4096 32 and 31, 16 heads of interleaved keys x 65536 110 and 121), 256 wide ahead in walks of 256
  // to 512 keys that run at once (64 x 512 20 and 35, 1 x 256 17 and 22; 1 x 128 19 and 16, 1 x 16384 40 and 32, 512 x 256 53 and 48).
  P.few = R <= 32 && (form < 2 ? a->NK >= 64 : a->NK >= 256 && a->NK <= 512 && heads <= cus);
  int64_t n = 1;
  if (P.few) {
    // one workgroup per CU (two of the narrow form, whose stages are half as large), every wave a share of at least two tiles
    const int nw = form == 2 ? 2 : 4;
    const int64_t tiles32 = ((int64_t)a->NK + 31) / 32;
    n = cus * (form == 0 ? 2 : 1) / (heads > 0 ? heads : 1);
    if (n > kMaxShares) n = kMaxShares;
    if (n > tiles32 / 2 / nw) n = tiles32 / 2 / nw;
    if (n < 1) n = 1;
    P.nsplit = (int)n;
    P.blocks_per_split = (int)((tiles32 + n * nw - 1) / (n * nw));
    return;
  }
  // As many shares as give every CU one workgroup, where that saves more blocks of a walk than the join costs: about 5 blocks' time and
  // one more for every 15 workgroups whose rows it reads, in the widest form, whose blocks take three times as long, 3 and one for 28
  // (64/128: N 4096, one head 68 us unsplit, 34 in 8 shares; 4 heads 77 and 67 in two; N 1024, 8 heads 27 and 36 in 4; 128/256: 61, 46).
  const int64_t nblk = ((int64_t)a->NK + kBlk - 1) / kBlk, groups = heads * P.tiles;
  n = groups > 0 ? std::min(cus / groups, nblk / 4) : 1;
  if (n > 1 && nblk - nblk / n < (form < 2 ? 5 + groups * n / 15 : 3 + groups * n / 28)) n = 1;
  if (n > 256) n = 256;
  if (n < 1) n = 1;
  P.blocks_per_split = (int)((nblk + n - 1) / n);
  if (P.blocks_per_split < 1) P.blocks_per_split = 1;
  P.nsplit = (int)((nblk + P.blocks_per_split - 1) / P.blocks_per_split);
  if (P.nsplit < 1) P.nsplit = 1;
}
// Which forward kernel, by the length of a workgroup's walk: halves that take turns start and join slower than four waves, and walk faster,
// above all where a CU has one workgroup.  Measured, us by turns and by four waves, 8 heads of 64/128, N x N:
//   at most one workgroup per CU   N 128: 16 and 12,  256: 18.3 and 16.3,  512: 23.1 and 24.5,  1024: 33 and 39,  2048: 55 and 76
//   8 per CU                       N 128: 119 and 68, 256: 126 and 81,  512: 161 and 124,  1024: 242 and 212,  2048: 415 and 409 (causal 266
//                                  and 258; 4 per CU 209 and 210, causal 139 and 157),  4096 (4 per CU): 381 and 403, causal 217 and 246
//   32/64, whose blocks are half as long, 4 to 8 per CU: 1024: 163 and 139, 2048: 280 and 266, 4096: 263 and 260, causal 152 and 165
bool takes_turns(const DiffParams& P, int form) {
  const int64_t groups = (int64_t)P.a.B * P.a.HK * P.tiles * P.nsplit;
  return form < 2 && P.blocks_per_split >= (groups <= device_cu_count() ? 8 : (form == 0 ? 64 : 32));
}
size_t forward_bytes(const DiffParams& P, int DV) {
  if (P.nsplit <= 1) return 0;
  const size_t rows = (size_t)P.nsplit * P.a.B * P.a.HK * P.G * P.a.NQ;
  return rows * (4 + 2 * (size_t)DV) * sizeof(float);
}
// The backward kernels' shares: of the keys of a query tile (dq), of the queries of a key tile (dkv).  A grid that fills the chip takes
// one share and stores its result; otherwise the shares' fp32 partial results are added by diff_sum_kernel.  Causal key tiles differ in
// length: in long walks dkv takes twice as many workgroups as run at a time (8192, 16 heads on 4, forward and backward: 1653 us with as
// many, 1446 with twice as many; 2048, where that leaves 8 blocks a share: 215 and 250), and 6 blocks are enough for a share where the grid
// has room (6 x 777, 6 heads on 2 of 32/64: 32 us in 3 shares, 23 in 6).
struct BackwardPlan {
  int dq_tiles, dq_shares, dq_blocks, dq_turns, dkv_tiles, dkv_shares;
  size_t delta, rows4, lampart, part;                      // floats
};
BackwardPlan plan_backward(const gc_diff_attention* a) {
  BackwardPlan p{};
  const int64_t cus = device_cu_count(), nkb = ((int64_t)a->NK + kBlk - 1) / kBlk, nqb = ((int64_t)a->NQ + kBlk - 1) / kBlk, G = a->H / a->HK;
  p.dq_tiles = (a->NQ + kRows - 1) / kRows;
  p.dkv_tiles = (a->NK + kRows - 1) / kRows;
  const int64_t dq_groups = (int64_t)a->B * a->H * p.dq_tiles;
  int64_t n = dq_groups > 0 ? std::max<int64_t>(1, std::min(cus / dq_groups, nkb / 4)) : 1;
  p.dq_turns = form_of(a) < 2 && dq_groups <= cus && 4 * dq_groups > cus && nkb / n >= 12;
  if (!p.dq_turns) n = shares_of(a, dq_groups, nkb, 10);
  p.dq_blocks = (int)((nkb + n - 1) / n);
  p.dq_shares = (int)((nkb + p.dq_blocks - 1) / p.dq_blocks);
  const int64_t groups = (int64_t)a->B * a->HK * p.dkv_tiles, steps = G * nqb;
  n = shares_of(a, groups, steps, a->causal && 4 * groups <= 3 * cus ? 6 : 10);
  if (a->causal && n < std::min(4 * cus / groups, steps / 16)) n = std::min(4 * cus / groups, steps / 16);
  if (n > 64) n = 64;
  p.dkv_shares = n < 2 ? 1 : (int)n;
  const size_t rows = (size_t)a->B * a->H * a->NQ, keys = (size_t)a->B * a->HK * a->NK;
  p.delta = (rows * 2 + 3) / 4 * 4;
  p.rows4 = rows * 4;
  p.lampart = ((size_t)a->B * a->H * p.dq_tiles * p.dq_shares + 3) / 4 * 4;
  const size_t dq = p.dq_shares > 1 ? (size_t)p.dq_shares * rows * 2 * a->d : 0, dkv = p.dkv_shares > 1 ? (size_t)p.dkv_shares * keys * (2 * a->d + a->dv) : 0;
  p.part = dq > dkv ? dq : dkv;                            // (used one after the other)
  return p;
}
size_t backward_bytes(const BackwardPlan& p) { return (p.delta + p.rows4 + p.lampart + p.part) * sizeof(float); }

template <int DK, int DV>
int launch_fwd(const DiffParams& P, hipStream_t s) {
  typedef Cfg<DK, DV> F;
  constexpr int lds = 2 * (2 * F::KB + F::VB);
  if (int e = ensure_dynamic_smem(reinterpret_cast<const void*>(diff_fwd_kernel<DK, DV>), lds)) return e;
  hipLaunchKernelGGL((diff_fwd_kernel<DK, DV>), dim3((unsigned)P.a.B * P.a.HK * P.tiles * P.nsplit), dim3(kThreads), lds, s, P);
  return check_hip(hipGetLastError(), "diff_fwd launch");
}
template <int DK, int DV>
int launch_turns(const DiffParams& P, hipStream_t s) {
  typedef TurnsCfg<DK, DV> X;
  if (int e = ensure_dynamic_smem(reinterpret_cast<const void*>(diff_fwd_turns_kernel<DK, DV>), X::LDS)) return e;
  hipLaunchKernelGGL((diff_fwd_turns_kernel<DK, DV>), dim3((unsigned)P.a.B * P.a.HK * P.tiles * P.nsplit), dim3(X::NW * 64), X::LDS, s, P);
  return check_hip(hipGetLastError(), "diff_fwd launch");
}
template <int DK, int DV>
int launch_few(const DiffParams& P, hipStream_t s) {
  typedef FewCfg<DK, DV> X;
  constexpr int lds = X::NW * 2 * X::STAGE;
  if (int e = ensure_dynamic_smem(reinterpret_cast<const void*>(diff_few_rows_kernel<DK, DV>), lds)) return e;
  hipLaunchKernelGGL((diff_few_rows_kernel<DK, DV>), dim3((unsigned)P.a.B * P.a.HK * P.nsplit), dim3(X::NW * 64), lds, s, P);
  return check_hip(hipGetLastError(), "diff_few_rows launch");
}
template <int DK, int DV>
int launch_dq(const DiffParams& P, hipStream_t s) {
  typedef Cfg<DK, DV> F;
  constexpr int lds = 2 * (2 * F::KB + F::VB);
  if (int e = ensure_dynamic_smem(reinterpret_cast<const void*>(diff_bwd_dq_kernel<DK, DV>), lds)) return e;
  hipLaunchKernelGGL((diff_bwd_dq_kernel<DK, DV>), dim3((unsigned)P.a.B * P.a.H * P.tiles * P.nsplit), dim3(kThreads), lds, s, P);
  return check_hip(hipGetLastError(), "diff_bwd_dq launch");
}
int launch_sum(const float* part, int shares, void* out0, size_t n0, void* out1, size_t n1, hipStream_t s) {
  hipLaunchKernelGGL(diff_sum_kernel, dim3((unsigned)(((n0 + n1) / 4 + kThreads - 1) / kThreads)), dim3(kThreads), 0, s, part, shares, (uint16_t*)out0, n0,
                     (uint16_t*)out1, n1);
  return check_hip(hipGetLastError(), "diff_sum launch");
}
template <int DK, int DV>
int launch_dq_turns(const DiffParams& P, hipStream_t s) {
  typedef TurnsCfg<DK, DV> X;
  if (int e = ensure_dynamic_smem(reinterpret_cast<const void*>(diff_bwd_dq_turns_kernel<DK, DV>), X::RING)) return e;
  hipLaunchKernelGGL((diff_bwd_dq_turns_kernel<DK, DV>), dim3((unsigned)P.a.B * P.a.H * P.tiles * P.nsplit), dim3(X::NW * 64), X::RING, s, P);
  return check_hip(hipGetLastError(), "diff_bwd_dq launch");
}
template <int DK, int DV, int OUT>
int launch_dkv(const DiffParams& P, hipStream_t s) {
  constexpr int lds = DkvCfg<DK, DV, OUT>::LDS;
  if (int e = ensure_dynamic_smem(reinterpret_cast<const void*>(diff_bwd_dkv_kernel<DK, DV, OUT>), lds)) return e;
  hipLaunchKernelGGL((diff_bwd_dkv_kernel<DK, DV, OUT>), dim3((unsigned)P.a.B * P.a.HK * P.tiles * P.nsplit), dim3(kThreads), lds, s, P);
  return check_hip(hipGetLastError(), "diff_bwd_dkv launch");
}

}  // namespace
}  // namespace gc

using namespace gc;

extern "C" size_t gc_diff_attention_workspace_bytes(const gc_diff_attention* desc, int backward) {
  if (desc == nullptr || desc->B <= 0 || desc->NQ <= 0 || desc->H <= 0 || desc->HK <= 0 || desc->H % desc->HK != 0) return 0;
  if (backward) return desc->NK > 0 ? backward_bytes(plan_backward(desc)) : 0;
  DiffParams P{};
  plan_forward(desc, P);
  return forward_bytes(P, kDV[form_of(desc)]);
}

extern "C" int gc_diff_attention_fwd(const gc_diff_attention* desc, void* workspace, size_t workspace_bytes, void* stream) {
  if (int e = check_desc(desc, false)) return e;
  if (desc->B == 0 || desc->NQ == 0) return GC_OK;
  DiffParams P{};
  plan_forward(desc, P);
  const int form = form_of(desc), DV = kDV[form];
  const size_t need = forward_bytes(P, DV);
  if (need > 0 && (misaligned(workspace) || workspace_bytes < need)) {
    set_error("differential attention: a 16-byte aligned workspace of %zu bytes is needed", need);
    return GC_WORKSPACE_TOO_SMALL;
  }
  const size_t rows = (size_t)P.nsplit * desc->B * desc->HK * P.G * desc->NQ;
  P.ml = static_cast<float*>(workspace);
  P.part = need > 0 ? P.ml + rows * 4 : nullptr;
  hipStream_t s = (hipStream_t)stream;
  {
    ProfScope ps(P.few ? "gc::diff_few_rows_kernel" : "gc::diff_fwd_kernel", 4.0 * desc->B * desc->H * (double)desc->NQ * desc->NK * (desc->d + desc->dv), s);
    int e;
    if (P.few) e = form == 0 ? launch_few<32, 64>(P, s) : (form == 1 ? launch_few<64, 128>(P, s) : launch_few<128, 256>(P, s));
    else if (takes_turns(P, form)) e = form == 0 ? launch_turns<32, 64>(P, s) : launch_turns<64, 128>(P, s);
    else e = form == 0 ? launch_fwd<32, 64>(P, s) : (form == 1 ? launch_fwd<64, 128>(P, s) : launch_fwd<128, 256>(P, s));
    if (e) return e;
  }
  if (P.nsplit > 1) {
    const size_t out_rows = (size_t)desc->B * desc->H * desc->NQ;
    if (P.nsplit > kFewShares) hipLaunchKernelGGL(diff_join_kernel, dim3((unsigned)out_rows), dim3(kJoinThreads), 0, s, P, DV);
    else if (form == 0) hipLaunchKernelGGL(diff_join_rows_kernel<64>, dim3((unsigned)((out_rows + 15) / 16)), dim3(kThreads), 0, s, P);
    else if (form == 1) hipLaunchKernelGGL(diff_join_rows_kernel<128>, dim3((unsigned)((out_rows + 7) / 8)), dim3(kThreads), 0, s, P);
    else hipLaunchKernelGGL(diff_join_rows_kernel<256>, dim3((unsigned)((out_rows + 3) / 4)), dim3(kThreads), 0, s, P);
    return check_hip(hipGetLastError(), "diff_join launch");
  }
  return GC_OK;
}

extern "C" int gc_diff_attention_bwd(const gc_diff_attention* desc, void* workspace, size_t workspace_bytes, void* stream) {
  if (int e = check_desc(desc, true)) return e;
  if (desc->B == 0 || desc->NQ == 0 || desc->NK == 0) {
    set_error("differential attention backward: an empty tensor has no gradient to compute");
    return GC_BAD_ARGUMENT;
  }
  const BackwardPlan plan = plan_backward(desc);
  const size_t need = backward_bytes(plan);
  if (misaligned(workspace) || workspace_bytes < need) {
    set_error("differential attention backward: a 16-byte aligned workspace of %zu bytes is needed", need);
    return GC_WORKSPACE_TOO_SMALL;
  }
  DiffParams P{};
  plan_forward(desc, P);
  const size_t rows = (size_t)desc->B * desc->H * desc->NQ, keys = (size_t)desc->B * desc->HK * desc->NK;
  P.delta = static_cast<float*>(workspace);
  P.rows4 = P.delta + plan.delta;
  P.lampart = P.rows4 + plan.rows4;
  P.part = P.lampart + plan.lampart;
  hipStream_t s = (hipStream_t)stream;
  const int form = form_of(desc);
  const double pairs = (double)desc->B * desc->H * desc->NQ * desc->NK;
  hipLaunchKernelGGL(diff_delta_kernel, dim3((unsigned)((rows * 16 + kThreads - 1) / kThreads)), dim3(kThreads), 0, s, P);
  if (check_hip(hipGetLastError(), "diff_delta launch")) return GC_HIP_ERROR;
  P.tiles = plan.dkv_tiles;
  P.nsplit = plan.dkv_shares;
  {
    ProfScope ps("gc::diff_bwd_dkv_kernel", pairs * (8.0 * desc->d + 4.0 * desc->dv), s);
    int e = form == 0 ? launch_dkv<32, 64, 3>(P, s) : (form == 1 ? launch_dkv<64, 128, 3>(P, s) : launch_dkv<128, 256, 1>(P, s));
    if (e == GC_OK && form == 2) e = launch_dkv<128, 256, 2>(P, s);
    if (e) return e;
  }
  if (P.nsplit > 1)
    if (int e = launch_sum(P.part, P.nsplit, desc->dk, keys * 2 * desc->d, desc->dv_out, keys * desc->dv, s)) return e;
  P.tiles = plan.dq_tiles;
  P.nsplit = plan.dq_shares;
  P.blocks_per_split = plan.dq_blocks;
  {
    ProfScope ps("gc::diff_bwd_dq_kernel", pairs * (8.0 * desc->d + 2.0 * desc->dv), s);
    int e;
    if (plan.dq_turns) e = form == 0 ? launch_dq_turns<32, 64>(P, s) : launch_dq_turns<64, 128>(P, s);
    else e = form == 0 ? launch_dq<32, 64>(P, s) : (form == 1 ? launch_dq<64, 128>(P, s) : launch_dq<128, 256>(P, s));
    if (e) return e;
  }
  if (P.nsplit > 1)
    if (int e = launch_sum(P.part, P.nsplit, desc->dq, rows * 2 * desc->d, nullptr, 0, s)) return e;
  hipLaunchKernelGGL(diff_dlam_kernel, dim3(desc->H), dim3(kThreads), 0, s, P);
  return check_hip(hipGetLastError(), "diff_dlam launch");
}
