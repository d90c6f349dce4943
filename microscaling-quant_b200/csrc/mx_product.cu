// Products of packed MX operands with their epilogue, dense and by expert:
//
//   acc[r, n] = sum_k x[r, k] w[n, k] 2^(sx[r, k/32] - 127) 2^(sw[n, k/32] - 127)        (float32, tensor cores)
//   y = act(acc + bias) (* up) + residual,  written as float32 / bf16 / f16 or packed again (32 columns per scale)
//
// x and w are row-major codes with blocks of 32 along K, as block.*.quantize_packed(axis=-1) writes them. sm_100's
// tcgen05.mma kind::mxf8f6f4 multiplies them as they are: codes and E8M0 bytes go from memory to shared memory to the
// tensor core, nothing is dequantized. The products are exact and the sums are held in float32 in TMEM, which the instruction cuts
// toward zero at every addition, where a float32 multiply-add rounds: the error against 64 bits is 6.0e-8, 1.1e-7, 2.2e-7 and
// 5.0e-7 of the norm at K = 1024, 2048, 4096 and 8192 (multiply-adds: 4.1e-8, 5.9e-8, 8.4e-8, 1.25e-7; three quarters of it a
// mean that makes the sums smaller; where K is split over a cluster, 8.3e-8 at 8192). There is no other accumulator.
//
// Two kernels share the operand staging:
//   k_mx_tile  256 rows of x by 256 rows of w per pair of CTAs, persistent, for many rows: the operations bound it.
//   k_mx_rows  128 rows of w by 16-64 rows of x per CTA, K split over a cluster, for few rows: reading w bounds it.
#include "common.cuh"
#include "mx_codes.cuh"
#include "mx_layout.cuh"
#include "tc.cuh"

#include <cooperative_groups.h>

namespace cg = cooperative_groups;
using namespace mxq;

namespace {

enum { kActNone = 0, kActRelu, kActGelu, kActGeluTanh, kActSilu, kActSwiglu, kActGeglu };
enum { kOutF32 = 0, kOutBf16, kOutF16, kOutPacked };

struct Args {
  const uint8_t *sx, *sw;      // E8M0 bytes, nb per row
  int nb;
  int sx_pitch, sw_pitch;      // bytes between the rows of sx and sw; what is behind a row's nb is 0 or never read
  int vec;                     // scale bytes are read 16, 4 or 1 at a time (alignment and the pitches allow it)
  const int32_t *offsets, *order;
  int experts;                 // 0: dense
  int per;                     // > 0: row r of the product is row order[r] / per of x
  int rows, xrows;             // rows of the product, rows of x
  int n, width;                // rows of w (per expert), columns of y
  int kblocks;                 // steps of 128 along K
  uint32_t idesc;
  uint32_t xbytes, wbytes;     // what one row of a stage's tile counts on the barrier
  const float* bias;
  const void* residual;
  int64_t residual_stride;
  void* out;
  uint8_t* out_scales;
  int64_t out_pitch, out_nb;
  int act, otype, ofmt;
  int vec_out;                 // y's (and the residual's) rows take 16-byte accesses
  int map_out;                 // k_mx_tile: whole staged rows of y leave by TMA
  unsigned* status;
  int64_t wait_cycles;
};

// ------------------------------------------------------------------------------------------ epilogue values
// A packed output turns an error of float32 into a whole step of the code where it meets a tie, so the epilogue keeps
// float32's accuracy relative to the result, in the tails too: within 16 units of 2^-24 by the sum of its roundings (the hardware's
// exp2 is good to 2^-22.5, its reciprocal to 2^-23), down to the smallest normal number. What an exponent's rounding loses,
// which its size multiplies, is carried: exp(a) = exp2(hi) (1 + r), hi = a log2(e) rounded, r = a - hi ln(2) by
// multiply-adds, ln(2) in two parts (Cody and Waite's reduction). Without the carrying the tails were 24 to 270 units off; it
// shows where K is short: 8192 x 8192 x 256 to bf16 takes 90 us with silu (87 without), 124 with gelu (107), 121 with gelu_tanh (95).
constexpr float kLog2E = 1.4426950408889634f, kLn2 = 0.6931471805599453f, kLn2Rest = (float)(0.6931471805599453 - (double)kLn2);
__device__ __forceinline__ float exp2_of(float x) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x));
  return e;
}
__device__ __forceinline__ float one_over(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// x / (1 + exp(t)) with exp(t) = 2^(2 hi) (1 + r), -100 <= t <= 93.9. The square and 2^-8 on both sides of the fraction keep what is
// left of a finite x to the last normal number (silu(-90) = -7.4e-38), where exp(t) itself would overflow; from t = 93 on the
// reciprocal is 0, and -Inf gives NaN, as -Inf * 0 does.
__device__ __forceinline__ float over_one_plus_exp(float x, float hi, float r) {
  constexpr float k = 0x1p-8f;
  const float h = exp2_of(hi);
  return x * k * one_over(__fmaf_rn(h * k, __fmaf_rn(h, r, h), k));
}
__device__ __forceinline__ float silu(float x) {
  const float t = fminf(fmaxf(-x, -100.0f), 93.5f), hi = t * (0.5f * kLog2E);
  return over_one_plus_exp(x, hi, __fmaf_rn(hi, -2.0f * kLn2Rest, __fmaf_rn(hi, -2.0f * kLn2, t)));
}
// x Phi(x). With z = |x| / sqrt(2) and t = 1 / (1 + z / 2), erfc(z) / 2 = t P(t) exp(-x^2 / 2), P a polynomial of degree
// 8 fitted here to the smallest relative error on 0 <= z <= 9.4 (4.2e-8, by iterated weighted least squares on
// Chebyshev points); Phi is that below zero and one minus that above. What x^2 / 2 loses in its own rounding is carried too.
__device__ __forceinline__ float gelu(float x) {
  const float a = fminf(fabsf(x), 19.5f), b = 0.5f * a, s = a * b, hi = s * -kLog2E;   // exp(-190) is 0
  const float t = one_over(__fmaf_rn(0.35355339059327376f, a, 1.0f));
  float e = exp2_of(hi);
  e = __fmaf_rn(e, __fmaf_rn(hi, -kLn2Rest, __fmaf_rn(hi, -kLn2, -s)) - __fmaf_rn(a, b, -s), e);
  float h = __fmaf_rn(t, -0.02942352555692196f, 0.14174368977546692f);
  h = __fmaf_rn(t, h, -0.24246817827224731f);
  h = __fmaf_rn(t, h, 0.13773120939731598f);
  h = __fmaf_rn(t, h, -0.012409592978656292f);
  h = __fmaf_rn(t, h, 0.10095827281475067f);
  h = __fmaf_rn(t, h, 0.12165011465549469f);
  h = __fmaf_rn(t, h, 0.14117400348186493f);
  h = __fmaf_rn(t, h, 0.1410439908504486f);
  h = h * t * e;
  return x * (x < 0.0f ? h : 1.0f - h);
}
// x (1 + tanh(u)) / 2 = x / (1 + exp(-2u)), u = sqrt(2 / pi) (x + 0.044715 x^3). -2u = x (k + m x^2) as a sum of two floats, with
// what each product's and sum's rounding left and the constants' own rest (k's head has 12 bits: the difference from it is exact)
__device__ __forceinline__ float gelu_tanh(float x) {
  constexpr float k = -1.595703125f, k_rest = (float)(-1.5957691216057308 - (double)k);
  constexpr float m = -0.07135481282609825f, m_rest = (float)(-0.07135481627260025 - (double)m);
  const float a = fminf(fmaxf(x, -10.28f), 10.28f), s = a * a;         // |t| is 93.9 there
  const float p = __fmaf_rn(s, m, k);
  float rest = __fmaf_rn(s, m, k - p) + k_rest;
  rest = __fmaf_rn(s, m_rest, __fmaf_rn(__fmaf_rn(a, a, -s), m, rest));
  const float t = a * p;
  rest = __fmaf_rn(a, rest, __fmaf_rn(a, p, -t));
  const float hi = t * (0.5f * kLog2E);
  return over_one_plus_exp(x, hi, __fmaf_rn(hi, -2.0f * kLn2, t) + __fmaf_rn(hi, -2.0f * kLn2Rest, rest));
}
// a NaN stays one
__device__ __forceinline__ float relu(float x) { return x < 0.0f ? 0.0f : x; }

// the switch outside the loop: one branch for all values
template <int N>
__device__ __forceinline__ void activate(int act, float (&v)[N]) {
  switch (act) {
    case kActRelu:
#pragma unroll
      for (int i = 0; i < N; i++) v[i] = relu(v[i]);
      break;
    case kActGelu:
    case kActGeglu:
#pragma unroll
      for (int i = 0; i < N; i++) v[i] = gelu(v[i]);
      break;
    case kActGeluTanh:
#pragma unroll
      for (int i = 0; i < N; i++) v[i] = gelu_tanh(v[i]);
      break;
    case kActSilu:
    case kActSwiglu:
#pragma unroll
      for (int i = 0; i < N; i++) v[i] = silu(v[i]);
      break;
    default: break;
  }
}

// ------------------------------------------------------------------------------------------ operand staging
constexpr int kMostExperts = 1024;
constexpr int kTileBytes = 128 * 128;                 // 128 rows of one K step

// 16 scale bytes of a row from K step 4g on (a step has 4): 0 beyond the row
__device__ __forceinline__ uint4 load_scales(const uint8_t* row, int g, int nb, int vec) {
  if (vec == 16) {                                     // the line and its neighbour come to L2 at the first touch
    uint4 v;
    asm volatile("ld.global.nc.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(row + (int64_t)g * 16));
    return v;
  }
  uint32_t w[4];
  if (vec == 4) {
#pragma unroll
    for (int j = 0; j < 4; j++)
      w[j] = g * 16 + j * 4 < nb ? __ldg(reinterpret_cast<const uint32_t*>(row + g * 16 + j * 4)) : 0u;
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  // rows at any byte: the aligned words that hold a byte of the row, shifted together; what is beyond the row is
  // cleared (a scale of the next row could be a NaN's)
  const uint8_t* from = row + (int64_t)g * 16;
  const int left = nb - g * 16, off = (int)(reinterpret_cast<uintptr_t>(from) & 3u);
  const uint32_t* words = reinterpret_cast<const uint32_t*>(from - off);
  uint32_t q[5];
#pragma unroll
  for (int j = 0; j < 5; j++) q[j] = 4 * j - off < left && 4 * j - off < 16 ? __ldg(words + j) : 0u;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    w[j] = __funnelshift_r(q[j], q[j + 1], 8 * off);
    const int have = left - 4 * j;
    if (have < 4) w[j] = have <= 0 ? 0u : w[j] & ((1u << (8 * have)) - 1u);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

struct Ring {
  int stage = 0;
  unsigned phase = 0;
  __device__ __forceinline__ void next(int stages) {
    if (++stage == stages) {
      stage = 0;
      phase ^= 1u;
    }
  }
};

// Scales on their way to a stage. The loader warp's lane holds, for each of G groups of 128 rows, the four rows lane,
// 32 + lane, 64 + lane and 96 + lane: their words stand side by side in the layout that copy_scales takes, so a step
// costs one 16-byte store per group.
template <int G>
struct ScaleRows {
  const uint8_t* row[4 * G];
  __device__ __forceinline__ void load(uint4 (&v)[4 * G], int g, const Args& a) const {
#pragma unroll
    for (int i = 0; i < 4 * G; i++) v[i] = load_scales(row[i], g, a.nb, a.vec);
  }
};
// step j of the four that v holds, to its place in the layout
template <int G>
__device__ __forceinline__ void put_words(const uint4 (&v)[4 * G], int j, uint8_t* to) {
  auto word = [j](const uint4& q) { return j == 0 ? q.x : j == 1 ? q.y : j == 2 ? q.z : q.w; };
#pragma unroll
  for (int i = 0; i < G; i++)
    *reinterpret_cast<uint4*>(to + (threadIdx.x & 31) * 16 + 512 * i) =
        make_uint4(word(v[4 * i]), word(v[4 * i + 1]), word(v[4 * i + 2]), word(v[4 * i + 3]));
}
// the same into the ring's next stage
template <int G>
__device__ __forceinline__ bool store_scales(const uint4 (&v)[4 * G], int j, const Args& a, uint8_t* area, int pitch, uint64_t* ready,
                                             uint64_t* empty, Ring& ring, int stages, const tc::Guard& guard) {
  if (!tc::wait_warp<false>(&empty[ring.stage], ring.phase ^ 1u, guard)) return false;
  put_words<G>(v, j, area + (size_t)ring.stage * pitch);
  __syncwarp();
  if (tc::elect()) tc::mbar_arrive(&ready[ring.stage]);
  ring.next(stages);
  return true;
}
// The words' way from the loader to the tensor core's view of shared memory, in a warp of its own: the fence waits
// for all that its thread has under way, and the loader has the next loads under way. far: the full barriers'
// shared::cluster address where they are in another CTA, else 0. Then the words are released to the cluster, which waits for
// everything that the SM has under way, about 1900 cycles a time.
__device__ __forceinline__ bool forward_scales(uint64_t* ready, uint64_t* full, uint32_t far, Ring& ring, int stages, const tc::Guard& guard) {
  if (!tc::wait_warp<false>(&ready[ring.stage], ring.phase, guard)) return false;
  if (tc::elect()) {
    fence_proxy_async();
    if (far) tc::mbar_arrive_remote(far + 8u * ring.stage);
    else tc::mbar_arrive(&full[ring.stage]);
  }
  __syncwarp();
  ring.next(stages);
  return true;
}

// where expert e's rows begin, whatever the offsets hold within the product's rows
__device__ __forceinline__ int row_begin(const Args& a, int e) { return min(max(a.offsets[e], 0), a.rows); }

// The experts' tiles in order, in shared memory: first[e] tiles are before expert e, whose rows begin at begin[e].
struct Table {
  int *first, *begin;
  __device__ __forceinline__ Table(void* at, int experts) : first(static_cast<int*>(at)), begin(first + experts + 1) {}
};
constexpr int table_bytes(int experts) { return 8 * (experts + 1); }

// one warp
__device__ void count_tiles(const Table& tab, const Args& a, int tile_rows, int per_row_tile) {
  const int lane = threadIdx.x & 31;
  int carry = 0;
  for (int base = 0; base < a.experts; base += 32) {
    const int e = base + lane;
    int t = 0;
    if (e < a.experts) {
      const int b = row_begin(a, e), c = row_begin(a, e + 1) - b;
      t = (c > 0 ? (c + tile_rows - 1) / tile_rows : 0) * per_row_tile;
      tab.begin[e] = b;
    }
    int s = t;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(~0u, s, d);
      if (lane >= d) s += up;
    }
    if (e < a.experts) tab.first[e + 1] = carry + s;
    carry += __shfl_sync(~0u, s, 31);
  }
  if (lane == 0) {
    tab.first[0] = 0;
    tab.begin[a.experts] = row_begin(a, a.experts);
  }
}

// Tile t: by expert, then column tile, then row tile, so that the CTAs at work at one time share w's tiles. Dense: row
// tiles in bands of 8 for the same reason.
struct Tile {
  int expert, row0, rows;              // its expert; first row of the product, rows of it in this tile
  int col;                     // column tile
  __device__ __forceinline__ void find(int t, const Args& a, const Table& tab, int tile_rows, int col_tiles) {
    if (a.experts == 0) {
      const int row_tiles = (a.rows + tile_rows - 1) / tile_rows;
      const int band = t / (kBand * col_tiles), in = t - band * kBand * col_tiles;
      const int high = min(kBand, row_tiles - band * kBand);
      expert = 0;
      col = in / high;
      row0 = (band * kBand + in % high) * tile_rows;
      rows = min(tile_rows, a.rows - row0);
      return;
    }
    int lo = 0, hi = a.experts;                        // first[lo] <= t < first[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (tab.first[mid] <= t) lo = mid; else hi = mid;
    }
    const int in = t - tab.first[lo], row_tiles = (tab.first[lo + 1] - tab.first[lo]) / col_tiles;
    expert = lo;
    col = in / row_tiles;
    row0 = tab.begin[lo] + (in - col * row_tiles) * tile_rows;
    rows = min(tile_rows, tab.begin[lo + 1] - row0);
  }
  static constexpr int kBand = 8;
};
// A warp's tiles one after the other: each lane finds one of the next 32, since a search takes about 1000 cycles
struct Tiles {
  Tile mine = {0, 0, 0, 0};
  int at = 0;
  // the tile `step` after the last one (the first: tile `from`), which exists
  __device__ __forceinline__ Tile next(int from, int step, int tiles, const Args& a, const Table& tab, int tile_rows, int col_tiles) {
    const int lane = threadIdx.x & 31;
    if (at == 0 && from + step * lane < tiles) mine.find(from + step * lane, a, tab, tile_rows, col_tiles);
    __syncwarp();
    Tile t;
    t.expert = __shfl_sync(~0u, mine.expert, at);
    t.row0 = __shfl_sync(~0u, mine.row0, at);
    t.rows = __shfl_sync(~0u, mine.rows, at);
    t.col = __shfl_sync(~0u, mine.col, at);
    at = (at + 1) & 31;
    return t;
  }
};
__device__ __forceinline__ int tile_count(const Args& a, const Table& tab, int tile_rows, int col_tiles) {
  return a.experts ? tab.first[a.experts] : (a.rows + tile_rows - 1) / tile_rows * col_tiles;
}

// the row of x that row r of the product is; a row beyond the tile stands for its last one and is never written
__device__ __forceinline__ int x_row(const Args& a, const Tile& t, int r) {
  r = t.row0 + min(r, t.rows - 1);
  if (a.per > 0) r = a.order[r] / a.per;
  return min(max(r, 0), a.xrows - 1);
}
__device__ __forceinline__ const uint8_t* w_scales(const Args& a, const Tile& t, int r) {
  return a.sw + ((int64_t)t.expert * a.n + min(r, a.n - 1)) * a.sw_pitch;
}

// ------------------------------------------------------------------------------------------------ many rows
// A pair of CTAs (cta_group::2) makes 256 rows by 256 features at a time: each holds 128 rows of x and half of the
// features of w, so that a stage brings 32 KB into each SM's shared memory and not the 48 KB of one CTA alone. Alone,
// the stage's arrival and the tensor core's reads are 192 bytes a cycle at the full rate, the shared memory moves
// 128; as a pair both are 128.
constexpr int kStages = 5;
constexpr int kStageBytes = 2 * kTileBytes;
// The scales come in groups of four steps (16 bytes of a row), in a ring of their own: the second CTA's words have to be
// released to the cluster, and a release for every step (about 1900 cycles, against the 512 of its products) doubled
// the kernel's time.
constexpr int kGroups = 4;
constexpr int kStepScales = 3 * 512;                   // x's 128 rows, all of w's 256
constexpr int kGroupScales = 4 * kStepScales;
constexpr int kWriters = 8;                            // epilogue warps
constexpr int kPassBytes = 32 * 128;                   // what one of them stages: 32 rows of 128 bytes

struct TileShared {
  uint64_t full[kStages], empty[kStages], acc_full, acc_free, last;
  uint64_t scales_ready[kGroups], scales_full[kGroups], scales_empty[kGroups];
  uint32_t tmem;
  int abort;
};
constexpr int kTileSmem = 1024 + kStages * kStageBytes + kGroups * kGroupScales + kWriters * kPassBytes + (int)sizeof(TileShared);

static_assert(kTileSmem + table_bytes(kMostExperts) <= 227 * 1024, "shared memory of a CTA");

// place of 16-byte piece j of a staged row: neighbouring rows in other banks
__device__ __forceinline__ uint8_t* piece(uint8_t* stage, int row, int j) { return stage + row * 128 + ((j ^ (row & 7)) << 4); }

// A warp's 32 staged rows to memory, `bytes` of each of the first `rows`. P: 16-byte pieces per staged row; vec:
// memory takes 16-byte accesses (then bytes is a multiple of 16), else it is written in elements of `size` bytes.
template <int P>
__device__ __forceinline__ void put_rows(uint8_t* stage, uint8_t* mem, int64_t pitch, int rows, int bytes, int size, bool vec) {
  const int lane = threadIdx.x & 31;
  if (vec) {
    const int j = lane % P, r0 = lane / P;
    uint8_t* to = mem + r0 * pitch + j * 16;
    uint4 v[P];
#pragma unroll
    for (int i = 0; i < P; i++) v[i] = *reinterpret_cast<const uint4*>(piece(stage, i * (32 / P) + r0, j));
    if (j * 16 < bytes) {
      pitch *= 32 / P;
#pragma unroll
      for (int i = 0; i < P; i++, to += pitch)
        if (i * (32 / P) + r0 < rows) *reinterpret_cast<uint4*>(to) = v[i];
    }
    return;
  }
  for (int r = 0; r < rows; r++)
    for (int b = lane * size; b < bytes; b += 32 * size) {
      const uint8_t* from = piece(stage, r, b >> 4) + (b & 15);
      uint8_t* to = mem + r * pitch + b;
      if (size == 4) *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(from);
      else if (size == 2) *reinterpret_cast<uint16_t*>(to) = *reinterpret_cast<const uint16_t*>(from);
      else *to = *from;
    }
}
// the other way, 128 bytes a row: under way when it returns (vec), to be waited for with cp.async.wait_all
__device__ __forceinline__ void get_rows(uint8_t* stage, const uint8_t* mem, int64_t pitch, int rows, int bytes, int size, bool vec) {
  const int lane = threadIdx.x & 31;
  if (vec) {
    const int j = lane & 7, r0 = lane >> 3;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int r = i * 4 + r0;
      if (r < rows && j * 16 < bytes)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(smem_addr(piece(stage, r, j))), "l"(mem + r * pitch + j * 16)
                     : "memory");
    }
    return;
  }
  for (int r = 0; r < rows; r++)
    for (int b = lane * size; b < bytes; b += 32 * size) {
      uint8_t* to = piece(stage, r, b >> 4) + (b & 15);
      const uint8_t* from = mem + r * pitch + b;
      if (size == 4) *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(from);
      else *reinterpret_cast<uint16_t*>(to) = *reinterpret_cast<const uint16_t*>(from);
    }
}

template <int OUT>
__device__ __forceinline__ float widen16(uint32_t h) {
  return OUT == kOutBf16 ? __uint_as_float(h << 16) : __half2float(__ushort_as_half((unsigned short)h));
}
template <int OUT>
__device__ __forceinline__ uint32_t narrow2(float lo, float hi) {
  if (OUT == kOutBf16) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&p);
  }
  const __half2 p = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}

// 32 columns of this lane's row into its staged row, at 16-byte piece j0 on; the residual's are there already
template <int OUT>
__device__ __forceinline__ void stage_row(bool residual, float (&y)[32], uint8_t* stage, int j0) {
  const int lane = threadIdx.x & 31;
  if (OUT == kOutF32) {
    if (residual) {
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const float4 q = *reinterpret_cast<const float4*>(piece(stage, lane, j0 + i));
        y[4 * i] += q.x;
        y[4 * i + 1] += q.y;
        y[4 * i + 2] += q.z;
        y[4 * i + 3] += q.w;
      }
    }
#pragma unroll
    for (int i = 0; i < 8; i++)
      *reinterpret_cast<float4*>(piece(stage, lane, j0 + i)) = make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
    return;
  }
  if (residual) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint4 q = *reinterpret_cast<const uint4*>(piece(stage, lane, j0 + i));
      const uint32_t h[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < 4; j++) {
        y[8 * i + 2 * j] += widen16<OUT>(h[j] & 0xffffu);
        y[8 * i + 2 * j + 1] += widen16<OUT>(h[j] >> 16);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; i++)
    *reinterpret_cast<uint4*>(piece(stage, lane, j0 + i)) =
        make_uint4(narrow2<OUT>(y[8 * i], y[8 * i + 1]), narrow2<OUT>(y[8 * i + 2], y[8 * i + 3]),
                   narrow2<OUT>(y[8 * i + 4], y[8 * i + 5]), narrow2<OUT>(y[8 * i + 6], y[8 * i + 7]));
}
// the same for a packed output: one block, of which `left` columns exist; returns its scale byte
template <int FMT>
__device__ __forceinline__ uint32_t stage_block(float (&y)[32], uint8_t* stage, int c, int left) {
  const int lane = threadIdx.x & 31;
  if (left < 32) {                                     // columns that do not exist
#pragma unroll
    for (int i = 0; i < 32; i++)
      if (i >= left) y[i] = 0.0f;
  }
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 32; i++) top = max(top, __float_as_uint(y[i]) & 0x7fffffffu);
  const uint32_t sb = scale_byte(top, FMT);
  const float inv = scale_inverse(sb);
  if (sb == 255u) {
#pragma unroll
    for (int i = 0; i < 32; i++) y[i] = 0.0f;
  }
#pragma unroll
  for (int i = 0; i < 32; i++) y[i] = __fmul_rn(y[i], inv);
  if (FMT == kFmtE2M1) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      w[i] = 0;
#pragma unroll
      for (int j = 0; j < 4; j++) w[i] |= (encode2(FMT, y[8 * i + 2 * j], y[8 * i + 2 * j + 1]) & 255u) << (8 * j);
    }
    *reinterpret_cast<uint4*>(piece(stage, lane, c)) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; i++)
      w[i] = encode2(FMT, y[4 * i], y[4 * i + 1]) | encode2(FMT, y[4 * i + 2], y[4 * i + 3]) << 16;
    *reinterpret_cast<uint4*>(piece(stage, lane, 2 * c)) = make_uint4(w[0], w[1], w[2], w[3]);
    *reinterpret_cast<uint4*>(piece(stage, lane, 2 * c + 1)) = make_uint4(w[4], w[5], w[6], w[7]);
  }
  return sb;
}
__device__ __forceinline__ uint32_t stage_block(int fmt, float (&y)[32], uint8_t* stage, int c, int left) {
  switch (fmt) {
    case kFmtE4M3: return stage_block<kFmtE4M3>(y, stage, c, left);
    case kFmtE5M2: return stage_block<kFmtE5M2>(y, stage, c, left);
    case kFmtE3M2: return stage_block<kFmtE3M2>(y, stage, c, left);
    case kFmtE2M3: return stage_block<kFmtE2M3>(y, stage, c, left);
    default: return stage_block<kFmtE2M1>(y, stage, c, left);
  }
}

// y += the biases of 32 columns, lane j's for column j
__device__ __forceinline__ void add_bias(float mine, float (&y)[32]) {
#pragma unroll
  for (int j = 0; j < 32; j++) y[j] += __shfl_sync(~0u, mine, j);
}

// Warp 0 loads the codes, warp 1 of the pair's first CTA issues the products, warps 2 and 3 bring the scales (in the second
// CTA warp 1 too), warps 4-11 write y: two per lane quarter, each with units of 64 columns.
//
// Measured (E4M3, bf16 y): 8192 x 8192 x 8192 434 us in a burst (2.53 PFLOP/s; 391 on a GPU that the power limit slowed
// less), 456 us back to back. Clock readings of the issuer, 4096 x 4096 x 4096, a pair's four tiles in 81500 cycles: 7900 to
// the first product (set-up 1900, the first scales and codes 6000), 65500 the products (512 a step of 128), 3400 at the tiles'
// ends (the shared columns' way out, the word to the next), 4700 in waits between; then the last tile's epilogue. The seven
// gated tiles of 4096 x 8192 x 2048 with packed y take 87 to 97 thousand: products 57, start 8 to 10, ends 6 to 8; the
// other 14 to 22 thousand have no cause yet. Short K shows the epilogue: 24576 rows by expert, 2048 x 1024: 81 us (85 with
// the staged rows written by the warps), 62 without it; 8192 x 8192 x 256 46 to 54 us.
//
// TMEM (512 columns, the same in both CTAs): two accumulators of 256 that share 64 columns, [0, 256) and [192, 448),
// and the stages' scale words in [448, 508). The epilogue of a tile drains the shared columns first and then lets the
// next tile's products start, so three quarters of it run beside them.
template <bool GATED, int OUT>
__global__ void __launch_bounds__(128 + 32 * kWriters, 1) __cluster_dims__(2, 1, 1)
    k_mx_tile(const __grid_constant__ CUtensorMap mx, const __grid_constant__ CUtensorMap mw, const __grid_constant__ CUtensorMap my,
              const __grid_constant__ Args a) {
  extern __shared__ uint8_t raw[];
  uint8_t* codes = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* passes = codes + kStages * kStageBytes;     // multiples of 1024 bytes, as the swizzle wants them
  uint8_t* scales = passes + kWriters * kPassBytes;
  TileShared& sh = *reinterpret_cast<TileShared*>(scales + kGroups * kGroupScales);
  const Table tab(&sh + 1, a.experts);
  const tc::Guard guard = {&sh.abort, a.status, a.wait_cycles};
  const int warp = __shfl_sync(~0u, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  constexpr int kCols = GATED ? 128 : 256;             // columns of y per tile
  const int col_tiles = (a.width + kCols - 1) / kCols;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; i++) {
      mbar_init(&sh.full[i], 1);                       // the first CTA's: the codes' bytes, both CTAs'
      mbar_init(&sh.empty[i], 1);
    }
    for (int i = 0; i < kGroups; i++) {
      mbar_init(&sh.scales_ready[i], 1);
      mbar_init(&sh.scales_full[i], 2);                // the first CTA's: both CTAs'
      mbar_init(&sh.scales_empty[i], 1);
    }
    mbar_init(&sh.acc_full, 1);
    mbar_init(&sh.acc_free, 2 * kWriters);             // the first CTA's: both CTAs' epilogue warps
    mbar_init(&sh.last, 1);
    sh.abort = 0;
    fence_mbar_init();
  }
  if (warp == 0 && tc::elect()) {
    tc::prefetch_map(&mw);
    tc::prefetch_map(&mx);
  }
  tc::wait_for_prior_grid();
  if (warp == 1) tc::tmem_alloc<true>(&sh.tmem, 512);
  if (warp == 2 && a.experts) count_tiles(tab, a, 256, col_tiles);
  tc::fence_before();
  cluster.sync();
  tc::fence_after();
  tc::start_next_grid();
  const uint32_t tmem = sh.tmem;
  const uint32_t full = tc::remote(sh.full, 0);
  const int tiles = tile_count(a, tab, 256, col_tiles);
  // the second half of a tile's w rows: the up projections, or the next 128 features
  const int second = GATED ? a.width : 128;
  // groups of scales `from`, from + step, ... on their way to the tensor core; the second CTA's by two warps in turn, so that
  // one's release passes beside the other's
  auto forward = [&](int from, int step) {
    const int per = (a.kblocks + 3) >> 2, groups = pair < tiles ? ((tiles - 1 - pair) / pairs + 1) * per : 0;
    const uint32_t far = rank ? tc::remote(sh.scales_full, 0) : 0u;
    Ring ring;
    if (from) ring.next(kGroups);
    for (int g = from; g < groups; g += step) {
      if (!forward_scales(sh.scales_ready, sh.scales_full, far, ring, kGroups, guard)) break;
      if (step == 2) ring.next(kGroups);
    }
  };

  if (warp == 0) {
    Ring ring;
    bool ok = true;
    Tiles list;
    int sent = 0;
    for (int i = pair; ok && i < tiles; i += pairs) {
      const Tile t = list.next(i, pairs, tiles, a, tab, 256, col_tiles);
      const int w0 = t.expert * a.n + t.col * kCols + (rank ? second : 0);
      for (int kb = 0; kb < a.kblocks; kb++) {
        ok = tc::wait_warp<true>(&sh.empty[ring.stage], ring.phase ^ 1u, guard);
        if (!ok) break;
        uint8_t* to = codes + ring.stage * kStageBytes;
        const uint32_t bar = full + 8u * ring.stage;
        if (tc::elect()) {
          if (rank == 0) mbar_expect_tx(&sh.full[ring.stage], 256 * (a.xbytes + a.wbytes));
          tc::tma_load_pair(to, &mx, kb * 128, t.row0 + rank * 128, bar);
          tc::tma_load_pair(to + kTileBytes, &mw, kb * 128, w0, bar);
        }
        __syncwarp();
        ring.next(kStages);
        sent++;
      }
    }
    if (!ok && lane == 0)                              // the loads under way land before the CTA leaves
      for (int s = 0; s < kStages && s < sent; s++) {
        ring.stage = ring.stage ? ring.stage - 1 : (ring.phase ^= 1u, kStages - 1);
        tc::settle(&sh.full[ring.stage], ring.phase, guard);
      }
  } else if (warp == 1) {
    if (rank == 0) {
      Ring ring, group;
      bool ok = true;
      int done = 0;
      for (int i = pair; ok && i < tiles; i += pairs, done++) {
        if (done) ok = tc::wait_warp<true>(&sh.acc_free, (done - 1) & 1, guard);
        if (!ok) break;
        const uint32_t acc = tmem + (done & 1 ? 192 : 0);
        for (int kb = 0; kb < a.kblocks; kb++) {
          ok = ((kb & 3) || tc::wait_warp<true>(&sh.scales_full[group.stage], group.phase, guard)) &&
               tc::wait_warp<true>(&sh.full[ring.stage], ring.phase, guard);
          if (!ok) break;
          tc::fence_after();
          const uint32_t at = smem_addr(codes + ring.stage * kStageBytes);
          const uint32_t sc = smem_addr(scales + group.stage * kGroupScales + (kb & 3) * kStepScales);
          const bool last = kb == a.kblocks - 1;
          const uint32_t ts = tmem + 448 + ring.stage * 12;
          const uint64_t da = tc::operand_desc(at), db = tc::operand_desc(at + kTileBytes);
          if (tc::elect()) {
#pragma unroll
            for (int j = 0; j < 3; j++) tc::copy_scales<true>(ts + 4 * j, tc::scale_desc(sc + 512 * j));
#pragma unroll
            for (int j = 0; j < 4; j++)                // 32 codes further: 2 units of 16 bytes
              tc::mma<true>(acc, da + 2 * j, db + 2 * j, tc::mma_desc_step(a.idesc, j), ts, ts + 4, kb > 0 || j > 0);
            tc::commit<true>(&sh.empty[ring.stage]);
            if (last || (kb & 3) == 3) tc::commit<true>(&sh.scales_empty[group.stage]);
            if (last) tc::commit<true>(&sh.acc_full);
          }
          __syncwarp();
          ring.next(kStages);
          if (last || (kb & 3) == 3) group.next(kGroups);
        }
      }
      if (!ok && tc::elect()) {
        tc::commit<true>(&sh.last);
        tc::settle(&sh.last, 0, guard);
      }
    } else {
      forward(1, 2);
    }
  } else if (warp == 2) {
    // x's 128 rows and w's 256. A group's words are on their way while the groups before them wait for their turn, over the
    // ends of the tiles too.
    const int per = (a.kblocks + 3) >> 2;
    ScaleRows<3> rows;
    uint4 v[12];
    Ring ring;
    Tiles list;
    bool ok = true;
    for (int i = pair; ok && i < tiles; i += pairs) {
      const Tile t = list.next(i, pairs, tiles, a, tab, 256, col_tiles);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int r = j * 32 + lane;
        rows.row[j] = a.sx + (int64_t)x_row(a, t, rank * 128 + r) * a.sx_pitch;
        rows.row[4 + j] = w_scales(a, t, t.col * kCols + r);
        rows.row[8 + j] = w_scales(a, t, t.col * kCols + r + second);
      }
      for (int g = 0; g < per; g++) {
        rows.load(v, g, a);
        ok = tc::wait_warp<true>(&sh.scales_empty[ring.stage], ring.phase ^ 1u, guard);
        if (!ok) break;
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (4 * g + j < a.kblocks) put_words<3>(v, j, scales + ring.stage * kGroupScales + j * kStepScales);
        __syncwarp();
        if (tc::elect()) tc::mbar_arrive(&sh.scales_ready[ring.stage]);
        ring.next(kGroups);
      }
    }
  } else if (warp == 3) {
    forward(0, rank ? 2 : 1);
  } else {
    Tiles list;
    int done = 0;
    const int q = warp & 3, set = (warp - 4) >> 2;     // lane quarter; which of its two warps
    uint8_t* stage = passes + (warp - 4) * kPassBytes;
    const uint32_t acc_free = tc::remote(&sh.acc_free, 0);
    constexpr int kUnits = kCols / 64;
    constexpr int size = OUT == kOutF32 ? 4 : OUT == kOutPacked ? 1 : 2;
    const bool nib = OUT == kOutPacked && a.ofmt == kFmtE2M1;
    // the stage's last rows have left it
    auto stage_free = [&] {
      if (lane == 0) tc::store_read();
      __syncwarp();
    };
    // the staged rows from column col on: by TMA where they are whole (it leaves out what is beyond y; by expert the
    // next expert's rows are), else by the warp
    auto put = [&](int row, int rows, int col, int cols) {
      if (a.map_out && (rows == 32 || a.experts == 0)) {
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) tc::tma_store(&my, col * size, row, stage);
      } else {
        __syncwarp();
        put_rows<8>(stage, static_cast<uint8_t*>(a.out) + (row * a.out_pitch + col) * size, a.out_pitch * size, rows, cols * size, size,
                    a.vec_out);
      }
      __syncwarp();
    };
    for (int i = pair; i < tiles; i += pairs, done++) {
      const Tile t = list.next(i, pairs, tiles, a, tab, 256, col_tiles);
      const int row = t.row0 + rank * 128 + q * 32;    // the warp's first
      const int rows = min(32, t.rows - rank * 128 - q * 32);
      // units in turn from the columns that the accumulators share on: the first accumulator's last unit, the
      // second's first
      auto unit_of = [&](int u) { return ((done & 1 ? 0 : kUnits - 1) + 2 * u + set) % kUnits; };
      // the residual's columns from col on go to the stage while the products and the activation are at work
      auto fetch = [&](int col) {
        if (!a.residual || rows <= 0 || col >= a.width) return;
        if (a.map_out) stage_free();
        get_rows(stage, static_cast<const uint8_t*>(a.residual) + (row * a.residual_stride + col) * size, a.residual_stride * size,
                   rows, min(128 / size, a.width - col) * size, size, a.vec_out);
      };
      // a unit's biases: column lane and column 32 + lane, of the gates and of the ups
      const float* bias = a.bias ? a.bias + (int64_t)t.expert * a.n : nullptr;
      float b[2] = {0.0f, 0.0f}, b_up[2] = {0.0f, 0.0f};
      auto fetch_bias = [&](int col) {
        if (!bias) return;
#pragma unroll
        for (int c = 0; c < 2; c++) {
          const int n = min(col + 32 * c + lane, a.width - 1);
          b[c] = __ldg(bias + n);
          if (GATED) b_up[c] = __ldg(bias + a.width + n);
        }
      };
      fetch(t.col * kCols + unit_of(0) * 64);
      fetch_bias(t.col * kCols + unit_of(0) * 64);
      const bool ok = tc::wait<true>(&sh.acc_full, done & 1, guard);
      __syncwarp();
      tc::fence_after();
      // the second warps' word that they are through with the tile before; the first warps give theirs below
      if (set == 1) {
        tc::fence_before();                            // their loads of that tile come before the word
        __syncwarp();
        if (lane == 0) tc::mbar_word_remote(acc_free);
      }
      const uint32_t acc = tmem + (done & 1 ? 192 : 0) + ((uint32_t)(q * 32) << 16);
#pragma unroll 1
      for (int u = 0; u < kUnits / 2; u++) {
        const int unit = unit_of(u), col0 = t.col * kCols + unit * 64;
        const bool live = rows > 0 && col0 < a.width;
        if (u > 0) {
          fetch(col0);
          fetch_bias(col0);
        }
        // The accumulator's shared columns leave TMEM before anything is done with them: of a gated tile's first unit
        // these are the gates' (second accumulator) or the ups'.
        const bool ups = GATED && !(done & 1);
        float y[32], next[32];
        tc::load32(acc + unit * 64 + (ups ? 128 : 0), y);
        tc::load32(acc + unit * 64 + (ups ? 160 : 32), next);
        if (set == 0 && u == 0) {                      // the next tile's products may start
          tc::fence_before();
          __syncwarp();
          if (lane == 0) tc::mbar_word_remote(acc_free);
        }
        // One body for both halves, not unrolled: straight-line code for 64 columns ran from the instruction cache's
        // second level, at 4 to 5 cycles an instruction.
#pragma unroll 1
        for (int c = 0; c < 2; c++) {
          const int col = col0 + c * 32, left = a.width - col;
          if (GATED) {
            float late[32];
            tc::load32(acc + (ups ? 0 : 128) + unit * 64 + c * 32, late);
            if (ups) {
#pragma unroll
              for (int j = 0; j < 32; j++) {
                const float up = y[j];
                y[j] = late[j];
                late[j] = up;
              }
            }
            if (bias) {
              add_bias(c ? b[1] : b[0], y);
              add_bias(c ? b_up[1] : b_up[0], late);
            }
            activate(a.act, y);
#pragma unroll
            for (int j = 0; j < 32; j++) y[j] *= late[j];
          } else {
            if (bias) add_bias(c ? b[1] : b[0], y);
            activate(a.act, y);
          }
          if (!ok) {
#pragma unroll
            for (int j = 0; j < 32; j++) y[j] = __uint_as_float(0x7fc00000u);
          }
          if (live && left > 0) {
            if (OUT == kOutPacked) {
              const uint32_t sb = stage_block(a.ofmt, y, stage, c, left);
              if (lane < rows) a.out_scales[(row + lane) * a.out_nb + (col >> 5)] = (uint8_t)sb;
            } else {
              if (c == 0 || OUT == kOutF32) {
                if (a.residual) {
                  asm volatile("cp.async.wait_all;\n" ::: "memory");
                  __syncwarp();
                } else if (a.map_out) {
                  stage_free();
                }
              }
              stage_row<OUT>(a.residual != nullptr, y, stage, OUT == kOutF32 ? 0 : 4 * c);
              if (OUT == kOutF32) {                    // 32 columns fill the stage
                put(row, rows, col, min(32, left));
                if (c == 0) fetch(col + 32);
              }
            }
          }
#pragma unroll
          for (int j = 0; j < 32; j++) y[j] = next[j];
        }
        if (OUT == kOutF32 || !live) continue;
        const int left = min(64, a.width - col0);
        if (OUT == kOutPacked) {
          uint8_t* out = static_cast<uint8_t*>(a.out) + row * a.out_pitch;
          __syncwarp();
          if (nib) put_rows<2>(stage, out + (col0 >> 1), a.out_pitch, rows, left >> 1, 1, a.vec_out);
          else put_rows<4>(stage, out + col0, a.out_pitch, rows, left, 1, a.vec_out);
          __syncwarp();
        } else {
          put(row, rows, col0, left);
        }
      }
    }
    if (a.map_out && lane == 0) tc::store_done();
  }
  __syncwarp();
  tc::fence_before();
  cluster.sync();
  tc::fence_after();
  if (warp == 1) tc::tmem_free<true>(tmem, 512);
}

// ------------------------------------------------------------------------------------------------- few rows
template <int BN>
struct RowsShape {
  static constexpr int kStageCodes = kTileBytes + BN * 128;
  static constexpr int kStageScales = 1024;            // w's 128 rows, x's up to 128
  static constexpr int kDepth = BN <= 32 ? 5 : BN == 64 ? 4 : 3;
  static constexpr int kSmem = 1024 + kDepth * (kStageCodes + kStageScales) + 256;
  static constexpr int kAcc = BN < 32 ? 32 : BN;       // accumulator columns
  static constexpr int kTmem = kAcc + kDepth * 8 <= 64 ? 64 : kAcc + kDepth * 8 <= 128 ? 128 : 256;
};

struct RowsShared {
  uint64_t full[5], empty[5], ready[5], acc_full, last;
  uint32_t tmem;
  int abort;
};
static_assert(sizeof(RowsShared) <= 256, "barriers");

// four columns of a row of y from column col on, all but the store's rounding done
__device__ __forceinline__ void write_four(const Args& a, float (&y)[4], int64_t row, int col, bool valid) {
  const int left = valid ? a.width - col : 0;
  if (a.otype == kOutPacked) {                         // eight lanes hold a block
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) top = max(top, i < left ? __float_as_uint(y[i]) & 0x7fffffffu : 0u);
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) top = max(top, __shfl_xor_sync(~0u, top, d));
    const uint32_t sb = scale_byte(top, a.ofmt);
    const float inv = scale_inverse(sb);
    if (left <= 0) return;
    if ((threadIdx.x & 7) == 0) a.out_scales[row * a.out_nb + (col >> 5)] = (uint8_t)sb;
#pragma unroll
    for (int i = 0; i < 4; i++) y[i] = i < left ? scaled(y[i], inv) : 0.0f;
    uint32_t lo = encode2(a.ofmt, y[0], y[1]), hi = encode2(a.ofmt, y[2], y[3]);
    uint8_t* to = static_cast<uint8_t*>(a.out) + row * a.out_pitch;
    if (a.ofmt == kFmtE2M1) {                          // the width is even
      to[col >> 1] = (uint8_t)lo;
      if (left > 2) to[(col >> 1) + 1] = (uint8_t)hi;
    } else if (left >= 4 && a.vec_out) {
      *reinterpret_cast<uint32_t*>(to + col) = lo | hi << 16;
    } else {
      lo |= hi << 16;
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (i < left) to[col + i] = (uint8_t)(lo >> (8 * i));
    }
    return;
  }
  if (left <= 0) return;
  const int64_t at = row * a.out_pitch + col, from = row * a.residual_stride + col;
  if (a.otype == kOutF32) {
    float* to = static_cast<float*>(a.out) + at;
    const float* r = a.residual ? static_cast<const float*>(a.residual) + from : nullptr;
    if (left >= 4 && a.vec_out) {
      float4 v = make_float4(y[0], y[1], y[2], y[3]);
      if (r) {
        const float4 q = *reinterpret_cast<const float4*>(r);
        v = make_float4(v.x + q.x, v.y + q.y, v.z + q.z, v.w + q.w);
      }
      *reinterpret_cast<float4*>(to) = v;
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (i < left) to[i] = r ? y[i] + r[i] : y[i];
    }
    return;
  }
  uint16_t* to = static_cast<uint16_t*>(a.out) + at;
  const uint16_t* r = a.residual ? static_cast<const uint16_t*>(a.residual) + from : nullptr;
  const bool bf = a.otype == kOutBf16, four = left >= 4 && a.vec_out;
  if (r) {
    uint16_t h[4] = {0, 0, 0, 0};
    if (four) {
      *reinterpret_cast<uint2*>(h) = *reinterpret_cast<const uint2*>(r);
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (i < left) h[i] = r[i];
    }
#pragma unroll
    for (int i = 0; i < 4; i++) y[i] += bf ? widen16<kOutBf16>(h[i]) : widen16<kOutF16>(h[i]);
  }
  const uint32_t lo = bf ? narrow2<kOutBf16>(y[0], y[1]) : narrow2<kOutF16>(y[0], y[1]);
  const uint32_t hi = bf ? narrow2<kOutBf16>(y[2], y[3]) : narrow2<kOutF16>(y[2], y[3]);
  if (four) {
    *reinterpret_cast<uint2*>(to) = make_uint2(lo, hi);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (i < left) to[i] = (uint16_t)((i < 2 ? lo : hi) >> (16 * (i & 1)));
  }
}

// Here w's rows are the A operand (128 lanes of TMEM) and x's the B operand (16 to 64 columns), so that a tile costs
// what its bytes of w cost. Measured, 16 rows by 16384 x 16384: E4M3 50 us (5.5 TB/s), FP4 34 us (4.2 TB/s: a stage
// holds half the bytes, and the time from a stage's release to its next product is the same). 1 row by 8192 x 2048:
// 7.6 us, of which the launch, the set-up and the cluster's two barriers are most.
//
// The cluster's CTAs each take a share of K; their partial sums meet in shared memory and are added in rank order (the
// same sum on every run), each CTA finishing its share of the rows of x.
template <int BN, bool GATED>
__global__ void __launch_bounds__(128, 2) k_mx_rows(const __grid_constant__ CUtensorMap mx, const __grid_constant__ CUtensorMap mw,
                                                 const __grid_constant__ Args a) {
  using S = RowsShape<BN>;
  extern __shared__ uint8_t raw[];
  uint8_t* codes = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* scales = codes + S::kDepth * S::kStageCodes;
  RowsShared& sh = *reinterpret_cast<RowsShared*>(scales + S::kDepth * S::kStageScales);
  const Table tab(&sh + 1, a.experts);
  const tc::Guard guard = {&sh.abort, a.status, a.wait_cycles};
  const int warp = __shfl_sync(~0u, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  constexpr int kCols = GATED ? 64 : 128;              // columns of y per tile
  const int col_tiles = (a.width + kCols - 1) / kCols;
  cg::cluster_group cluster = cg::this_cluster();
  const int split = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();

  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kDepth; i++) {
      mbar_init(&sh.full[i], 2);                       // the codes' bytes and the scales
      mbar_init(&sh.empty[i], 1);
      mbar_init(&sh.ready[i], 1);
    }
    mbar_init(&sh.acc_full, 1);
    mbar_init(&sh.last, 1);
    sh.abort = 0;
    fence_mbar_init();
  }
  if (warp == 0 && tc::elect()) {
    tc::prefetch_map(&mw);
    tc::prefetch_map(&mx);
  }
  tc::wait_for_prior_grid();
  if (warp == 1) tc::tmem_alloc<false>(&sh.tmem, S::kTmem);
  if (warp == 2 && a.experts) count_tiles(tab, a, BN, col_tiles);
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  tc::start_next_grid();
  const uint32_t tmem = sh.tmem;
  Tile t;
  const bool work = (int)blockIdx.x / split < tile_count(a, tab, BN, col_tiles);  // the same for the whole cluster
  if (work) t.find(blockIdx.x / split, a, tab, BN, col_tiles);
  const int k0 = (int)((int64_t)a.kblocks * rank / split), k1 = (int)((int64_t)a.kblocks * (rank + 1) / split);
  const bool busy = work && k1 > k0;

  if (busy && warp == 0) {
    Ring ring;
    bool ok = true;
    int sent = 0;
    int4 rows = make_int4(0, 0, 0, 0);
    if (a.per > 0 && lane < BN / 4)
      rows = make_int4(x_row(a, t, 4 * lane), x_row(a, t, 4 * lane + 1), x_row(a, t, 4 * lane + 2), x_row(a, t, 4 * lane + 3));
    const int w0 = t.expert * a.n + t.col * kCols;
    for (int kb = k0; kb < k1; kb++) {
      ok = tc::wait_warp<false>(&sh.empty[ring.stage], ring.phase ^ 1u, guard);
      if (!ok) break;
      uint8_t* to = codes + ring.stage * S::kStageCodes;
      uint64_t* bar = &sh.full[ring.stage];
      if (tc::elect()) {
        mbar_expect_tx(bar, 128 * a.wbytes + BN * a.xbytes);
        tma_load_2d(to, &mw, kb * 128, w0, bar);
        if (GATED) tma_load_2d(to + kTileBytes / 2, &mw, kb * 128, w0 + a.width, bar);
        if (a.per == 0) tma_load_2d(to + kTileBytes, &mx, kb * 128, t.row0, bar);
      }
      __syncwarp();
      if (a.per > 0 && lane < BN / 4) tc::tma_gather4(to + kTileBytes + lane * 512, &mx, kb * 128, rows, bar);
      ring.next(S::kDepth);
      sent++;
    }
    if (!ok && lane == 0)
      for (int s = 0; s < S::kDepth && s < sent; s++) {
        ring.stage = ring.stage ? ring.stage - 1 : (ring.phase ^= 1u, S::kDepth - 1);
        tc::settle(&sh.full[ring.stage], ring.phase, guard);
      }
  } else if (busy && warp == 1) {
    Ring ring;
    bool ok = true;
    for (int kb = k0; kb < k1; kb++) {
      ok = tc::wait_warp<false>(&sh.full[ring.stage], ring.phase, guard);
      if (!ok) break;
      tc::fence_after();
      const uint32_t at = smem_addr(codes + ring.stage * S::kStageCodes);
      const uint32_t sc = smem_addr(scales + ring.stage * S::kStageScales);
      const uint32_t ts = tmem + S::kAcc + ring.stage * 8;
      const uint64_t da = tc::operand_desc(at), db = tc::operand_desc(at + kTileBytes);
      if (tc::elect()) {
        tc::copy_scales<false>(ts, tc::scale_desc(sc));
        tc::copy_scales<false>(ts + 4, tc::scale_desc(sc + 512));
#pragma unroll
        for (int j = 0; j < 4; j++)
          tc::mma<false>(tmem, da + 2 * j, db + 2 * j, tc::mma_desc_step(a.idesc, j), ts, ts + 4, kb > k0 || j > 0);
        tc::commit<false>(&sh.empty[ring.stage]);
        if (kb == k1 - 1) tc::commit<false>(&sh.acc_full);
      }
      __syncwarp();
      ring.next(S::kDepth);
    }
    if (!ok && tc::elect()) {
      tc::commit<false>(&sh.last);
      tc::settle(&sh.last, 0, guard);
    }
  } else if (busy && warp == 2) {
    ScaleRows<2> rows;                                 // w's 128 rows; x's, the last repeated up to 128
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int r = j * 32 + lane;
      rows.row[j] = w_scales(a, t, t.col * kCols + (GATED && r >= 64 ? a.width + r - 64 : r));
      rows.row[4 + j] = a.sx + (int64_t)x_row(a, t, r) * a.sx_pitch;
    }
    Ring ring;
    uint4 now[8], nxt[8];
    int g = k0 >> 2;
    const int last = (k1 - 1) >> 2;
    bool ok = true;
    rows.load(now, g, a);
    for (; g <= last && ok; g++) {
      if (g < last) rows.load(nxt, g + 1, a);
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (g * 4 + j >= k0 && g * 4 + j < k1 && ok)
          ok = store_scales<2>(now, j, a, scales, S::kStageScales, sh.ready, sh.empty, ring, S::kDepth, guard);
#pragma unroll
      for (int i = 0; i < 8; i++) now[i] = nxt[i];
    }
  } else if (busy) {
    Ring ring;
    bool ok = true;
    for (int kb = k0; kb < k1 && ok; kb++) ok = forward_scales(sh.ready, sh.full, 0u, ring, S::kDepth, guard);
  }
  __syncwarp();

  // partial sums, [row of x][feature], over the codes' stages, which are all consumed
  float* part = reinterpret_cast<float*>(codes);
  if (work) {
    const bool ok = !busy || tc::wait<false>(&sh.acc_full, 0, guard);
    __syncwarp();
    tc::fence_after();
    const uint32_t acc = tmem + ((uint32_t)(warp * 32) << 16);
#pragma unroll 1
    for (int c = 0; c < BN; c += 16) {
      float v[16];
      tc::load16(acc + c, v);
#pragma unroll
      for (int j = 0; j < 16; j++)
        part[(c + j) * 128 + warp * 32 + lane] = !busy ? 0.0f : ok ? v[j] : __uint_as_float(0x7fc00000u);
    }
  }
  tc::fence_before();
  if (split > 1) cluster.sync(); else __syncthreads();
  tc::fence_after();
  if (work) {
    // a row of kCols columns by kCols / 4 lanes, rows dealt out to the cluster's warps
    constexpr int kLanes = kCols / 4, kRows = 32 / kLanes;
    const float* bias = a.bias ? a.bias + (int64_t)t.expert * a.n : nullptr;
    const int f = lane % kLanes * 4, col = t.col * kCols + f;
    float b[4] = {0.0f, 0.0f, 0.0f, 0.0f}, b_up[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (bias) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int n = min(col + i, a.width - 1);
        b[i] = __ldg(bias + n);
        if (GATED) b_up[i] = __ldg(bias + a.width + n);
      }
    }
    for (int base = (rank * 4 + warp) * kRows; base < t.rows; base += split * 4 * kRows) {
      const int r = base + lane / kLanes, at = min(r, t.rows - 1) * 128 + f;
      float y[4] = {0.0f, 0.0f, 0.0f, 0.0f}, up[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
      for (int s = 0; s < split; s++) {
        const float* from = split > 1 ? cluster.map_shared_rank(part, s) : part;
        const float4 v = *reinterpret_cast<const float4*>(from + at);
        y[0] += v.x;
        y[1] += v.y;
        y[2] += v.z;
        y[3] += v.w;
        if (GATED) {
          const float4 u = *reinterpret_cast<const float4*>(from + at + 64);
          up[0] += u.x;
          up[1] += u.y;
          up[2] += u.z;
          up[3] += u.w;
        }
      }
#pragma unroll
      for (int i = 0; i < 4; i++) y[i] += b[i];
      activate(a.act, y);
      if (GATED) {
#pragma unroll
        for (int i = 0; i < 4; i++) y[i] *= up[i] + b_up[i];
      }
      write_four(a, y, (int64_t)t.row0 + r, col, r < t.rows);
    }
  }
  if (split > 1) cluster.sync(); else __syncthreads();  // the partial sums are read before their CTA leaves
  if (warp == 1) tc::tmem_free<false>(tmem, S::kTmem);
}

// --------------------------------------------------------------------------------------------------- host
struct Operand {
  const uint8_t* codes;
  int64_t rows, pitch;
  bool nibbles;
};
int map_of(CUtensorMap* m, const Operand& o, int64_t K, int box) {
  return encode_tmap_codes(m, o.codes, o.nibbles, (uint64_t)o.rows, (uint64_t)K, (uint64_t)o.pitch, (uint32_t)box);
}

template <int BN, bool GATED>
int launch_rows(Args& a, const Operand& x, const Operand& w, int64_t K, int64_t tiles, int split, int fx, int fw, cudaStream_t st) {
  using S = RowsShape<BN>;
  CUtensorMap mx, mw;
  if (int rc = map_of(&mx, x, K, a.per > 0 ? 1 : BN)) return rc;
  if (int rc = map_of(&mw, w, K, GATED ? 64 : 128)) return rc;
  a.idesc = tc::mma_desc(fw, fx, 128, BN);
  const int smem = S::kSmem + (a.experts ? table_bytes(a.experts) : 0);
  auto f = k_mx_rows<BN, GATED>;
  if (int rc = allow_smem((const void*)f, S::kSmem + table_bytes(kMostExperts))) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * split));
  cfg.blockDim = dim3(128);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = split;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  return check_cuda(cudaLaunchKernelEx(&cfg, f, mx, mw, a), "product (few rows)");
}

template <bool GATED, int OUT>
int launch_tile(Args& a, const Operand& x, const Operand& w, int64_t K, int64_t tiles, int fx, int fw, cudaStream_t st) {
  CUtensorMap mx, mw, my;
  if (int rc = map_of(&mx, x, K, 128)) return rc;
  if (int rc = map_of(&mw, w, K, 128)) return rc;
  // y as bytes, in the stage's rows of 128; a tile's first byte in its row is a 32-bit coordinate
  const int size = OUT == kOutF32 ? 4 : 2;
  a.map_out = OUT != kOutPacked && a.vec_out && (int64_t)a.width * size < (1ll << 31);
  my = mx;
  if (a.map_out)
    if (int rc = encode_tmap_codes(&my, a.out, false, (uint64_t)a.rows, (uint64_t)a.width * size, (uint64_t)a.out_pitch * size, 32)) return rc;
  a.idesc = tc::mma_desc(fx, fw, 256, 256);
  const int smem = kTileSmem + (a.experts ? table_bytes(a.experts) : 0);
  auto f = k_mx_tile<GATED, OUT>;
  if (int rc = allow_smem((const void*)f, kTileSmem + table_bytes(kMostExperts))) return rc;
  const int64_t pairs = sm_count() / 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * (tiles < pairs ? tiles : pairs)));
  cfg.blockDim = dim3(128 + 32 * kWriters);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, f, mx, mw, my, a), "product");
}

int64_t up_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// How a product is cut up: by k_mx_rows in tiles of bn rows with K split, or by k_mx_tile
struct Cut {
  bool few;
  int bn, split;
  int64_t tiles;
};
Cut cut_of(const Args& a, bool gated, int64_t kblocks) {
  // rows that share a tile of w: all of them, or an expert's share
  const int64_t share = a.experts ? up_div(a.rows, a.experts) : a.rows;
  const int64_t groups = a.experts ? (a.experts < a.rows ? a.experts : a.rows) : 1;
  const int64_t cols = up_div(a.width, gated ? 64 : 128);
  Cut c;
  // Tiles of few rows: as many as there are; by expert several times the mean, since the longest expert's second tile
  // would read w again (64 experts of 2048 x 1024 with 8 rows each at random: 37 us with tiles of 16, 33 with 32 and
  // 64).
  c.bn = a.experts ? (share <= 2 ? 16 : share <= 8 ? 32 : 64) : share <= 16 ? 16 : share <= 32 ? 32 : 64;
  c.tiles = (a.experts ? a.rows / c.bn + groups : up_div(a.rows, c.bn)) * cols;
  // Which kernel, measured on E4M3: dense 4096 x 4096, M = 256: 14.9 us by few rows, 16.9 by many, M = 384: 19.0 and
  // 17.4; 2048 x 2048, M = 512: 12.4 and 12.4; 8192 x 2048, M = 128: 12.5 and 12.7, M = 256: 14.5 and 12.9. By
  // expert, 64 experts 2048 x 1024: 1 row each 22 and 28, 4 rows 38 and 37, 8 rows 39 and 37, 12 rows 40 and 38; 2048 x
  // 2048: 8 rows 59 and 66, 12 rows 60 and 66; 8 experts 4096 x 2048, 32 rows: 14 and 20.
  c.few = a.experts ? share <= 8 || c.tiles <= 4 * sm_count() : c.tiles <= sm_count();
  c.split = 1;
  if (!c.few) {
    c.tiles = (a.experts ? a.rows / 256 + groups : up_div(a.rows, 256)) * up_div(a.width, gated ? 128 : 256);
    return c;
  }
  // K split over a cluster while that gives every SM two CTAs at most and each CTA two steps at least
  while (c.split < 8 && c.tiles * c.split * 2 <= 2 * sm_count() && kblocks >= c.split * 4) c.split *= 2;
  return c;
}

template <bool GATED>
int launch(Args& a, const Cut& c, const Operand& x, const Operand& w, int64_t K, int fx, int fw, cudaStream_t st) {
  if (!c.few) {
    switch (a.otype) {
      case kOutF32: return launch_tile<GATED, kOutF32>(a, x, w, K, c.tiles, fx, fw, st);
      case kOutBf16: return launch_tile<GATED, kOutBf16>(a, x, w, K, c.tiles, fx, fw, st);
      case kOutF16: return launch_tile<GATED, kOutF16>(a, x, w, K, c.tiles, fx, fw, st);
      default: return launch_tile<GATED, kOutPacked>(a, x, w, K, c.tiles, fx, fw, st);
    }
  }
  switch (c.bn) {
    case 16: return launch_rows<16, GATED>(a, x, w, K, c.tiles, c.split, fx, fw, st);
    case 32: return launch_rows<32, GATED>(a, x, w, K, c.tiles, c.split, fx, fw, st);
    default: return launch_rows<64, GATED>(a, x, w, K, c.tiles, c.split, fx, fw, st);
  }
}

bool aligned(const void* p, int64_t n) { return reinterpret_cast<uintptr_t>(p) % (uintptr_t)n == 0; }

// An operand as a caller has it: codes of a format (pitch in bytes) or, type > 0, floats of type - 1 (pitch in
// elements)
struct Given {
  const void* data;
  const uint8_t* scales;
  int64_t rows, pitch;
  int fmt, type;
};
int mma_format(int fmt) { return fmt == kFmtE4M3 ? tc::kE4M3 : fmt == kFmtE5M2 ? tc::kE5M2 : tc::kE2M1; }
int64_t codes_pitch(int64_t K) { return up_div(K, 16) * 16; }
// whether the tensor maps take the codes as they are; rows that are gathered one by one must be 8-bit codes
bool direct(const Given& o, int64_t K, bool gathered) {
  if (o.type > 0) return false;
  if (o.fmt == kFmtE4M3 || o.fmt == kFmtE5M2) return aligned(o.data, 16) && o.pitch % 16 == 0;
  return o.fmt == kFmtE2M1 && !gathered && aligned(o.data, 32) && o.pitch % 32 == 0 && K % 128 == 0;
}
// Scale rows of an operand that is laid out come to 16 bytes too where they are at odd bytes (63 of them a row, 777 x 1000:
// the product takes 15 us instead of 18); rows of a word or less are one load either way.
bool scales_at_odd_bytes(int64_t K) { return K > 128 && up_div(K, 32) % 4 != 0; }
int64_t scales_pitch(int64_t K) { return scales_at_odd_bytes(K) ? up_div(K, 512) * 16 : up_div(K, 32); }
int64_t room(const Given& o, int64_t K, bool gathered) {
  if (direct(o, K, gathered)) return 0;
  const bool scales = o.type > 0 || scales_at_odd_bytes(K);
  return up_div(o.rows * (codes_pitch(K) + (scales ? scales_pitch(K) : 0)), 128) * 128;
}
// rows in the plan's order: their codes at codes_pitch(K), whatever the pitch of x, then their scales
int64_t sorted_room(int64_t rows, int64_t K) { return up_div(rows * (codes_pitch(K) + up_div(K, 32)), 128) * 128; }
// The operand as the kernels read it, laid out in `at` (room() bytes) where need be: floats are packed by a launch here,
// codes are left to the caller's `job`
int lay(const Given& o, int64_t K, bool gathered, uint8_t* at, Operand* out, const uint8_t** scales, int* pitch_of_scales, int* fmt,
        LayJob* job, cudaStream_t st) {
  const bool odd = scales_at_odd_bytes(K);
  *job = {};
  *scales = o.scales;
  *pitch_of_scales = (int)up_div(K, 32);
  *fmt = o.fmt;
  if (direct(o, K, gathered)) {
    *out = {static_cast<const uint8_t*>(o.data), o.rows, o.pitch, o.fmt == kFmtE2M1};
    return MXQ_OK;
  }
  const int64_t pitch = codes_pitch(K);
  *out = {at, o.rows, pitch, false};
  if (o.fmt != kFmtE5M2) *fmt = kFmtE4M3;
  uint8_t* sc = at + o.rows * pitch;
  if (o.type > 0 || odd) {
    *scales = sc;
    *pitch_of_scales = (int)scales_pitch(K);
  }
  if (o.type > 0) return pack_rows_to(o.data, o.type - 1, o.pitch, at, pitch, sc, *pitch_of_scales, o.rows, K, o.fmt, st);
  *job = {static_cast<const uint8_t*>(o.data), o.pitch, at, pitch, o.rows, K, o.fmt, 0, o.scales, odd ? sc : nullptr, *pitch_of_scales};
  return MXQ_OK;
}

int check_operand(const char* who, const char* what, const Given& o, int64_t K) {
  MXQ_REQUIRE(o.fmt != kFmtNone, MXQ_ERR_VALUE, "%s: %s has no MX element format", who, what);
  MXQ_REQUIRE(o.type >= 0 && o.type <= 1 + kOutF16, MXQ_ERR_VALUE, "%s: type %d of %s", who, o.type, what);
  MXQ_REQUIRE(o.fmt != kFmtE2M1 || K % 2 == 0 || o.type > 0, MXQ_ERR_VALUE, "%s: FP4 codes of %s pair up, K is %lld", who, what, (long long)K);
  const int64_t least = o.type > 0 || o.fmt != kFmtE2M1 ? K : K / 2;
  MXQ_REQUIRE(o.rows <= 1 || o.pitch >= least, MXQ_ERR_VALUE, "%s: rows of %s are %lld apart and K is %lld", who, what, (long long)o.pitch,
              (long long)K);
  return MXQ_OK;
}

int product(const char* who, Args& a, const Given& gx, const Given& gw, int64_t K, const mxq_product_spec* s, void* workspace,
            int64_t workspace_bytes, cudaStream_t st) {
  if (int rc = check_operand(who, "x", gx, K)) return rc;
  if (int rc = check_operand(who, "w", gw, K)) return rc;
  MXQ_REQUIRE(s->activation >= kActNone && s->activation <= kActGeglu, MXQ_ERR_VALUE, "%s: activation %d", who, s->activation);
  MXQ_REQUIRE(s->out >= kOutF32 && s->out <= kOutPacked, MXQ_ERR_VALUE, "%s: output type %d", who, s->out);
  const bool gated = s->activation >= kActSwiglu;
  MXQ_REQUIRE(!gated || a.n % 2 == 0, MXQ_ERR_VALUE, "%s: a gated activation needs an even number of rows of w, got %d", who, a.n);
  a.width = gated ? a.n / 2 : a.n;
  a.act = s->activation;
  a.otype = s->out;
  a.ofmt = kFmtE4M3;
  a.out_pitch = a.width;
  a.out_nb = up_div(a.width, 32);
  if (s->out == kOutPacked) {
    a.ofmt = format_of(s->out_e, s->out_m);
    MXQ_REQUIRE(a.ofmt != kFmtNone, MXQ_ERR_VALUE, "%s: (e=%d, m=%d) is not an MX element format", who, s->out_e, s->out_m);
    MXQ_REQUIRE(a.out_scales != nullptr && a.residual == nullptr, MXQ_ERR_VALUE, "%s: a packed output needs scales and takes no residual", who);
    if (a.ofmt == kFmtE2M1) {
      MXQ_REQUIRE(a.width % 2 == 0, MXQ_ERR_VALUE, "%s: packed FP4 needs an even width, got %d", who, a.width);
      a.out_pitch = a.width / 2;
    }
  }
  const int size = s->out == kOutF32 ? 4 : s->out == kOutPacked ? 1 : 2;
  a.vec_out = a.out_pitch * size % 16 == 0 && aligned(a.out, 16) &&
              (a.residual == nullptr || (a.residual_stride * size % 16 == 0 && aligned(a.residual, 16)));
  a.kblocks = (int)up_div(K, 128);
  const Cut cut = cut_of(a, gated, a.kblocks);
  // Rows that the plan scatters are fetched one by one by k_mx_rows in tiles of up to 32 (tile::gather4: four rows an
  // instruction, about 65 cycles each), and brought into the plan's order first for larger tiles: 64 experts 2048 x
  // 2048, 384 rows each: 330 us fetched, 154 sorted; 8 experts 4096 x 4096, 16 rows each: 36 and 33.
  const bool sorted = a.per > 0 && (!cut.few || cut.bn > 32);
  const int64_t room_x = room(gx, K, a.per > 0), room_w = room(gw, K, false), room_s = sorted ? sorted_room(a.rows, K) : 0;
  const int64_t need = room_x + room_w + room_s;
  MXQ_REQUIRE(a.rows == 0 || a.width == 0 || need == 0 || (workspace != nullptr && aligned(workspace, 16) && workspace_bytes >= need),
              MXQ_ERR_VALUE, "%s: needs a workspace of %lld bytes, 16-byte aligned", who, (long long)need);
  if (a.rows == 0 || a.width == 0) return MXQ_OK;
  a.status = wait_status_word();
  if (!a.status) return MXQ_ERR_CUDA;
  Operand x, w;
  int fmtx, fmtw;
  uint8_t* at = static_cast<uint8_t*>(workspace);
  LayJob lay_x, lay_w;
  if (int rc = lay(gx, K, a.per > 0, at, &x, &a.sx, &a.sx_pitch, &fmtx, &lay_x, st)) return rc;
  if (int rc = lay(gw, K, false, at + room_x, &w, &a.sw, &a.sw_pitch, &fmtw, &lay_w, st)) return rc;
  if (int rc = lay_rows(lay_x, lay_w, st)) return rc;
  a.nb = (int)up_div(K, 32);
  if (sorted) {
    uint8_t* codes = at + room_x + room_w;
    const int64_t pitch = codes_pitch(K);
    uint8_t* scales = codes + a.rows * pitch;
    if (int rc = gather_rows(x.codes, a.sx, x.pitch, a.sx_pitch, a.order, a.per, a.xrows, a.rows, K, codes, pitch, scales, st)) return rc;
    x = {codes, a.rows, pitch, false};
    a.sx = scales;
    a.sx_pitch = a.nb;
    a.xrows = a.rows;
    a.per = 0;
  }
  const int fx = mma_format(fmtx), fw = mma_format(fmtw);
  auto scales_by = [&](int n) { return a.sx_pitch % n == 0 && a.sw_pitch % n == 0 && aligned(a.sx, n) && aligned(a.sw, n); };
  a.vec = scales_by(16) ? 16 : scales_by(4) ? 4 : 1;
  // a load of FP4 codes counts the bytes read, half of those that it fills
  a.xbytes = fmtx == kFmtE2M1 ? 64 : 128;
  a.wbytes = fmtw == kFmtE2M1 ? 64 : 128;
  if (a.wait_cycles == 0) a.wait_cycles = tc::kWaitCycles;
  else a.xbytes += 16;                                 // the test of the waits: bytes that never come
  return gated ? launch<true>(a, cut, x, w, K, fx, fw, st) : launch<false>(a, cut, x, w, K, fx, fw, st);
}

int check_sizes(const char* who, int64_t rows, int64_t N, int64_t K, int64_t experts) {
  MXQ_REQUIRE(rows >= 0 && rows < (1ll << 30) && N >= 0 && K >= 1 && K < (1ll << 30) && experts >= 1 && experts * N < (1ll << 30),
              MXQ_ERR_VALUE, "%s: bad sizes (rows %lld, N %lld, K %lld, experts %lld)", who, (long long)rows, (long long)N,
              (long long)K, (long long)experts);
  return MXQ_OK;
}

}  // namespace

namespace mxq {
unsigned product_wait_timeouts() { return read_wait_timeouts(); }
}  // namespace mxq

extern "C" int64_t mxq_product_workspace(const void* x, int64_t x_pitch, int64_t x_rows, const uint8_t* w, int64_t w_pitch, int64_t w_rows,
                                         int64_t K, int64_t gathered_slots, const mxq_product_spec* s) {
  if (s == nullptr || K < 1 || x_rows < 0 || w_rows < 0 || gathered_slots < 0) return -1;
  return room({x, nullptr, x_rows, x_pitch, format_of(s->x_e, s->x_m), s->x_type}, K, gathered_slots > 0) +
         room({w, nullptr, w_rows, w_pitch, format_of(s->w_e, s->w_m), 0}, K, false) + (gathered_slots > 0 ? sorted_room(gathered_slots, K) : 0);
}

extern "C" int mxq_linear_packed(const void* x, const uint8_t* x_scales, int64_t x_pitch, int64_t M, const uint8_t* w,
                                 const uint8_t* w_scales, int64_t w_pitch, int64_t N, int64_t K, const mxq_product_spec* spec,
                                 const float* bias, const void* residual, int64_t residual_stride, void* out,
                                 uint8_t* out_scales, void* workspace, int64_t workspace_bytes, void* stream) {
  MXQ_REQUIRE(spec != nullptr, MXQ_ERR_VALUE, "linear_packed: no spec");
  if (int rc = check_sizes("linear_packed", M, N, K, 1)) return rc;
  Args a = {};
  a.rows = a.xrows = (int)M;
  a.n = (int)N;
  a.bias = bias;
  a.residual = residual;
  a.residual_stride = residual_stride;
  a.out = out;
  a.out_scales = out_scales;
  return product("linear_packed", a, {x, x_scales, M, x_pitch, format_of(spec->x_e, spec->x_m), spec->x_type},
                 {w, w_scales, N, w_pitch, format_of(spec->w_e, spec->w_m), 0}, K, spec, workspace, workspace_bytes, as_stream(stream));
}

extern "C" int mxq_testing_product_timeout(const uint8_t* x, const uint8_t* x_scales, int64_t M, const uint8_t* w,
                                           const uint8_t* w_scales, int64_t N, int64_t K, float* y, int64_t wait_cycles,
                                           void* stream) {
  if (int rc = check_sizes("testing_product_timeout", M, N, K, 1)) return rc;
  MXQ_REQUIRE(wait_cycles >= 1 && wait_cycles <= (1 << 22), MXQ_ERR_VALUE, "testing_product_timeout: wait_cycles must be in [1, 2^22]");
  const mxq_product_spec spec = {4, 3, 4, 3, MXQ_ACT_NONE, MXQ_OUT_F32, 0, 0, 0};
  Args a = {};
  a.rows = a.xrows = (int)M;
  a.n = (int)N;
  a.out = y;
  a.wait_cycles = wait_cycles;
  return product("testing_product_timeout", a, {x, x_scales, M, K, kFmtE4M3, 0}, {w, w_scales, N, K, kFmtE4M3, 0}, K, &spec, nullptr, 0,
                 as_stream(stream));
}

extern "C" int mxq_experts_packed(const void* x, const uint8_t* x_scales, int64_t x_pitch, int64_t x_rows, const uint8_t* w,
                                  const uint8_t* w_scales, int64_t w_pitch, int64_t experts, int64_t N, int64_t K,
                                  const int32_t* offsets, const int32_t* order, int64_t slots, int64_t per,
                                  const mxq_product_spec* spec, const float* bias, void* out, uint8_t* out_scales,
                                  void* workspace, int64_t workspace_bytes, void* stream) {
  MXQ_REQUIRE(spec != nullptr, MXQ_ERR_VALUE, "experts_packed: no spec");
  if (int rc = check_sizes("experts_packed", slots, N, K, experts)) return rc;
  MXQ_REQUIRE(experts <= kMostExperts, MXQ_ERR_UNSUPPORTED, "experts_packed: at most %d experts, got %lld", kMostExperts,
              (long long)experts);
  MXQ_REQUIRE(per >= 0 && per < (1ll << 30) &&
                  (slots == 0 || (x_rows >= 1 && x_rows < (1ll << 30) && (per == 0 ? x_rows >= slots : x_rows * per >= slots))),
              MXQ_ERR_VALUE, "experts_packed: %lld rows of x do not serve %lld slots, %lld per row", (long long)x_rows,
              (long long)slots, (long long)per);
  Args a = {};
  a.offsets = offsets;
  a.order = order;
  a.experts = (int)experts;
  a.per = (int)per;
  a.rows = (int)slots;
  a.xrows = (int)x_rows;
  a.n = (int)N;
  a.bias = bias;
  a.out = out;
  a.out_scales = out_scales;
  return product("experts_packed", a, {x, x_scales, x_rows, x_pitch, format_of(spec->x_e, spec->x_m), spec->x_type},
                 {w, w_scales, experts * N, w_pitch, format_of(spec->w_e, spec->w_m), 0}, K, spec, workspace, workspace_bytes,
                 as_stream(stream));
}
