// Operands of the packed products brought to the layout that the tensor maps take: codes of any MX format as 8-bit
// codes at a pitch of 16 bytes (k_lay_codes), and float rows packed on the way in (k_pack_rows). Both read their
// input once and write their output once; they are bound by those bytes. 8192 x 8192: packing float32 50 us (6.7
// TB/s), bf16 33 us (6.1); FP6 codes laid out 22.5 us (6.0; 24 with 64-bit indexes), FP4 21 us (4.9; 24), E4M3 rows of 8184
// 27 us (4.9; 28.5).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "mx_codes.cuh"
#include "mx_layout.cuh"

using namespace mxq;

namespace {

// The product that comes next on the stream may be launched while this grid is at work (it waits for its end before it
// reads anything).
__device__ __forceinline__ void start_next_grid() { asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory"); }

// four codes of one row -> one 32-bit word of 8-bit codes; `in` points at the row, c is a multiple of 4
__device__ __forceinline__ uint32_t lay4(const uint8_t* in, int64_t c, int64_t K, int fmt) {
  uint32_t w = 0;
  if (fmt == kFmtE2M1) {
    const uint32_t lo = in[c >> 1], hi = c + 2 < K ? in[(c >> 1) + 1] : 0u;
    return widen2(fmt, lo) | widen2(fmt, hi) << 16;
  }
#pragma unroll
  for (int j = 0; j < 4; j++)
    if (c + j < K) w |= (uint32_t)in[c + j] << (8 * j);
  if (fmt == kFmtE4M3 || fmt == kFmtE5M2) return w;
  return widen2(fmt, w & 0xffffu) | widen2(fmt, w >> 16) << 16;
}

// A thread per 16 codes of the output; its place beyond K is written as zeros (the tensor map never reads it). Then, for
// scale rows that are brought to a pitch of 16 bytes too, a thread per 16 of their bytes: zeros beyond the row, which
// the products do read. I: the index type, 32 bits while the threads' work is less than 2^31 (for the division).
template <typename I>
__device__ __forceinline__ void lay_codes(const LayJob& job, I first, I stride) {
  const int64_t K = job.K, pitch = job.pitch, out_pitch = job.out_pitch;
  const I per = (I)(out_pitch >> 4), n = (I)job.rows * per;
  const int fmt = job.fmt, vec = job.vec;
  const uint8_t* __restrict__ codes = job.codes;
  uint8_t* __restrict__ to_codes = job.to_codes;
  for (I i = first; i < n; i += stride) {
    const I at = i / per;
    const int64_t r = at, c = (int64_t)(i - at * per) << 4;
    const uint8_t* row = codes + r * pitch;
    uint32_t w[4];
    if (vec && c + 16 <= K) {                      // the row's words are aligned: 16 codes in one or two loads
      if (fmt == kFmtE2M1) {
        const uint2 q = __ldg(reinterpret_cast<const uint2*>(row + (c >> 1)));
        w[0] = widen2(fmt, q.x & 255u) | widen2(fmt, (q.x >> 8) & 255u) << 16;
        w[1] = widen2(fmt, (q.x >> 16) & 255u) | widen2(fmt, q.x >> 24) << 16;
        w[2] = widen2(fmt, q.y & 255u) | widen2(fmt, (q.y >> 8) & 255u) << 16;
        w[3] = widen2(fmt, (q.y >> 16) & 255u) | widen2(fmt, q.y >> 24) << 16;
      } else {
        const uint2 q0 = __ldg(reinterpret_cast<const uint2*>(row + c)), q1 = __ldg(reinterpret_cast<const uint2*>(row + c) + 1);
        w[0] = q0.x;
        w[1] = q0.y;
        w[2] = q1.x;
        w[3] = q1.y;
        if (fmt != kFmtE4M3 && fmt != kFmtE5M2) {
#pragma unroll
          for (int j = 0; j < 4; j++) w[j] = widen2(fmt, w[j] & 0xffffu) | widen2(fmt, w[j] >> 16) << 16;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++) w[j] = c + 4 * j < K ? lay4(row, c + 4 * j, K, fmt) : 0u;
    }
    *reinterpret_cast<uint4*>(to_codes + r * out_pitch + c) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  if (job.to_scales == nullptr) return;
  const int nb = (int)((K + 31) / 32);
  const I groups = (I)(job.scales_pitch >> 4), m = (I)job.rows * groups;
  for (I i = first; i < m; i += stride) {
    const int64_t r = i / groups;
    const int at = (int)(i - (I)r * groups) << 4;
    const uint8_t* row = job.scales + r * nb;
    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int j = 0; j < 16; j++)
      if (at + j < nb) w[j >> 2] |= (uint32_t)__ldg(row + at + j) << (8 * (j & 3));
    *reinterpret_cast<uint4*>(job.to_scales + r * job.scales_pitch + at) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// one or two operands in one launch: the blocks from `second` on take the other
template <typename I>
__global__ void __launch_bounds__(256) k_lay_codes(LayJob one, LayJob two, unsigned second) {
  start_next_grid();
  if (blockIdx.x < second)
    lay_codes<I>(one, (I)blockIdx.x * blockDim.x + threadIdx.x, (I)second * blockDim.x);
  else
    lay_codes<I>(two, (I)(blockIdx.x - second) * blockDim.x + threadIdx.x, (I)(gridDim.x - second) * blockDim.x);
}

// A warp per row of the product: the codes and scale bytes of the row of x that its slot takes, side by side in the
// order of the slots. x's rows may be any multiple of 16 bytes apart; of each only its K codes are read (the last row may end
// the caller's memory), and they are written at a pitch of their own, zeros up to it.
__global__ void __launch_bounds__(256) k_gather_rows(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t pitch,
                                                     int scales_pitch, const int* __restrict__ order, int per, int x_rows, int64_t slots,
                                                     int64_t K, int nb, uint8_t* __restrict__ to_codes, int64_t to_pitch,
                                                     uint8_t* __restrict__ to_scales) {
  start_next_grid();
  const int64_t r = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (r >= slots) return;
  const int slot = order[r];
  if (slot < 0) return;                                // a place without a slot: nobody reads it
  const int64_t from = min(slot / per, x_rows - 1);
  const uint4* a = reinterpret_cast<const uint4*>(codes + from * pitch);
  uint4* b = reinterpret_cast<uint4*>(to_codes + r * to_pitch);
#pragma unroll 4
  for (int64_t i = lane; i < K / 16; i += 32) b[i] = __ldg(a + i);
  if (const int left = (int)(K % 16)) {                // the last piece, byte by byte
    const int64_t at = K - left;
    if (lane < 16) to_codes[r * to_pitch + at + lane] = lane < left ? __ldg(codes + from * pitch + at + lane) : (uint8_t)0;
  }
  for (int i = lane; i < nb; i += 32) to_scales[r * nb + i] = __ldg(scales + from * scales_pitch + i);
}

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }

// Two lanes per block of 32: 16 values each, the block's largest |value| by a shuffle. VEC: 16-byte loads. I: the index
// type, 32 bits while the lanes are fewer than 2^31 (the division by the blocks of a row is what it is for).
template <typename T, bool VEC, int FMT, typename I>
__global__ void __launch_bounds__(256) k_pack_rows(const T* __restrict__ x, int64_t x_stride, uint8_t* __restrict__ codes,
                                                   int64_t out_pitch, uint8_t* __restrict__ scales, int64_t scales_pitch,
                                                   int64_t rows, int64_t K) {
  start_next_grid();
  constexpr int N = 16;
  const I nb = (I)((K + 31) / 32), n = (I)(rows * (int64_t)nb * 2), stride = (I)gridDim.x * blockDim.x;
  const I whole = (n + 31) / 32 * 32;                  // whole warps stay for the shuffle
  for (I i = (I)blockIdx.x * blockDim.x + threadIdx.x; i < whole; i += stride) {
    const I b = i >> 1, r = b / nb;
    const int64_t c = (int64_t)(b - r * nb) * 32 + (int)(i & 1) * N;
    const bool live = i < n;
    const T* from = x + (int64_t)r * x_stride + c;
    float v[N];
    if (VEC && live && c + N <= K) {
      uint4 t[sizeof(T)];
#pragma unroll
      for (int j = 0; j < (int)sizeof(T); j++) t[j] = __ldg(reinterpret_cast<const uint4*>(from) + j);
#pragma unroll
      for (int j = 0; j < N; j++) v[j] = to_float<T>(reinterpret_cast<const T*>(t)[j]);
    } else {
#pragma unroll
      for (int j = 0; j < N; j++) v[j] = live && c + j < K ? to_float<T>(from[j]) : 0.0f;
    }
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < N; j++) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
    top = max(top, __shfl_xor_sync(~0u, top, 1));
    const uint32_t sb = scale_byte(top, FMT);
    const float inv = scale_inverse(sb);
    uint32_t q[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      uint32_t h[2];
#pragma unroll
      for (int p = 0; p < 2; p++) {
        h[p] = encode2(FMT, __fmul_rn(v[4 * j + 2 * p], inv), __fmul_rn(v[4 * j + 2 * p + 1], inv));
        if (FMT > kFmtE5M2) h[p] = widen2(FMT, h[p]);
      }
      q[j] = sb == 255u ? 0u : h[0] | h[1] << 16;      // a block with an Inf or a NaN: its scale says so
    }
    if (!live) continue;
    if ((i & 1) == 0) {
      if (scales_pitch == (int64_t)nb) {
        scales[b] = (uint8_t)sb;
      } else {                                         // a pitch beyond the row is read as zeros
        const int at = (int)(b - r * nb);
        uint8_t* to = scales + (int64_t)r * scales_pitch;
        to[at] = (uint8_t)sb;
        if (at + 1 == (int)nb)
          for (int64_t j = nb; j < scales_pitch; j++) to[j] = 0;
      }
    }
    if (c < out_pitch)                                 // the pitch is a multiple of 16, as c is
      *reinterpret_cast<uint4*>(codes + (int64_t)r * out_pitch + c) = make_uint4(q[0], q[1], q[2], q[3]);
  }
}

template <typename T, int FMT>
int pack_rows(const void* x, int64_t x_stride, uint8_t* codes, int64_t out_pitch, uint8_t* scales, int64_t scales_pitch, int64_t rows,
              int64_t K, cudaStream_t st) {
  const int64_t n = rows * ((K + 31) / 32) * 2;
  const unsigned grid = grid_for(n, 256, 16);
  const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && x_stride * (int64_t)sizeof(T) % 16 == 0;
  const bool small = n < (1ll << 31) - (int64_t)grid * 256 - 64;
  auto f = vec ? (small ? k_pack_rows<T, true, FMT, uint32_t> : k_pack_rows<T, true, FMT, int64_t>)
               : (small ? k_pack_rows<T, false, FMT, uint32_t> : k_pack_rows<T, false, FMT, int64_t>);
  f<<<grid, 256, 0, st>>>(static_cast<const T*>(x), x_stride, codes, out_pitch, scales, scales_pitch, rows, K);
  return MXQ_LAUNCH_CHECK("pack_rows");
}
template <typename T>
int pack_rows(const void* x, int64_t x_stride, uint8_t* codes, int64_t out_pitch, uint8_t* scales, int64_t scales_pitch, int64_t rows,
              int64_t K, int fmt, cudaStream_t st) {
  switch (fmt) {
    case kFmtE4M3: return pack_rows<T, kFmtE4M3>(x, x_stride, codes, out_pitch, scales, scales_pitch, rows, K, st);
    case kFmtE5M2: return pack_rows<T, kFmtE5M2>(x, x_stride, codes, out_pitch, scales, scales_pitch, rows, K, st);
    case kFmtE3M2: return pack_rows<T, kFmtE3M2>(x, x_stride, codes, out_pitch, scales, scales_pitch, rows, K, st);
    case kFmtE2M3: return pack_rows<T, kFmtE2M3>(x, x_stride, codes, out_pitch, scales, scales_pitch, rows, K, st);
    default: return pack_rows<T, kFmtE2M1>(x, x_stride, codes, out_pitch, scales, scales_pitch, rows, K, st);
  }
}

}  // namespace

namespace mxq {
int gather_rows(const uint8_t* codes, const uint8_t* scales, int64_t pitch, int scales_pitch, const int* order, int per, int x_rows,
                int64_t slots, int64_t K, uint8_t* to_codes, int64_t to_pitch, uint8_t* to_scales, cudaStream_t st) {
  k_gather_rows<<<(unsigned)((slots + 7) / 8), 256, 0, st>>>(codes, scales, pitch, scales_pitch, order, per, x_rows, slots, K,
                                                             (int)((K + 31) / 32), to_codes, to_pitch, to_scales);
  return MXQ_LAUNCH_CHECK("gather_rows");
}

static unsigned lay_grid(const LayJob& j) {
  return j.rows > 0 ? grid_for(j.rows * (j.out_pitch / 16), 256, 16) : 0u;     // a row has more codes than scales
}
int lay_rows(LayJob one, LayJob two, cudaStream_t st) {
  const unsigned a = lay_grid(one), b = lay_grid(two);
  if (a + b == 0) return MXQ_OK;
  for (LayJob* j : {&one, &two}) j->vec = reinterpret_cast<uintptr_t>(j->codes) % 8 == 0 && j->pitch % 8 == 0;
  const int64_t most = (one.rows * one.out_pitch > two.rows * two.out_pitch ? one.rows * one.out_pitch : two.rows * two.out_pitch) / 16;
  auto f = most < (1ll << 31) - (int64_t)(a + b) * 256 ? k_lay_codes<uint32_t> : k_lay_codes<int64_t>;
  f<<<a + b, 256, 0, st>>>(one, two, a);
  return MXQ_LAUNCH_CHECK("lay_codes");
}

int pack_rows_to(const void* x, int type, int64_t x_stride, uint8_t* codes, int64_t out_pitch, uint8_t* scales, int64_t scales_pitch,
                 int64_t rows, int64_t K, int fmt, cudaStream_t st) {
  if (rows == 0) return MXQ_OK;
  if (type == MXQ_OUT_F32) return pack_rows<float>(x, x_stride, codes, out_pitch, scales, scales_pitch, rows, K, fmt, st);
  if (type == MXQ_OUT_BF16) return pack_rows<__nv_bfloat16>(x, x_stride, codes, out_pitch, scales, scales_pitch, rows, K, fmt, st);
  if (type == MXQ_OUT_F16) return pack_rows<__half>(x, x_stride, codes, out_pitch, scales, scales_pitch, rows, K, fmt, st);
  return set_error(MXQ_ERR_VALUE, "pack_rows: type %d", type);
}
}  // namespace mxq

extern "C" int mxq_lay_codes(const uint8_t* codes, int64_t in_pitch, uint8_t* out, int64_t out_pitch, int64_t rows, int64_t K,
                             int32_t e, int32_t m, void* stream) {
  const int fmt = format_of(e, m);
  MXQ_REQUIRE(fmt != kFmtNone, MXQ_ERR_VALUE, "lay_codes: (e=%d, m=%d) is not an MX element format", e, m);
  MXQ_REQUIRE(rows >= 0 && K >= 1 && out_pitch >= K && out_pitch % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0,
              MXQ_ERR_VALUE, "lay_codes: rows %lld, K %lld, output pitch %lld", (long long)rows, (long long)K, (long long)out_pitch);
  MXQ_REQUIRE(fmt != kFmtE2M1 || K % 2 == 0, MXQ_ERR_VALUE, "lay_codes: FP4 codes pair up, K is %lld", (long long)K);
  return lay_rows({codes, in_pitch, out, out_pitch, rows, K, fmt, 0, nullptr, nullptr, 0}, {}, as_stream(stream));
}

extern "C" int mxq_pack_rows(const void* x, int32_t type, int64_t x_stride, uint8_t* codes, int64_t out_pitch, uint8_t* scales,
                             int64_t rows, int64_t K, int32_t e, int32_t m, void* stream) {
  const int fmt = format_of(e, m);
  MXQ_REQUIRE(fmt != kFmtNone, MXQ_ERR_VALUE, "pack_rows: (e=%d, m=%d) is not an MX element format", e, m);
  MXQ_REQUIRE(rows >= 0 && K >= 1 && out_pitch >= K && out_pitch % 16 == 0 && reinterpret_cast<uintptr_t>(codes) % 16 == 0,
              MXQ_ERR_VALUE, "pack_rows: rows %lld, K %lld, output pitch %lld", (long long)rows, (long long)K, (long long)out_pitch);
  return pack_rows_to(x, type, x_stride, codes, out_pitch, scales, (K + 31) / 32, rows, K, fmt, as_stream(stream));
}
