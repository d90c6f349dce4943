// Operands of the packed products brought to the layout that the tensor maps take: codes of any MX format as 8-bit codes
// at a pitch of 16 bytes (k_lay_codes), and float rows packed on the way in (k_pack_rows). Both read their input once and
// write their output once; they are bound by those bytes.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "mx_codes.cuh"

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

// a thread per 16 codes of the output; its place beyond K is written as zeros (the tensor map never reads it)
__global__ void __launch_bounds__(256) k_lay_codes(const uint8_t* __restrict__ in, int64_t in_pitch, uint8_t* __restrict__ out,
                                                   int64_t out_pitch, int64_t rows, int64_t K, int fmt, int vec) {
  start_next_grid();
  const int64_t per = out_pitch >> 4, n = rows * per, stride = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += stride) {
    const int64_t r = i / per, c = (i - r * per) << 4;
    const uint8_t* row = in + r * in_pitch;
    uint32_t w[4];
    if (vec && c + 16 <= K) {                          // the row's words are aligned: 16 codes in one or two loads
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
    *reinterpret_cast<uint4*>(out + r * out_pitch + c) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// A warp per row of the product: the codes and scale bytes of the row of x that its slot takes, side by side in the order
// of the slots.
__global__ void __launch_bounds__(256) k_gather_rows(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t pitch,
                                                     const int* __restrict__ order, int per, int x_rows, int64_t slots, int nb,
                                                     uint8_t* __restrict__ to_codes, uint8_t* __restrict__ to_scales) {
  start_next_grid();
  const int64_t r = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (r >= slots) return;
  const int slot = order[r];
  if (slot < 0) return;                                // a place without a slot: nobody reads it
  const int64_t from = min(slot / per, x_rows - 1);
  const uint4* a = reinterpret_cast<const uint4*>(codes + from * pitch);
  uint4* b = reinterpret_cast<uint4*>(to_codes + r * pitch);
#pragma unroll 4
  for (int64_t i = lane; i < pitch / 16; i += 32) b[i] = __ldg(a + i);
  for (int i = lane; i < nb; i += 32) to_scales[r * nb + i] = __ldg(scales + from * nb + i);
}

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }

// Four lanes per block of 32: 8 values each, the block's largest |value| by two shuffles. VEC: 16-byte loads.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) k_pack_rows(const T* __restrict__ x, int64_t x_stride, uint8_t* __restrict__ codes,
                                                   int64_t out_pitch, uint8_t* __restrict__ scales, int64_t rows, int64_t K, int fmt) {
  start_next_grid();
  const int64_t nb = (K + 31) / 32, n = rows * nb * 4, stride = (int64_t)gridDim.x * blockDim.x;
  const int64_t n32 = (n + 31) / 32 * 32;              // whole warps stay for the shuffles
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n32; i += stride) {
    const int64_t b = i >> 2, r = b / nb, c = (b - r * nb) * 32 + (i & 3) * 8;
    float v[8];
    uint32_t top = 0;
    const bool live = i < n;
    if (VEC && live && c + 8 <= K) {
      const uint4* from = reinterpret_cast<const uint4*>(x + r * x_stride + c);
      T t[8];
#pragma unroll
      for (int j = 0; j < (int)(sizeof(T) / 2); j++) reinterpret_cast<uint4*>(t)[j] = __ldg(from + j);
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = to_float<T>(t[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = live && c + j < K ? to_float<T>(x[r * x_stride + c + j]) : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < 8; j++) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
    top = max(top, __shfl_xor_sync(~0u, top, 1));
    top = max(top, __shfl_xor_sync(~0u, top, 2));
    const uint32_t sb = scale_byte(top, fmt);
    const float inv = scale_inverse(sb);
    uint32_t q[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      q[j] = encode2(fmt, scaled(v[2 * j], inv), scaled(v[2 * j + 1], inv));
      if (fmt > kFmtE5M2) q[j] = widen2(fmt, q[j]);
    }
    if (!live) continue;
    if ((i & 3) == 0) scales[b] = (uint8_t)sb;
    if (c < out_pitch)                                 // the pitch is a multiple of 16, c of 8
      *reinterpret_cast<uint2*>(codes + r * out_pitch + c) = make_uint2(q[0] | q[1] << 16, q[2] | q[3] << 16);
  }
}

template <typename T>
int pack_rows(const void* x, int64_t x_stride, uint8_t* codes, int64_t out_pitch, uint8_t* scales, int64_t rows, int64_t K, int fmt,
              cudaStream_t st) {
  const int64_t n = rows * ((K + 31) / 32) * 4;
  const unsigned grid = grid_for(n, 256, 16);
  const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && x_stride * (int64_t)sizeof(T) % 16 == 0;
  if (vec)
    k_pack_rows<T, true><<<grid, 256, 0, st>>>(static_cast<const T*>(x), x_stride, codes, out_pitch, scales, rows, K, fmt);
  else
    k_pack_rows<T, false><<<grid, 256, 0, st>>>(static_cast<const T*>(x), x_stride, codes, out_pitch, scales, rows, K, fmt);
  return MXQ_LAUNCH_CHECK("pack_rows");
}

}  // namespace

namespace mxq {
int gather_rows(const uint8_t* codes, const uint8_t* scales, int64_t pitch, const int* order, int per, int x_rows, int64_t slots, int nb,
                uint8_t* to_codes, uint8_t* to_scales, cudaStream_t st) {
  k_gather_rows<<<(unsigned)((slots + 7) / 8), 256, 0, st>>>(codes, scales, pitch, order, per, x_rows, slots, nb, to_codes, to_scales);
  return MXQ_LAUNCH_CHECK("gather_rows");
}
}  // namespace mxq

extern "C" int mxq_lay_codes(const uint8_t* codes, int64_t in_pitch, uint8_t* out, int64_t out_pitch, int64_t rows, int64_t K,
                             int32_t e, int32_t m, void* stream) {
  const int fmt = format_of(e, m);
  MXQ_REQUIRE(fmt != kFmtNone, MXQ_ERR_VALUE, "lay_codes: (e=%d, m=%d) is not an MX element format", e, m);
  MXQ_REQUIRE(rows >= 0 && K >= 1 && out_pitch >= K && out_pitch % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0,
              MXQ_ERR_VALUE, "lay_codes: rows %lld, K %lld, output pitch %lld", (long long)rows, (long long)K, (long long)out_pitch);
  MXQ_REQUIRE(fmt != kFmtE2M1 || K % 2 == 0, MXQ_ERR_VALUE, "lay_codes: FP4 codes pair up, K is %lld", (long long)K);
  if (rows == 0) return MXQ_OK;
  const int vec = reinterpret_cast<uintptr_t>(codes) % 8 == 0 && in_pitch % 8 == 0;
  k_lay_codes<<<grid_for(rows * (out_pitch / 16), 256, 16), 256, 0, as_stream(stream)>>>(codes, in_pitch, out, out_pitch, rows, K, fmt, vec);
  return MXQ_LAUNCH_CHECK("lay_codes");
}

extern "C" int mxq_pack_rows(const void* x, int32_t type, int64_t x_stride, uint8_t* codes, int64_t out_pitch, uint8_t* scales,
                             int64_t rows, int64_t K, int32_t e, int32_t m, void* stream) {
  const int fmt = format_of(e, m);
  MXQ_REQUIRE(fmt != kFmtNone, MXQ_ERR_VALUE, "pack_rows: (e=%d, m=%d) is not an MX element format", e, m);
  MXQ_REQUIRE(rows >= 0 && K >= 1 && out_pitch >= K && out_pitch % 16 == 0 && reinterpret_cast<uintptr_t>(codes) % 16 == 0,
              MXQ_ERR_VALUE, "pack_rows: rows %lld, K %lld, output pitch %lld", (long long)rows, (long long)K, (long long)out_pitch);
  if (rows == 0) return MXQ_OK;
  cudaStream_t st = as_stream(stream);
  if (type == MXQ_OUT_F32) return pack_rows<float>(x, x_stride, codes, out_pitch, scales, rows, K, fmt, st);
  if (type == MXQ_OUT_BF16) return pack_rows<__nv_bfloat16>(x, x_stride, codes, out_pitch, scales, rows, K, fmt, st);
  if (type == MXQ_OUT_F16) return pack_rows<__half>(x, x_stride, codes, out_pitch, scales, rows, K, fmt, st);
  return set_error(MXQ_ERR_VALUE, "pack_rows: type %d", type);
}
