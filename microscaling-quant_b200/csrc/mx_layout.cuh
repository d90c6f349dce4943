// What the packed products take from mx_layout.cu: operands brought to the layout that their tensor maps and scale loads
// want. Host functions; each launches on the stream that it is given.
#pragma once
#include <cuda_runtime.h>
#include <cstdint>

namespace mxq {

// Rows of codes to 8-bit codes at a pitch of 16 bytes and, where to_scales is given, their scale rows to a pitch of 16
// bytes, zeros behind them. No rows: nothing to do.
struct LayJob {
  const uint8_t* codes;
  int64_t pitch;
  uint8_t* to_codes;
  int64_t out_pitch, rows, K;
  int fmt;
  int vec;                     // set by lay_rows: the rows of codes take 8-byte loads
  const uint8_t* scales;
  uint8_t* to_scales;
  int64_t scales_pitch;
};
int lay_rows(LayJob one, LayJob two, cudaStream_t st);

// Rows of floats (type: MXQ_OUT_*) to codes and scales, each at its pitch, with zeros behind a row of scales.
int pack_rows_to(const void* x, int type, int64_t x_stride, uint8_t* codes, int64_t out_pitch, uint8_t* scales, int64_t scales_pitch,
                 int64_t rows, int64_t K, int fmt, cudaStream_t st);

// The rows of x that the slots of a plan take, in the plan's order: K codes of each to a pitch of their own (a multiple of 16
// and at least K; zeros up to the next multiple of 16), ceil(K / 32) scale bytes side by side.
int gather_rows(const uint8_t* codes, const uint8_t* scales, int64_t pitch, int scales_pitch, const int* order, int per, int x_rows,
                int64_t slots, int64_t K, uint8_t* to_codes, int64_t to_pitch, uint8_t* to_scales, cudaStream_t st);

}  // namespace mxq
