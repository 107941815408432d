// generated by lego_amd (python -m lego_amd.build) -- do not edit; edit the generator
#pragma once
#include <hip/hip_runtime.h>

hipError_t lego_transpose_any_launch(const void*, void*, int, int, int, hipStream_t);
hipError_t lego_transpose_f32_64x128_w64x8_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_transpose_f32_64x128_w32x8_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_transpose_f32_32x256_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_transpose_f32_64x64_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_transpose_f32_128x32_edge_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_transpose_f32_64x128_edge_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_transpose_f32_128x32_ragged_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_transpose_f32_64x64_ragged_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_transpose_f32_128x64_ragged_launch(const void*, void*, int, int, hipStream_t);
// picks the first tiling that divides the shape; any other shape takes the tiling with vectors at any element and edge tests, a tiny matrix the one-element-per-access kernel
inline hipError_t lego_transpose_f32_dispatch(const void* in, void* out, int rows, int cols, hipStream_t stream) {
  if (rows % 4096 == 0 && cols % 1024 == 0 && 2ull * rows * cols * 4 <= 1610612736ull) return lego_transpose_f32_64x128_w64x8_launch(in, out, rows, cols, stream);
  if (rows % 2048 == 0 && cols % 1024 == 0 && 2ull * rows * cols * 4 <= 1610612736ull) return lego_transpose_f32_64x128_w32x8_launch(in, out, rows, cols, stream);
  if (rows % 32 == 0 && cols % 256 == 0 && 1ull * rows * cols >= 2097152ull) return lego_transpose_f32_32x256_launch(in, out, rows, cols, stream);
  if (rows % 64 == 0 && cols % 64 == 0) return lego_transpose_f32_64x64_launch(in, out, rows, cols, stream);
  if (rows % 4 == 0 && cols % 4 == 0 && 1ull * rows * cols >= 33554432ull && 1ull * rows * cols <= 402653184ull) return lego_transpose_f32_128x32_edge_launch(in, out, rows, cols, stream);
  if (rows % 4 == 0 && cols % 4 == 0 && 1ull * rows * cols >= 33554432ull) return lego_transpose_f32_64x128_edge_launch(in, out, rows, cols, stream);
  if (rows % 1 == 0 && cols % 1 == 0 && rows >= 4 && cols >= 4 && 1ull * rows * cols >= 3145728ull) return lego_transpose_f32_128x32_ragged_launch(in, out, rows, cols, stream);
  if (rows % 1 == 0 && cols % 1 == 0 && rows >= 4 && cols >= 4 && 1ull * rows * cols >= 16384ull) return lego_transpose_f32_64x64_ragged_launch(in, out, rows, cols, stream);
  return lego_transpose_any_launch(in, out, rows, cols, 4, stream);
}
// matrices whose base is only element aligned (a sliced view): the tilings whose vectors sit at any element
inline hipError_t lego_transpose_f32_dispatch_any_base(const void* in, void* out, int rows, int cols, hipStream_t stream) {
  if (rows >= 4 && cols >= 4 && 1ull * rows * cols >= 3145728ull) return lego_transpose_f32_128x32_ragged_launch(in, out, rows, cols, stream);
  if (rows >= 4 && cols >= 4 && 1ull * rows * cols >= 16384ull) return lego_transpose_f32_64x64_ragged_launch(in, out, rows, cols, stream);
  return lego_transpose_any_launch(in, out, rows, cols, 4, stream);
}
// tiling number `tiling` of the list above, for a shape it takes (16-byte aligned bases); the caller compares tilings with it
inline hipError_t lego_transpose_f32_tiling(int tiling, const void* in, void* out, int rows, int cols, hipStream_t stream) {
  if (tiling == 0 && rows % 4096 == 0 && cols % 1024 == 0) return lego_transpose_f32_64x128_w64x8_launch(in, out, rows, cols, stream);      // 64 x 128
  if (tiling == 1 && rows % 2048 == 0 && cols % 1024 == 0) return lego_transpose_f32_64x128_w32x8_launch(in, out, rows, cols, stream);      // 64 x 128
  if (tiling == 2 && rows % 32 == 0 && cols % 256 == 0) return lego_transpose_f32_32x256_launch(in, out, rows, cols, stream);      // 32 x 256
  if (tiling == 3 && rows % 64 == 0 && cols % 64 == 0) return lego_transpose_f32_64x64_launch(in, out, rows, cols, stream);      // 64 x 64
  if (tiling == 4 && rows % 4 == 0 && cols % 4 == 0) return lego_transpose_f32_128x32_edge_launch(in, out, rows, cols, stream);      // 128 x 32
  if (tiling == 5 && rows % 4 == 0 && cols % 4 == 0) return lego_transpose_f32_64x128_edge_launch(in, out, rows, cols, stream);      // 64 x 128
  if (tiling == 6 && rows % 1 == 0 && cols % 1 == 0 && rows >= 4 && cols >= 4) return lego_transpose_f32_128x32_ragged_launch(in, out, rows, cols, stream);      // 128 x 32
  if (tiling == 7 && rows % 1 == 0 && cols % 1 == 0 && rows >= 4 && cols >= 4) return lego_transpose_f32_64x64_ragged_launch(in, out, rows, cols, stream);      // 64 x 64
  if (tiling == 8 && rows % 1 == 0 && cols % 1 == 0 && rows >= 4 && cols >= 4) return lego_transpose_f32_128x64_ragged_launch(in, out, rows, cols, stream);      // 128 x 64
  return hipErrorInvalidValue;
}

hipError_t lego_transpose_f16_64x256_w128x8_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_transpose_f16_64x256_w64x8_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_transpose_f16_64x256_w32x8_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_transpose_f16_64x256_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_transpose_f16_64x64_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_transpose_f16_256x64_edge_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_transpose_f16_256x64_ragged_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_transpose_f16_64x64_ragged_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_transpose_f16_128x128_edge_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_transpose_f16_128x128_ragged_launch(const void*, void*, int, int, hipStream_t);
// picks the first tiling that divides the shape; any other shape takes the tiling with vectors at any element and edge tests, a tiny matrix the one-element-per-access kernel
inline hipError_t lego_transpose_f16_dispatch(const void* in, void* out, int rows, int cols, hipStream_t stream) {
  if (rows % 8192 == 0 && cols % 2048 == 0) return lego_transpose_f16_64x256_w128x8_launch(in, out, rows, cols, stream);
  if (rows % 4096 == 0 && cols % 2048 == 0) return lego_transpose_f16_64x256_w64x8_launch(in, out, rows, cols, stream);
  if (rows % 2048 == 0 && cols % 2048 == 0) return lego_transpose_f16_64x256_w32x8_launch(in, out, rows, cols, stream);
  if (rows % 64 == 0 && cols % 256 == 0 && 1ull * rows * cols >= 2097152ull) return lego_transpose_f16_64x256_launch(in, out, rows, cols, stream);
  if (rows % 64 == 0 && cols % 64 == 0) return lego_transpose_f16_64x64_launch(in, out, rows, cols, stream);
  if (rows % 8 == 0 && cols % 8 == 0 && 1ull * rows * cols >= 33554432ull) return lego_transpose_f16_256x64_edge_launch(in, out, rows, cols, stream);
  if (rows % 1 == 0 && cols % 1 == 0 && rows >= 8 && cols >= 8 && 1ull * rows * cols >= 41943040ull) return lego_transpose_f16_256x64_ragged_launch(in, out, rows, cols, stream);
  if (rows % 1 == 0 && cols % 1 == 0 && rows >= 8 && cols >= 8 && 1ull * rows * cols >= 16384ull) return lego_transpose_f16_64x64_ragged_launch(in, out, rows, cols, stream);
  return lego_transpose_any_launch(in, out, rows, cols, 2, stream);
}
// matrices whose base is only element aligned (a sliced view): the tilings whose vectors sit at any element
inline hipError_t lego_transpose_f16_dispatch_any_base(const void* in, void* out, int rows, int cols, hipStream_t stream) {
  if (rows >= 8 && cols >= 8 && 1ull * rows * cols >= 41943040ull) return lego_transpose_f16_256x64_ragged_launch(in, out, rows, cols, stream);
  if (rows >= 8 && cols >= 8 && 1ull * rows * cols >= 16384ull) return lego_transpose_f16_64x64_ragged_launch(in, out, rows, cols, stream);
  return lego_transpose_any_launch(in, out, rows, cols, 2, stream);
}
// tiling number `tiling` of the list above, for a shape it takes (16-byte aligned bases); the caller compares tilings with it
inline hipError_t lego_transpose_f16_tiling(int tiling, const void* in, void* out, int rows, int cols, hipStream_t stream) {
  if (tiling == 0 && rows % 8192 == 0 && cols % 2048 == 0) return lego_transpose_f16_64x256_w128x8_launch(in, out, rows, cols, stream);      // 64 x 256
  if (tiling == 1 && rows % 4096 == 0 && cols % 2048 == 0) return lego_transpose_f16_64x256_w64x8_launch(in, out, rows, cols, stream);      // 64 x 256
  if (tiling == 2 && rows % 2048 == 0 && cols % 2048 == 0) return lego_transpose_f16_64x256_w32x8_launch(in, out, rows, cols, stream);      // 64 x 256
  if (tiling == 3 && rows % 64 == 0 && cols % 256 == 0) return lego_transpose_f16_64x256_launch(in, out, rows, cols, stream);      // 64 x 256
  if (tiling == 4 && rows % 64 == 0 && cols % 64 == 0) return lego_transpose_f16_64x64_launch(in, out, rows, cols, stream);      // 64 x 64
  if (tiling == 5 && rows % 8 == 0 && cols % 8 == 0) return lego_transpose_f16_256x64_edge_launch(in, out, rows, cols, stream);      // 256 x 64
  if (tiling == 6 && rows % 1 == 0 && cols % 1 == 0 && rows >= 8 && cols >= 8) return lego_transpose_f16_256x64_ragged_launch(in, out, rows, cols, stream);      // 256 x 64
  if (tiling == 7 && rows % 1 == 0 && cols % 1 == 0 && rows >= 8 && cols >= 8) return lego_transpose_f16_64x64_ragged_launch(in, out, rows, cols, stream);      // 64 x 64
  if (tiling == 8 && rows % 8 == 0 && cols % 8 == 0) return lego_transpose_f16_128x128_edge_launch(in, out, rows, cols, stream);      // 128 x 128
  if (tiling == 9 && rows % 1 == 0 && cols % 1 == 0 && rows >= 8 && cols >= 8) return lego_transpose_f16_128x128_ragged_launch(in, out, rows, cols, stream);      // 128 x 128
  return hipErrorInvalidValue;
}

hipError_t lego_softmax_f16_w1_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_f16_w1_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_f16_w2_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_f16_w2_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_f16_w4_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_f16_w4_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_f16_w8_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_f16_w8_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_f32_w1_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_f32_w1_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_f32_w4_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_f32_w4_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_f32_w8_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_f32_w8_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_f16s_w1_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_f16s_w1_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_f32s_w1_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_f32s_w1_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_f16s_w4_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_f16s_w4_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_f32s_w4_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_f32s_w4_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_f16s_w8_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_f16s_w8_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_bf16s_w8_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_bf16s_w8_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_f32s_w8_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_f32s_w8_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_f16_w16_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_f16_w16_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_f32_w16_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_f32_w16_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_f16s_w16_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_f16s_w16_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_f32s_w16_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_f32s_w16_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_bf16_w1_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_bf16_w1_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_bf16_w4_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_bf16_w4_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_bf16_w8_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_bf16_w8_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_bf16_w16_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_bf16_w16_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_bf16s_w1_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_bf16s_w1_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_bf16s_w4_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_bf16s_w4_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_bf16s_w16_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_bf16s_w16_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_f16_l16_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_f16_l16_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_f16s_l16_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_f16s_l16_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_f16_l32_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_f16_l32_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_f16s_l32_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_f16s_l32_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_bf16_l16_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_bf16_l16_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_bf16s_l16_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_bf16s_l16_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_bf16_l32_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_bf16_l32_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_bf16s_l32_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_bf16s_l32_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_f32_l16_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_f32_l16_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_f32s_l16_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_f32s_l16_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_f32_l32_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_f32_l32_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_f32s_l32_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_layernorm_fwd_f32s_l32_launch(const void*, void*, const void*, const void*, float*, float*, int, int, float, hipStream_t);
hipError_t lego_softmax_long_f16_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_softmax_long_bf16_launch(const void*, void*, int, int, hipStream_t);
hipError_t lego_softmax_long_f32_launch(const void*, void*, int, int, hipStream_t);
#define LEGO_ROWWISE_MAX_N 32768
#define LEGO_ROWWISE_MAX_N_SMALL_TEAMS 16384
// waves per row: one wave keeps short rows free of barriers, four waves keep the
// register footprint of long rows small enough for full occupancy, sixteen (a whole
// workgroup of 1024 lanes) hold the rows that four cannot
inline int lego_rowwise_default_wpr(int n) { return n <= 2048 ? 1 : n <= 16384 ? 4 : 16; }
// 16-bit rows of whole vectors: eight waves (a workgroup of 512 lanes, two to four vectors per lane) for long
// rows of tall matrices, where they measure 3-5 % above four waves; fewer rows leave too few workgroups
// ... and two waves (two rows per workgroup) for 2049-4096 rows of 2049-4096 elements: one round of workgroups on
// the 256 CUs instead of two (4096 x 4096: softmax 4.9 -> 5.4 TB/s, LayerNorm 4.4 -> 5.0; no gain from 8192 rows on)
// ... and for rows of 1537-2048 elements, which one wave holds as four vectors per lane, of matrices of 16384 rows
// and more (2-5 % above one wave there, 1-11 % below it at 8192 rows)
inline int lego_rowwise_f16_wpr(int m, int n) { return n > 6144 && n <= 16384 && m >= 4096 ? 8 : n > 2048 && n <= 4096 && m > 2048 && m <= 4096 ? 2 : n > 1536 && n <= 2048 && m >= 16384 ? 2 : lego_rowwise_default_wpr(n); }

unsigned lego_layernorm_bwd_groups(int M, int N);
unsigned lego_layernorm_bwd_f32_groups(int M, int N);
unsigned lego_layernorm_bwd_bf16_groups(int M, int N);
hipError_t lego_layernorm_bwd_f32_launch(const void*, const void*, const void*, const float*, const float*, void*, void*, void*, float*, int, int, int, hipStream_t);
hipError_t lego_layernorm_bwd_bf16_launch(const void*, const void*, const void*, const float*, const float*, void*, void*, void*, float*, int, int, int, hipStream_t);
hipError_t lego_layernorm_bwd_f16_launch(const void*, const void*, const void*, const float*, const float*, void*, void*, void*, float*, int, int, int, hipStream_t);
#define LEGO_LAYERNORM_BWD_MAX_N 32768

hipError_t lego_gemm_f16_nn_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_f16_nn_t128x128_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_f16_nn_t128x128_deep_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_f16_nt_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_f16_nt_t128x128_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_f16_nt_t128x128_deep_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_f16_tn_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_f16_tn_t128x128_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_f16_tn_t128x128_deep_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_f16_tt_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_f16_tt_t128x128_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_f16_tt_t128x128_deep_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_bf16_nn_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_bf16_nn_t128x128_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_bf16_nn_t128x128_deep_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_bf16_nt_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_bf16_nt_t128x128_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_bf16_nt_t128x128_deep_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_bf16_tn_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_bf16_tn_t128x128_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_bf16_tn_t128x128_deep_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_bf16_tt_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_bf16_tt_t128x128_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_bf16_tt_t128x128_deep_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_bf16h_nn_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_bf16h_nn_t128x128_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_bf16h_nn_t128x128_deep_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_bf16h_nt_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_bf16h_nt_t128x128_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_bf16h_nt_t128x128_deep_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_bf16h_tn_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_bf16h_tn_t128x128_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_bf16h_tn_t128x128_deep_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_bf16h_tt_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_bf16h_tt_t128x128_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_bf16h_tt_t128x128_deep_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_e4m3_nn_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_e4m3_nn_t128x128_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_e4m3_nn_t128x128_deep_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_e4m3_nt_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_e4m3_nt_t128x128_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_e4m3_nt_t128x128_deep_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_e4m3_tn_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_e4m3_tn_t128x128_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_e4m3_tn_t128x128_deep_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_e4m3_tt_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_e4m3_tt_t128x128_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_e4m3_tt_t128x128_deep_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_e5m2_nn_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_e5m2_nn_t128x128_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_e5m2_nn_t128x128_deep_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_e5m2_nt_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_e5m2_nt_t128x128_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_e5m2_nt_t128x128_deep_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_e5m2_tn_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_e5m2_tn_t128x128_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_e5m2_tn_t128x128_deep_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_e5m2_tt_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_e5m2_tt_t128x128_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_e5m2_tt_t128x128_deep_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_f16_nn_t128x128_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_f16_nn_t128x128_deep_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_f16_nt_t128x128_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_f16_nt_t128x128_deep_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_f16_tn_t128x128_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_f16_tn_t128x128_deep_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_f16_tt_t128x128_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_f16_tt_t128x128_deep_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_bf16_nn_t128x128_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_bf16_nn_t128x128_deep_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_bf16_nt_t128x128_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_bf16_nt_t128x128_deep_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_bf16_tn_t128x128_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_bf16_tn_t128x128_deep_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_bf16_tt_t128x128_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_bf16_tt_t128x128_deep_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_bf16h_nn_t128x128_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_bf16h_nn_t128x128_deep_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_bf16h_nt_t128x128_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_bf16h_nt_t128x128_deep_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_bf16h_tn_t128x128_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_bf16h_tn_t128x128_deep_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_bf16h_tt_t128x128_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_bf16h_tt_t128x128_deep_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_e4m3_nn_t128x128_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_e4m3_nn_t128x128_deep_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_e4m3_nt_t128x128_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_e4m3_nt_t128x128_deep_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_e4m3_tn_t128x128_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_e4m3_tn_t128x128_deep_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_e4m3_tt_t128x128_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_e4m3_tt_t128x128_deep_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_e5m2_nn_t128x128_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_e5m2_nn_t128x128_deep_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_e5m2_nt_t128x128_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_e5m2_nt_t128x128_deep_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_e5m2_tn_t128x128_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_e5m2_tn_t128x128_deep_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_e5m2_tt_t128x128_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_gemm_e5m2_tt_t128x128_deep_splitk_launch(const void*, const void*, void*, int, int, int, int, int, float*, hipStream_t);
hipError_t lego_grouped_gemm_f16_launch(const void* const*, const void* const*, void* const*, const int*, int, hipStream_t);
hipError_t lego_grouped_gemm_f16_t128x128_launch(const void* const*, const void* const*, void* const*, const int*, int, hipStream_t);
hipError_t lego_grouped_gemm_f16_t128x128_deep_launch(const void* const*, const void* const*, void* const*, const int*, int, hipStream_t);
hipError_t lego_grouped_gemm_f16_t128x128_deep_parts_launch(const void* const*, const void* const*, void* const*, const int*, int, int, float*, hipStream_t);
hipError_t lego_gemm_f16_nn_w2x4_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_f16_nn_m32_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_f16_nt_m32_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_f16_tn_m32_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_f16_tt_m32_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_bf16_nn_m32_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_bf16_nt_m32_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_bf16_tn_m32_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_bf16_tt_m32_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_bf16h_nn_m32_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_bf16h_nt_m32_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_bf16h_tn_m32_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_bf16h_tt_m32_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_gemm_f16_nn_stamps_launch(const void*, const void*, void*, int, int, int, int, hipStream_t);
hipError_t lego_grouped_gemm_f16_stamps_launch(const void* const*, const void* const*, void* const*, const int*, int, hipStream_t);
hipError_t lego_grouped_gemm_f16_stamps_split_launch(const void* const*, const void* const*, void* const*, const int*, int, int, hipStream_t);
hipError_t lego_gemm_stamps_read(unsigned long long*, int);
hipError_t lego_gemm_any_launch(const void*, const void*, void*, int, int, int, int, int, int, int, hipStream_t);
hipError_t lego_gemm_rows_launch(const void*, const void*, void*, int, int, int, int, int, int, hipStream_t);
hipError_t lego_grouped_gemm_f16_split_launch(const void* const*, const void* const*, void* const*, const int*, int, int, hipStream_t);
#define LEGO_GEMM_BM 256
#define LEGO_GEMM_BN 256
#define LEGO_GEMM_BK 64
#define LEGO_GEMM_BK_8BIT 128
#define LEGO_GROUPED_MAX_GROUPS 64

hipError_t lego_nw_i32_launch(const int*, int*, int, int, hipStream_t);
unsigned long long lego_nw_i32_strips_words(int);
hipError_t lego_nw_i32_strips_launch(const int*, int*, int, int, unsigned long long*, hipStream_t);
#define LEGO_NW_TILE 64

hipError_t lego_stencil_f32_launch(const float*, float*, const float*, int, int, int, int, int, hipStream_t);
hipError_t lego_stencil_f32_plan(int, int, int, int, int*);
#define LEGO_STENCIL_BRICK 8
#define LEGO_STENCIL_MAX_RADIUS 3
#define LEGO_STENCIL_STAR_MAX_RADIUS 4

hipError_t lego_lud_f32_launch(float*, int, hipStream_t);
hipError_t lego_lud_f32_plan(int, int*, int, int*);
#define LEGO_LUD_BLOCK 64

struct AttentionArgs;
struct RotaryArgs;
struct TreeArgs;
hipError_t lego_tree_f16_d64_launch(const TreeArgs&, int, hipStream_t);
hipError_t lego_tree_f16_d96_launch(const TreeArgs&, int, hipStream_t);
hipError_t lego_tree_f16_d128_launch(const TreeArgs&, int, hipStream_t);
hipError_t lego_tree_bf16_d64_launch(const TreeArgs&, int, hipStream_t);
hipError_t lego_tree_bf16_d96_launch(const TreeArgs&, int, hipStream_t);
hipError_t lego_tree_bf16_d128_launch(const TreeArgs&, int, hipStream_t);
#define LEGO_TREE_LEAST 2
hipError_t lego_attention_fwd_f16_d64_launch(const AttentionArgs&, hipStream_t);
hipError_t lego_attention_fwd_f16_d96_launch(const AttentionArgs&, hipStream_t);
hipError_t lego_attention_fwd_f16_d128_launch(const AttentionArgs&, hipStream_t);
hipError_t lego_attention_fwd_bf16_d64_launch(const AttentionArgs&, hipStream_t);
hipError_t lego_attention_fwd_bf16_d96_launch(const AttentionArgs&, hipStream_t);
hipError_t lego_attention_fwd_bf16_d128_launch(const AttentionArgs&, hipStream_t);
hipError_t lego_attention_bwd_f16_d64_launch(const AttentionArgs&, hipStream_t);
hipError_t lego_attention_bwd_f16_d96_launch(const AttentionArgs&, hipStream_t);
hipError_t lego_attention_bwd_f16_d128_launch(const AttentionArgs&, hipStream_t);
hipError_t lego_attention_bwd_bf16_d64_launch(const AttentionArgs&, hipStream_t);
hipError_t lego_attention_bwd_bf16_d96_launch(const AttentionArgs&, hipStream_t);
hipError_t lego_attention_bwd_bf16_d128_launch(const AttentionArgs&, hipStream_t);
hipError_t lego_attention_tiles_launch(const int*, int2*, int, int, hipStream_t);
hipError_t lego_attention_order_launch(const AttentionArgs&, hipStream_t);
hipError_t lego_attention_delta_launch(const AttentionArgs&, int, hipStream_t);
hipError_t lego_attention_join_launch(const AttentionArgs&, int, hipStream_t);
hipError_t lego_rotary_launch(const RotaryArgs&, int, int, int, int, hipStream_t);
#define LEGO_ATTENTION_MAX_HEAD 128
#define LEGO_ATTENTION_ORDERED 512
#define LEGO_ROTARY_MAX_PART 256
