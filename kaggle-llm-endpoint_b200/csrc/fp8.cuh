// 8-bit floating point (e4m3) products with one scale per 128 x 128 weight block and per 128-wide group of an
// activation row (fp8.cu): the group scale, and the interface between the quantiser and the product.
#pragma once
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace cbmoe {

constexpr int kFp8Group = 128;       // columns of one scale; also one 128-byte swizzle row of an operand tile
constexpr int kFp8TileN = 256;       // weight rows per output tile (SwiGLU: 128 of gate and 128 of up)

// The scale of a group whose largest magnitude is `top`: the least power of two s >= 2^-100 with top <= 448 s, so that
// x / s is exact and the only rounding is the one to e4m3 (the same codes whatever the order of evaluation). NaN for an
// infinite or NaN maximum: every value of such a group then stands for NaN, as its row's products do. *inv = 1 / s.
__device__ __forceinline__ float fp8_group_scale(float top, float* inv) {
  if (!(top < __uint_as_float(0x7f800000u))) {
    *inv = __uint_as_float(0x7fc00000u);
    return *inv;
  }
  const uint32_t b = __float_as_uint(fmaxf(top, 0x1.cp-92f));                          // 448 * 2^-100
  const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);     // 448 = 1.75 * 2^8
  *inv = __uint_as_float((uint32_t)(127 - e) << 23);
  return __uint_as_float((uint32_t)(127 + e) << 23);
}

// Maximum that keeps a NaN (fmaxf drops it).
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

struct Fp8Gemm {
  int rows, K;             // weight rows per expert (of each matrix) and inputs
  int E;
  const void* xq;          // e4m3 [x_rows][ldx]
  long long ldx;
  int x_rows;
  int repeated;            // dense, up to 32 tokens: xq holds row n at n, 32 + n, 64 + n and 96 + n
  const float* xs;         // [x_rows][ldxs], ldxs = fp8_scale_stride(K), 16-byte aligned
  int ldxs;
  const void* w0;          // e4m3 [E][rows][ldw]; w1: up, beside w0 = gate (SwiGLU), else null
  const void* w1;
  long long ldw;
  const float* s0;         // [E][ceil(rows / 128)][ceil(K / 128)]
  const float* s1;
  const int* pass_expert;  // passes of up to `mt` consecutive rows of one expert (null: dense, x_rows rows)
  const int* pass_row0;
  const int* pass_cnt;
  const int* n_pass;
  float limit;             // SwiGLU clamp
  void* out;               // one matrix: [x_rows][rows] of out_type
  int out_type;
  float* part;             // fp8_part_bytes(mt): partial sums of tiles that several CTAs share
  int* arrived;            // fp8_arrived() counters, zero before the launch
  uint8_t* hq;             // SwiGLU: e4m3 [x_rows][ceil(rows / 128) * 128] and its scales [x_rows][fp8_scale_stride(rows)]
  float* hs;
};

// Row stride of the scales that the library keeps for itself: four blocks are one 16-byte load.
inline int fp8_scale_stride(int K) { return ((K + kFp8Group - 1) / kFp8Group + 3) & ~3; }
// This file's own error word (common.cuh), after the device is synchronized.
int fp8_device_errors(int clear, int* out_host);
// Token rows per pass of the product kernel: 32, 64, 128 or 256 (a pair of CTAs).
int fp8_pass_tokens(long long slots, int E);
size_t fp8_part_bytes(int mt);
int fp8_arrived();         // counters of one launch: 8 for each tile that can be shared (fewer than the SMs)
int launch_fp8_gemm(const Fp8Gemm& g, int mt, cudaStream_t s);
// x [N][K] (row stride ldx elements) -> e4m3 rows q (stride ldq bytes, columns K.. up to ldq zero where a unit of 8
// reaches past K) and scales s [..][lds]; with row_slot, row n goes to the k rows row_slot[n][:] in [0, R).
// With `repeat` (row_slot null) row n goes to the rows n + 32 j, j < repeat, its scales to row n only.
// Clears zero[0, n_zero) on the way (the counters of the products that follow).
int launch_fp8_quantize(const void* x, int type, int N, int K, long long ldx, uint8_t* q, long long ldq, float* s, int lds,
                        const int* row_slot, int k, int R, int repeat, int* zero, int n_zero, cudaStream_t stream);

}  // namespace cbmoe
