// Products in 8-bit floating point (e4m3): fp8_linear and the routed experts on such tables.
//
//   y[n, r] = sum_b sx[n, b] * sw[r / 128, b] * sum_{c in block b} xq[n, c] * wq[r, c]
//
// fp8_gemm_kernel, one CTA per SM, 10 warps:
//   warp 0     TMA producer: per 128-column block the tile's MT x 128 B of tokens and 2 x 128 x 128 B of weights (128-byte
//              swizzle), into a ring of stages
//   warp 1     TMEM owner and MMA issuer (one thread): 4 tcgen05.mma kind::f8f6f4 (M 128 x N 256 x K 32) per block into
//              one of two 256-column accumulators
//   warps 2-9  promotion and epilogue: a block's 128 x 256 partial sums leave TMEM while the tensor core works on the next
//              block; acc += partial * (sx * sw) in fp32 registers (32 rows x 128 columns per warp). Tokens are the M side,
//              so a thread owns one token row: both scales are scalars for its columns.
// The block's partial sum is exact enough to be added as it is: e4m3 products are exact in fp32 and the tensor core sums
// them in fp32 (measured: 1e-8 relative over K = 128).
// With two matrices (gate, up: 128 columns each) the epilogue forms swiglu_clamped(gate, up), takes each row's maximum
// over its 128 columns and stores e4m3 codes and the scale: the down product's input, never in 16 bits.
// Every wait is bounded; a role that gives up sets CBMOE_DEVERR_TIMEOUT and falls through to the final barrier.
#include <cudaTypedefs.h>

#include "fp8.cuh"
#include "grouped.cuh"
#include "layer.cuh"
#include "profile.cuh"
#include "umma.cuh"

namespace cbmoe {

namespace {

// ------------------------------------------------------------------------------------------------- quantiser
template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32(float v) { return v; }

// 16 lanes per group of 128, 8 values each. Bound by the reads of x; with row_slot a token is read and quantised once
// and its k copies are written, so the sorted rows cost their own bytes only.
template <typename T>
__global__ void __launch_bounds__(256) fp8_quantize_kernel(const T* __restrict__ x, int N, int K, long long ldx,
                                                           int vec, uint8_t* __restrict__ q, long long ldq,
                                                           float* __restrict__ s, const int* __restrict__ row_slot,
                                                           int k, int R) {
  griddep_wait();
  griddep_launch();
  const int KB = (K + kFp8Group - 1) / kFp8Group;
  const long long total = (long long)N * KB;
  const int l = threadIdx.x & 15;
  const bool wide = ldq % 8 == 0 && (reinterpret_cast<uintptr_t>(q) & 7) == 0;
  for (long long g0 = (blockIdx.x * 256LL + (threadIdx.x & ~31)) / 16; g0 < total; g0 += gridDim.x * 16LL) {
    const long long g = g0 + ((threadIdx.x >> 4) & 1);
    const bool in = g < total;
    const int n = in ? (int)(g / KB) : 0, kb = in ? (int)(g - (long long)n * KB) : 0;
    const int c0 = kb * kFp8Group + 8 * l;
    float v[8];
    const T* src = x + (size_t)n * ldx + c0;
    if (in && vec && c0 + 8 <= K) {
      union {
        uint4 u[sizeof(T) * 8 / 16];
        T t[8];
      } b;
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) * 8 / 16; ++i) b.u[i] = reinterpret_cast<const uint4*>(src)[i];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = to_f32<T>(b.t[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = in && c0 + i < K ? to_f32<T>(src[i]) : 0.f;
    }
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max_nan(top, fabsf(v[i]));
#pragma unroll
    for (int m = 8; m > 0; m >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, m));
    float inv;
    const float sc = fp8_group_scale(top, &inv);
    const uint2 o = make_uint2(fp8_pack4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv),
                               fp8_pack4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv));
    if (!in) continue;
    const int copies = row_slot != nullptr ? k : 1;
    for (int j = 0; j < copies; ++j) {
      const int r = row_slot != nullptr ? row_slot[(size_t)n * k + j] : n;
      if (r < 0 || r >= R) continue;
      uint8_t* dst = q + (size_t)r * ldq + c0;
      if (wide && c0 + 8 <= ldq) {
        *reinterpret_cast<uint2*>(dst) = o;
      } else {
        for (int i = 0; i < 8 && c0 + i < K; ++i) dst[i] = (uint8_t)((i < 4 ? o.x : o.y) >> (8 * (i & 3)));
      }
      if (l == 0) s[(size_t)r * KB + kb] = sc;
    }
  }
}

// --------------------------------------------------------------------------------------------------- product
constexpr int kFp8Threads = 10 * 32;
constexpr int kW0 = 2;                                   // first promotion warp
constexpr int kBHalf = 128 * 128;                        // 128 weight rows of one block

template <int MT>
struct Fp8Cfg {
  static constexpr int kATile = MT * 128;
  static constexpr int kStage = kATile + 2 * kBHalf;
  static constexpr int kNStage = MT == 128 ? 4 : (MT == 64 ? 5 : 6);
  static constexpr int kBarOff = kNStage * kStage;
  static constexpr int kSmem = 1024 + kBarOff + 256 + 4 * 2 * 2 * 32 * 4;   // + row maxima of the SwiGLU epilogue
  static_assert(kSmem <= 227 * 1024, "shared memory budget");
};

struct Fp8Params {
  Fp8Gemm g;
  int KB, RB, NT;          // column blocks, 128-row blocks per matrix, output tiles per pass
};

struct Fp8Item {
  int e, row0, cnt, nt;
};

template <int MT>
__device__ __forceinline__ int fp8_items(const Fp8Params& p) {
  return (p.g.pass_expert ? *p.g.n_pass : (p.g.x_rows + MT - 1) / MT) * p.NT;
}

template <int MT>
__device__ __forceinline__ Fp8Item fp8_item(const Fp8Params& p, int item) {
  const int pass = item / p.NT, nt = item % p.NT;
  if (p.g.pass_expert == nullptr) return {0, pass * MT, min(MT, p.g.x_rows - pass * MT), nt};
  return {p.g.pass_expert[pass], p.g.pass_row0[pass], p.g.pass_cnt[pass], nt};
}

__device__ __forceinline__ void fma2(unsigned long long& acc, uint32_t lo, uint32_t hi, unsigned long long sc) {
  unsigned long long d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(d), "l"(sc));
}

__device__ __forceinline__ unsigned long long pair_of(float v) {
  unsigned long long d;
  asm("mov.b64 %0, {%1, %1};" : "=l"(d) : "r"(__float_as_uint(v)));
  return d;
}

__device__ __forceinline__ float lo_of(unsigned long long v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float hi_of(unsigned long long v) { return __uint_as_float((uint32_t)(v >> 32)); }

// Accumulator pair i (columns 2i, 2i + 1) of a thread's 128 columns.
#define CBMOE_ACC(a, c) (((c) & 1) ? hi_of((a)[(c) >> 1]) : lo_of((a)[(c) >> 1]))

template <typename OUT>
__device__ __forceinline__ OUT out_of(float v);
template <>
__device__ __forceinline__ float out_of(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 out_of(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half out_of(float v) { return __float2half_rn(v); }

// silu(min(g, L)) * clip(u, -L, L) (model.py:119-122) that keeps a NaN, so that a bad row shows.
__device__ __forceinline__ float swiglu_keep_nan(float g, float u, float limit) {
  g = g > limit ? limit : g;
  u = u > limit ? limit : (u < -limit ? -limit : u);
  return silu_f(g) * u;
}

template <int MT, bool SWIGLU, typename OUT>
__global__ void __launch_bounds__(kFp8Threads, 1) fp8_gemm_kernel(const Fp8Params p,
                                                                  const __grid_constant__ CUtensorMap map_x,
                                                                  const __grid_constant__ CUtensorMap map_w0,
                                                                  const __grid_constant__ CUtensorMap map_w1) {
  using C = Fp8Cfg<MT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kBarOff);
  uint64_t* empty = full + C::kNStage;
  uint64_t* d_full = empty + C::kNStage;    // [2]
  uint64_t* d_empty = d_full + 2;           // [2]
  uint64_t* swap = d_empty + 2;             // [4]: the two warps of a row quadrant exchange row maxima
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(swap + 4);
  float* row_max = reinterpret_cast<float*>(smem + C::kBarOff + 256);   // [2 items][4 quadrants][2 halves][32]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kNStage; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&d_full[i], 1);
      mbar_init(&d_empty[i], 8);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&swap[i], 2);
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc(tmem_slot, 512);
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&map_x);
    prefetch_tmap(&map_w0);
    prefetch_tmap(&map_w1);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  griddep_wait();
  griddep_launch();
  const int n_items = fp8_items<MT>(p);

  if (warp == 0) {
    if (lane == 0) {
      int st = 0;
      uint32_t ph = 0;
      for (int item = blockIdx.x; item < n_items; item += gridDim.x) {
        const Fp8Item it = fp8_item<MT>(p, item);
        const int wrow = it.e * p.g.rows + it.nt * (SWIGLU ? 128 : 256);
        for (int kb = 0; kb < p.KB; ++kb) {
          if (!mbar_wait_sleepy(&empty[st], ph ^ 1)) goto done;
          uint8_t* a = smem + st * C::kStage;
          mbar_arrive_expect_tx(&full[st], C::kStage);
          tma_load_2d(a, &map_x, kb * kFp8Group, it.row0, &full[st]);
          tma_load_2d(a + C::kATile, &map_w0, kb * kFp8Group, wrow, &full[st]);
          tma_load_2d(a + C::kATile + kBHalf, SWIGLU ? &map_w1 : &map_w0, kb * kFp8Group, SWIGLU ? wrow : wrow + 128,
                      &full[st]);
          if (++st == C::kNStage) {
            st = 0;
            ph ^= 1;
          }
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_e4m3_m128(kFp8TileN);
      int st = 0;
      uint32_t ph = 0, n = 0;
      for (int item = blockIdx.x; item < n_items; item += gridDim.x) {
        for (int kb = 0; kb < p.KB; ++kb, ++n) {
          const int buf = n & 1;
          if (!mbar_wait(&d_empty[buf], ((n >> 1) & 1) ^ 1) || !mbar_wait(&full[st], ph)) goto done;
          tc_fence_after();
          // Rows MT.. of the M side are whatever follows in the stage (weights): their sums are never read.
          const uint32_t sbase = smem_addr(smem + st * C::kStage);
          const uint64_t ad = sw128_desc(sbase), bd = sw128_desc(sbase + C::kATile);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) umma_fp8(tmem + buf * kFp8TileN, ad + 2 * kk, bd + 2 * kk, idesc, kk != 0);
          umma_commit(&empty[st]);
          umma_commit(&d_full[buf]);
          if (++st == C::kNStage) {
            st = 0;
            ph ^= 1;
          }
        }
      }
    }
  } else {
    const int q = warp & 3;                  // TMEM lane quadrant this warp may read
    const int half = (warp - kW0) >> 2;
    uint32_t n = 0, local = 0;
    for (int item = blockIdx.x; item < n_items; item += gridDim.x) {
      const Fp8Item it = fp8_item<MT>(p, item);
      const int m = 32 * q + lane;
      const bool live = 32 * q < it.cnt, mine = m < it.cnt;
      const size_t xrow = (size_t)it.row0 + (mine ? m : 0);
      const float* sx = p.g.xs + xrow * p.KB;
      const float *sa, *sb;                  // scales of this thread's columns 0-63 and 64-127
      if constexpr (SWIGLU) {
        sa = p.g.s0 + ((size_t)it.e * p.RB + it.nt) * p.KB;
        sb = p.g.s1 + ((size_t)it.e * p.RB + it.nt) * p.KB;
      } else {
        sa = p.g.s0 + ((size_t)it.e * p.RB + min(2 * it.nt + half, p.RB - 1)) * p.KB;
        sb = sa;
      }
      unsigned long long acc[64];
#pragma unroll
      for (int i = 0; i < 64; ++i) acc[i] = 0;
      float x_next = live ? sx[0] : 0.f, a_next = sa[0], b_next = sb[0];
      for (int kb = 0; kb < p.KB; ++kb, ++n) {
        const int buf = n & 1;
        const unsigned long long fa = pair_of(x_next * a_next), fb = pair_of(x_next * b_next);
        if (live && kb + 1 < p.KB) {
          x_next = sx[kb + 1];
          a_next = sa[kb + 1];
          if constexpr (SWIGLU) b_next = sb[kb + 1];
          else b_next = a_next;
        }
        if (!mbar_wait(&d_full[buf], (n >> 1) & 1)) goto done;
        tc_fence_after();
        if (live) {
          const uint32_t t0 = tmem + buf * kFp8TileN + ((uint32_t)(32 * q) << 16);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t v[32];
            const int col = SWIGLU ? (c < 2 ? 64 * half + 32 * c : 128 + 64 * half + 32 * (c - 2)) : 128 * half + 32 * c;
            tmem_ld32(t0 + col, v);
#pragma unroll
            for (int i = 0; i < 16; ++i) fma2(acc[16 * c + i], v[2 * i], v[2 * i + 1], c < 2 ? fa : fb);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&d_empty[buf]);
      }
      if constexpr (SWIGLU) {
        const int col0 = it.nt * 128 + 64 * half;
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 64; ++i) {
          const float h = col0 + i < p.g.rows ? swiglu_keep_nan(CBMOE_ACC(acc, i), CBMOE_ACC(acc, 64 + i), p.g.limit) : 0.f;
          top = max_nan(top, fabsf(h));
          if (i & 1) acc[i >> 1] = (acc[i >> 1] & 0xffffffffull) | ((unsigned long long)__float_as_uint(h) << 32);
          else acc[i >> 1] = (acc[i >> 1] & ~0xffffffffull) | __float_as_uint(h);
        }
        float* mx = row_max + ((local & 1) * 4 + q) * 64;
        mx[half * 32 + lane] = top;
        __syncwarp();
        if (lane == 0) mbar_arrive(&swap[q]);
        if (!mbar_wait(&swap[q], local & 1)) goto done;
        top = max_nan(top, mx[(half ^ 1) * 32 + lane]);
        float inv;
        const float sc = fp8_group_scale(top, &inv);
        if (mine) {
          uint4* dst = reinterpret_cast<uint4*>(p.g.hq + xrow * ((size_t)p.RB * 128) + col0);
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int c = 16 * u + 4 * i;
              w[i] = fp8_pack4(CBMOE_ACC(acc, c) * inv, CBMOE_ACC(acc, c + 1) * inv, CBMOE_ACC(acc, c + 2) * inv,
                               CBMOE_ACC(acc, c + 3) * inv);
            }
            dst[u] = make_uint4(w[0], w[1], w[2], w[3]);
          }
          if (half == 0) p.g.hs[xrow * p.RB + it.nt] = sc;
        }
      } else if (mine) {
        const int col0 = it.nt * 256 + 128 * half, rows = p.g.rows;
        OUT* dst = static_cast<OUT*>(p.g.out) + xrow * rows + col0;
        constexpr int kU = 16 / (int)sizeof(OUT);
        if (rows % kU == 0 && (reinterpret_cast<uintptr_t>(p.g.out) & 15) == 0) {
#pragma unroll
          for (int u = 0; u < 128 / kU; ++u) {
            union {
              uint4 v;
              OUT o[kU];
            } b;
#pragma unroll
            for (int i = 0; i < kU; ++i) b.o[i] = out_of<OUT>(CBMOE_ACC(acc, u * kU + i));
            if (col0 + u * kU < rows) reinterpret_cast<uint4*>(dst)[u] = b.v;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 128; ++i)
            if (col0 + i < rows) dst[i] = out_of<OUT>(CBMOE_ACC(acc, i));
        }
      }
      ++local;
    }
  }
done:
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// e4m3 matrix [rows][K] with row stride ld bytes: 128-byte x box_rows boxes, 128-byte swizzle, zeros out of bounds.
int make_fp8_map(CUtensorMap* map, const void* base, int K, long long rows, long long ld, int box_rows) {
  auto fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(tensor_map_encoder());
  if (fn == nullptr) return CBMOE_ERR_CUDA;
  const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld};
  const cuuint32_t box[2] = {(cuuint32_t)kFp8Group, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? CBMOE_OK : CBMOE_ERR_CUDA;
}

template <int MT, bool SWIGLU, typename OUT>
int launch_t(const Fp8Gemm& g, cudaStream_t stream) {
  using C = Fp8Cfg<MT>;
  Fp8Params p;
  p.g = g;
  p.KB = (g.K + kFp8Group - 1) / kFp8Group;
  p.RB = (g.rows + 127) / 128;
  p.NT = SWIGLU ? p.RB : (p.RB + 1) / 2;
  CUtensorMap mx, m0, m1;
  int rc = make_fp8_map(&mx, g.xq, g.K, g.x_rows, g.ldx, MT);
  if (!rc) rc = make_fp8_map(&m0, g.w0, g.K, (long long)g.E * g.rows, g.ldw, 128);
  if (!rc) rc = make_fp8_map(&m1, SWIGLU ? g.w1 : g.w0, g.K, (long long)g.E * g.rows, g.ldw, 128);
  if (rc) return rc;
  auto kern = fp8_gemm_kernel<MT, SWIGLU, OUT>;
  static PerDevice s_attr;
  long long set = 0;
  rc = per_device(s_attr, [&](long long& v) -> int {
    CBMOE_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    v = 1;
    return CBMOE_OK;
  }, &set);
  if (rc) return rc;
  prof_begin(kProfOther, stream);
  CBMOE_CUDA_TRY(launch_pdl(kern, dim3(num_sms()), dim3(kFp8Threads), C::kSmem, stream, p, mx, m0, m1));
  prof_end(kProfOther, stream);
  CBMOE_CUDA_TRY(cudaGetLastError());
  return CBMOE_OK;
}

template <int MT>
int launch_mt(const Fp8Gemm& g, cudaStream_t s) {
  if (g.w1 != nullptr) return launch_t<MT, true, float>(g, s);
  if (g.out_type == CBMOE_BF16) return launch_t<MT, false, __nv_bfloat16>(g, s);
  if (g.out_type == CBMOE_F16) return launch_t<MT, false, __half>(g, s);
  return launch_t<MT, false, float>(g, s);
}

bool aligned(const void* p, int n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
bool type_ok(int t) { return t == CBMOE_BF16 || t == CBMOE_F16 || t == CBMOE_F32; }
int blocks_of(int K) { return (K + kFp8Group - 1) / kFp8Group; }

}  // namespace

int fp8_pass_tokens(long long slots, int E) { return slots <= 32LL * E ? 32 : (slots <= 64LL * E ? 64 : 128); }

int launch_fp8_gemm(const Fp8Gemm& g, int mt, cudaStream_t s) {
  if (mt == 32) return launch_mt<32>(g, s);
  if (mt == 64) return launch_mt<64>(g, s);
  return launch_mt<128>(g, s);
}

int launch_fp8_quantize(const void* x, int type, int N, int K, long long ldx, uint8_t* q, long long ldq, float* s,
                        const int* row_slot, int k, int R, cudaStream_t stream) {
  const long long groups = (long long)N * blocks_of(K);
  long long blocks = (groups + 15) / 16, cap = (long long)num_sms() * 16;
  if (blocks > cap) blocks = cap;
  const int size = type == CBMOE_F32 ? 4 : 2;
  const int vec = aligned(x, 16) && ldx * size % 16 == 0;
  prof_begin(kProfOther, stream);
  if (type == CBMOE_BF16)
    CBMOE_CUDA_TRY(launch_pdl(fp8_quantize_kernel<__nv_bfloat16>, dim3((int)blocks), dim3(256), 0, stream,
                              static_cast<const __nv_bfloat16*>(x), N, K, ldx, vec, q, ldq, s, row_slot, k, R));
  else if (type == CBMOE_F16)
    CBMOE_CUDA_TRY(launch_pdl(fp8_quantize_kernel<__half>, dim3((int)blocks), dim3(256), 0, stream,
                              static_cast<const __half*>(x), N, K, ldx, vec, q, ldq, s, row_slot, k, R));
  else
    CBMOE_CUDA_TRY(launch_pdl(fp8_quantize_kernel<float>, dim3((int)blocks), dim3(256), 0, stream,
                              static_cast<const float*>(x), N, K, ldx, vec, q, ldq, s, row_slot, k, R));
  prof_end(kProfOther, stream);
  CBMOE_CUDA_TRY(cudaGetLastError());
  return CBMOE_OK;
}

namespace {

// Workspace of a product with a quantised input: q [N][blocks * 128] | s [N][blocks].
struct LinearWs {
  size_t s, total;
};
LinearWs linear_ws(int N, int K) {
  LinearWs w;
  w.s = lyr::align_up((size_t)N * blocks_of(K) * kFp8Group);
  w.total = w.s + lyr::align_up((size_t)N * blocks_of(K) * 4);
  return w;
}

struct ExpertsWs {
  size_t plan, xq, xs, hq, hs, y, total;
  int mt, Rp;
  lyr::PlanLayoutHost L;
};
ExpertsWs experts_ws(int E, int H, int I, int N, int k, int y_type) {
  ExpertsWs w;
  const long long S = (long long)N * k;
  w.mt = fp8_pass_tokens(S, E);
  w.L = lyr::host_plan_layout(N, k, E, 1, w.mt);
  w.Rp = (int)S;                                        // blocks of one row: the sorted rows are [0, S)
  w.plan = 0;
  w.xq = lyr::align_up((size_t)w.L.off[13] * 4);
  w.xs = w.xq + lyr::align_up((size_t)S * blocks_of(H) * kFp8Group);
  w.hq = w.xs + lyr::align_up((size_t)S * blocks_of(H) * 4);
  w.hs = w.hq + lyr::align_up((size_t)S * blocks_of(I) * kFp8Group);
  w.y = w.hs + lyr::align_up((size_t)S * blocks_of(I) * 4);
  w.total = w.y + lyr::align_up((size_t)S * H * (y_type == CBMOE_F32 ? 4 : 2));
  return w;
}

bool fp8_table_ok(const void* q, const float* s, long long ld, long long rows, int K) {
  return q && s && aligned(q, 16) && aligned(s, 4) && ld >= K && ld % 16 == 0 && rows <= 0x7fffffffLL;
}

bool fp8_experts_ok(const cbmoe_fp8_experts* ex) {
  return ex && ex->E > 0 && ex->E <= 1024 && ex->H > 0 && ex->I > 0 && ex->H <= (1 << 20) && ex->I <= (1 << 20) &&
         fp8_table_ok(ex->gate, ex->gate_s, ex->ld_in, (long long)ex->E * ex->I, ex->H) &&
         fp8_table_ok(ex->up, ex->up_s, ex->ld_in, (long long)ex->E * ex->I, ex->H) &&
         fp8_table_ok(ex->down, ex->down_s, ex->ld_down, (long long)ex->E * ex->H, ex->I);
}

}  // namespace

}  // namespace cbmoe

using namespace cbmoe;

extern "C" int cbmoe_fp8_quantize(const void* x, int type, int N, int K, long long ldx, uint8_t* q, long long ldq,
                                  float* s, cudaStream_t stream) {
  if (!type_ok(type) || N < 0 || K <= 0 || ldx < K || ldq < K) return CBMOE_ERR_INVALID;
  if (N == 0) return CBMOE_OK;
  if (!x || !q || !s) return CBMOE_ERR_INVALID;
  return launch_fp8_quantize(x, type, N, K, ldx, q, ldq, s, nullptr, 1, N, stream);
}

extern "C" size_t cbmoe_fp8_linear_workspace_bytes(int N, int K, int rows, int x_type) {
  if (N < 0 || K <= 0 || rows <= 0) return 0;
  if (x_type == CBMOE_E4M3) return 0;
  return type_ok(x_type) ? linear_ws(N, K).total : 0;
}

extern "C" int cbmoe_fp8_linear(const void* q, long long ldq, const float* s, int rows, int K, const void* x,
                                int x_type, long long ldx, const float* xs, int N, void* y, int y_type,
                                void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  if (rows <= 0 || K <= 0 || N < 0 || !type_ok(y_type) || !fp8_table_ok(q, s, ldq, rows, K)) return CBMOE_ERR_INVALID;
  const bool ready = x_type == CBMOE_E4M3;
  if (!ready && !type_ok(x_type)) return CBMOE_ERR_INVALID;
  if (N == 0) return CBMOE_OK;
  if (!x || !y || ldx < K || (ready && (!xs || ldx % 16 || !aligned(x, 16)))) return CBMOE_ERR_INVALID;
  Fp8Gemm g{};
  g.rows = rows;
  g.K = K;
  g.E = 1;
  g.x_rows = N;
  g.w0 = q;
  g.ldw = ldq;
  g.s0 = s;
  g.out = y;
  g.out_type = y_type;
  if (ready) {
    g.xq = x;
    g.ldx = ldx;
    g.xs = xs;
  } else {
    const LinearWs W = linear_ws(N, K);
    if (!workspace || workspace_bytes < W.total || !aligned(workspace, 256)) return CBMOE_ERR_WORKSPACE;
    uint8_t* xq = static_cast<uint8_t*>(workspace);
    float* sc = reinterpret_cast<float*>(xq + W.s);
    g.ldx = (long long)blocks_of(K) * kFp8Group;
    const int rc = launch_fp8_quantize(x, x_type, N, K, ldx, xq, g.ldx, sc, nullptr, 1, N, stream);
    if (rc) return rc;
    g.xq = xq;
    g.xs = sc;
  }
  return launch_fp8_gemm(g, fp8_pass_tokens(N, 1), stream);
}

extern "C" size_t cbmoe_fp8_experts_workspace_bytes(const cbmoe_fp8_experts* ex, int N, int k, int y_type) {
  if (!ex || ex->E <= 0 || ex->H <= 0 || ex->I <= 0 || N < 0 || k <= 0 || !type_ok(y_type)) return 0;
  return experts_ws(ex->E, ex->H, ex->I, N, k, y_type).total;
}

extern "C" int cbmoe_fp8_experts_apply(const cbmoe_fp8_experts* ex, const uint16_t* x, int N, const int32_t* idx,
                                       const float* w, int k, float limit, void* y, int y_type, void* workspace,
                                       size_t workspace_bytes, cudaStream_t stream) {
  if (!fp8_experts_ok(ex) || N < 0 || k <= 0 || k > 64 || !type_ok(y_type)) return CBMOE_ERR_INVALID;
  if (N == 0) return CBMOE_OK;
  if (!x || !idx || !w || !y) return CBMOE_ERR_INVALID;
  if ((long long)N * k > (1 << 30)) return CBMOE_ERR_UNSUPPORTED;
  const ExpertsWs W = experts_ws(ex->E, ex->H, ex->I, N, k, y_type);
  if (!workspace || workspace_bytes < W.total || !aligned(workspace, 256)) return CBMOE_ERR_WORKSPACE;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  int32_t* plan = reinterpret_cast<int32_t*>(ws + W.plan);
  int rc = launch_route_plan(idx, w, N, k, ex->E, 1, W.mt, plan, stream, nullptr, 0);
  if (rc) return rc;
  const int32_t* row_slot = plan + W.L.off[9];
  Fp8Gemm g{};
  g.E = ex->E;
  g.rows = ex->I;
  g.K = ex->H;
  g.ldx = (long long)blocks_of(ex->H) * kFp8Group;
  g.x_rows = W.Rp;
  g.xq = ws + W.xq;
  g.xs = reinterpret_cast<const float*>(ws + W.xs);
  rc = launch_fp8_quantize(x, CBMOE_BF16, N, ex->H, ex->H, ws + W.xq, g.ldx, reinterpret_cast<float*>(ws + W.xs),
                           row_slot, k, W.Rp, stream);
  if (rc) return rc;
  g.w0 = ex->gate;
  g.w1 = ex->up;
  g.ldw = ex->ld_in;
  g.s0 = ex->gate_s;
  g.s1 = ex->up_s;
  g.pass_expert = plan + W.L.off[10];
  g.pass_row0 = plan + W.L.off[11];
  g.pass_cnt = plan + W.L.off[12];
  g.n_pass = plan + W.L.off[5];
  g.limit = limit;
  g.hq = ws + W.hq;
  g.hs = reinterpret_cast<float*>(ws + W.hs);
  rc = launch_fp8_gemm(g, W.mt, stream);
  if (rc) return rc;
  Fp8Gemm d = g;
  d.rows = ex->H;
  d.K = ex->I;
  d.xq = g.hq;
  d.ldx = (long long)blocks_of(ex->I) * kFp8Group;
  d.xs = g.hs;
  d.w0 = ex->down;
  d.w1 = nullptr;
  d.ldw = ex->ld_down;
  d.s0 = ex->down_s;
  d.s1 = nullptr;
  d.hq = nullptr;
  d.hs = nullptr;
  d.out = ws + W.y;
  d.out_type = y_type;
  rc = launch_fp8_gemm(d, W.mt, stream);
  if (rc) return rc;
  return cbmoe_unpermute(ws + W.y, y_type, W.Rp, ex->H, row_slot, w, N, k, y, stream);
}
