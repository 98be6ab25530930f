// Tokens into expert order and back, forward and backward, over a routing plan (cbmoe_route_plan): the row gather and
// the weighted combine of the layer (resident.py:144-165) as operators of their own, with their gradients.
//
//   permute             xs[r] = x[tok_row[r]], zero rows where tok_row[r] < 0
//   unpermute           y[t] = sum_j w[t, j] ys[row_slot[t, j]]      (without w: the plain sum, permute's gradient)
//   unpermute backward  dys[row_slot[t, j]] = w[t, j] dy[t], zero rows where tok_row < 0; dw[t, j] = <dy[t], ys[row]>
//
// All three are bound by memory, so each walks the tokens, not the sorted rows: a token's row is read once and its k
// sorted rows are written (or read) once, and no row is touched twice. A sorted row belongs to one slot, so nothing is
// added by atomics: sums run over j in order, in fp32, rounded once. Rows outside [0, R) in row_slot are empty slots.
// Measured on one B200, 4096 tokens x 8 slots, rows of 5120 bf16 (about 375 MB a direction, 57 us at the copy rate):
// permute 67 us, unpermute 68 us; backward of the weighted form 150 us for 108 us of bytes (it reads ys and writes dys).
// Looking a slot's row up once per token and not once per unit took the plan, permute and its gradient from 198 to 184 us.
#include <cuda_fp16.h>

#include "decode.cuh"
#include "layer.cuh"
#include "profile.cuh"

namespace cbmoe {

namespace {

constexpr int kPermThreads = 128;

template <typename T>
struct Elem;
template <>
struct Elem<__nv_bfloat16> {
  static __device__ float to(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __nv_bfloat16 from(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Elem<__half> {
  static __device__ float to(__half v) { return __half2float(v); }
  static __device__ __half from(float v) { return __float2half_rn(v); }
};
template <>
struct Elem<float> {
  static __device__ float to(float v) { return v; }
  static __device__ float from(float v) { return v; }
};

// VB bytes of a row as one unit: the most of 16, 8, 4 and 2 that rows and pointers are aligned to.
// 4096 x 8 rows of 2564 bf16 (8 bytes): permute 41 us, unpermute 56, backward 90; by single elements 76, 117 and 151.
template <typename T, int VB>
struct alignas(VB) Vec {
  static constexpr int n = VB / (int)sizeof(T);
  T v[n];
};

// The sums of a unit of T as O.
template <typename T, int VB, typename O>
using Out = Vec<O, Vec<T, VB>::n * (int)sizeof(O)>;

// Zero rows of `out` where tok_row < 0: a warp looks at up to 32 rows at a time, at fewer where there are enough warps
// (a row of padding is a warp's work: 528 rows of 1411 halfs by 17 warps took 15 us).
template <typename V>
__device__ __forceinline__ void zero_padding(V* out, const int32_t* __restrict__ tok_row, int R, int HV, int warp0,
                                             int n_warps) {
  const int lane = threadIdx.x & 31;
  const int step = min(32, (R + n_warps - 1) / n_warps);
  for (long long base = (long long)step * warp0; base < R; base += (long long)step * n_warps) {
    const int r = (int)base + lane;
    unsigned todo = __ballot_sync(0xffffffffu, lane < step && r < R && tok_row[r < R ? r : R - 1] < 0);
    while (todo) {
      const int row = (int)base + __ffs(todo) - 1;
      todo &= todo - 1;
      V z{};
      for (int c = lane; c < HV; c += 32) out[(size_t)row * HV + c] = z;
    }
  }
}

// A token's k rows are looked up once by the threads that copy or sum it: `tpt` threads a token (32 for narrow rows).
template <typename T, int VB>
__global__ void __launch_bounds__(kPermThreads) permute_kernel(const Vec<T, VB>* __restrict__ x, int Tn, int HV,
                                                               const int32_t* __restrict__ row_slot, int k,
                                                               const int32_t* __restrict__ tok_row, int R,
                                                               Vec<T, VB>* __restrict__ xs, int tok_blocks, int tpt) {
  griddep_wait();
  griddep_launch();
  if ((int)blockIdx.x >= tok_blocks) {
    if (blockIdx.y == 0)
      zero_padding(xs, tok_row, R, HV, ((int)blockIdx.x - tok_blocks) * (kPermThreads / 32) + (threadIdx.x >> 5),
                   ((int)gridDim.x - tok_blocks) * (kPermThreads / 32));
    return;
  }
  const int per = kPermThreads / tpt, c0 = threadIdx.x % tpt + tpt * blockIdx.y, dc = tpt * gridDim.y;
  for (int t = blockIdx.x * per + threadIdx.x / tpt; t < Tn; t += tok_blocks * per) {
    for (int j0 = 0; j0 < k; j0 += 8) {
      int r[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        r[j] = j0 + j < k ? row_slot[(size_t)t * k + j0 + j] : -1;
        if (r[j] >= R) r[j] = -1;
      }
      for (int c = c0; c < HV; c += dc) {
        const Vec<T, VB> v = x[(size_t)t * HV + c];
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (r[j] >= 0) xs[(size_t)r[j] * HV + c] = v;
      }
    }
  }
}

// Rows of T, sums rounded to O.
template <typename T, int VB, typename O>
__global__ void __launch_bounds__(kPermThreads) unpermute_kernel(const Vec<T, VB>* __restrict__ ys, int R, int HV,
                                                                 const int32_t* __restrict__ row_slot,
                                                                 const float* __restrict__ w, int Tn, int k,
                                                                 Out<T, VB, O>* __restrict__ y, int tpt) {
  using V = Vec<T, VB>;
  griddep_wait();
  griddep_launch();
  const int per = kPermThreads / tpt, c0 = threadIdx.x % tpt + tpt * blockIdx.y, dc = tpt * gridDim.y;
  for (int t = blockIdx.x * per + threadIdx.x / tpt; t < Tn; t += gridDim.x * per) {
    // Units under 16 bytes are many, so their rows are looked up once per token (8 slots at most): 61 -> 56 us for 4096 x 8
    // rows of 2564 bf16, 84 -> 64 for 2562. With whole units the registers that it holds cost more: 42 -> 49 for 2560.
    if constexpr (VB < 16) {
      int r[8];
      float wt[8];
      const auto look_up = [&](int j0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          r[j] = j0 + j < k ? row_slot[(size_t)t * k + j0 + j] : -1;
          if (r[j] >= R) r[j] = -1;
          wt[j] = r[j] >= 0 && w != nullptr ? w[(size_t)t * k + j0 + j] : 1.f;
        }
      };
      look_up(0);
      for (int c = c0; c < HV; c += dc) {
        float acc[V::n] = {};
        for (int j0 = 0; j0 < k; j0 += 8) {
          V v[8];
          if (k > 8) look_up(j0);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (r[j] >= 0) v[j] = ys[(size_t)r[j] * HV + c];
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (r[j] >= 0) {
#pragma unroll
              for (int q = 0; q < V::n; ++q) acc[q] = fmaf(wt[j], Elem<T>::to(v[j].v[q]), acc[q]);
            }
        }
        Out<T, VB, O> o;
#pragma unroll
        for (int q = 0; q < V::n; ++q) o.v[q] = Elem<O>::from(acc[q]);
        y[(size_t)t * HV + c] = o;
      }
    } else {
      for (int c = c0; c < HV; c += dc) {
        float acc[V::n] = {};
        for (int j0 = 0; j0 < k; j0 += 8) {   // 8 rows in flight
          V v[8];
          float wt[8];
          bool in[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int r = j0 + j < k ? row_slot[(size_t)t * k + j0 + j] : -1;
            in[j] = r >= 0 && r < R;
            wt[j] = in[j] && w != nullptr ? w[(size_t)t * k + j0 + j] : 1.f;
            if (in[j]) v[j] = ys[(size_t)r * HV + c];
          }
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (in[j]) {
#pragma unroll
              for (int q = 0; q < V::n; ++q) acc[q] = fmaf(wt[j], Elem<T>::to(v[j].v[q]), acc[q]);
            }
        }
        Out<T, VB, O> o;
#pragma unroll
        for (int q = 0; q < V::n; ++q) o.v[q] = Elem<O>::from(acc[q]);
        y[(size_t)t * HV + c] = o;
      }
    }
  }
}

constexpr int kBackThreads = 128;

// One CTA per token (grid-stride): dy[t] is read once per 8 slots, dw by a fixed-order block sum.
template <typename T, int VB>
__global__ void __launch_bounds__(kBackThreads) unpermute_backward_kernel(
    const Vec<T, VB>* __restrict__ dy, const Vec<T, VB>* __restrict__ ys, int R, int HV,
    const int32_t* __restrict__ row_slot, const int32_t* __restrict__ tok_row, const float* __restrict__ w, int Tn,
    int k, Vec<T, VB>* __restrict__ dys, float* __restrict__ dw, int tok_blocks) {
  using V = Vec<T, VB>;
  __shared__ float red[8][kBackThreads / 32];
  griddep_wait();
  griddep_launch();
  if ((int)blockIdx.x >= tok_blocks) {
    zero_padding(dys, tok_row, R, HV, ((int)blockIdx.x - tok_blocks) * (kBackThreads / 32) + (threadIdx.x >> 5),
                 ((int)gridDim.x - tok_blocks) * (kBackThreads / 32));
    return;
  }
  for (int t = blockIdx.x; t < Tn; t += tok_blocks) {
    for (int j0 = 0; j0 < k; j0 += 8) {
      int r[8];
      float wt[8], dot[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        r[j] = j0 + j < k ? row_slot[(size_t)t * k + j0 + j] : -1;
        if (r[j] >= R) r[j] = -1;
        wt[j] = r[j] >= 0 && w != nullptr ? w[(size_t)t * k + j0 + j] : 1.f;
        dot[j] = 0.f;
      }
      for (int c = threadIdx.x; c < HV; c += kBackThreads) {
        const V d = dy[(size_t)t * HV + c];
        V v[8];
        if (dw != nullptr) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (r[j] >= 0) v[j] = ys[(size_t)r[j] * HV + c];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (r[j] < 0) continue;
          V o;
#pragma unroll
          for (int q = 0; q < V::n; ++q) {
            const float g = Elem<T>::to(d.v[q]);
            o.v[q] = Elem<T>::from(wt[j] * g);
            if (dw != nullptr) dot[j] = fmaf(g, Elem<T>::to(v[j].v[q]), dot[j]);
          }
          if (dys != nullptr) dys[(size_t)r[j] * HV + c] = o;
        }
      }
      if (dw == nullptr) continue;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], m);
        if ((threadIdx.x & 31) == 0) red[j][threadIdx.x >> 5] = dot[j];
      }
      __syncthreads();
      if (threadIdx.x < 8 && j0 + (int)threadIdx.x < k) {
        float s = 0.f;
#pragma unroll
        for (int u = 0; u < kBackThreads / 32; ++u) s += red[threadIdx.x][u];
        dw[(size_t)t * k + j0 + threadIdx.x] = s;   // 0 for an empty slot
      }
      __syncthreads();
    }
  }
}

int blocks_for(long long total, int threads, int per_sm) {
  const long long b = (total + threads - 1) / threads, cap = (long long)num_sms() * per_sm;
  return (int)(b < 1 ? 1 : (b > cap ? cap : b));
}

// Threads that share a token, and blocks beside the token blocks that clear padding rows.
int threads_per_token(int HV) { return HV <= 64 ? 32 : (HV <= 256 ? 64 : 128); }
// Blocks along a row where the tokens alone do not fill the GPU (a single token: its columns over as many SMs).
int row_blocks(int HV, int tpt, int tok_blocks) {
  const int want = 2 * num_sms() / tok_blocks, most = (HV + tpt - 1) / tpt;
  return want < 1 ? 1 : (want < most ? want : most);
}
int pad_blocks(int R, int threads) {
  const long long b = ((long long)R * 32 + threads - 1) / threads, cap = num_sms();
  return (int)(b > cap ? cap : b);
}

// The backward of 16-bit rows moves 8 bytes a thread at most: 8 rows of ys in whole units hold 32 registers more and leave
// fewer warps. 4096 x 8 rows of 5120 bf16: 150 us against 172; of 2560: 82 against 105.
int back_unit(int type, int unit) { return type != CBMOE_F32 && unit == 16 ? 8 : unit; }
size_t elem_size(int type) { return type == CBMOE_F32 ? 4 : 2; }

int unit_bytes(int type, int H, const void* a, const void* b, const void* c = nullptr) {
  const uintptr_t all = (uintptr_t)H * elem_size(type) | reinterpret_cast<uintptr_t>(a) |
                        reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c) | 16;
  return (int)(all & (~all + 1));   // the lowest bit that is set
}

template <typename T, int VB>
int permute_t(const void* x, int Tn, int H, const int32_t* row_slot, int k, const int32_t* tok_row, int R, void* xs,
              cudaStream_t s) {
  using V = Vec<T, VB>;
  const int HV = H / V::n, tpt = threads_per_token(HV), tb = blocks_for(Tn, kPermThreads / tpt, 64);
  CBMOE_CUDA_TRY(launch_pdl(permute_kernel<T, VB>, dim3(tb + pad_blocks(R, kPermThreads), row_blocks(HV, tpt, tb)),
                            dim3(kPermThreads), 0, s,
                            static_cast<const V*>(x), Tn, HV, row_slot, k, tok_row, R, static_cast<V*>(xs), tb, tpt));
  return CBMOE_OK;
}

template <typename T, int VB, typename O = T>
int unpermute_t(const void* ys, int R, int H, const int32_t* row_slot, const float* w, int Tn, int k, void* y,
                cudaStream_t s) {
  using V = Vec<T, VB>;
  const int HV = H / V::n;
  const int tpt = threads_per_token(HV), tb = blocks_for(Tn, kPermThreads / tpt, 64);
  CBMOE_CUDA_TRY(launch_pdl(unpermute_kernel<T, VB, O>, dim3(tb, row_blocks(HV, tpt, tb)), dim3(kPermThreads), 0, s,
                            static_cast<const V*>(ys), R, HV, row_slot, w, Tn, k, static_cast<Out<T, VB, O>*>(y), tpt));
  return CBMOE_OK;
}

template <typename T, int VB>
int unpermute_backward_t(const void* dy, const void* ys, int R, int H, const int32_t* row_slot, const int32_t* tok_row,
                         const float* w, int Tn, int k, void* dys, float* dw, cudaStream_t s) {
  using V = Vec<T, VB>;
  const int HV = H / V::n, tb = blocks_for(Tn, 1, 64);
  const int pb = dys != nullptr ? pad_blocks(R, kBackThreads) : 0;
  CBMOE_CUDA_TRY(launch_pdl(unpermute_backward_kernel<T, VB>, dim3(tb + pb), dim3(kBackThreads), 0, s,
                            static_cast<const V*>(dy), static_cast<const V*>(ys), R, HV, row_slot, tok_row, w, Tn, k,
                            static_cast<V*>(dys), dw, tb));
  return CBMOE_OK;
}

bool type_ok(int t) { return t == CBMOE_BF16 || t == CBMOE_F16 || t == CBMOE_F32; }

// Elements of `size` bytes at each of the pointers.
template <typename... P>
bool aligned(size_t size, const P*... p) {
  return ((reinterpret_cast<uintptr_t>(p) | ...) & (size - 1)) == 0;
}

// The kernels' strided loops count in 32 bits: a count and the largest step (a row's columns over 2 * 148 blocks of 128
// threads) stay below 2^31.
bool counts_ok(int T, int R, int H, int k) {
  constexpr int kMost = 0x7fff0000;
  return T <= kMost && R <= kMost && H <= kMost && k <= kMost;
}

}  // namespace

// f<T, VB>(args...) for the type and the unit's bytes.
#define CBMOE_BY_UNIT(f, T, unit, ...) \
  ((unit) == 16 ? f<T, 16>(__VA_ARGS__) : (unit) == 8 ? f<T, 8>(__VA_ARGS__) : f<T, 4>(__VA_ARGS__))
#define CBMOE_BY_TYPE(f, type, unit, ...)                                                     \
  ((type) == CBMOE_F32    ? CBMOE_BY_UNIT(f, float, unit, __VA_ARGS__)                        \
   : (type) == CBMOE_BF16 ? ((unit) == 2 ? f<__nv_bfloat16, 2>(__VA_ARGS__)                   \
                                         : CBMOE_BY_UNIT(f, __nv_bfloat16, unit, __VA_ARGS__)) \
                          : ((unit) == 2 ? f<__half, 2>(__VA_ARGS__) : CBMOE_BY_UNIT(f, __half, unit, __VA_ARGS__)))

namespace {

template <typename T, int VB>
int unpermute_to_bf16(const void* ys, int R, int H, const int32_t* row_slot, const float* w, int Tn, int k, void* y,
                      cudaStream_t s) {
  return unpermute_t<T, VB, __nv_bfloat16>(ys, R, H, row_slot, w, Tn, k, y, s);
}
template <typename T, int VB>
int unpermute_to_f16(const void* ys, int R, int H, const int32_t* row_slot, const float* w, int Tn, int k, void* y,
                     cudaStream_t s) {
  return unpermute_t<T, VB, __half>(ys, R, H, row_slot, w, Tn, k, y, s);
}

}  // namespace

// The expert layer's combine: fp32 slots, y in any type. 4096 x 8 rows of 5120 into fp32: 130 us, 115 at the copy rate.
int launch_unpermute_f32(const float* ys, int R, int H, const int32_t* row_slot, const float* w, int T, int k, void* y,
                         int y_type, cudaStream_t stream) {
  // 16-bit rows of y are half as wide as those of ys: a unit of y is aligned where twice its address is
  const uintptr_t y_as = reinterpret_cast<uintptr_t>(y) * (y_type == CBMOE_F32 ? 1 : 2);
  const int unit = unit_bytes(CBMOE_F32, H, ys, reinterpret_cast<const void*>(y_as));
  prof_begin(kProfCombine, stream);
  const int rc = y_type == CBMOE_F32 ? CBMOE_BY_UNIT(unpermute_t, float, unit, ys, R, H, row_slot, w, T, k, y, stream)
                 : y_type == CBMOE_BF16
                     ? CBMOE_BY_UNIT(unpermute_to_bf16, float, unit, ys, R, H, row_slot, w, T, k, y, stream)
                     : CBMOE_BY_UNIT(unpermute_to_f16, float, unit, ys, R, H, row_slot, w, T, k, y, stream);
  prof_end(kProfCombine, stream);
  if (rc) return rc;
  CBMOE_CUDA_TRY(cudaGetLastError());
  return CBMOE_OK;
}

}  // namespace cbmoe

using namespace cbmoe;

extern "C" int cbmoe_permute(const void* x, int type, int T, int H, const int32_t* row_slot, int k,
                             const int32_t* tok_row, int R, void* xs, cudaStream_t stream) {
  if (!type_ok(type) || T < 0 || H <= 0 || k <= 0 || R < 0) return CBMOE_ERR_INVALID;
  if ((T > 0 && (!x || !row_slot)) || (R > 0 && (!tok_row || !xs))) return CBMOE_ERR_INVALID;
  if (!aligned(elem_size(type), x, xs) || !aligned(4, row_slot, tok_row)) return CBMOE_ERR_INVALID;
  if (!counts_ok(T, R, H, k)) return CBMOE_ERR_UNSUPPORTED;
  if (R == 0) return CBMOE_OK;
  prof_begin(kProfOther, stream);
  const int rc = CBMOE_BY_TYPE(permute_t, type, unit_bytes(type, H, x, xs), x, T, H, row_slot, k, tok_row, R, xs, stream);
  prof_end(kProfOther, stream);
  if (rc) return rc;
  CBMOE_CUDA_TRY(cudaGetLastError());
  return CBMOE_OK;
}

extern "C" int cbmoe_unpermute(const void* ys, int type, int R, int H, const int32_t* row_slot, const float* w, int T,
                               int k, void* y, cudaStream_t stream) {
  if (!type_ok(type) || T < 0 || H <= 0 || k <= 0 || R < 0) return CBMOE_ERR_INVALID;
  if (T > 0 && (!row_slot || !y || (R > 0 && !ys))) return CBMOE_ERR_INVALID;
  if (!aligned(elem_size(type), ys, y) || !aligned(4, row_slot, w)) return CBMOE_ERR_INVALID;
  if (!counts_ok(T, R, H, k)) return CBMOE_ERR_UNSUPPORTED;
  if (T == 0) return CBMOE_OK;
  prof_begin(kProfCombine, stream);
  const int rc = CBMOE_BY_TYPE(unpermute_t, type, unit_bytes(type, H, ys, y), ys, R, H, row_slot, w, T, k, y, stream);
  prof_end(kProfCombine, stream);
  if (rc) return rc;
  CBMOE_CUDA_TRY(cudaGetLastError());
  return CBMOE_OK;
}

extern "C" int cbmoe_unpermute_backward(const void* dy, const void* ys, int type, int R, int H,
                                        const int32_t* row_slot, const int32_t* tok_row, const float* w, int T, int k,
                                        void* dys, float* dw, cudaStream_t stream) {
  if (!type_ok(type) || T < 0 || H <= 0 || k <= 0 || R < 0) return CBMOE_ERR_INVALID;
  if ((T > 0 && (!dy || !row_slot)) || (dw && R > 0 && !ys) || (dys && R > 0 && !tok_row)) return CBMOE_ERR_INVALID;
  if (!aligned(elem_size(type), dy, ys, dys) || !aligned(4, row_slot, tok_row, w, dw)) return CBMOE_ERR_INVALID;
  if (!counts_ok(T, R, H, k)) return CBMOE_ERR_UNSUPPORTED;
  if (!dys && !dw) return CBMOE_OK;
  if (T == 0 && (!dys || R == 0)) return CBMOE_OK;
  prof_begin(kProfCombine, stream);
  const int unit = back_unit(type, unit_bytes(type, H, dy, dys, ys));
  const int rc = CBMOE_BY_TYPE(unpermute_backward_t, type, unit, dy, ys, R, H, row_slot, tok_row, w, T, k, dys, dw,
                               stream);
  prof_end(kProfCombine, stream);
  if (rc) return rc;
  CBMOE_CUDA_TRY(cudaGetLastError());
  return CBMOE_OK;
}
