// Products in 8-bit floating point (e4m3): fp8_linear and the routed experts on such tables.
//
//   y[n, r] = sum_b sx[n, b] * sw[r / 128, b] * sum_{c in block b} xq[n, c] * wq[r, c]
//
// fp8_gemm_kernel, one CTA per SM, 12 warps:
//   warp 0      TMA producer: per 128-column block the tile's MT x 128 B of tokens and 2 x 128 x 128 B of weights (128-byte
//               swizzle), into a ring of stages
//   warp 1      TMEM owner and MMA issuer (one thread): 4 tcgen05.mma kind::f8f6f4 (M 128 x N 256 x K 32) per block into
//               one of two 256-column accumulators
//   warps 4-11  promotion and epilogue: a block's 128 x 256 partial sums leave TMEM while the tensor core works on the next
//               block; acc += partial * (sx * sw) in fp32 registers (32 rows x 128 columns per warp). Tokens are the M side,
//               so a thread owns one token row: both scales are scalars for its columns. These warps take the registers
//               that the first warpgroup gives up (128 accumulators + two 32-column loads in turn a thread).
// The block's partial sum is exact enough to be added as it is: e4m3 products are exact in fp32 and the tensor core sums
// them in fp32 (measured: 1e-8 relative over K = 128).
// With many rows (MT = 256) two CTAs of a cluster work as a pair (cta_group::2, M = 256): each brings 128 tokens and half
// of the weight tile, so a block costs an SM 32 KB of shared-memory writes and 32 KB of operand reads where a CTA alone
// costs it 48 and 48, which at 128 B a clock is more than the 512 clocks of its MMAs (measured at 4096 x 5120 x 12288:
// alone 1300 clocks a block, 1070 with the promotion left out).
// With two matrices (gate, up: 128 columns each) the epilogue forms swiglu_clamped(gate, up), takes each row's maximum
// over its 128 columns and stores e4m3 codes and the scale: the down product's input, never in 16 bits.
// Work: whole waves of output tiles, one tile per CTA; the tiles left over are cut along K into equal ranges of blocks, one
// per CTA (Fp8Sched), so that few rows (a single token: all of the time) still use every SM and the memory behind it. A
// tile's ranges leave fp32 partial sums in the workspace; the last to arrive adds them in range order (the same bits on
// every call) and runs the epilogue.
// Every wait is bounded; a role that gives up sets CBMOE_DEVERR_TIMEOUT and falls through to the final barrier.
#define CBMOE_OWN_UNIT
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
                                                           float* __restrict__ s, int lds,
                                                           const int* __restrict__ row_slot, int k, int R, int* __restrict__ zero, int n_zero) {
  griddep_wait();
  griddep_launch();
  for (int i = blockIdx.x * 256 + threadIdx.x; i < n_zero; i += gridDim.x * 256) zero[i] = 0;
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
      if (l == 0) s[(size_t)r * lds + kb] = sc;
    }
  }
}

// --------------------------------------------------------------------------------------------------- product
constexpr int kFp8Threads = 12 * 32;
constexpr int kW0 = 4;                                   // first promotion warp
constexpr int kBHalf = 128 * 128;                        // 128 weight rows of one block
constexpr int kRegsIdle = 40, kRegsWork = 232;           // 128 * 40 + 256 * 232 = 384 * 168, the launch's registers

template <int MT>
struct Fp8Cfg {
  static constexpr bool kPair = MT == 256;               // two CTAs, 128 tokens each
  static constexpr int kRows = kPair ? 128 : MT;         // tokens of a CTA's tile
  static constexpr int kATile = kRows * 128;
  static constexpr int kStage = kATile + (kPair ? 1 : 2) * kBHalf;
  static constexpr int kNStage = kPair ? 6 : (MT == 128 ? 4 : (MT == 64 ? 5 : 6));
  static constexpr int kBarOff = kNStage * kStage;
  static constexpr int kMaxOff = kBarOff + 256;          // row maxima [2][4 quadrants][2 halves][32] f32
  static constexpr int kFlagOff = kMaxOff + 2048;        // [2][4] int
  static constexpr int kSmem = 1024 + kFlagOff + 32;
  static_assert(kSmem <= 227 * 1024, "shared memory budget");
};

struct Fp8Params {
  Fp8Gemm g;
  int KB, RB, NT;          // column blocks, 128-row blocks per matrix, output tiles per pass
  int hs_ld;               // row stride of hs
  int xs_wide;             // xs rows are 16-byte aligned
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

// A worker's (a CTA's, or a pair's) share of the tiles, in segments (tile, blocks [kb0, kb1)).
struct Fp8Seg {
  int item, kb0, kb1;
};
struct Fp8Sched {
  int waves, first, KB, chunk, u, u1, i, worker, G;

  // Ranges shorter than 4 blocks would spend more on joining them than on their sums.
  // Worker `w` of `G` (a CTA, or a pair).
  __device__ __forceinline__ Fp8Sched(int n_items, int kb, int w, int g) : KB(kb), i(0), worker(w), G(g) {
    const int rem = n_items % G;
    waves = n_items / G;
    first = waves * G;
    chunk = max((rem * KB + G - 1) / G, min(KB, 4));
    u = min(rem * KB, worker * chunk);
    u1 = min(rem * KB, u + chunk);
  }
  __device__ __forceinline__ bool next(Fp8Seg& s) {
    if (i < waves) {
      s = {i * G + worker, 0, KB};
      ++i;
      return true;
    }
    if (u >= u1) return false;
    const int t = u / KB, kb0 = u - t * KB, kb1 = min(KB, kb0 + u1 - u);
    s = {first + t, kb0, kb1};
    u += kb1 - kb0;
    return true;
  }
  // The workers [c0, c1] that share a left-over tile, and where a worker's partial sums of it lie.
  __device__ __forceinline__ void sharers(int item, int& c0, int& c1) const {
    const int b = (item - first) * KB;
    c0 = b / chunk;
    c1 = (b + KB - 1) / chunk;
  }
  __device__ __forceinline__ int slot(int w, int item) const { return 2 * w + (w * chunk / KB == item - first ? 0 : 1); }
};

template <typename OUT>
__device__ __forceinline__ OUT out_of(float v);
template <>
__device__ __forceinline__ float out_of(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 out_of(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half out_of(float v) { return __float2half_rn(v); }

__device__ __forceinline__ void store32(void* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
               "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// silu(min(g, L)) * clip(u, -L, L) (model.py:119-122) that keeps a NaN, so that a bad row shows.
__device__ __forceinline__ float swiglu_keep_nan(float g, float u, float limit) {
  g = g > limit ? limit : g;
  u = u > limit ? limit : (u < -limit ? -limit : u);
  return silu_f(g) * u;
}

// The two warps of a row quadrant wait for one another (bounded); `n` counts their meetings.
__device__ __forceinline__ bool pair_meet(uint64_t* bar, uint32_t& n) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
  return mbar_wait(bar, n++ & 1);
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
  uint64_t* meet = d_empty + 2;             // [4]
  uint64_t* peer = meet + 4;                // [kNStage] pair, in rank 0: the other CTA's stage is full
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(peer + C::kNStage);
  float* row_max = reinterpret_cast<float*>(smem + C::kMaxOff);
  volatile int* flag = reinterpret_cast<volatile int*>(smem + C::kFlagOff);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kNStage; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
      mbar_init(&peer[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&d_full[i], 1);
      mbar_init(&d_empty[i], C::kPair ? 16 : 8);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&meet[i], 2);
    fence_mbar_init();
  }
  if (warp == 1) {
    if constexpr (C::kPair) tmem_alloc_pair(tmem_slot, 512);
    else tmem_alloc(tmem_slot, 512);
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&map_x);
    prefetch_tmap(&map_w0);
    prefetch_tmap(&map_w1);
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (C::kPair) cluster_sync();    // the other CTA's barriers are set up
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int rank = C::kPair ? (int)cluster_rank() : 0, group = C::kPair ? 2 : 1;
  griddep_wait();
  griddep_launch();

  if (warp < kW0) {
    regs_give_up<kRegsIdle>();
    Fp8Sched sched(fp8_items<MT>(p), p.KB, blockIdx.x / group, gridDim.x / group);
    Fp8Seg sg;
    // Whole warps walk these loops and one elected lane issues: addresses and descriptors stay in uniform registers, which
    // halves the instructions of an issue (measured beside the promotion warps: 870 -> 760 clocks a block).
    int st = 0;
    uint32_t ph = 0;
    if (warp == 0) {
      while (sched.next(sg)) {
        const Fp8Item it = fp8_item<MT>(p, sg.item);
        const int wrow = it.e * p.g.rows + it.nt * (SWIGLU ? 128 : 256), xrow = it.row0 + 128 * rank;
#pragma unroll 1
        for (int kb = sg.kb0; kb < sg.kb1; ++kb) {
          if (!mbar_wait(&empty[st], ph ^ 1)) goto done;
          uint8_t* a = smem + st * C::kStage;
          if (elect_one()) {
            mbar_arrive_expect_tx(&full[st], C::kStage);
            tma_load_2d(a, &map_x, kb * kFp8Group, xrow, &full[st]);
            if (!C::kPair || rank == 0) tma_load_2d(a + C::kATile, &map_w0, kb * kFp8Group, wrow, &full[st]);
            if (!C::kPair || rank == 1)
              tma_load_2d(a + C::kATile + (C::kPair ? 0 : kBHalf), SWIGLU ? &map_w1 : &map_w0, kb * kFp8Group,
                          SWIGLU ? wrow : wrow + 128, &full[st]);
          }
          __syncwarp();
          if (++st == C::kNStage) {
            st = 0;
            ph ^= 1;
          }
        }
      }
    } else if (warp == 1 && rank == 1) {
      // The pair's MMAs are issued by rank 0: tell it which of this CTA's stages are full.
      while (sched.next(sg)) {
#pragma unroll 1
        for (int kb = sg.kb0; kb < sg.kb1; ++kb) {
          if (!mbar_wait(&full[st], ph)) goto done;
          if (elect_one()) mbar_arrive_remote(&peer[st], 0);
          __syncwarp();
          if (++st == C::kNStage) {
            st = 0;
            ph ^= 1;
          }
        }
      }
    } else if (warp == 1) {
      constexpr uint32_t idesc = idesc_e4m3(C::kPair ? 256 : 128, kFp8TileN);
      const uint64_t desc0 = sw128_desc(smem_addr(smem));
      uint32_t buf = 0, dph = 1;
      while (sched.next(sg)) {
#pragma unroll 1
        for (int kb = sg.kb0; kb < sg.kb1; ++kb) {
          if (!mbar_wait(&d_empty[buf], dph) || !mbar_wait(&full[st], ph)) goto done;
          if (C::kPair && !mbar_wait(&peer[st], ph)) goto done;
          tc_fence_after();
          // Rows kRows.. of the M side are whatever follows in the stage (weights): their sums are never read.
          const uint64_t ad = desc0 + (uint32_t)st * (C::kStage >> 4), bd = ad + (C::kATile >> 4);
          const uint32_t d = tmem + buf * kFp8TileN;
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
              if constexpr (C::kPair) umma_fp8_pair(d, ad + 2 * kk, bd + 2 * kk, idesc, kk != 0);
              else umma_fp8(d, ad + 2 * kk, bd + 2 * kk, idesc, kk != 0);
            }
            if constexpr (C::kPair) {
              umma_commit_pair(&empty[st]);
              umma_commit_pair(&d_full[buf]);
            } else {
              umma_commit(&empty[st]);
              umma_commit(&d_full[buf]);
            }
          }
          __syncwarp();
          if (++st == C::kNStage) {
            st = 0;
            ph ^= 1;
          }
          buf ^= 1;
          dph ^= buf ^ 1;
        }
      }
    }
  } else {
    regs_take<kRegsWork>();
    Fp8Sched sched(fp8_items<MT>(p), p.KB, blockIdx.x / group, gridDim.x / group);
    Fp8Seg sg;
    const int q = warp & 3;                  // TMEM lane quadrant this warp may read
    const int half = (warp - kW0) >> 2;
    uint32_t n = 0, met = 0;
    auto d_read = [&](int buf) {             // to the CTA that issues the MMAs
      if (rank == 0) mbar_arrive(&d_empty[buf]);
      else mbar_arrive_remote(&d_empty[buf], 0);
    };
    while (sched.next(sg)) {
      Fp8Item it = fp8_item<MT>(p, sg.item);
      it.row0 += 128 * rank;                 // this CTA's rows of the tile
      it.cnt -= 128 * rank;
      const int m = 32 * q + lane;
      const bool live = 32 * q < it.cnt, mine = m < it.cnt;
      const size_t xrow = mine ? (size_t)it.row0 + m : 0;
      const float* sx = p.g.xs + xrow * p.g.ldxs;
      const float *sa, *sb;                  // scales of this thread's columns 0-63 and 64-127
      if constexpr (SWIGLU) {
        sa = p.g.s0 + ((size_t)it.e * p.RB + it.nt) * p.KB;
        sb = p.g.s1 + ((size_t)it.e * p.RB + it.nt) * p.KB;
      } else {
        sa = p.g.s0 + ((size_t)it.e * p.RB + min(2 * it.nt + half, p.RB - 1)) * p.KB;
        sb = sa;
      }
      float acc[128];
#pragma unroll
      for (int i = 0; i < 128; ++i) acc[i] = 0.f;
      // Scales come four blocks ahead of their use (a load's latency under the tiles' traffic is longer than a block):
      // this row's own, four blocks at a time; the weights', one block per lane.
      auto row_scales = [&](int kb) {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (p.xs_wide && kb % 4 == 0) {
          if (kb < sg.kb1) v = *reinterpret_cast<const float4*>(sx + kb);
        } else {
          if (kb < sg.kb1) v.x = sx[kb];
          if (kb + 1 < sg.kb1) v.y = sx[kb + 1];
          if (kb + 2 < sg.kb1) v.z = sx[kb + 2];
          if (kb + 3 < sg.kb1) v.w = sx[kb + 3];
        }
        return v;
      };
      float4 xn = row_scales(sg.kb0), xc = xn;
      float wa = 0.f, wb = 0.f, wa_n = 0.f, wb_n = 0.f;
      if (sg.kb0 + lane < sg.kb1) {
        wa_n = sa[sg.kb0 + lane];
        if constexpr (SWIGLU) wb_n = sb[sg.kb0 + lane];
      }
      // Not unrolled: 128 multiply-adds a turn fill the instruction cache that the MMA issuer shares.
#pragma unroll 1
      for (int kb = sg.kb0; kb < sg.kb1; ++kb) {
        const int at = kb - sg.kb0;
        if (at % 4 == 0) {
          xc = xn;
          xn = row_scales(kb + 4);
        }
        if (at % 32 == 0) {
          wa = wa_n, wb = wb_n;
          if (kb + 32 + lane < sg.kb1) {
            wa_n = sa[kb + 32 + lane];
            if constexpr (SWIGLU) wb_n = sb[kb + 32 + lane];
          }
        }
        const int buf = n & 1;
        const float fa = xc.x * __shfl_sync(0xffffffffu, wa, at);
        const float fb = SWIGLU ? xc.x * __shfl_sync(0xffffffffu, wb, at) : fa;
        xc.x = xc.y, xc.y = xc.z, xc.z = xc.w;
        if (!mbar_wait(&d_full[buf], (n >> 1) & 1)) goto done;
        ++n;
        tc_fence_after();
        if (live) {
          const uint32_t t0 = tmem + buf * kFp8TileN + ((uint32_t)(32 * q) << 16);
          // 16 columns at a time: the two warps of a scheduler take turns between a load and its multiply-adds, and
          // 128 + 16 registers a thread leave nothing to spill (loads of 32 columns or two in flight measured the same
          // in a loop of their own, 350-370 clocks a block, and spilled here).
#pragma unroll
          for (int c = 0; c < 8; ++c) {       // 0-3 gate and 4-7 up; or 8 in a row
            float v[16];
            tmem_ld16(t0 + (SWIGLU ? (c < 4 ? 64 * half + 16 * c : 64 + 64 * half + 16 * c) : 128 * half + 16 * c), v);
            if (c == 7) {                     // all of this block is in registers
              tc_fence_before();
              __syncwarp();
              if (lane == 0) d_read(buf);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[16 * c + i] = fmaf(v[i], c < 4 ? fa : fb, acc[16 * c + i]);
          }
        } else if (lane == 0) {
          d_read(buf);
        }
      }
      const int rows = p.g.rows;
      if (sg.kb0 == 0 && sg.kb1 == p.KB) {
        // ------------------------------------------------------------- the whole sum: this thread's row, 128 columns
        if constexpr (SWIGLU) {
          const int col0 = it.nt * 128 + 64 * half;
          float top = 0.f;
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            float h[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              h[c] = col0 + 2 * i + c < rows
                         ? swiglu_keep_nan(acc[2 * i + c], acc[64 + 2 * i + c], p.g.limit)
                         : 0.f;
              top = max_nan(top, fabsf(h[c]));
            }
            acc[2 * i] = h[0];
            acc[2 * i + 1] = h[1];
          }
          float* mx = row_max + ((met & 1) * 4 + q) * 64;
          mx[half * 32 + lane] = top;
          if (!pair_meet(&meet[q], met)) goto done;
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
                w[i] = fp8_pack4(acc[c] * inv, acc[c + 1] * inv, acc[c + 2] * inv,
                                 acc[c + 3] * inv);
              }
              dst[u] = make_uint4(w[0], w[1], w[2], w[3]);
            }
            if (half == 0) p.g.hs[xrow * p.hs_ld + it.nt] = sc;
          }
        } else if (mine) {
          const int col0 = it.nt * 256 + 128 * half;
          OUT* dst = static_cast<OUT*>(p.g.out) + xrow * rows + col0;
          constexpr int kU = 32 / (int)sizeof(OUT);        // one 32-byte store: a whole sector of this row
          if (rows % kU == 0 && (reinterpret_cast<uintptr_t>(p.g.out) & 31) == 0) {
#pragma unroll
            for (int u = 0; u < 128 / kU; ++u) {
              union {
                uint32_t w[8];
                OUT o[kU];
              } b;
#pragma unroll
              for (int i = 0; i < kU; ++i) b.o[i] = out_of<OUT>(acc[u * kU + i]);
              if (col0 + u * kU < rows) store32(dst + u * kU, b.w);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 128; ++i)
              if (col0 + i < rows) dst[i] = out_of<OUT>(acc[i]);
          }
        }
        continue;
      }
      // ----------------------------------------------- a range of the sum: partial sums [slot][rank][half][row][128 columns]
      int c0, c1;
      sched.sharers(sg.item, c0, c1);
      auto part = [&](int w, int row) {
        const size_t at = ((size_t)sched.slot(w, sg.item) * group + rank) * 2 + half;
        return reinterpret_cast<float4*>(p.g.part) + (at * C::kRows + row) * 32;
      };
      int* arrived = p.g.arrived + ((sg.item - sched.first) * group + rank) * 8;
      if (mine) {
        float4* dst = part(sched.worker, m);
#pragma unroll
        for (int i = 0; i < 32; ++i)
          __stcg(dst + i, make_float4(acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3]));
      }
      __threadfence();
      bool last;
      if constexpr (SWIGLU) {
        if (!pair_meet(&meet[q], met)) goto done;          // both halves are written
        if (half == 0 && lane == 0) {
          flag[(met & 1) * 4 + q] = atomicAdd(&arrived[q], 1) == c1 - c0;
          __threadfence();
        }
        const int at = (met & 1) * 4 + q;
        if (!pair_meet(&meet[q], met)) goto done;
        last = flag[at] != 0;
      } else {
        int old = 0;
        __syncwarp();
        if (lane == 0) old = atomicAdd(&arrived[4 * half + q], 1);
        last = __shfl_sync(0xffffffffu, old, 0) == c1 - c0;
      }
      if (!last) continue;
      __threadfence();
      // The last worker of the tile: lanes take columns now (4 each), rows one after another.
      const int nr = min(32, it.cnt - 32 * q);
      // 8 rows at a time, so that 8 loads (16 for two matrices) are under way at once.
      for (int r0 = 0; r0 < nr; r0 += 8) {
        float4 sum[8];                       // SwiGLU: gate columns in x, y and up columns in z, w
#pragma unroll
        for (int r = 0; r < 8; ++r) sum[r] = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int c = c0; c <= c1; ++c) {
          const float4* src = part(c, 32 * q + r0);
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            if (r0 + r >= nr) break;
            float4 a;
            if constexpr (SWIGLU) {
              const float2* s2 = reinterpret_cast<const float2*>(src + 32 * r);
              const float2 g = __ldcg(s2 + lane), u = __ldcg(s2 + 32 + lane);
              a = make_float4(g.x, g.y, u.x, u.y);
            } else {
              a = __ldcg(src + 32 * r + lane);
            }
            sum[r].x += a.x;
            sum[r].y += a.y;
            sum[r].z += a.z;
            sum[r].w += a.w;
          }
        }
        if constexpr (SWIGLU) {
          const int col0 = it.nt * 128 + 64 * half + 2 * lane;
          float* mx = row_max + ((met & 1) * 4 + q) * 64;
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            sum[r].x = col0 < rows ? swiglu_keep_nan(sum[r].x, sum[r].z, p.g.limit) : 0.f;
            sum[r].y = col0 + 1 < rows ? swiglu_keep_nan(sum[r].y, sum[r].w, p.g.limit) : 0.f;
            float top = max_nan(fabsf(sum[r].x), fabsf(sum[r].y));
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, d));
            if (lane == 0) mx[half * 32 + r] = top;
          }
          if (!pair_meet(&meet[q], met)) goto done;
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            if (r0 + r >= nr) break;
            float inv;
            const float sc = fp8_group_scale(max_nan(mx[r], mx[32 + r]), &inv);
            const size_t row = (size_t)it.row0 + 32 * q + r0 + r;
            *reinterpret_cast<uint16_t*>(p.g.hq + row * ((size_t)p.RB * 128) + col0) = (uint16_t)__nv_cvt_float2_to_fp8x2(
                make_float2(sum[r].x * inv, sum[r].y * inv), __NV_SATFINITE, __NV_E4M3);
            if (half == 0 && lane == 0) p.g.hs[row * p.hs_ld + it.nt] = sc;
          }
        } else {
          const int col0 = it.nt * 256 + 128 * half + 4 * lane;
          const bool wide = rows % 4 == 0 && (reinterpret_cast<uintptr_t>(p.g.out) & 15) == 0;
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            if (r0 + r >= nr) break;
            struct alignas(4 * sizeof(OUT)) Out4 {
              OUT o[4];
            } b = {{out_of<OUT>(sum[r].x), out_of<OUT>(sum[r].y), out_of<OUT>(sum[r].z), out_of<OUT>(sum[r].w)}};
            OUT* dst = static_cast<OUT*>(p.g.out) + ((size_t)it.row0 + 32 * q + r0 + r) * rows + col0;
            if (wide) {
              if (col0 < rows) *reinterpret_cast<Out4*>(dst) = b;
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (col0 + i < rows) dst[i] = b.o[i];
            }
          }
        }
      }
    }
  }
done:
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if constexpr (C::kPair) cluster_sync();    // neither CTA leaves while the other may reach into it
  if (warp == 1) {
    tc_fence_after();
    if constexpr (C::kPair) tmem_dealloc_pair(tmem, 512);
    else tmem_dealloc(tmem, 512);
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
  p.hs_ld = fp8_scale_stride(g.rows);
  p.xs_wide = g.ldxs % 4 == 0 && (reinterpret_cast<uintptr_t>(g.xs) & 15) == 0;
  p.NT = SWIGLU ? p.RB : (p.RB + 1) / 2;
  CUtensorMap mx, m0, m1;
  int rc = make_fp8_map(&mx, g.xq, g.K, g.x_rows, g.ldx, C::kRows);
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
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(C::kPair ? num_sms() & ~1 : num_sms());
  cfg.blockDim = dim3(kFp8Threads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = C::kPair ? 2 : 1;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  CBMOE_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, p, mx, m0, m1));
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

int fp8_pass_tokens(long long slots, int E) {
  return slots <= 32LL * E ? 32 : (slots <= 64LL * E ? 64 : (slots <= 128LL * E ? 128 : 256));
}

int fp8_device_errors(int clear, int* out_host) {
  CBMOE_CUDA_TRY(cudaMemcpyFromSymbol(out_host, g_device_errors, sizeof(int)));
  const int zero = 0;
  if (clear && *out_host) CBMOE_CUDA_TRY(cudaMemcpyToSymbol(g_device_errors, &zero, sizeof(int)));
  return CBMOE_OK;
}

size_t fp8_part_bytes(int mt) { return (size_t)num_sms() * 2 * (mt < 128 ? mt : 128) * kFp8TileN * 4; }

int fp8_arrived() { return num_sms() * 8; }

int launch_fp8_gemm(const Fp8Gemm& g, int mt, cudaStream_t s) {
  if (mt == 32) return launch_mt<32>(g, s);
  if (mt == 64) return launch_mt<64>(g, s);
  if (mt == 128) return launch_mt<128>(g, s);
  return launch_mt<256>(g, s);
}

int launch_fp8_quantize(const void* x, int type, int N, int K, long long ldx, uint8_t* q, long long ldq, float* s, int lds,
                        const int* row_slot, int k, int R, int* zero, int n_zero, cudaStream_t stream) {
  const long long groups = (long long)N * blocks_of(K);
  long long blocks = (groups + 15) / 16, cap = (long long)num_sms() * 16;
  if (blocks > cap) blocks = cap;
  const int size = type == CBMOE_F32 ? 4 : 2;
  const int vec = aligned(x, 16) && ldx * size % 16 == 0;
  prof_begin(kProfOther, stream);
  if (type == CBMOE_BF16)
    CBMOE_CUDA_TRY(launch_pdl(fp8_quantize_kernel<__nv_bfloat16>, dim3((int)blocks), dim3(256), 0, stream,
                              static_cast<const __nv_bfloat16*>(x), N, K, ldx, vec, q, ldq, s, lds, row_slot, k, R, zero,
                              n_zero));
  else if (type == CBMOE_F16)
    CBMOE_CUDA_TRY(launch_pdl(fp8_quantize_kernel<__half>, dim3((int)blocks), dim3(256), 0, stream,
                              static_cast<const __half*>(x), N, K, ldx, vec, q, ldq, s, lds, row_slot, k, R, zero,
                              n_zero));
  else
    CBMOE_CUDA_TRY(launch_pdl(fp8_quantize_kernel<float>, dim3((int)blocks), dim3(256), 0, stream,
                              static_cast<const float*>(x), N, K, ldx, vec, q, ldq, s, lds, row_slot, k, R, zero,
                              n_zero));
  prof_end(kProfOther, stream);
  CBMOE_CUDA_TRY(cudaGetLastError());
  return CBMOE_OK;
}

namespace {

// Workspace of a product: partial sums | counters | q [N][blocks * 128] | s [N][blocks] (the last two where x is quantised
// here).
struct LinearWs {
  size_t arrived, xq, xs, total;
  int mt;
};
LinearWs linear_ws(int N, int K, bool ready) {
  LinearWs w;
  w.mt = fp8_pass_tokens(N, 1);
  w.arrived = lyr::align_up(fp8_part_bytes(w.mt));
  w.xq = w.arrived + lyr::align_up((size_t)fp8_arrived() * 4);
  w.xs = w.xq + (ready ? 0 : lyr::align_up((size_t)N * blocks_of(K) * kFp8Group));
  w.total = w.xs + (ready ? 0 : lyr::align_up((size_t)N * fp8_scale_stride(K) * 4));
  return w;
}

// Workspace of the layer: plan | partial sums | counters (gate/up, down) | xq, xs (sorted rows) | hq, hs | slot outputs.
struct ExpertsWs {
  size_t plan, part, arrived, xq, xs, hq, hs, y, total;
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
  w.part = lyr::align_up((size_t)w.L.off[13] * 4);
  w.arrived = w.part + lyr::align_up(fp8_part_bytes(w.mt));
  w.xq = w.arrived + lyr::align_up((size_t)fp8_arrived() * 2 * 4);
  w.xs = w.xq + lyr::align_up((size_t)S * blocks_of(H) * kFp8Group);
  w.hq = w.xs + lyr::align_up((size_t)S * fp8_scale_stride(H) * 4);
  w.hs = w.hq + lyr::align_up((size_t)S * blocks_of(I) * kFp8Group);
  w.y = w.hs + lyr::align_up((size_t)S * fp8_scale_stride(I) * 4);
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
  return launch_fp8_quantize(x, type, N, K, ldx, q, ldq, s, blocks_of(K), nullptr, 1, N, nullptr, 0, stream);
}

extern "C" size_t cbmoe_fp8_linear_workspace_bytes(int N, int K, int rows, int x_type) {
  if (N < 0 || K <= 0 || rows <= 0) return 0;
  return x_type == CBMOE_E4M3 || type_ok(x_type) ? linear_ws(N, K, x_type == CBMOE_E4M3).total : 0;
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
  const LinearWs W = linear_ws(N, K, ready);
  if (!workspace || workspace_bytes < W.total || !aligned(workspace, 256)) return CBMOE_ERR_WORKSPACE;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  g.part = reinterpret_cast<float*>(ws);
  g.arrived = reinterpret_cast<int*>(ws + W.arrived);
  if (ready) {
    CBMOE_CUDA_TRY(cudaMemsetAsync(g.arrived, 0, (size_t)fp8_arrived() * 4, stream));
    g.xq = x;
    g.ldx = ldx;
    g.xs = xs;
    g.ldxs = blocks_of(K);
  } else {
    float* sc = reinterpret_cast<float*>(ws + W.xs);
    g.ldxs = fp8_scale_stride(K);
    g.ldx = (long long)blocks_of(K) * kFp8Group;
    const int rc = launch_fp8_quantize(x, x_type, N, K, ldx, ws + W.xq, g.ldx, sc, g.ldxs, nullptr, 1, N, g.arrived,
                                       fp8_arrived(), stream);
    if (rc) return rc;
    g.xq = ws + W.xq;
    g.xs = sc;
  }
  return launch_fp8_gemm(g, W.mt, stream);
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
  int* arrived = reinterpret_cast<int*>(ws + W.arrived);
  Fp8Gemm g{};
  g.E = ex->E;
  g.rows = ex->I;
  g.K = ex->H;
  g.ldx = (long long)blocks_of(ex->H) * kFp8Group;
  g.x_rows = W.Rp;
  g.ldxs = fp8_scale_stride(ex->H);
  g.xq = ws + W.xq;
  g.xs = reinterpret_cast<const float*>(ws + W.xs);
  rc = launch_fp8_quantize(x, CBMOE_BF16, N, ex->H, ex->H, ws + W.xq, g.ldx, reinterpret_cast<float*>(ws + W.xs), g.ldxs,
                           row_slot, k, W.Rp, arrived, 2 * fp8_arrived(), stream);
  if (rc) return rc;
  g.part = reinterpret_cast<float*>(ws + W.part);
  g.arrived = arrived;
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
  d.ldxs = fp8_scale_stride(ex->I);
  d.w0 = ex->down;
  d.w1 = nullptr;
  d.ldw = ex->ld_down;
  d.s0 = ex->down_s;
  d.s1 = nullptr;
  d.arrived = arrived + fp8_arrived();
  d.hq = nullptr;
  d.hs = nullptr;
  d.out = ws + W.y;
  d.out_type = y_type;
  rc = launch_fp8_gemm(d, W.mt, stream);
  if (rc) return rc;
  return cbmoe_unpermute(ws + W.y, y_type, W.Rp, ex->H, row_slot, w, N, k, y, stream);
}
