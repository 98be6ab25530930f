// Products in 8-bit floating point (e4m3): fp8_linear and the routed experts on such tables.
//
//   y[n, r] = sum_b sx[n, b] * sw[r / 128, b] * sum_{c in block b} xq[n, c] * wq[r, c]
//
// fp8_gemm_kernel, one CTA per SM, 12 warps:
//   warp 0      TMA producer: per 128-column block the tile's MT x 128 B of tokens and 2 x 128 x 128 B of weights (128-byte
//               swizzle), into a ring of stages
//   warp 1      TMEM owner and MMA issuer (one elected lane): 4 tcgen05.mma kind::f8f6f4 (M 128 x N 256 x K 32) per block
//               into one of two 256-column accumulators (tiles of 128 or 64 weight rows: 2 or 4 blocks side by side)
//   warps 4-11  promotion and epilogue: a block's 128 x 256 partial sums leave TMEM while the tensor core works on the next
//               block; acc += partial * (sx * sw) in fp32 registers (32 rows x 128 columns per warp; up to 32 tokens a pass
//               lie four times in the M side and a warp has 32 rows x a quarter of that). Tokens are the M side,
//               so a thread owns one token row: both scales are scalars for its columns. These warps take the registers
//               that the first warpgroup gives up (128 accumulators and a 16-column load a thread).
// The block's partial sum is exact enough to be added as it is: e4m3 products are exact in fp32 and the tensor core sums
// them in fp32 (measured: 1e-8 relative over K = 128).
// With many rows (MT = 256) two CTAs of a cluster work as a pair (cta_group::2, M = 256): each brings 128 tokens and half
// of the weight tile, 32 KB of loads a block where a CTA alone takes 48. What bounds it (one B200, 4096 x 12288 -> 9472):
// 1.88-1.92 PFLOP/s; a loop of its own that only loads and multiplies takes 380 us of the 500 because the clock falls to
// 1.06 GHz under the power cap, reading TMEM adds 45 us, the fp32 multiply-adds 45 us; the rest are the tiles' ends.
// With two matrices (gate, up: 128 columns each) the epilogue forms swiglu_clamped(gate, up), takes each row's maximum
// over its 128 columns and stores e4m3 codes and the scale: the down product's input, never in 16 bits.
// Work: whole waves of output tiles, one tile per CTA (pair). Tiles left over are cut along K into equal ranges of blocks
// where that pays (Fp8Sched): always for pairs, which wait for arithmetic; else only where there are fewer tiles than half
// of the SMs. A tile's ranges leave fp32 partial sums in the workspace; the last to arrive adds them in range order (the
// same bits on every call) and runs the epilogue. Few tokens take narrower tiles, so that enough SMs stream weights.
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
                                                           const int* __restrict__ row_slot, int k, int R, int repeat,
                                                           int* __restrict__ zero, int n_zero) {
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
    const int copies = row_slot != nullptr ? k : repeat;
    for (int j = 0; j < copies; ++j) {
      const int r = row_slot != nullptr ? row_slot[(size_t)n * k + j] : n + 32 * j;
      if (r < 0 || r >= R) continue;
      uint8_t* dst = q + (size_t)r * ldq + c0;
      if (wide && c0 + 8 <= ldq) {
        *reinterpret_cast<uint2*>(dst) = o;
      } else {
        for (int i = 0; i < 8 && c0 + i < K; ++i) dst[i] = (uint8_t)((i < 4 ? o.x : o.y) >> (8 * (i & 3)));
      }
      if (l == 0 && (row_slot != nullptr || j == 0)) s[(size_t)r * lds + kb] = sc;
    }
  }
}

// Scales that come with codes [N][KB] -> rows padded to whole 16-byte groups; clears the product's counters on the way.
// Where q is given, also the codes [N][K], N <= 32, four times into q (rows n + 32 j of KB * 128 bytes).
__global__ void __launch_bounds__(256) fp8_scales_kernel(const float* __restrict__ xs, int N, int KB, int ld,
                                                         float* __restrict__ out, const uint8_t* __restrict__ x, int K,
                                                         long long ldx, uint8_t* __restrict__ q, int* __restrict__ zero,
                                                         int n_zero) {
  griddep_wait();
  griddep_launch();
  const long long total = (long long)N * ld, at = blockIdx.x * 256LL + threadIdx.x, step = gridDim.x * 256LL;
  for (long long i = at; i < n_zero; i += step) zero[i] = 0;
  for (long long i = at; i < total; i += step) {
    const long long n = i / ld;
    const int kb = (int)(i - n * ld);
    out[i] = kb < KB ? xs[n * KB + kb] : 0.f;
  }
  if (q == nullptr) return;
  const int units = (K + 15) / 16;
  for (long long i = at; i < (long long)N * units; i += step) {
    const int n = (int)(i / units), c = (int)(i - (long long)n * units) * 16;
    const uint8_t* src = x + n * ldx + c;
    union {
      uint4 v;
      uint8_t b[16];
    } u;
    if (c + 16 <= K) {
      u.v = *reinterpret_cast<const uint4*>(src);
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) u.b[e] = c + e < K ? src[e] : 0;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4*>(q + (size_t)(n + 32 * j) * KB * kFp8Group + c) = u.v;
  }
}

// --------------------------------------------------------------------------------------------------- product
constexpr int kFp8Threads = 12 * 32;
constexpr int kW0 = 4;                                   // first promotion warp
constexpr int kRegsIdle = 40, kRegsWork = 232;           // 128 * 40 + 256 * 232 = 384 * 168, the launch's registers

// MT tokens and TN weight rows per tile (two matrices: TN / 2 of each).
template <int MT, int TN>
struct Fp8Cfg {
  static constexpr bool kPair = MT == 256;               // two CTAs, 128 tokens each
  static constexpr int kRows = kPair ? 128 : MT;         // tokens of a CTA's tile
  // 32 tokens lie four times in the 128 rows of the M side: each TMEM lane quadrant holds all of them and its warps take a
  // quarter of the columns. (Once, all columns would be read and summed by the two warps of one scheduler: the layer of 160
  // experts at 8 tokens then took 312 us, not 224.) Dense rows lie four times in memory, one load a block; a pass of an
  // expert loads its rows four times.
  static constexpr int kCopies = MT == 32 ? 4 : 1;
  static constexpr int kATile = kCopies * kRows * 128;
  static constexpr int kBTile = (kPair ? TN / 2 : TN) * 128;
  // Column blocks per stage and per accumulator (256 columns in all): a hand-over costs some 500 clocks of the issuer and
  // of the promotion warps whatever its size, so narrow tiles take several blocks at once.
  static constexpr int kU = 256 / TN;
  static constexpr int kStage = kU * (kATile + kBTile);
  static constexpr int kRest = 1024 + 2048 + 32 + 512;
  static constexpr int kNStage = (227 * 1024 - kRest) / kStage < 16 ? (227 * 1024 - kRest) / kStage : 16;
  static constexpr int kMaxOff = kNStage * kStage;       // row maxima [2][4 quadrants][2 halves][32] f32
  static constexpr int kFlagOff = kMaxOff + 2048;        // [2][4] int
  static constexpr int kBarOff = kFlagOff + 32;
  static constexpr int kSmem = 1024 + kBarOff + 512;
  static_assert((2 * kNStage + 9) * 8 <= 512, "barriers");
  static_assert(kSmem <= 227 * 1024, "shared memory budget");
  // The tensor core reads 128 rows of the M side whatever MT: past a block's tokens that is still its stage.
  static_assert((kU - 1) * kATile + 128 * 128 <= kStage, "M side inside the stage");
};

struct Fp8Params {
  Fp8Gemm g;
  int KB, RB, NT;          // column blocks, 128-row blocks per matrix, output tiles per pass
  int hs_ld;               // row stride of hs
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

// A worker's (a CTA's, or a pair's) share of the tiles, in segments (tile, units [kb0, kb1) of kU column blocks).
struct Fp8Seg {
  int item, kb0, kb1;
};
struct Fp8Sched {
  int waves, first, KB, chunk, u, u1, i, worker, G;

  // Worker `w` of `g` (a CTA, or a pair). Pairs cut whatever is left over: with many rows the SMs' arithmetic is what
  // counts. Alone, a CTA with few rows waits for memory, which half of the SMs keep busy: tiles are cut only where there
  // are fewer than that. Ranges below 4 (8) blocks would spend more on joining than on their sums.
  __device__ __forceinline__ Fp8Sched(int n_items, int kb, int w, int g, bool pair) : KB(kb), i(0), worker(w), G(g) {
    const int rem = n_items % G;
    waves = n_items / G;
    first = waves * G;
    chunk = pair ? 4 : (waves == 0 && 2 * rem <= G ? 8 : KB);
    chunk = max((rem * KB + G - 1) / G, min(KB, chunk));
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

// A thread's W sums to the columns [col0, col0 + W) of its row, as far as the matrix goes: whole 32-byte sectors where
// rows allow them (a lane per row, so narrower stores would leave the sectors in pieces).
template <int W, typename OUT, int N>
__device__ __forceinline__ void store_row(void* out, size_t row, int rows, int col0, const float (&acc)[N]) {
  const int end = min(rows - col0, W);
  OUT* dst = static_cast<OUT*>(out) + row * rows + col0;
  constexpr int kB = W * (int)sizeof(OUT) < 32 ? 16 : 32, kU = kB / (int)sizeof(OUT);
  if (rows % kU == 0 && (reinterpret_cast<uintptr_t>(out) & (kB - 1)) == 0) {
#pragma unroll
    for (int u = 0; u < W / kU; ++u) {
      if (u * kU < end) {
        union {
          uint32_t w[kB / 4];
          OUT o[kU];
        } b;
#pragma unroll
        for (int i = 0; i < kU; ++i) b.o[i] = out_of<OUT>(acc[u * kU + i]);
        if constexpr (kB == 32) store32(dst + u * kU, b.w);
        else *reinterpret_cast<uint4*>(dst + u * kU) = make_uint4(b.w[0], b.w[1], b.w[2], b.w[3]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (i < end) dst[i] = out_of<OUT>(acc[i]);
  }
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
  return mbar_wait_brief(bar, n++ & 1);
}

template <int MT, int TN, bool SWIGLU>
__global__ void __launch_bounds__(kFp8Threads, 1) fp8_gemm_kernel(const Fp8Params p,
                                                                  const __grid_constant__ CUtensorMap map_x,
                                                                  const __grid_constant__ CUtensorMap map_w0,
                                                                  const __grid_constant__ CUtensorMap map_w1) {
  using C = Fp8Cfg<MT, TN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kBarOff);   // [kNStage]
  uint64_t* empty = full + C::kNStage;      // [kNStage]
  uint64_t* d_full = empty + C::kNStage;    // [2]
  uint64_t* d_empty = d_full + 2;           // [2]
  uint64_t* meet = d_empty + 2;             // [4]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(meet + 4);
  float* row_max = reinterpret_cast<float*>(smem + C::kMaxOff);
  volatile int* flag = reinterpret_cast<volatile int*>(smem + C::kFlagOff);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kNStage; ++i) {
      mbar_init(&full[i], C::kPair && cluster_rank() == 0 ? 2 : 1);   // rank 0 of a pair: the other CTA's loads too
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&d_full[i], 1);
      mbar_init(&d_empty[i], C::kPair ? 16 : 8);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&meet[i], C::kCopies > 1 ? 8 : 2);
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
  const int KBU = (p.KB + C::kU - 1) / C::kU;               // units of a whole sum
  auto schedule = [&]() { return Fp8Sched(fp8_items<MT>(p), KBU, blockIdx.x / group, gridDim.x / group, C::kPair); };

  if (warp < kW0) {
    regs_give_up<kRegsIdle>();
    // Whole warps walk these loops and one elected lane issues: addresses and descriptors stay in uniform registers, which
    // halves the instructions of an issue (measured beside the promotion warps: 870 -> 760 clocks a block).
    int st = 0;
    uint32_t ph = 0;
    if (warp == 0) {
      auto weights = [&](const Fp8Item& it, int u, int st) {
        const int wrow = it.e * p.g.rows + it.nt * (SWIGLU ? TN / 2 : TN);
        uint8_t* b = smem + st * C::kStage + C::kU * C::kATile;
#pragma unroll
        for (int j = 0; j < C::kU; ++j) {
          const int x = (u * C::kU + j) * kFp8Group;        // past K: zeros
          if (!C::kPair || rank == 0) tma_load_2d(b + j * C::kBTile, &map_w0, x, wrow, &full[st]);
          if (!C::kPair || rank == 1)
            tma_load_2d(b + j * C::kBTile + (C::kPair ? 0 : TN / 2 * 128), SWIGLU ? &map_w1 : &map_w0, x,
                        SWIGLU ? wrow : wrow + TN / 2, &full[st]);
        }
      };
      Fp8Sched sched = schedule();
      Fp8Seg sg, sn;
      bool have = sched.next(sg);
      Fp8Item it{};
      if (have) it = fp8_item<MT>(p, sg.item);
      while (have) {
        const bool have_n = sched.next(sn);
        Fp8Item itn{};
        if (have_n) itn = fp8_item<MT>(p, sn.item);         // under way while this segment's loads are issued
        const int xrow = it.row0 + 128 * rank;
#pragma unroll 1
        for (int u = sg.kb0; u < sg.kb1; ++u) {
          if (!mbar_wait_brief(&empty[st], ph ^ 1)) goto late;
          if (elect_one()) {
            mbar_arrive_expect_tx(&full[st], C::kStage);
            weights(it, u, st);
#pragma unroll
            for (int j = 0; j < C::kU; ++j)
              for (int i = 0; i < (p.g.repeated ? 1 : C::kCopies); ++i)
                tma_load_2d(smem + st * C::kStage + j * C::kATile + i * C::kRows * 128, &map_x, (u * C::kU + j) * kFp8Group,
                            xrow, &full[st]);
          }
          __syncwarp();
          if (++st == C::kNStage) {
            st = 0;
            ph ^= 1;
          }
        }
        sg = sn;
        it = itn;
        have = have_n;
      }
    } else if (warp == 1 && rank == 1) {
      // The pair's MMAs are issued by rank 0: tell it which of this CTA's stages are full.
      Fp8Sched sched = schedule();
      Fp8Seg sg;
      while (sched.next(sg)) {
#pragma unroll 1
        for (int kb = sg.kb0; kb < sg.kb1; ++kb) {
          if (!mbar_wait_brief(&full[st], ph)) goto late;
          if (elect_one()) mbar_arrive_remote(&full[st], 0);
          __syncwarp();
          if (++st == C::kNStage) {
            st = 0;
            ph ^= 1;
          }
        }
      }
    } else if (warp == 1) {
      Fp8Sched sched = schedule();
      Fp8Seg sg;
      constexpr uint32_t idesc = idesc_e4m3(C::kPair ? 256 : 128, TN);
      const uint64_t desc0 = sw128_desc(smem_addr(smem));
      uint32_t buf = 0, dph = 1;
      while (sched.next(sg)) {
#pragma unroll 1
        for (int u = sg.kb0; u < sg.kb1; ++u) {
          if (!mbar_wait_brief(&d_empty[buf], dph) || !mbar_wait_brief(&full[st], ph)) goto late;
          tc_fence_after();
          // Rows kRows.. of the M side are whatever follows in the stage: their sums are never read.
          const uint64_t a0 = desc0 + (uint32_t)(st * (C::kStage >> 4)), b0 = a0 + (C::kU * C::kATile >> 4);
          const uint32_t d = tmem + buf * 256;
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < 4 * C::kU; ++kk) {
              const uint64_t ad = a0 + (kk / 4) * (C::kATile >> 4) + 2 * (kk % 4);
              const uint64_t bd = b0 + (kk / 4) * (C::kBTile >> 4) + 2 * (kk % 4);
              if constexpr (C::kPair) umma_fp8_pair(d, ad, bd, idesc, kk % 4 != 0);
              else umma_fp8(d + (kk / 4) * TN, ad, bd, idesc, kk % 4 != 0);
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
    Fp8Sched sched = schedule();
    const int q = warp & 3;                  // TMEM lane quadrant this warp may read
    const int half = (warp - kW0) >> 2;
    const int qq = C::kCopies > 1 ? q : 0;   // quarter of the columns
    const int m = C::kCopies > 1 ? lane : 32 * q + lane;   // this thread's row of the CTA's tile
    constexpr int AC = TN / 2 / C::kCopies;  // columns of a warp (SwiGLU: half of gate, half of up)
    constexpr int LW = AC < 16 ? AC : 16;    // columns of a load
    uint64_t* const meet_bar = &meet[C::kCopies > 1 ? 0 : q];
    uint32_t n = 0, met = 0;
    auto d_read = [&](int buf) {             // to the CTA that issues the MMAs
      __syncwarp();
      if constexpr (C::kPair) mbar_arrive_remote(&d_empty[buf], 0, lane == 0);
      else mbar_arrive_if(&d_empty[buf], lane == 0);
    };
    auto item_of = [&](const Fp8Seg& s) {
      Fp8Item it = fp8_item<MT>(p, s.item);
      it.row0 += 128 * rank;                 // this CTA's rows of the tile
      it.cnt -= 128 * rank;
      return it;
    };
    // A tile's place in the plan is fetched while the tile before it is summed.
    Fp8Seg sg{}, sn{};
    Fp8Item it{}, itn{};
    bool have = sched.next(sg);
    if (have) it = item_of(sg);
    while (have) {
      const bool live = m - lane < it.cnt, mine = m < it.cnt;
      const size_t xrow = mine ? (size_t)it.row0 + m : 0;
      const bool have_n = sched.next(sn);
      if (have_n) itn = item_of(sn);         // under way while this tile is summed
      float acc[AC];
#pragma unroll
      for (int i = 0; i < AC; ++i) acc[i] = 0.f;
      // This row's scales, four blocks at a time (rows are padded to whole groups: fp8_scale_stride), and the weights', a
      // block per lane: of this half's 128-row block, or of gate and up. Fetched at least four blocks ahead of their use: a
      // load's latency under the tiles' traffic is longer than a block.
      const float* sx = p.g.xs + xrow * p.g.ldxs;
      const int blk = SWIGLU ? it.nt : min((it.nt * TN + half * (TN / 2) + AC * qq) / 128, p.RB - 1), kb0 = sg.kb0 * C::kU;
      const float* sa = p.g.s0 + ((size_t)it.e * p.RB + blk) * p.KB;
      const float* sb = SWIGLU ? p.g.s1 + ((size_t)it.e * p.RB + blk) * p.KB : sa;
      auto row_scales = [&](int kb) { return *reinterpret_cast<const float4*>(sx + min(kb, (p.KB - 1) & ~3)); };
      float4 xn = row_scales(kb0 & ~3), xc = xn;
      float wa = 0.f, wb = 0.f;
      float wa_n = kb0 + lane < p.KB ? sa[kb0 + lane] : 0.f, wb_n = SWIGLU && kb0 + lane < p.KB ? sb[kb0 + lane] : 0.f;
      // Not unrolled: 128 multiply-adds a turn fill the instruction cache that the MMA issuer shares.
#pragma unroll 1
      for (int u = sg.kb0; u < sg.kb1; ++u, ++n) {
        const int kb = u * C::kU, i32 = (kb - kb0) % 32, buf = n & 1;
        if (kb % 4 == 0 || kb == kb0) {
          xc = xn;
          xn = row_scales((kb & ~3) + 4);
          if (kb % 4 >= 2) xc.x = xc.z, xc.y = xc.w;         // a range that begins inside a group
          if (kb % 2 != 0) xc.x = xc.y, xc.y = xc.z, xc.z = xc.w;
        }
        if (i32 == 0) {
          wa = wa_n, wb = wb_n;
          const int k = kb + 32 + lane;
          if (k < p.KB) {
            wa_n = sa[k];
            if constexpr (SWIGLU) wb_n = sb[k];
          }
        }
        float fa[C::kU], fb = 0.f;
#pragma unroll
        for (int j = 0; j < C::kU; ++j) {
          fa[j] = (j == 0 ? xc.x : (j == 1 ? xc.y : (j == 2 ? xc.z : xc.w))) * __shfl_sync(0xffffffffu, wa, i32 + j);
          if (C::kU > 1 && kb + j >= p.KB) fa[j] = 0.f;      // past K the products are zero, the scales are not
        }
        if constexpr (SWIGLU) fb = xc.x * __shfl_sync(0xffffffffu, wb, i32);
        if constexpr (C::kU == 1) xc.x = xc.y, xc.y = xc.z, xc.z = xc.w;
        if constexpr (C::kU == 2) xc.x = xc.z, xc.y = xc.w;
        if (!mbar_wait_brief(&d_full[buf], (n >> 1) & 1)) goto late;
        tc_fence_after();
        if (live) {
          const uint32_t t0 = tmem + buf * 256 + ((uint32_t)(32 * q) << 16);
          // 16 columns at a time: the two warps of a scheduler take turns between a load and its multiply-adds, and
          // 128 + 16 registers a thread leave nothing to spill (one spilled register in this loop costs more than any
          // longer load gains).
          constexpr int kLoads = 128 / C::kCopies / LW;
#pragma unroll
          for (int c = 0; c < kLoads; ++c) {    // SwiGLU: gate, then up; else kU blocks
            float v[LW];
            const int j = SWIGLU ? 0 : LW * c / AC, at = LW * c % AC;
            const int col = SWIGLU ? (at < AC / 2 ? 0 : 128) + 64 * half + AC / 2 * qq + at % (AC / 2)
                                   : j * TN + TN / 2 * half + AC * qq + at;
            if constexpr (LW == 16) tmem_ld16(t0 + col, v);
            else tmem_ld8(t0 + col, v);
            if (c == kLoads - 1) {              // all of this unit is in registers
              tc_fence_before();
              d_read(buf);
            }
            const float f = SWIGLU && at >= AC / 2 ? fb : fa[j];
#pragma unroll
            for (int i = 0; i < LW; ++i) acc[at + i] = fmaf(v[i], f, acc[at + i]);
          }
        } else {
          d_read(buf);
        }
      }
      bool whole = true;
      if (sg.kb1 - sg.kb0 < KBU) {
        // ---------------- a range of the sum: partial sums [slot][rank][half][quarter][4-column group][row], 512
        // contiguous bytes a store
        int c0, c1;
        sched.sharers(sg.item, c0, c1);
        auto part = [&](int w) {
          const size_t at = (((size_t)sched.slot(w, sg.item) * group + rank) * 2 + half) * C::kCopies + qq;
          return reinterpret_cast<float4*>(p.g.part) + at * (AC / 4) * C::kRows + m;
        };
        if (mine) {
          float4* dst = part(sched.worker);
#pragma unroll
          for (int i = 0; i < AC / 4; ++i)
            __stcg(dst + i * C::kRows, make_float4(acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3]));
        }
        __threadfence();
        int* arrived = p.g.arrived + ((sg.item - sched.first) * group + rank) * 8;
        if constexpr (SWIGLU) {                            // one decision for all of a row
          if (!pair_meet(meet_bar, met)) goto late;        // both are written
          const int at = (met & 1) * 4 + (C::kCopies > 1 ? 0 : q);
          if (half == 0 && lane == 0 && (C::kCopies == 1 || q == 0)) flag[at] = atomicAdd(&arrived[q], 1) == c1 - c0;
          if (!pair_meet(meet_bar, met)) goto late;
          whole = flag[at] != 0;
        } else {
          int old = 0;
          __syncwarp();
          if (lane == 0) old = atomicAdd(&arrived[4 * half + q], 1);
          whole = __shfl_sync(0xffffffffu, old, 0) == c1 - c0;
        }
        if (whole) __threadfence();
        // The last worker to arrive adds the tile's ranges in their order, 8 loads under way at once.
#pragma unroll
        for (int i = 0; i < AC; ++i) acc[i] = 0.f;
        if (whole && mine) {
          for (int w = c0; w <= c1; ++w) {
            const float4* src = part(w);
            constexpr int kStep = AC / 4 < 8 ? AC / 4 : 8;
#pragma unroll
            for (int i = 0; i < AC / 4; i += kStep) {
              float4 v[kStep];
#pragma unroll
              for (int j = 0; j < kStep; ++j) v[j] = __ldcg(src + (i + j) * C::kRows);
#pragma unroll
              for (int j = 0; j < kStep; ++j) {
                acc[4 * (i + j)] += v[j].x;
                acc[4 * (i + j) + 1] += v[j].y;
                acc[4 * (i + j) + 2] += v[j].z;
                acc[4 * (i + j) + 3] += v[j].w;
              }
            }
          }
        }
      }
      // ------------------------------------------------------------------- the whole sum: this thread's row, its columns
      const int rows = p.g.rows;
      if (whole) {
        if constexpr (SWIGLU) {
          static_assert(!SWIGLU || TN == 256, "a row's maximum over 128 columns is taken inside one tile");
          constexpr int GW = AC / 2;
          const int col0 = it.nt * 128 + 64 * half + GW * qq;
          float top = 0.f;
#pragma unroll
          for (int i = 0; i < GW; ++i) {
            acc[i] = col0 + i < rows ? swiglu_keep_nan(acc[i], acc[GW + i], p.g.limit) : 0.f;
            top = max_nan(top, fabsf(acc[i]));
          }
          if constexpr (C::kCopies > 1) {
            float* mx = row_max + (met & 1) * 256;
            mx[(half * 4 + q) * 32 + lane] = top;
            if (!pair_meet(meet_bar, met)) goto late;
#pragma unroll
            for (int i = 0; i < 8; ++i) top = max_nan(top, mx[i * 32 + lane]);
          } else {
            float* mx = row_max + ((met & 1) * 4 + q) * 64;
            mx[half * 32 + lane] = top;
            if (!pair_meet(meet_bar, met)) goto late;
            top = max_nan(top, mx[(half ^ 1) * 32 + lane]);
          }
          float inv;
          const float sc = fp8_group_scale(top, &inv);
          if (mine) {
            uint4* dst = reinterpret_cast<uint4*>(p.g.hq + xrow * ((size_t)p.RB * 128) + col0);
#pragma unroll
            for (int u = 0; u < GW / 16; ++u) {
              uint32_t w[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int c = 16 * u + 4 * i;
                w[i] = fp8_pack4(acc[c] * inv, acc[c + 1] * inv, acc[c + 2] * inv, acc[c + 3] * inv);
              }
              dst[u] = make_uint4(w[0], w[1], w[2], w[3]);
            }
            if (half == 0 && qq == 0) p.g.hs[xrow * p.hs_ld + it.nt] = sc;
          }
        } else if (mine) {
          const int col0 = it.nt * TN + half * (TN / 2) + AC * qq;
          if (p.g.out_type == CBMOE_BF16) store_row<AC, __nv_bfloat16>(p.g.out, xrow, rows, col0, acc);
          else if (p.g.out_type == CBMOE_F16) store_row<AC, __half>(p.g.out, xrow, rows, col0, acc);
          else store_row<AC, float>(p.g.out, xrow, rows, col0, acc);
        }
      }
      sg = sn;
      it = itn;
      have = have_n;
    }
  }
  if (false) {
  late:
    atomicOr(&g_device_errors, CBMOE_DEVERR_TIMEOUT);
  }
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

template <int MT, int TN, bool SWIGLU>
int launch_t(const Fp8Gemm& g, cudaStream_t stream) {
  using C = Fp8Cfg<MT, TN>;
  Fp8Params p;
  p.g = g;
  p.KB = (g.K + kFp8Group - 1) / kFp8Group;
  p.RB = (g.rows + 127) / 128;
  p.NT = SWIGLU ? p.RB : (g.rows + TN - 1) / TN;
  p.hs_ld = fp8_scale_stride(g.rows);
  CUtensorMap mx, m0, m1;
  int rc = make_fp8_map(&mx, g.xq, g.K, g.repeated ? 128 : g.x_rows, g.ldx, g.repeated ? 128 : C::kRows);
  if (!rc) rc = make_fp8_map(&m0, g.w0, g.K, (long long)g.E * g.rows, g.ldw, TN / 2);
  if (!rc) rc = make_fp8_map(&m1, SWIGLU ? g.w1 : g.w0, g.K, (long long)g.E * g.rows, g.ldw, TN / 2);
  if (rc) return rc;
  auto kern = fp8_gemm_kernel<MT, TN, SWIGLU>;
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

// Weight rows per tile with few tokens. Dense: by how many tiles that gives. Measured on one B200, quantiser included:
// 5120 -> 12288, 64 tokens: 48 tiles of 256 28.9 us, 96 of 128 19.1, 192 of 64 22.8; 77 x 5000 -> 1411: 6 of 256 27.3, 12 of
// 128 22.3, 23 of 64 18.7. Experts with up to 32 rows a pass load the tokens four times, so a block more per stage costs
// four more loads: 256 (54 experts: 227 us against 242 at 128).
template <int MT>
int launch_few(const Fp8Gemm& g, cudaStream_t s) {
  if (g.w1 != nullptr) return launch_t<MT, 256, true>(g, s);
  if (MT == 32 && g.pass_expert != nullptr) return launch_t<MT, 256, false>(g, s);
  const long long passes = g.pass_expert ? (g.x_rows < g.E ? g.x_rows : g.E) : (g.x_rows + MT - 1) / MT;
  if (passes * ((g.rows + 255) / 256) >= 2LL * num_sms()) return launch_t<MT, 256, false>(g, s);
  if (passes * ((g.rows + 127) / 128) >= num_sms() / 2) return launch_t<MT, 128, false>(g, s);
  return launch_t<MT, 64, false>(g, s);
}

bool aligned(const void* p, int n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
bool type_ok(int t) { return t == CBMOE_BF16 || t == CBMOE_F16 || t == CBMOE_F32; }
int elem_size(int t) { return t == CBMOE_F32 ? 4 : 2; }
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
  if (mt == 32) return launch_few<32>(g, s);
  if (mt == 64) return launch_few<64>(g, s);
  if (mt == 128) return launch_few<128>(g, s);
  if (g.w1 != nullptr) return launch_t<256, 256, true>(g, s);
  return launch_t<256, 256, false>(g, s);
}

int launch_fp8_quantize(const void* x, int type, int N, int K, long long ldx, uint8_t* q, long long ldq, float* s, int lds,
                        const int* row_slot, int k, int R, int repeat, int* zero, int n_zero, cudaStream_t stream) {
  const long long groups = (long long)N * blocks_of(K);
  long long blocks = (groups + 15) / 16, cap = (long long)num_sms() * 16;
  if (blocks > cap) blocks = cap;
  const int size = elem_size(type);
  const int vec = aligned(x, 16) && ldx * size % 16 == 0;
  prof_begin(kProfOther, stream);
  if (type == CBMOE_BF16)
    CBMOE_CUDA_TRY(launch_pdl(fp8_quantize_kernel<__nv_bfloat16>, dim3((int)blocks), dim3(256), 0, stream,
                              static_cast<const __nv_bfloat16*>(x), N, K, ldx, vec, q, ldq, s, lds, row_slot, k, R, repeat,
                              zero, n_zero));
  else if (type == CBMOE_F16)
    CBMOE_CUDA_TRY(launch_pdl(fp8_quantize_kernel<__half>, dim3((int)blocks), dim3(256), 0, stream,
                              static_cast<const __half*>(x), N, K, ldx, vec, q, ldq, s, lds, row_slot, k, R, repeat, zero,
                              n_zero));
  else
    CBMOE_CUDA_TRY(launch_pdl(fp8_quantize_kernel<float>, dim3((int)blocks), dim3(256), 0, stream,
                              static_cast<const float*>(x), N, K, ldx, vec, q, ldq, s, lds, row_slot, k, R, repeat, zero,
                              n_zero));
  prof_end(kProfOther, stream);
  CBMOE_CUDA_TRY(cudaGetLastError());
  return CBMOE_OK;
}

namespace {

// Workspace of a product: partial sums | counters | q [rows][blocks * 128] |
// scales [N][fp8_scale_stride].
struct LinearWs {
  size_t arrived, xq, xs, total;
  int mt;
};
LinearWs linear_ws(int N, int K, bool ready) {
  LinearWs w;
  w.mt = fp8_pass_tokens(N, 1);
  w.arrived = lyr::align_up(fp8_part_bytes(w.mt));
  w.xq = w.arrived + lyr::align_up((size_t)fp8_arrived() * 4);
  const int q_rows = w.mt == 32 ? 128 : (ready ? 0 : N);   // up to 32 tokens lie there four times
  w.xs = w.xq + lyr::align_up((size_t)q_rows * blocks_of(K) * kFp8Group);
  w.total = w.xs + lyr::align_up((size_t)N * fp8_scale_stride(K) * 4);
  return w;
}

// Workspace of the layer: plan | partial sums | counters (gate/up, down) | xq, xs (sorted rows) | hq, hs | slot outputs.
// The slots' outputs are fp32 whatever the type of y: the weighted sum is rounded once, and a slot may lie outside the
// range of fp16 where the sum does not. (160 experts x 4096 tokens, bf16 out: 1877 us a call; with slots in bf16, a second
// rounding, 1728: the combine moves 57 us more of bytes, the down product stores twice as much at its tiles' ends.)
struct ExpertsWs {
  size_t plan, part, arrived, xq, xs, hq, hs, y, total;
  int mt, Rp;
  lyr::PlanLayoutHost L;
};
ExpertsWs experts_ws(int E, int H, int I, int N, int k) {
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
  w.total = w.y + lyr::align_up((size_t)S * H * 4);
  return w;
}

bool fp8_table_ok(const void* q, const float* s, long long ld, long long rows, int K) {
  // (the row coordinates of a tile's end have to fit 32 bits)
  return q && s && aligned(q, 16) && aligned(s, 4) && ld >= K && ld % 16 == 0 && rows <= 0x7ffffe00LL;
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
  if (!x || !q || !s || !aligned(x, elem_size(type)) || !aligned(s, 4)) return CBMOE_ERR_INVALID;
  if (K > (1 << 30)) return CBMOE_ERR_UNSUPPORTED;                    // columns in 32 bits
  return launch_fp8_quantize(x, type, N, K, ldx, q, ldq, s, blocks_of(K), nullptr, 1, N, 1, nullptr, 0, stream);
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
  if (N > (1 << 30) || K > (1 << 24)) return CBMOE_ERR_UNSUPPORTED;   // counts of tiles and blocks in 32 bits
  if (!x || !y || ldx < K || !aligned(y, elem_size(y_type))) return CBMOE_ERR_INVALID;
  if (ready ? !xs || ldx % 16 || !aligned(x, 16) || !aligned(xs, 4) : !aligned(x, elem_size(x_type)))
    return CBMOE_ERR_INVALID;
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
    float* sc = reinterpret_cast<float*>(ws + W.xs);
    g.xq = x;
    g.ldx = ldx;
    g.xs = sc;
    g.ldxs = fp8_scale_stride(K);
    if (W.mt == 32) {
      g.xq = ws + W.xq;
      g.ldx = (long long)blocks_of(K) * kFp8Group;
      g.repeated = 1;
    }
    const long long blocks = ((long long)N * (W.mt == 32 ? K / 16 + g.ldxs : g.ldxs) + 255) / 256, cap = num_sms() * 8;
    prof_begin(kProfOther, stream);
    CBMOE_CUDA_TRY(launch_pdl(fp8_scales_kernel, dim3((int)(blocks < cap ? blocks : cap)), dim3(256), 0, stream, xs, N,
                              blocks_of(K), g.ldxs, sc, static_cast<const uint8_t*>(x), K, ldx,
                              W.mt == 32 ? ws + W.xq : static_cast<uint8_t*>(nullptr), g.arrived, fp8_arrived()));
    prof_end(kProfOther, stream);
    CBMOE_CUDA_TRY(cudaGetLastError());
  } else {
    float* sc = reinterpret_cast<float*>(ws + W.xs);
    g.ldxs = fp8_scale_stride(K);
    g.ldx = (long long)blocks_of(K) * kFp8Group;
    g.repeated = W.mt == 32;
    const int rc = launch_fp8_quantize(x, x_type, N, K, ldx, ws + W.xq, g.ldx, sc, g.ldxs, nullptr, 1,
                                       g.repeated ? 128 : N, g.repeated ? 4 : 1, g.arrived,
                                       fp8_arrived(), stream);
    if (rc) return rc;
    g.xq = ws + W.xq;
    g.xs = sc;
  }
  return launch_fp8_gemm(g, W.mt, stream);
}

extern "C" size_t cbmoe_fp8_experts_workspace_bytes(const cbmoe_fp8_experts* ex, int N, int k, int y_type) {
  if (!ex || ex->E <= 0 || ex->H <= 0 || ex->I <= 0 || N < 0 || k <= 0 || !type_ok(y_type)) return 0;
  return experts_ws(ex->E, ex->H, ex->I, N, k).total;
}

extern "C" int cbmoe_fp8_experts_apply(const cbmoe_fp8_experts* ex, const uint16_t* x, int N, const int32_t* idx,
                                       const float* w, int k, float limit, void* y, int y_type, void* workspace,
                                       size_t workspace_bytes, cudaStream_t stream) {
  if (!fp8_experts_ok(ex) || N < 0 || k <= 0 || k > 64 || !type_ok(y_type)) return CBMOE_ERR_INVALID;
  if (N == 0) return CBMOE_OK;
  if (!x || !idx || !w || !y) return CBMOE_ERR_INVALID;
  if (!aligned(x, 2) || !aligned(idx, 4) || !aligned(w, 4) || !aligned(y, elem_size(y_type))) return CBMOE_ERR_INVALID;
  if ((long long)N * k > (1 << 30)) return CBMOE_ERR_UNSUPPORTED;
  const ExpertsWs W = experts_ws(ex->E, ex->H, ex->I, N, k);
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
                           row_slot, k, W.Rp, 1, arrived, 2 * fp8_arrived(), stream);
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
  d.out_type = CBMOE_F32;
  rc = launch_fp8_gemm(d, W.mt, stream);
  if (rc) return rc;
  return launch_unpermute_f32(reinterpret_cast<const float*>(ws + W.y), W.Rp, ex->H, row_slot, w, N, k, y, y_type,
                              stream);
}
