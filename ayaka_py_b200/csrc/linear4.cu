// Products of 8-bit rows and 4-bit weights (microscale.cuh), both in blocks of 32 columns that share a power of two, on tcgen05
// with the scales in tensor memory (kind::mxf8f6f4): nothing is decoded in front of the tensor cores.
//
//   linear:  C[t, n] = act(sum_k a[t, k] W[n, k] + bias[n]) (+ residual[t, n])
//   gated:   rows in 8 bits of act(sum_k a[t, k] G[n, k]) * (sum_k a[t, k] U[n, k])
//
// Weights lie in column blocks of 128 (64 bytes of codes a row), their scales beside them as the tensor cores take them.  The
// copy engine spreads sixteen codes over sixteen bytes on their way into shared memory.
//
// Every wait is bounded; one that runs out records a code (101 ... 119) in an error word and the CTA winds down: whoever gave up, its copies
// in flight and its MMAs are waited for before it leaves.
#include <cuda.h>

#include <mutex>
#include <type_traits>

#include "microscale.cuh"
#include "tcgen05.cuh"

namespace {

constexpr int BLOCK_K = 128;                    // columns of a stage: 128 bytes a row in shared memory, 64 of a weight's row in memory
constexpr int TILE_N = 128;                     // features of a CTA
constexpr int W_BYTES = TILE_N * BLOCK_K;       // a weight tile in shared memory; half of it travels
constexpr int SCALE_BYTES = 512;                // the scales of 128 rows and four blocks
constexpr int QUADS = 4;                        // the rows' scales come for four column blocks at a time, into a ring of four such
constexpr int QUAD_BYTES = 4 * SCALE_BYTES;

struct Args {
  void* C;                       // linear: bfloat16 or float32 [T, N]; gated: codes [T, N]
  uint8_t* out_scales;           // gated
  const uint8_t* a_scales;
  const uint8_t* w_scales[2];
  const float* bias;
  const float* residual;
  int* error;
  long long a_scale_stride, out_scale_stride;
  int T, N, K;
  int n_blocks;                  // the weight's rows in whole 128
  int act, out_bf16;
};

// What has to be known to wind a CTA down where a warp has given up, in shared memory behind the barriers.
struct Ends {
  uint32_t tmem;                 // the address of tensor memory
  int issued;                    // stages whose operands are copied
  int gave_up;
  int quads, tiles;              // many rows: quads of scales that are copied, tiles whose last product is committed
};

// A wait for other warps of the CTA, bounded.  (That it gives up at once, to test what comes after, is a constant of a build of its own: a
// flag in the arguments cost 2 to 9 % of a launch, a vote of a warp's lanes up to 6.  Lanes poll side by side, and give up so.)
__device__ __forceinline__ bool hand_over(uint32_t bar, uint32_t parity, int* error, int code) {
#ifdef AYK_IMPATIENT
  if (mbar_test(bar, parity)) return true;
  atomicExch(error, code);
  return false;
#else
  return mbar_wait_short(bar, parity, error, code);
#endif
}
__device__ __forceinline__ bool hand_over_warp(uint32_t bar, uint32_t parity, int* error, int code) {
#ifdef AYK_IMPATIENT
  return __all_sync(0xffffffffu, hand_over(bar, parity, error, code));
#else
  return hand_over(bar, parity, error, code);
#endif
}

// The scales of row t for column block kb, the first block in the low byte; zeros (2^-127) beyond the matrix.
__device__ __forceinline__ uint32_t row_scales(const Args& a, int t, int kb) {
  const int blocks = a.K / MX_BLOCK - 4 * kb;
  if (t >= a.T || blocks <= 0) return 0u;
  const uint8_t* at = a.a_scales + (size_t)t * a.a_scale_stride + 4 * kb;
  if (blocks >= 4) return *reinterpret_cast<const uint32_t*>(at);
  uint32_t word = at[0];
  if (blocks > 1) word |= (uint32_t)at[1] << 8;
  if (blocks > 2) word |= (uint32_t)at[2] << 16;
  return word;
}

// The activations of the tensor-core epilogues, of which the squared ReLU's maximum would take a NaN to 0: here a row that is no number
// stays so under every one (max.NaN is one instruction as well).
template <int ACT>
__device__ __forceinline__ float activated(float x, int act) {
  if constexpr (ACT == AYK_ACT_RELU2) {
    float r;
    asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(x));
    return r * r;
  } else {
    return apply_activation_tc<ACT>(x, act);
  }
}

// One feature n (a lane's) of CNT rows from t on.  Linear: bias, activation, residual (every load before the first store: the
// residual may be C), rounding.  Gated: the warp's 32 features are a block, whose largest magnitude makes the scale.
// `inside`: n is a feature (of a gated product all 32 or none).
template <bool GATED, int ACT, int CNT>
__device__ __forceinline__ void finish_rows(const Args& a, int t, int n, bool inside, const float (&v)[CNT], const float (&u)[CNT]) {
  if constexpr (GATED) {
#pragma unroll
    for (int j = 0; j < CNT; ++j) {
      const float y = activated<ACT>(v[j], a.act) * u[j];
      const uint32_t code = mx_scale_code(__reduce_max_sync(0xffffffffu, magnitude_bits(y)));
      if (inside && t + j < a.T) {
        ((uint8_t*)a.C)[(size_t)(t + j) * a.N + n] = (uint8_t)e4m3_pair(y * mx_inverse(code), 0.f);
        if ((threadIdx.x & 31) == 0) a.out_scales[(size_t)(t + j) * a.out_scale_stride + n / MX_BLOCK] = (uint8_t)code;
      }
    }
  } else if (inside) {
    const float b = a.bias ? a.bias[n] : 0.f;
    float r[CNT];
#pragma unroll
    for (int j = 0; j < CNT; ++j) r[j] = a.residual && t + j < a.T ? a.residual[(size_t)(t + j) * a.N + n] : 0.f;
#pragma unroll
    for (int j = 0; j < CNT; ++j) {
      if (t + j < a.T) {
        const float y = activated<ACT>(v[j] + b, a.act) + r[j];
        const size_t at = (size_t)(t + j) * a.N + n;
        if (a.out_bf16) ((__nv_bfloat16*)a.C)[at] = __float2bfloat16_rn(y);
        else ((float*)a.C)[at] = y;
      }
    }
  }
}

// The activation as a constant of the code that `run` is compiled to; the ones that few products use share one copy.
template <typename Run>
__device__ __forceinline__ void with_activation(int act, Run run) {
  if (act == AYK_ACT_NONE) run(std::integral_constant<int, AYK_ACT_NONE>());
  else if (act == AYK_ACT_SILU) run(std::integral_constant<int, AYK_ACT_SILU>());
  else if (act == AYK_ACT_GELU_TANH) run(std::integral_constant<int, AYK_ACT_GELU_TANH>());
  else if (act == AYK_ACT_RELU2) run(std::integral_constant<int, AYK_ACT_RELU2>());
  else run(std::integral_constant<int, -1>());
}

// ---------------------------------------------------------------- few rows --
// A CTA takes 128 features as the MMA's M side and BT rows as its N side, so that a handful of rows streams every weight byte
// once; the CTAs of a cluster along z share the tile, each with a part of its column blocks, and exchange their 32-bit sums
// through shared memory.  Bound by the weight's bytes where there are enough, else by the way of one launch: 8 x 16384 x 4096
// (36 MB) 8.4 us with the weight in L2, 9.6 with weights from memory in turn (3.7 TB/s; each further 36 MB 6 us, 6.1 TB/s); 1 x 1600 x
// 4800 4.1 us, 128 x 128 alone 1.9.  The MMAs (128 x 16 x 32, 40 clocks: 128 rows' 32 bytes leave shared memory at 128 a clock) would
// take weights at twice the memory's rate.  Tried, 8 x 16384 x 4096 from memory: three or four stages a CTA 10.9, 10.3; one CTA to a
// multiprocessor, so that the next launch's fits beside it, 11.2.
//
// Warp 0: copies; warp 1: MMA issue, tensor memory; warps 2 ... 5 (64 rows: 2 ... 9): the rows' scales while the main loop runs,
// then the epilogue.
template <int BT, bool GATED>
struct Few {
  static constexpr int MATRICES = GATED ? 2 : 1;
  static constexpr int ROW_BYTES = BT * BLOCK_K;
  static constexpr int TILE_BYTES = MATRICES * W_BYTES + ROW_BYTES;
  static constexpr int STAGES = GATED ? (BT <= 16 ? 5 : BT <= 32 ? 4 : 3) : (BT <= 16 ? 5 : BT <= 32 ? 4 : 6);
  static constexpr int PLACES = GATED || BT > 32 ? 1 : 2;                    // CTAs that a multiprocessor's shared memory holds
  static constexpr int EPILOGUE = BT <= 32 ? 128 : 256;                      // threads
  static constexpr int THREADS = 64 + EPILOGUE;
  static constexpr int TX = MATRICES * (W_BYTES / 2 + SCALE_BYTES) + ROW_BYTES;
  static constexpr int ACCUMULATORS = MATRICES * BT;
  static constexpr int SCALE_COLUMNS = 4 * (MATRICES + 1);                   // of a stage
  static constexpr int USED = ACCUMULATORS + STAGES * SCALE_COLUMNS;
  static constexpr int TMEM = USED <= 64 ? 64 : USED <= 128 ? 128 : USED <= 256 ? 256 : 512;
  // shared memory, from a 1024-byte boundary on
  static constexpr int AT_W_SCALES = STAGES * TILE_BYTES;
  static constexpr int AT_ROW_SCALES = AT_W_SCALES + STAGES * MATRICES * SCALE_BYTES;
  static constexpr int AT_BARS = AT_ROW_SCALES + QUADS * QUAD_BYTES;
  static constexpr int AT_SUMS = AT_BARS + 256;
  // features of a tile that one CTA of the cluster finishes; of a gated product whole blocks of 32, so that some CTAs may finish none
  __host__ __device__ static constexpr int share(int splits) { return GATED ? (splits >= 4 ? 32 : splits >= 2 ? 64 : 128) : (TILE_N + splits - 1) / splits; }
  static constexpr int sums_bytes(int splits) { return MATRICES * splits * share(splits) * BT * 4; }
  static constexpr int smem(int splits) { return 1024 + AT_SUMS + sums_bytes(splits); }
};

template <int BT, bool GATED>
__global__ void __launch_bounds__(Few<BT, GATED>::THREADS, 1)
linear4_few_kernel(const __grid_constant__ CUtensorMap map_w0, const __grid_constant__ CUtensorMap map_w1,
                   const __grid_constant__ CUtensorMap map_a, const Args args) {
  using L = Few<BT, GATED>;
  constexpr int STAGES = L::STAGES, MATRICES = L::MATRICES;
  constexpr uint32_t IDESC = make_idesc_mx(TILE_N, BT, MX_E2M1, MX_E4M3);
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw), tiles = (raw + 1023u) & ~1023u;
  const uint32_t w_scales = tiles + L::AT_W_SCALES, row_ring = tiles + L::AT_ROW_SCALES, bars = tiles + L::AT_BARS, sums = tiles + L::AT_SUMS;
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (STAGES + s); };
  auto scales_full = [&](int q) { return bars + 8u * (2 * STAGES + q); };
  auto scales_empty = [&](int q) { return bars + 8u * (2 * STAGES + QUADS + q); };
  const uint32_t done_bar = bars + 8u * (2 * STAGES + 2 * QUADS), tmem_slot = done_bar + 8u;
  volatile Ends* ends = (volatile Ends*)(smem_raw + (tmem_slot - raw));

  const int warp = warp_number(), lane = threadIdx.x & 31;
  const int n0 = blockIdx.x * TILE_N, t0 = blockIdx.y * BT;
  const int splits = gridDim.z, z = blockIdx.z;
  const int total = (args.K + BLOCK_K - 1) / BLOCK_K, base = total / splits, extra = total % splits;
  const int kb0 = z * base + min(z, extra), num_kb = base + (z < extra ? 1 : 0);      // >= 1 by the host's choice

  if (threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w0) : "memory");
    if (GATED) asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w1) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_a) : "memory");
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int q = 0; q < QUADS; ++q) {
      mbar_init(scales_full(q), 1);
      mbar_init(scales_empty(q), 1);
    }
    mbar_init(done_bar, 1);
    ends->gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"(L::TMEM) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_arrive();              // matched by cluster_wait() in every role: nobody sends sums to a CTA that has not started
  tc_fence_after();
  const uint32_t tmem = uniform(*(volatile uint32_t*)(smem_raw + (tmem_slot - raw)));
  pdl_trigger();                 // after the allocation: a successor that is placed early waits for this grid with tensor memory in hand

  bool ok = true;
  if (warp == 0) {
    if (elect_one()) {
      auto load_weights = [&](int i, int s) {
        const uint32_t at = tiles + s * L::TILE_BYTES;
        tma_load_3d(at, &map_w0, 0, n0, kb0 + i, full_bar(s));
        if (GATED) tma_load_3d(at + W_BYTES, &map_w1, 0, n0, kb0 + i, full_bar(s));
        for (int m = 0; m < MATRICES; ++m)
          bulk_load(w_scales + (s * MATRICES + m) * SCALE_BYTES, args.w_scales[m] + ((size_t)(kb0 + i) * args.n_blocks + blockIdx.x) * SCALE_BYTES,
                    SCALE_BYTES, full_bar(s));
      };
      auto load_rows = [&](int i, int s) {
        tma_load_2d(tiles + s * L::TILE_BYTES + MATRICES * W_BYTES, &map_a, (kb0 + i) * BLOCK_K, t0, full_bar(s));
      };
      // the weights do not depend on the kernels before this one: their first stages start at once
      const int pre = min(num_kb, STAGES);
      for (int i = 0; i < pre; ++i) {
        mbar_expect_tx(full_bar(i), L::TX);
        load_weights(i, i);
      }
      pdl_wait();
      for (int i = 0; i < pre; ++i) load_rows(i, i);
      int issued = pre, s = 0;
      uint32_t parity = 0;
      for (int i = pre; i < num_kb; ++i) {
        ok = hand_over(empty_bar(s), parity, args.error, 101);
        if (!ok) break;
        mbar_expect_tx(full_bar(s), L::TX);
        load_weights(i, s);
        load_rows(i, s);
        issued = i + 1;
        if (++s == STAGES) { s = 0; parity ^= 1u; }
      }
      ends->issued = issued;
      if (!ok) ends->gave_up = 1;
    }
    __syncwarp();
    cluster_wait();
  } else if (warp == 1) {
    if (elect_one()) {
      const uint64_t weights0 = make_desc(tiles), rows0 = make_desc(tiles + MATRICES * W_BYTES), w_scales0 = make_desc_scales(w_scales), row_scales0 = make_desc_scales(row_ring);
      uint32_t bar = full_bar(0), at = 0, scales_at = 0, columns = tmem + L::ACCUMULATORS, parity = 0;      // this stage's: barrier, 16-byte units from the first on, scales
      uint32_t q = 0, quad_parity = 0;
      for (int i = 0; i < num_kb; ++i) {
        if ((i & 3) == 0) ok = hand_over(scales_full(q), quad_parity, args.error, 103);
        ok = ok && hand_over(bar, parity, args.error, 104);
        if (!ok) break;
        tc_fence_after();
        // A stage's scales have columns of their own: by the time the stage comes round again the MMAs that read them are done.
        tmem_cp_scales(columns, row_scales0 + (uint64_t)(q * (QUAD_BYTES >> 4) + (i & 3) * (SCALE_BYTES >> 4)));
#pragma unroll
        for (int m = 0; m < MATRICES; ++m) tmem_cp_scales(columns + 4 * (m + 1), w_scales0 + scales_at + (uint64_t)(m * (SCALE_BYTES >> 4)));
        const uint64_t weights = weights0 + at, rows = rows0 + at;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
#pragma unroll
          for (int m = 0; m < MATRICES; ++m)
            umma_mx(tmem + m * BT, weights + (uint64_t)(m * (W_BYTES >> 4) + 2 * k), rows + (uint64_t)(2 * k), idesc_mx_block(IDESC, k), columns + 4 * (m + 1), columns,
                    (i > 0 || k > 0) ? 1u : 0u);
        }
        umma_commit(bar + 8u * STAGES);
        bar += 8u;
        at += L::TILE_BYTES >> 4;
        scales_at += MATRICES * (SCALE_BYTES >> 4);
        columns += L::SCALE_COLUMNS;
        if (bar == full_bar(STAGES)) { bar = full_bar(0); at = scales_at = 0; columns = tmem + L::ACCUMULATORS; parity ^= 1u; }
        if ((i & 3) == 3) {
          umma_commit(scales_empty(q));
          if (++q == QUADS) { q = 0; quad_parity ^= 1u; }
        }
      }
      umma_commit(done_bar);     // arrives when every MMA issued so far is done
      if (!ok) ends->gave_up = 1;
    }
    __syncwarp();
    cluster_wait();
  } else {
    const int quarter = warp & 3, w = warp - 2;
    pdl_wait();
    for (int quad = w; w < QUADS && quad * 4 < num_kb; quad += 4) {          // quad q is warp q % 4's, and so is its place in the ring
      uint32_t words[(BT + 31) / 32][4];
#pragma unroll
      for (int j = 0; j < (BT + 31) / 32; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int i = quad * 4 + k, r = 32 * j + lane;
          words[j][k] = i < num_kb && r < BT ? row_scales(args, t0 + r, kb0 + i) : 0u;
        }
      if (quad >= QUADS && !hand_over_warp(scales_empty(w), ((uint32_t)(quad / QUADS) & 1u) ^ 1u, args.error, 105)) break;
#pragma unroll
      for (int j = 0; j < (BT + 31) / 32; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(row_ring + w * QUAD_BYTES + k * SCALE_BYTES + lane * 16 + j * 4), "r"(words[j][k]) : "memory");
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(scales_full(w));
    }
    __syncwarp();
    cluster_wait();
    ok = mbar_wait(done_bar, 0u, args.error, 106);
    tc_fence_after();
    const uint32_t quarter_at = tmem + ((uint32_t)(quarter * 32) << 16);
    const int first = 16 * (w / 4), step = L::EPILOGUE / 8;       // two warps to a quarter of the features: every other 16 rows each
    if (splits == 1) {
      const int n = n0 + quarter * 32 + lane;
      with_activation(args.act, [&](auto act) {
#pragma unroll 1
        for (int c = first; c < BT && t0 + c < args.T; c += step) {
          uint32_t r[MATRICES][16];
#pragma unroll
          for (int m = 0; m < MATRICES; ++m) tmem_ld16(quarter_at + (uint32_t)(m * BT + c), r[m]);
          tmem_ld_wait();
          float v[MATRICES][16];
#pragma unroll
          for (int m = 0; m < MATRICES; ++m)
#pragma unroll
            for (int j = 0; j < 16; ++j) v[m][j] = __uint_as_float(r[m][j]);
          finish_rows<GATED, decltype(act)::value, 16>(args, t0 + c, n, n < args.N, v[0], v[MATRICES - 1]);
        }
      });
    } else {
      // Sums go to the CTA that finishes their features, [matrix][split][four rows][feature]: neighbouring lanes 16 bytes apart.
      const int per = L::share(splits), local = quarter * 32 + lane;
      const uint32_t mine = map_to_cta(sums, (uint32_t)(local / per)) + 16u * (uint32_t)(local % per);
#pragma unroll
      for (int m = 0; m < MATRICES; ++m) {
#pragma unroll 1
        for (int c = first; c < BT && t0 + c < args.T; c += step) {
          uint32_t r[16];
          tmem_ld16(quarter_at + (uint32_t)(m * BT + c), r);
          tmem_ld_wait();
#pragma unroll
          for (int q = 0; q < 4; ++q)
            st_cluster_v4(mine + 16u * (uint32_t)(((m * splits + z) * (BT / 4) + c / 4 + q) * per), __uint_as_float(r[4 * q]),
                          __uint_as_float(r[4 * q + 1]), __uint_as_float(r[4 * q + 2]), __uint_as_float(r[4 * q + 3]));
        }
      }
    }
  }
  __syncwarp();
  if (splits > 1) {
    cluster_sync_all();          // every sum is where it belongs, and nobody leaves before
    if (warp >= 2) {
      const int per = L::share(splits), mine = min(per, TILE_N - z * per);      // none of a gated product's fifth CTA on
      const float4* part = (const float4*)(smem_raw + (sums - raw));
      with_activation(args.act, [&](auto act) {
#pragma unroll 1
        for (int p = threadIdx.x - 64; p < mine * (BT / 4); p += L::EPILOGUE) {
          const int f = p % mine, four = p / mine, t = t0 + 4 * four, n = n0 + z * per + f;
          if (t >= args.T) break;              // a warp's lanes have the same four rows where a block's scale is made (per >= 32)
          float v[MATRICES][4];
#pragma unroll
          for (int m = 0; m < MATRICES; ++m) {
            const float4* at = part + ((size_t)m * splits * (BT / 4) + four) * per + f;
            v[m][0] = v[m][1] = v[m][2] = v[m][3] = 0.f;
#pragma unroll 2
            for (int y = 0; y < splits; ++y) {                   // in the splits' order, whoever came first
              const float4 x = at[y * (BT / 4) * per];
              v[m][0] += x.x; v[m][1] += x.y; v[m][2] += x.z; v[m][3] += x.w;
            }
          }
          finish_rows<GATED, decltype(act)::value, 4>(args, t, n, n < args.N, v[0], v[MATRICES - 1]);
        }
      });
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::TMEM) : "memory");
  if (threadIdx.x == 0 && ends->gave_up) {       // each stage's last copies may not have been waited for (they are, where the MMAs ran)
    for (int i = max(0, ends->issued - STAGES); i < ends->issued; ++i) mbar_wait(full_bar(i % STAGES), (uint32_t)(i / STAGES) & 1u, args.error, 102);
  }
}

// --------------------------------------------------------------- many rows --
// Persistent CTAs over tiles of 128 rows (the MMA's M side, a row to a lane of tensor memory) by BN features (its N side; of a
// gated product BN of each matrix, one behind the other), two accumulators in tensor memory so that a tile's epilogue runs under the
// next one's main loop.  An epilogue thread owns a row and stores runs of features.  Bound by the MMAs and what the operands' and
// results' ways cost beside them: 4096 x 4096 x 16384 208 us (2.64 PFLOP/s) in short runs; without the epilogue 177, without the
// operands' copies 162, the MMAs alone 146; 243 us in long ones, where the power cap holds the clock at 1.3 to 1.6 GHz.
//
// Scales travel for four column blocks (a quad) at a time, as they lie in memory.  Four warps, one to a quarter of the lanes of
// tensor memory, put them there: the rows' turned (16 bytes come for each row), the weights' shifted so that a tile's first feature has
// the first column (the MMA takes its scales from a whole group of four columns on, and a tile may start at any 32 features).
// Copied by tcgen05.cp from shared memory, in order with the MMAs, they held those up: 2048 x 4096 x 4096 41 us against 30.
// (Pairs of CTAs, 256 rows and cta_group::2, were built: as fast with tcgen05.cp, three times slower with scales that the warps of both
// bring, for the issuing thread then waits for the other CTA at every column block.)
//
// Warp 0: the operands' copies; warp 1: MMA issue, tensor memory; warps 2, 3, 12, 13: scales; warps 4 ... 11: epilogue, two to a
// quarter of the rows, each with every other run of features; warp 14: the scales' copies.
constexpr int TILE_T = 128;
constexpr int MANY_THREADS = 480;
constexpr int ROWS_BYTES = TILE_T * BLOCK_K;
constexpr int MANY_MOST_STAGES = 8;
constexpr int MANY_QUADS = 2;                   // places of the ring of scales as they come
constexpr int MANY_MOST_BLOCKS = 3;             // of 128 features' scales that a tile of 224 touches
constexpr int MANY_BARS_BYTES = 288;            // barriers (three to a stage) and what lies behind them
static_assert(8 * (3 * MANY_MOST_STAGES + 4 + 2 * MANY_QUADS) + sizeof(Ends) <= MANY_BARS_BYTES && MANY_BARS_BYTES % 16 == 0, "barriers");

struct ManyShape {
  int BN, stages, m_tiles, n_tiles;
  int groups;                    // of four columns of scales: of 128 rows, and of 128 features of the MMA's N side (the last one not full perhaps)
  int w_touched;                 // aligned groups of 128 features that a tile touches at most
  int turned;                    // rows of the result start anywhere: not on 32-byte boundaries
  int smem;
};

// Eight words on a 32-byte boundary in one store: a whole sector of a lane's row, where two stores of half would be sent one by one.
__device__ __forceinline__ void store_32(void* at, const uint32_t* p) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(at), "r"(p[0]), "r"(p[1]), "r"(p[2]), "r"(p[3]), "r"(p[4]), "r"(p[5]),
               "r"(p[6]), "r"(p[7]) : "memory");
}

__device__ __forceinline__ void load_32(const float* at, float* v) {
  asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]) : "l"(at) : "memory");
}

// 16 features n ... of row t, linear, where every row's start on a 32-byte boundary.
template <int ACT>
__device__ __forceinline__ void finish_features(const Args& a, int t, int n, const uint32_t (&r)[16]) {
  if (t >= a.T) return;
  const size_t at = (size_t)t * a.N + n;
  float v[16], res[16];
  if (a.residual) {
    load_32(a.residual + at, res);
    load_32(a.residual + at + 8, res + 8);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float4 b = a.bias ? reinterpret_cast<const float4*>(a.bias + n)[j] : make_float4(0.f, 0.f, 0.f, 0.f);
    v[4 * j] = __uint_as_float(r[4 * j]) + b.x; v[4 * j + 1] = __uint_as_float(r[4 * j + 1]) + b.y;
    v[4 * j + 2] = __uint_as_float(r[4 * j + 2]) + b.z; v[4 * j + 3] = __uint_as_float(r[4 * j + 3]) + b.w;
  }
#pragma unroll
  for (int j = 0; j < 16; ++j) v[j] = activated<ACT>(v[j], a.act);
  if (a.residual) {
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] += res[j];
  }
  if (a.out_bf16) {
    uint32_t p[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const __nv_bfloat162 two = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
      p[j] = *reinterpret_cast<const uint32_t*>(&two);
    }
    store_32((__nv_bfloat16*)a.C + at, p);
  } else {
    uint32_t p[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) p[j] = __float_as_uint(v[j]);
    store_32((float*)a.C + at, p);
    store_32((float*)a.C + at + 8, p + 8);
  }
}

// The same for rows that start anywhere: a warp turns its 32 rows (from t0 on), 32 features at a time, in shared memory and writes them row
// by row, a lane to a feature.  (5000 x 128 x 2001, us: 13.0; lanes that write their own rows, 2 bytes to a sector, 85; pieces of 8
// bytes shifted into line through shared memory 16.9, whole sectors 27, for a row's ends then take longer than its middle.  2000
// features, in whole sectors as they are, 6.7.)
constexpr int TURNED_ROW = 33;                  // words: a column's neighbours are on other banks
constexpr int TURNED_BYTES = 8 * 32 * TURNED_ROW * 4;
template <int ACT, typename O>
__device__ __forceinline__ void finish_turned(const Args& a, uint32_t sums, float* mine, int t0, int n0, int columns) {
  const int lane = threadIdx.x & 31, rows = min(32, a.T - t0);
#pragma unroll 1
  for (int c = 0; c < columns && n0 + c < a.N; c += 32) {
    uint32_t r[32];
    tmem_ld32(sums + c, r);                     // of a last half run, what lies behind it too
    tmem_ld_wait();
#pragma unroll
    for (int j = 0; j < 32; ++j) mine[lane * TURNED_ROW + j] = __uint_as_float(r[j]);
    __syncwarp();
    const int n = n0 + c + lane;
    if (c + lane < columns && n < a.N) {
      const float b = a.bias ? a.bias[n] : 0.f;
      O* out = (O*)a.C + (size_t)t0 * a.N + n;
      const float* add = a.residual + (size_t)t0 * a.N + n;
      for (int first = 0; first < rows; first += 8) {
        float res[8];
        if (a.residual) {
#pragma unroll
          for (int i = 0; i < 8; ++i) res[i] = first + i < rows ? add[(size_t)i * a.N] : 0.f;
          add += (size_t)8 * a.N;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float y = activated<ACT>(mine[(first + i) * TURNED_ROW + lane] + b, a.act);
          if (a.residual) y += res[i];
          if (first + i < rows) *out = from_float<O>(y);
          out += a.N;
        }
      }
    }
    __syncwarp();
  }
}

// A block of 32 features of row t, gated: the scale and the codes of one thread.
template <int ACT>
__device__ __forceinline__ void finish_block(const Args& a, int t, int n, const uint32_t (&g)[32], const uint32_t (&u)[32]) {
  if (t >= a.T || n >= a.N) return;
  float v[32];
  uint32_t largest = 0u;
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    v[j] = activated<ACT>(__uint_as_float(g[j]), a.act) * __uint_as_float(u[j]);
    largest = max(largest, magnitude_bits(v[j]));
  }
  const uint32_t code = mx_scale_code(largest);
  const float inverse = mx_inverse(code);
  uint32_t p[8];
#pragma unroll
  for (int j = 0; j < 8; ++j)
    p[j] = e4m3_pair(v[4 * j] * inverse, v[4 * j + 1] * inverse) | (e4m3_pair(v[4 * j + 2] * inverse, v[4 * j + 3] * inverse) << 16);
  store_32((uint8_t*)a.C + (size_t)t * a.N + n, p);
  a.out_scales[(size_t)t * a.out_scale_stride + n / MX_BLOCK] = (uint8_t)code;
}

__device__ __forceinline__ void lds_v4(uint32_t at, uint32_t* w) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
}
// Where a warp gave up: the last tile's MMAs, each stage's last copies and the scales' last ones.  (Not inline: instructions that no launch runs
// stood in the way of those behind them.)
__device__ __noinline__ void wait_for_the_last(uint32_t sums, uint32_t parity, uint32_t full, int issued, int stages, uint32_t come, int quads, int* error) {
  mbar_wait(sums, parity, error, 112);
  for (int i = max(0, issued - stages); i < issued; ++i) mbar_wait(full + 8u * (i % stages), (uint32_t)(i / stages) & 1u, error, 112);
  for (int i = max(0, quads - MANY_QUADS); i < quads; ++i) mbar_wait(come + 8u * (i % MANY_QUADS), (uint32_t)(i / MANY_QUADS) & 1u, error, 112);
}
template <bool GATED>
__global__ void __launch_bounds__(MANY_THREADS, 1)
linear4_many_kernel(const __grid_constant__ CUtensorMap map_w0, const __grid_constant__ CUtensorMap map_w1, const __grid_constant__ CUtensorMap map_a,
                    const __grid_constant__ CUtensorMap map_s, const Args args, const ManyShape shape) {
  constexpr int MATRICES = GATED ? 2 : 1;
  extern __shared__ uint8_t smem_raw[];
  const int BN = shape.BN, stages = shape.stages;
  const int weight_bytes = BN * BLOCK_K, tile_bytes = ROWS_BYTES + MATRICES * weight_bytes, groups = shape.groups;
  const int quad_bytes = (1 + MATRICES * shape.w_touched) * QUAD_BYTES;      // as they come: rows [128][16], features [matrix][column block][group][512]
  const uint32_t raw = smem_u32(smem_raw), tiles = (raw + 1023u) & ~1023u, come = tiles + stages * tile_bytes, bars = come + MANY_QUADS * quad_bytes;
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (MANY_MOST_STAGES + s); };
  auto sums_full = [&](int b) { return bars + 8u * (2 * MANY_MOST_STAGES + b); };
  auto sums_empty = [&](int b) { return bars + 8u * (2 * MANY_MOST_STAGES + 2 + b); };
  auto come_full = [&](int q) { return bars + 8u * (2 * MANY_MOST_STAGES + 4 + q); };
  auto come_empty = [&](int q) { return bars + 8u * (2 * MANY_MOST_STAGES + 4 + MANY_QUADS + q); };
  auto scaled_bar = [&](int s) { return bars + 8u * (2 * MANY_MOST_STAGES + 4 + 2 * MANY_QUADS + s); };
  const uint32_t tmem_slot = scaled_bar(MANY_MOST_STAGES);
  volatile Ends* ends = (volatile Ends*)(smem_raw + (tmem_slot - raw));

  const int warp = warp_number(), lane = threadIdx.x & 31;
  const int num_kb = (args.K + BLOCK_K - 1) / BLOCK_K;
  const int num_tiles = shape.m_tiles * shape.n_tiles;

  if (threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w0) : "memory");
    if (GATED) asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w1) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_a) : "memory");
    for (int s = 0; s < stages; ++s) {
      mbar_init(full_bar(s), 1);             // the operands' copies alone, so that they can be waited for whatever became of the scales
      mbar_init(scaled_bar(s), 4);           // the four warps that bring the scales
      mbar_init(empty_bar(s), 1);
    }
    for (int q = 0; q < MANY_QUADS; ++q) {
      mbar_init(come_full(q), 1);
      mbar_init(come_empty(q), 4);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(sums_full(b), 1);
      mbar_init(sums_empty(b), 8);
    }
    ends->gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(*(volatile uint32_t*)(smem_raw + (tmem_slot - raw)));
  pdl_trigger();                 // after the allocation, see above

  bool ok = true;
  if (warp == 0) {
    if (elect_one()) {
      pdl_wait();
      const uint32_t tx = ROWS_BYTES + MATRICES * weight_bytes / 2;        // codes count as they travel, two to a byte
      const uint32_t bars_end = full_bar(stages), to_empty = empty_bar(0) - full_bar(0);
      uint32_t bar = full_bar(0), at = tiles, parity = 1;                  // a barrier's first wait by the opposite parity returns at once
      int issued = 0;
      for (int tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x) {
        const int t0 = tile % shape.m_tiles * TILE_T, n0 = tile / shape.m_tiles * BN;
        for (int kb = 0; kb < num_kb; ++kb) {
          ok = hand_over(bar + to_empty, parity, args.error, 111);
          if (!ok) break;
          mbar_expect_tx(bar, tx);
          tma_load_2d(at, &map_a, kb * BLOCK_K, t0, bar);
          tma_load_3d(at + ROWS_BYTES, &map_w0, 0, n0, kb, bar);
          if (GATED) tma_load_3d(at + ROWS_BYTES + weight_bytes, &map_w1, 0, n0, kb, bar);
          ++issued;
          bar += 8u;
          at += tile_bytes;
          if (bar == bars_end) { bar = full_bar(0); at = tiles; parity ^= 1u; }
        }
      }
      ends->issued = issued;
      if (!ok) ends->gave_up = 1;
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t idesc = make_idesc_mx(TILE_T, MATRICES * BN, MX_E4M3, MX_E2M1);
      const uint32_t bars_end = full_bar(stages), to_empty = empty_bar(0) - full_bar(0), to_scaled = scaled_bar(0) - full_bar(0), all_sums = 2 * MATRICES * BN;
      const uint64_t rows0 = make_desc(tiles), weights0 = make_desc(tiles + ROWS_BYTES);
      uint32_t bar = full_bar(0), at = 0, parity = 0, columns = tmem + all_sums;      // this stage's: barrier, 16-byte units from the first on, scales
      int it = 0;
      for (int tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x, ++it) {
        const uint32_t buffer = it & 1, sums = tmem + buffer * MATRICES * BN;
        if (it >= 2) ok = hand_over(sums_empty(buffer), ((uint32_t)(it >> 1) & 1u) ^ 1u, args.error, 113);
        for (int kb = 0; kb < num_kb && ok; ++kb) {
          ok = hand_over(bar + to_scaled, parity, args.error, 119) && hand_over(bar, parity, args.error, 114);
          if (!ok) break;
          tc_fence_after();
          const uint64_t rows = rows0 + at, weights = weights0 + at;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_mx(sums, rows + (uint64_t)(2 * k), weights + (uint64_t)(2 * k), idesc_mx_block(idesc, k), columns, columns + 4, (kb > 0 || k > 0) ? 1u : 0u);
          umma_commit(bar + to_empty);
          bar += 8u;
          at += tile_bytes >> 4;
          columns += 4 * groups;
          if (bar == bars_end) { bar = full_bar(0); at = 0; columns = tmem + all_sums; parity ^= 1u; }
        }
        umma_commit(sums_full(buffer));
      }
      ends->tiles = it;
      if (!ok) ends->gave_up = 1;
    }
    __syncwarp();
  } else if (warp == 14) {
    if (elect_one()) {
      int quads = 0;
      pdl_wait();
      for (int tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x) {
        const int t0 = tile % shape.m_tiles * TILE_T, n0 = tile / shape.m_tiles * BN, block0 = n0 / TILE_N;
        const int blocks = min((n0 % TILE_N + BN + TILE_N - 1) / TILE_N, args.n_blocks - block0);
        for (int first = 0; first < num_kb; first += 4, ++quads) {
          const int q = quads % MANY_QUADS, kbs = min(4, num_kb - first);
          if (quads >= MANY_QUADS) ok = hand_over(come_empty(q), ((uint32_t)(quads / MANY_QUADS) & 1u) ^ 1u, args.error, 116);
          if (!ok) break;
          mbar_expect_tx(come_full(q), QUAD_BYTES + MATRICES * kbs * blocks * SCALE_BYTES);
          tma_load_2d(come + q * quad_bytes, &map_s, 4 * first, t0, come_full(q));
          for (int m = 0; m < MATRICES; ++m)
            for (int k = 0; k < kbs; ++k)      // [matrix][column block][group]: a column block's groups lie side by side in memory too
              bulk_load(come + q * quad_bytes + QUAD_BYTES + (m * 4 + k) * shape.w_touched * SCALE_BYTES,
                        args.w_scales[m] + ((size_t)(first + k) * args.n_blocks + block0) * SCALE_BYTES, blocks * SCALE_BYTES, come_full(q));
        }
      }
      ends->quads = quads;
      if (!ok) ends->gave_up = 1;
    }
    __syncwarp();
  } else if (warp < 4 || warp >= 12) {
    const uint32_t lanes = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + 2 * MATRICES * BN, bars_end = full_bar(stages), to_empty = empty_bar(0) - full_bar(0), to_scaled = scaled_bar(0) - full_bar(0);
    uint32_t bar = full_bar(0), columns = lanes, parity = 1;       // of the stage: the scales' columns are free when the operands' place is
    int quad = 0;
    for (int tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x) {
      const int shift = tile / shape.m_tiles * BN % TILE_N / 32;
      for (int first = 0; first < num_kb && ok; first += 4, ++quad) {
        const int q = quad % MANY_QUADS;
        const uint32_t from = come + q * quad_bytes + lane * 16;
        ok = hand_over_warp(come_full(q), (uint32_t)(quad / MANY_QUADS) & 1u, args.error, 115);
        if (!ok) break;
        uint32_t r[4][4];                    // rows lane, lane + 32, ...: 16 bytes are a row's four column blocks
#pragma unroll
        for (int j = 0; j < 4; ++j) lds_v4(from + j * 512, r[j]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (first + k >= num_kb || !ok) continue;
          ok = hand_over_warp(bar + to_empty, parity, args.error, 118);
          if (!ok) continue;
          tc_fence_after();
          tmem_st4(columns, r[0][k], r[1][k], r[2][k], r[3][k]);
          uint32_t w[MATRICES][4 * MANY_MOST_BLOCKS + 4];          // this lane's columns of the groups, in a row
#pragma unroll
          for (int m = 0; m < MATRICES; ++m) {
#pragma unroll
            for (int g = 0; g < MANY_MOST_BLOCKS; ++g)
              if (g < shape.w_touched) lds_v4(from + QUAD_BYTES + ((m * 4 + k) * shape.w_touched + g) * SCALE_BYTES, w[m] + 4 * g);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[m][4 * MANY_MOST_BLOCKS + j] = 0u;
            if (shift & 1)
#pragma unroll
              for (int j = 0; j < 4 * MANY_MOST_BLOCKS; ++j) w[m][j] = w[m][j + 1];
            if (shift & 2)
#pragma unroll
              for (int j = 0; j < 4 * MANY_MOST_BLOCKS; ++j) w[m][j] = w[m][j + 2];
          }
          if (GATED) {                       // the second matrix's behind the first one's: one, two or three columns on
#pragma unroll
            for (int j = 5; j >= 1; --j) w[0][j] = 32 * j < BN ? w[0][j] : BN == 32 ? w[MATRICES - 1][j - 1] : BN == 64 ? w[MATRICES - 1][max(j - 2, 0)] : w[MATRICES - 1][max(j - 3, 0)];
          }
#pragma unroll
          for (int g = 0; g < MANY_MOST_BLOCKS - 1; ++g)
            if (g < groups - 1) tmem_st4(columns + 4 * (1 + g), w[0][4 * g], w[0][4 * g + 1], w[0][4 * g + 2], w[0][4 * g + 3]);
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar + to_scaled);
          bar += 8u;
          columns += 4 * groups;
          if (bar == bars_end) { bar = full_bar(0); columns = lanes; parity ^= 1u; }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(come_empty(q));
      }
    }
    if (!ok) ends->gave_up = 1;
  } else {
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    pdl_wait();
    with_activation(args.act, [&](auto act) {
      constexpr int ACT = decltype(act)::value;
      int it = 0;
      for (int tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x, ++it) {
        const int buffer = it & 1, t = tile % shape.m_tiles * TILE_T + quarter * 32 + lane, n0 = tile / shape.m_tiles * BN;
        ok = hand_over_warp(sums_full(buffer), (uint32_t)(it >> 1) & 1u, args.error, 117);
        if (!ok) break;
        tc_fence_after();
        const uint32_t sums = tmem + ((uint32_t)(quarter * 32) << 16) + buffer * MATRICES * BN;
        if constexpr (GATED) {
#pragma unroll 1
          for (int c = half * 32; c < BN && n0 + c < args.N; c += 64) {
            uint32_t g[32], u[32];
            tmem_ld32(sums + c, g);
            tmem_ld32(sums + BN + c, u);
            tmem_ld_wait();
            finish_block<ACT>(args, t, n0 + c, g, u);
          }
        } else if (shape.turned) {
          float* mine = (float*)(smem_raw + (bars + MANY_BARS_BYTES - raw)) + (warp - 4) * 32 * TURNED_ROW;
          const int from = half * (BN / 2);
          if (args.out_bf16) finish_turned<ACT, __nv_bfloat16>(args, sums + from, mine, t - lane, n0 + from, BN / 2);
          else finish_turned<ACT, float>(args, sums + from, mine, t - lane, n0 + from, BN / 2);
        } else {
#pragma unroll 1
          for (int c = half * 16; c < BN && n0 + c < args.N; c += 32) {
            uint32_t r[16];
            tmem_ld16(sums + c, r);
            tmem_ld_wait();
            finish_features<ACT>(args, t, n0 + c, r);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(sums_empty(buffer));
      }
    });
    if (!ok) ends->gave_up = 1;
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    if (ends->gave_up) {
      const int last = ends->tiles - 1;
      wait_for_the_last(sums_full(last & 1), (uint32_t)(last >> 1) & 1u, full_bar(0), ends->issued, stages, come_full(0), ends->quads, args.error);
      __syncwarp();
    }
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// ------------------------------------------------------------------- host --

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn g_encode = nullptr;
int* g_error_host = nullptr;     // mapped pinned memory: the kernels write, the host reads without a copy
int* g_error_dev = nullptr;
std::mutex g_mutex;

int setup() {
  std::lock_guard<std::mutex> lock(g_mutex);
  if (g_encode && g_error_dev) return 0;
  void* fn = nullptr;
  cudaDriverEntryPointQueryResult q;
  cudaError_t err = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q);
  if (err != cudaSuccess || fn == nullptr || q != cudaDriverEntryPointSuccess) return ayk_fail("ayk_linear4: cuTensorMapEncodeTiled is not available from this driver");
  if (!g_error_host) {
    // the first call may be one that is captured, which bars its thread from allocations unless it says that they may be made
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    cudaThreadExchangeStreamCaptureMode(&mode);
    err = cudaHostAlloc((void**)&g_error_host, sizeof(int), cudaHostAllocMapped | cudaHostAllocPortable);
    cudaThreadExchangeStreamCaptureMode(&mode);
    if (err != cudaSuccess) return ayk_fail("ayk_linear4: cudaHostAlloc: %s", cudaGetErrorString(err));
    *g_error_host = 0;
  }
  err = cudaHostGetDevicePointer((void**)&g_error_dev, g_error_host, 0);
  if (err != cudaSuccess) return ayk_fail("ayk_linear4: cudaHostGetDevicePointer: %s", cudaGetErrorString(err));
  g_encode = (EncodeTiledFn)fn;
  return 0;
}

// Rows of codes [T, K], rows `stride` bytes apart: boxes of 128 columns.
int encode_rows(CUtensorMap* map, const void* p, long long T, int K, long long stride, int box) {
  cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)T}, strides[1] = {(cuuint64_t)stride};
  cuuint32_t boxes[2] = {BLOCK_K, (cuuint32_t)box}, step[2] = {1, 1};
  const CUresult r = g_encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(p), dims, strides, boxes, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return ayk_fail("ayk_linear4: cuTensorMapEncodeTiled of the rows failed with %d", (int)r);
  return 0;
}
// The rows' scales, rows `stride` bytes apart: boxes of 16 bytes (four column blocks) and 128 rows.
int encode_scales(CUtensorMap* map, const void* p, long long T, int K, long long stride) {
  cuuint64_t dims[2] = {(cuuint64_t)(K / MX_BLOCK), (cuuint64_t)T}, strides[1] = {(cuuint64_t)stride};
  cuuint32_t boxes[2] = {16, TILE_T}, step[2] = {1, 1};
  const CUresult r = g_encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(p), dims, strides, boxes, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return ayk_fail("ayk_linear4: cuTensorMapEncodeTiled of the rows' scales failed with %d", (int)r);
  return 0;
}
// A weight's codes [K / 128][rows][128]: boxes of `box` rows, spread to a byte each.
int encode_weight(CUtensorMap* map, const void* p, int rows, int K, int box) {
  cuuint64_t dims[3] = {BLOCK_K, (cuuint64_t)rows, (cuuint64_t)((K + BLOCK_K - 1) / BLOCK_K)};
  cuuint64_t strides[2] = {BLOCK_K / 2, (cuuint64_t)rows * (BLOCK_K / 2)};
  cuuint32_t boxes[3] = {BLOCK_K, (cuuint32_t)box, 1}, step[3] = {1, 1, 1};
  const CUresult r = g_encode(map, CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B, 3, const_cast<void*>(p), dims, strides, boxes, step,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return ayk_fail("ayk_linear4: cuTensorMapEncodeTiled of the weight failed with %d", (int)r);
  return 0;
}

// ----------------------------------------------------------------- choices --
// CTAs along K to a tile of the few-row kernel, 1 ... 8.  The clusters of a launch should run at once: with one CTA to a multiprocessor
// a B200 of 148 takes so many clusters of 1, 2, ... 8 (the driver's occupancy; a cluster stays within a group of multiprocessors), with
// two as many as were seen to run side by side (S CTAs of 8 column blocks each: 70 clusters of four 6.3 us, 72 10.0; 33 of eight 6.6, 34
// 10.0).  Among those, the least time: column blocks one after the other, 0.25 us each (two matrices 0.33), 0.6 for the exchange of the
// sums, and of a gated product the epilogue, which four CTAs share.  (us with 1, 2, 4, 8: 8 x 4096 x 4096 9.5, 6.6, 5.4, 5.7; 64 x 6400 x
// 1600 14.4, 10.0, 7.1, 6.3; 50 x 2976 x 4226, 34 tiles, 8.5, 7.2, 11.3, 15.1 and with 3 6.8; gated 16 x 768 x 768 5.4, 3.8, 3.6, 3.4.)
template <int BT, bool GATED>
constexpr int MOST_SPLITS = GATED && BT >= 64 ? 4 : 8;           // what the sums leave of shared memory

template <int BT, bool GATED>
int few_clusters(int splits, int sms) {      // that run at once
  constexpr int one[8] = {148, 74, 45, 33, 26, 22, 15, 15}, two[8] = {296, 148, 90, 66, 52, 44, 32, 32};
  return (Few<BT, GATED>::PLACES == 2 ? two : one)[splits - 1] * sms / 148;
}
template <int BT, bool GATED>
int few_splits(int T, int N, int K, int sms) {
  const long long tiles = (long long)((N + TILE_N - 1) / TILE_N) * ((T + BT - 1) / BT);
  const int blocks = (K + BLOCK_K - 1) / BLOCK_K;
  int best = 1;
  double least = 0;
  for (int s = 1; s <= MOST_SPLITS<BT, GATED> && s <= blocks; ++s) {
    if ((s > 1 && tiles > few_clusters<BT, GATED>(s, sms)) || Few<BT, GATED>::smem(s) > 232448) continue;
    const double us = (GATED ? 0.33 : 0.25) * ((blocks + s - 1) / s) + (s > 1 ? 0.6 : 0) + (GATED ? (1.0 + 0.05 * BT) / (s < 4 ? s : 4) : 0);
    if (least == 0 || us < least) {
      best = s;
      least = us;
    }
  }
  return best;
}

// Microseconds of the two kernels, fitted to graphs of 20 launches each on a B200 (N and K from 768 to 16384, 65 to 1024 rows): per wave of
// CTAs a fixed part and one per column block.  The estimates are 0.78 to 1.21 times what the kernel for few rows takes (0.97 in the median),
// but 0.88 to 1.53 times what the one for many takes (1.25): they are of a form of it whose scales were copied by tcgen05.cp.  Both sides of
// the choice as they are now, us few / many: 128 x 6400 x 1600 7.4 / 12.5, 1024 x 6400 x 1600 29.5 / 14.1, 128 x 4096 x 16384 21.9 / 10.6, gated
// 128 x 16384 x 4096 28.4 / 36.9, each of which goes to the quicker one; but 512 x 6400 x 1600 14.8 / 13.0, gated 256 x 4096 x 4096 17.7 / 12.2
// (to the quicker one) and gated 384 x 6400 x 1600 23.5 / 16.2: of 112 products 18 go to the slower kernel, which costs 7 to 45 % there.
template <bool GATED>
double few_us(int T, int N, int K, int sms) {
  const int splits = few_splits<64, GATED>(T, N, K, sms), blocks = (K + BLOCK_K - 1) / BLOCK_K;
  const long long tiles = (long long)((N + TILE_N - 1) / TILE_N) * ((T + 63) / 64), at_once = few_clusters<64, GATED>(splits, sms);
  return 1.2 + (double)((tiles + at_once - 1) / at_once) * ((GATED ? 5.0 : 3.2) + (GATED ? 0.335 : 0.22) * ((blocks + splits - 1) / splits));
}

// The many-row kernel's tile width, with its time: wider tiles cost less a feature and fill the last wave less.
template <bool GATED>
ManyShape many_shape(int T, int N, int K, int sms, int turned, double* us) {
  constexpr int MATRICES = GATED ? 2 : 1;
  const int widths[6] = {224, 192, 128, 96, 64, 32};
  const int blocks = (K + BLOCK_K - 1) / BLOCK_K;
  ManyShape best{};
  *us = 0;
  for (int i = GATED ? 3 : 0; i < 6; ++i) {
    ManyShape s{};
    s.BN = widths[i];
    s.m_tiles = (T + TILE_T - 1) / TILE_T;
    s.n_tiles = (N + s.BN - 1) / s.BN;
    s.groups = 1 + (MATRICES * s.BN + TILE_N - 1) / TILE_N;
    s.w_touched = ((TILE_N % s.BN == 0 ? 0 : s.BN == 192 ? 64 : 96) + s.BN + TILE_N - 1) / TILE_N;      // a tile starts so far behind a group at most
    const int stage = ROWS_BYTES + MATRICES * s.BN * BLOCK_K;
    s.turned = turned;
    s.smem = 1024 + MANY_QUADS * (1 + MATRICES * s.w_touched) * QUAD_BYTES + MANY_BARS_BYTES + (turned ? TURNED_BYTES : 0);
    s.stages = (232448 - s.smem) / stage;
    if (s.stages > (512 - 2 * MATRICES * s.BN) / (4 * s.groups)) s.stages = (512 - 2 * MATRICES * s.BN) / (4 * s.groups);      // columns of scales
    if (s.stages > MANY_MOST_STAGES) s.stages = MANY_MOST_STAGES;
    s.smem += s.stages * stage;
    const long long tiles = (long long)s.m_tiles * s.n_tiles;
    const double block = GATED ? 0.33 + 0.0012 * s.BN : 0.262 + 0.00057 * s.BN;
    const double time = 2.5 + 0.005 * s.BN + (double)((tiles + sms - 1) / sms) * blocks * block;
    if (*us == 0 || time < *us) {
      best = s;
      *us = time;
    }
  }
  return best;
}

// Up to 64 rows every weight byte goes by once in the few-row kernel; above, the quicker one, where its grid has room.
constexpr int FEW_MOST_TILES = 65535;      // of rows: a grid's second side
template <bool GATED>
bool takes_few(int T, int N, int K, int sms) {
  double many;
  if (T <= 64) return true;
  if ((T + 63) / 64 > FEW_MOST_TILES) return false;
  many_shape<GATED>(T, N, K, sms, 0, &many);
  return few_us<GATED>(T, N, K, sms) < many;
}

template <int BT, bool GATED>
int launch_few(const CUtensorMap& w0, const CUtensorMap& w1, const CUtensorMap& a, const Args& args, const char* name, cudaStream_t stream) {
  using L = Few<BT, GATED>;
  constexpr int MOST = MOST_SPLITS<BT, GATED>;
  static_assert(L::smem(MOST) <= 232448 && L::smem(1) <= 232448, "shared memory");
  static_assert(L::USED <= 512 && 8 * (2 * L::STAGES + 2 * QUADS + 2) <= 256 && L::AT_BARS % 16 == 0, "layout");
  const int tiles_n = (args.N + TILE_N - 1) / TILE_N, tiles_t = (args.T + BT - 1) / BT;
  AYK_REQUIRE(tiles_t <= FEW_MOST_TILES, "%s: too many rows (%d)", name, args.T);
  const int splits = few_splits<BT, GATED>(args.T, args.N, args.K, ayk_sm_count());
  static AykPerDevice configured;
  {
    std::lock_guard<std::mutex> lock(g_mutex);
    bool& done = configured.here();
    if (!done) {
      int most = 0;
      for (int s = 1; s <= MOST; ++s) most = L::smem(s) > most && L::smem(s) <= 232448 ? L::smem(s) : most;
      const cudaError_t err = cudaFuncSetAttribute(linear4_few_kernel<BT, GATED>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
      if (err != cudaSuccess) return ayk_fail("%s: shared memory %d: %s", name, most, cudaGetErrorString(err));
      done = true;
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(tiles_n, tiles_t, splits);
  cfg.blockDim = dim3(L::THREADS);
  cfg.dynamicSmemBytes = L::smem(splits);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = splits;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ayk_pdl_enabled() ? 2 : 1;
  cudaLaunchKernelEx(&cfg, linear4_few_kernel<BT, GATED>, w0, w1, a, args);
  return ayk_check_launch(name);
}

template <bool GATED>
int launch_many(const void* codes0, const void* codes1, const void* a, long long a_stride, const Args& args, const char* name, cudaStream_t stream) {
  const bool turned = !GATED && !(args.N % 16 == 0 && (uintptr_t)args.C % 32 == 0 && (uintptr_t)args.bias % 16 == 0 && (uintptr_t)args.residual % 32 == 0);
  double us;
  const ManyShape s = many_shape<GATED>(args.T, args.N, args.K, ayk_sm_count(), turned, &us);
  const long long tiles = (long long)s.m_tiles * s.n_tiles;
  AYK_REQUIRE(tiles <= 0x7fffffff - 65536, "%s: too many rows (%d) and columns (%d)", name, args.T, args.N);
  CUtensorMap w0, w1, rows, row_scales;
  const int padded = args.n_blocks * TILE_N;
  if (encode_weight(&w0, codes0, padded, args.K, s.BN) != 0 || (GATED && encode_weight(&w1, codes1, padded, args.K, s.BN) != 0) ||
      encode_rows(&rows, a, args.T, args.K, a_stride, TILE_T) != 0 || encode_scales(&row_scales, args.a_scales, args.T, args.K, args.a_scale_stride) != 0)
    return -1;
  static AykPerDevice configured;
  {
    std::lock_guard<std::mutex> lock(g_mutex);
    bool& done = configured.here();
    if (!done) {
      const cudaError_t err = cudaFuncSetAttribute(linear4_many_kernel<GATED>, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448);
      if (err != cudaSuccess) return ayk_fail("%s: shared memory: %s", name, cudaGetErrorString(err));
      done = true;
    }
  }
  const int sms = ayk_sm_count();
  ayk_launch(linear4_many_kernel<GATED>, dim3((unsigned)(tiles < sms ? tiles : sms)), dim3(MANY_THREADS), (size_t)s.smem, stream, w0, GATED ? w1 : w0, rows,
             row_scales, args, s);
  return ayk_check_launch(name);
}

int check(const char* name, const void* a, long long a_stride, const void* a_scales, long long a_scale_stride, long long T, int N, int K, int act) {
  AYK_REQUIRE(N > 0 && K > 0 && K % MX_BLOCK == 0, "%s: a product of %d columns over rows of %d (whole blocks of %d)", name, N, K, MX_BLOCK);
  AYK_REQUIRE(T >= 0 && T <= 0x7fffffff - 256 && N <= 0x7fffffff - 256 && K <= 0x7fffffff - 256, "%s: too many rows (%lld) or columns (%d, %d)", name, T, N, K);
  AYK_REQUIRE(act >= AYK_ACT_NONE && act <= AYK_ACT_SILU, "%s: unknown activation %d", name, act);
  AYK_REQUIRE((uintptr_t)a % 16 == 0 && a_stride % 16 == 0 && a_stride >= K, "%s: rows of codes must lie on 16-byte boundaries", name);
  AYK_REQUIRE((uintptr_t)a_scales % 16 == 0 && a_scale_stride % 16 == 0 && a_scale_stride >= K / MX_BLOCK, "%s: rows of scales must lie on 16-byte boundaries", name);
  return 0;
}

}  // namespace

AYK_EXPORT int ayk_linear4_error() { return g_error_host ? *g_error_host : 0; }
AYK_EXPORT void ayk_linear4_clear_error() { if (g_error_host) *g_error_host = 0; }

// What a product of these sizes runs as: rows of a tile (16, 32 or 64: the few-row kernel, with `parts` CTAs along K to a tile; 128:
// the many-row kernel, with tiles `parts` features wide).  Host arithmetic.
AYK_EXPORT int ayk_linear4_plan(int T, int N, int K, int gated, int sms, int* parts) {
  AYK_REQUIRE(T >= 1 && N >= 1 && K >= MX_BLOCK && K % MX_BLOCK == 0 && sms >= 1 && T <= 0x7fffffff - 256 && N <= 0x7fffffff - 256 && K <= 0x7fffffff - 256,
              "ayk_linear4_plan: no product of %d rows of %d columns and %d features on %d SMs", T, K, N, sms);
  double us;
  if (!(gated ? takes_few<true>(T, N, K, sms) : takes_few<false>(T, N, K, sms))) {
    *parts = gated ? many_shape<true>(T, N, K, sms, 0, &us).BN : many_shape<false>(T, N, K, sms, N % 16 != 0, &us).BN;
    return TILE_T;
  }
  if (T <= 16) *parts = gated ? few_splits<16, true>(T, N, K, sms) : few_splits<16, false>(T, N, K, sms);
  else if (T <= 32) *parts = gated ? few_splits<32, true>(T, N, K, sms) : few_splits<32, false>(T, N, K, sms);
  else *parts = gated ? few_splits<64, true>(T, N, K, sms) : few_splits<64, false>(T, N, K, sms);
  return T <= 16 ? 16 : T <= 32 ? 32 : 64;
}

// The arguments come as one block of memory: a call with fifteen of them from Python takes 0.6 us more.
//
// a [T, K] e4m3 (rows a_stride bytes apart) and its scales; codes and scales of the weight [N, K] as laid out (see the head); C
// [T, N] float32 or bfloat16; bias, residual float32 or null (the residual may be a float32 C).
struct Linear4Call {
  void* C;
  const void *a, *a_scales;
  long long a_stride, a_scale_stride;
  const void *codes, *scales;
  const float *bias, *residual;
  long long T;
  int N, K, act, out_dtype;
  cudaStream_t stream;
};
AYK_EXPORT int ayk_linear4(const Linear4Call* call) {
  const Linear4Call c = *call;
  if (check("ayk_linear4", c.a, c.a_stride, c.a_scales, c.a_scale_stride, c.T, c.N, c.K, c.act) != 0) return -1;
  AYK_REQUIRE(c.out_dtype == AYK_DTYPE_F32 || c.out_dtype == AYK_DTYPE_BF16, "ayk_linear4: unknown output dtype %d", c.out_dtype);
  if (c.T == 0) return 0;
  if (setup() != 0) return -1;
  Args args{};
  args.C = c.C; args.a_scales = (const uint8_t*)c.a_scales; args.a_scale_stride = c.a_scale_stride; args.w_scales[0] = (const uint8_t*)c.scales;
  args.bias = c.bias; args.residual = c.residual; args.error = g_error_dev; args.T = (int)c.T; args.N = c.N; args.K = c.K;
  args.n_blocks = (c.N + TILE_N - 1) / TILE_N; args.act = c.act; args.out_bf16 = c.out_dtype == AYK_DTYPE_BF16;
  if (!takes_few<false>(args.T, args.N, args.K, ayk_sm_count())) return launch_many<false>(c.codes, c.codes, c.a, c.a_stride, args, "ayk_linear4", c.stream);
  const int bt = c.T <= 16 ? 16 : c.T <= 32 ? 32 : 64;
  CUtensorMap mw, ma;
  if (encode_weight(&mw, c.codes, args.n_blocks * TILE_N, c.K, TILE_N) != 0 || encode_rows(&ma, c.a, c.T, c.K, c.a_stride, bt) != 0) return -1;
  switch (bt) {
    case 16: return launch_few<16, false>(mw, mw, ma, args, "ayk_linear4", c.stream);
    case 32: return launch_few<32, false>(mw, mw, ma, args, "ayk_linear4", c.stream);
    default: return launch_few<64, false>(mw, mw, ma, args, "ayk_linear4", c.stream);
  }
}

// out [T, N] e4m3 and out_scales (rows out_scale_stride bytes apart) of act(a gate^T) * (a up^T).
struct GatedLinear4Call {
  void *out, *out_scales;
  long long out_scale_stride;
  const void *a, *a_scales;
  long long a_stride, a_scale_stride;
  const void *gate_codes, *gate_scales, *up_codes, *up_scales;
  long long T;
  int N, K, act;
  cudaStream_t stream;
};
AYK_EXPORT int ayk_gated_linear4(const GatedLinear4Call* call) {
  const GatedLinear4Call c = *call;
  if (check("ayk_gated_linear4", c.a, c.a_stride, c.a_scales, c.a_scale_stride, c.T, c.N, c.K, c.act) != 0) return -1;
  AYK_REQUIRE(c.N % MX_BLOCK == 0, "ayk_gated_linear4: a row of %d is not whole blocks of %d", c.N, MX_BLOCK);
  AYK_REQUIRE((uintptr_t)c.out % 32 == 0, "ayk_gated_linear4: codes must lie on 32-byte boundaries");
  if (c.T == 0) return 0;
  if (setup() != 0) return -1;
  Args args{};
  args.C = c.out; args.out_scales = (uint8_t*)c.out_scales; args.out_scale_stride = c.out_scale_stride;
  args.a_scales = (const uint8_t*)c.a_scales; args.a_scale_stride = c.a_scale_stride;
  args.w_scales[0] = (const uint8_t*)c.gate_scales; args.w_scales[1] = (const uint8_t*)c.up_scales; args.error = g_error_dev;
  args.T = (int)c.T; args.N = c.N; args.K = c.K; args.n_blocks = (c.N + TILE_N - 1) / TILE_N; args.act = c.act;
  if (!takes_few<true>(args.T, args.N, args.K, ayk_sm_count())) return launch_many<true>(c.gate_codes, c.up_codes, c.a, c.a_stride, args, "ayk_gated_linear4", c.stream);
  const int bt = c.T <= 16 ? 16 : c.T <= 32 ? 32 : 64;
  CUtensorMap mg, mu, ma;
  if (encode_weight(&mg, c.gate_codes, args.n_blocks * TILE_N, c.K, TILE_N) != 0 || encode_weight(&mu, c.up_codes, args.n_blocks * TILE_N, c.K, TILE_N) != 0 ||
      encode_rows(&ma, c.a, c.T, c.K, c.a_stride, bt) != 0)
    return -1;
  switch (bt) {
    case 16: return launch_few<16, true>(mg, mu, ma, args, "ayk_gated_linear4", c.stream);
    case 32: return launch_few<32, true>(mg, mu, ma, args, "ayk_gated_linear4", c.stream);
    default: return launch_few<64, true>(mg, mu, ma, args, "ayk_gated_linear4", c.stream);
  }
}
