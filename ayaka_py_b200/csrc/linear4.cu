// Products of 8-bit rows and 4-bit weights (microscale.cuh), both in blocks of 32 columns that share a power of two:
//
//   linear:  C[t, n] = act(sum_k a[t, k] W[n, k] + bias[n]) (+ residual[t, n])
//   gated:   rows in 8 bits of act(sum_k a[t, k] G[n, k]) * (sum_k a[t, k] U[n, k])
//
// Weights lie in tiles of 128 x 128 (a row of a tile: 64 bytes), their scales beside them as the tensor cores take them.
#include "microscale.cuh"

namespace {

constexpr int TILE = 128;
constexpr int FEATURES = 32, TOKENS = 16, THREADS = 256;

struct Matrix {
  const uint8_t* codes;
  const uint8_t* scales;
};

__device__ __forceinline__ float e2m1_float(uint32_t code) {
  const int m = code & 7;
  const float v = m < 2 ? 0.5f * (float)m : (1.0f + 0.5f * (float)(m & 1)) * (float)(1 << ((m >> 1) - 1));
  return code & 8 ? -v : v;
}

// A block of 32 features (the lanes) and 16 tokens (two to a warp); K goes by in tiles of 128 columns.
template <bool GATED>
__global__ void __launch_bounds__(THREADS)
linear4_kernel(void* C, uint8_t* out_scales, long long out_scale_stride, const uint8_t* a, long long a_stride, const uint8_t* a_scales,
               long long a_scale_stride, Matrix m0, Matrix m1, const float* __restrict__ bias, const float* residual, int T, int N, int K,
               int act, int out_bf16) {
  __shared__ float at[TOKENS][TILE + 1], wt[GATED ? 2 : 1][FEATURES][TILE + 1];
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n0 = blockIdx.x * FEATURES, t0 = blockIdx.y * TOKENS, n = n0 + lane;
  const int blocks_k = (K + TILE - 1) / TILE;
  float sum[GATED ? 2 : 1][2] = {};
  for (int kb = 0; kb < blocks_k; ++kb) {
    __syncthreads();
    for (int i = threadIdx.x; i < TOKENS * TILE; i += THREADS) {
      const int r = i / TILE, c = i % TILE, t = t0 + r, k = kb * TILE + c;
      at[r][c] = t < T && k < K ? e4m3_float(a[(size_t)t * a_stride + k]) * mx_scale(a_scales[(size_t)t * a_scale_stride + k / MX_BLOCK]) : 0.f;
    }
    for (int g = 0; g < (GATED ? 2 : 1); ++g) {
      const Matrix m = g ? m1 : m0;
      const size_t tile = (size_t)(n0 / TILE) * blocks_k + kb;
      for (int i = threadIdx.x; i < FEATURES * TILE / 2; i += THREADS) {
        const int r = i / (TILE / 2), c = i % (TILE / 2), tr = n0 % TILE + r;
        const uint32_t pair = m.codes[(tile * TILE + tr) * (TILE / 2) + c];
        const float s = mx_scale(m.scales[tile * 512 + (tr % 32) * 16 + (tr / 32) * 4 + c / 16]);
        wt[g][r][2 * c] = e2m1_float(pair & 15) * s;
        wt[g][r][2 * c + 1] = e2m1_float(pair >> 4) * s;
      }
    }
    __syncthreads();
    for (int c = 0; c < TILE; ++c)
#pragma unroll
      for (int g = 0; g < (GATED ? 2 : 1); ++g)
#pragma unroll
        for (int j = 0; j < 2; ++j) sum[g][j] = fmaf(at[warp * 2 + j][c], wt[g][lane][c], sum[g][j]);
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int t = t0 + warp * 2 + j;
    if (t >= T) continue;
    if constexpr (GATED) {
      const float v = apply_activation(sum[0][j], act) * sum[1][j];      // N is whole blocks of 32
      const uint32_t code = mx_scale_code(__reduce_max_sync(0xffffffffu, magnitude_bits(v)));
      ((uint8_t*)C)[(size_t)t * N + n] = (uint8_t)e4m3_pair(v * mx_inverse(code), 0.f);
      if (lane == 0) out_scales[(size_t)t * out_scale_stride + n0 / MX_BLOCK] = (uint8_t)code;
    } else if (n < N) {
      const size_t at_c = (size_t)t * N + n;
      const float v = apply_activation(sum[0][j] + (bias ? bias[n] : 0.f), act) + (residual ? residual[at_c] : 0.f);
      if (out_bf16) ((__nv_bfloat16*)C)[at_c] = __float2bfloat16_rn(v);
      else ((float*)C)[at_c] = v;
    }
  }
}

int check(const char* name, long long T, int N, int K, int act) {
  AYK_REQUIRE(N > 0 && K > 0 && K % MX_BLOCK == 0, "%s: a product of %d columns over rows of %d (whole blocks of %d)", name, N, K, MX_BLOCK);
  AYK_REQUIRE(T >= 0 && T <= 65535ll * TOKENS, "%s: too many rows (%lld)", name, T);
  AYK_REQUIRE(act >= AYK_ACT_NONE && act <= AYK_ACT_SILU, "%s: unknown activation %d", name, act);
  return 0;
}

}  // namespace

AYK_EXPORT int ayk_linear4(void* C, const void* a, long long a_stride, const void* a_scales, long long a_scale_stride, const void* codes,
                           const void* scales, const float* bias, const float* residual, long long T, int N, int K, int act, int out_dtype,
                           cudaStream_t stream) {
  if (check("ayk_linear4", T, N, K, act) != 0) return -1;
  AYK_REQUIRE(out_dtype == AYK_DTYPE_F32 || out_dtype == AYK_DTYPE_BF16, "ayk_linear4: unknown output dtype %d", out_dtype);
  if (T == 0) return 0;
  const Matrix m{(const uint8_t*)codes, (const uint8_t*)scales};
  ayk_launch(linear4_kernel<false>, dim3((N + FEATURES - 1) / FEATURES, (unsigned)((T + TOKENS - 1) / TOKENS)), dim3(THREADS), 0, stream, C,
             (uint8_t*)nullptr, 0ll, (const uint8_t*)a, a_stride, (const uint8_t*)a_scales, a_scale_stride, m, m, bias, residual, (int)T, N, K,
             act, out_dtype == AYK_DTYPE_BF16);
  return ayk_check_launch("ayk_linear4");
}

AYK_EXPORT int ayk_gated_linear4(void* out, void* out_scales, long long out_scale_stride, const void* a, long long a_stride, const void* a_scales,
                                 long long a_scale_stride, const void* gate_codes, const void* gate_scales, const void* up_codes,
                                 const void* up_scales, long long T, int N, int K, int act, cudaStream_t stream) {
  if (check("ayk_gated_linear4", T, N, K, act) != 0) return -1;
  AYK_REQUIRE(N % MX_BLOCK == 0, "ayk_gated_linear4: a row of %d is not whole blocks of %d", N, MX_BLOCK);
  if (T == 0) return 0;
  const Matrix g{(const uint8_t*)gate_codes, (const uint8_t*)gate_scales}, u{(const uint8_t*)up_codes, (const uint8_t*)up_scales};
  ayk_launch(linear4_kernel<true>, dim3(N / FEATURES, (unsigned)((T + TOKENS - 1) / TOKENS)), dim3(THREADS), 0, stream, out,
             (uint8_t*)out_scales, out_scale_stride, (const uint8_t*)a, a_stride, (const uint8_t*)a_scales, a_scale_stride, g, u,
             (const float*)nullptr, (const float*)nullptr, (int)T, N, K, act, 0);
  return ayk_check_launch("ayk_gated_linear4");
}
