// Rows in 8 bits (microscale.cuh) from rows in 32 or 16: as they are, or as the root-mean-square norm of the residual
// stream, which takes a sublayer's result on the way:
//
//   x += y;  h = x / sqrt(mean(x^2) + eps) * w;  per block of 32 columns: scale 2^e, codes e4m3(h / 2^e)
//
// The sum of squares, the norm and the block's scale are 32-bit; the code is the one rounding.
#include "microscale.cuh"

namespace {

constexpr int THREADS = 256;

// One block per row; a warp takes 32 columns at a time, a lane one of them.
template <typename X, typename Y, bool NORM>
__global__ void __launch_bounds__(THREADS)
rows8_kernel(uint8_t* __restrict__ out, uint8_t* scales, long long scale_stride, X* x, long long x_stride, const Y* y,
             long long y_stride, const float* __restrict__ w, int K, float eps) {
  __shared__ float red[THREADS / 32];
  pdl_trigger();
  pdl_wait();
  X* row = x + (size_t)blockIdx.x * x_stride;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float inv = 1.f;
  if constexpr (NORM) {
    float s = 0.f;
    for (int k = threadIdx.x; k < K; k += THREADS) {
      float v = to_float<X>(row[k]);
      if (y) {
        v += to_float<Y>(y[(size_t)blockIdx.x * y_stride + k]);
        row[k] = from_float<X>(v);
      }
      s = fmaf(v, v, s);
    }
    s = warp_sum(s);
    if (lane == 0) red[warp] = s;
    __syncthreads();
    s = 0.f;
    for (int i = 0; i < THREADS / 32; ++i) s += red[i];
    inv = 1.0f / sqrtf(s / (float)K + eps);
  }
  for (int b = warp; b < K / MX_BLOCK; b += THREADS / 32) {
    const int k = b * MX_BLOCK + lane;
    float v = to_float<X>(row[k]);
    if constexpr (NORM) v *= inv * w[k];
    const uint32_t code = mx_scale_code(__reduce_max_sync(0xffffffffu, magnitude_bits(v)));
    out[(size_t)blockIdx.x * K + k] = (uint8_t)e4m3_pair(v * mx_inverse(code), 0.f);
    if (lane == 0) scales[(size_t)blockIdx.x * scale_stride + b] = (uint8_t)code;
  }
}

}  // namespace

// codes [T, K] and scales (rows `scale_stride` bytes apart) of x [T, K], rows `x_stride` numbers apart.
AYK_EXPORT int ayk_rows8(void* codes, void* scales, long long scale_stride, const void* x, long long x_stride, long long T, int K, int dtype,
                         cudaStream_t stream) {
  AYK_REQUIRE(K > 0 && K % MX_BLOCK == 0, "ayk_rows8: a row of %d is not whole blocks of %d", K, MX_BLOCK);
  AYK_REQUIRE(dtype == AYK_DTYPE_F32 || dtype == AYK_DTYPE_BF16, "ayk_rows8: unknown dtype %d", dtype);
  AYK_REQUIRE(T >= 0 && T <= 0x7fffffff, "ayk_rows8: too many rows");
  if (T == 0) return 0;
  uint8_t *c = (uint8_t*)codes, *s = (uint8_t*)scales;
  if (dtype == AYK_DTYPE_F32)
    ayk_launch(rows8_kernel<float, float, false>, dim3((unsigned)T), dim3(THREADS), 0, stream, c, s, scale_stride, (float*)x, x_stride,
               (const float*)nullptr, 0ll, (const float*)nullptr, K, 0.f);
  else
    ayk_launch(rows8_kernel<__nv_bfloat16, float, false>, dim3((unsigned)T), dim3(THREADS), 0, stream, c, s, scale_stride, (__nv_bfloat16*)x,
               x_stride, (const float*)nullptr, 0ll, (const float*)nullptr, K, 0.f);
  return ayk_check_launch("ayk_rows8");
}

// x (float32) += y (float32 or bfloat16; null: nothing), and codes and scales of the norm of the new x.
AYK_EXPORT int ayk_rmsnorm_rows8(void* codes, void* scales, long long scale_stride, void* x, long long x_stride, const void* y, long long y_stride,
                                 int y_dtype, const float* w, long long T, int K, float eps, cudaStream_t stream) {
  AYK_REQUIRE(K > 0 && K % MX_BLOCK == 0, "ayk_rmsnorm_rows8: a row of %d is not whole blocks of %d", K, MX_BLOCK);
  AYK_REQUIRE(y_dtype == AYK_DTYPE_F32 || y_dtype == AYK_DTYPE_BF16, "ayk_rmsnorm_rows8: unknown dtype %d", y_dtype);
  AYK_REQUIRE(T >= 0 && T <= 0x7fffffff, "ayk_rmsnorm_rows8: too many rows");
  if (T == 0) return 0;
  uint8_t *c = (uint8_t*)codes, *s = (uint8_t*)scales;
  if (y_dtype == AYK_DTYPE_F32)
    ayk_launch(rows8_kernel<float, float, true>, dim3((unsigned)T), dim3(THREADS), 0, stream, c, s, scale_stride, (float*)x, x_stride,
               (const float*)y, y_stride, w, K, eps);
  else
    ayk_launch(rows8_kernel<float, __nv_bfloat16, true>, dim3((unsigned)T), dim3(THREADS), 0, stream, c, s, scale_stride, (float*)x, x_stride,
               (const __nv_bfloat16*)y, y_stride, w, K, eps);
  return ayk_check_launch("ayk_rmsnorm_rows8");
}
