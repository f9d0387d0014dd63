// Rows in 8 bits (microscale.cuh) from rows in 32 or 16: as they are, or as the root-mean-square norm of the residual
// stream, which takes a sublayer's result on the way:
//
//   x += y;  h = x / sqrt(mean(x^2) + eps) * w;  per block of 32 columns: scale 2^e, codes e4m3(h / 2^e)
//
// The sum of squares, the norm and the block's scale are 32-bit; the code is the one rounding.
//
// Bound by memory (norm of 8192 x 4096 with a bfloat16 y, 370 MB: 56.9 us, 6.5 TB/s) or, for few rows, by the way of one launch (1 x 768 1.6 us,
// 8 x 1600 rows 1.0): every number is read once and kept in registers between the sum and the codes.  A thread holds runs of eight
// numbers, four neighbouring threads a block; a row's threads make its sum of squares through shuffles and one exchange.
#include "microscale.cuh"

namespace {

constexpr int RUN = 8;

// `pieces`: of 32 bytes (2), of 16 (1) or number by number (0), as the rows lie.  A float32 run in one piece: 62.0 -> 56.9 us for the norm
// of 8192 x 4096 over three inputs in turn (5.97 -> 6.50 TB/s).
__device__ __forceinline__ void load_run(const float* p, int pieces, float (&v)[RUN]) {
  if (pieces == 2) {
    asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]) : "l"(p) : "memory");
  } else if (pieces == 1) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int j = 0; j < RUN; ++j) v[j] = p[j];
  }
}
__device__ __forceinline__ void load_run(const __nv_bfloat16* p, int pieces, float (&v)[RUN]) {
  if (pieces) {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = __uint_as_float(w[j] << 16);
      v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int j = 0; j < RUN; ++j) v[j] = __bfloat162float(p[j]);
  }
}
__device__ __forceinline__ void store_run(float* p, int pieces, const float (&v)[RUN]) {
  if (pieces == 2) {
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]) : "memory");
  } else if (pieces == 1) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
#pragma unroll
    for (int j = 0; j < RUN; ++j) p[j] = v[j];
  }
}

// Run i of a row (`there`: it exists) to its codes and, with its three neighbours, its scale.  Whole warps.
__device__ __forceinline__ void quantise_run(uint8_t* codes, uint8_t* scales, int i, bool there, const float (&v)[RUN]) {
  uint32_t largest = 0u;
#pragma unroll
  for (int j = 0; j < RUN; ++j) largest = max(largest, magnitude_bits(v[j]));
  largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
  largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
  const uint32_t code = mx_scale_code(largest);
  const float inverse = mx_inverse(code);
  if (there) {
    uint2 p;
    p.x = e4m3_pair(v[0] * inverse, v[1] * inverse) | (e4m3_pair(v[2] * inverse, v[3] * inverse) << 16);
    p.y = e4m3_pair(v[4] * inverse, v[5] * inverse) | (e4m3_pair(v[6] * inverse, v[7] * inverse) << 16);
    *reinterpret_cast<uint2*>(codes + (size_t)RUN * i) = p;
    if ((i & 3) == 0) scales[i >> 2] = (uint8_t)code;
  }
}

// A row's threads are blockDim.x, whole warps; blockDim.y rows to a block (several only of one warp each).  ITEMS runs to a
// thread, kept in registers; 0: a row too long for that, whose x is read a second time.
template <typename X, typename Y, bool NORM, int ITEMS>
__global__ void rows8_kernel(uint8_t* codes, uint8_t* scales, long long scale_stride, const X* x_in, float* x_out, long long x_stride, const Y* y,
                             long long y_stride, const float* __restrict__ w, long long rows, int K, float eps, int x_pieces, int y_pieces, int w_pieces) {
  __shared__ float red[32];
  if (gridDim.x <= AYK_FEW_BLOCKS) pdl_trigger();
  const long long r = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  const bool mine = r < rows;                  // whole warps: a row has its own
  const int runs = K / RUN, threads = blockDim.x;
  const X* row = x_in + (mine ? r : 0) * x_stride;
  const Y* add = y ? y + (mine ? r : 0) * y_stride : nullptr;
  codes += (mine ? r : 0) * K;
  scales += (mine ? r : 0) * scale_stride;
  pdl_wait();

  // eight numbers of the row, which takes y's on the way
  auto fetch = [&](int i, float (&v)[RUN]) {
    load_run(row + RUN * i, x_pieces, v);
    if (NORM && add) {
      float u[RUN];
      load_run(add + RUN * i, y_pieces, u);
#pragma unroll
      for (int j = 0; j < RUN; ++j) v[j] += u[j];
      store_run(x_out + r * x_stride + RUN * i, x_pieces, v);
    }
  };
  auto total = [&](float s) {
    s = warp_sum(s);
    if (threads > 32) {
      if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
      __syncthreads();
      s = 0.f;
      for (int i = 0; i < threads / 32; ++i) s += red[i];
    }
    return s;
  };
  auto norm_run = [&](int i, float inv, float (&v)[RUN]) {
    float g[RUN];
    load_run(w + RUN * i, w_pieces, g);
#pragma unroll
    for (int j = 0; j < RUN; ++j) v[j] = v[j] * inv * g[j];
  };

  if constexpr (ITEMS > 0) {
    float v[ITEMS][RUN];
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      const int i = threadIdx.x + k * threads;
#pragma unroll
      for (int j = 0; j < RUN; ++j) v[k][j] = 0.f;
      if (mine && i < runs) fetch(i, v[k]);
    }
    float inv = 1.f;
    if constexpr (NORM) {
#pragma unroll
      for (int k = 0; k < ITEMS; ++k)
#pragma unroll
        for (int j = 0; j < RUN; ++j) s = fmaf(v[k][j], v[k][j], s);
      inv = 1.0f / sqrtf(total(s) / (float)K + eps);
    }
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      const int i = threadIdx.x + k * threads;
      const bool there = mine && i < runs;
      if (NORM && there) norm_run(i, inv, v[k]);
      quantise_run(codes, scales, i, there, v[k]);
    }
  } else {
    float inv = 1.f;
    if constexpr (NORM) {
      float s = 0.f;
      for (int i = threadIdx.x; i < runs; i += threads) {
        float v[RUN];
        fetch(i, v);
#pragma unroll
        for (int j = 0; j < RUN; ++j) s = fmaf(v[j], v[j], s);
      }
      inv = 1.0f / sqrtf(total(s) / (float)K + eps);
    }
    for (int first = 0; first < runs; first += threads) {
      const int i = first + threadIdx.x;
      float v[RUN] = {};
      if (i < runs) {
        load_run(row + RUN * i, x_pieces, v);               // this thread's own stores, where the row was changed
        if constexpr (NORM) norm_run(i, inv, v);
      }
      quantise_run(codes, scales, i, i < runs, v);
    }
  }
}

constexpr int MOST_THREADS = 512, MOST_ITEMS = 4;

template <typename X, typename Y, bool NORM>
int launch(const char* name, uint8_t* codes, uint8_t* scales, long long scale_stride, const X* x, long long x_stride, const Y* y, long long y_stride,
           const float* w, long long T, int K, float eps, cudaStream_t stream) {
  AYK_REQUIRE(K > 0 && K % MX_BLOCK == 0, "%s: a row of %d is not whole blocks of %d", name, K, MX_BLOCK);
  AYK_REQUIRE(T >= 0 && T <= 0x7fffffff, "%s: too many rows (%lld)", name, T);
  AYK_REQUIRE((uintptr_t)codes % 16 == 0, "%s: codes must lie on 16-byte boundaries", name);
  if (T == 0) return 0;
  auto pieces = [](const void* p, long long stride, size_t size) {
    const uintptr_t bits = (uintptr_t)p | (uintptr_t)(stride * (long long)size);
    return bits % 32 == 0 ? 2 : bits % 16 == 0 ? 1 : 0;
  };
  // Few rows: as few runs to a thread as MOST_THREADS allow, for a row is a chain of loads, a sum and stores.  Many rows: 48 bytes of
  // loads under way to a thread at least (8192 x 4096, us with one, two, four runs to a thread: bfloat16 rows 21.8, 17.9, 16.4, norm
  // alone 44.7, 35.0, 34.8; norm with y, which has 48 a run, 56.9, 58.2 with one and two).
  const int runs = K / RUN, bytes = RUN * (int)(sizeof(X) + (y ? sizeof(Y) : 0));
  int items = 1;
  if (T >= 4 * ayk_sm_count())
    while (items < MOST_ITEMS && items * bytes < 48 && runs / (2 * items) >= 32) items *= 2;
  while (items <= MOST_ITEMS && (runs + items - 1) / items > MOST_THREADS) items *= 2;
  const int threads = items > MOST_ITEMS ? MOST_THREADS : ((runs + items - 1) / items + 31) / 32 * 32;
  const dim3 block(threads, threads == 32 ? 4 : 1);
  const dim3 grid((unsigned)((T + block.y - 1) / block.y));
  float* x_out = (float*)const_cast<X*>(x);
#define ROWS8_LAUNCH(ITEMS) \
  ayk_launch(rows8_kernel<X, Y, NORM, ITEMS>, grid, block, 0, stream, codes, scales, scale_stride, x, x_out, x_stride, y, y_stride, w, T, K, eps, pieces(x, x_stride, sizeof(X)), \
             pieces(y, y_stride, sizeof(Y)), pieces(w, 0, 4))
  if (items == 1) ROWS8_LAUNCH(1);
  else if (items == 2) ROWS8_LAUNCH(2);
  else if (items == 4) ROWS8_LAUNCH(4);
  else ROWS8_LAUNCH(0);
#undef ROWS8_LAUNCH
  return ayk_check_launch(name);
}

}  // namespace

// The arguments come as one block of memory (a call with a dozen of them from Python takes 0.5 us more).  Codes [T, K] and scales
// (rows `scale_stride` bytes apart) of x [T, K], rows `x_stride` numbers apart; with a norm's weight w: x (float32) += y (float32
// or bfloat16; null: nothing), and codes and scales of the norm of the new x.
struct Rows8Call {
  void *codes, *scales;
  long long scale_stride;
  void* x;
  long long x_stride;
  const void* y;
  long long y_stride;
  const float* w;
  long long T;
  int K, x_dtype, y_dtype;
  float eps;
  cudaStream_t stream;
};
AYK_EXPORT int ayk_rows8(const Rows8Call* call) {
  const Rows8Call c = *call;
  AYK_REQUIRE((c.x_dtype == AYK_DTYPE_F32 || c.x_dtype == AYK_DTYPE_BF16) && (c.y_dtype == AYK_DTYPE_F32 || c.y_dtype == AYK_DTYPE_BF16),
              "ayk_rows8: unknown dtypes %d, %d", c.x_dtype, c.y_dtype);
  AYK_REQUIRE(c.w ? c.x_dtype == AYK_DTYPE_F32 : c.y == nullptr, "ayk_rows8: the norm is of a float32 stream, and y is added to such a one");
  uint8_t *codes = (uint8_t*)c.codes, *scales = (uint8_t*)c.scales;
  const float* none = nullptr;
  if (!c.w) {
    if (c.x_dtype == AYK_DTYPE_F32) return launch<float, float, false>("ayk_rows8", codes, scales, c.scale_stride, (const float*)c.x, c.x_stride, none, 0, none, c.T, c.K, 0.f, c.stream);
    return launch<__nv_bfloat16, float, false>("ayk_rows8", codes, scales, c.scale_stride, (const __nv_bfloat16*)c.x, c.x_stride, none, 0, none, c.T, c.K, 0.f, c.stream);
  }
  if (c.y_dtype == AYK_DTYPE_F32)
    return launch<float, float, true>("ayk_rows8", codes, scales, c.scale_stride, (const float*)c.x, c.x_stride, (const float*)c.y, c.y_stride, c.w, c.T, c.K, c.eps, c.stream);
  return launch<float, __nv_bfloat16, true>("ayk_rows8", codes, scales, c.scale_stride, (const float*)c.x, c.x_stride, (const __nv_bfloat16*)c.y, c.y_stride, c.w, c.T, c.K,
                                            c.eps, c.stream);
}
