// Products of few rows with a weight held in 4 bits, and its packing.
//
// W[n, k] = scale[n, k / group] * (code - 8).  Words of 8 codes; in each block of 128 columns word w
// is stored at place (w % 4) * 4 + w / 4 (see mtorch_cuda.h).
#include "runtime.h"

namespace mt {

// place of word w in its block of 16 words, and back (the map is a 4 x 4 transpose)
__host__ __device__ __forceinline__ int w4_place(int w) { return (w & 3) * 4 + (w >> 2); }

struct Linear4Params {
  int M, N, K, Kp, group;
  const void* x; int64_t ldx;
  const uint32_t* words;
  const __nv_bfloat16* scales;
  const void* bias;
  void* y; int64_t ldy;
};

// One warp per (output column, 8 rows): lanes stride over the words of the weight's row.
template <typename T>
__global__ void __launch_bounds__(128) linear4_simple_kernel(const Linear4Params p) {
  const int n = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int m0 = blockIdx.y * 8;
  if (n >= p.N) return;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const T* x = static_cast<const T*>(p.x);
  for (int i = lane; i < p.Kp / 8; i += 32) {
    const int k0 = (i & ~15) * 8 + w4_place(i & 15) * 8;
    const uint32_t word = p.words[(int64_t)n * (p.Kp / 8) + i];
    const float s = __bfloat162float(p.scales[(int64_t)n * (p.Kp / p.group) + k0 / p.group]);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (k0 + j >= p.K) break;
      const float w = s * (float)((int)((word >> (4 * j)) & 15u) - 8);
#pragma unroll
      for (int m = 0; m < 8; ++m)
        if (m0 + m < p.M) acc[m] = fmaf(to_f32<T>(x[(int64_t)(m0 + m) * p.ldx + k0 + j]), w, acc[m]);
    }
  }
#pragma unroll
  for (int m = 0; m < 8; ++m) {
    const float v = warp_sum(acc[m]);
    if (lane == 0 && m0 + m < p.M) {
      const float b = p.bias ? to_f32<T>(static_cast<const T*>(p.bias)[n]) : 0.f;
      static_cast<T*>(p.y)[(int64_t)(m0 + m) * p.ldy + n] = from_f32<T>(v + b);
    }
  }
}

// One thread per word of 8 columns; the group's maximum over 4, 8 or 16 neighbouring threads.
template <typename T>
__global__ void __launch_bounds__(256) weight4_pack_kernel(int32_t* words, __nv_bfloat16* scales, const T* w,
                                                           int64_t ldw, int N, int K, int Kp, int group) {
  const int W = Kp / 8;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const bool live = idx < (int64_t)N * W;  // W is a multiple of 16: whole groups are live or not
  const int64_t n = live ? idx / W : 0;
  const int i = live ? (int)(idx - n * W) : 0;
  float x[8], top = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int k = i * 8 + j;
    x[j] = live && k < K ? to_f32<T>(w[n * ldw + k]) : 0.f;
    top = fmaxf(top, fabsf(x[j]));
  }
  for (int o = 1; o < group / 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (!live) return;
  const __nv_bfloat16 sb = __float2bfloat16_rn(__fmul_rn(top, 1.0f / 7.0f));
  const float s = __bfloat162float(sb);
  uint32_t word = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float c = s > 0.f ? fminf(fmaxf(rintf(__fdiv_rn(x[j], s)), -8.f), 7.f) : 0.f;
    word |= (uint32_t)((int)c + 8) << (4 * j);
  }
  words[n * W + (i & ~15) + w4_place(i & 15)] = (int32_t)word;
  if (i % (group / 8) == 0) scales[n * (Kp / group) + i * 8 / group] = sb;
}

template <typename T>
__global__ void __launch_bounds__(256) weight4_unpack_kernel(T* w, int64_t ldw, const uint32_t* words,
                                                             const __nv_bfloat16* scales, int N, int K, int Kp,
                                                             int group) {
  const int W = Kp / 8;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (idx >= (int64_t)N * W) return;
  const int64_t n = idx / W;
  const int i = (int)(idx - n * W);
  const uint32_t word = words[n * W + (i & ~15) + w4_place(i & 15)];
  const float s = __bfloat162float(scales[n * (Kp / group) + i * 8 / group]);
  T* dst = w + n * ldw + i * 8;
  alignas(16) T v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = from_f32<T>(s * (float)((int)((word >> (4 * j)) & 15u) - 8));
  if (i * 8 + 8 <= K && (reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
#pragma unroll
    for (int j = 0; j < (int)sizeof(T) / 2; ++j) reinterpret_cast<uint4*>(dst)[j] = reinterpret_cast<uint4*>(v)[j];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i * 8 + j < K) dst[j] = v[j];
  }
}

static int64_t w4_padded(int64_t K) { return (K + 127) / 128 * 128; }

static int w4_check(int64_t N, int64_t K, int64_t group, int dtype, const char* what) {
  if (N < 0 || K < 0 || N > INT32_MAX || K > INT32_MAX - 128) return fail(MT_ERR_INVALID, "%s: bad sizes", what);
  if (group != 32 && group != 64 && group != 128)
    return fail(MT_ERR_INVALID, "%s: group %lld (32, 64 or 128)", what, (long long)group);
  if (dtype != MT_F32 && dtype != MT_BF16 && dtype != MT_F16) return fail(MT_ERR_UNSUPPORTED, "%s: dtype", what);
  if (N * (w4_padded(K) / 8) > (int64_t)INT32_MAX * 256) return fail(MT_ERR_UNSUPPORTED, "%s: weight too large", what);
  return MT_OK;
}

size_t linear_weight4_workspace(const mt_linear_weight4_desc&) { return 0; }

int run_linear_weight4(const mt_linear_weight4_desc& d, void*, size_t, cudaStream_t st) {
  int rc = w4_check(d.N, d.K, d.group, d.dtype, "linear_weight4");
  if (rc) return rc;
  if (d.M < 0 || d.M > INT32_MAX || d.ldx < 0 || d.ldy < 0) return fail(MT_ERR_INVALID, "linear_weight4: bad sizes");
  if (d.M == 0 || d.N == 0) return MT_OK;
  if (!d.y || (d.K && (!d.x || !d.words || !d.scales))) return fail(MT_ERR_INVALID, "linear_weight4: null operand");
  if ((uintptr_t)d.words % 16) return fail(MT_ERR_INVALID, "linear_weight4: words have to be 16-byte aligned");
  Linear4Params p{};
  p.M = (int)d.M; p.N = (int)d.N; p.K = (int)d.K; p.Kp = (int)w4_padded(d.K); p.group = (int)d.group;
  p.x = d.x; p.ldx = d.ldx;
  p.words = reinterpret_cast<const uint32_t*>(d.words);
  p.scales = static_cast<const __nv_bfloat16*>(d.scales);
  p.bias = d.bias; p.y = d.y; p.ldy = d.ldy;
  if ((d.M + 7) / 8 > 65535) return fail(MT_ERR_UNSUPPORTED, "linear_weight4: too many rows");
  dim3 grid((unsigned)((d.N + 3) / 4), (unsigned)((d.M + 7) / 8));
  switch (d.dtype) {
    case MT_F32: linear4_simple_kernel<float><<<grid, 128, 0, st>>>(p); break;
    case MT_BF16: linear4_simple_kernel<__nv_bfloat16><<<grid, 128, 0, st>>>(p); break;
    default: linear4_simple_kernel<__half><<<grid, 128, 0, st>>>(p); break;
  }
  return check_launch("linear_weight4");
}

int run_weight4_pack(int32_t* words, void* scales, const void* w, int dtype, int64_t ldw, int64_t N, int64_t K,
                     int64_t group, cudaStream_t st) {
  int rc = w4_check(N, K, group, dtype, "weight4_pack");
  if (rc) return rc;
  if (N == 0 || K == 0) return MT_OK;
  if (!words || !scales || !w) return fail(MT_ERR_INVALID, "weight4_pack: null operand");
  const int64_t Kp = w4_padded(K);
  const unsigned grid = (unsigned)((N * (Kp / 8) + 255) / 256);
  auto* sc = static_cast<__nv_bfloat16*>(scales);
  switch (dtype) {
    case MT_F32:
      weight4_pack_kernel<float><<<grid, 256, 0, st>>>(words, sc, static_cast<const float*>(w), ldw, (int)N, (int)K,
                                                       (int)Kp, (int)group);
      break;
    case MT_BF16:
      weight4_pack_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(words, sc, static_cast<const __nv_bfloat16*>(w), ldw,
                                                               (int)N, (int)K, (int)Kp, (int)group);
      break;
    default:
      weight4_pack_kernel<__half><<<grid, 256, 0, st>>>(words, sc, static_cast<const __half*>(w), ldw, (int)N, (int)K,
                                                        (int)Kp, (int)group);
  }
  return check_launch("weight4_pack");
}

int run_weight4_unpack(void* w, int dtype, int64_t ldw, const int32_t* words, const void* scales, int64_t N, int64_t K,
                       int64_t group, cudaStream_t st) {
  int rc = w4_check(N, K, group, dtype, "weight4_unpack");
  if (rc) return rc;
  if (N == 0 || K == 0) return MT_OK;
  if (!words || !scales || !w) return fail(MT_ERR_INVALID, "weight4_unpack: null operand");
  const int64_t Kp = w4_padded(K);
  const unsigned grid = (unsigned)((N * (Kp / 8) + 255) / 256);
  const auto* wd = reinterpret_cast<const uint32_t*>(words);
  const auto* sc = static_cast<const __nv_bfloat16*>(scales);
  switch (dtype) {
    case MT_F32:
      weight4_unpack_kernel<float><<<grid, 256, 0, st>>>(static_cast<float*>(w), ldw, wd, sc, (int)N, (int)K, (int)Kp,
                                                         (int)group);
      break;
    case MT_BF16:
      weight4_unpack_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(static_cast<__nv_bfloat16*>(w), ldw, wd, sc, (int)N,
                                                                 (int)K, (int)Kp, (int)group);
      break;
    default:
      weight4_unpack_kernel<__half><<<grid, 256, 0, st>>>(static_cast<__half*>(w), ldw, wd, sc, (int)N, (int)K,
                                                          (int)Kp, (int)group);
  }
  return check_launch("weight4_unpack");
}

}  // namespace mt
