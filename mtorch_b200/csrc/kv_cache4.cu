// Writing to and reading from the paged 4-bit key / value cache (attention over it:
// window_attention_split.cu).
//
// One thread per word of 8 channels, 8 neighbouring threads per group of 64 channels: the group's
// minimum and maximum come from three shuffles.  Bound by memory: the values are read once and 36
// bytes are written per 64 channels.
#include "runtime.h"

namespace mt {

// n / d for n < 2^31 by a multiplication (d >= 1; division by an invariant integer, Granlund and Montgomery 1994): m = floor(2^32 (2^s - d) / d) + 1 with s = ceil(log2 d)
struct FastDiv {
  uint32_t d, m, s;
  FastDiv() = default;
  explicit FastDiv(uint32_t div) : d(div), s(0) {
    while ((1ull << s) < div) ++s;
    m = (uint32_t)((((1ull << s) - div) << 32) / div + 1);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(m, n) + n) >> s; }
};

struct Cache4Params {
  FastDiv by_words, by_inner;  // D / 8; heads (append), threads' tokens (read)
  const int32_t* table;
  int64_t table_stride;
  int max_pages, page_shift, num_pages;
  int Hkv, D, T;
  int items;  // ceil(T / tokens of a thread) * Hkv * D / 8: threads of one sequence
  const int32_t* starts;
  int32_t* words[2];
  __half2* scales[2];  // (scale, zero)
  const void* in[2];
  void* out[2];
  int64_t st[2][4];
  bool vec;  // 8 channels are one aligned vector (16-bit types: 16 bytes, fp32: two of 16)
};

// Index of (token t of sequence b, head h) in units of heads' rows, -1 where it has no place.
__device__ __forceinline__ int64_t cache4_row(const Cache4Params& p, int64_t b, int h, int t) {
  const int64_t at = (int64_t)p.starts[b] + t;
  const int64_t pi = at >> p.page_shift;
  if (at < 0 || pi >= p.max_pages) return -1;
  const int page = p.table[b * p.table_stride + pi];
  if (page < 0 || page >= p.num_pages) return -1;
  const int slot = (int)(at & ((1 << p.page_shift) - 1));
  return (((int64_t)page * p.Hkv + h) << p.page_shift) + slot;
}

template <typename T>
struct Vec8 {
  alignas(16) T v[8];
};
template <typename T>
__device__ __forceinline__ Vec8<T> load8(const T* src, int64_t st, bool vec) {
  Vec8<T> x;
  if (vec) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(x.v)[i] = reinterpret_cast<const uint4*>(src)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x.v[i] = src[i * st];
  }
  return x;
}

constexpr int kAppendTokens = 1, kReadTokens = 4;  // consecutive tokens of a thread

// minimum and maximum that keep a NaN
__device__ __forceinline__ float min_nan(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// The code word and (scale, zero) of eight channels of a group of 64, whose other channels neighbouring lanes hold.
// A NaN in the group makes its scale and zero NaN, as does a group of one infinity only (max - min): it reads back as NaN.
template <typename T>
__device__ __forceinline__ uint32_t quantise8(const Vec8<T>& in, __half2& scale_zero) {
  float x[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = to_f32<T>(in.v[j]);
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int j = 1; j < 8; ++j) {
    lo = min_nan(lo, x[j]);
    hi = max_nan(hi, x[j]);
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  const __half zero = __float2half_rn(min_nan(max_nan(lo, -65504.f), 65504.f));
  const __half scale = __float2half_rn(min_nan(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f), 65504.f));
  scale_zero = __halves2half2(scale, zero);
  const float z = __half2float(zero), s = __half2float(scale);
  // code = clamp(rint((x - z) / s), 0, 15), ties to the even code.  The quotient by a multiplication is within 2^-22 of
  // itself of the divided one, so it rounds to the same code unless it is that near to a tie (within 2^-18 up to
  // 15.5); then the word's quotients are divided as the definition says.  1.5 * 2^23 added to a number rounds it to a
  // whole one, which stands in the sum's low bits.
  constexpr float kRound = 12582912.f;
  uint32_t word = 0;
  if (s > 0.f) {
    const float inv = 1.f / s;
    float tie = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float q = fminf(fmaxf(__fmul_rn(__fsub_rn(x[j], z), inv), 0.f), 15.f);
      const float r = __fadd_rn(q, kRound);
      tie = fmaxf(tie, fabsf(q - (r - kRound)));
      word |= (__float_as_uint(r) & 15u) << (4 * j);
    }
    if (tie > 0.5f - 3.8e-6f) {
      word = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float c = fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x[j], z), s)), 0.f), 15.f);
        word |= (uint32_t)c << (4 * j);
      }
    }
  }
  return word;
}

// A thread takes the same word of K and of V: the index arithmetic and the look into the table are shared.  18 MB of keys and
// values take 14, 16, 18 us with 1, 2, 4 tokens a thread: the arithmetic of a word (about 100 instructions)
// wants warps more than loads in flight.  Reading back, 8 us with 4 tokens, 10.5 with one.
template <typename T>
__global__ void __launch_bounds__(256) cache4_append_kernel(const Cache4Params p) {
  const uint32_t idx = blockIdx.x * 256u + threadIdx.x;
  const int64_t b = blockIdx.y;
  const uint32_t W = p.D / 8;
  const bool live = idx < (uint32_t)p.items;  // whole groups of 8 threads are live or not
  const uint32_t i = live ? idx : 0;
  const uint32_t r = p.by_words.div(i), w = i - r * W;
  const int tq = p.by_inner.div(r), h = r - (uint32_t)tq * p.Hkv, t0 = tq * kAppendTokens;
  Vec8<T> in[2][kAppendTokens];
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    const T* src = static_cast<const T*>(p.in[kv]) + b * p.st[kv][0] + h * p.st[kv][1] + t0 * p.st[kv][2] +
                   (int64_t)w * 8 * p.st[kv][3];
#pragma unroll
    for (int u = 0; u < kAppendTokens; ++u) {
      in[kv][u] = load8<T>(src, p.st[kv][3], p.vec);
      if (t0 + u + 1 < p.T) src += p.st[kv][2];  // (tokens past the last repeat it)
    }
  }
#pragma unroll
  for (int u = 0; u < kAppendTokens; ++u) {
    const int64_t row = live && t0 + u < p.T ? cache4_row(p, b, h, t0 + u) : -1;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      __half2 sz;
      const uint32_t word = quantise8<T>(in[kv][u], sz);
      if (row >= 0) {
        p.words[kv][row * W + w] = (int32_t)word;
        if ((w & 7) == 0) p.scales[kv][row * (W / 8) + (w >> 3)] = sz;
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256) cache4_read_kernel(const Cache4Params p) {
  const uint32_t idx = blockIdx.x * 256u + threadIdx.x;
  const int64_t b = blockIdx.y;
  if (idx >= (uint32_t)p.items) return;
  const uint32_t W = p.D / 8;
  const uint32_t r = p.by_words.div(idx), w = idx - r * W;
  const int h = p.by_inner.div(r), t0 = (r - (uint32_t)h * p.by_inner.d) * kReadTokens;
  uint32_t word[2][kReadTokens];
  __half2 sz[2][kReadTokens];
#pragma unroll
  for (int u = 0; u < kReadTokens; ++u) {
    const int64_t row = t0 + u < p.T ? cache4_row(p, b, h, t0 + u) : -1;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      word[kv][u] = row >= 0 ? (uint32_t)p.words[kv][row * W + w] : 0u;
      sz[kv][u] = row >= 0 ? p.scales[kv][row * (W / 8) + (w >> 3)] : __half2(__ushort_as_half(0), __ushort_as_half(0));
    }
  }
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    T* dst = static_cast<T*>(p.out[kv]) + b * p.st[kv][0] + h * p.st[kv][1] + t0 * p.st[kv][2] +
             (int64_t)w * 8 * p.st[kv][3];
#pragma unroll
    for (int u = 0; u < kReadTokens; ++u) {
      if (t0 + u >= p.T) break;
      const float2 f = __half22float2(sz[kv][u]);
      Vec8<T> o;
#pragma unroll
      for (int j = 0; j < 8; ++j)  // 2^23 | code as a number, minus 2^23: the code
        o.v[j] = from_f32<T>(fmaf(__uint_as_float(0x4b000000u | ((word[kv][u] >> (4 * j)) & 15u)) - 8388608.f, f.x, f.y));
      if (p.vec) {
#pragma unroll
        for (int j = 0; j < (int)sizeof(T) / 2; ++j)
          reinterpret_cast<uint4*>(dst)[j] = reinterpret_cast<const uint4*>(o.v)[j];
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) dst[j * p.st[kv][3]] = o.v[j];
      }
      dst += p.st[kv][2];
    }
  }
}

int validate_kv_cache4(const mt_kv_cache4& c) {
  if (c.num_pages < 0 || c.num_pages > INT32_MAX || c.Hkv <= 0 || c.Hkv > 65535)
    return fail(MT_ERR_INVALID, "kv_cache4: bad sizes");
  if (c.page_size < 16 || c.page_size > 1024 || (c.page_size & (c.page_size - 1)))
    return fail(MT_ERR_INVALID, "kv_cache4: page_size %lld is not a power of two from 16 to 1024",
                (long long)c.page_size);
  if (c.D < 64 || c.D > 256 || c.D % 64)
    return fail(MT_ERR_INVALID, "kv_cache4: head dim %lld is not a multiple of 64 up to 256", (long long)c.D);
  if (c.num_pages && (!c.k_words || !c.k_scales || !c.v_words || !c.v_scales))
    return fail(MT_ERR_INVALID, "kv_cache4: null cache array");
  for (const void* a : {(const void*)c.k_words, (const void*)c.k_scales, (const void*)c.v_words,
                        (const void*)c.v_scales})
    if ((uintptr_t)a % 16) return fail(MT_ERR_INVALID, "kv_cache4: cache arrays have to be 16-byte aligned");
  return MT_OK;
}

static int cache4_params(Cache4Params& p, const mt_kv_cache4& c, const void* k, const int64_t* ks, const void* v,
                         const int64_t* vs, int dtype, int64_t B, int64_t T, const int32_t* table,
                         int64_t table_stride, int64_t max_pages, const int32_t* starts, int tokens, const char* what) {
  int rc = validate_kv_cache4(c);
  if (rc) return rc;
  if (dtype != MT_F32 && dtype != MT_BF16 && dtype != MT_F16) return fail(MT_ERR_UNSUPPORTED, "%s: dtype", what);
  if (B < 0 || T < 0 || T > INT32_MAX || max_pages < 0 || max_pages > INT32_MAX)
    return fail(MT_ERR_INVALID, "%s: bad sizes", what);
  if (B && T && (!k || !v || !starts || (max_pages && !table))) return fail(MT_ERR_INVALID, "%s: null operand", what);
  p.table = table; p.table_stride = table_stride; p.max_pages = (int)max_pages;
  p.page_shift = __builtin_ctzll((unsigned long long)c.page_size);
  p.num_pages = (int)c.num_pages;
  p.Hkv = (int)c.Hkv; p.D = (int)c.D; p.T = (int)T;
  if (T * c.Hkv > INT32_MAX / 64) return fail(MT_ERR_UNSUPPORTED, "%s: too many tokens", what);
  p.items = (int)((T + tokens - 1) / tokens * c.Hkv * (c.D / 8));
  p.starts = starts;
  p.by_words = FastDiv((uint32_t)(c.D / 8));
  p.words[0] = c.k_words; p.words[1] = c.v_words;
  p.scales[0] = static_cast<__half2*>(c.k_scales); p.scales[1] = static_cast<__half2*>(c.v_scales);
  const int es = dtype_size(dtype);
  p.vec = true;
  for (int i = 0; i < 2; ++i) {
    const int64_t* s = i ? vs : ks;
    for (int j = 0; j < 4; ++j) p.st[i][j] = s[j];
    p.vec = p.vec && s[3] == 1 && (uintptr_t)(i ? v : k) % 16 == 0;
    for (int j = 0; j < 3; ++j) p.vec = p.vec && (s[j] * es) % 16 == 0;
  }
  return MT_OK;
}

// Sequences stand in the grid's second axis, larger batches in several launches: the one from sequence b on.
constexpr int64_t kMaxGridY = 65535;
static dim3 cache4_grid(Cache4Params& p, int64_t b, int64_t B, const int32_t* table, const int32_t* starts) {
  p.table = table ? table + b * p.table_stride : nullptr;
  p.starts = starts + b;
  return dim3((unsigned)((p.items + 255) / 256), (unsigned)std::min(B - b, kMaxGridY));
}

int run_kv_cache4_append(const mt_kv_cache4& c, const void* k, const int64_t* ks, const void* v, const int64_t* vs,
                         int dtype, int64_t B, int64_t T, const int32_t* table, int64_t table_stride,
                         int64_t max_pages, const int32_t* starts, cudaStream_t st) {
  Cache4Params p{};
  int rc = cache4_params(p, c, k, ks, v, vs, dtype, B, T, table, table_stride, max_pages, starts, kAppendTokens,
                         "kv_cache4_append");
  if (rc || B == 0 || p.items == 0) return rc;
  p.by_inner = FastDiv((uint32_t)c.Hkv);
  const int64_t es = dtype_size(dtype);
  for (int64_t b = 0; b < B && !rc; b += kMaxGridY) {
    p.in[0] = static_cast<const char*>(k) + b * ks[0] * es;
    p.in[1] = static_cast<const char*>(v) + b * vs[0] * es;
    const dim3 grid = cache4_grid(p, b, B, table, starts);
    switch (dtype) {
      case MT_F32: cache4_append_kernel<float><<<grid, 256, 0, st>>>(p); break;
      case MT_BF16: cache4_append_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(p); break;
      default: cache4_append_kernel<__half><<<grid, 256, 0, st>>>(p); break;
    }
    rc = check_launch("kv_cache4_append");
  }
  return rc;
}

int run_kv_cache4_read(const mt_kv_cache4& c, void* k, const int64_t* ks, void* v, const int64_t* vs, int dtype,
                       int64_t B, int64_t T, const int32_t* table, int64_t table_stride, int64_t max_pages,
                       const int32_t* starts, cudaStream_t st) {
  Cache4Params p{};
  int rc = cache4_params(p, c, k, ks, v, vs, dtype, B, T, table, table_stride, max_pages, starts, kReadTokens,
                         "kv_cache4_read");
  if (rc || B == 0 || p.items == 0) return rc;
  p.by_inner = FastDiv((uint32_t)((T + kReadTokens - 1) / kReadTokens));
  const int64_t es = dtype_size(dtype);
  for (int64_t b = 0; b < B && !rc; b += kMaxGridY) {
    p.out[0] = static_cast<char*>(k) + b * ks[0] * es;
    p.out[1] = static_cast<char*>(v) + b * vs[0] * es;
    const dim3 grid = cache4_grid(p, b, B, table, starts);
    switch (dtype) {
      case MT_F32: cache4_read_kernel<float><<<grid, 256, 0, st>>>(p); break;
      case MT_BF16: cache4_read_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(p); break;
      default: cache4_read_kernel<__half><<<grid, 256, 0, st>>>(p); break;
    }
    rc = check_launch("kv_cache4_read");
  }
  return rc;
}

}  // namespace mt
