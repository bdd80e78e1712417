// Rotary positions with several axes on the heads of one or two tensors.
//
// Pair i of a head turns by angle = fp32(position[axis(i)] * frequency[i]):
//   (x, y) -> (x cos - y sin, x sin + y cos), with -angle for the inverse (= the gradient).
// Bound by memory: every element is read and written once; the sine and cosine of a (token, pair)
// are computed once per thread and used for all the heads that the thread walks through.
#include "runtime.h"

namespace mt {

struct RotaryParams {
  int64_t tokens;  // B * S
  int S, D, Hq, Hk, pairs;
  int axes, axis_end[MT_ROTARY_MAX_AXES];
  float sign;  // +1 forward, -1 inverse
  const int32_t* pos;
  int64_t pos_axis, pos_batch;
  const float* freq;
  const void* in[2];
  void* out[2];
  int64_t is[2][4], os[2][4];
  int heads_per_block;  // heads (q then k) that one blockIdx.y walks through
};

__device__ __forceinline__ void rotary_sincos(const RotaryParams& p, int64_t b, int s, int pair, float& sn, float& cs) {
  int a = 0;
  while (a + 1 < p.axes && pair >= p.axis_end[a]) ++a;
  const float at = (float)p.pos[a * p.pos_axis + b * p.pos_batch + s];
  sincosf(__fmul_rn(at, p.freq[pair]), &sn, &cs);
  sn *= p.sign;
}

// (x, y) turned; explicit roundings, the same for every kernel here
__device__ __forceinline__ void rotary_turn(float& x, float& y, float sn, float cs) {
  const float a = __fmaf_rn(x, cs, -__fmul_rn(y, sn));
  y = __fmaf_rn(x, sn, __fmul_rn(y, cs));
  x = a;
}

// One thread per (token, element or pair of elements), any strides.
template <typename T>
__global__ void __launch_bounds__(256) rotary_any_kernel(const RotaryParams p, const bool inter) {
  const int items = p.D - p.pairs;  // pairs, then the copied elements
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t tok = idx / items;
  const int c = (int)(idx - tok * items);
  if (tok >= p.tokens) return;
  const int64_t b = tok / p.S;
  const int s = (int)(tok - b * p.S);
  const bool pair = c < p.pairs;
  float sn = 0.f, cs = 1.f;
  if (pair) rotary_sincos(p, b, s, c, sn, cs);
  const int d0 = pair ? (inter ? 2 * c : c) : c + p.pairs;
  const int d1 = inter ? 2 * c + 1 : c + p.pairs;
  const int h0 = blockIdx.y * p.heads_per_block, h1 = min(p.Hq + p.Hk, h0 + p.heads_per_block);
#pragma unroll 4
  for (int h = h0; h < h1; ++h) {
    const int w = h < p.Hq ? 0 : 1;
    const int hh = w ? h - p.Hq : h;
    const T* src = static_cast<const T*>(p.in[w]) + b * p.is[w][0] + hh * p.is[w][1] + s * p.is[w][2];
    T* dst = static_cast<T*>(p.out[w]) + b * p.os[w][0] + hh * p.os[w][1] + s * p.os[w][2];
    if (pair) {
      float x = to_f32<T>(src[d0 * p.is[w][3]]), y = to_f32<T>(src[d1 * p.is[w][3]]);
      rotary_turn(x, y, sn, cs);
      dst[d0 * p.os[w][3]] = from_f32<T>(x);
      dst[d1 * p.os[w][3]] = from_f32<T>(y);
    } else {
      dst[d0 * p.os[w][3]] = src[d0 * p.is[w][3]];
    }
  }
}

template <int BYTES> struct RotaryVec;
template <> struct RotaryVec<16> { using type = uint4; };
template <> struct RotaryVec<8> { using type = uint2; };
template <> struct RotaryVec<4> { using type = uint32_t; };

// VEC elements (up to 16 bytes) at a time.  Split pairs: a thread holds channels c .. c + VEC - 1 and their partners
// `pairs` further on (pairs is a multiple of VEC), or VEC copied channels.  Interleaved pairs: a thread holds VEC
// channels, VEC / 2 pairs, those at and past `pairs` copied.  The angles of a (token, channel) are computed once
// for all the heads the thread walks through, four heads' loads ahead of their use.
template <typename T, int VEC, bool INTER>
__global__ void __launch_bounds__(256) rotary_vec_kernel(const RotaryParams p) {
  using V = typename RotaryVec<VEC * sizeof(T)>::type;
  constexpr int NP = INTER ? VEC / 2 : VEC;  // pairs of a thread
  constexpr int NV = INTER ? 1 : 2;          // vectors of a thread
  const int items = INTER ? p.D / VEC : (p.D - p.pairs) / VEC;
  const uint32_t idx = blockIdx.x * 256u + threadIdx.x;
  const uint32_t tok = idx / items;
  if (tok >= p.tokens) return;
  const int c = (idx - tok * items) * VEC;
  const int64_t b = tok / (uint32_t)p.S;
  const int s = tok - (uint32_t)b * p.S;
  // first channel of each vector; copied channels of split pairs follow the second halves
  const bool turns = INTER ? c / 2 < p.pairs : c < p.pairs;
  const int d0 = INTER || turns ? c : c + p.pairs, d1 = c + p.pairs;
  float sn[NP], cs[NP];
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    const int pair = INTER ? c / 2 + j : c + j;
    sn[j] = 0.f;
    cs[j] = 1.f;
    if (pair < p.pairs) rotary_sincos(p, b, s, pair, sn[j], cs[j]);
  }
  const int h0 = blockIdx.y * p.heads_per_block, h1 = min(p.Hq + p.Hk, h0 + p.heads_per_block);
  constexpr int U = 4;  // heads in flight
  for (int h = h0; h < h1; h += U) {
    V in[U][NV];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int hh = min(h + u, h1 - 1), w = hh < p.Hq ? 0 : 1;
      const T* src = static_cast<const T*>(p.in[w]) + b * p.is[w][0] + (w ? hh - p.Hq : hh) * p.is[w][1] + s * p.is[w][2];
      in[u][0] = *reinterpret_cast<const V*>(src + d0);
      if (!INTER && turns) in[u][NV - 1] = *reinterpret_cast<const V*>(src + d1);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (h + u >= h1) break;
      const int hh = h + u, w = hh < p.Hq ? 0 : 1;
      T* dst = static_cast<T*>(p.out[w]) + b * p.os[w][0] + (w ? hh - p.Hq : hh) * p.os[w][1] + s * p.os[w][2];
      if (turns) {
        T* e = reinterpret_cast<T*>(&in[u][0]);
        T* f = reinterpret_cast<T*>(&in[u][NV - 1]);
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          T& xr = INTER ? e[2 * j] : e[j];
          T& yr = INTER ? e[2 * j + 1] : f[j];
          float x = to_f32<T>(xr), y = to_f32<T>(yr);
          rotary_turn(x, y, sn[j], cs[j]);
          if (!INTER || c / 2 + j < p.pairs) {
            xr = from_f32<T>(x);
            yr = from_f32<T>(y);
          }
        }
        if (!INTER) *reinterpret_cast<V*>(dst + d1) = in[u][NV - 1];
      }
      *reinterpret_cast<V*>(dst + d0) = in[u][0];
    }
  }
}

// Largest vector (elements) that every row of the tensors allows; 1: none.
static int rotary_vec(const mt_rotary_desc& d) {
  const int es = dtype_size(d.dtype);
  for (int vec = 16 / es; vec > 1; vec /= 2) {
    bool ok = d.D % vec == 0 && (d.interleaved || d.pairs % vec == 0);
    for (int i = 0; i < 4; ++i) {
      const bool second = i & 1;
      if (second && !d.Hk) continue;
      if (!second && !d.Hq) continue;
      const void* base = i < 2 ? (second ? d.k : d.q) : (second ? d.k_out : d.q_out);
      const int64_t* st = i < 2 ? (second ? d.k_strides : d.q_strides) : (second ? d.k_out_strides : d.q_out_strides);
      ok = ok && st[3] == 1 && (uintptr_t)base % (vec * es) == 0 && st[0] % vec == 0 && st[1] % vec == 0 && st[2] % vec == 0;
    }
    if (ok) return vec;
  }
  return 1;
}

template <typename T, int VEC>
static void rotary_vec_launch(bool inter, dim3 grid, const RotaryParams& p, cudaStream_t st) {
  if (inter) rotary_vec_kernel<T, VEC, true><<<grid, 256, 0, st>>>(p);
  else rotary_vec_kernel<T, VEC, false><<<grid, 256, 0, st>>>(p);
}

template <typename T>
static int rotary_launch(const mt_rotary_desc& d, RotaryParams& p, cudaStream_t st) {
  const int heads = p.Hq + p.Hk;
  const int vec = p.tokens * p.D < UINT32_MAX - 256 ? rotary_vec(d) : 1;  // (the vector kernel counts in 32 bits)
  const int64_t items = p.tokens * (vec > 1 ? (d.interleaved ? p.D / vec : (p.D - p.pairs) / vec) : p.D - p.pairs);
  const int64_t blocks = (items + 255) / 256;
  if (blocks > INT32_MAX) return fail(MT_ERR_UNSUPPORTED, "rotary: too many elements");
  // heads are shared out over CTAs until the GPU is full: few tokens leave nothing else to share
  int64_t parts = std::min<int64_t>(heads, std::max<int64_t>(1, (12LL * num_sms() + blocks - 1) / blocks));
  p.heads_per_block = (int)((heads + parts - 1) / parts);
  dim3 grid((unsigned)blocks, (unsigned)((heads + p.heads_per_block - 1) / p.heads_per_block));
  const bool inter = d.interleaved != 0;
  if (vec > 1) {
    if (vec * (int)sizeof(T) == 16) rotary_vec_launch<T, 16 / sizeof(T)>(inter, grid, p, st);
    else if (vec * (int)sizeof(T) == 8) rotary_vec_launch<T, 8 / sizeof(T)>(inter, grid, p, st);
    else if constexpr (sizeof(T) == 2) rotary_vec_launch<T, 2>(inter, grid, p, st);
  } else {
    rotary_any_kernel<T><<<grid, 256, 0, st>>>(p, inter);
  }
  return check_launch("rotary");
}

int run_rotary(const mt_rotary_desc& d, cudaStream_t st) {
  if (d.B < 0 || d.S < 0 || d.D <= 0 || d.Hq < 0 || d.Hk < 0) return fail(MT_ERR_INVALID, "rotary: bad sizes");
  if (d.axes < 1 || d.axes > MT_ROTARY_MAX_AXES)
    return fail(MT_ERR_INVALID, "rotary: 1 to %d axes", MT_ROTARY_MAX_AXES);
  int64_t at = 0;
  for (int a = 0; a < d.axes; ++a) {
    if (d.axis_end[a] < at) return fail(MT_ERR_INVALID, "rotary: axis_end has to grow");
    at = d.axis_end[a];
  }
  if (at != d.pairs || d.pairs < 0 || 2 * d.pairs > d.D)
    return fail(MT_ERR_INVALID, "rotary: %lld pairs (axes end at %lld) for head dim %lld", (long long)d.pairs,
                (long long)at, (long long)d.D);
  if (d.D > (1 << 20) || d.S > INT32_MAX || d.Hq + d.Hk > 65535)
    return fail(MT_ERR_UNSUPPORTED, "rotary: sizes past the kernel's range");
  if (d.dtype != MT_F32 && d.dtype != MT_BF16 && d.dtype != MT_F16) return fail(MT_ERR_UNSUPPORTED, "rotary: dtype");
  if (d.B == 0 || d.S == 0 || d.Hq + d.Hk == 0) return MT_OK;
  if ((d.Hq && (!d.q || !d.q_out)) || (d.Hk && (!d.k || !d.k_out)) || (d.pairs && (!d.positions || !d.frequencies)))
    return fail(MT_ERR_INVALID, "rotary: null operand");
  RotaryParams p{};
  p.tokens = d.B * d.S;
  p.S = (int)d.S; p.D = (int)d.D; p.Hq = (int)d.Hq; p.Hk = (int)d.Hk; p.pairs = (int)d.pairs;
  p.axes = d.axes;
  for (int a = 0; a < d.axes; ++a) p.axis_end[a] = (int)d.axis_end[a];
  p.sign = d.inverse ? -1.f : 1.f;
  p.pos = d.positions; p.pos_axis = d.pos_axis_stride; p.pos_batch = d.pos_batch_stride;
  p.freq = d.frequencies;
  p.in[0] = d.q; p.in[1] = d.k; p.out[0] = d.q_out; p.out[1] = d.k_out;
  for (int i = 0; i < 4; ++i) {
    p.is[0][i] = d.q_strides[i]; p.is[1][i] = d.k_strides[i];
    p.os[0][i] = d.q_out_strides[i]; p.os[1][i] = d.k_out_strides[i];
  }
  switch (d.dtype) {
    case MT_F32: return rotary_launch<float>(d, p, st);
    case MT_BF16: return rotary_launch<__nv_bfloat16>(d, p, st);
    default: return rotary_launch<__half>(d, p, st);
  }
}

}  // namespace mt
