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

template <typename T>
static int rotary_launch(const mt_rotary_desc& d, RotaryParams& p, cudaStream_t st) {
  const int heads = p.Hq + p.Hk;
  const int64_t items = p.tokens * (p.D - p.pairs);
  const int64_t blocks = (items + 255) / 256;
  if (blocks > INT32_MAX) return fail(MT_ERR_UNSUPPORTED, "rotary: too many elements");
  int64_t parts = std::min<int64_t>(heads, std::max<int64_t>(1, (4LL * num_sms() + blocks - 1) / blocks));
  p.heads_per_block = (int)((heads + parts - 1) / parts);
  dim3 grid((unsigned)blocks, (unsigned)((heads + p.heads_per_block - 1) / p.heads_per_block));
  rotary_any_kernel<T><<<grid, 256, 0, st>>>(p, d.interleaved != 0);
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
