// Attention with a sliding window and sinks: the choice of the kernel (16-bit prompts: window_attention_sm100.cu; few queries
// over 16-bit keys and over the 4-bit cache: window_attention_split.cu), the kernels in fp32, and the join of split keys.
//
// One pass over the keys with the running maximum and sum of the softmax in fp32:
//   m' = max(m, s), l' = l 2^(m - m') + 2^(s - m'), o' = o 2^(m - m') + 2^(s - m') v.
// Only blocks of keys that a row of the tile can see are visited.  Few rows leave most of the GPU
// idle, so their keys are split over CTAs; the partial (m, l, o) go to the workspace and are joined
// by a second kernel.
#include <algorithm>
#include <cmath>

#include "window_attention.cuh"

namespace mt {

constexpr int kRowTile = 4;    // rows per CTA of attn_rows_kernel
constexpr int kRowBlock = 16;  // keys per step of a warp

enum { KV_ALIGNED = 0, KV_STRIDED = 1 };

// One CTA (4 warps) = kRowTile rows of one (batch entry, key head) and one share of their keys.
// A group of 8 lanes works on one key: a lane holds 4 channels of every 32.
template <typename T, int DCH, int KIND>
__global__ void __launch_bounds__(128) attn_rows_kernel(const AttnParams p) {
  constexpr int DP = DCH * 32;
  __shared__ float sq[kRowTile][DP];
  __shared__ float so[4][kRowTile][DP];
  __shared__ float2 sml[4][kRowTile];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l8 = lane & 7, grp = lane >> 3;
  const int bk = blockIdx.y, b = bk / p.Hkv, hk = bk % p.Hkv;
  const int r0 = blockIdx.z * kRowTile, nr = min(kRowTile, p.rows - r0);
  const SeqPos sp = seq_pos(p, b, false);

  for (int i = threadIdx.x; i < kRowTile * DP; i += 128) {
    const int r = i / DP, d = i % DP;
    float x = 0.f;
    if (r < nr && d < p.D) {
      const int qi = (r0 + r) / p.g, h = hk * p.g + (r0 + r) % p.g;
      x = to_f32<T>(static_cast<const T*>(p.q)[b * p.qs[0] + h * p.qs[1] + qi * p.qs[2] + d * p.qs[3]]);
    }
    sq[r][d] = x * p.scale_log2;
  }
  __syncthreads();

  RowKeys rk[kRowTile];
#pragma unroll
  for (int r = 0; r < kRowTile; ++r) rk[r] = row_keys(p, sp, sp.start + (r0 + min(r, nr - 1)) / p.g);
  const BlockList bl = block_list<kRowBlock>(p, sp, sp.start + r0 / p.g, sp.start + (r0 + nr - 1) / p.g);
  const int per = (bl.count + p.splits - 1) / p.splits;
  const int i0 = blockIdx.x * per, i1 = min(bl.count, i0 + per);

  float m[kRowTile], l[kRowTile], o[kRowTile][DCH][4];
#pragma unroll
  for (int r = 0; r < kRowTile; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int c = 0; c < DCH; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[r][c][j] = 0.f;
  }

  for (int i = i0 + warp; i < i1; i += 4) {
    const int k0 = bl.block(i) * kRowBlock;
#pragma unroll 1
    for (int it = 0; it < kRowBlock / 4; ++it) {
      const int kk = it * 4 + grp, key = k0 + kk;
      const bool live = key < sp.n;
      auto load = [&](int which, float (&x)[DCH][4]) {
#pragma unroll
        for (int c = 0; c < DCH; ++c) {
          const int d = c * 32 + l8 * 4;
#pragma unroll
          for (int j = 0; j < 4; ++j) x[c][j] = 0.f;
          if (!live || d >= p.D) continue;
          const int64_t* s = which ? p.vs : p.ks;
          const T* src = static_cast<const T*>(which ? p.v : p.k) + b * s[0] + hk * s[1] + key * s[2];
          if (KIND == KV_ALIGNED) {
            alignas(16) T raw[4];
            if (sizeof(T) == 4) *reinterpret_cast<uint4*>(raw) = *reinterpret_cast<const uint4*>(src + d);
            else *reinterpret_cast<uint2*>(raw) = *reinterpret_cast<const uint2*>(src + d);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[c][j] = to_f32<T>(raw[j]);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (d + j < p.D) x[c][j] = to_f32<T>(src[(d + j) * s[3]]);
          }
        }
      };
      float kf[DCH][4], vf[DCH][4];
      load(0, kf);
      load(1, vf);
#pragma unroll
      for (int r = 0; r < kRowTile; ++r) {
        if (r >= nr) break;
        float s = 0.f;
#pragma unroll
        for (int c = 0; c < DCH; ++c) {
          const float4 qv = *reinterpret_cast<const float4*>(&sq[r][c * 32 + l8 * 4]);
          s = fmaf(qv.x, kf[c][0], s);
          s = fmaf(qv.y, kf[c][1], s);
          s = fmaf(qv.z, kf[c][2], s);
          s = fmaf(qv.w, kf[c][3], s);
        }
#pragma unroll
        for (int x = 1; x < 8; x <<= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        if (!live || !rk[r].sees(key)) continue;
        // a score of -infinity weighs nothing, also as the first one; a NaN stays in m and makes the row's weights NaN
        const float mn = max_nan(m[r], s);
        const float corr = m[r] == -INFINITY ? 0.f : exp2f(m[r] - mn), e = s == -INFINITY ? 0.f : exp2f(s - mn);
        m[r] = mn;
        l[r] = fmaf(l[r], corr, e);
#pragma unroll
        for (int c = 0; c < DCH; ++c)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[r][c][j] = fmaf(o[r][c][j], corr, e * vf[c][j]);
      }
    }
  }

  // join the four key groups of the warp, then the four warps
#pragma unroll
  for (int r = 0; r < kRowTile; ++r) {
    float top = max_nan(m[r], __shfl_xor_sync(0xffffffffu, m[r], 8));
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 16));
    const float f = m[r] == -INFINITY ? 0.f : exp2f(m[r] - top);
    float ls = l[r] * f;
    ls += __shfl_xor_sync(0xffffffffu, ls, 8);
    ls += __shfl_xor_sync(0xffffffffu, ls, 16);
    if (lane == 0) sml[warp][r] = make_float2(top, ls);
#pragma unroll
    for (int c = 0; c < DCH; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float x = m[r] == -INFINITY ? 0.f : o[r][c][j] * f;
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        if (grp == 0) so[warp][r][c * 32 + l8 * 4 + j] = x;
      }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < nr * DP; i += 128) {
    const int r = i / DP, d = i % DP;
    if (d >= p.D) continue;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) top = max_nan(top, sml[w][r].x);
    float ls = 0.f, x = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w)
      if (sml[w][r].x != -INFINITY) {
        const float f = exp2f(sml[w][r].x - top);
        ls = fmaf(sml[w][r].y, f, ls);
        x = fmaf(so[w][r][d], f, x);
      }
    if (p.splits > 1) {
      const int64_t row = ((int64_t)blockIdx.x * p.B * p.Hkv + bk) * p.rows + r0 + r;
      p.part_o[row * p.D + d] = x;
      if (d == 0) p.part_ml[row] = make_float2(top, ls);
    } else {
      const int qi = (r0 + r) / p.g, h = hk * p.g + (r0 + r) % p.g;
      static_cast<T*>(p.o)[b * p.os[0] + h * p.os[1] + qi * p.os[2] + d * p.os[3]] =
          from_f32<T>(ls == 0.f ? 0.f : x / ls);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Many queries in fp32 (and 16-bit rows that the tensor-core kernel cannot map): tiles of 64 queries of a head by 64
// keys in shared memory, fp32 products on the FMA units.  A thread (ty, tx) of 16 x 16 holds 4 x 4 scores and
// 4 x (DP / 16) outputs; Q, K and P lie transposed, so that a step of a product is two 16-byte reads for 16 FMAs.
// Bound by the FMA units (128 a cycle and SM); a tile past the window, or past the sinks, is not visited.
constexpr int kTile = 64;

template <typename T, int DP>
__global__ void __launch_bounds__(256, DP <= 128 ? 2 : 1) attn_tile_kernel(const AttnParams p, const bool aligned) {
  extern __shared__ float4 tile_smem[];
  float* Qs = reinterpret_cast<float*>(tile_smem);  // [DP][64]
  float* Ks = Qs + DP * kTile;                      // [DP][64]
  float* Vs = Ks + DP * kTile;                      // [64][DP]
  float* Ps = Vs + DP * kTile;                      // [64 keys][64 queries]
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int bh = blockIdx.x, b = bh / p.H, h = bh % p.H, hk = h / p.g;
  const int q0 = (gridDim.y - 1 - blockIdx.y) * kTile, q1 = min(p.Sq, q0 + kTile) - 1;  // (the longest rows first)
  const SeqPos sp = seq_pos(p, b, false);
  const BlockList bl = block_list<kTile>(p, sp, sp.start + q0, sp.start + q1);
  const RowKeys ra = row_keys(p, sp, sp.start + q0), rz = row_keys(p, sp, sp.start + q1);

  // four channels of row `row` of a tensor; zeros where there are none
  auto load4 = [&](const void* base, const int64_t* st, int64_t head, int row, bool live, int d) -> float4 {
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    if (live && d < p.D) {
      const T* src = static_cast<const T*>(base) + b * st[0] + head * st[1] + row * st[2];
      if (aligned) {
        alignas(16) T raw[4];
        if (sizeof(T) == 4) *reinterpret_cast<uint4*>(raw) = *reinterpret_cast<const uint4*>(src + d);
        else *reinterpret_cast<uint2*>(raw) = *reinterpret_cast<const uint2*>(src + d);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = to_f32<T>(raw[j]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (d + j < p.D) x[j] = to_f32<T>(src[(d + j) * st[3]]);
      }
    }
    return make_float4(x[0], x[1], x[2], x[3]);
  };

  for (int i = tid; i < kTile * (DP / 4); i += 256) {
    const int r = i % kTile, d = i / kTile * 4;
    const float4 x = load4(p.q, p.qs, h, q0 + r, q0 + r < p.Sq, d);
    Qs[d * kTile + r] = x.x * p.scale_log2;
    Qs[(d + 1) * kTile + r] = x.y * p.scale_log2;
    Qs[(d + 2) * kTile + r] = x.z * p.scale_log2;
    Qs[(d + 3) * kTile + r] = x.w * p.scale_log2;
  }
  float m[4], l[4], o[4][DP / 16];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int j = 0; j < DP / 16; ++j) o[i][j] = 0.f;
  }
  for (int t = 0; t < bl.count; ++t) {
    const int k0 = bl.block(t) * kTile;
    __syncthreads();
    for (int i = tid; i < kTile * (DP / 4); i += 256) {
      const int r = i % kTile, d = i / kTile * 4;  // K: neighbouring threads take neighbouring keys
      const float4 x = load4(p.k, p.ks, hk, k0 + r, k0 + r < sp.n, d);
      Ks[d * kTile + r] = x.x;
      Ks[(d + 1) * kTile + r] = x.y;
      Ks[(d + 2) * kTile + r] = x.z;
      Ks[(d + 3) * kTile + r] = x.w;
      const int rv = i / (DP / 4), dv = i % (DP / 4) * 4;  // V: neighbouring channels
      *reinterpret_cast<float4*>(&Vs[rv * DP + dv]) = load4(p.v, p.vs, hk, k0 + rv, k0 + rv < sp.n, dv);
    }
    __syncthreads();
    float s[4][4] = {};
#pragma unroll 8
    for (int d = 0; d < DP; ++d) {
      const float4 q = *reinterpret_cast<const float4*>(&Qs[d * kTile + ty * 4]);
      const float4 k = *reinterpret_cast<const float4*>(&Ks[d * kTile + tx * 4]);
      const float qv[4] = {q.x, q.y, q.z, q.w}, kv[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = fmaf(qv[i], kv[j], s[i][j]);
    }
    if (!(k0 + kTile - 1 <= ra.hi && (k0 >= rz.lo || k0 + kTile - 1 < ra.sk))) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const RowKeys rk = row_keys(p, sp, sp.start + min(q0 + ty * 4 + i, q1));
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (!rk.sees(k0 + tx * 4 + j)) s[i][j] = -INFINITY;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float mx = fmaxf(fmaxf(s[i][0], s[i][1]), fmaxf(s[i][2], s[i][3]));
#pragma unroll
      for (int x = 1; x < 16; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
      mx = fmaxf(mx, m[i]);
      const float mu = mx == -INFINITY ? 0.f : mx, corr = exp2f(m[i] - mu);
      m[i] = mx;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = exp2f(s[i][j] - mu);
        sum += s[i][j];
      }
      l[i] = fmaf(l[i], corr, sum);  // of this thread's keys; joined at the end
#pragma unroll
      for (int j = 0; j < DP / 16; ++j) o[i][j] *= corr;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *reinterpret_cast<float4*>(&Ps[(tx * 4 + j) * kTile + ty * 4]) = make_float4(s[0][j], s[1][j], s[2][j], s[3][j]);
    __syncthreads();
#pragma unroll 4
    for (int k = 0; k < kTile; ++k) {
      const float4 pv = *reinterpret_cast<const float4*>(&Ps[k * kTile + ty * 4]);
      const float pr[4] = {pv.x, pv.y, pv.z, pv.w};
#pragma unroll
      for (int c = 0; c < DP / 64; ++c) {
        const float4 v = *reinterpret_cast<const float4*>(&Vs[k * DP + c * 64 + tx * 4]);
        const float vv[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[i][c * 4 + j] = fmaf(pr[i], vv[j], o[i][c * 4 + j]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], x);
    const int qi = q0 + ty * 4 + i;
    if (qi >= p.Sq) continue;
    const float inv = l[i] > 0.f ? 1.f / l[i] : 0.f;
    T* dst = static_cast<T*>(p.o) + b * p.os[0] + h * p.os[1] + qi * p.os[2];
#pragma unroll
    for (int c = 0; c < DP / 64; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int d = c * 64 + tx * 4 + j;
        if (d < p.D) dst[d * p.os[3]] = from_f32<T>(o[i][c * 4 + j] * inv);
      }
  }
}

// One CTA joins the shares of one row: groups of threads take shares in turn, a thread holds 4 channels (or
// single ones where D is no multiple of 4), so that all the reads of a row are in flight at once.
constexpr int kJoinThreads = 256;
constexpr int kMaxSplits = 512;

template <typename T>
__global__ void __launch_bounds__(kJoinThreads) attn_join_kernel(const AttnParams p) {
  __shared__ float w[kMaxSplits];
  __shared__ float red[kJoinThreads * 4];
  __shared__ float s_top[kJoinThreads / 32], s_sum[kJoinThreads / 32];
  // launched while the kernel before it still runs (see join_launch): wait for its results
  cudaGridDependencySynchronize();
  const int64_t total = (int64_t)p.B * p.Hkv * p.rows;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  float2 ml[kMaxSplits / kJoinThreads];
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kMaxSplits / kJoinThreads; ++i) {
    const int s = tid + i * kJoinThreads;
    ml[i] = s < p.splits ? p.part_ml[s * total + row] : make_float2(-INFINITY, 0.f);
    top = fmaxf(top, ml[i].x);
  }
  top = warp_max(top);
  if (lane == 0) s_top[warp] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kJoinThreads / 32; ++i) top = fmaxf(top, s_top[i]);
  float ls = 0.f;
#pragma unroll
  for (int i = 0; i < kMaxSplits / kJoinThreads; ++i) {
    const int s = tid + i * kJoinThreads;
    const float f = ml[i].x == -INFINITY ? 0.f : exp2f(ml[i].x - top);
    if (s < p.splits) w[s] = f;
    ls = fmaf(ml[i].y, f, ls);
  }
  ls = warp_sum(ls);
  if (lane == 0) s_sum[warp] = ls;
  __syncthreads();
  ls = 0.f;
#pragma unroll
  for (int i = 0; i < kJoinThreads / 32; ++i) ls += s_sum[i];

  const bool vec = p.D % 4 == 0;
  const int n = vec ? p.D / 4 : p.D, groups = max(1, kJoinThreads / n);
  const int g = tid / n, c = tid % n;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  if (g < groups) {
#pragma unroll 4
    for (int s = g; s < p.splits; s += groups) {
      const float f = w[s];
      if (f == 0.f) continue;  // an empty share wrote no o
      const float* src = p.part_o + (s * total + row) * p.D;
      if (vec) {
        const float4 v = reinterpret_cast<const float4*>(src)[c];
        x.x = fmaf(v.x, f, x.x);
        x.y = fmaf(v.y, f, x.y);
        x.z = fmaf(v.z, f, x.z);
        x.w = fmaf(v.w, f, x.w);
      } else {
        x.x = fmaf(src[c], f, x.x);
      }
    }
  }
  reinterpret_cast<float4*>(red)[tid] = x;
  __syncthreads();
  const int64_t bk = row / p.rows;
  const int r = (int)(row - bk * p.rows);
  const int b = (int)(bk / p.Hkv), hk = (int)(bk % p.Hkv);
  T* dst = static_cast<T*>(p.o) + b * p.os[0] + (hk * p.g + r % p.g) * p.os[1] + (r / p.g) * p.os[2];
  for (int d = tid; d < p.D; d += kJoinThreads) {
    const int at = vec ? d : d * 4, step = n * 4;
    float y = 0.f;
    for (int i = 0; i < groups; ++i) y += red[i * step + at];
    dst[d * p.os[3]] = from_f32<T>(ls == 0.f ? 0.f : y / ls);
  }
}

// ---------------------------------------------------------------------------------------------
// host

// Keys that one row can see at most.
static int64_t span_keys(int64_t Sk, int64_t Sq, int causal, int64_t window, int64_t sinks) {
  if (window <= 0) return Sk;
  return std::min(Sk, (causal ? window : 2 * window - 1) + Sq - 1 + sinks + 2 * kRowBlock);
}

// Shares of the keys: enough CTAs to fill the GPU a few times, each with at least 8 blocks of keys.  A step of few tokens (one
// tile of rows a key head) is cut finer, more rows pay more for the join.  fp32, us with 2, 4 and 8 CTAs an SM: one token of
// 8 sequences, 32 / 8 heads of 128, window 4096: 105, 115, 107 (floor 41); of 24 sequences, 16 heads of 64, 4096 keys: 233, 240,
// 193 (124); 2 / 8 heads, 30000 keys: 40, 37, 37; 32 queries of 4 x 16 heads, 500 keys, 4 and 8: 56, 60; 200 of 16 / 4 heads over
// 4000 keys, window 1000: 194, 211.
static int choose_splits(int64_t ctas, int64_t tiles, int64_t keys) {
  const int64_t want = ((tiles == 1 ? 8LL : 4LL) * num_sms() + ctas - 1) / ctas;
  const int64_t most = std::max<int64_t>(1, keys / (8 * kRowBlock));
  return (int)std::max<int64_t>(1, std::min<int64_t>(std::min(want, most), kMaxSplits));
}

static size_t part_bytes(int splits, int64_t rows, int64_t D) {
  if (splits <= 1) return 0;
  return align_up((size_t)splits * rows * sizeof(float2), 256) + (size_t)splits * rows * D * sizeof(float);
}

static int rows_splits(int64_t B, int64_t H, int64_t Hkv, int64_t Sq, int64_t Sk, int causal, int64_t window,
                       int64_t sinks) {
  const int64_t tiles = (Sq * (H / Hkv) + kRowTile - 1) / kRowTile;
  return choose_splits(B * Hkv * tiles, tiles, span_keys(Sk, Sq, causal, window, sinks));
}

// Rows of head dim channels are whole 16-byte vectors of a 16-bit type.
static bool aligned16(const void* base, const int64_t* s, int64_t D) {
  return s[3] == 1 && D % 8 == 0 && (uintptr_t)base % 16 == 0 && s[0] % 8 == 0 && s[1] % 8 == 0 && s[2] % 8 == 0;
}

static bool takes_split(const mt_window_attention_desc& d) {
  return d.dtype != MT_F32 && aligned16(d.k, d.k_strides, d.D) && aligned16(d.v, d.v_strides, d.D);
}

// The tensor-core kernel (tiles of 256 queries of a head) or the split kernel (which reads the keys anew for each 16 rows
// of a key head, but spreads them over the GPU)?  By the time that each takes: about 2 us per 128 keys and round of CTAs
// (a prompt of 8192 in 4 rounds of 18 tiles: 148 us) behind a start of 5 us, against 4 TB/s of keys and values
// (one token of 8 sequences: 131 MB in 32 us) behind 8 us.  Tiles and split keys: 33 queries of 2 heads over 4000 keys 60
// and 15 us; 100 of 8 heads over 1000 25 and 17; 300 of 16 heads over 300 10 and 29; 2048 of 16 heads 37 and 242.
static bool takes_sm100(const mt_window_attention_desc& d) {
  if (!window_sm100_takes(d)) return false;
  if (!takes_split(d)) return true;
  if (d.Sq <= 16) return false;  // a step of a few tokens: the start is what counts, and three tensor maps take the host longer
  const double rounds = std::ceil((double)(d.B * d.H * ((d.Sq + 255) / 256)) / num_sms());
  const double span = (double)span_keys(d.Sk, std::min<int64_t>(d.Sq, 256), d.causal, d.window, d.sinks);
  const int64_t rows = d.Sq * (d.H / d.Hkv);
  const double few = (double)span_keys(d.Sk, std::min(d.Sq, (16 + d.H / d.Hkv - 1) / (d.H / d.Hkv)), d.causal, d.window, d.sinks);
  const double tiles_us = 5.0 + rounds * std::ceil(span / 128) * 2.0;
  const double split_us = 8.0 + (double)(d.B * d.Hkv * ((rows + 15) / 16)) * few * d.D * 4.0 / 4e6;
  return tiles_us < split_us;
}

// fp32 (and what neither of the two takes): tiles of 64 queries from 24 queries of a head an SM on, else rows with the keys
// split.  Tiles and rows, us, by queries of all heads: 1200 (300 of 4 heads over 600 keys) 77 and 40; 2048 (32 of 4 x 16, 500)
// 79 and 56; 3200 (200 of 16, 4000, window 1000) 216 and 194; 3600 (150 of 24, 300) 42 and 56; 4000 (2000 of 2, window 256) 42
// and 49; 4160 (130 of 2 x 16, 1000) 154 and 161; 8704 (17 of 64 x 8, 1000, heads of 128) 631 and 667; 72000 (1500 of 3 x 16, 1500)
// 541 and 1704.
static bool takes_tiles(const mt_window_attention_desc& d) {
  return d.Sq > 16 && d.B * d.H * d.Sq >= 24 * num_sms();
}

static int window_splits(const mt_window_attention_desc& d) {
  if (takes_sm100(d)) return 1;
  if (takes_split(d))
    return split_count(d.B * d.Hkv, d.Sq * (d.H / d.Hkv), span_keys(d.Sk, d.Sq, d.causal, d.window, d.sinks));
  if (takes_tiles(d)) return 1;
  return rows_splits(d.B, d.H, d.Hkv, d.Sq, d.Sk, d.causal, d.window, d.sinks);
}

static int cache_splits(const mt_kv_cache4_attention_desc& d) {
  return split_count(d.B * d.cache.Hkv, d.Sq * (d.H / d.cache.Hkv),
                     span_keys(d.max_pages * d.cache.page_size, d.Sq, 1, d.window, d.sinks));
}

// The partial results are stored 16 bytes at a time.
static int check_workspace(const void* ws, size_t bytes, size_t need, const char* what) {
  if (!need) return MT_OK;
  if (!ws || bytes < need) return fail(MT_ERR_WORKSPACE, "%s: workspace too small", what);
  if ((uintptr_t)ws % 16) return fail(MT_ERR_INVALID, "%s: the workspace has to be 16-byte aligned", what);
  return MT_OK;
}

static void bind_workspace(AttnParams& p, void* ws) {
  const size_t rows = (size_t)p.B * p.Hkv * p.rows;
  p.part_ml = static_cast<float2*>(ws);
  p.part_o = reinterpret_cast<float*>(static_cast<char*>(ws) + align_up((size_t)p.splits * rows * sizeof(float2), 256));
}

template <typename T>
static int join_launch(const AttnParams& p, cudaStream_t st) {
  const int64_t rows = (int64_t)p.B * p.Hkv * p.rows;
  if (rows > INT32_MAX) return fail(MT_ERR_UNSUPPORTED, "window_attention: too many rows");
  // programmatic launch: the CTAs come up while the last shares are computed, which hides the launch
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)rows);
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = st;
  cudaLaunchAttribute at = {};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  int rc = cuda_check(cudaLaunchKernelEx(&cfg, attn_join_kernel<T>, p), "attention_join");
  return rc ? rc : check_launch("attention_join");
}

static int join(const AttnParams& p, int dtype, cudaStream_t st) {
  return dtype == MT_F16 ? join_launch<__half>(p, st) : join_launch<__nv_bfloat16>(p, st);
}

template <typename T, int KIND>
static int rows_launch(const AttnParams& p, cudaStream_t st) {
  const int64_t tiles = (p.rows + kRowTile - 1) / kRowTile;
  if ((int64_t)p.B * p.Hkv > 65535 || tiles > 65535)
    return fail(MT_ERR_UNSUPPORTED, "window_attention: batch * key heads or rows past the grid");
  dim3 grid((unsigned)p.splits, (unsigned)(p.B * p.Hkv), (unsigned)tiles);
  const int dch = (p.D + 31) / 32;
  if (dch <= 2) attn_rows_kernel<T, 2, KIND><<<grid, 128, 0, st>>>(p);
  else if (dch <= 4) attn_rows_kernel<T, 4, KIND><<<grid, 128, 0, st>>>(p);
  else attn_rows_kernel<T, 8, KIND><<<grid, 128, 0, st>>>(p);
  int rc = check_launch("attention_rows");
  if (rc || p.splits == 1) return rc;
  return join_launch<T>(p, st);
}

template <typename T, int DP>
static int tile_launch(const AttnParams& p, bool aligned, cudaStream_t st) {
  constexpr int smem = (3 * DP + kTile) * kTile * 4;
  auto kern = attn_tile_kernel<T, DP>;
  static bool attr[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!attr[dev & 63]) {
    int rc = cuda_check(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "attention tile smem attribute");
    if (rc) return rc;
    attr[dev & 63] = true;
  }
  const int64_t tiles = (p.Sq + kTile - 1) / kTile;
  if ((int64_t)p.B * p.H > INT32_MAX || tiles > 65535)
    return fail(MT_ERR_UNSUPPORTED, "window_attention: batch * heads or queries past the grid");
  kern<<<dim3((unsigned)(p.B * p.H), (unsigned)tiles), 256, smem, st>>>(p, aligned);
  return check_launch("attention_tile");
}

static int check_common(int64_t B, int64_t H, int64_t Hkv, int64_t Sq, int64_t Sk, int64_t D, int64_t window,
                        int64_t sinks, double scale, const char* what) {
  if (B < 0 || H <= 0 || Hkv <= 0 || Sq < 0 || Sk < 0 || D <= 0 || window < 0 || sinks < 0)
    return fail(MT_ERR_INVALID, "%s: bad sizes", what);
  if (H % Hkv) return fail(MT_ERR_INVALID, "%s: %lld heads are no multiple of %lld key heads", what, (long long)H,
                           (long long)Hkv);
  if (D > 256) return fail(MT_ERR_UNSUPPORTED, "%s: head dim > 256", what);
  if (!(scale == scale) || scale > 1e30 || scale < -1e30) return fail(MT_ERR_INVALID, "%s: scale", what);
  if (Sq > kMaxKeys || Sk > kMaxKeys || B > INT32_MAX || Sq * (H / Hkv) > INT32_MAX / 2)
    return fail(MT_ERR_UNSUPPORTED, "%s: sizes past the kernels' range", what);
  return MT_OK;
}

static int clamp_window(int64_t w) { return w <= 0 || w >= kNoWindow ? kNoWindow : (int)w; }

static int validate_window(const mt_window_attention_desc& d) {
  int rc = check_common(d.B, d.H, d.Hkv, d.Sq, d.Sk, d.D, d.window, d.sinks, d.scale, "window_attention");
  if (rc) return rc;
  if (d.dtype != MT_F32 && d.dtype != MT_BF16 && d.dtype != MT_F16)
    return fail(MT_ERR_UNSUPPORTED, "window_attention: dtype");
  if (d.B && d.Sq && (!d.q || !d.o || (d.Sk && (!d.k || !d.v))))
    return fail(MT_ERR_INVALID, "window_attention: null operand");
  return MT_OK;
}

int window_attention_path(const mt_window_attention_desc& d) {
  if (validate_window(d)) return 0;
  return takes_sm100(d) ? MT_WINDOW_PATH_TC : takes_split(d) ? MT_WINDOW_PATH_SPLIT
                      : takes_tiles(d) ? MT_WINDOW_PATH_TILES : MT_WINDOW_PATH_ROWS;
}

// The kernels of few rows have a (batch entry, key head) in the grid's second axis: larger batches go in parts.
constexpr int64_t kMaxBatchHeads = 65535;
static int64_t batch_part(int64_t B, int64_t Hkv) { return std::min(B, std::max<int64_t>(1, kMaxBatchHeads / Hkv)); }

static mt_window_attention_desc batch_from(const mt_window_attention_desc& d, int64_t b, int64_t n) {
  mt_window_attention_desc p = d;
  const int64_t es = dtype_size(d.dtype);
  auto at = [&](const void* base, const int64_t* st) { return static_cast<const char*>(base) + b * st[0] * es; };
  p.B = n;
  if (d.starts) p.starts = d.starts + b;
  if (d.lengths) p.lengths = d.lengths + b;
  p.q = at(d.q, d.q_strides);
  p.o = const_cast<char*>(at(d.o, d.o_strides));
  if (d.k) p.k = at(d.k, d.k_strides);
  if (d.v) p.v = at(d.v, d.v_strides);
  return p;
}
static mt_kv_cache4_attention_desc batch_from(const mt_kv_cache4_attention_desc& d, int64_t b, int64_t n) {
  mt_kv_cache4_attention_desc p = d;
  p.B = n;
  p.lengths = d.lengths + b;
  if (d.block_table) p.block_table = d.block_table + b * d.table_stride;
  p.q = static_cast<const char*>(d.q) + b * d.q_strides[0] * 2;
  p.o = static_cast<char*>(d.o) + b * d.o_strides[0] * 2;
  return p;
}
static bool in_parts(const mt_window_attention_desc& d) {
  return batch_part(d.B, d.Hkv) < d.B && !takes_sm100(d) && (takes_split(d) || !takes_tiles(d));
}
static bool in_parts(const mt_kv_cache4_attention_desc& d) { return batch_part(d.B, d.cache.Hkv) < d.B; }

// `run` on parts of `per` batch entries, the last one the rest; or the larger of the two parts' workspaces.
template <typename Desc, typename Run>
static int run_parts(const Desc& d, int64_t per, Run run) {
  int rc = MT_OK;
  for (int64_t b = 0; b < d.B && !rc; b += per) rc = run(batch_from(d, b, std::min(per, d.B - b)));
  return rc;
}
template <typename Desc, typename Size>
static size_t parts_workspace(const Desc& d, int64_t per, Size size) {
  const int64_t rest = d.B % per;
  return std::max(size(batch_from(d, 0, per)), rest ? size(batch_from(d, d.B - rest, rest)) : 0);
}

size_t window_attention_workspace(const mt_window_attention_desc& d) {
  if (validate_window(d) || d.B == 0 || d.Sq == 0) return 0;
  if (in_parts(d)) return parts_workspace(d, batch_part(d.B, d.Hkv), window_attention_workspace);
  const int splits = window_splits(d);
  if (takes_split(d) && split_joins_in_cluster(d.B * d.Hkv, d.Sq * (d.H / d.Hkv), splits)) return 0;
  return part_bytes(splits, d.B * d.H * d.Sq, d.D);
}

// 4 channels are one aligned vector
static bool aligned4(const void* base, const int64_t* s, int64_t D, int es) {
  if (s[3] != 1 || D % 4 || (uintptr_t)base % (4 * es)) return false;
  return s[0] % 4 == 0 && s[1] % 4 == 0 && s[2] % 4 == 0;
}

template <typename T>
static int window_dispatch(const mt_window_attention_desc& d, const AttnParams& p, cudaStream_t st) {
  const bool kv4 = aligned4(d.k, d.k_strides, d.D, sizeof(T)) && aligned4(d.v, d.v_strides, d.D, sizeof(T));
  if (takes_tiles(d)) {
    const bool all4 = kv4 && aligned4(d.q, d.q_strides, d.D, sizeof(T));
    switch ((d.D + 63) / 64) {
      case 1: return tile_launch<T, 64>(p, all4, st);
      case 2: return tile_launch<T, 128>(p, all4, st);
      case 3: return tile_launch<T, 192>(p, all4, st);
      default: return tile_launch<T, 256>(p, all4, st);
    }
  }
  if (kv4) return rows_launch<T, KV_ALIGNED>(p, st);
  return rows_launch<T, KV_STRIDED>(p, st);
}

int run_window_attention(const mt_window_attention_desc& d, void* ws, size_t ws_bytes, cudaStream_t st) {
  int rc = validate_window(d);
  if (rc || d.B == 0 || d.Sq == 0) return rc;
  if (in_parts(d)) {
    rc = check_workspace(ws, ws_bytes, window_attention_workspace(d), "window_attention");
    if (rc) return rc;
    return run_parts(d, batch_part(d.B, d.Hkv),
                     [&](const mt_window_attention_desc& p) { return run_window_attention(p, ws, ws_bytes, st); });
  }
  AttnParams p{};
  p.B = (int)d.B; p.H = (int)d.H; p.Hkv = (int)d.Hkv; p.g = (int)(d.H / d.Hkv);
  p.Sq = (int)d.Sq; p.Sk = (int)d.Sk; p.D = (int)d.D; p.rows = p.g * p.Sq;
  p.causal = d.causal != 0;
  p.window = clamp_window(d.window);
  p.sinks = (int)std::min<int64_t>(d.sinks, kNoWindow);
  p.scale_log2 = (float)(d.scale * 1.4426950408889634);
  p.starts = d.starts; p.lengths = d.lengths;
  p.q = d.q; p.k = d.k; p.v = d.v; p.o = d.o;
  for (int i = 0; i < 4; ++i) {
    p.qs[i] = d.q_strides[i]; p.ks[i] = d.k_strides[i]; p.vs[i] = d.v_strides[i]; p.os[i] = d.o_strides[i];
  }
  p.splits = window_splits(d);
  rc = check_workspace(ws, ws_bytes, window_attention_workspace(d), "window_attention");
  if (rc) return rc;
  bind_workspace(p, ws);
  if (takes_sm100(d)) return run_window_sm100(d, p, st);
  if (takes_split(d)) {
    p.q_vec = aligned16(d.q, d.q_strides, d.D);
    rc = run_split_attention(p, d.dtype, false, st);
    return rc || p.splits == 1 || p.cluster ? rc : join(p, d.dtype, st);
  }
  switch (d.dtype) {
    case MT_F32: return window_dispatch<float>(d, p, st);
    case MT_BF16: return window_dispatch<__nv_bfloat16>(d, p, st);
    default: return window_dispatch<__half>(d, p, st);
  }
}

static int validate_cache_attention(const mt_kv_cache4_attention_desc& d) {
  int rc = validate_kv_cache4(d.cache);
  if (rc) return rc;
  if (d.max_pages < 0 || d.max_pages > INT32_MAX) return fail(MT_ERR_INVALID, "kv_cache4_attention: max_pages");
  rc = check_common(d.B, d.H, d.cache.Hkv, d.Sq, d.max_pages * d.cache.page_size, d.cache.D, d.window, d.sinks, d.scale,
                    "kv_cache4_attention");
  if (rc) return rc;
  if (d.dtype != MT_BF16 && d.dtype != MT_F16)
    return fail(MT_ERR_UNSUPPORTED, "kv_cache4_attention: queries are bf16 or f16");
  if (d.B && d.Sq && (!d.q || !d.o || !d.lengths || (d.max_pages && !d.block_table)))
    return fail(MT_ERR_INVALID, "kv_cache4_attention: null operand");
  return MT_OK;
}

size_t kv_cache4_attention_workspace(const mt_kv_cache4_attention_desc& d) {
  if (validate_cache_attention(d) || d.B == 0 || d.Sq == 0) return 0;
  if (in_parts(d)) return parts_workspace(d, batch_part(d.B, d.cache.Hkv), kv_cache4_attention_workspace);
  const int splits = cache_splits(d);
  if (split_joins_in_cluster(d.B * d.cache.Hkv, d.Sq * (d.H / d.cache.Hkv), splits)) return 0;
  return part_bytes(splits, d.B * d.H * d.Sq, d.cache.D);
}

int run_kv_cache4_attention(const mt_kv_cache4_attention_desc& d, void* ws, size_t ws_bytes, cudaStream_t st) {
  int rc = validate_cache_attention(d);
  if (rc || d.B == 0 || d.Sq == 0) return rc;
  if (in_parts(d)) {
    rc = check_workspace(ws, ws_bytes, kv_cache4_attention_workspace(d), "kv_cache4_attention");
    if (rc) return rc;
    return run_parts(d, batch_part(d.B, d.cache.Hkv),
                     [&](const mt_kv_cache4_attention_desc& p) { return run_kv_cache4_attention(p, ws, ws_bytes, st); });
  }
  AttnParams p{};
  p.B = (int)d.B; p.H = (int)d.H; p.Hkv = (int)d.cache.Hkv; p.g = (int)(d.H / d.cache.Hkv);
  p.Sq = (int)d.Sq; p.Sk = (int)(d.max_pages * d.cache.page_size); p.D = (int)d.cache.D; p.rows = p.g * p.Sq;
  p.causal = 1;
  p.window = clamp_window(d.window);
  p.sinks = (int)std::min<int64_t>(d.sinks, kNoWindow);
  p.scale_log2 = (float)(d.scale * 1.4426950408889634);
  p.lengths = d.lengths;
  p.q = d.q; p.o = d.o;
  for (int i = 0; i < 4; ++i) {
    p.qs[i] = d.q_strides[i]; p.os[i] = d.o_strides[i];
  }
  p.words[0] = reinterpret_cast<const uint32_t*>(d.cache.k_words);
  p.words[1] = reinterpret_cast<const uint32_t*>(d.cache.v_words);
  p.scales[0] = static_cast<const __half2*>(d.cache.k_scales);
  p.scales[1] = static_cast<const __half2*>(d.cache.v_scales);
  p.table = d.block_table; p.table_stride = d.table_stride;
  p.num_pages = (int)d.cache.num_pages;
  p.page_shift = __builtin_ctzll((unsigned long long)d.cache.page_size);
  p.splits = cache_splits(d);
  rc = check_workspace(ws, ws_bytes, kv_cache4_attention_workspace(d), "kv_cache4_attention");
  if (rc) return rc;
  bind_workspace(p, ws);
  p.q_vec = aligned16(d.q, d.q_strides, d.cache.D);
  rc = run_split_attention(p, d.dtype, true, st);
  return rc || p.splits == 1 || p.cluster ? rc : join(p, d.dtype, st);
}

}  // namespace mt
