// Attention of few query rows over many keys (16-bit keys and values, or the paged 4-bit cache):
// the keys are split over warps and CTAs, and read once for all the query rows of a key head.
//
// The products run on mma.m16n8k16 with the KEYS on the 16-row side and up to 8 * NT query rows on the
// 8-column side: S^T = K Q^T, then O^T = V^T P^T.  The work is bound by reading K and V (a decoder's step
// has 1 to 16 rows a key head), so the tensor cores only have to keep the arithmetic out of the way; with
// the keys on the M side a fragment of K or V is exactly what a lane loads from memory, 16 bytes (or 8 / 4
// bytes of codes) at a time, with no shared memory between: the k order of a product is free, and the
// codes are unpacked into fragments with one shift and one logic instruction per pair.
//
// Codes as operands: bf16 takes 0x4300 | c = 128 + c, exact; f16 takes the code's bits as they are, a
// subnormal c * 2^-24, exact too.  With value = zero + scale c,
//   q.k = scale (q.(128 + c)) + (zero - 128 scale) sum(q)   per 64 channels,
// on fp32 sums that start anew for each 16 keys.  V's codes run over thousands of keys into one
// sum, which an offset of 128 would bias (the tensor core truncates), so they are centred exactly:
//   o = sum p scale (c - 8) + sum p (zero + 8 scale),
// with p scale rounded to bf16 (for f16 queries too: p scale spans more than f16's exponents).
//
// The running maximum is raised only when a score passes it by more than 2^8 ("lazy"): then the warp
// reduces the maximum and rescales; otherwise a block of 16 keys costs one vote.
#include <algorithm>

#include "window_attention.cuh"

namespace mt {

constexpr int kSplitWarps = 4;
constexpr float kSplitLazy = 8.0f;
constexpr int kMinChunk = 16;  // blocks of 16 keys that a CTA takes at least

__device__ __forceinline__ float ex2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <bool F16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (F16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// transpose of an 8 x 8 matrix of 16-bit elements spread over the warp (row lane / 4, columns 2 (lane % 4) ..)
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// two codes at bits 4i and 16 + 4i as 128 + c (bf16) or c * 2^-24 (f16)
template <bool F16>
__device__ __forceinline__ uint32_t code_pair(uint32_t w, int i) {
  return ((w >> (4 * i)) & 0x000f000fu) | (F16 ? 0u : 0x43004300u);
}
// the same two codes minus 8, exact in bf16
__device__ __forceinline__ uint32_t code_pair_centred(uint32_t w, int i) {
  const uint32_t x = code_pair<false>(w, i);
  __nv_bfloat162 v = *reinterpret_cast<const __nv_bfloat162*>(&x);
  v = __hsub2(v, __nv_bfloat162(__ushort_as_bfloat16(0x4308), __ushort_as_bfloat16(0x4308)));  // 136
  return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ uint4 ldg16(const void* p) { return __ldg(static_cast<const uint4*>(p)); }

// One CTA: kSplitWarps warps over one chunk of the key blocks of (b, hk) for 8 * NT query rows.
// DC: blocks of 64 channels.  In a lane, n = lane / 4 and t = lane % 4.
template <bool F16, bool PAGED, int DC, int NT>
__global__ void __launch_bounds__(kSplitWarps * 32) attn_split_kernel(const AttnParams p) {
  using T = typename std::conditional<F16, __half, __nv_bfloat16>::type;
  constexpr int ROWS = 8 * NT;
  constexpr int DP = 64 * DC;
  constexpr bool PF16 = F16 && !PAGED;  // type of P and V's operands
  __shared__ float so[ROWS][DP + 4];
  __shared__ float2 sml[kSplitWarps][ROWS];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = lane >> 2, t = lane & 3;
  const int bk = blockIdx.y, b = bk / p.Hkv, hk = bk % p.Hkv;
  const int r0 = blockIdx.z * ROWS, nr = min(ROWS, p.rows - r0);
  const SeqPos sp = seq_pos(p, b, PAGED);
  const int pmin = sp.start + r0 / p.g, pmax = sp.start + (r0 + nr - 1) / p.g;
  const BlockList bl = block_list<16>(p, sp, pmin, pmax);

  // chunk: the same for every CTA of the grid, so that sequences of different lengths fill it evenly
  float total = 0.f;  // blocks of the whole batch; a guide only, but the same in every CTA
  for (int i = lane; i < p.B; i += 32) {
    const SeqPos s = seq_pos(p, i, PAGED);
    total += (float)block_list<16>(p, s, s.start + r0 / p.g, s.start + (r0 + nr - 1) / p.g).count;
  }
  total = warp_sum(total) * (float)(p.Hkv * gridDim.z) / (float)p.target;
  int per = max(kMinChunk, (int)fminf(ceilf(total), (float)bl.count));
  per = max(per, (bl.count + (int)gridDim.x - 1) / (int)gridDim.x);
  const int i0 = (int)min((int64_t)blockIdx.x * per, (int64_t)bl.count), i1 = min(bl.count, i0 + per);
  const int64_t out_row = ((int64_t)blockIdx.x * p.B * p.Hkv + bk) * p.rows + r0;
  if (i0 >= i1 && gridDim.x > 1) {
    if (threadIdx.x < nr) p.part_ml[out_row + threadIdx.x] = make_float2(-INFINITY, 0.f);
    return;
  }

  // Q fragments: dense, 8 channels at 32 c + 8 t of row n; paged, the channel order of the codes' pairs
  uint32_t qf[NT][2 * DC][4];
  float qsum[NT][DC][2];
#pragma unroll
  for (int x = 0; x < NT; ++x) {
    const int r = r0 + 8 * x + n;
    const bool live = 8 * x + n < nr;
    const T* src = static_cast<const T*>(p.q);
    if (live) src += b * p.qs[0] + (int64_t)(hk * p.g + r % p.g) * p.qs[1] + (int64_t)(r / p.g) * p.qs[2];
#pragma unroll
    for (int c = 0; c < 2 * DC; ++c) {
      const int base = PAGED ? (c >> 1) * 64 + t * 16 + (c & 1) * 8 : c * 32 + t * 8;
      T v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[j] = live && base + j < p.D ? src[(base + j) * p.qs[3]] : from_f32<T>(0.f);
      const uint16_t* u = reinterpret_cast<const uint16_t*>(v);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        qf[x][c][j] = PAGED ? (u[j] | (uint32_t)u[j + 4] << 16) : (u[2 * j] | (uint32_t)u[2 * j + 1] << 16);
      if (PAGED) {
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) s += to_f32<T>(v[j]);
        s += __shfl_xor_sync(0xffffffffu, s, 1);
        s += __shfl_xor_sync(0xffffffffu, s, 2);
        const float s0 = __shfl_sync(0xffffffffu, s, 8 * t), s1 = __shfl_sync(0xffffffffu, s, 8 * t + 4);
        qsum[x][c >> 1][0] = (c & 1) ? qsum[x][c >> 1][0] + s0 : s0;
        qsum[x][c >> 1][1] = (c & 1) ? qsum[x][c >> 1][1] + s1 : s1;
      }
    }
  }
  // keys that the rows of this lane's columns (2t, 2t + 1) see; keys that all rows see, that any row sees
  RowKeys rk[NT][2];
#pragma unroll
  for (int x = 0; x < NT; ++x)
#pragma unroll
    for (int j = 0; j < 2; ++j) rk[x][j] = row_keys(p, sp, sp.start + (r0 + min(8 * x + 2 * t + j, nr - 1)) / p.g);
  const RowKeys ra = row_keys(p, sp, pmin), rz = row_keys(p, sp, pmax);

  float m[NT][2], l[NT][2], cor[NT][DC][2], o[DC][4][NT][4];
#pragma unroll
  for (int x = 0; x < NT; ++x)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      m[x][j] = -INFINITY;
      l[x][j] = 0.f;
#pragma unroll
      for (int c = 0; c < DC; ++c) cor[x][c][j] = 0.f;
    }
#pragma unroll
  for (int c = 0; c < DC; ++c)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[c][j][x][e] = 0.f;

  // ---- loads: K and V of one block of 16 keys into registers ----
  uint4 kd[PAGED ? 1 : 2 * DC][2];
  uint2 kq[PAGED ? DC : 1][2];
  uint4 vd[PAGED ? 1 : DC][4];
  uint32_t vq[PAGED ? DC : 1][4];
  __half2 ksc[PAGED ? DC : 1][2], vsc[PAGED ? DC : 1][2];
  const T* kbase = static_cast<const T*>(p.k) + b * p.ks[0] + hk * p.ks[1];
  const T* vbase = static_cast<const T*>(p.v) + b * p.vs[0] + hk * p.vs[1];

  auto page_of = [&](int i) -> int {
    if (!PAGED || i >= i1) return -1;
    return __ldg(p.table + b * p.table_stride + ((bl.block(i) * 16) >> p.page_shift));
  };
  // row of the cache's arrays where block i starts (page -1 where the page does not exist)
  auto cache_row = [&](int i, int page) -> int64_t {
    return (((int64_t)page * p.Hkv + hk) << p.page_shift) + ((bl.block(i) * 16) & ((1 << p.page_shift) - 1));
  };
  auto load_k = [&](int i, int page) {
    if (PAGED) {
      if (i >= i1 || page < 0 || page >= p.num_pages) return;
      const int64_t row = cache_row(i, page);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t rr = row + n + 8 * h;
#pragma unroll
        for (int c = 0; c < DC; ++c) {
          kq[c][h] = __ldg(reinterpret_cast<const uint2*>(p.words[0] + rr * (DP / 8) + c * 8 + t * 2));
          ksc[c][h] = __ldg(p.scales[0] + rr * DC + c);
        }
      }
    } else {
      const int k0 = bl.block(i) * 16;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int key = k0 + n + 8 * h;
        const T* src = kbase + (int64_t)key * p.ks[2] + t * 8;
#pragma unroll
        for (int c = 0; c < 2 * DC; ++c)
          kd[c][h] = (i < i1 && key < sp.n && c * 32 + t * 8 < p.D) ? ldg16(src + c * 32) : make_uint4(0, 0, 0, 0);
      }
    }
  };
  auto load_v = [&](int i, int page) {
    if (PAGED) {
      if (i >= i1 || page < 0 || page >= p.num_pages) return;
      const int64_t row = cache_row(i, page);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t rr = row + 2 * t + (e & 1) + (e >> 1) * 8;
#pragma unroll
        for (int c = 0; c < DC; ++c) vq[c][e] = __ldg(p.words[1] + rr * (DP / 8) + c * 8 + n);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int c = 0; c < DC; ++c) vsc[c][h] = __ldg(p.scales[1] + (row + n + 8 * h) * DC + c);
    } else {
      const int k0 = bl.block(i) * 16;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = k0 + 2 * t + (e & 1) + (e >> 1) * 8;
        // a key that no row sees counts as zeros, whatever stands there
        const bool live = i < i1 && key < sp.n && ((key >= ra.lo && key <= rz.hi) || key < rz.sk);
        const T* src = vbase + (int64_t)key * p.vs[2] + n * 8;
#pragma unroll
        for (int c = 0; c < DC; ++c)
          vd[c][e] = (live && c * 64 + n * 8 < p.D) ? ldg16(src + c * 64) : make_uint4(0, 0, 0, 0);
      }
    }
  };

  int i = i0 + warp;
  int page = page_of(i), page_next = page_of(i + kSplitWarps);
  load_k(i, page);
  load_v(i, page);
  for (; i < i1; i += kSplitWarps) {
    const int k0 = bl.block(i) * 16;
    // ---- S^T = K Q^T: sc[.][0,1] key n, sc[.][2,3] key n + 8; columns 2t, 2t + 1 ----
    float sc[NT][4];
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[x][e] = 0.f;
    if (PAGED) {
#pragma unroll
      for (int c = 0; c < DC; ++c) {
        float acc[NT][4];
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[x][e] = 0.f;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint32_t w0 = u ? kq[c][0].y : kq[c][0].x, w1 = u ? kq[c][1].y : kq[c][1].x;
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const uint32_t a[4] = {code_pair<F16>(w0, 2 * s), code_pair<F16>(w1, 2 * s),
                                   code_pair<F16>(w0, 2 * s + 1), code_pair<F16>(w1, 2 * s + 1)};
#pragma unroll
            for (int x = 0; x < NT; ++x) mma16816<F16>(acc[x], a, qf[x][2 * c + u][2 * s], qf[x][2 * c + u][2 * s + 1]);
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float s = __low2float(ksc[c][h]), z = __high2float(ksc[c][h]);
          const float f = F16 ? s * 16777216.f : s;
          const float off = F16 ? z : fmaf(-128.f, s, z);
#pragma unroll
          for (int x = 0; x < NT; ++x)
#pragma unroll
            for (int j = 0; j < 2; ++j)
              sc[x][2 * h + j] += fmaf(f, acc[x][2 * h + j], off * qsum[x][c][j]);
        }
      }
    } else {
#pragma unroll
      for (int c = 0; c < 2 * DC; ++c) {
        const uint32_t a0[4] = {kd[c][0].x, kd[c][1].x, kd[c][0].y, kd[c][1].y};
        const uint32_t a1[4] = {kd[c][0].z, kd[c][1].z, kd[c][0].w, kd[c][1].w};
#pragma unroll
        for (int x = 0; x < NT; ++x) {
          mma16816<F16>(sc[x], a0, qf[x][c][0], qf[x][c][1]);
          mma16816<F16>(sc[x], a1, qf[x][c][2], qf[x][c][3]);
        }
      }
    }
    const bool missing = PAGED && (page < 0 || page >= p.num_pages);
    load_k(i + kSplitWarps, page_next);

    // ---- softmax ----
    const bool full = !missing && k0 + 15 <= ra.hi && (k0 >= rz.lo || k0 + 15 < ra.sk);
    bool over = false;
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float s = sc[x][e] * p.scale_log2;
        if (!full && (missing || !rk[x][e & 1].sees(k0 + n + 8 * (e >> 1)))) s = -INFINITY;
        sc[x][e] = s;
        over |= s > m[x][e & 1] + kSplitLazy;
      }
    if (__any_sync(0xffffffffu, over)) {
#pragma unroll
      for (int x = 0; x < NT; ++x) {
        float corr[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float mx = fmaxf(sc[x][j], sc[x][2 + j]);
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          mx = fmaxf(mx, m[x][j]);
          corr[j] = m[x][j] == -INFINITY ? 0.f : ex2f(m[x][j] - mx);
          m[x][j] = mx;
          l[x][j] *= corr[j];
#pragma unroll
          for (int c = 0; c < DC; ++c) cor[x][c][j] *= corr[j];
        }
#pragma unroll
        for (int c = 0; c < DC; ++c)
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[c][j][x][e] *= corr[e & 1];
      }
    }
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float mu = m[x][e & 1] == -INFINITY ? 0.f : m[x][e & 1];
        sc[x][e] = ex2f(sc[x][e] - mu);
        l[x][e & 1] += sc[x][e];
      }

    // ---- O^T += V^T P^T ----
    uint32_t pb[NT][2];
    if (!PAGED) {
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          pb[x][h] = transpose8x8(PF16 ? pack_f16x2(sc[x][2 * h], sc[x][2 * h + 1])
                                       : pack_bf16x2(sc[x][2 * h], sc[x][2 * h + 1]));
    }
#pragma unroll
    for (int c = 0; c < DC; ++c) {
      if (PAGED) {
        float s[2], z[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          s[h] = __low2float(vsc[c][h]);
          z[h] = fmaf(8.f, s[h], __high2float(vsc[c][h]));
        }
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float e0 = sc[x][2 * h] * s[h], e1 = sc[x][2 * h + 1] * s[h];
            float g0 = sc[x][2 * h] * z[h], g1 = sc[x][2 * h + 1] * z[h];
            if (!full) {  // scales of slots that hold nothing may be NaN
              if (sc[x][2 * h] == 0.f) e0 = g0 = 0.f;
              if (sc[x][2 * h + 1] == 0.f) e1 = g1 = 0.f;
            }
            cor[x][c][0] += g0;
            cor[x][c][1] += g1;
            pb[x][h] = transpose8x8(pack_bf16x2(e0, e1));
          }
        const uint32_t lo0 = __byte_perm(vq[c][0], vq[c][1], 0x5410), hi0 = __byte_perm(vq[c][0], vq[c][1], 0x7632);
        const uint32_t lo1 = __byte_perm(vq[c][2], vq[c][3], 0x5410), hi1 = __byte_perm(vq[c][2], vq[c][3], 0x7632);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t w0 = j < 2 ? lo0 : hi0, w1 = j < 2 ? lo1 : hi1;
          const int q = (2 * j) & 3;
          const uint32_t a[4] = {code_pair_centred(w0, q), code_pair_centred(w0, q + 1), code_pair_centred(w1, q),
                                 code_pair_centred(w1, q + 1)};
#pragma unroll
          for (int x = 0; x < NT; ++x) mma16816<false>(o[c][j][x], a, pb[x][0], pb[x][1]);
        }
      } else {
        const uint32_t* e0 = reinterpret_cast<const uint32_t*>(&vd[c][0]);
        const uint32_t* e1 = reinterpret_cast<const uint32_t*>(&vd[c][1]);
        const uint32_t* e2 = reinterpret_cast<const uint32_t*>(&vd[c][2]);
        const uint32_t* e3 = reinterpret_cast<const uint32_t*>(&vd[c][3]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t a[4] = {__byte_perm(e0[j], e1[j], 0x5410), __byte_perm(e0[j], e1[j], 0x7632),
                                 __byte_perm(e2[j], e3[j], 0x5410), __byte_perm(e2[j], e3[j], 0x7632)};
#pragma unroll
          for (int x = 0; x < NT; ++x) mma16816<PF16>(o[c][j][x], a, pb[x][0], pb[x][1]);
        }
      }
    }
    load_v(i + kSplitWarps, page_next);
    page = page_next;
    page_next = page_of(i + 2 * kSplitWarps);
  }

  // ---- join the lanes (sums), then the warps ----
#pragma unroll
  for (int x = 0; x < NT; ++x)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) {
        l[x][j] += __shfl_xor_sync(0xffffffffu, l[x][j], d);
        if (PAGED)
#pragma unroll
          for (int c = 0; c < DC; ++c) cor[x][c][j] += __shfl_xor_sync(0xffffffffu, cor[x][c][j], d);
      }
      if (n == 0) sml[warp][8 * x + 2 * t + j] = make_float2(m[x][j], l[x][j]);
    }
  __syncthreads();
  float f[NT][2];
#pragma unroll
  for (int x = 0; x < NT; ++x)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kSplitWarps; ++w) top = fmaxf(top, sml[w][8 * x + 2 * t + j].x);
      f[x][j] = m[x][j] == -INFINITY ? 0.f : ex2f(m[x][j] - top);
    }
  for (int w = 0; w < kSplitWarps; ++w) {
    if (warp == w) {
#pragma unroll
      for (int c = 0; c < DC; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int x = 0; x < NT; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float* dst = &so[8 * x + 2 * t + (e & 1)][64 * c + 8 * n + 2 * j + (e >> 1)];
              const float v = (o[c][j][x][e] + (PAGED ? cor[x][c][e & 1] : 0.f)) * f[x][e & 1];
              *dst = w ? *dst + v : v;
            }
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < nr * DP; i += kSplitWarps * 32) {
    const int r = i / DP, d = i % DP;
    if (d >= p.D) continue;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kSplitWarps; ++w) top = fmaxf(top, sml[w][r].x);
    float ls = 0.f;
#pragma unroll
    for (int w = 0; w < kSplitWarps; ++w)
      if (sml[w][r].x != -INFINITY) ls = fmaf(sml[w][r].y, ex2f(sml[w][r].x - top), ls);
    if (gridDim.x > 1) {
      p.part_o[(out_row + r) * p.D + d] = so[r][d];
      if (d == 0) p.part_ml[out_row + r] = make_float2(top, ls);
    } else {
      const int qi = (r0 + r) / p.g, h = hk * p.g + (r0 + r) % p.g;
      static_cast<T*>(p.o)[b * p.os[0] + h * p.os[1] + qi * p.os[2] + d * p.os[3]] =
          from_f32<T>(ls > 0.f ? so[r][d] / ls : 0.f);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// host

// Query rows a key head that the split kernel takes (more rows: the tiled kernels read K and V less often).
int split_tile_rows(int64_t rows) { return rows <= 8 ? 8 : 16; }

int split_count(int64_t bk, int64_t rows, int64_t keys) {
  const int tr = split_tile_rows(rows);
  const int64_t ctas = bk * ((rows + tr - 1) / tr);
  const int64_t most = std::max<int64_t>(1, (keys / 16 + kMinChunk - 1) / kMinChunk);
  // a few times more than fill the GPU: room for sequences longer than the mean
  const int64_t want = (16LL * num_sms() + ctas - 1) / ctas;
  return (int)std::max<int64_t>(1, std::min<int64_t>(std::min(want, most), 512));
}

template <bool F16, bool PAGED, int DC>
static int split_launch_dc(AttnParams& p, cudaStream_t st) {
  const int tr = split_tile_rows(p.rows);
  const int64_t tiles = (p.rows + tr - 1) / tr;
  if ((int64_t)p.B * p.Hkv > 65535 || tiles > 65535)
    return fail(MT_ERR_UNSUPPORTED, "window_attention: batch * key heads or rows past the grid");
  dim3 grid((unsigned)p.splits, (unsigned)(p.B * p.Hkv), (unsigned)tiles);
  p.target = 8 * num_sms();
  if (tr == 8) attn_split_kernel<F16, PAGED, DC, 1><<<grid, kSplitWarps * 32, 0, st>>>(p);
  else attn_split_kernel<F16, PAGED, DC, 2><<<grid, kSplitWarps * 32, 0, st>>>(p);
  return check_launch("attention_split");
}

template <bool F16, bool PAGED>
static int split_launch(AttnParams& p, cudaStream_t st) {
  switch ((p.D + 63) / 64) {
    case 1: return split_launch_dc<F16, PAGED, 1>(p, st);
    case 2: return split_launch_dc<F16, PAGED, 2>(p, st);
    case 3: return split_launch_dc<F16, PAGED, 3>(p, st);
    default: return split_launch_dc<F16, PAGED, 4>(p, st);
  }
}

int run_split_attention(AttnParams& p, int dtype, bool paged, cudaStream_t st) {
  if (dtype == MT_F16) return paged ? split_launch<true, true>(p, st) : split_launch<true, false>(p, st);
  return paged ? split_launch<false, true>(p, st) : split_launch<false, false>(p, st);
}

}  // namespace mt
