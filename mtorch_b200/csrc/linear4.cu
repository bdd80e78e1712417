// Products of few rows with a weight held in 4 bits, and its packing.
//
// W[n, k] = scale[n, k / group] * (code - 8).  Words of 8 codes; in each block of 128 columns word w
// is stored at place (w % 4) * 4 + w / 4 (see mtorch_cuda.h).
//
// linear4_kernel: Y^T = W X^T on mma.m16n8k16 with the weight's rows on the 16-row side and up to 8 * NT rows of X
// on the 8-column side.  Bound by reading W, and next by unpacking it: a lane's 16 bytes are words t, t + 4, t + 8,
// t + 12 of a block of 128 columns, which are its fragments for 8 products of 16 columns.  A code's 4 bits at the low
// end of a 16-bit lane are the number c * 2^-133 in bf16 (c * 2^-24 in f16), a subnormal that mma multiplies exactly,
// at bits 4..7 sixteen times that: one AND makes two operands, one shift serves half a word.  The two places have
// sums of their own (a sixteenth put on X instead would cost f16 values below 2^-10 their last bits).  X is laid out once
// per CTA as operands in shared memory (bf16 times 2^80, to stay clear of fp32's subnormals), with the sums of -8 x
// per row and group beside it, which take the codes' offset off: y += scale (low - 8 sum x + high / 16), in fp32 per
// group of columns.  A warp brings its blocks of W with its own cp.async into a ring; no barrier stands between
// the warps but at the end of a tile.
//
// Rows of X that this cannot hold, with an infinity, a NaN or (bf16, fp32) a largest value outside 2^-46..2^47, are
// found while X is laid out; their outputs are summed up as they stand, a warp an output (w4_direct): infinity times a
// weight is then what it has to be, and not NaN.  One such row of 8192 -> 28672 takes 174 us in the place of 40, 13 of
// 5000 -> 4099 204 in the place of 20.
//
// fp32 X goes as three bf16 parts (8 + 8 + 8 bits) in three rows of their own, added at the end.
#include <algorithm>

#include "runtime.h"

namespace mt {

// place of word w in its block of 16 words, and back (the map is a 4 x 4 transpose)
__host__ __device__ __forceinline__ int w4_place(int w) { return (w & 3) * 4 + (w >> 2); }

struct Linear4Params {
  int M, N, K, Kp, group;
  const void* x; int64_t ldx;
  bool x_vec;  // 8 columns of a row of X are aligned 16-byte vectors
  const uint32_t* words;
  const __nv_bfloat16* scales;
  const void* bias;
  void* y; int64_t ldy;
};

template <bool F16>
__device__ __forceinline__ void w4_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
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

// the same on sums of zero
template <bool F16>
__device__ __forceinline__ void w4_mma_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (F16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

// Rows of the products that one row of X becomes.
template <typename T> constexpr int w4_parts() { return sizeof(T) == 4 ? 3 : 1; }

// A code counts c * 2^-24 in f16, c * 2^-133 in bf16 against operands scaled by 2^80.  (The scale leaves room on both
// sides: X up to 2^47 fits, and weights and rows whose products are as small as 2^-73 do not underflow.)
template <typename T>
__device__ __forceinline__ constexpr float w4_unit() {
  return std::is_same<T, __half>::value ? 16777216.f : 9007199254740992.f;  // 2^24, 2^53
}

// Largest |x| of eight columns as bits of the type (of fp32: bits of fp32), a NaN above all.
template <typename T>
__device__ __forceinline__ uint32_t w4_top(const uint4 (&raw)[sizeof(T) / 2]) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(raw);
  if constexpr (sizeof(T) == 4) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, w[j] & 0x7fffffffu);
    return m;
  } else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const T2* v = reinterpret_cast<const T2*>(w);
    const T2 m = __hmax2_nan(__hmax2_nan(__habs2(v[0]), __habs2(v[1])), __hmax2_nan(__habs2(v[2]), __habs2(v[3])));
    const uint32_t u = *reinterpret_cast<const uint32_t*>(&m);
    return max(u & 0x7fffu, u >> 16 & 0x7fffu);
  }
}
// whether a row of this largest value has to be summed up as it stands
template <typename T>
__device__ __forceinline__ bool w4_odd(uint32_t top) {
  if (std::is_same<T, __half>::value) return top >= 0x7c00u;
  constexpr int sh = sizeof(T) == 4 ? 23 : 7;
  return top >= (127u + 47u) << sh || (top != 0 && top < (127u - 46u) << sh);
}

// Eight columns of X as operands: pairs (0, 4), (1, 5), (2, 6), (3, 7); bf16 times 2^80, f16 as it is.  `part`: which of the three bf16 parts of
// fp32.  Returns -8 times the columns' sum in the operands' unit.
template <typename T>
__device__ __forceinline__ float w4_operands(const uint4 (&raw)[sizeof(T) / 2], int part, uint4& out) {
  constexpr bool F16 = std::is_same<T, __half>::value;
  const T* e = reinterpret_cast<const T*>(raw);
  float sum = 0.f;
  uint32_t w[4];
  if constexpr (sizeof(T) == 2) {
    const uint4 r = raw[0];
    w[0] = __byte_perm(r.x, r.z, 0x5410);
    w[1] = __byte_perm(r.x, r.z, 0x7632);
    w[2] = __byte_perm(r.y, r.w, 0x5410);
    w[3] = __byte_perm(r.y, r.w, 0x7632);
    if (!F16) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        __nv_bfloat162& v = *reinterpret_cast<__nv_bfloat162*>(&w[j]);
        const __nv_bfloat16 f = __ushort_as_bfloat16(0x6780);  // 2^80
        v = __hmul2(v, __nv_bfloat162(f, f));
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += to_f32<T>(e[j]);
  } else {
    constexpr float f = 1208925819614629174706176.f;  // 2^80
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float x = to_f32<T>(e[j]);
      const float hi = __bfloat162float(__float2bfloat16_rn(x));
      const float mid = __bfloat162float(__float2bfloat16_rn(x - hi));
      v[j] = __bfloat162float(__float2bfloat16_rn(part == 0 ? hi : part == 1 ? mid : x - hi - mid));
      sum += v[j];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = pack_bf16x2(v[j] * f, v[j + 4] * f);
  }
  out = make_uint4(w[0], w[1], w[2], w[3]);
  return sum * (-8.f / w4_unit<T>());
}

// 16 bytes to shared memory
__device__ __forceinline__ void w4_cp_async(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// Shared memory of a CTA for `rows` operand rows: the warps' sums, the rings, X's operands, the sums of -8 x.
template <int GROUP, int MT, int NT, int WARPS>
struct W4Smem {
  static constexpr int STAGES = 3;
  static constexpr int RING = STAGES * MT * 1024;  // a warp's: 16 MT rows of 64 bytes a block
  static __host__ __device__ int pitch(int Kp) { return Kp * 2 + 64; }  // of an operand row: two rows meet no bank twice
  static __host__ __device__ int red(int rows) { return 2 * WARPS * rows * (16 * MT + 4) * 4; }
  static __host__ __device__ int ops(int rows, int Kp) { return rows * pitch(Kp); }
  static __host__ __device__ int sums(int Kp) { return Kp / GROUP * 8 * NT * 4; }
  static __host__ __device__ int total(int rows, int Kp) { return red(rows) + WARPS * RING + ops(rows, Kp) + sums(Kp) + 16; }
};

// Eight columns of a row x of X from column k on, zeros past K.
template <typename T>
__device__ __forceinline__ void w4_load8(const T* x, int k, int K, bool vec, uint4 (&raw)[sizeof(T) / 2]) {
  const T* src = x + k;
  if (vec && k + 8 <= K) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) raw[i] = __ldg(reinterpret_cast<const uint4*>(src) + i);
  } else {
    T* e = reinterpret_cast<T*>(raw);
#pragma unroll
    for (int j = 0; j < 8; ++j) e[j] = k + j < K ? src[j] : from_f32<T>(0.f);
  }
}

// sum of x w over a row of X and a row of W by one warp, in fp32
template <typename T, int GROUP>
__device__ __noinline__ float w4_direct(const T* x, const uint32_t* words, const __nv_bfloat16* scales, int K, bool vec) {
  float v = 0.f;
  for (int i = threadIdx.x & 31; i * 8 < K; i += 32) {
    uint4 raw[sizeof(T) / 2];
    w4_load8<T>(x, i * 8, K, vec, raw);
    const T* e = reinterpret_cast<const T*>(raw);
    const uint32_t word = __ldg(words + (i & ~15) + w4_place(i & 15));
    const float s = __bfloat162float(scales[i * 8 / GROUP]);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i * 8 + j < K) v = fmaf(to_f32<T>(e[j]), s * (float)((int)(word >> (4 * j) & 15u) - 8), v);
  }
  return warp_sum(v);
}

// A CTA takes a run of strips of 16 rows of W (outputs), the same number for all but a strip, and goes through them MT at
// a time against up to 8 * NT operand rows; its warps take blocks of 128 columns in turn and add up in shared memory.
// The rings run on across the tiles: the next tile's first blocks come while this one is finished.
template <typename T, int GROUP, int MT, int NT, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, 1) linear4_kernel(const Linear4Params p) {
  constexpr bool F16 = std::is_same<T, __half>::value;
  constexpr int PARTS = w4_parts<T>();
  constexpr int GPB = 128 / GROUP;  // groups of a block
  constexpr int OUT = 16 * MT;
  using Smem = W4Smem<GROUP, MT, NT, WARPS>;
  extern __shared__ __align__(16) uint8_t w4_smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = lane >> 2, t = lane & 3;
  const int blocks = p.Kp / 128, rows = p.M * PARTS;
  float* red = reinterpret_cast<float*>(w4_smem);  // [2][WARPS][rows][OUT + 4]
  uint8_t* ring = w4_smem + Smem::red(rows) + warp * Smem::RING;
  uint8_t* ops = w4_smem + Smem::red(rows) + WARPS * Smem::RING;
  float* sums = reinterpret_cast<float*>(ops + Smem::ops(rows, p.Kp));  // [group][8 NT]
  uint32_t* odd_smem = reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(sums) + Smem::sums(p.Kp));
  const uint32_t ring_u32 = smem_u32(ring);
  const int pitch_x = Smem::pitch(p.Kp);
  const int strips = (p.N + 15) / 16;
  const int s0 = (int)((int64_t)strips * blockIdx.x / gridDim.x), s1 = (int)((int64_t)strips * (blockIdx.x + 1) / gridDim.x);
  const int last_row = min(p.N, s1 * 16) - 1;

  // step q of this warp: block (q % per_tile) * WARPS + warp of the tile at strip s0 + q / per_tile * MT
  const int per_tile = (blocks + WARPS - 1) / WARPS;
  // the next step to bring: chunk t of rows n + 8 i (rows past the CTA's repeat its last)
  const int64_t pitch = p.Kp / 2;
  const uint8_t* wsrc[2 * MT];
  int ln0 = s0 * 16, lkb = warp, lq = 0;
  auto start_tile = [&]() {
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i)
      wsrc[i] = reinterpret_cast<const uint8_t*>(p.words) + min(ln0 + 8 * i + n, last_row) * pitch + warp * 64 + t * 16;
  };
  start_tile();
  auto load = [&](int stage) {
    if (ln0 <= last_row && lkb < blocks) {
      const uint32_t dst = ring_u32 + stage * (MT * 1024) + lane * 16;
#pragma unroll
      for (int i = 0; i < 2 * MT; ++i) w4_cp_async(dst + i * 512, wsrc[i]);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    lkb += WARPS;
    if (++lq == per_tile) {
      lq = 0;
      lkb = warp;
      ln0 += OUT;
      start_tile();
    } else {
#pragma unroll
      for (int i = 0; i < 2 * MT; ++i) wsrc[i] += WARPS * 64;
    }
  };
  uint2 sc = make_uint2(0, 0);  // scales of row `lane` of the tile in the next block, as they come
  const __nv_bfloat16* srow;
  auto scales_of = [&](int n0) {
    srow = p.scales + (int64_t)min(n0 + (lane & (OUT - 1)), last_row) * (p.Kp / GROUP);
  };
  auto load_scales = [&](int kb) {
    if (kb >= blocks) return;
    const __nv_bfloat16* s = srow + kb * GPB;
    if (GPB == 4) sc = __ldg(reinterpret_cast<const uint2*>(s));
    else if (GPB == 2) sc.x = __ldg(reinterpret_cast<const uint32_t*>(s));
    else sc.x = __ldg(reinterpret_cast<const uint16_t*>(s));
  };
#pragma unroll
  for (int s = 0; s < Smem::STAGES - 1; ++s) load(s);
  scales_of(s0 * 16);
  load_scales(warp);

  // X's operands: a warp takes 32 chunks of 8 columns of a row at a time (a group's chunks are neighbouring lanes)
  const int chunks = p.Kp / 8, segs = (chunks + 31) / 32, tasks = rows * segs;
  constexpr int U = 4;  // loads in flight
  bool odd = false;
  for (int task0 = warp; task0 < tasks; task0 += U * WARPS) {
    uint4 raw[U][sizeof(T) / 2];
    int row[U], ch[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int task = min(task0 + u * WARPS, tasks - 1);
      row[u] = task / segs;
      ch[u] = (task - row[u] * segs) * 32 + lane;
      w4_load8<T>(static_cast<const T*>(p.x) + (int64_t)(row[u] / PARTS) * p.ldx, ch[u] * 8, p.K, p.x_vec, raw[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint4 o;
      odd |= w4_odd<T>(w4_top<T>(raw[u]));
      float sum = w4_operands<T>(raw[u], row[u] % PARTS, o);
#pragma unroll
      for (int d = 1; d < GROUP / 8; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      if (task0 + u * WARPS < tasks && ch[u] < chunks) {
        *reinterpret_cast<uint4*>(ops + row[u] * pitch_x + ch[u] * 16) = o;
        if (ch[u] % (GROUP / 8) == 0) sums[ch[u] / (GROUP / 8) * (8 * NT) + row[u]] = sum;
      }
    }
  }
  uint32_t odd_rows = 0;  // bit m: row m is summed up as it stands
  if (__syncthreads_or(odd)) {  // eight columns of some row: look at whole rows
    if (threadIdx.x == 0) *odd_smem = 0;
    __syncthreads();
    for (int m = warp; m < p.M; m += WARPS) {
      uint32_t top = 0;
      for (int c = lane; c < chunks; c += 32) {
        uint4 raw[sizeof(T) / 2];
        w4_load8<T>(static_cast<const T*>(p.x) + (int64_t)m * p.ldx, c * 8, p.K, p.x_vec, raw);
        top = max(top, w4_top<T>(raw));
      }
      top = __reduce_max_sync(0xffffffffu, top);
      if (lane == 0 && w4_odd<T>(top)) atomicOr(odd_smem, 1u << m);
    }
    __syncthreads();
    odd_rows = *odd_smem;
  }

  const uint8_t* xrow[NT];  // this lane's operand rows (rows past the last repeat it; their sums are not stored)
#pragma unroll
  for (int x = 0; x < NT; ++x) xrow[x] = ops + min(8 * x + n, rows - 1) * pitch_x + t * 16;
  float y[MT][NT][4];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int e = 0; e < 4; ++e) y[i][x][e] = 0.f;
  int stage = 0, buf = 0, q = 0, kb = warp;
  for (int n0 = s0 * 16; n0 <= last_row;) {
    if (kb < blocks) {
      asm volatile("cp.async.wait_group %0;" ::"n"(Smem::STAGES - 2) : "memory");
      __syncwarp();
      const uint8_t* st = ring + stage * (MT * 1024) + lane * 16;
      uint2 sn[MT][2];  // this block's scales; the next block's start to come
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          sn[i][h].x = __shfl_sync(0xffffffffu, sc.x, 16 * i + 8 * h + n);
          sn[i][h].y = GPB == 4 ? __shfl_sync(0xffffffffu, sc.y, 16 * i + 8 * h + n) : 0u;
        }
      if (q + 1 < per_tile) load_scales(kb + WARPS);
      uint4 xb[4][NT];
      float2 s8[GPB][NT];
#pragma unroll
      for (int x = 0; x < NT; ++x) {
#pragma unroll
        for (int j = 0; j < 4; ++j) xb[j][x] = *reinterpret_cast<const uint4*>(xrow[x] + kb * 256 + j * 64);
#pragma unroll
        for (int g = 0; g < GPB; ++g)
          s8[g][x] = *reinterpret_cast<const float2*>(sums + (kb * GPB + g) * (8 * NT) + 8 * x + 2 * t);
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const uint4 c0 = *reinterpret_cast<const uint4*>(st + i * 1024), c1 = *reinterpret_cast<const uint4*>(st + i * 1024 + 512);
        // sums over the codes at bits 0..3, and 16 times those over the codes at bits 4..7 (one chain for both, the
        // second divided before the first start, saves the additions and takes 36.3 us for 34.9 at 8192 -> 28672, one row)
        float lo[NT][4], hi[NT][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // 32 columns
          const bool fresh = (j * 32) % GROUP == 0;
          const uint32_t w0 = j == 0 ? c0.x : j == 1 ? c0.y : j == 2 ? c0.z : c0.w, v0 = w0 >> 8;
          const uint32_t w1 = j == 0 ? c1.x : j == 1 ? c1.y : j == 2 ? c1.z : c1.w, v1 = w1 >> 8;
          const uint32_t al[4] = {w0 & 0x000f000fu, w1 & 0x000f000fu, v0 & 0x000f000fu, v1 & 0x000f000fu};
          const uint32_t ah[4] = {w0 & 0x00f000f0u, w1 & 0x00f000f0u, v0 & 0x00f000f0u, v1 & 0x00f000f0u};
#pragma unroll
          for (int x = 0; x < NT; ++x) {
            if (fresh) {
              w4_mma_zero<F16>(lo[x], al, xb[j][x].x, xb[j][x].z);
              w4_mma_zero<F16>(hi[x], ah, xb[j][x].y, xb[j][x].w);
            } else {
              w4_mma<F16>(lo[x], al, xb[j][x].x, xb[j][x].z);
              w4_mma<F16>(hi[x], ah, xb[j][x].y, xb[j][x].w);
            }
          }
          if ((j * 32 + 32) % GROUP == 0) {
            const int g = j * 32 / GROUP;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t w = g < 2 ? sn[i][h].x : sn[i][h].y;
              const float s = __uint_as_float(g & 1 ? w & 0xffff0000u : w << 16);
#pragma unroll
              for (int x = 0; x < NT; ++x) {
                y[i][x][2 * h] = fmaf(s, fmaf(hi[x][2 * h], 0.0625f, lo[x][2 * h] + s8[g][x].x), y[i][x][2 * h]);
                y[i][x][2 * h + 1] = fmaf(s, fmaf(hi[x][2 * h + 1], 0.0625f, lo[x][2 * h + 1] + s8[g][x].y), y[i][x][2 * h + 1]);
              }
            }
          }
        }
      }
    }
    if (q + 1 == per_tile) {
      scales_of(n0 + OUT);
      load_scales(warp);
    }
    __syncwarp();
    int next = stage + Smem::STAGES - 1;
    if (next >= Smem::STAGES) next -= Smem::STAGES;
    load(next);
    if (++stage == Smem::STAGES) stage = 0;
    kb += WARPS;
    if (++q < per_tile) continue;
    // the tile is done: add the warps' sums (two buffers, so that one barrier a tile is enough)
    float* mine = red + (buf * WARPS + warp) * rows * (OUT + 4);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 8 * x + 2 * t + (e & 1);
          if (r < rows) mine[r * (OUT + 4) + 16 * i + n + 8 * (e >> 1)] = y[i][x][e];
          y[i][x][e] = 0.f;
        }
    __syncthreads();
    for (int i = threadIdx.x; i < p.M * OUT; i += WARPS * 32) {
      const int m = i / OUT, c = i % OUT;
      if (n0 + c > last_row || (odd_rows >> m & 1u)) continue;
      float v = 0.f;
#pragma unroll
      for (int part = 0; part < PARTS; ++part)
#pragma unroll
        for (int k = 0; k < WARPS; ++k) v += red[((buf * WARPS + k) * rows + m * PARTS + part) * (OUT + 4) + c];
      v *= w4_unit<T>();
      if (p.bias) v += to_f32<T>(static_cast<const T*>(p.bias)[n0 + c]);
      static_cast<T*>(p.y)[(int64_t)m * p.ldy + n0 + c] = from_f32<T>(v);
    }
    for (uint32_t left = odd_rows; left; left &= left - 1) {
      const int m = __ffs(left) - 1;
      for (int c = warp; c < OUT && n0 + c <= last_row; c += WARPS) {
        const int64_t n = n0 + c;
        float v = w4_direct<T, GROUP>(static_cast<const T*>(p.x) + (int64_t)m * p.ldx, p.words + n * (p.Kp / 8),
                                      p.scales + n * (p.Kp / GROUP), p.K, p.x_vec);
        if (p.bias) v += to_f32<T>(static_cast<const T*>(p.bias)[n0 + c]);
        if (lane == 0) static_cast<T*>(p.y)[(int64_t)m * p.ldy + n0 + c] = from_f32<T>(v);
      }
    }
    buf ^= 1;
    n0 += OUT;
    q = 0;
    kb = warp;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
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

// ---- many rows: products of f16 copies on the tensor-core GEMM ----
//
// scale * (code - 8) has at most 8 + 3 significant bits, which f16 holds and bf16 does not, and bf16 X fits f16's 11 bits
// too.  Only the ranges differ: each row of W and of X is multiplied by a power of two that takes its largest finite value
// near the top of f16's range, and the GEMM's epilogue takes the fp32 sums back by both.  What stands 2^28 (W) or 2^21
// (X) below its row's largest value is rounded to 2^-40 of that.  fp32 X goes in two parts of 11 bits (what is left is
// 2^-24 of a value): x1 and 2^11 x2 side by side, against w and 2^-11 w.
// So the same row gives the same sums here and in linear4_kernel up to their order.

// the power of two that takes the largest finite |x| of `bits` (fp32, as unsigned) to 2^to .. 2^(to + 1)
__device__ __forceinline__ int w4_shift(uint32_t bits, int to) { return to + 127 - (int)(bits >> 23); }

struct W4CopyParams {
  Linear4Params p;
  __half *wh, *xh;              // [N, parts * Kp], [M, parts * Kp]
  int *row_shift, *col_shift;   // [M], [N]
  int w_blocks;                 // CTAs that copy W, eight rows each; the others copy a row of X each
};

// Zeros past K in both.
template <typename T>
__global__ void __launch_bounds__(256) linear4_copy_kernel(const W4CopyParams c) {
  constexpr int PARTS = sizeof(T) == 4 ? 2 : 1;
  __shared__ uint32_t tops[8];
  const Linear4Params& p = c.p;
  const int W = p.Kp / 8;
  if (blockIdx.x < c.w_blocks) {  // a warp per row of W
    const int64_t n = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (n >= p.N) return;
    const __nv_bfloat16* sc = p.scales + n * (p.Kp / p.group);
    uint32_t top = 0;
    for (int i = lane; i * p.group < p.K; i += 32) {
      const uint32_t u = __float_as_uint(__bfloat162float(sc[i])) & 0x7fffffffu;
      if (u < 0x7f800000u) top = max(top, u);
    }
    const int b = w4_shift(__reduce_max_sync(0xffffffffu, top), 11);  // 8 scale: at most 2^15
    if (lane == 0) c.col_shift[n] = b;
    uint4* out = reinterpret_cast<uint4*>(c.wh) + n * PARTS * W;
#pragma unroll 4
    for (int i = lane; i < W; i += 32) {
      const uint32_t word = __ldg(p.words + n * W + (i & ~15) + w4_place(i & 15));
      const float s = ldexp_f32(__bfloat162float(sc[i * 8 / p.group]), b);
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = i * 8 + j < p.K ? s * (float)((int)(word >> (4 * j) & 15u) - 8) : 0.f;
#pragma unroll
      for (int part = 0; part < PARTS; ++part) {
        out[part * W + i] = make_uint4(pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3]), pack_f16x2(v[4], v[5]), pack_f16x2(v[6], v[7]));
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= 1.f / 2048.f;
      }
    }
    return;
  }
  const int64_t m = blockIdx.x - c.w_blocks;
  const T* row = static_cast<const T*>(p.x) + m * p.ldx;
  uint32_t top = 0;
  for (int i = threadIdx.x; i * 8 < p.K; i += 256) {
    uint4 raw[sizeof(T) / 2];
    w4_load8<T>(row, i * 8, p.K, p.x_vec, raw);
    const T* e = reinterpret_cast<const T*>(raw);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t u = __float_as_uint(to_f32<T>(e[j])) & 0x7fffffffu;
      if (u < 0x7f800000u) top = max(top, u);
    }
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, tops[i]);
  const int a = w4_shift(top, 14);
  if (threadIdx.x == 0) c.row_shift[m] = a;
  uint4* out = reinterpret_cast<uint4*>(c.xh) + m * PARTS * W;
  for (int i = threadIdx.x; i < W; i += 256) {
    uint4 raw[sizeof(T) / 2];
    w4_load8<T>(row, i * 8, p.K, p.x_vec, raw);
    const T* e = reinterpret_cast<const T*>(raw);
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = ldexp_f32(to_f32<T>(e[j]), a);
#pragma unroll
    for (int part = 0; part < PARTS; ++part) {
      out[part * W + i] = make_uint4(pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3]), pack_f16x2(v[4], v[5]), pack_f16x2(v[6], v[7]));
#pragma unroll
      for (int j = 0; j < 8; ++j)  // (an infinity or NaN stands in the first part)
        v[j] = isfinite(v[j]) ? (v[j] - __half2float(__float2half_rn(v[j]))) * 2048.f : 0.f;
    }
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

constexpr int kW4Smem = 227 * 1024;

// Operand rows that fit a CTA of this shape.
template <int GROUP, int MT, int NT, int WARPS>
static int w4_fit(int Kp) {
  using Smem = W4Smem<GROUP, MT, NT, WARPS>;
  const int left = kW4Smem - Smem::total(0, Kp);
  return left <= 0 ? 0 : std::min(8 * NT, left / (Smem::red(1) + Smem::ops(1, Kp)));
}

// Rows of X that a launch takes at most, 0 where not even one fits: one strip at a time but where every SM has two and the
// registers allow it (up to 8 operand rows): X's operands are then read once for both.
struct W4Fit {
  int one, two, four, most;  // by NT
};
template <int GROUP>
static W4Fit w4_fits(int Kp, int N, int parts) {
  W4Fit f{};
  f.one = (N > 16 * num_sms() ? w4_fit<GROUP, 2, 1, 16>(Kp) : w4_fit<GROUP, 1, 1, 16>(Kp)) / parts;
  f.two = w4_fit<GROUP, 1, 2, 16>(Kp) / parts;
  f.four = w4_fit<GROUP, 1, 4, 8>(Kp) / parts;
  f.most = std::max(f.one, std::max(f.two, f.four));
  return f;
}

// linear4_kernel, which reads W once a launch, or copies and the GEMM?  16-bit rows: up to two launches, three where W has 2^26
// values.  fp32, whose copies are larger and go through the GEMM in passes: two, three from 2^22 and six from 2^26 values
// on.  Launches against copies, us, 16-bit rows: 768 -> 2304, 32 / 64 rows (1 / 2 launches) 9 and 16 / 17 and 16; 4096 -> 4096,
// 32 / 48 (2 / 3) 30 and 40 / 44 and 40; 5000 -> 4099, 32 / 48 (2 / 3) 49 and 54 / 73 and 54; 8192 -> 28672, 16 / 32 (2 / 4) 108
// and 243 / 276 and 241; 28672 -> 8192, 1 / 4 / 8 (1 / 2 / 4) 34 and 322 / 75 and 278 / 276 and 279.  fp32: 768 -> 2304, 16 / 24
// (2 / 3) 24 and 28 / 35 and 28; 4096 -> 4096, 16 / 24 (3 / 4) 81 and 92 / 116 and 93; 8192 -> 28672, 16 / 24 (6 / 8) 385 and 475 /
// 525 and 485; 28672 -> 8192, 6 / 8 (6 / 8) 612 and 724 / 815 and 723.
static bool w4_few(const mt_linear_weight4_desc& d) {
  const int64_t Kp = w4_padded(d.K);
  const int parts = d.dtype == MT_F32 ? 3 : 1;
  if (Kp > kW4Smem) return false;  // (one row's operands take 2 bytes a column)
  const int most = (d.group == 32   ? w4_fits<32>((int)Kp, (int)d.N, parts)
                    : d.group == 64 ? w4_fits<64>((int)Kp, (int)d.N, parts)
                                    : w4_fits<128>((int)Kp, (int)d.N, parts)).most;
  const int64_t values = d.N * Kp;
  const int64_t launches = d.dtype == MT_F32 ? (values < (1 << 22) ? 2 : values < (1 << 26) ? 3 : 6) : values < (1 << 26) ? 2 : 3;
  return d.M <= launches * most;
}

template <typename T, int GROUP, int MT, int NT, int WARPS>
static int linear4_launch(const Linear4Params& p, int rows_x, cudaStream_t st) {
  auto kern = linear4_kernel<T, GROUP, MT, NT, WARPS>;
  static bool attr[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!attr[dev & 63]) {
    int rc = cuda_check(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kW4Smem), "linear4 smem attribute");
    if (rc) return rc;
    attr[dev & 63] = true;
  }
  Linear4Params q = p;
  const int strips = (p.N + 15) / 16;
  const unsigned grid = (unsigned)std::min((strips + MT - 1) / MT, num_sms());
  for (int m = 0; m < p.M; m += rows_x) {
    q.x = static_cast<const T*>(p.x) + (int64_t)m * p.ldx;
    q.y = static_cast<T*>(p.y) + (int64_t)m * p.ldy;
    q.M = std::min(rows_x, p.M - m);
    kern<<<grid, WARPS * 32, W4Smem<GROUP, MT, NT, WARPS>::total(q.M * w4_parts<T>(), p.Kp), st>>>(q);
    int rc = check_launch("linear_weight4");
    if (rc) return rc;
  }
  return MT_OK;
}

// Rows of X are shared out evenly over the launches.
template <typename T, int GROUP>
static int linear4_dispatch(const Linear4Params& p, cudaStream_t st) {
  const W4Fit f = w4_fits<GROUP>(p.Kp, p.N, w4_parts<T>());
  const int launches = (p.M + f.most - 1) / f.most, rows = (p.M + launches - 1) / launches;
  if (rows <= f.one)
    return p.N > 16 * num_sms() ? linear4_launch<T, GROUP, 2, 1, 16>(p, rows, st) : linear4_launch<T, GROUP, 1, 1, 16>(p, rows, st);
  if (rows <= f.two) return linear4_launch<T, GROUP, 1, 2, 16>(p, rows, st);
  return linear4_launch<T, GROUP, 1, 4, 8>(p, rows, st);
}

template <typename T>
static int linear4_run(const Linear4Params& p, cudaStream_t st) {
  switch (p.group) {
    case 32: return linear4_dispatch<T, 32>(p, st);
    case 64: return linear4_dispatch<T, 64>(p, st);
    default: return linear4_dispatch<T, 128>(p, st);
  }
}

static int validate_linear4(const mt_linear_weight4_desc& d) {
  int rc = w4_check(d.N, d.K, d.group, d.dtype, "linear_weight4");
  if (rc) return rc;
  if (d.M < 0 || d.M > INT32_MAX || d.ldx < 0 || d.ldy < 0) return fail(MT_ERR_INVALID, "linear_weight4: bad sizes");
  if (d.M == 0 || d.N == 0) return MT_OK;
  if (!d.y || (d.K && (!d.x || !d.words || !d.scales))) return fail(MT_ERR_INVALID, "linear_weight4: null operand");
  if ((uintptr_t)d.words % 16 || (uintptr_t)d.scales % 8)
    return fail(MT_ERR_INVALID, "linear_weight4: words have to be 16-byte, scales 8-byte aligned");
  return MT_OK;
}

// Memory of the products of many rows: f16 copies of W and X and their rows' shifts.
struct W4Many {
  size_t w, x, row_shift, col_shift, gemm, total;
};
static mt_gemm_desc w4_gemm(const mt_linear_weight4_desc& d, const W4Many& w, char* ws) {
  mt_gemm_desc g{};
  g.M = d.M; g.N = d.N; g.K = w4_padded(d.K) * (d.dtype == MT_F32 ? 2 : 1); g.batch = 1;
  g.dtype = MT_F16; g.out_dtype = d.dtype;
  g.A = ws + w.x; g.lda = g.K;
  g.B = ws + w.w; g.ldb = g.K; g.b_trans = 1;
  g.D = d.y; g.ldd = d.ldy;
  g.bias = d.bias; g.bias_dtype = d.dtype;
  g.alpha = 1.f;
  return g;
}
static W4Many w4_many(const mt_linear_weight4_desc& d) {
  W4Many m{};
  const size_t row = (size_t)w4_padded(d.K) * (d.dtype == MT_F32 ? 4 : 2);  // bytes of a row of a copy
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at = align_up(at + bytes, 1024);
    return here;
  };
  m.w = take((size_t)d.N * row);
  m.x = take((size_t)d.M * row);
  m.row_shift = take((size_t)d.M * 4);
  m.col_shift = take(align_up((size_t)d.N, 32) * 4);
  m.gemm = at;
  m.total = at + gemm_workspace(w4_gemm(d, m, reinterpret_cast<char*>(1024)));
  return m;
}

constexpr int64_t kW4Pass = 1024;

template <typename T>
static int linear4_many(const mt_linear_weight4_desc& d, const Linear4Params& p, char* ws, size_t ws_bytes, cudaStream_t st) {
  const W4Many w = w4_many(d);
  W4CopyParams c{};
  c.p = p;
  c.wh = reinterpret_cast<__half*>(ws + w.w);
  c.xh = reinterpret_cast<__half*>(ws + w.x);
  c.row_shift = reinterpret_cast<int*>(ws + w.row_shift);
  c.col_shift = reinterpret_cast<int*>(ws + w.col_shift);
  c.w_blocks = (p.N + 7) / 8;
  if ((int64_t)c.w_blocks + d.M > INT32_MAX) return fail(MT_ERR_UNSUPPORTED, "linear_weight4: too many rows");
  linear4_copy_kernel<T><<<(unsigned)(c.w_blocks + p.M), 256, 0, st>>>(c);
  int rc = check_launch("linear_weight4 copies");
  if (rc) return rc;
  const mt_gemm_desc all = w4_gemm(d, w, ws);
  if (d.dtype != MT_F32) return run_gemm_shifted(all, c.row_shift, c.col_shift, ws + w.gemm, ws_bytes - w.gemm, st);
  // fp32: the tensor core's accumulator drops what does not fit in each step of 16 columns, which grows to 1e-5 of the
  // result at 4000 columns.  So the second parts have sums of their own, and the first parts' columns go 1024 at a time; Y
  // adds up the passes in fp32.
  for (int64_t k = -1; k < p.Kp && !rc; k = k < 0 ? 0 : k + kW4Pass) {
    mt_gemm_desc g = all;
    const int64_t at = k < 0 ? p.Kp : k;
    g.K = k < 0 ? p.Kp : std::min<int64_t>(kW4Pass, p.Kp - k);
    g.A = static_cast<const __half*>(all.A) + at;
    g.B = static_cast<const __half*>(all.B) + at;
    if (k >= 0) {
      g.bias = nullptr;
      g.C = g.D; g.ldc = g.ldd; g.beta = 1.f;
    }
    rc = run_gemm_shifted(g, c.row_shift, c.col_shift, ws + w.gemm, ws_bytes - w.gemm, st);
  }
  return rc;
}

size_t linear_weight4_workspace(const mt_linear_weight4_desc& d) {
  if (validate_linear4(d) || w4_few(d) || d.M == 0 || d.N == 0 || d.K == 0) return 0;
  return w4_many(d).total;
}

int run_linear_weight4(const mt_linear_weight4_desc& d, void* ws, size_t ws_bytes, cudaStream_t st) {
  int rc = validate_linear4(d);
  if (rc || d.M == 0 || d.N == 0) return rc;
  Linear4Params p{};
  p.M = (int)d.M; p.N = (int)d.N; p.K = (int)d.K; p.Kp = (int)w4_padded(d.K); p.group = (int)d.group;
  p.x = d.x; p.ldx = d.ldx;
  p.x_vec = (uintptr_t)d.x % 16 == 0 && (d.ldx * dtype_size(d.dtype)) % 16 == 0;
  p.words = reinterpret_cast<const uint32_t*>(d.words);
  p.scales = static_cast<const __nv_bfloat16*>(d.scales);
  p.bias = d.bias; p.y = d.y; p.ldy = d.ldy;
  if (!w4_few(d) && d.K > 0) {
    if (!ws || ws_bytes < linear_weight4_workspace(d)) return fail(MT_ERR_WORKSPACE, "linear_weight4: workspace too small");
    if ((uintptr_t)ws % 16) return fail(MT_ERR_INVALID, "linear_weight4: the workspace has to be 16-byte aligned");
    char* mem = static_cast<char*>(ws);
    switch (d.dtype) {
      case MT_F32: return linear4_many<float>(d, p, mem, ws_bytes, st);
      case MT_BF16: return linear4_many<__nv_bfloat16>(d, p, mem, ws_bytes, st);
      default: return linear4_many<__half>(d, p, mem, ws_bytes, st);
    }
  }
  switch (d.dtype) {
    case MT_F32: return linear4_run<float>(p, st);
    case MT_BF16: return linear4_run<__nv_bfloat16>(p, st);
    default: return linear4_run<__half>(p, st);
  }
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
