// Products of few rows with a weight held in 4 bits, and its packing.
//
// W[n, k] = scale[n, k / group] * (code - 8).  Words of 8 codes; in each block of 128 columns word w
// is stored at place (w % 4) * 4 + w / 4 (see mtorch_cuda.h).
//
// linear4_kernel: Y^T = W X^T on mma.m16n8k16 with the weight's rows on the 16-row side and up to 8 * NT rows of X
// on the 8-column side.  Bound by reading W: a lane's 16 bytes are words t, t + 4, t + 8, t + 12 of a block of 128
// columns, which are its fragments for 8 products of 16 columns; no shared memory stands between.  A code's
// 4 bits at the low end of a 16-bit lane are the number c * 2^-133 in bf16 (c * 2^-24 in f16), a subnormal that mma
// multiplies exactly, at bits 4..7 sixteen times that: one AND makes two operands, one shift serves half a word.  X
// is scaled to match while it is loaded (bf16 by 2^64; channels at bits 4..7 by another 1/16).  The code's offset
// is taken off with one more product per step, of a constant row of eights: the same fp32 rounding as the
// others, so nothing is left of it but sum x (c - 8).  Per group of columns: y += scale (acc - acc8), in fp32.
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

constexpr int kW4Warps = 8;

// Rows of the products that one row of X becomes.
template <typename T> constexpr int w4_parts() { return sizeof(T) == 4 ? 3 : 1; }

// Eight columns of X at k as operands: pairs (0, 4), (1, 5), (2, 6), (3, 7), scaled as the codes' places ask.
// `part`: which of the three bf16 parts of fp32.
template <typename T>
__device__ __forceinline__ uint4 w4_load_x(const T* x, int k, int K, bool vec, int part) {
  float v[8];
  if (vec && k + 8 <= K) {
    uint4 raw[sizeof(T) / 2];
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) raw[i] = __ldg(reinterpret_cast<const uint4*>(x + k) + i);
    const T* e = reinterpret_cast<const T*>(raw);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = to_f32<T>(e[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = k + j < K ? to_f32<T>(x[k + j]) : 0.f;
  }
  constexpr bool F16 = std::is_same<T, __half>::value;
  if (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float hi = __bfloat162float(__float2bfloat16_rn(v[j]));
      const float mid = __bfloat162float(__float2bfloat16_rn(v[j] - hi));
      v[j] = part == 0 ? hi : part == 1 ? mid : v[j] - hi - mid;
    }
  }
  constexpr float even = F16 ? 1.f : 18446744073709551616.f, odd = even / 16.f;  // 2^64, 2^60
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float f = j & 1 ? odd : even;
    w[j] = F16 ? pack_f16x2(v[j] * f, v[j + 4] * f) : pack_bf16x2(v[j] * f, v[j + 4] * f);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// One CTA: 16 * MT rows of W (outputs) against 8 * NT rows of operands; the 8 warps take blocks of 128 columns in
// turn and add up in shared memory.
template <typename T, int GROUP, int MT, int NT>
__global__ void __launch_bounds__(kW4Warps * 32, MT * NT < 4 ? 2 : 1) linear4_kernel(const Linear4Params p) {
  constexpr bool F16 = std::is_same<T, __half>::value;
  constexpr int PARTS = w4_parts<T>();
  constexpr int GPB = 128 / GROUP;  // groups of a block
  constexpr int OUT = 16 * MT, COL = 8 * NT;
  __shared__ float red[kW4Warps][COL][OUT + 4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * OUT, row0 = blockIdx.y * COL;
  const int rows = p.M * PARTS;
  const int blocks = p.Kp / 128;

  const T* xrow[NT];
  int part[NT];
  bool live[NT];
#pragma unroll
  for (int x = 0; x < NT; ++x) {
    const int r = row0 + 8 * x + n;
    live[x] = r < rows;
    part[x] = r % PARTS;
    xrow[x] = static_cast<const T*>(p.x) + (int64_t)(live[x] ? r / PARTS : 0) * p.ldx;
  }
  // rows n and n + 8 of each tile of W; rows past N repeat the last
  const uint4* wrow[MT][2];
  const __nv_bfloat16* srow[MT][2];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t r = min(n0 + 16 * i + n + 8 * h, p.N - 1);
      wrow[i][h] = reinterpret_cast<const uint4*>(p.words + r * (p.Kp / 8)) + t;
      srow[i][h] = p.scales + r * (p.Kp / GROUP);
    }

  float y[MT][NT][4];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int e = 0; e < 4; ++e) y[i][x][e] = 0.f;

  uint4 w[MT][2];
  __nv_bfloat16 sc[MT][2][GPB];
  auto load_w = [&](int kb) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        w[i][h] = __ldg(wrow[i][h] + kb * 4);
        if (GPB == 4) *reinterpret_cast<uint2*>(sc[i][h]) = __ldg(reinterpret_cast<const uint2*>(srow[i][h] + kb * GPB));
        else if (GPB == 2) *reinterpret_cast<uint32_t*>(sc[i][h]) = __ldg(reinterpret_cast<const uint32_t*>(srow[i][h] + kb * GPB));
        else sc[i][h][0] = srow[i][h][kb];
      }
  };
  if (warp < blocks) load_w(warp);
  for (int kb = warp; kb < blocks; kb += kW4Warps) {
    uint4 wc[MT][2];
    float sf[MT][2][GPB];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        wc[i][h] = w[i][h];
#pragma unroll
        for (int g = 0; g < GPB; ++g) sf[i][h][g] = __bfloat162float(sc[i][h][g]);
      }
    if (kb + kW4Warps < blocks) load_w(kb + kW4Warps);
    float acc[MT][NT][4], acc8[NT][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // 32 columns
      if ((j * 32) % GROUP == 0) {
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            acc8[x][e] = 0.f;
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[i][x][e] = 0.f;
          }
      }
      uint4 xb[NT];
#pragma unroll
      for (int x = 0; x < NT; ++x)
        xb[x] = live[x] ? w4_load_x<T>(xrow[x], kb * 128 + j * 32 + t * 8, p.K, p.x_vec, part[x]) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t eights[4] = {0x00080008u, 0x00080008u, 0x00800080u, 0x00800080u};
#pragma unroll
        for (int x = 0; x < NT; ++x) w4_mma<F16>(acc8[x], eights, e ? xb[x].z : xb[x].x, e ? xb[x].w : xb[x].y);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          uint32_t w0 = j == 0 ? wc[i][0].x : j == 1 ? wc[i][0].y : j == 2 ? wc[i][0].z : wc[i][0].w;
          uint32_t w1 = j == 0 ? wc[i][1].x : j == 1 ? wc[i][1].y : j == 2 ? wc[i][1].z : wc[i][1].w;
          if (e) {
            w0 >>= 8;
            w1 >>= 8;
          }
          const uint32_t a[4] = {w0 & 0x000f000fu, w1 & 0x000f000fu, w0 & 0x00f000f0u, w1 & 0x00f000f0u};
#pragma unroll
          for (int x = 0; x < NT; ++x) w4_mma<F16>(acc[i][x], a, e ? xb[x].z : xb[x].x, e ? xb[x].w : xb[x].y);
        }
      }
      if ((j * 32 + 32) % GROUP == 0) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int x = 0; x < NT; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              y[i][x][e] = fmaf(sf[i][e >> 1][j * 32 / GROUP], acc[i][x][e] - acc8[x][e], y[i][x][e]);
      }
    }
  }
  constexpr float unit = F16 ? 16777216.f : 590295810358705651712.f;  // 2^24, 2^69
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int e = 0; e < 4; ++e) red[warp][8 * x + 2 * t + (e & 1)][16 * i + n + 8 * (e >> 1)] = y[i][x][e] * unit;
  __syncthreads();
  const int m0 = row0 / PARTS, ms = min(COL / PARTS, p.M - m0);
  for (int i = threadIdx.x; i < ms * OUT; i += kW4Warps * 32) {
    const int m = i / OUT, c = i % OUT;
    if (n0 + c >= p.N) continue;
    float v = 0.f;
#pragma unroll
    for (int q = 0; q < PARTS; ++q)
#pragma unroll
      for (int k = 0; k < kW4Warps; ++k) v += red[k][m * PARTS + q][c];
    if (p.bias) v += to_f32<T>(static_cast<const T*>(p.bias)[n0 + c]);
    static_cast<T*>(p.y)[(int64_t)(m0 + m) * p.ldy + n0 + c] = from_f32<T>(v);
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

// Rows of X that go through linear4_kernel; more go through an unpacked copy of W and the tensor-core GEMM.
constexpr int64_t kW4MaxRows = 64;

template <typename T, int GROUP, int MT, int NT>
static void linear4_launch(const Linear4Params& p, cudaStream_t st) {
  constexpr int per = 8 * NT / w4_parts<T>();  // rows of X a tile
  Linear4Params q = p;
  dim3 grid((unsigned)((p.N + 16 * MT - 1) / (16 * MT)), 1);
  // fp32: 8 NT operand rows hold (8 NT / 3) whole rows of X
  for (int m = 0; m < p.M; m += per) {
    q.x = static_cast<const T*>(p.x) + (int64_t)m * p.ldx;
    q.y = static_cast<T*>(p.y) + (int64_t)m * p.ldy;
    q.M = std::min(per, p.M - m);
    linear4_kernel<T, GROUP, MT, NT><<<grid, kW4Warps * 32, 0, st>>>(q);
  }
}

template <typename T, int GROUP>
static void linear4_dispatch(const Linear4Params& p, cudaStream_t st) {
  const int rows = p.M * w4_parts<T>();
  // 64 rows of W a CTA where that still gives every SM two CTAs: X's operands are then made once for four tiles
  bool wide = p.N >= 64 * 2 * num_sms(), mid = p.N >= 32 * 2 * num_sms();
  if (getenv("MT_W4")) { int v = atoi(getenv("MT_W4")); wide = v == 4; mid = v >= 2; }
  if (rows <= 8) {
    if (wide) linear4_launch<T, GROUP, 4, 1>(p, st);
    else if (mid) linear4_launch<T, GROUP, 2, 1>(p, st);
    else linear4_launch<T, GROUP, 1, 1>(p, st);
  } else if (rows <= 16) {
    if (mid) linear4_launch<T, GROUP, 2, 2>(p, st);
    else linear4_launch<T, GROUP, 1, 2>(p, st);
  } else {
    if (mid) linear4_launch<T, GROUP, 2, 4>(p, st);
    else linear4_launch<T, GROUP, 1, 4>(p, st);
  }
}

template <typename T>
static int linear4_run(const Linear4Params& p, cudaStream_t st) {
  switch (p.group) {
    case 32: linear4_dispatch<T, 32>(p, st); break;
    case 64: linear4_dispatch<T, 64>(p, st); break;
    default: linear4_dispatch<T, 128>(p, st);
  }
  return check_launch("linear_weight4");
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

// Unpacked weight rows: a pitch of 16-byte multiples for the GEMM's tensor maps.
static int64_t w4_pitch(const mt_linear_weight4_desc& d) { return (d.K + 7) / 8 * 8; }

static mt_gemm_desc w4_gemm(const mt_linear_weight4_desc& d, void* w) {
  mt_gemm_desc g{};
  g.M = d.M; g.N = d.N; g.K = d.K; g.batch = 1;
  g.dtype = g.out_dtype = d.dtype;
  g.A = d.x; g.lda = d.ldx;
  g.B = w; g.ldb = w4_pitch(d); g.b_trans = 1;
  g.D = d.y; g.ldd = d.ldy;
  g.bias = d.bias; g.bias_dtype = d.dtype;
  g.alpha = 1.f;
  return g;
}
static size_t w4_copy_bytes(const mt_linear_weight4_desc& d) {
  return align_up((size_t)d.N * w4_pitch(d) * dtype_size(d.dtype), 1024);
}

size_t linear_weight4_workspace(const mt_linear_weight4_desc& d) {
  if (validate_linear4(d) || d.M <= kW4MaxRows || d.N == 0 || d.K == 0) return 0;
  return w4_copy_bytes(d) + gemm_workspace(w4_gemm(d, reinterpret_cast<void*>(1024)));
}

int run_linear_weight4(const mt_linear_weight4_desc& d, void* ws, size_t ws_bytes, cudaStream_t st) {
  int rc = validate_linear4(d);
  if (rc || d.M == 0 || d.N == 0) return rc;
  if (d.M > kW4MaxRows && d.K > 0) {
    if (!ws || ws_bytes < linear_weight4_workspace(d)) return fail(MT_ERR_WORKSPACE, "linear_weight4: workspace too small");
    rc = run_weight4_unpack(ws, d.dtype, w4_pitch(d), d.words, d.scales, d.N, d.K, d.group, st);
    if (rc) return rc;
    const size_t copy = w4_copy_bytes(d);
    return run_gemm(w4_gemm(d, ws), static_cast<char*>(ws) + copy, ws_bytes - copy, st);
  }
  Linear4Params p{};
  p.M = (int)d.M; p.N = (int)d.N; p.K = (int)d.K; p.Kp = (int)w4_padded(d.K); p.group = (int)d.group;
  p.x = d.x; p.ldx = d.ldx;
  p.x_vec = (uintptr_t)d.x % 16 == 0 && (d.ldx * dtype_size(d.dtype)) % 16 == 0;
  p.words = reinterpret_cast<const uint32_t*>(d.words);
  p.scales = static_cast<const __nv_bfloat16*>(d.scales);
  p.bias = d.bias; p.y = d.y; p.ldy = d.ldy;
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
