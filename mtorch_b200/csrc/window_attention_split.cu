// Attention of few query rows over many keys (16-bit keys and values, or the paged 4-bit cache):
// the keys are split over warps and CTAs, and read once for all the query rows of a key head.
//
// The products run on mma.m16n8k16 with the KEYS on the 16-row side and up to 8 * NT query rows on the
// 8-column side: S^T = K Q^T, then O^T = V^T P^T.  The work is bound by reading K and V (a decoder's step
// has 1 to 16 rows a key head), so the tensor cores only have to keep the arithmetic out of the way; with
// the keys on the M side a fragment of K or V is what a lane reads from its warp's ring (cp.async, no
// barrier between warps), 16 bytes or 8 / 4 bytes of codes at a time: the k order of a product is free, and
// the codes are unpacked into fragments with one shift and one logic instruction per pair.
//
// Codes as operands: the 4 bits of a code at the low end of a 16-bit lane ARE the number c * 2^-133 in
// bf16 (c * 2^-24 in f16), a subnormal that mma multiplies exactly; at bits 4..7 they are 16 times that.  One
// AND makes two operands, one shift serves half a word.  Queries are multiplied by a power of two (exact), one
// for the CTA's rows, that takes the largest finite value among them to 2^63..2^64 in bf16 (the products stay far from
// fp32's own subnormals, and no value passes bf16's range), to 2^14..2^15 in f16.  Channels at bits 4..7 get a sixteenth,
// which costs an f16 value bits only where it is 2^24 below the largest.  With value = zero + scale c:
//   q.k = scale (q.c) + zero sum(q)  per 64 channels,
//   o   = sum (p scale) c + sum p zero,
// with p scale rounded to bf16 (for f16 queries too, whose exponents are too few for p scale; they get the rounding's
// rest in a second product).  That rounding meets c - 8 rather than c, because what is added for zero is p (zero + 8 scale) - 8 round(p scale):
// the codes of a key centre around 8, and the error of a rounded weight is halved.  bf16 queries go without the second
// product: 24 sequences of 4096..16384 codes take 80 us without and 91 with it, and are off by 0.0017 of the result
// against 64 bits in both, which is the result's rounding to bf16.
// Over 16-bit keys the weights have two parts in both types (one part: 0.0023 off for bf16, two: 0.0016, the result's own
// rounding; 8 sequences of 4096 keys 32.2 -> 32.35 us).
//
// The running maximum is raised only when a score passes it by more than 2^8 ("lazy"): then the warp
// reduces the maximum and rescales; otherwise a block of 16 keys costs one vote.
#include <algorithm>

#include "window_attention.cuh"

namespace mt {

constexpr int kSplitWarps = 4;
constexpr float kSplitLazy = 8.0f;
constexpr int kMinChunk = 16;     // blocks of 16 keys that a CTA takes at least
constexpr int kSplitCluster = 8;  // up to so many chunks are joined within a cluster

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
// the same on accumulators of zero
template <bool F16>
__device__ __forceinline__ void mma16816_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
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
// transpose of an 8 x 8 matrix of 16-bit elements spread over the warp (row lane / 4, columns 2 (lane % 4) ..)
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// operands of codes i and i + 4 of a word: c * u, or 16 c * u for odd i (u = 2^-133 in bf16, 2^-24 in f16)
__device__ __forceinline__ uint32_t code_pair(uint32_t w, uint32_t w8, int i) {
  return (i & 2 ? w8 : w) & (i & 1 ? 0x00f000f0u : 0x000f000fu);
}
constexpr float kPow64 = 18446744073709551616.f;          // 2^64
constexpr float kPow69 = 32.f * kPow64;                    // 2^69 = 2^133 / 2^64
__device__ __forceinline__ float pow2f(int n) { return __int_as_float((n + 127) << 23); }  // -126 <= n <= 127
// |a| and |b|, the larger of each half; NaN is dropped
template <bool F16>
__device__ __forceinline__ uint32_t max_abs2(uint32_t a, uint32_t b) {
  if (F16) {
    const __half2 m = __hmax2(__habs2(*reinterpret_cast<const __half2*>(&a)), __habs2(*reinterpret_cast<const __half2*>(&b)));
    return *reinterpret_cast<const uint32_t*>(&m);
  }
  const __nv_bfloat162 m =
      __hmax2(__habs2(*reinterpret_cast<const __nv_bfloat162*>(&a)), __habs2(*reinterpret_cast<const __nv_bfloat162*>(&b)));
  return *reinterpret_cast<const uint32_t*>(&m);
}

// 16 bytes to shared memory, zeros when !live
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
// 16 bytes to shared memory where `on`
__device__ __forceinline__ void cp_async16_if(uint32_t dst, const void* src, bool on) {
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %2, 0;\n @p cp.async.cg.shared.global [%0], [%1], 16;\n}\n" ::"r"(dst),
               "l"(src), "r"((int)on)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A warp's ring of steps (KB blocks of 16 keys) in shared memory, filled by the warp's own cp.async (no barrier
// between warps).  The 16-byte chunks are placed so that the fragment reads meet no bank twice:
//   16-bit rows (8 DC chunks): chunk ch of K row r at ch ^ kswz(r), of V row r at ch ^ (r & 7);
//   rows of codes (2 DC chunks, DC halves of 32 bytes): a block's V rows in the order 0 2 4 .. 1 3 5 .., then half
//   c of the row at place r at c ^ (r / 2) for DC = 2, c ^ r for DC = 4.
template <bool PAGED, int DC, int KB>
struct SplitRing {
  static constexpr int ROW = PAGED ? 32 * DC : 128 * DC;         // bytes of a row of K or V
  static constexpr int SCALES = PAGED ? KB * 16 * 4 * DC : 0;    // bytes of a step's scales of K or V
  static constexpr int RUN = KB * 16 * ROW;                      // bytes of a step's K or V
  static constexpr int STAGE = 2 * (RUN + SCALES);
  static constexpr int STAGES = PAGED && KB == 1 ? 4 : 3;
  static constexpr int BYTES = STAGE * STAGES;                   // a warp's
  static constexpr int V = RUN, KS = 2 * RUN, VS = KS + SCALES;  // offsets in a stage; K at 0
  static_assert(!PAGED || 4 * DC * KB <= 16, "a step's scales are one instruction of the warp");
  static __device__ __forceinline__ int kswz(int r) { return ((r & 1) << 2) | ((r >> 1) & 3); }
  static __device__ __forceinline__ int half(int c, int r) { return DC == 2 ? c ^ ((r >> 1) & 1) : DC == 4 ? c ^ (r & 3) : c; }
  static __device__ __forceinline__ int vplace(int r) { return (r & 16) | ((r & 15) >> 1) | ((r & 1) << 3); }
};

// One CTA: kSplitWarps warps over one chunk of the steps (KB blocks of 16 keys, of one page) of (b, hk) for
// 8 * NT query rows.  DC: blocks of 64 channels.  CLUSTER: the chunks of a row tile are a cluster, which joins them (a
// variant of its own: the code costs registers).  In a lane, n = lane / 4 and t = lane % 4.
template <bool F16, bool PAGED, int DC, int NT, int KB, bool CLUSTER>
__global__ void __launch_bounds__(kSplitWarps * 32, DC * NT <= 2 ? (PAGED ? 4 : 2) : 1) attn_split_kernel(const AttnParams p) {
  using T = typename std::conditional<F16, __half, __nv_bfloat16>::type;
  constexpr int ROWS = 8 * NT;
  constexpr int DP = 64 * DC;
  constexpr bool PF16 = F16 && !PAGED;  // type of P and V's operands
  using Ring = SplitRing<PAGED, DC, KB>;
  constexpr int STEP = 16 * KB;  // keys
  static_assert(ROWS * (DP + 4) * 4 <= Ring::BYTES, "the ring holds a warp's result at the end");
  extern __shared__ __align__(16) uint8_t split_smem[];
  __shared__ float2 sml[kSplitWarps][ROWS];
  __shared__ RowKeys srk[ROWS];
  __shared__ float sinv[ROWS];
  __shared__ float2 sfin[ROWS];  // maximum and sum of the CTA's share

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = lane >> 2, t = lane & 3;
  const int bk = blockIdx.y, b = bk / p.Hkv, hk = bk % p.Hkv;
  const int r0 = blockIdx.z * ROWS, nr = min(ROWS, p.rows - r0);
  const SeqPos sp = seq_pos(p, b, PAGED);
  const int q0 = r0 / p.g, q1 = (r0 + nr - 1) / p.g;  // queries of the rows
  const int pmin = sp.start + q0, pmax = sp.start + q1;
  const BlockList bl = block_list<STEP>(p, sp, pmin, pmax);

  // chunk: about the same for every CTA of the grid, so that sequences of different lengths fill it evenly
  int per = bl.count;
  if (gridDim.x > 1) {
    float total = 0.f;  // steps of the whole batch; a guide only, but the same in every CTA
    for (int i = lane; i < p.B; i += 32) {
      const SeqPos s = seq_pos(p, i, PAGED);
      total += (float)block_list<STEP>(p, s, s.start + q0, s.start + q1).count;
    }
    total = warp_sum(total) * (float)(p.Hkv * gridDim.z) / (float)p.target;
    per = max(kMinChunk / KB, (int)fminf(ceilf(total), (float)bl.count));
    const int chunks = min((bl.count + per - 1) / per, (int)gridDim.x);
    per = chunks > 0 ? (bl.count + chunks - 1) / chunks : 1;  // of one length within the sequence
  }
  const int i0 = (int)min((int64_t)blockIdx.x * per, (int64_t)bl.count), i1 = min(bl.count, i0 + per);
  const int64_t out_row = ((int64_t)blockIdx.x * p.B * p.Hkv + bk) * p.rows + r0;
  if (i0 >= i1 && gridDim.x > 1 && !CLUSTER) {
    if (threadIdx.x < nr) p.part_ml[out_row + threadIdx.x] = make_float2(-INFINITY, 0.f);
    return;
  }

  // keys that each row sees; keys that all rows see (ra.hi, rz.lo, ra.sk), that any row sees (ra.lo, rz.hi, rz.sk)
  if (threadIdx.x < ROWS) srk[threadIdx.x] = row_keys(p, sp, sp.start + (r0 + min((int)threadIdx.x, nr - 1)) / p.g);
  const RowKeys ra = row_keys(p, sp, pmin), rz = row_keys(p, sp, pmax);
  __syncthreads();

  constexpr float kShift = PAGED ? 64.f : 0.f;  // p = 2^(score - m + kShift)
  float m[NT][2], thr[NT][2], negm[NT][2], l[NT][2], cor[NT][DC][2], o[DC][4][NT][4];
  float psum[PAGED ? DC : 1][NT][4];  // sums of the rounded weights, as a product with ones
#pragma unroll
  for (int x = 0; x < NT; ++x)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      m[x][j] = thr[x][j] = -INFINITY;
      negm[x][j] = kShift;
      l[x][j] = 0.f;
#pragma unroll
      for (int c = 0; c < DC; ++c) cor[x][c][j] = 0.f;
    }
#pragma unroll
  for (int c = 0; c < DC; ++c)
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
#pragma unroll
        for (int j = 0; j < 4; ++j) o[c][j][x][e] = 0.f;
        psum[PAGED ? c : 0][x][e] = 0.f;
      }

  // ---- loads: steps of keys into this warp's ring ----
  uint8_t* ring = split_smem + warp * Ring::BYTES;
  const uint32_t ring_u32 = smem_u32(ring);
  const int64_t es = sizeof(T);
  // sources: paged, this lane's chunk of a step's words and scales; dense, the head's first row
  constexpr int CH = PAGED ? 2 * DC : 8 * DC;  // chunks of a row
  const uint8_t *ksrc, *vsrc, *ssrc = nullptr;
  if (PAGED) {
    const uint64_t head = ((uint64_t)hk << p.page_shift);  // rows
    ksrc = reinterpret_cast<const uint8_t*>(p.words[0]) + head * Ring::ROW + lane * 16;
    vsrc = reinterpret_cast<const uint8_t*>(p.words[1]) + head * Ring::ROW + lane * 16;
    ssrc = reinterpret_cast<const uint8_t*>(p.scales[lane >> 4]) + head * (4 * DC) + (lane & 15) * 16;
  } else {
    ksrc = static_cast<const uint8_t*>(p.k) + (b * p.ks[0] + hk * p.ks[1]) * es;
    vsrc = static_cast<const uint8_t*>(p.v) + (b * p.vs[0] + hk * p.vs[1]) * es;
  }
  // where chunk j * 32 + lane goes (the offsets of j > 0 are constants for DC <= 2)
  auto kdst = [&](int j) {
    const int r = (j * 32 + lane) / CH, ch = (j * 32 + lane) % CH;
    return PAGED ? r * Ring::ROW + Ring::half(ch >> 1, r) * 32 + (ch & 1) * 16 : r * Ring::ROW + (ch ^ Ring::kswz(r)) * 16;
  };
  auto vdst = [&](int j) {
    const int r = (j * 32 + lane) / CH, ch = (j * 32 + lane) % CH;
    const int v = Ring::vplace(r);
    return PAGED ? v * Ring::ROW + Ring::half(ch >> 1, v) * 32 + (ch & 1) * 16 : r * Ring::ROW + (ch ^ (r & 7)) * 16;
  };
  const uint32_t kdst0 = kdst(0), vdst0 = vdst(0);
  const uint32_t sdst = (lane >> 4 ? Ring::VS : Ring::KS) + (lane & 15) * 16;
  const int32_t* table = p.table + b * p.table_stride;
  // row (in units of 16) of step i in the cache's arrays (of head 0), kNoRow where its page does not exist; steps
  // past the chunk look at its last one
  constexpr uint32_t kNoRow = 0xffffffffu;
  const uint32_t page_blocks = (uint32_t)p.Hkv << (p.page_shift - 4);
  auto cache_row = [&](int i) -> uint32_t {
    const int k0 = bl.block(min(i, i1 - 1)) * STEP;
    const int page = __ldg(table + (k0 >> p.page_shift));
    const uint32_t row = (uint32_t)page * page_blocks + ((k0 & ((1 << p.page_shift) - 1)) >> 4);
    return i < i1 && (uint32_t)page < (uint32_t)p.num_pages ? row : kNoRow;
  };
  // brings step i to `stage`
  auto load = [&](int i, uint32_t row, int stage) {
    const uint32_t dst = ring_u32 + stage * Ring::STAGE;
    if (PAGED) {
      const bool on = row != kNoRow;
      const uint8_t* ks = ksrc + (uint64_t)row * (16 * Ring::ROW);
      const uint8_t* vs = vsrc + (uint64_t)row * (16 * Ring::ROW);
#pragma unroll
      for (int j = 0; j < KB * DC; ++j) {
        // 32 chunks are 16 / DC rows: rows + 8 (DC = 2) or + 16 keep the swizzle, V's places move by 4 and 16
        const uint32_t ko = DC <= 2 ? kdst0 + j * 512 : kdst(j);
        const uint32_t vo = DC == 1 ? vdst0 + j * 512 : DC == 2 ? vdst0 + ((j & 1) * 4 + (j >> 1) * 16) * Ring::ROW : vdst(j);
        cp_async16_if(dst + ko, ks + j * 512, on);
        cp_async16_if(dst + Ring::V + vo, vs + j * 512, on);
      }
      cp_async16_if(dst + sdst, ssrc + (uint64_t)row * (16 * 4 * DC), on && (lane & 15) < 4 * DC * KB);
    } else if (i < i1) {
      const int k0 = bl.block(i) * STEP;
      // channels past D are zeros; RPI rows an instruction where rows do not straddle instructions
      if (32 % CH == 0 && k0 + STEP <= sp.n && (k0 + STEP - 1 <= rz.hi && (k0 >= ra.lo || k0 + STEP - 1 < rz.sk))) {
        constexpr int RPI = 32 / CH > 0 ? 32 / CH : 1;
        const int r = lane / CH, ch = lane % CH;
        const uint8_t* ks = ksrc + ((k0 + r) * p.ks[2] + ch * 8) * es;
        const uint8_t* vs = vsrc + ((k0 + r) * p.vs[2] + ch * 8) * es;
        const int64_t kstep = RPI * p.ks[2] * es, vstep = RPI * p.vs[2] * es;
        const bool in = ch * 8 < p.D;
#pragma unroll
        for (int j = 0; j < STEP / RPI; ++j) {
          cp_async16(dst + kdst(j), in ? ks : ksrc, in);
          cp_async16(dst + Ring::V + vdst(j), in ? vs : vsrc, in);
          ks += kstep;
          vs += vstep;
        }
      } else {
#pragma unroll 1
        for (int j = 0; j < STEP * CH / 32; ++j) {
          const int r = (j * 32 + lane) / CH, ch = (j * 32 + lane) % CH;
          const int key = k0 + r;
          const bool in = key < sp.n && ch * 8 < p.D;
          // a key that no row sees counts as zeros in V, whatever stands there
          const bool seen = in && ((key >= ra.lo && key <= rz.hi) || key < rz.sk);
          cp_async16(dst + kdst(j), in ? ksrc + (key * p.ks[2] + ch * 8) * es : ksrc, in);
          cp_async16(dst + Ring::V + vdst(j), seen ? vsrc + (key * p.vs[2] + ch * 8) * es : vsrc, seen);
        }
      }
    }
    cp_async_commit();
  };

  // this lane's fragments in a stage
  int koff[DC], voff[DC];
#pragma unroll
  for (int c = 0; c < DC; ++c) {
    koff[c] = n * Ring::ROW + Ring::half(c, n) * 32 + t * 8;              // rows n, n + 8
    voff[c] = Ring::V + t * Ring::ROW + Ring::half(c, t) * 32 + n * 4;    // places t (+ 8, 4, 12): rows 2t, 2t + 1, 2t + 8, 2t + 9
  }

  int i = i0 + warp;
  uint32_t row_next = kNoRow;   // of the next step to bring: looked up a step early
  uint32_t missing_steps = 0;   // bit s: step i + s W has no page
  if (PAGED && i0 < i1) row_next = cache_row(i);
#pragma unroll
  for (int s = 0; s < Ring::STAGES - 1; ++s) {
    load(i + s * kSplitWarps, row_next, s);
    if (PAGED && i0 < i1) {
      missing_steps |= (uint32_t)(row_next == kNoRow) << s;
      row_next = cache_row(i + (s + 1) * kSplitWarps);
    }
  }
  // Q fragments (while the first keys are on their way): dense, 8 channels at 32 c + 8 t of row n; paged, the channel order of the codes' pairs
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
      alignas(16) T raw[8];
      if (p.q_vec) {  // (D is a multiple of 8)
        *reinterpret_cast<uint4*>(raw) = live && base < p.D ? __ldg(reinterpret_cast<const uint4*>(src + base)) : make_uint4(0, 0, 0, 0);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) raw[j] = live && base + j < p.D ? src[(base + j) * p.qs[3]] : from_f32<T>(0.f);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) qf[x][c][j] = reinterpret_cast<const uint32_t*>(raw)[j];
    }
  }
  int kq = 0;  // queries over codes are multiplied by 2^kq
  if (PAGED) {
    constexpr uint32_t kInf = F16 ? 0x7c00u : 0x7f80u;
    uint32_t top2 = 0;
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int c = 0; c < 2 * DC; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) top2 = max_abs2<F16>(top2, qf[x][c][j]);
    uint32_t top = __reduce_max_sync(0xffffffffu, max(top2 & 0xffffu, top2 >> 16));
    if (top >= kInf) {  // an infinity: the largest of the others
      top = 0;
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int c = 0; c < 2 * DC; ++c)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t u0 = qf[x][c][j] & 0x7fffu, u1 = qf[x][c][j] >> 16 & 0x7fffu;
            top = max(top, max(u0 < kInf ? u0 : 0u, u1 < kInf ? u1 : 0u));
          }
      top = __reduce_max_sync(0xffffffffu, top);
    }
    const uint16_t top16 = (uint16_t)top;
    kq = (F16 ? 14 : 63) + 127 - (int)(__float_as_uint(to_f32<T>(*reinterpret_cast<const T*>(&top16))) >> 23);
  }
  const float q_up[2] = {pow2f(kq >> 1), pow2f(kq - (kq >> 1))};
  // scores, their running maximum m and the bound `thr` past which it is raised are in units of 1 / score_scale
  // (base 2); over codes a product counts 2^-24 (f16) or 2^-133.  Past 2^120 (queries near the end of bf16's range)
  // it makes no difference between scores that far apart.
  const int unit = (F16 ? 24 : 133) - kq;
  const float score_scale =
      !PAGED ? fmaxf(fabsf(p.scale_log2), 1e-30f)
             : fmaxf(fminf(fabsf(p.scale_log2) * pow2f(unit >> 1) * pow2f(unit - (unit >> 1)), kPow64 * 72057594037927936.f),
                     1.17549435e-38f);  // 2^120, 2^-126
#pragma unroll
  for (int x = 0; x < NT; ++x)
#pragma unroll
    for (int c = 0; c < 2 * DC; ++c) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = qf[x][c][j];
      const T* raw = reinterpret_cast<const T*>(w);
      float v[8];
      uint16_t u[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = to_f32<T>(raw[j]);
        if (p.scale_log2 < 0.f) v[j] = -v[j];  // the maximum is taken of unscaled scores
        if (PAGED) v[j] = v[j] * q_up[0] * q_up[1];
        const T h = from_f32<T>(PAGED && (j & 1) ? v[j] * 0.0625f : v[j]);
        u[j] = *reinterpret_cast<const uint16_t*>(&h);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        qf[x][c][j] = PAGED ? (u[j] | (uint32_t)u[j + 4] << 16) : (u[2 * j] | (uint32_t)u[2 * j + 1] << 16);
      if (PAGED) {
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) s += v[j];
        s *= F16 ? 1.f / 16777216.f : 1.f / kPow69 / kPow64;  // the unit of q.c below
        s += __shfl_xor_sync(0xffffffffu, s, 1);
        s += __shfl_xor_sync(0xffffffffu, s, 2);
        const float s0 = __shfl_sync(0xffffffffu, s, 8 * t), s1 = __shfl_sync(0xffffffffu, s, 8 * t + 4);
        qsum[x][c >> 1][0] = (c & 1) ? qsum[x][c >> 1][0] + s0 : s0;
        qsum[x][c >> 1][1] = (c & 1) ? qsum[x][c >> 1][1] + s1 : s1;
      }
    }
  int stage = 0;
  for (; i < i1; i += kSplitWarps) {
    const int k0 = bl.block(i) * STEP;
    cp_async_wait<Ring::STAGES - 2>();
    __syncwarp();
    const uint8_t* st = ring + stage * Ring::STAGE;
    // ---- S^T = K Q^T: sc[.][.][0,1] key n of a block, [2,3] key n + 8; columns 2t, 2t + 1 ----
    float sc[KB][NT][4];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      if (PAGED) {
#pragma unroll
        for (int c = 0; c < DC; ++c) {
          float acc[NT][4];
          uint2 kq[2];
          float2 ksc[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            kq[h] = *reinterpret_cast<const uint2*>(st + koff[c] + (kb * 16 + 8 * h) * Ring::ROW);
            ksc[h] = __half22float2(*reinterpret_cast<const __half2*>(st + n * (4 * DC) + Ring::KS + ((kb * 16 + 8 * h) * DC + c) * 4));
          }
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint32_t w0 = u ? kq[0].y : kq[0].x, w1 = u ? kq[1].y : kq[1].x;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t a[4] = {code_pair(w0, w0 >> 8, 2 * e), code_pair(w1, w1 >> 8, 2 * e),
                                     code_pair(w0, w0 >> 8, 2 * e + 1), code_pair(w1, w1 >> 8, 2 * e + 1)};
#pragma unroll
              for (int x = 0; x < NT; ++x) {
                if (u + e == 0) mma16816_zero<F16>(acc[x], a, qf[x][2 * c + u][2 * e], qf[x][2 * c + u][2 * e + 1]);
                else mma16816<F16>(acc[x], a, qf[x][2 * c + u][2 * e], qf[x][2 * c + u][2 * e + 1]);
              }
            }
          }
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int x = 0; x < NT; ++x)
#pragma unroll
              for (int j = 0; j < 2; ++j)
                sc[kb][x][2 * h + j] =
                    fmaf(ksc[h].y, qsum[x][c][j], c ? fmaf(ksc[h].x, acc[x][2 * h + j], sc[kb][x][2 * h + j])
                                                    : ksc[h].x * acc[x][2 * h + j]);
        }
      } else {
#pragma unroll
        for (int c = 0; c < 2 * DC; ++c) {
          const uint8_t* r0p = st + (kb * 16 + n) * Ring::ROW;
          const uint4 k0v = *reinterpret_cast<const uint4*>(r0p + (((c * 4 + t) ^ Ring::kswz(n)) * 16));
          const uint4 k1v = *reinterpret_cast<const uint4*>(r0p + 8 * Ring::ROW + (((c * 4 + t) ^ Ring::kswz(n)) * 16));
          const uint32_t a0[4] = {k0v.x, k1v.x, k0v.y, k1v.y}, a1[4] = {k0v.z, k1v.z, k0v.w, k1v.w};
#pragma unroll
          for (int x = 0; x < NT; ++x) {
            if (c == 0) mma16816_zero<F16>(sc[kb][x], a0, qf[x][c][0], qf[x][c][1]);
            else mma16816<F16>(sc[kb][x], a0, qf[x][c][0], qf[x][c][1]);
            mma16816<F16>(sc[kb][x], a1, qf[x][c][2], qf[x][c][3]);
          }
        }
      }
    }

    // ---- softmax ----
    const bool missing = PAGED && (missing_steps & 1u);
    const bool full = !missing && k0 + STEP - 1 <= ra.hi && (k0 >= rz.lo || k0 + STEP - 1 < ra.sk);
    if (!full) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (missing || !srk[8 * x + 2 * t + (e & 1)].sees(k0 + kb * 16 + n + 8 * (e >> 1))) sc[kb][x][e] = -INFINITY;
      if (PAGED) {  // scales of slots that hold nothing may be NaN
        for (int j = lane; j < STEP * DC; j += 32) {
          const int key = k0 + j / DC;
          if (missing || !((key >= ra.lo && key <= rz.hi) || key < rz.sk))
            reinterpret_cast<uint32_t*>(ring + stage * Ring::STAGE + Ring::VS)[j] = 0u;
        }
        __syncwarp();
      }
    }
    bool over = false;
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float top = max_nan(sc[0][x][j], sc[0][x][2 + j]);
        if (KB == 2) top = max_nan(top, max_nan(sc[KB - 1][x][j], sc[KB - 1][x][2 + j]));
        over |= !(top <= thr[x][j]);  // (a NaN too: it stays in m, and all the weights to come are NaN)
      }
    if (__any_sync(0xffffffffu, over)) {
#pragma unroll
      for (int x = 0; x < NT; ++x) {
        float corr[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float mx = max_nan(sc[0][x][j], sc[0][x][2 + j]);
          if (KB == 2) mx = max_nan(mx, max_nan(sc[KB - 1][x][j], sc[KB - 1][x][2 + j]));
          mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          mx = max_nan(mx, m[x][j]);
          corr[j] = m[x][j] == -INFINITY ? 0.f : ex2f((m[x][j] - mx) * score_scale);
          m[x][j] = mx;
          thr[x][j] = mx + kSplitLazy / score_scale;
          negm[x][j] = mx == -INFINITY ? kShift : fmaf(-mx, score_scale, kShift);
          l[x][j] *= corr[j];
#pragma unroll
          for (int c = 0; c < DC; ++c) {
            cor[x][c][j] *= corr[j];
            if (PAGED) psum[PAGED ? c : 0][x][j] *= corr[j];
          }
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
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sc[kb][x][e] = ex2f(fmaf(sc[kb][x][e], score_scale, negm[x][e & 1]));
          l[x][e & 1] += sc[kb][x][e];
        }

    // ---- O^T += V^T P^T ----
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      uint32_t pb[NT][2], pl[NT][2];  // weights, and what their rounding left (over codes: of f16 queries)
      if (!PAGED) {
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float e0 = sc[kb][x][2 * h], e1 = sc[kb][x][2 * h + 1];
            if (PF16) {
              const uint32_t w = pack_f16x2(e0, e1);
              const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
              pb[x][h] = transpose8x8(w);
              pl[x][h] = transpose8x8(pack_f16x2(e0 - f.x, e1 - f.y));
            } else {
              const uint32_t w = pack_bf16x2(e0, e1);
              pb[x][h] = transpose8x8(w);
              pl[x][h] = transpose8x8(pack_bf16x2(e0 - __uint_as_float(w << 16), e1 - __uint_as_float(w & 0xffff0000u)));
            }
          }
      }
#pragma unroll
      for (int c = 0; c < DC; ++c) {
        if (PAGED) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float2 vsc =
                __half22float2(*reinterpret_cast<const __half2*>(st + n * (4 * DC) + Ring::VS + ((kb * 16 + 8 * h) * DC + c) * 4));
            const float f = vsc.x, z = fmaf(8.f, vsc.x, vsc.y);
#pragma unroll
            for (int x = 0; x < NT; ++x) {
              cor[x][c][0] = fmaf(sc[kb][x][2 * h], z, cor[x][c][0]);
              cor[x][c][1] = fmaf(sc[kb][x][2 * h + 1], z, cor[x][c][1]);
              const float e0 = sc[kb][x][2 * h] * f, e1 = sc[kb][x][2 * h + 1] * f;
              const uint32_t w = pack_bf16x2(e0, e1);
              pb[x][h] = transpose8x8(w);
              if (F16)
                pl[x][h] = transpose8x8(pack_bf16x2(e0 - __uint_as_float(w << 16), e1 - __uint_as_float(w & 0xffff0000u)));
            }
          }
          const uint32_t ones[4] = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
#pragma unroll
          for (int x = 0; x < NT; ++x) {
            mma16816<false>(psum[PAGED ? c : 0][x], ones, pb[x][0], pb[x][1]);
            if (F16) mma16816<false>(psum[PAGED ? c : 0][x], ones, pl[x][0], pl[x][1]);
          }
          uint32_t vq[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            vq[e] = *reinterpret_cast<const uint32_t*>(st + voff[c] + (kb * 16 + (e & 1) * 8 + (e >> 1) * 4) * Ring::ROW);
          const uint32_t lo0 = __byte_perm(vq[0], vq[1], 0x5410), hi0 = __byte_perm(vq[0], vq[1], 0x7632);
          const uint32_t lo1 = __byte_perm(vq[2], vq[3], 0x5410), hi1 = __byte_perm(vq[2], vq[3], 0x7632);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t w0 = j < 2 ? lo0 : hi0, w1 = j < 2 ? lo1 : hi1;
            const int q = (2 * j) & 3;  // codes 2j and 2j + 1 at bits 4q, 4q + 4 of both halves
            const uint32_t a[4] = {code_pair(w0, w0 >> 8, q), code_pair(w0, w0 >> 8, q + 1), code_pair(w1, w1 >> 8, q),
                                   code_pair(w1, w1 >> 8, q + 1)};
#pragma unroll
            for (int x = 0; x < NT; ++x) {
              mma16816<false>(o[c][j][x], a, pb[x][0], pb[x][1]);
              if (F16) mma16816<false>(o[c][j][x], a, pl[x][0], pl[x][1]);
            }
          }
        } else {
          uint32_t e0[4], e1[4], e2[4], e3[4];
          auto row = [&](int r, uint32_t (&w)[4]) {
            const uint4 x = *reinterpret_cast<const uint4*>(st + Ring::V + (kb * 16 + r) * Ring::ROW + (((c * 8 + n) ^ (r & 7)) * 16));
            w[0] = x.x;
            w[1] = x.y;
            w[2] = x.z;
            w[3] = x.w;
          };
          row(2 * t, e0);
          row(2 * t + 1, e1);
          row(2 * t + 8, e2);
          row(2 * t + 9, e3);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t a[4] = {__byte_perm(e0[j], e1[j], 0x5410), __byte_perm(e0[j], e1[j], 0x7632),
                                   __byte_perm(e2[j], e3[j], 0x5410), __byte_perm(e2[j], e3[j], 0x7632)};
#pragma unroll
            for (int x = 0; x < NT; ++x) {
              mma16816<PF16>(o[c][j][x], a, pb[x][0], pb[x][1]);
              mma16816<PF16>(o[c][j][x], a, pl[x][0], pl[x][1]);
            }
          }
        }
      }
    }
    __syncwarp();
    int next = stage + Ring::STAGES - 1;  // the stage that the step before this one emptied
    if (next >= Ring::STAGES) next -= Ring::STAGES;
    load(i + (Ring::STAGES - 1) * kSplitWarps, row_next, next);
    if (++stage == Ring::STAGES) stage = 0;
    if (PAGED) {
      missing_steps = (missing_steps | (uint32_t)(row_next == kNoRow) << (Ring::STAGES - 1)) >> 1;
      row_next = cache_row(i + Ring::STAGES * kSplitWarps);
    }
  }
  cp_async_wait<0>();

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
      if (PAGED)
#pragma unroll
        for (int c = 0; c < DC; ++c) cor[x][c][j] = fmaf(-8.f, psum[PAGED ? c : 0][x][j], cor[x][c][j]);
      if (n == 0) sml[warp][8 * x + 2 * t + j] = make_float2(m[x][j] * score_scale, PAGED ? l[x][j] / kPow64 : l[x][j]);
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
      f[x][j] = m[x][j] == -INFINITY ? 0.f : ex2f(m[x][j] * score_scale - top);
    }
  if (threadIdx.x < nr) {  // maximum and sum of the CTA's share, or 1 / sum
    const int r = threadIdx.x;
    float top = -INFINITY, ls = 0.f;
#pragma unroll
    for (int w = 0; w < kSplitWarps; ++w) top = max_nan(top, sml[w][r].x);
#pragma unroll
    for (int w = 0; w < kSplitWarps; ++w)
      if (sml[w][r].x != -INFINITY) ls = fmaf(sml[w][r].y, ex2f(sml[w][r].x - top), ls);
    if (CLUSTER) sfin[r] = make_float2(top, ls);
    if (gridDim.x > 1 && !CLUSTER) p.part_ml[out_row + r] = make_float2(top, ls);
    sinv[r] = ls == 0.f ? 0.f : 1.f / ls;
  }
  __syncwarp();
  float* mine = reinterpret_cast<float*>(ring);
#pragma unroll
  for (int c = 0; c < DC; ++c)
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float v[8];  // channels 64 c + 8 n ..
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float y = o[c][j][x][2 * e + r];  // codes at bits 4..7 (rows n + 8) count 16 times
            if (PAGED) y = fmaf(y, e ? kPow69 / 16.f : kPow69, cor[x][c][r] / kPow64);
            v[2 * j + e] = y * f[x][r];
          }
        float4* dst = reinterpret_cast<float4*>(mine + (8 * x + 2 * t + r) * (DP + 4) + 64 * c + 8 * n);
        dst[0] = make_float4(v[0], v[1], v[2], v[3]);
        dst[1] = make_float4(v[4], v[5], v[6], v[7]);
      }
  __syncthreads();
  if constexpr (CLUSTER) {
    // each CTA adds up its warps, then takes its part of the outputs over all the CTAs' sums in their shared memory,
    // which saves the join's launch (4 tokens on 1000 keys of 4 heads of codes: 12.4 -> 10.7 us)
    constexpr int U = ROWS * DP / 4 / (kSplitWarps * 32);
    float4 own[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = threadIdx.x + u * kSplitWarps * 32, r = i / (DP / 4), d = i % (DP / 4) * 4;
      own[u] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kSplitWarps; ++w) {
        const float4 y = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(split_smem + w * Ring::BYTES) + r * (DP + 4) + d);
        own[u] = make_float4(own[u].x + y.x, own[u].y + y.y, own[u].z + y.z, own[u].w + y.w);
      }
    }
    __syncthreads();
    float* sum = reinterpret_cast<float*>(split_smem);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = threadIdx.x + u * kSplitWarps * 32;
      *reinterpret_cast<float4*>(sum + i / (DP / 4) * (DP + 4) + i % (DP / 4) * 4) = own[u];
    }
    cluster_sync();
    const int n_cta = gridDim.x;
    for (int i = blockIdx.x * kSplitWarps * 32 + threadIdx.x; i < nr * (DP / 4); i += n_cta * kSplitWarps * 32) {
      const int r = i / (DP / 4), d = i % (DP / 4) * 4;
      float2 ml[kSplitCluster];
      float top = -INFINITY, ls = 0.f;
#pragma unroll
      for (int c = 0; c < kSplitCluster; ++c) {
        ml[c] = make_float2(-INFINITY, 0.f);
        if (c < n_cta) asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(ml[c].x), "=f"(ml[c].y) : "r"(mapa_rank(&sfin[r], c)) : "memory");
        top = fmaxf(top, ml[c].x);
      }
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int c = 0; c < kSplitCluster; ++c) {
        if (ml[c].x == -INFINITY) continue;  // (a chunk that saw nothing)
        const float f = ex2f(ml[c].x - top);
        float4 y;
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(y.x), "=f"(y.y), "=f"(y.z), "=f"(y.w)
                     : "r"(mapa_rank(sum + r * (DP + 4) + d, c))
                     : "memory");
        ls = fmaf(ml[c].y, f, ls);
        x = make_float4(fmaf(y.x, f, x.x), fmaf(y.y, f, x.y), fmaf(y.z, f, x.z), fmaf(y.w, f, x.w));
      }
      if (d >= p.D) continue;  // D is a multiple of 8
      const float inv = ls == 0.f ? 0.f : 1.f / ls;
      const int qi = (r0 + r) / p.g, h = hk * p.g + (r0 + r) % p.g;
      T* dst = static_cast<T*>(p.o) + b * p.os[0] + h * p.os[1] + qi * p.os[2];
      const float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) dst[(d + j) * p.os[3]] = from_f32<T>(v[j] * inv);
    }
    __syncwarp();
    cluster_sync();  // the sums stay until everybody has read them
    return;
  }
  for (int i = threadIdx.x; i < nr * (DP / 4); i += kSplitWarps * 32) {
    const int r = i / (DP / 4), d = i % (DP / 4) * 4;
    float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kSplitWarps; ++w) {
      const float4 y = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(split_smem + w * Ring::BYTES) + r * (DP + 4) + d);
      x[0] += y.x;
      x[1] += y.y;
      x[2] += y.z;
      x[3] += y.w;
    }
    if (d >= p.D) continue;  // D is a multiple of 8
    if (gridDim.x > 1) {
      *reinterpret_cast<float4*>(p.part_o + (out_row + r) * p.D + d) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
      const int qi = (r0 + r) / p.g, h = hk * p.g + (r0 + r) % p.g;
      T* dst = static_cast<T*>(p.o) + b * p.os[0] + h * p.os[1] + qi * p.os[2];
#pragma unroll
      for (int j = 0; j < 4; ++j) dst[(d + j) * p.os[3]] = from_f32<T>(x[j] * sinv[r]);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// host

// Query rows a key head that the split kernel takes (more rows: the tiled kernels read K and V less often).
int split_tile_rows(int64_t rows) { return rows <= 8 ? 8 : 16; }

// A grid of at most two CTAs an SM, all resident at once, is joined in clusters; larger ones in a launch of their own: a
// cluster starts when all its CTAs have room, and those without keys hold theirs until it ends.  Join's launch, cluster at
// 2000 keys, 8 key heads of 128 channels, 16-bit rows, 1, 4, 12, 40 sequences: 10.4, 12.4, 25, 54 us against 10.4, 12.4,
// 35, 147; codes of 64 channels, 1, 2, 4, 12, 40: 8.5, 9.8, 10.4, 14.9, 31 against 8.3, 8.6, 9.9, 16.9, 41.
bool split_joins_in_cluster(int64_t bk, int64_t rows, int splits) {
  const int tr = split_tile_rows(rows);
  return splits > 1 && splits <= kSplitCluster && bk * ((rows + tr - 1) / tr) * splits <= 2 * num_sms();
}

int split_count(int64_t bk, int64_t rows, int64_t keys) {
  const int tr = split_tile_rows(rows);
  const int64_t ctas = bk * ((rows + tr - 1) / tr);
  const int64_t most = std::max<int64_t>(1, (keys / 16 + kMinChunk - 1) / kMinChunk);
  // a few times more than fill the GPU: room for sequences longer than the mean
  const int64_t want = (16LL * num_sms() + ctas - 1) / ctas;
  return (int)std::max<int64_t>(1, std::min<int64_t>(std::min(want, most), 512));
}

template <bool F16, bool PAGED, int DC, int NT, int KB, bool CLUSTER>
static int split_launch_cluster(AttnParams& p, dim3 grid, cudaStream_t st) {
  constexpr int smem = kSplitWarps * SplitRing<PAGED, DC, KB>::BYTES;
  auto kern = attn_split_kernel<F16, PAGED, DC, NT, KB, CLUSTER>;
  static int resident[64] = {};  // CTAs an SM holds
  int dev = 0;
  cudaGetDevice(&dev);
  int& res = resident[dev & 63];
  if (!res) {
    int n = 0;
    int rc = cuda_check(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem),
                        "attention split smem attribute");
    if (!rc)
      rc = cuda_check(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, kSplitWarps * 32, smem),
                      "attention split occupancy");
    if (rc) return rc;
    res = std::max(n, 1);
  }
  // chunks for three waves over the codes (arithmetic counts, the waves even out) and one and a half over 16-bit
  // rows, where a chunk's start costs more: 24 sequences of 4096..16384 codes take 111, 83, 83, 79, 80 us with 2, 3,
  // 8, 12, 16 CTAs an SM (4 resident), 8 sequences of 4096 16-bit keys 33, 32, 35, 37 with 2, 3, 4, 8 (2 resident)
  p.target = num_sms() * (PAGED ? 3 * res : (3 * res + 1) / 2);
  if (!CLUSTER) {
    kern<<<grid, kSplitWarps * 32, smem, st>>>(p);
    return check_launch("attention_split");
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kSplitWarps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at = {};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = grid.x;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  int rc = cuda_check(cudaLaunchKernelEx(&cfg, kern, (const AttnParams)p), "attention_split");
  return rc ? rc : check_launch("attention_split");
}

template <bool F16, bool PAGED, int DC, int NT, int KB>
static int split_launch_kernel(AttnParams& p, dim3 grid, cudaStream_t st) {
  return p.cluster ? split_launch_cluster<F16, PAGED, DC, NT, KB, true>(p, grid, st)
                   : split_launch_cluster<F16, PAGED, DC, NT, KB, false>(p, grid, st);
}

template <bool F16, bool PAGED, int DC>
static int split_launch_dc(AttnParams& p, cudaStream_t st) {
  const int tr = split_tile_rows(p.rows);
  const int64_t tiles = (p.rows + tr - 1) / tr;
  if ((int64_t)p.B * p.Hkv > 65535 || tiles > 65535)
    return fail(MT_ERR_UNSUPPORTED, "window_attention: batch * key heads or rows past the grid");
  dim3 grid((unsigned)p.splits, (unsigned)(p.B * p.Hkv), (unsigned)tiles);
  // two blocks a step where pages allow it and the scales fit one instruction: control and votes are shared
  // (cache4_batch of the benchmark, pages of 64)
  constexpr int KB2 = PAGED && DC <= 2 ? 2 : 1;
  if (KB2 == 2 && p.page_shift >= 5) {
    return tr == 8 ? split_launch_kernel<F16, PAGED, DC, 1, KB2>(p, grid, st)
                   : split_launch_kernel<F16, PAGED, DC, 2, KB2>(p, grid, st);
  }
  return tr == 8 ? split_launch_kernel<F16, PAGED, DC, 1, 1>(p, grid, st)
                 : split_launch_kernel<F16, PAGED, DC, 2, 1>(p, grid, st);
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
  p.cluster = split_joins_in_cluster((int64_t)p.B * p.Hkv, p.rows, p.splits);
  if (paged && ((int64_t)p.num_pages * p.Hkv << (p.page_shift - 4)) >= 0xffffffffLL)
    return fail(MT_ERR_UNSUPPORTED, "kv_cache4_attention: more than 2^36 tokens and heads in the cache");
  if (dtype == MT_F16) return paged ? split_launch<true, true>(p, st) : split_launch<true, false>(p, st);
  return paged ? split_launch<false, true>(p, st) : split_launch<false, false>(p, st);
}

}  // namespace mt
