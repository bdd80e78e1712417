// Attention with a sliding window and sinks on the 5th-generation tensor cores, for many queries
// (bf16 / f16, head dims up to 128).
//
// One CTA = two tiles of 128 query rows of one (batch entry, head); the tiles of 128 keys that any of the rows
// sees (the sinks' tiles, then the window's) stream through TMA rings of K and V, 128-byte swizzled.
//   warp 0      producer: Q once and K(0) (before the barriers' first use), then K(j + 1), V(j), ..
//   warp 1      MMA issuer: S_x = Q_x K^T into TMEM (fp32), then O_x += P_x V with P_x as the TMEM operand: it
//               overwrites the low half of S_x's columns, so the probabilities never touch shared memory.
//   warps 4..11 one softmax warpgroup per query tile, one row per thread: the row's 128 scores are read once into
//               registers (these warps take the registers that the first four give up); p = 2^(s scale - m) in fp32, the sums in fp32, P rounded to 16 bits.
// O stays in TMEM for all the key tiles.  The running maximum m is raised only when a score passes it by more than
// 2^8; the warp then rescales its rows of O in TMEM.  While one warpgroup exponentiates, the tensor core works for
// the other tile: 128 x 128 scores take 1024 cycles of the exponential unit (16 a cycle) and, at head dim 128,
// 1024 cycles of the tensor core, so both are near their limits.
//
// P has the bits of its 16-bit type and no second part (the split kernel's has): the rest would be a second P V product,
// 1000 cycles more for the tensor core that already works 2400 of a tile pair's 3160, and five more instructions a
// pair of scores for the softmax, which is what the rest waits for.  A prompt of 8192 tokens (bf16) is off by 0.0022 of 64 bits with it, 0.0016 is the rounding of
// the result alone (f16: 0.00025 and 0.00021).
//
// Keys that a row does not see weigh exactly zero: their K may be anything, their V anything finite (a NaN or an infinity in V
// at a key that only other rows of the tile see is 0 * NaN).  NaN among the scores of a row makes the row NaN.
//
// The products of one thread complete in order, so the barrier behind S_x(j + 1) also says that O_x holds tile j,
// and P_x(j) is read before S_x(j + 1) overwrites it.  All waits are bounded (timeout -> device error word, return).
#include "window_attention.cuh"

namespace mt {

MT_STATUS_READER(read_status_window_attention)

constexpr int kWaTile = 128;  // queries per tile, keys per tile
constexpr int kWaThreads = 384;  // producer, MMA issuer, two idle warps; two softmax warpgroups
// registers: 384 threads start with 168 each; 128 * 72 + 256 * 216 = 384 * 168
constexpr int kWaRegsIssue = 72, kWaRegsSoftmax = 216;
constexpr float kWaLazy = 8.0f;
constexpr int kWaPoly = 2;  // of 8 pairs of exponentials, those on the FMA pipe

struct WaParams {
  AttnParams a;
  int out_vec;  // output rows take 16-byte stores
};

__device__ __forceinline__ float wa_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// maxima that keep a NaN: a row with a NaN among the scores that it sees has to end as NaN
__device__ __forceinline__ float wa_max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float wa_max2(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ uint64_t wa_pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void wa_unpack2(uint64_t r, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r));
}
__device__ __forceinline__ uint64_t wa_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t wa_add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// subnormal numbers to zero
__device__ __forceinline__ uint64_t wa_flush2(uint64_t a) {
  uint64_t r;
  asm("mul.rn.ftz.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(wa_pack2(1.f, 1.f)));
  return r;
}

// maximum of 128 values, eight independent chains
__device__ __forceinline__ float wa_max128(const uint32_t (&r)[128]) {
  float m[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) m[i] = __uint_as_float(r[i]);
#pragma unroll
  for (int k = 8; k + 16 <= 128; k += 16)
#pragma unroll
    for (int i = 0; i < 8; ++i) m[i] = wa_max3(m[i], __uint_as_float(r[k + i]), __uint_as_float(r[k + 8 + i]));
#pragma unroll
  for (int i = 0; i < 8; ++i) m[i] = wa_max2(m[i], __uint_as_float(r[120 + i]));
  return wa_max3(wa_max3(m[0], m[1], m[2]), wa_max3(m[3], m[4], m[5]), wa_max2(m[6], m[7]));
}

// 2^x of two values on the FMA pipe: x = i + f with |f| <= 1/2, a polynomial for 2^f (minimax in relative error by the
// Remez exchange: 7.5e-5 for degree 3, 2.6e-6 for degree 4, a fraction of P's rounding to bf16 / f16), i added to
// the exponent.  x at or below -126 (a hidden key's is -inf) gives 0: there the polynomial's value is just below
// 2^-126, and the last product flushes it, so that a hidden key's V counts nothing however large it is.
template <bool F16>
__device__ __forceinline__ void wa_exp2_poly(float& a0, float& a1) {
  a0 = fmaxf(a0, -126.f);
  a1 = fmaxf(a1, -126.f);
  const uint64_t x = wa_pack2(a0, a1);
  const uint64_t t = wa_add2(x, wa_pack2(12582912.f, 12582912.f));  // 1.5 * 2^23: rounds to a whole number
  const uint64_t i = wa_add2(t, wa_pack2(-12582912.f, -12582912.f));
  const uint64_t f = wa_fma2(i, wa_pack2(-1.f, -1.f), x);
  uint64_t y;
  if (F16) {
    y = wa_fma2(wa_pack2(0.009570102f, 0.009570102f), f, wa_pack2(0.05591786f, 0.05591786f));
    y = wa_fma2(y, f, wa_pack2(0.24024745f, 0.24024745f));
    y = wa_fma2(y, f, wa_pack2(0.69312181f, 0.69312181f));
    y = wa_fma2(y, f, wa_pack2(0.99999926f, 0.99999926f));
  } else {
    y = wa_fma2(wa_pack2(0.05517167f, 0.05517167f), f, wa_pack2(0.24261112f, 0.24261112f));
    y = wa_fma2(y, f, wa_pack2(0.69326099f, 0.69326099f));
    y = wa_fma2(y, f, wa_pack2(0.99992807f, 0.99992807f));
  }
  float t0, t1;
  wa_unpack2(t, t0, t1);
  wa_unpack2(y, a0, a1);
  a0 = __uint_as_float(__float_as_uint(a0) + (__float_as_uint(t0) << 23));
  a1 = __uint_as_float(__float_as_uint(a1) + (__float_as_uint(t1) << 23));
  wa_unpack2(wa_flush2(wa_pack2(a0, a1)), a0, a1);
}

// bits c of the 32 columns from `base` on that a row sees
__device__ __forceinline__ uint32_t wa_row_bits(const RowKeys& rk, int base) {
  const int lo = rk.lo - base, hi = rk.hi - base, sk = rk.sk - base;
  const uint32_t ge = lo <= 0 ? ~0u : lo >= 32 ? 0u : ~0u << lo;
  const uint32_t le = hi < 0 ? 0u : hi >= 31 ? ~0u : (2u << hi) - 1u;
  const uint32_t first = sk <= 0 ? 0u : sk >= 32 ? ~0u : (1u << sk) - 1u;
  return (ge & le) | first;
}

__device__ __forceinline__ void wa_tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

// Products issued by the elected lane of a warp that runs as one: addresses, loop counters and descriptors then stay
// in uniform registers, which the instruction takes its operands from.  A descriptor is passed as its low word; the
// high word is the same for all operands here (8 rows of 128 bytes = 1024, version, 128-byte swizzle).
constexpr uint32_t kWaDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
// low words: rows along K (Q, K: the next 64 channels are another tile); rows along N (V: 64 channels of one key are
// 128 bytes, the next 64 channels lie `chunk` bytes on)
__device__ __forceinline__ uint32_t wa_desc_k(uint32_t addr) { return ((addr & 0x3FFFF) >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t wa_desc_n(uint32_t addr, uint32_t chunk) {
  return ((addr & 0x3FFFF) >> 4) | ((chunk >> 4) << 16);
}
// D (+)= A B^T, both in shared memory
__device__ __forceinline__ void wa_mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t acc,
                                          uint32_t leader) {
  asm volatile(
      "{\n .reg .pred p, q;\n .reg .b64 da, db;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n mov.b64 da, {%1, %6};\n"
      " mov.b64 db, {%2, %6};\n @q tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n}\n" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(acc), "r"(leader), "n"(kWaDescHi)
      : "memory");
}
// D (+)= A B with A in TMEM (16-bit, two K elements a column)
__device__ __forceinline__ void wa_mma_ts(uint32_t d, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc, uint32_t acc,
                                          uint32_t leader) {
  asm volatile(
      "{\n .reg .pred p, q;\n .reg .b64 db;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n mov.b64 db, {%2, %6};\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n}\n" ::"r"(d),
      "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"(acc), "r"(leader), "n"(kWaDescHi)
      : "memory");
}
__device__ __forceinline__ void wa_commit(uint64_t* bar, uint32_t leader) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
      " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(smem_u32(bar)),
      "r"(leader)
      : "memory");
}
__device__ __forceinline__ uint32_t wa_elect() {
  uint32_t r;
  asm volatile("{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n selp.u32 %0, 1, 0, q;\n}\n" : "=r"(r));
  return r;
}

// After a wait that expired: what this CTA has in flight may still land, so nothing leaves before it has, or a bound.
__device__ __forceinline__ void wa_drain(uint64_t* bar, uint32_t parity) {
  const long long start = clock64();
  while (!mbar_try_wait(bar, parity) && clock64() - start < kWaitBudgetCycles / 8) {
  }
}

template <int DP>
struct WaCfg {
  static constexpr int TILE = kWaTile * DP * 2;  // bytes of a tile of Q, K or V
  static constexpr int CHUNK = kWaTile * 128;    // 64 channels of a tile
  static constexpr int STAGES_K = DP == 128 ? 3 : 4, STAGES_V = DP == 128 ? 2 : 4;
  static constexpr int SMEM = (2 + STAGES_K + STAGES_V) * TILE + 1024 + 512;
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

template <int DP, bool F16>
__global__ void __launch_bounds__(kWaThreads, 1)
    window_attention_sm100_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                                  const __grid_constant__ CUtensorMap tmV, const __grid_constant__ WaParams wp) {
  using Cfg = WaCfg<DP>;
  constexpr int CHUNKS = DP / 64;
  constexpr int FMT = F16 ? 0 : 1;
  constexpr uint32_t idesc_s = make_idesc(FMT, kWaTile, kWaTile);
  constexpr uint32_t idesc_o = make_idesc(FMT, kWaTile, DP) | (1u << 16);  // B (V) MN-major
  const AttnParams& p = wp.a;

  extern __shared__ uint8_t wa_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(wa_smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + 2 * Cfg::TILE;
  uint8_t* sV = sK + Cfg::STAGES_K * Cfg::TILE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + Cfg::STAGES_V * Cfg::TILE);
  uint64_t* q_full = bars;                        // 1
  uint64_t* v_raw = bars + 1;                     // a V tile whose tail is zeroed before use
  uint64_t* k_full = bars + 2;
  uint64_t* k_empty = k_full + Cfg::STAGES_K;
  uint64_t* v_full = k_empty + Cfg::STAGES_K;
  uint64_t* v_empty = v_full + Cfg::STAGES_V;
  uint64_t* s_full = v_empty + Cfg::STAGES_V;     // [2]
  uint64_t* p_full = s_full + 2;                  // [2][2]: the first and the second 64 keys of P_x
  uint64_t* o_done = p_full + 4;                  // [2]
  uint64_t* mma_idle = o_done + 2;                // after an expired wait: the products issued so far are done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mma_idle + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // the last queries first: with a causal mask they have the most key tiles, and the short CTAs fill the end
  const int bh = blockIdx.x, b = bh / p.H, h = bh % p.H, hk = h / p.g;
  const int qbase = (gridDim.y - 1 - blockIdx.y) * (2 * kWaTile);
  const SeqPos sp = seq_pos(p, b, false);

  // key tiles: of both query tiles together, and of each
  const int qlast = min(p.Sq, qbase + 2 * kWaTile) - 1;
  const BlockList bl = block_list<kWaTile>(p, sp, sp.start + qbase, sp.start + qlast);
  auto tiles_of = [&](int x) -> BlockList {
    const int q0 = qbase + x * kWaTile, q1 = min(p.Sq, q0 + kWaTile) - 1;
    return q1 < q0 ? BlockList{0, 0, 0} : block_list<kWaTile>(p, sp, sp.start + q0, sp.start + q1);
  };
  // step i of the list concerns the query tile whose list is t
  auto active = [&](const BlockList& t, int i) -> bool {
    const int tile = bl.block(i);
    return i < bl.count && (tile < t.first || (tile >= t.from && tile < t.from + t.count - t.first));
  };

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(v_raw, 1);
    for (int s = 0; s < Cfg::STAGES_K; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
    }
    for (int s = 0; s < Cfg::STAGES_V; ++s) {
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&s_full[x], 1);
      mbar_init(&p_full[2 * x], kWaTile);
      mbar_init(&p_full[2 * x + 1], kWaTile);
      mbar_init(&o_done[x], 1);
    }
    mbar_init(mma_idle, 1);
    *abort_flag = 0;
    fence_barrier_init();
    if (bl.count > 0) {  // Q and the first K tile come while the rest is set up
      mbar_arrive_expect_tx(q_full, 2 * Cfg::TILE);
      for (int x = 0; x < 2; ++x)
        for (int c = 0; c < CHUNKS; ++c)
          tma_load_4d(sQ + x * Cfg::TILE + c * Cfg::CHUNK, &tmQ, q_full, c * 64, qbase + x * kWaTile, h, b);
      mbar_arrive_expect_tx(&k_full[0], Cfg::TILE);
      for (int c = 0; c < CHUNKS; ++c)
        tma_load_4d(sK + c * Cfg::CHUNK, &tmK, &k_full[0], c * 64, bl.block(0) * kWaTile, hk, b);
    }
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;  // S_x at 128 x, O_x at 256 + 128 x

  if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kWaRegsIssue));
  if (warp == 0) {
    // ---------------- producer ----------------
    int ks = 1, vs = 0;
    uint32_t kph = 0, vph = 0;
    bool ok = true;
    int k_loads = bl.count > 0, v_loads = 0;  // so far, without the tile of V that is fixed (it can only be the last one)
    bool raw_load = false;
    auto load_k = [&](int i) {
      if (lane == 0 && ok) {
        ok = mbar_wait(&k_empty[ks], kph ^ 1, 71, abort_flag);
        if (ok) {
          ++k_loads;
          mbar_arrive_expect_tx(&k_full[ks], Cfg::TILE);
          for (int c = 0; c < CHUNKS; ++c)
            tma_load_4d(sK + ks * Cfg::TILE + c * Cfg::CHUNK, &tmK, &k_full[ks], c * 64, bl.block(i) * kWaTile, hk, b);
        }
      }
      if (++ks == Cfg::STAGES_K) {
        ks = 0;
        kph ^= 1;
      }
    };
    for (int i = 0; i < bl.count; ++i) {
      if (i + 1 < bl.count) load_k(i + 1);
      const int k0 = bl.block(i) * kWaTile;
      // keys at n and beyond may hold anything: a tile with such keys of the tensor gets zeros there
      const int live = min(kWaTile, sp.n - k0);
      const bool fix = live < kWaTile && sp.n < p.Sk;
      if (lane == 0 && ok) {
        ok = mbar_wait(&v_empty[vs], vph ^ 1, 72, abort_flag);
        if (ok) {
          uint64_t* bar = fix ? v_raw : &v_full[vs];
          raw_load = fix;
          v_loads += !fix;
          mbar_arrive_expect_tx(bar, Cfg::TILE);
          for (int c = 0; c < CHUNKS; ++c)
            tma_load_4d(sV + vs * Cfg::TILE + c * Cfg::CHUNK, &tmV, bar, c * 64, k0, hk, b);
          if (fix) ok = mbar_wait(v_raw, 0, 73, abort_flag);  // at most one tile of a sequence
        }
      }
      ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
      if (!ok) break;
      if (fix) {
        for (int j = live * 8 + lane; j < kWaTile * 8; j += 32)
          for (int c = 0; c < CHUNKS; ++c)
            *reinterpret_cast<uint4*>(sV + vs * Cfg::TILE + c * Cfg::CHUNK + j * 16) = make_uint4(0, 0, 0, 0);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_full[vs]);
      }
      if (++vs == Cfg::STAGES_V) {
        vs = 0;
        vph ^= 1;
      }
    }
    if (lane == 0 && *abort_flag && bl.count > 0) {
      wa_drain(q_full, 0);
      for (int n = max(0, k_loads - Cfg::STAGES_K); n < k_loads; ++n) wa_drain(&k_full[n % Cfg::STAGES_K], (n / Cfg::STAGES_K) & 1);
      for (int n = max(0, v_loads - Cfg::STAGES_V); n < v_loads; ++n) wa_drain(&v_full[n % Cfg::STAGES_V], (n / Cfg::STAGES_V) & 1);
      if (raw_load) wa_drain(v_raw, 0);
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer (the whole warp runs it, one lane issues) ----------------
    if (bl.count > 0) {
      const uint32_t leader = wa_elect();
      const uint32_t q_lo = wa_desc_k(smem_u32(sQ)), k_lo = wa_desc_k(smem_u32(sK)), v_lo = wa_desc_n(smem_u32(sV), Cfg::CHUNK);
      const BlockList t0 = tiles_of(0), t1 = tiles_of(1);
      auto wait = [&](uint64_t* bar, uint32_t parity, int site) -> bool {
        return __all_sync(0xffffffffu, mbar_wait(bar, parity, site, abort_flag));
      };
      int ks = 0, vs = 0;
      uint32_t kph = 0, vph = 0;
      int done0 = 0, done1 = 0;
      auto issue_s = [&](int x) {
        const uint32_t qa = q_lo + x * (Cfg::TILE >> 4), ka = k_lo + ks * (Cfg::TILE >> 4);
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
          const int off = ((kk / 4) * Cfg::CHUNK + (kk % 4) * 32) >> 4;
          wa_mma_ss(tmem + x * 128, qa + off, ka + off, idesc_s, kk > 0, leader);
        }
        wa_commit(&s_full[x], leader);
      };
      // O_x += P_x V: the first half's products run under the second half's exponentials
      auto issue_pv = [&](int x, int done) -> bool {
        const uint32_t va = v_lo + vs * (Cfg::TILE >> 4);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (!wait(&p_full[2 * x + half], done & 1, 77)) return false;
          tc_fence_after();
#pragma unroll
          for (int kk = half * 4; kk < half * 4 + 4; ++kk)
            wa_mma_ts(tmem + 256 + x * 128, tmem + x * 128 + kk * 8, va + kk * (2048 >> 4), idesc_o, done > 0 || kk > 0, leader);
        }
        return true;
      };
      bool ok = wait(q_full, 0, 74) && wait(&k_full[0], 0, 75);
      bool a0 = active(t0, 0), a1 = active(t1, 0);
      if (ok) {
        tc_fence_after();
        if (a0) issue_s(0);
        if (a1) issue_s(1);
        wa_commit(&k_empty[0], leader);
        ks = 1;
      }
      for (int i = 0; ok && i < bl.count; ++i) {
        const bool more = i + 1 < bl.count;
        const bool n0 = active(t0, i + 1), n1 = active(t1, i + 1);
        // every tile has to arrive before its stage is handed back, also one that no row needs
        ok = wait(&v_full[vs], vph, 76);
        if (ok && a0) {
          ok = issue_pv(0, done0);
          if (++done0 == t0.count) wa_commit(&o_done[0], leader);
        }
        ok = ok && (!more || wait(&k_full[ks], kph, 78));
        tc_fence_after();
        if (ok && n0) issue_s(0);
        if (ok && a1) {
          ok = issue_pv(1, done1);
          if (++done1 == t1.count) wa_commit(&o_done[1], leader);
        }
        if (ok && n1) issue_s(1);
        if (!ok) break;
        wa_commit(&v_empty[vs], leader);
        if (++vs == Cfg::STAGES_V) {
          vs = 0;
          vph ^= 1;
        }
        if (more) {
          wa_commit(&k_empty[ks], leader);
          if (++ks == Cfg::STAGES_K) {
            ks = 0;
            kph ^= 1;
          }
        }
        a0 = n0;
        a1 = n1;
      }
      if (!ok || *abort_flag) {
        wa_commit(mma_idle, leader);
        wa_drain(mma_idle, 0);
      }
    }
  } else if (warp >= 4) {
    // ---------------- softmax ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kWaRegsSoftmax));
    const int x = (warp - 4) >> 2;
    const BlockList mine = tiles_of(x);
    const int quarter = warp & 3;  // the TMEM lanes that this warp can reach
    const int row = quarter * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const uint32_t t_s = tmem + x * 128 + lane_off, t_o = tmem + 256 + x * 128 + lane_off;
    const int q0 = qbase + x * kWaTile, qi = q0 + row;
    // keys that all rows of the tile see: up to all_hi, from all_lo on or below all_sk
    const RowKeys ra = row_keys(p, sp, sp.start + q0);
    const int all_hi = ra.hi, all_sk = ra.sk, all_lo = row_keys(p, sp, sp.start + min(q0 + kWaTile, p.Sq) - 1).lo;
    const float sl = p.scale_log2;
    const uint64_t sl2 = wa_pack2(sl, sl);
    float m = -INFINITY, thr = -INFINITY, l = 0.f;
    bool ok = true;
    int k = 0;
    for (int i = 0; i < bl.count; ++i) {
      if (!active(mine, i)) continue;
      if (!mbar_wait(&s_full[x], k & 1, 79, abort_flag)) {
        ok = false;
        break;
      }
      tc_fence_after();
      uint32_t r[128];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(t_s + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&r[c * 32]));
      tmem_ld_wait();
      const int k0 = bl.block(i) * kWaTile;
      if (!(k0 + kWaTile - 1 <= all_hi && (k0 >= all_lo || k0 + kWaTile - 1 < all_sk))) {
        const RowKeys rk = row_keys(p, sp, sp.start + min(qi, p.Sq - 1));
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t bits = wa_row_bits(rk, k0 + w * 32);
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (!(bits & (1u << c))) r[w * 32 + c] = 0xff800000u;
        }
      }
      const float top = wa_max128(r);
      // A NaN stays in m (the comparison with it is false), as does what infinity - infinity gives: from then on
      // every weight of the row is NaN.  The polynomial alone would turn a NaN score into a number.
      if (__any_sync(0xffffffffu, !(top <= thr))) {
        float mn = wa_max2(m, top);
        if (mn == INFINITY) mn = NAN;
        const float corr = m == -INFINITY ? 0.f : wa_ex2((m - mn) * sl);
        m = mn;
        thr = m + kWaLazy / sl;
        l *= corr;
        if (k > 0) {  // O holds the tiles before this one (S of this tile is complete)
#pragma unroll
          for (int c = 0; c < DP; c += 16) {
            uint32_t v[16];
            asm volatile(
                "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
                  "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                : "r"(t_o + c));
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * corr);
            tmem_st16(t_o + c, v);
          }
        }
      }
      const float negm = m == -INFINITY ? 0.f : -m * sl;
      const uint64_t negm2 = wa_pack2(negm, negm);
      uint64_t sum[2] = {wa_pack2(0.f, 0.f), wa_pack2(0.f, 0.f)};
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int c = half * 32; c < half * 32 + 32; ++c) {  // in place: word c of P from scores 2c, 2c + 1
          float a0, a1;
          wa_unpack2(wa_fma2(wa_pack2(__uint_as_float(r[2 * c]), __uint_as_float(r[2 * c + 1])), sl2, negm2), a0, a1);
          if (c % 8 < kWaPoly) {
            wa_exp2_poly<F16>(a0, a1);
          } else {
            a0 = wa_ex2(a0);
            a1 = wa_ex2(a1);
          }
          sum[c & 1] = wa_add2(sum[c & 1], wa_pack2(a0, a1));
          r[c] = F16 ? pack_f16x2(a0, a1) : pack_bf16x2(a0, a1);
        }
        wa_tmem_st32(t_s + half * 32, &r[half * 32]);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&p_full[2 * x + half]);
      }
      float s0, s1;
      wa_unpack2(wa_add2(sum[0], sum[1]), s0, s1);
      l += s0 + s1;
      ++k;
    }
    if (ok && k > 0) ok = mbar_wait(&o_done[x], 0, 80, abort_flag);
    if (ok && q0 < p.Sq) {
      tc_fence_after();
      const float inv = m > -INFINITY && l > 0.f ? 1.f / l : 0.f;  // m: -inf where the row saw no key
      const int64_t off = b * p.os[0] + h * p.os[1] + (int64_t)qi * p.os[2];
#pragma unroll
      for (int c = 0; c < DP; c += 32) {
        uint32_t v[32];
        if (k > 0) {
          tmem_ld32(t_o + c, v);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = 0u;
        }
        if (qi >= p.Sq) continue;
        if (wp.out_vec) {
          uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.o) + off + c);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (c + j * 8 >= p.D) break;
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float y0 = __uint_as_float(v[j * 8 + 2 * e]) * inv, y1 = __uint_as_float(v[j * 8 + 2 * e + 1]) * inv;
              w[e] = F16 ? pack_f16x2(y0, y1) : pack_bf16x2(y0, y1);
            }
            dst[j] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (c + j < p.D)
              store_from_f32(p.o, off + (c + j) * p.os[3], F16 ? MT_F16 : MT_BF16, __uint_as_float(v[j]) * inv);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------------------------------------
// host

// 4-D map {D, S, heads, batch} of a strided [B, Hx, S, D] view, boxes of 64 channels x 128 rows, 128-byte swizzle.
static int wa_map(CUtensorMap* m, int dtype, const void* base, int64_t B, int64_t Hx, int64_t S, int64_t D,
                  const int64_t* st) {
  uint64_t dims[4] = {(uint64_t)D, (uint64_t)S, (uint64_t)Hx, (uint64_t)B};
  uint64_t strides[3] = {(uint64_t)(S > 1 ? st[2] * 2 : 16), (uint64_t)(Hx > 1 ? st[1] * 2 : 16),
                         (uint64_t)(B > 1 ? st[0] * 2 : 16)};
  uint32_t box[4] = {64, kWaTile, 1, 1};
  return make_tensor_map(m, dtype, 4, base, dims, strides, box, 128);
}

// A 16-bit view that a map can describe.
static bool wa_mappable(const void* base, const int64_t* st, int64_t B, int64_t Hx, int64_t S, int64_t D) {
  if ((uintptr_t)base % 16 || (st[3] != 1 && D > 1) || D % 8) return false;
  const int64_t n[3] = {B, Hx, S};
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1 && (st[i] <= 0 || st[i] % 8 || st[i] * 2 >= (1LL << 40))) return false;
  return true;
}

bool window_sm100_takes(const mt_window_attention_desc& d) {
  return d.dtype != MT_F32 && d.D <= 128 && d.scale > 0 && d.Sk > 0 && d.B * d.H <= INT32_MAX &&
         wa_mappable(d.q, d.q_strides, d.B, d.H, d.Sq, d.D) && wa_mappable(d.k, d.k_strides, d.B, d.Hkv, d.Sk, d.D) &&
         wa_mappable(d.v, d.v_strides, d.B, d.Hkv, d.Sk, d.D);
}

template <int DP, bool F16>
static int wa_launch(const mt_window_attention_desc& d, const AttnParams& a, cudaStream_t st) {
  auto kern = window_attention_sm100_kernel<DP, F16>;
  static bool attr[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!attr[dev & 63]) {
    int rc = cuda_check(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, WaCfg<DP>::SMEM),
                        "window attention smem attribute");
    if (rc) return rc;
    attr[dev & 63] = true;
  }
  CUtensorMap mq, mk, mv;
  int rc = wa_map(&mq, d.dtype, d.q, d.B, d.H, d.Sq, d.D, d.q_strides);
  if (!rc) rc = wa_map(&mk, d.dtype, d.k, d.B, d.Hkv, d.Sk, d.D, d.k_strides);
  if (!rc) rc = wa_map(&mv, d.dtype, d.v, d.B, d.Hkv, d.Sk, d.D, d.v_strides);
  if (rc) return rc;
  WaParams p{};
  p.a = a;
  p.out_vec = d.o_strides[3] == 1 && (uintptr_t)d.o % 16 == 0 && d.o_strides[0] % 8 == 0 && d.o_strides[1] % 8 == 0 &&
              d.o_strides[2] % 8 == 0;
  const int64_t blocks = (d.Sq + 2 * kWaTile - 1) / (2 * kWaTile);
  if (blocks > 65535) return fail(MT_ERR_UNSUPPORTED, "window_attention: too many queries");
  dim3 grid((unsigned)(d.B * d.H), (unsigned)blocks);
  kern<<<grid, kWaThreads, WaCfg<DP>::SMEM, st>>>(mq, mk, mv, p);
  return check_launch("window_attention_sm100");
}

int run_window_sm100(const mt_window_attention_desc& d, const AttnParams& a, cudaStream_t st) {
  if (d.D <= 64) return d.dtype == MT_F16 ? wa_launch<64, true>(d, a, st) : wa_launch<64, false>(d, a, st);
  return d.dtype == MT_F16 ? wa_launch<128, true>(d, a, st) : wa_launch<128, false>(d, a, st);
}

}  // namespace mt
