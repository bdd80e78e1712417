// Attention with a sliding window and sinks on the 5th-generation tensor cores, for many queries
// (bf16 / f16, head dims up to 128).
//
// One CTA = two tiles of 128 query rows of one (batch entry, head); the tiles of 128 keys that any of the rows
// sees (the sinks' tiles, then the window's) stream through TMA rings of K and V, 128-byte swizzled.
//   warp 0      producer: Q once, then K(0), K(j + 1), V(j), ..
//   warp 1      MMA issuer: S_x = Q_x K^T into TMEM (fp32), then O_x += P_x V with P_x as the TMEM operand: it
//               overwrites the low half of S_x's columns, so the probabilities never touch shared memory.
//   warps 4..11 one softmax warpgroup per query tile, one row per thread: the row's 128 scores are read once into
//               registers (these warps take the registers that the first four give up); p = 2^(s scale - m) in fp32, the sums in fp32, P rounded to 16 bits.
// O stays in TMEM for all the key tiles.  The running maximum m is raised only when a score passes it by more than
// 2^8; the warp then rescales its rows of O in TMEM.  While one warpgroup exponentiates, the tensor core works for
// the other tile: 128 x 128 scores take 1024 cycles of the exponential unit (16 a cycle) and, at head dim 128,
// 1024 cycles of the tensor core, so both are near their limits.
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

struct WaParams {
  AttnParams a;
  int out_vec;  // output rows take 16-byte stores
};

__device__ __forceinline__ float wa_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float wa_max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
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

// maximum of 128 values, four independent chains
__device__ __forceinline__ float wa_max128(const uint32_t (&r)[128]) {
  float m[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) m[i] = __uint_as_float(r[i]);
#pragma unroll
  for (int k = 4; k + 8 <= 128; k += 8)
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = wa_max3(m[i], __uint_as_float(r[k + i]), __uint_as_float(r[k + 4 + i]));
#pragma unroll
  for (int i = 0; i < 4; ++i) m[i] = fmaxf(m[i], __uint_as_float(r[124 + i]));
  return fmaxf(wa_max3(m[0], m[1], m[2]), m[3]);
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

// D (+)= A (TMEM, 16-bit, two K elements a column) * B (shared memory descriptor)
__device__ __forceinline__ void wa_umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(
          d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Operand whose rows along N are contiguous (V: 64 channels of one key = 128 bytes, swizzled; 8 keys = 1024 bytes):
// the next 64 channels lie `chunk` bytes on, the next 8 keys 1024.
__device__ __forceinline__ uint64_t wa_desc_mn(uint32_t addr, uint32_t chunk) {
  uint64_t d = 0;
  d |= (uint64_t)((addr & 0x3FFFF) >> 4);
  d |= (uint64_t)(chunk >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;  // SWIZZLE_128B
  return d;
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
  uint64_t* p_full = s_full + 2;                  // [2]
  uint64_t* o_done = p_full + 2;                  // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_done + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int bh = blockIdx.y, b = bh / p.H, h = bh % p.H, hk = h / p.g;
  const int qbase = blockIdx.x * (2 * kWaTile);
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
      mbar_init(&p_full[x], kWaTile);
      mbar_init(&o_done[x], 1);
    }
    *abort_flag = 0;
    fence_barrier_init();
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
    if (lane == 0 && bl.count > 0) {
      tma_prefetch_desc(&tmQ);
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
      mbar_arrive_expect_tx(q_full, 2 * Cfg::TILE);
      for (int x = 0; x < 2; ++x)
        for (int c = 0; c < CHUNKS; ++c)
          tma_load_4d(sQ + x * Cfg::TILE + c * Cfg::CHUNK, &tmQ, q_full, c * 64, qbase + x * kWaTile, h, b);
    }
    int ks = 0, vs = 0;
    uint32_t kph = 0, vph = 0;
    bool ok = true;
    auto load_k = [&](int i) {
      if (lane == 0 && ok) {
        ok = mbar_wait(&k_empty[ks], kph ^ 1, 71, abort_flag);
        if (ok) {
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
    if (bl.count > 0) load_k(0);
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
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    if (lane == 0 && bl.count > 0) {
      const uint32_t q_addr = smem_u32(sQ), k_addr = smem_u32(sK), v_addr = smem_u32(sV);
      bool ok = mbar_wait(q_full, 0, 74, abort_flag);
      int ks = 0, vs = 0;
      uint32_t kph = 0, vph = 0;
      const BlockList tx[2] = {tiles_of(0), tiles_of(1)};
      int done[2] = {0, 0};
      auto issue_s = [&](int x) {
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk)
          umma_f16(tmem + x * 128, sdesc_sw128(q_addr + x * Cfg::TILE + (kk / 4) * Cfg::CHUNK + (kk % 4) * 32),
                   sdesc_sw128(k_addr + ks * Cfg::TILE + (kk / 4) * Cfg::CHUNK + (kk % 4) * 32), idesc_s, kk > 0);
        umma_commit(&s_full[x]);
      };
      ok = ok && mbar_wait(&k_full[0], 0, 75, abort_flag);
      if (ok) {
        tc_fence_after();
#pragma unroll
        for (int x = 0; x < 2; ++x)
          if (active(tx[x], 0)) issue_s(x);
        umma_commit(&k_empty[0]);
        ks = 1 % Cfg::STAGES_K;
      }
      for (int i = 0; ok && i < bl.count; ++i) {
        bool have_k = false, have_v = false;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (ok && active(tx[x], i)) {
            if (!have_v) ok = mbar_wait(&v_full[vs], vph, 76, abort_flag);
            have_v = true;
            ok = ok && mbar_wait(&p_full[x], done[x] & 1, 77, abort_flag);
            if (!ok) continue;
            tc_fence_after();
#pragma unroll
            for (int kk = 0; kk < kWaTile / 16; ++kk)
              wa_umma_ts(tmem + 256 + x * 128, tmem + x * 128 + kk * 8,
                         wa_desc_mn(v_addr + vs * Cfg::TILE + kk * 2048, Cfg::CHUNK), idesc_o, done[x] > 0 || kk > 0);
            if (++done[x] == tx[x].count) umma_commit(&o_done[x]);
          }
          if (ok && active(tx[x], i + 1)) {
            if (!have_k) ok = mbar_wait(&k_full[ks], kph, 78, abort_flag);
            have_k = true;
            if (!ok) continue;
            tc_fence_after();
            issue_s(x);
          }
        }
        // a tile that no row needed still has to arrive before its stage is handed back
        if (ok && !have_v) ok = mbar_wait(&v_full[vs], vph, 76, abort_flag);
        if (ok && !have_k && i + 1 < bl.count) ok = mbar_wait(&k_full[ks], kph, 78, abort_flag);
        if (!ok) break;
        umma_commit(&v_empty[vs]);
        if (++vs == Cfg::STAGES_V) {
          vs = 0;
          vph ^= 1;
        }
        if (i + 1 < bl.count) {
          umma_commit(&k_empty[ks]);
          if (++ks == Cfg::STAGES_K) {
            ks = 0;
            kph ^= 1;
          }
        }
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
    const RowKeys rk = row_keys(p, sp, sp.start + min(qi, p.Sq - 1));
    // keys that all rows of the tile see
    const RowKeys ra = row_keys(p, sp, sp.start + q0), rz = row_keys(p, sp, sp.start + min(q0 + kWaTile, p.Sq) - 1);
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
      if (!(k0 + kWaTile - 1 <= ra.hi && (k0 >= rz.lo || k0 + kWaTile - 1 < ra.sk))) {
        const int lo = rk.lo - k0, hi = rk.hi - k0, sk = rk.sk - k0;
#pragma unroll
        for (int c = 0; c < 128; ++c)
          if (!((c >= lo && c <= hi) || c < sk)) r[c] = 0xff800000u;
      }
      const float top = wa_max128(r);
      if (__any_sync(0xffffffffu, top > thr)) {
        const float mn = fmaxf(m, top);
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
        uint32_t pk[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          float a0, a1;
          wa_unpack2(wa_fma2(wa_pack2(__uint_as_float(r[half * 64 + 2 * c]), __uint_as_float(r[half * 64 + 2 * c + 1])),
                             sl2, negm2), a0, a1);
          a0 = wa_ex2(a0);
          a1 = wa_ex2(a1);
          sum[c & 1] = wa_add2(sum[c & 1], wa_pack2(a0, a1));
          pk[c] = F16 ? pack_f16x2(a0, a1) : pack_bf16x2(a0, a1);
        }
        wa_tmem_st32(t_s + half * 32, pk);
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&p_full[x]);
      float s0, s1;
      wa_unpack2(wa_add2(sum[0], sum[1]), s0, s1);
      l += s0 + s1;
      ++k;
    }
    if (ok && k > 0) ok = mbar_wait(&o_done[x], 0, 80, abort_flag);
    if (ok && q0 < p.Sq) {
      tc_fence_after();
      const float inv = l > 0.f ? 1.f / l : 0.f;
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
  return d.dtype != MT_F32 && d.D <= 128 && d.scale > 0 && d.Sk > 0 && d.B * d.H <= 65535 &&
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
  dim3 grid((unsigned)((d.Sq + 2 * kWaTile - 1) / (2 * kWaTile)), (unsigned)(d.B * d.H));
  kern<<<grid, kWaThreads, WaCfg<DP>::SMEM, st>>>(mq, mk, mv, p);
  return check_launch("window_attention_sm100");
}

int run_window_sm100(const mt_window_attention_desc& d, const AttnParams& a, cudaStream_t st) {
  if (d.D <= 64) return d.dtype == MT_F16 ? wa_launch<64, true>(d, a, st) : wa_launch<64, false>(d, a, st);
  return d.dtype == MT_F16 ? wa_launch<128, true>(d, a, st) : wa_launch<128, false>(d, a, st);
}

}  // namespace mt
