// What the attention kernels over a window of keys share: parameters, and which keys a tile of
// query rows has to visit.
#pragma once

#include "runtime.h"

namespace mt {

constexpr int kNoWindow = 1 << 29;  // window of calls without one; longer windows mean the same
constexpr int kMaxKeys = 1 << 28;   // keys and queries of a sequence
constexpr int kMaxStart = 1 << 29;  // first positions are clamped to +-kMaxStart (sums stay below 2^31)

// Rows of one (batch entry, key head): r = query * g + (head within the group), g = H / Hkv.
struct AttnParams {
  int B, H, Hkv, g, Sq, Sk, D, rows;  // Sk: keys (dense), or max_pages * page_size (paged)
  int causal, window, sinks;          // window kNoWindow: none
  float scale_log2;                   // softmax scale * log2(e)
  const int32_t* starts;              // NULL: Sk - Sq (dense), n - Sq (paged)
  const int32_t* lengths;             // NULL: Sk
  const void* q; int64_t qs[4];
  void* o; int64_t os[4];
  // dense keys and values
  const void* k; int64_t ks[4];
  const void* v; int64_t vs[4];
  // paged, 4 bits
  const uint32_t* words[2];
  const __half2* scales[2];
  const int32_t* table; int64_t table_stride;
  int num_pages, page_shift;
  // split keys: partial results in the workspace
  int splits;
  int q_vec;        // 8 channels of q are one aligned 16-byte vector (attn_split_kernel)
  int cluster;      // the splits of a row tile are a cluster and join there (attn_split_kernel)
  int target;       // CTAs that the work is cut into (attn_split_kernel)
  float2* part_ml;  // [split][B * Hkv * rows] (maximum in base 2, sum)
  float* part_o;    // [split][B * Hkv * rows][D], not divided by the sum
};

// A maximum that keeps a NaN: a query whose scores hold one has to end as NaN, also where shares of its keys are joined.
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// Keys n and the first query's position of one batch entry.
struct SeqPos {
  int n, start;
};
__device__ __forceinline__ SeqPos seq_pos(const AttnParams& p, int b, bool paged) {
  SeqPos s;
  s.n = p.lengths ? min(max(p.lengths[b], 0), p.Sk) : p.Sk;
  s.start = p.starts ? min(max(p.starts[b], -kMaxStart), kMaxStart) : (paged ? s.n : p.Sk) - p.Sq;
  return s;
}

// Keys that a query at position `pos` sees: [0, sk) and [lo, hi].
struct RowKeys {
  int lo, hi, sk;
  __device__ __forceinline__ bool sees(int j) const { return (j >= lo && j <= hi) || j < sk; }
};
__device__ __forceinline__ RowKeys row_keys(const AttnParams& p, const SeqPos& s, int pos) {
  RowKeys r;
  r.lo = p.window == kNoWindow ? 0 : max(0, pos - p.window + 1);
  r.hi = p.causal ? pos : (p.window == kNoWindow ? s.n - 1 : pos + p.window - 1);
  r.hi = min(r.hi, s.n - 1);
  r.sk = min(p.sinks, s.n);
  if (p.causal) r.sk = min(r.sk, pos + 1);
  return r;
}

// Blocks of BN keys that any of the queries at positions pmin..pmax visits: `first` blocks from
// key 0 on (sinks), then blocks from `from` on; `count` in all.
struct BlockList {
  int first, from, count;
  __device__ __forceinline__ int block(int i) const { return i < first ? i : from + i - first; }
};
template <int BN>
__device__ __forceinline__ BlockList block_list(const AttnParams& p, const SeqPos& s, int pmin, int pmax) {
  const RowKeys a = row_keys(p, s, pmin), z = row_keys(p, s, pmax);
  BlockList l;
  l.first = z.sk > 0 ? (z.sk + BN - 1) / BN : 0;
  l.from = max(a.lo / BN, l.first);
  const int last = z.hi >= a.lo ? z.hi / BN : -1;
  l.count = l.first + max(0, last - l.from + 1);
  return l;
}

// window_attention_split.cu: few query rows over 16-bit keys (16-byte aligned rows) or the 4-bit cache
int split_count(int64_t bk, int64_t rows, int64_t keys);
bool split_joins_in_cluster(int64_t bk, int64_t rows, int splits);  // no workspace and no join launch then
int run_split_attention(AttnParams& p, int dtype, bool paged, cudaStream_t st);

// window_attention_sm100.cu: many queries over 16-bit keys, head dims up to 128
bool window_sm100_takes(const mt_window_attention_desc& d);
int run_window_sm100(const mt_window_attention_desc& d, const AttnParams& a, cudaStream_t st);

}  // namespace mt
