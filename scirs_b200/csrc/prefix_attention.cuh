// What the kernels of the shared-prefix attention have in common (prefix_attention.cu, tails and joining;
// prefix_attention_sm100.cu, the prefix on tcgen05).
#pragma once

#include "host_common.h"

namespace scirs {
namespace prefix {

using bf16 = __nv_bfloat16;
constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kTile = 16;  // keys per step of a warp
constexpr int kStages = 3;
constexpr int kStep = kTile * kWarps;  // keys per step of a CTA: split lengths are multiples

struct Params {
  const bf16 *q, *k, *v;
  bf16* out;
  const int *tables, *lens, *qlens, *pages;  // qlens may be null: Q each
  float *part_o, *part_ml;                   // [B Q H, slots, HD], [B Q H, slots, 2]
  long q_sb, q_st, q_sh;                     // element strides of q
  int table_stride, max_pages, num_pages;
  int B, Q, H, Hkv, G, HD, bs;
  int L;                // tokens of the prefix
  int P;                // slots of a row that the prefix may take
  int per_p, rt_p;      // prefix items of item_kernel: keys a split, row tiles (0: tcgen05 takes the prefix)
  int T, rt_t;          // tails: splits (slots P .. P + T - 1), row tiles of a sequence
  // prefix on tcgen05: row tiles of tc_rows rows of one cached head against tc_blocks key blocks; a CTA takes
  // tc_share consecutive blocks of all row tiles' blocks laid end to end
  int tc_rows, tc_tiles, tc_blocks, tc_streams, tc_box, tc_share;
  float scale_log2;
  DevStatus* st;
};

struct Seq {
  int len, ql, start;  // tokens, queries, first key that is read through the sequence's own chain
};

__device__ __forceinline__ Seq seq_of(const Params& p, int b, bool report = false) {
  Seq s;
  s.len = max(p.lens[b], 0);
  if ((long)s.len > (long)p.max_pages * p.bs) {  // not addressable
    if (report) report_status(p.st, kStBounds, 95, (unsigned)s.len);
    s.len = p.max_pages * p.bs;
  }
  s.ql = p.qlens != nullptr ? min(max(p.qlens[b], 0), p.Q) : p.Q;
  if (s.ql == 0) s.len = 0;
  s.start = s.len - s.ql + 1 >= p.L ? p.L : 0;
  return s;
}

// Keys of a split of a sequence's tail: an even share, in whole steps.
__device__ __forceinline__ int tail_share(const Params& p, const Seq& s) {
  const int n = max(s.len - s.start, 0);
  return ((n + p.T - 1) / p.T + kStep - 1) / kStep * kStep;
}

// A K or V row (one token, one head) of the pool, in elements; -1 where the chain names no page of the pool.
__device__ __forceinline__ long pool_row(const Params& p, const int* pages, int max_pages, int key, int hk) {
  const int pi = key / p.bs;
  if (pi >= max_pages) return -1;
  const int page = pages[pi];
  if (!input_in_range(page, p.num_pages, p.st, 96)) return -1;
  return (((long)page * p.bs + key % p.bs) * p.Hkv + hk) * p.HD;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool full) {
  const int n = full ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Row r (of all rows of a cached head) of the batch: its query, or null where it takes no part in the prefix.
__device__ __forceinline__ const bf16* prefix_query(const Params& p, int r, int hk) {
  if (r >= p.B * p.Q * p.G) return nullptr;
  const int bt = r / p.G, b = bt / p.Q, t = bt % p.Q;
  const Seq s = seq_of(p, b);
  if (t >= s.ql || s.start != p.L) return nullptr;
  return p.q + b * p.q_sb + t * p.q_st + (long)(hk * p.G + r % p.G) * p.q_sh;
}

// The prefix on tcgen05: plans the split (p.P and the tc_ fields), launches.
void plan_prefix_tc(Params& p, int sms);
void launch_prefix_tc(const Params& p, cudaStream_t st);

}  // namespace prefix
}  // namespace scirs
