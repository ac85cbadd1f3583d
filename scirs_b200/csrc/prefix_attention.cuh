// What the kernels of the shared-prefix attention have in common (prefix_attention.cu, tails and joining;
// prefix_attention_sm100.cu, the prefix on tcgen05).
#pragma once

#include "host_common.h"

namespace scirs {
namespace prefix {

using bf16 = __nv_bfloat16;
constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kTile = 16;  // keys per step of a warp: split lengths are multiples
constexpr int kSpareParts = 32;  // parts of a row that spare items take, at most, where items take the prefix too
constexpr float kRaise = 8.f;  // a running maximum is raised only past 2^8

struct Params {
  const bf16 *q, *k, *v;
  bf16* out;
  const int *tables, *lens, *qlens, *pages;  // qlens may be null: Q each
  float *part_o, *part_ml;                   // [B Q H, slots, HD], [B Q H, slots, 2]
  long q_sb, q_st, q_sh;                     // element strides of q
  int max_pages, num_pages;                  // (tables are [B, max_pages])
  int B, Q, H, Hkv, G, HD, bs;
  int L;                // tokens of the prefix
  int P, T;             // splits of the prefix and of a tail, and their slots: 0 .. P - 1, P .. P + T - 1
  int per_p;            // item_kernel: keys of a prefix split
  int rt_p, rt_t;       // item_kernel: row tiles of the prefix (0: tcgen05 takes it), of a tail
  int pages_max;        // pages of the prefix
  int items;            // of item_kernel
  int spare;            // items behind those, which take more parts of the sequences that end inside the prefix
  int box;              // keys of a TMA box (0: cp.async)
  uint32_t bs_mul;      // division by bs (see page_of)
  int bs_shift;
  // prefix on tcgen05: row tiles of tc_rows rows of one cached head against tc_blocks key blocks; a CTA takes
  // tc_share consecutive blocks of all row tiles' blocks laid end to end
  int tc_rows, tc_tiles, tc_blocks, tc_streams, tc_box, tc_share;
  float scale_log2;
  DevStatus* st;
};

struct Seq {
  int len, ql, start;  // tokens, queries, first key that is read through the sequence's own chain
};

__device__ __forceinline__ Seq seq_from(const Params& p, int len, int ql, bool report) {
  Seq s;
  s.len = max(len, 0);
  if ((long)s.len > (long)p.max_pages * p.bs) {  // not addressable
    if (report) report_status(p.st, kStBounds, 95, (unsigned)s.len);
    s.len = p.max_pages * p.bs;
  }
  s.ql = min(max(ql, 0), p.Q);
  if (s.ql == 0) s.len = 0;
  s.start = s.len - s.ql + 1 >= p.L ? p.L : 0;
  return s;
}

__device__ __forceinline__ Seq seq_of(const Params& p, int b) {
  return seq_from(p, p.lens[b], p.qlens != nullptr ? p.qlens[b] : p.Q, false);
}

// The tiles of a sequence's tail begin at multiples of kTile, the first one perhaps before the tail does; the
// keys from there, and a split's share of them.
__device__ __forceinline__ int first_key(const Seq& s) { return s.start & ~(kTile - 1); }
__device__ __forceinline__ int tail_keys(const Seq& s) { return s.len > s.start ? s.len - first_key(s) : 0; }
__device__ __forceinline__ int tail_share(const Seq& s, int parts) {
  return ((tail_keys(s) + parts - 1) / parts + kTile - 1) / kTile * kTile;
}

// A sequence that ends inside the prefix is read by itself from its first key, up to L of them, where T goes by the
// tails behind the prefix. Only the device knows which these are: where they would take long, their keys are cut into
// T + spare_parts shares, and the spare items, as many to each of them as there are for all that the batch has, take
// those behind the T-th.
__device__ __forceinline__ bool ends_inside(const Params& p, const Seq& s) { return s.start != p.L && s.len > 0; }

// How many there are (the same in all lanes).
__device__ __forceinline__ int count_inside(const Params& p, int lane) {
  int n = 0;
#pragma unroll 1
  for (int b = lane; b < p.B; b += 32) n += ends_inside(p, seq_of(p, b));
  return __reduce_add_sync(0xffffffffu, n);
}
// The k-th of them, from 0.
__device__ __forceinline__ int nth_inside(const Params& p, int k, int lane) {
  for (int b0 = 0;; b0 += 32) {
    const int b = b0 + lane;
    const uint32_t on = __ballot_sync(0xffffffffu, b < p.B && ends_inside(p, seq_of(p, b)));
    if (k < __popc(on)) return b0 + __fns(on, 0, k + 1);
    if (b0 + 32 >= p.B) return 0;  // (not reached)
    k -= __popc(on);
  }
}
__device__ __forceinline__ int spare_parts(const Params& p, int inside) {
  return min(p.spare / (inside * p.Hkv * p.rt_t), p.rt_p == 0 ? p.P : kSpareParts);
}
// Where the slots of such a row begin: with tcgen05 (rt_p = 0) at the prefix's, of which it has none; items write
// their part of every row.
__device__ __forceinline__ int spare_at(const Params& p) { return p.rt_p == 0 ? 0 : p.P + p.T; }
// Slots of a row.
__host__ __device__ __forceinline__ int slots_of(const Params& p) {
  return p.P + p.T + (p.spare > 0 && p.rt_p > 0 ? p.T + kSpareParts : 0);
}

// key / bs for 0 <= key < 2^31: multiplication by the rounded-up reciprocal (Granlund & Montgomery, 1994).
__device__ __forceinline__ int page_of(const Params& p, int key) {
  return (int)(((uint64_t)(uint32_t)key * p.bs_mul) >> p.bs_shift);
}

// The largest value, NaN if one is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// A K or V row (one token, one head) of the pool, in elements; -1 where the chain names no page of the pool.
__device__ __forceinline__ long pool_row(const Params& p, const int* pages, int max_pages, int key, int hk) {
  const int pi = page_of(p, key);
  if (pi >= max_pages) return -1;
  const int page = pages[pi];
  if (!input_in_range(page, p.num_pages, p.st, 96)) return -1;
  return (((long)page * p.bs + key - pi * p.bs) * p.Hkv + hk) * p.HD;
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

__device__ __forceinline__ void tma_load_5d(void* smem_dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1,
                                            int c2, int c3, int c4) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
      "[%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(smem_u32(smem_dst)),
      "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
      : "memory");
}

// A tensor map of a pool with boxes of `rows` slots of `halves` 64-column halves of one head (head_dim 64 or 128).
CUtensorMap pool_map(const Params& p, const bf16* pool, int rows, int halves);

// The kernels of one call overlap at their ends: each may start when the one before it has started all its
// CTAs, and waits for its completion where it needs it, at the latest before it ends itself, so that what comes
// behind the last one finds all of them done. The first one waits for everything in front of the call.
__device__ __forceinline__ void allow_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Launch; `overlap`: may start before the kernel in front of it in the stream has ended.
template <typename... P, typename... A>
void launch(void (*kern)(P...), unsigned grid, int threads, int smem, cudaStream_t st, bool overlap, const A&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = overlap ? 1 : 0;
  SCIRS_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kern, args...));
}

// The prefix on tcgen05: plans the split (p.P and the tc_ fields), launches.
void plan_prefix_tc(Params& p, int sms);
void launch_prefix_tc(const Params& p, cudaStream_t st);

}  // namespace prefix
}  // namespace scirs
