// Verification of drafted tokens against the target's probabilities, for a batch, from given random
// numbers (rejection sampling: Leviathan et al., 2023).
//
// Sequence b has n_b drafted tokens x_i with the draft's probabilities q_i and the target's p_i
// (i = 0 .. n_b; p_{n_b} follows the last draft). Draft i is kept while
//     q_i(x_i) > 0 ?  u_i q_i(x_i) < p_i(x_i)  or  u_i < threshold  :  p_i(x_i) > 0
// and at the first place r that is not kept (r = n_b: none) one token is drawn from the weights
//     max(p_r - q_r, 0), or p_r where those are all zero;  p_{n_b} where every draft was kept:
// the first v whose cumulative weight exceeds u_n times the total.
//
// What it costs: 2 n gathered values, then ONE row of p and one of q a sequence, read once: bound by
// memory for a batch, by the chain of dependent loads for one sequence. A cluster of 8 CTAs takes a
// sequence (one CTA, where a batch is large and its rows are short); each of its 64 warps sums a
// contiguous segment of the row, the 64 sums are exchanged through distributed shared memory, and the CTA
// that owns the segment with the answer reads that segment again (from L2) to find it. The answer is a
// whole number that must not depend on rounding next to a border, so products, differences and sums are
// formed in 64 bits (u q and p - q of 32-bit values are exact there) in a fixed order.
//
// Measured: 256 sequences of 8 drafts over 131072 tokens (246 MB of rows) 61 us, 4.0 TB/s, 0.61 of the device's
// copy rate: a CTA reads its 131 KB only after the accepted drafts are known and is idle in the two exchanges
// behind it (an order of steps, which reads of the next sequence's row could fill, not a bound of the device).
// 64 of 5 over 50257 in bf16 12 us and one of 4 in fp32 8 us: the chain tokens -> gathers -> row -> sums ->
// segment, five dependent trips to memory.
//
// Reference parity: scirs2-neural/src/inference/speculative/rejection_sampling.rs:180-330
// (SpeculativeDecoder::rejection_sampling_step, one sequence on the host).
#include "host_common.h"

#include <cooperative_groups.h>
#include <cuda_fp16.h>

namespace scirs {
namespace verify {

namespace cg = cooperative_groups;

constexpr int kCluster = 8, kThreads = 256, kWarps = kThreads / 32;
constexpr int kMaxSegs = kCluster * kWarps;  // two to a lane

struct Params {
  const void *target, *draft;  // draft may be null: it is certain of its tokens
  const long* tokens;
  const float* u;
  const int* lens;  // may be null: n each
  int* accepted;
  long* out;
  long ts_b, ts_i, ds_b, ds_i;  // element strides of target and draft
  int n, V;
  double threshold;
};

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }

__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Inclusive prefix sum over the lanes.
__device__ __forceinline__ double warp_scan_d(double v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double w = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += w;
  }
  return v;
}

// The row that the token is drawn from.
template <typename T>
struct Row {
  const T *p, *q;  // q null: nothing, or one at `certain`, is taken off
  int certain;
  // Weight of entry v; what is not a positive finite number counts as nothing.
  __device__ __forceinline__ double weight(float pv, float qv) const {
    const double d = (double)pv - (double)qv;
    return d > 0.0 && d < INFINITY ? d : 0.0;
  }
  __device__ __forceinline__ double at(int v) const {
    return weight(to_f(p[v]), q != nullptr ? to_f(q[v]) : (v == certain ? 1.f : 0.f));
  }
};

// VEC: the rows begin at multiples of 16 bytes, so that a lane reads 16 of them at a time.
// CL: CTAs of a sequence.
template <typename T, bool VEC, int CL>
__global__ void __cluster_dims__(CL, 1, 1) __launch_bounds__(kThreads, 5) verify_kernel(const Params a) {
  constexpr int kSegs = CL * kWarps;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = blockIdx.x, b = blockIdx.y;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  __shared__ int kept_s, hit_s, last_s;
  __shared__ double seg_sum[kWarps];  // read by the whole cluster
  __shared__ double all_sum[kMaxSegs], scan_s[kThreads], wsum[kWarps];

  const T* tb = reinterpret_cast<const T*>(a.target) + b * a.ts_b;
  const T* db = a.draft != nullptr ? reinterpret_cast<const T*>(a.draft) + b * a.ds_b : nullptr;
  const long* tok = a.tokens + (long)b * a.n;
  const float* u = a.u + (long)b * (a.n + 1);
  const int nb = a.lens != nullptr ? min(max(a.lens[b], 0), a.n) : a.n;

  // how many drafts are kept: every CTA of the cluster finds out for itself
  if (warp == 0) {
    int kept = 0;
    for (int i0 = 0; i0 < nb; i0 += 32) {
      const int i = i0 + lane;
      bool keep = false;
      if (i < nb) {
        const long x = tok[i];
        if (x >= 0 && x < a.V) {
          const double p = to_f(tb[i * a.ts_i + x]), q = db != nullptr ? to_f(db[i * a.ds_i + x]) : 1.f, ui = u[i];
          keep = q <= 0.0 ? p > 0.0 : ui < 1.0 && (ui * q < p || ui < a.threshold);
        }
      }
      const unsigned m = __ballot_sync(0xffffffffu, keep);
      const int run = m == 0xffffffffu ? 32 : __ffs(~m) - 1;
      kept += run;
      if (run < 32) break;
    }
    if (lane == 0) kept_s = kept;
  }
  __syncthreads();
  const int kept = kept_s;

  Row<T> row;
  row.p = tb + kept * a.ts_i;
  row.q = kept < nb && db != nullptr ? db + kept * a.ds_i : nullptr;
  row.certain = -1;
  if (kept < nb && db == nullptr) {
    const long x = tok[kept];
    row.certain = x >= 0 && x < a.V ? (int)x : -1;
  }
  bool residual = row.q != nullptr || row.certain >= 0;

  constexpr int kVec = VEC ? 16 / (int)sizeof(T) : 1;
  const int seg_len = ((a.V + kSegs - 1) / kSegs + kVec - 1) / kVec * kVec;
  int found;  // the segment that holds the answer, -1: every weight is zero
  double base, target;
  while (true) {
    {
      const int s0 = (rank * kWarps + warp) * seg_len, s1 = min(s0 + seg_len, a.V);
      double s = 0.0;
      if (VEC) {
        const int whole = s0 + max(s1 - s0, 0) / kVec * kVec;
#pragma unroll 4
        for (int v = s0 + lane * kVec; v < whole; v += 32 * kVec) {
          union {
            uint4 u;
            T t[kVec];
          } x, y;
          x.u = __ldg(reinterpret_cast<const uint4*>(row.p + v));
          y.u = row.q != nullptr ? __ldg(reinterpret_cast<const uint4*>(row.q + v)) : make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int e = 0; e < kVec; ++e)
            s += row.weight(to_f(x.t[e]), row.q != nullptr ? to_f(y.t[e]) : (v + e == row.certain ? 1.f : 0.f));
        }
        if (whole + lane < s1) s += row.at(whole + lane);  // (fewer than kVec at the row's end)
      } else {
#pragma unroll 16
        for (int v = s0 + lane; v < s1; v += 32) s += row.at(v);
      }
      s = warp_sum_d(s);
      if (lane == 0) seg_sum[warp] = s;
    }
    cluster.sync();
    if (tid < kMaxSegs) all_sum[tid] = tid < kSegs ? cluster.map_shared_rank(seg_sum, tid / kWarps)[tid % kWarps] : 0.0;
    __syncthreads();
    cluster.barrier_arrive();  // (waited for before seg_sum is written again, and before this CTA leaves)
    // prefix sums of the segments, two to a lane; every warp computes the same
    const double s0 = all_sum[2 * lane], s1 = all_sum[2 * lane + 1];
    const double inc = warp_scan_d(s0 + s1, lane);
    double exc = __shfl_up_sync(0xffffffffu, inc, 1);
    if (lane == 0) exc = 0.0;
    const double total = __shfl_sync(0xffffffffu, inc, 31);
    target = (double)u[a.n] * total;
    const bool h0 = s0 > 0.0 && exc + s0 > target, h1 = s1 > 0.0 && inc > target;
    const unsigned hit = __ballot_sync(0xffffffffu, h0 || h1), any = __ballot_sync(0xffffffffu, s0 > 0.0 || s1 > 0.0);
    if (any == 0u && residual) {  // nothing is left of the target's row: draw from the row itself
      residual = false;
      row.q = nullptr;
      row.certain = -1;
      cluster.barrier_wait();
      continue;
    }
    // the first segment past the target; rounding may leave none: the last one with weight
    const int l = hit != 0u ? __ffs(hit) - 1 : 31 - __clz(any);
    const bool second = hit != 0u ? !h0 : s1 > 0.0;
    found = any == 0u ? -1 : __shfl_sync(0xffffffffu, 2 * lane + (second ? 1 : 0), l & 31);
    base = __shfl_sync(0xffffffffu, second ? exc + s0 : exc, l & 31);
    break;
  }

  if (rank == 0)
    for (int i = tid; i <= a.n; i += kThreads) {
      if (i == kept) {
        if (found < 0) a.out[(long)b * (a.n + 1) + i] = -1;
        a.accepted[b] = kept;
      } else {
        a.out[(long)b * (a.n + 1) + i] = i < kept ? tok[i] : -1;
      }
    }
  cluster.barrier_wait();
  if (found < 0 || found / kWarps != rank) return;

  // the owner reads the segment again, a short run to each thread
  const int s0 = found * seg_len, s1 = min(s0 + seg_len, a.V);
  const int per = (seg_len + kThreads - 1) / kThreads;
  const int v0 = min(s0 + tid * per, s1), v1 = min(v0 + per, s1);
  double s = 0.0;
  for (int v = v0; v < v1; ++v) s += row.at(v);
  const double inc = warp_scan_d(s, lane);
  if (lane == 31) wsum[warp] = inc;
  if (tid == 0) {
    hit_s = kThreads;
    last_s = 0;
  }
  __syncthreads();
  double off = base;
  for (int w = 0; w < warp; ++w) off += wsum[w];
  scan_s[tid] = off + inc;
  if (s > 0.0) {
    if (off + inc > target) atomicMin(&hit_s, tid);
    atomicMax(&last_s, tid);
  }
  __syncthreads();
  if (tid != (hit_s < kThreads ? hit_s : last_s)) return;
  double run = tid > 0 ? scan_s[tid - 1] : base;
  int token = -1;
  for (int v = v0; v < v1; ++v) {
    const double w = row.at(v);
    if (w <= 0.0) continue;
    run += w;
    token = v;
    if (run > target) break;
  }
  a.out[(long)b * (a.n + 1) + kept] = token;
}

}  // namespace verify

// target [B, n + 1, V] and draft [B, n, V] (or none): fp32, bf16 or fp16 with contiguous rows; tokens int64
// [B, n]; uniforms fp32 [B, n + 1]; lens int32 [B] (or none). Returns (accepted int32 [B], tokens int64
// [B, n + 1]).
std::tuple<torch::Tensor, torch::Tensor> draft_verify(torch::Tensor target, c10::optional<torch::Tensor> draft,
                                                      torch::Tensor tokens, torch::Tensor uniforms,
                                                      c10::optional<torch::Tensor> lens, double threshold) {
  CHECK_CUDA_TENSOR(target);
  TORCH_CHECK(target.dim() == 3 && target.size(1) >= 1 && target.size(2) >= 1, "target probabilities [B, n + 1, V]");
  const int64_t B = target.size(0), n = target.size(1) - 1, V = target.size(2);
  // (places in a row are 32-bit numbers; the end of the last segment lies up to a segment behind the row's)
  TORCH_CHECK(V < (1LL << 30) && B < 65536 && n < (1LL << 30), "draft_verify: too large");
  auto rows = [&](const torch::Tensor& t, const char* what, int64_t count) {
    TORCH_CHECK(t.device() == target.device() && t.scalar_type() == target.scalar_type() && t.dim() == 3 &&
                    t.size(0) == B && t.size(1) == count && t.size(2) == V && (V == 1 || t.stride(2) == 1),
                what, " must be [", num(B), ", ", num(count), ", ", num(V), "] with contiguous rows of the target's type");
  };
  rows(target, "target probabilities", n + 1);
  const bool has_draft = draft.has_value() && draft->defined(), has_lens = lens.has_value() && lens->defined();
  if (has_draft) rows(*draft, "draft probabilities", n);
  auto flat = [&](const torch::Tensor& t, const char* what, at::ScalarType ty, int64_t count) {
    TORCH_CHECK(t.device() == target.device() && t.scalar_type() == ty && t.is_contiguous() && t.numel() == count,
                what, ": contiguous ", ty, " with ", num(count), " values on the target's device");
  };
  flat(tokens, "draft tokens", at::kLong, B * n);
  flat(uniforms, "uniforms", at::kFloat, B * (n + 1));
  if (has_lens) flat(*lens, "draft lengths", at::kInt, B);
  c10::cuda::CUDAGuard guard(target.get_device());
  auto accepted = at::empty({B}, target.options().dtype(at::kInt));
  auto out = at::empty({B, n + 1}, target.options().dtype(at::kLong));
  if (B == 0) return {accepted, out};
  verify::Params a{};
  a.target = target.data_ptr();
  a.draft = has_draft ? draft->data_ptr() : nullptr;
  a.tokens = reinterpret_cast<const long*>(tokens.data_ptr<int64_t>());
  a.u = uniforms.data_ptr<float>();
  a.lens = has_lens ? lens->data_ptr<int>() : nullptr;
  a.accepted = accepted.data_ptr<int>();
  a.out = reinterpret_cast<long*>(out.data_ptr<int64_t>());
  a.ts_b = target.stride(0);
  a.ts_i = target.stride(1);
  a.ds_b = has_draft ? draft->stride(0) : 0;
  a.ds_i = has_draft ? draft->stride(1) : 0;
  a.n = (int)n;
  a.V = (int)V;
  a.threshold = threshold;
  const auto aligned = [](const torch::Tensor& t) {
    const int64_t v = 16 / t.element_size();
    return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && t.stride(0) % v == 0 && t.stride(1) % v == 0;
  };
  // 16 bytes a lane where a warp's segment gives every lane four of them: 256 rows of 131072 fp32 82 -> 66 us
  // against single values, but 64 rows of 50257 bf16 12.5 -> 17.4 us (99 vectors for the 32 lanes of a warp)
  const bool vec = V >= (int64_t)verify::kMaxSegs * 32 * 4 * (16 / target.element_size()) && aligned(target) &&
                   (!has_draft || aligned(*draft));
  // one CTA a sequence where a cluster's eight would queue up for longer than it reads the row: that grows with B
  // in rounds of CTAs, the row with V. Eight -> one: 256 rows of 2505 16.0 -> 7.4 us, of 32769 32 -> 29, 128 of 8191
  // 11.0 -> 11.1, 64 of 256 5.7 -> 4.8, but 64 of 8191 7.0 -> 10.8 and 32 of 2505 5.2 -> 6.8.
  const bool solo = !vec && 2 * V <= B * B;
#define SCIRS_VERIFY_CL(T_, V_, CL_) \
  verify::verify_kernel<T_, V_, CL_><<<dim3(CL_, (unsigned)B), verify::kThreads, 0, cur_stream()>>>(a)
#define SCIRS_VERIFY(T_)                              \
  if (vec)                                            \
    SCIRS_VERIFY_CL(T_, true, verify::kCluster);      \
  else if (solo)                                      \
    SCIRS_VERIFY_CL(T_, false, 1);                    \
  else                                                \
    SCIRS_VERIFY_CL(T_, false, verify::kCluster);     \
  break;
  switch (target.scalar_type()) {
    case at::kFloat:
      SCIRS_VERIFY(float)
    case at::kBFloat16:
      SCIRS_VERIFY(__nv_bfloat16)
    case at::kHalf:
      SCIRS_VERIFY(__half)
    default:
      TORCH_CHECK(false, "probabilities must be fp32, bf16 or fp16, got ", target.scalar_type());
  }
#undef SCIRS_VERIFY
#undef SCIRS_VERIFY_CL
  SCIRS_CHECK_LAUNCH();
  return {accepted, out};
}

}  // namespace scirs
