// Attention over the paged cache for a batch whose sequences begin with the same tokens: the shared
// prefix is read once for all of them, each sequence's own tail by itself, and the partial softmaxes
// are joined.
//
// q [B, Q, H, HD] holds the newest q_len <= Q tokens of each sequence (Q = 1: plain decoding; more:
// drafted tokens to be scored). With len tokens in sequence b, query t stands at position
// len - q_len + t and sees the keys up to its own: limit = len - q_len + t + 1 of them. A row with
// t >= q_len, or without keys, gives zeros. H query heads share Hkv cached ones, G = H / Hkv.
//
//   rows of one cached head: r = (b Q + t) G + g, so a prefix item works on 16 MT consecutive r of the
//   whole batch against keys [0, L) of prefix_pages; a tail item on the Q G rows of one sequence against
//   keys [L, len) of its own chain. Both kinds split their keys, and every split writes (max, sum,
//   unnormalised O) of its rows; the combine kernel joins them:
//     o = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i.
//   A sequence some of whose queries end inside the prefix (it is shorter, or padding) is read by itself
//   from its first key, so that in a prefix item a row sees every key or none.
//
// Tiles: a warp walks its keys 16 at a time, K and V rows of one head copied by cp.async (16 bytes a
// lane, swizzled so that ldmatrix is free of conflicts) into a ring of its own, so the warps of a CTA
// never wait for one another; S = Q K^T and O += P V by mma.sync m16n8k16 with the running max and sum
// in registers. Bound by memory as long as few rows share a key.
//
// Masked places: keys past the limit get P = 0 by selection, and slots past the length are never read.
// Where a tile holds keys that only some rows see and one of its V values is infinite or NaN, P V is
// formed row by row without the masked keys, since 0 * NaN would reach the rows that do not see it.
//
// Reference parity: scirs2-neural/src/inference/paged_attention.rs:113-283 (one query over one page
// chain), block_manager.rs:196-280 (SharedPrefixCache: the pages a prefix's sequences share).
#include "prefix_attention.cuh"

namespace scirs {
namespace prefix {

__device__ __forceinline__ void ldsm4(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int HDP>
struct Cfg {
  static constexpr int ROW = HDP * 2;                 // bytes of a K or V row
  static constexpr int KV = kTile * ROW;              // bytes of a K or V tile
  static constexpr int WARP = kStages * 2 * KV;       // a warp's ring
  static constexpr int SMEM = kWarps * WARP;
  // merging the warps at the end reuses the rings: per warp 16 MT rows of O
  static constexpr int merge(int mt) { return kWarps * 16 * mt * (HDP + 2) * 4; }
  static constexpr int smem(int mt) { return SMEM > merge(mt) ? SMEM : merge(mt); }
};

// Byte offset of 16-byte chunk c of row r inside a tile: the chunk index is mixed with the row so that
// eight rows' equal chunks (one ldmatrix phase) fall into different banks.
template <int HDP>
__device__ __forceinline__ uint32_t tile_at(int r, int c) {
  return (uint32_t)(r * Cfg<HDP>::ROW + ((c & ~7) | ((c ^ r) & 7)) * 16);
}

template <int HDP, int MT>
__global__ void __launch_bounds__(kThreads) item_kernel(const Params p) {
  using C = Cfg<HDP>;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int M = 16 * MT;

  // ---- which rows against which keys
  int i = blockIdx.x;
  const int prefix_items = p.P * p.Hkv * p.rt_p;  // none when tcgen05 takes the prefix
  const bool is_prefix = i < prefix_items;
  int hk, r0, r_end, k0, k1, slot, max_pages;
  const int* pages;
  if (is_prefix) {
    slot = i % p.P;
    i /= p.P;
    r0 = (i % p.rt_p) * M;
    hk = i / p.rt_p;
    r_end = p.B * p.Q * p.G;
    k0 = slot * p.per_p;
    k1 = min(k0 + p.per_p, p.L);
    pages = p.pages;
    max_pages = (p.L + p.bs - 1) / p.bs;
  } else {
    i -= prefix_items;
    const int t = i % p.T;
    i /= p.T;
    hk = i % p.Hkv;
    i /= p.Hkv;
    const int b = i / p.rt_t;
    const Seq s = seq_of(p, b, threadIdx.x == 0);
    const int share = tail_share(p, s);
    k0 = s.start + t * share;
    k1 = min(k0 + share, s.len);
    slot = p.P + t;
    r0 = b * p.Q * p.G + (i % p.rt_t) * M;
    r_end = (b + 1) * p.Q * p.G;
    pages = p.tables + (long)b * p.table_stride;
    max_pages = p.max_pages;
    if (k0 >= k1) return;  // the combine kernel knows the splits that hold keys
  }

  // ---- this thread's rows: r0 + 16 mt + lane / 4 (+ 8)
  int limit[MT][2];
  uint32_t qf[MT][HDP / 16][4];
  int lo = 0x7fffffff;  // the smallest limit of a row that sees any of these keys
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = r0 + 16 * mt + 8 * h + (lane >> 2);
      int lim = 0;
      const bf16* src = nullptr;
      if (r < r_end) {
        const int bt = r / p.G, b = bt / p.Q, t = bt % p.Q;
        const Seq s = seq_of(p, b);
        if (t < s.ql && (!is_prefix || s.start == p.L)) lim = max(s.len - s.ql + t + 1, 0);
        src = p.q + b * p.q_sb + t * p.q_st + (long)(hk * p.G + r % p.G) * p.q_sh;
      }
      limit[mt][h] = lim;
      if (lim > k0) lo = min(lo, lim);
#pragma unroll
      for (int kk = 0; kk < HDP / 16; ++kk)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int d = kk * 16 + e * 8 + (lane & 3) * 2;
          qf[mt][kk][e * 2 + h] = (src != nullptr && d < p.HD) ? *reinterpret_cast<const uint32_t*>(src + d) : 0u;
        }
    }
  lo = __reduce_min_sync(0xffffffffu, lo);

  float o[MT][HDP / 8][4];
  float m_run[MT][2], l_run[MT][2];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
    for (int n = 0; n < HDP / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[mt][n][e] = 0.f;
    m_run[mt][0] = m_run[mt][1] = -INFINITY;
    l_run[mt][0] = l_run[mt][1] = 0.f;
  }

  // ---- the ring of this warp: K tiles then V tiles
  uint8_t* ring = smem + warp * C::WARP;
  const uint32_t ring_a = smem_u32(ring);
  const int chunks = p.HD / 8;  // 16-byte chunks that a row has; the rest of a padded row stays zero
  if (chunks < HDP / 8) {
    for (int j = lane; j < C::WARP / 16; j += 32) reinterpret_cast<uint4*>(ring)[j] = make_uint4(0, 0, 0, 0);
    __syncwarp();
  }
  const int first = k0 + warp * kTile;
  const int steps = first < k1 ? (k1 - first + kStep - 1) / kStep : 0;
  uint32_t valid[kStages - 1];  // of the steps on their way: the keys that are read (bit = key)

  auto load = [&](int j, int s) -> uint32_t {
    const int key = first + j * kStep + lane;  // lanes 0-15 look their key's page up
    const long off = lane < kTile && key < k1 ? pool_row(p, pages, max_pages, key, hk) : -1;
    constexpr int RPI = 32 / (HDP / 8);  // rows per instruction
    const int c = lane % (HDP / 8);
#pragma unroll
    for (int j2 = 0; j2 < kTile / RPI; ++j2) {
      const int r = j2 * RPI + lane / (HDP / 8);
      const long ro = __shfl_sync(0xffffffffu, off, r);
      if (c < chunks) {
        const uint32_t d = ring_a + s * 2 * C::KV + tile_at<HDP>(r, c);
        const long e = (ro < 0 ? 0 : ro) + c * 8;
        cp_async16(d, p.k + e, ro >= 0);
        cp_async16(d + C::KV, p.v + e, ro >= 0);
      }
    }
    return __ballot_sync(0xffffffffu, off >= 0);
  };

#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) {
    valid[s] = s < steps ? load(s, s) : 0u;
    cp_commit();
  }

  for (int j = 0; j < steps; ++j) {
    const int s = j % kStages;
    cp_wait<kStages - 2>();
    __syncwarp();
    uint32_t vm;
    {
      const int sn = (j + kStages - 1) % kStages;
      vm = valid[0];
#pragma unroll
      for (int e = 0; e + 2 < kStages; ++e) valid[e] = valid[e + 1];
      valid[kStages - 2] = j + kStages - 1 < steps ? load(j + kStages - 1, sn) : 0u;
      cp_commit();
    }
    const uint32_t ka = ring_a + s * 2 * C::KV, va = ka + C::KV;
    const int key0 = first + j * kStep;

    // S = Q K^T: two 8-key column groups
    float sc[MT][2][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[mt][n][e] = 0.f;
#pragma unroll
    for (int kk = 0; kk < HDP / 16; ++kk) {
      uint32_t kb[4];  // (keys 0-7, dims 0-7), (keys 0-7, dims 8-15), (keys 8-15, ...)
      ldsm4(kb, ka + tile_at<HDP>((lane & 7) + ((lane >> 4) & 1) * 8, kk * 2 + ((lane >> 3) & 1)));
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        mma16816(sc[mt][0], qf[mt][kk], kb[0], kb[1]);
        mma16816(sc[mt][1], qf[mt][kk], kb[2], kb[3]);
      }
    }
    // softmax step: this thread holds keys key0 + 8 n + 2 (lane & 3) + {0, 1} of its rows
    const bool masked = vm != 0xffffu || key0 + kTile > lo;
    uint32_t pa[MT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float x[4];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int kl = n * 8 + (lane & 3) * 2 + e;
            const float v = sc[mt][n][2 * h + e] * p.scale_log2;
            x[n * 2 + e] = !masked || (((vm >> kl) & 1u) && key0 + kl < limit[mt][h]) ? v : -INFINITY;
          }
        if (!masked && limit[mt][h] <= k0) x[0] = x[1] = x[2] = x[3] = -INFINITY;  // a row that sees nothing here
        float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mn = fmaxf(m_run[mt][h], mx);
        const float ref = mn == -INFINITY ? 0.f : mn;
        const float alpha = ex2_fast(m_run[mt][h] - ref);  // 2^-inf = 0 before the first key
        m_run[mt][h] = mn;
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = ex2_fast(x[e] - ref);
          sum += x[e];
        }
        l_run[mt][h] = l_run[mt][h] * alpha + sum;  // this thread's keys; the four lanes are added up at the end
        pa[mt][h] = pack_bf16x2(x[0], x[1]);
        pa[mt][2 + h] = pack_bf16x2(x[2], x[3]);
#pragma unroll
        for (int n = 0; n < HDP / 8; ++n) {
          o[mt][n][2 * h] *= alpha;
          o[mt][n][2 * h + 1] *= alpha;
        }
      }
    // a tile with keys that only some rows see: look for V values that a zero would not cancel
    bool odd = false;
    if (key0 + kTile > lo) {
      for (int c = lane; c < kTile * chunks; c += 32) {
        const uint4 w = *reinterpret_cast<const uint4*>(ring + s * 2 * C::KV + C::KV + tile_at<HDP>(c / chunks, c % chunks));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t x = (&w.x)[e];
          odd |= (x & 0x7f80u) == 0x7f80u || (x & 0x7f800000u) == 0x7f800000u;
        }
      }
      odd = __any_sync(0xffffffffu, odd);
    }
    if (!odd) {
      // O += P V
#pragma unroll
      for (int n2 = 0; n2 < HDP / 16; ++n2) {
        uint32_t vb[4];  // (keys 0-7, dims 0-7), (keys 8-15, dims 0-7), (keys 0-7, dims 8-15), ...
        ldsm4_t(vb, va + tile_at<HDP>(lane & 15, n2 * 2 + (lane >> 4)));
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          mma16816(o[mt][n2 * 2], pa[mt], vb[0], vb[1]);
          mma16816(o[mt][n2 * 2 + 1], pa[mt], vb[2], vb[3]);
        }
      }
    } else {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll 1
        for (int kl = 0; kl < kTile; ++kl) {
          const int owner = (lane & ~3) | ((kl & 7) >> 1);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t w = __shfl_sync(0xffffffffu, kl < 8 ? pa[mt][h] : pa[mt][2 + h], owner);
            const float pv = (kl & 1) ? bf16_hi(w) : bf16_lo(w);
            const bool sees = ((vm >> kl) & 1u) && key0 + kl < limit[mt][h];
#pragma unroll
            for (int n = 0; n < HDP / 8; ++n) {
              const uint32_t x = *reinterpret_cast<const uint32_t*>(ring + s * 2 * C::KV + C::KV + tile_at<HDP>(kl, n) +
                                                                    (lane & 3) * 4);
              if (sees) {
                o[mt][n][2 * h] = fmaf(pv, bf16_lo(x), o[mt][n][2 * h]);
                o[mt][n][2 * h + 1] = fmaf(pv, bf16_hi(x), o[mt][n][2 * h + 1]);
              }
            }
          }
        }
    }
    __syncwarp();  // the tile has been read before the next step's copies overwrite it
  }
  cp_wait<0>();

  // ---- join the four warps, write this split's part of every row
  __syncthreads();
  float* mo = reinterpret_cast<float*>(smem);           // [warp][M][HDP]
  float* mml = mo + kWarps * M * HDP;                   // [warp][M][2]
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = 16 * mt + 8 * h + (lane >> 2);
      float l = l_run[mt][h];
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      if ((lane & 3) == 0) {
        mml[(warp * M + r) * 2] = m_run[mt][h];
        mml[(warp * M + r) * 2 + 1] = l;
      }
#pragma unroll
      for (int n = 0; n < HDP / 8; ++n)
        *reinterpret_cast<float2*>(mo + (warp * M + r) * HDP + n * 8 + (lane & 3) * 2) =
            make_float2(o[mt][n][2 * h], o[mt][n][2 * h + 1]);
    }
  __syncthreads();
  const int slots = p.P + p.T;
  for (int r = warp; r < M && r0 + r < r_end; r += kWarps) {
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, mml[(w * M + r) * 2]);
    const float ref = m == -INFINITY ? 0.f : m;
    float f[kWarps], l = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      f[w] = ex2_fast(mml[(w * M + r) * 2] - ref);
      l += f[w] * mml[(w * M + r) * 2 + 1];
    }
    const int gr = r0 + r, bt = gr / p.G, head = hk * p.G + gr % p.G;
    const long at = ((long)bt * p.H + head) * slots + slot;
    for (int d = lane; d < p.HD; d += 32) {
      float acc = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w)
        if (f[w] != 0.f) acc += f[w] * mo[(w * M + r) * HDP + d];
      p.part_o[at * p.HD + d] = acc;
    }
    if (lane == 0) {
      p.part_ml[at * 2] = m;
      p.part_ml[at * 2 + 1] = l;
    }
  }
}

// One CTA per output row; its warps take every fourth part.
__global__ void __launch_bounds__(128) combine_kernel(const Params p) {
  const long row = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __shared__ float4 acc_s[4][32];
  __shared__ float den_s[4];
  const int b = (int)(row / ((long)p.Q * p.H));
  const int t = (int)(row / p.H % p.Q);
  const Seq s = seq_of(p, b);
  const int share = tail_share(p, s), n = max(s.len - s.start, 0);
  // the slots that hold parts of this row: the prefix's, if the sequence takes part in it, and its tail's
  int np = 0;  // prefix slots
  if (t < s.ql && s.start == p.L) {
    np = p.P;
    if (p.tc_share > 0) {
      // the CTAs whose blocks meet the row tile's
      const int h = (int)(row % p.H), hk = h / p.G, r = (b * p.Q + t) * p.G + h % p.G;
      const int first = (hk * p.tc_tiles + r / p.tc_rows) * p.tc_blocks;
      np = ((first + p.tc_blocks - 1) / p.tc_share - first / p.tc_share + 1) * p.tc_streams;
    }
  }
  const int nt = t < s.ql && n > 0 ? (n + share - 1) / share : 0;  // tail slots
  const int slots = p.P + p.T;
  const float* ml = p.part_ml + row * slots * 2;
  const float* po = p.part_o + row * slots * p.HD;
  const auto slot_of = [&](int j) { return j < np ? j : p.P + j - np; };
  float m = -INFINITY;
  for (int j = lane; j < np + nt; j += 32) m = fmaxf(m, ml[2 * slot_of(j)]);
  m = warp_max(m);
  const float ref = m == -INFINITY ? 0.f : m;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float den = 0.f;
  const bool on = 4 * lane < p.HD;
#pragma unroll 4
  for (int j = warp; j < np + nt; j += 4) {
    const int i = slot_of(j);
    const float2 v = *reinterpret_cast<const float2*>(ml + 2 * i);
    const float4 o = on ? *reinterpret_cast<const float4*>(po + (long)i * p.HD + 4 * lane) : acc;
    const float w = ex2_fast(v.x - ref);
    if (w != 0.f) {  // (a part without keys holds nothing)
      den += w * v.y;
      acc.x += w * o.x;
      acc.y += w * o.y;
      acc.z += w * o.z;
      acc.w += w * o.w;
    }
  }
  acc_s[warp][lane] = acc;
  if (lane == 0) den_s[warp] = den;
  __syncthreads();
  if (warp != 0 || !on) return;
#pragma unroll
  for (int w = 1; w < 4; ++w) {
    const float4 o = acc_s[w][lane];
    acc.x += o.x;
    acc.y += o.y;
    acc.z += o.z;
    acc.w += o.w;
    den += den_s[w];
  }
  uint2 out = make_uint2(0u, 0u);
  if (den != 0.f) {
    const float inv = 1.f / den;
    out = make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
  }
  *reinterpret_cast<uint2*>(p.out + row * p.HD + 4 * lane) = out;
}

}  // namespace prefix

// q [B, Q, H, HD] bf16 (inner dimension contiguous) -> [B, Q, H, HD] bf16. Pools [num_pages, block_size,
// Hkv, HD] bf16; tables int32 [B, max_pages] (each sequence's whole chain), lens int32 [B], pages int32
// [>= ceil(L / block_size)] (the prefix's chain), qlens int32 [B] or none.
constexpr int64_t kTcRows = 32, kTcKeys = 256;

torch::Tensor paged_prefix_attention(torch::Tensor q, torch::Tensor k_pool, torch::Tensor v_pool, torch::Tensor tables,
                                     torch::Tensor lens, torch::Tensor pages, int64_t L,
                                     c10::optional<torch::Tensor> qlens, double scale) {
  CHECK_CUDA_TENSOR(q);
  CHECK_DTYPE(q, at::kBFloat16);
  CHECK_DTYPE(k_pool, at::kBFloat16);
  CHECK_DTYPE(v_pool, at::kBFloat16);
  TORCH_CHECK(q.dim() == 4, "q must be [B, Q, H, HD]");
  const int64_t B = q.size(0), Q = q.size(1), H = q.size(2), HD = q.size(3);
  TORCH_CHECK(k_pool.dim() == 4 && k_pool.sizes() == v_pool.sizes() && k_pool.is_contiguous() &&
                  v_pool.is_contiguous() && k_pool.size(3) == HD,
              "pools must be contiguous [num_pages, block_size, Hkv, ", num(HD), "]");
  const int64_t num_pages = k_pool.size(0), bs = k_pool.size(1), Hkv = k_pool.size(2);
  TORCH_CHECK(HD % 8 == 0 && HD >= 8 && HD <= 128, "head_dim must be a multiple of 8 up to 128, got ", num(HD));
  TORCH_CHECK(Hkv > 0 && bs > 0 && H > 0 && H % Hkv == 0, "query heads must be a multiple of the cached heads");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(k_pool.data_ptr()) % 16 == 0 &&
                  reinterpret_cast<uintptr_t>(v_pool.data_ptr()) % 16 == 0,
              "pools must be 16-byte aligned");
  const bool has_ql = qlens.has_value() && qlens->defined();
  auto ints = [&](const torch::Tensor& t, const char* what) {
    TORCH_CHECK(t.scalar_type() == at::kInt && t.is_contiguous() && t.device() == q.device(), what,
                ": contiguous int32 on q's device");
  };
  ints(tables, "block tables");
  ints(lens, "sequence lengths");
  ints(pages, "prefix pages");
  if (has_ql) ints(*qlens, "query lengths");
  TORCH_CHECK(k_pool.device() == q.device() && v_pool.device() == q.device(), "pools and q on different devices");
  TORCH_CHECK(tables.dim() == 2 && tables.size(0) == B && lens.numel() == B && (!has_ql || qlens->numel() == B),
              "one table row, length and query length per sequence");
  const int64_t max_pages = tables.size(1);
  TORCH_CHECK(num_pages > 0 || L == 0, "an empty pool holds no prefix");
  TORCH_CHECK(L >= 0 && L <= pages.numel() * bs && L <= max_pages * bs, "a prefix of ", num(L),
              " tokens is longer than its pages or than a chain");
  TORCH_CHECK(max_pages * bs < (1LL << 30) && B * Q * H < (1LL << 30), "paged attention: too large");
  c10::cuda::CUDAGuard guard(q.get_device());
  auto out = at::empty({B, Q, H, HD}, q.options());
  if (out.numel() == 0) return out;
  if (q.stride(3) != 1 || q.stride(0) % 8 || q.stride(1) % 8 || q.stride(2) % 8 ||
      reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 != 0)
    q = q.clone(at::MemoryFormat::Contiguous);  // (contiguous() would keep a contiguous tensor at an odd offset)
  prefix::Params p{};
  p.q = reinterpret_cast<const prefix::bf16*>(q.data_ptr());
  p.k = reinterpret_cast<const prefix::bf16*>(k_pool.data_ptr());
  p.v = reinterpret_cast<const prefix::bf16*>(v_pool.data_ptr());
  p.out = reinterpret_cast<prefix::bf16*>(out.data_ptr());
  p.tables = tables.data_ptr<int>();
  p.lens = lens.data_ptr<int>();
  p.qlens = has_ql ? qlens->data_ptr<int>() : nullptr;
  p.pages = pages.data_ptr<int>();
  p.q_sb = q.stride(0);
  p.q_st = q.stride(1);
  p.q_sh = q.stride(2);
  p.table_stride = p.max_pages = (int)max_pages;
  p.num_pages = (int)num_pages;
  p.B = (int)B;
  p.Q = (int)Q;
  p.H = (int)H;
  p.Hkv = (int)Hkv;
  p.G = (int)(H / Hkv);
  p.HD = (int)HD;
  p.bs = (int)bs;
  p.L = (int)L;
  p.scale_log2 = (float)(scale * 1.4426950408889634);
  p.st = status_ptr(q.get_device());

  const int64_t seq_rows = Q * p.G, rows = B * seq_rows;
  const int sms = num_sms(q.get_device());
  const bool tc = L >= kTcKeys && rows > kTcRows;
  const int mt = std::max(L > 0 && !tc ? rows : 0, seq_rows) > 16 ? 2 : 1;
  p.rt_p = L > 0 && !tc ? (int)((rows + 16 * mt - 1) / (16 * mt)) : 0;
  p.rt_t = (int)((seq_rows + 16 * mt - 1) / (16 * mt));
  // equal shares of keys for about four items per SM
  const int64_t span = max_pages * bs - L;
  const int64_t work = Hkv * (p.rt_p * L + B * p.rt_t * span);
  int64_t unit = work / (4LL * sms);
  unit = std::max<int64_t>(256, (unit + prefix::kStep - 1) / prefix::kStep * prefix::kStep);
  p.P = tc ? 0 : (int)((L + unit - 1) / unit);
  p.per_p = (int)unit;
  p.T = (int)std::max<int64_t>(1, (span + unit - 1) / unit);
  if (tc) prefix::plan_prefix_tc(p, sms);
  const int slots = p.P + p.T;
  auto part_o = at::empty({B * Q * H, slots, HD}, q.options().dtype(at::kFloat));
  auto part_ml = at::empty({B * Q * H, slots, 2}, q.options().dtype(at::kFloat));
  p.part_o = part_o.data_ptr<float>();
  p.part_ml = part_ml.data_ptr<float>();
  const int64_t items = Hkv * ((int64_t)p.rt_p * p.P + B * p.rt_t * p.T);
  if (tc) {
    prefix::launch_prefix_tc(p, cur_stream());
    SCIRS_CHECK_LAUNCH();
  }
  TORCH_CHECK(items < (1LL << 31), "paged attention: too large");
  auto st = cur_stream();
#define SCIRS_ITEMS(HDP_, MT_)                                              \
  {                                                                         \
    auto kern = prefix::item_kernel<HDP_, MT_>;                             \
    set_max_smem((const void*)kern, prefix::Cfg<HDP_>::smem(MT_));          \
    kern<<<(unsigned)items, prefix::kThreads, prefix::Cfg<HDP_>::smem(MT_), st>>>(p); \
  }
  if (HD <= 64) {
    if (mt == 1) SCIRS_ITEMS(64, 1) else SCIRS_ITEMS(64, 2)
  } else {
    if (mt == 1) SCIRS_ITEMS(128, 1) else SCIRS_ITEMS(128, 2)
  }
#undef SCIRS_ITEMS
  SCIRS_CHECK_LAUNCH();
  prefix::combine_kernel<<<(unsigned)(B * Q * H), 128, 0, st>>>(p);
  SCIRS_CHECK_LAUNCH();
  return out;
}

}  // namespace scirs
