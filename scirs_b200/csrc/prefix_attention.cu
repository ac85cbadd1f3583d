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
//   from its first key, so that in a prefix item a row sees every key or none. Behind long prefixes spare items
//   take parts of such sequences.
//
// An item belongs to a CTA of four warps. Each walks every fourth tile of 16 keys, K and V rows of one head
// copied into a ring of its own: by TMA where head_dim is 64 or 128 and the page size a multiple of 8, else by
// cp.async (16 bytes a lane, the same swizzle, free of bank conflicts for ldmatrix); S = Q K^T and O += P V by
// mma.sync m16n8k16 with the running max and sum in registers. The warps meet once, at the end. What bounds
// an item is the chain length -> page ids -> first tile (so page ids are read 32 boxes at a time, and before
// the length where the split does not depend on it), and memory over many items.
//
// P is rounded to bf16, as the tensor cores take it beside V; its sum is formed from the unrounded values, and
// maxima, sums and O are fp32. That puts the output off by up to 2^-8 sum p |v| next to its own rounding: 1.9e-3 to
// 2.4e-3 of its 2-norm on random inputs, 1.7e-3 with P in fp32. P as two bf16 terms would take that back at twice the
// MMAs of P V, which run one after the other with the softmax.
//
// Masked places (keys past a row's limit, slots past the length or before the item's first key) get P = 0
// by selection. Where a tile has any and one of its V values is infinite or NaN, P V is formed row by row
// without the masked keys, since 0 * NaN would reach the rows that do not see them.
//
// Measured (tails alone): 256 sequences of 512 tokens on average, 8 cached heads of 128 (537 MB), 100 us, 5.4 TB/s,
// 0.82 of the device's copy rate; 64 of 256 (67 MB) 23 us, where an item's start is half of its time; 4 sequences
// of 32 tokens and a prefix of 512, 12 heads of 64, 4.9 us. Joining 2048 rows of 20 parts 9 us, 8192 of 9 12 us.
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
  static constexpr int HALF = kTile * 128;           // 64 columns of a K or V tile
  static constexpr int KV = HALF * (HDP / 64);       // a K or V tile
  static constexpr int STAGES = 3;
  static constexpr int WARP = STAGES * 2 * KV;       // a warp's ring
  // joining the warps at the end reuses the rings: 16 MT rows of O and (max, sum) a warp
  static constexpr int smem(int mt) {
    const int merge = kWarps * 16 * mt * (HDP + 2) * 4;
    return (kWarps * WARP > merge ? kWarps * WARP : merge) + 1024;
  }
  // per SM, by registers and shared memory
  static constexpr int ctas(int mt) { return HDP == 64 && mt == 1 ? 3 : 2; }
};

// Byte offset of 16-byte chunk c of row r inside a tile: [64-column half][row][128 bytes], the chunk index
// mixed with the row (TMA's 128-byte swizzle), so that eight rows' equal chunks (one ldmatrix phase) fall
// into different banks.
template <int HDP>
__device__ __forceinline__ uint32_t tile_at(int r, int c) {
  return (uint32_t)((c >> 3) * Cfg<HDP>::HALF + r * 128 + ((c ^ r) & 7) * 16);
}

// W: warps of an item; the CTA's four warps take one item together, or one each. SPARE: there are spare items.
template <int HDP, int MT, bool TMA, int W, bool SPARE>
__global__ void __launch_bounds__(kThreads, Cfg<HDP>::ctas(MT)) item_kernel(const __grid_constant__ CUtensorMap map_k,
                                                                             const __grid_constant__ CUtensorMap map_v,
                                                                             const Params p) {
  using C = Cfg<HDP>;
  constexpr int M = 16 * MT;
  allow_next();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full_s[kWarps][C::STAGES];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part_w = warp % W;  // which of the item's warps this is
  uint64_t* full = full_s[warp];
  uint8_t* ring = smem + warp * C::WARP;
  const uint32_t ring_a = smem_u32(ring);

  // ---- which rows against which keys. Neighbouring items are the cached heads of the same keys, which lie
  // side by side in a page.
  int i = blockIdx.x * (kWarps / W) + warp / W;
  if (i >= p.items + (SPARE ? p.spare : 0)) {
    wait_for_previous();
    return;
  }
  const bool is_spare = SPARE && i >= p.items;
  if (is_spare) i -= p.items;
  const int hk = i % p.Hkv;
  i /= p.Hkv;
  const bool is_prefix = !is_spare && i < p.P * p.rt_p;  // (rt_p = 0 when tcgen05 takes the prefix)
  int r0, r_end, split, slot, b = 0;  // (slot: where this part of a row goes)
  const int* pages;
  if (is_prefix) {
    slot = split = i % p.P;
    r0 = i / p.P * M;
    r_end = p.B * p.Q * p.G;
    pages = p.pages;
  } else {
    if (is_spare) {  // a part of a row tile of one of the sequences that end inside the prefix
      const int inside = count_inside(p, lane), parts = inside > 0 ? spare_parts(p, inside) : 0;
      if (i >= inside * p.rt_t * parts) {
        wait_for_previous();
        return;
      }
      split = p.T + i % parts;
      i /= parts;
      b = nth_inside(p, i / p.rt_t, lane);
      i %= p.rt_t;
    } else {
      i -= p.P * p.rt_p;
      split = i % p.T;
      slot = p.P + split;
      i /= p.T;
      b = i / p.rt_t;
      i -= b * p.rt_t;
    }
    r0 = b * p.Q * p.G + i * M;
    r_end = (b + 1) * p.Q * p.G;
    pages = p.tables + (long)b * p.max_pages;
  }
  const int max_pages = is_prefix ? p.pages_max : p.max_pages;

  // ---- page ids: with TMA a lane holds the page and slot of one box, 32 boxes of this warp's tiles at a time
  // (tile j of the warp begins at base + (W j + its part) 16); with cp.async lanes 0-15 hold one tile's keys
  const int runs = TMA ? kTile / p.box : 1;  // boxes of a tile
  int base = is_prefix ? split * p.per_p : p.L & ~(kTile - 1), k1 = 0x7fffffff;
  int page = -2, at = 0, batch = 0;
  auto look_up = [&](int j) {  // TMA: the boxes of tiles j, j + 1, ..; cp.async: the keys of tile j
    const int key = TMA ? base + (((j + lane / runs) * W + part_w) * kTile + lane % runs * p.box)
                        : base + (j * W + part_w) * kTile + lane;
    const int pi = page_of(p, key);
    page = (TMA || lane < kTile) && key >= 0 && key < k1 && pi < max_pages ? pages[pi] : -2;
    at = key - pi * p.bs;
    batch = j;
  };
  // the whole tail in one item: its pages can be read before its length is known
  const bool early = TMA && (is_prefix || (p.T == 1 && !is_spare));
  if (early) look_up(0);

  int k0, len = 0, ql = 0;
  if (is_prefix) {
    k0 = base;
    k1 = min(base + p.per_p, p.L);
  } else {
    const Seq s = seq_from(p, p.lens[b], p.qlens != nullptr ? p.qlens[b] : p.Q, lane == 0 && part_w == 0);
    int parts = p.T;
    if (SPARE && ends_inside(p, s)) {
      parts += spare_parts(p, count_inside(p, lane));
      slot = spare_at(p) + split;
    }
    const int share = tail_share(s, parts);
    const int first = first_key(s) + split * share;
    k0 = max(first, s.start);
    k1 = min(first + share, s.len);
    if (k0 >= k1) {  // the combine kernel knows the splits that hold keys
      wait_for_previous();
      return;
    }
    len = s.len;
    ql = s.ql;
    if (first != base || !early) {
      base = first;
      if (TMA) look_up(0);
    }
  }
  const int tiles = max((k1 - base + kTile - 1) / kTile - part_w + W - 1, 0) / W;  // of this warp
  if (lane == 0) {
    for (int s = 0; s < C::STAGES; ++s) mbar_init(&full[s], 1);
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  const int chunks = p.HD / 8;  // 16-byte chunks that a row has; the rest of a padded row stays zero
  if (!TMA && chunks < HDP / 8)
    for (int j = lane; j < C::WARP / 16; j += 32) reinterpret_cast<uint4*>(ring)[j] = make_uint4(0, 0, 0, 0);
  __syncwarp();

  // Copy tile j into a stage; returns which of its keys are to be used (bit = key).
  auto copy = [&](int j, int stage) -> uint32_t {
    uint32_t valid;
    uint8_t* dst = ring + stage * 2 * C::KV;
    const int key0 = base + (j * W + part_w) * kTile;
    if (TMA) {
      if ((j - batch + 1) * runs > 32) look_up(j);
      // boxes of the whole tile, or, a lane each, of 8 keys and one half of the columns; a box that is not
      // read is taken off the bytes to wait for
      const int from = (j - batch) * runs;
      const int pg0 = __shfl_sync(0xffffffffu, page, from), sl0 = __shfl_sync(0xffffffffu, at, from);
      if (runs == 1) {
        const bool good = pg0 != -2 && input_in_range(pg0, p.num_pages, p.st, 96);
        if (lane == 0) {
          mbar_arrive_expect_tx(&full[stage], good ? 2 * C::KV : 0);
          if (good) {
            tma_load_5d(dst, &map_k, &full[stage], 0, sl0, 0, hk, pg0);
            tma_load_5d(dst + C::KV, &map_v, &full[stage], 0, sl0, 0, hk, pg0);
          }
        }
        valid = good ? 0xffffu : 0u;
      } else {
        const int pg1 = __shfl_sync(0xffffffffu, page, from + 1), sl1 = __shfl_sync(0xffffffffu, at, from + 1);
        // (ids that were read before the length may lie past the chain's end)
        const int q = lane & 1, h = lane >> 2, pg = !q ? pg0 : key0 + 8 < k1 ? pg1 : -2;
        const bool good = pg != -2 && input_in_range(pg, p.num_pages, p.st, 96);
        const uint32_t ok = __ballot_sync(0xffffffffu, good) & 3u;
        if (lane == 0) mbar_arrive_expect_tx(&full[stage], __popc(ok) * C::KV);
        __syncwarp();
        if (h < HDP / 64 && good)
          tma_load_5d(dst + (lane >> 1 & 1) * C::KV + h * C::HALF + q * 1024, (lane & 2) ? &map_v : &map_k,
                      &full[stage], 0, q ? sl1 : sl0, h, hk, pg);
        valid = (ok & 1u ? 0xffu : 0u) | (ok & 2u ? 0xff00u : 0u);
      }
    } else {
      if (batch != j || j == 0) look_up(j);
      const bool good = page != -2 && input_in_range(page, p.num_pages, p.st, 96);
      const long off = good ? (((long)page * p.bs + at) * p.Hkv + hk) * p.HD : -1;
      constexpr int RPI = 32 / (HDP / 8);  // rows per instruction
      const int c = lane % (HDP / 8);
#pragma unroll
      for (int n = 0; n < kTile / RPI; ++n) {
        const int r = n * RPI + lane / (HDP / 8);
        const long ro = __shfl_sync(0xffffffffu, off, r);
        if (c < chunks) {
          const uint32_t d = smem_u32(dst) + tile_at<HDP>(r, c);
          const long e = (ro < 0 ? 0 : ro) + c * 8;
          cp_async16(d, p.k + e, ro >= 0);
          cp_async16(d + C::KV, p.v + e, ro >= 0);
        }
      }
      cp_commit();
      valid = __ballot_sync(0xffffffffu, good);
      look_up(j + 1);  // (in time for the next tile)
    }
    if (key0 < k0) valid &= 0xffffu << (k0 - key0);
    if (key0 + kTile > k1) valid &= 0xffffu >> (key0 + kTile - k1);
    return valid;
  };

  int limit[MT][2];  // keys that rows r0 + 16 mt + lane / 4 (+ 8) see
  uint32_t qf[MT][HDP / 16][4];
  float o[MT][HDP / 8][4];
  float m_run[MT][2], l_run[MT][2];
  int lo = 0x7fffffff;  // the smallest limit of a row that sees any of these keys
  int flying = 0, next = 0, s = 0, sw = 0;  // tiles on their way, the next one to copy; stages to read and to write
  uint32_t phase = 0;
  uint64_t valid_q = 0;  // 16 bits a tile on its way
  for (int j = 0; j < tiles;) {
    // (every piece of code stands in the loop once: what is fetched for the first time costs a short call most)
    while (next < tiles && flying < C::STAGES) {
      valid_q |= (uint64_t)copy(next, sw) << (16 * flying);
      ++next;
      ++flying;
      sw = sw + 1 == C::STAGES ? 0 : sw + 1;
    }
    if (j == 0) {  // the queries, while the first tiles are on their way
      const bf16* src[MT][2];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = r0 + 16 * mt + 8 * h + (lane >> 2);
          const int bt = r / p.G, rb = bt / p.Q, t = bt - rb * p.Q;
          src[mt][h] = r < r_end ? p.q + rb * p.q_sb + t * p.q_st + (long)(hk * p.G + r - bt * p.G) * p.q_sh : nullptr;
          int lim = 0;
          if (r < r_end) {
            if (is_prefix) {
              const Seq q = seq_of(p, rb);
              if (t < q.ql && q.start == p.L) lim = q.len - q.ql + t + 1;
            } else if (t < ql) {
              lim = max(len - ql + t + 1, 0);
            }
          }
          limit[mt][h] = lim;
          if (lim > k0) lo = min(lo, lim);
          m_run[mt][h] = -INFINITY;
          l_run[mt][h] = 0.f;
#pragma unroll
          for (int n = 0; n < HDP / 8; ++n) o[mt][n][2 * h] = o[mt][n][2 * h + 1] = 0.f;
        }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int kk = 0; kk < HDP / 16; ++kk)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int d = kk * 16 + (e >> 1) * 8 + (lane & 3) * 2;
            qf[mt][kk][e] = src[mt][e & 1] != nullptr && d < p.HD
                                ? __ldg(reinterpret_cast<const uint32_t*>(src[mt][e & 1] + d))
                                : 0u;
          }
      lo = __reduce_min_sync(0xffffffffu, lo);
    }
    if (TMA) {
      if (!mbar_wait(&full[s], phase, p.st, 97, nullptr)) break;
    } else {
      if (flying > 2)
        cp_wait<2>();
      else if (flying == 2)
        cp_wait<1>();
      else
        cp_wait<0>();
    }
    __syncwarp();
    const uint32_t vm = (uint32_t)valid_q & 0xffffu;  // the tile's keys that are used
    const int key0 = base + (j * W + part_w) * kTile;
    ++j;
    valid_q >>= 16;
    --flying;
    uint8_t* const vt = ring + s * 2 * C::KV + C::KV;
    const uint32_t ka = ring_a + s * 2 * C::KV, va = ka + C::KV;

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
    float alpha[MT][2];
    bool rescale = false;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float x[4] = {sc[mt][0][2 * h], sc[mt][0][2 * h + 1], sc[mt][1][2 * h], sc[mt][1][2 * h + 1]};
        if (masked) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int kl = (e >> 1) * 8 + (lane & 3) * 2 + (e & 1);
            if (!((vm >> kl) & 1u) || key0 + kl >= limit[mt][h]) x[e] = -INFINITY;
          }
        } else if (limit[mt][h] <= k0) {
          x[0] = x[1] = x[2] = x[3] = -INFINITY;  // a row that sees nothing here
        }
        float mx = max_nan(max_nan(x[0], x[1]), x[2], x[3]);
        mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        mx *= p.scale_log2;
        // the reference maximum is raised only when it grew by more than 2^8: P stays below 2^8
        alpha[mt][h] = 1.f;
        if (mx > m_run[mt][h] + kRaise) {
          alpha[mt][h] = ex2_fast(m_run[mt][h] - mx);  // 2^-inf = 0 before the first key
          m_run[mt][h] = mx;
          rescale = true;
        }
        if (!(mx < INFINITY)) m_run[mt][h] = NAN;  // a score that is NaN or infinite makes the row NaN
        const float ref = m_run[mt][h] == -INFINITY ? 0.f : m_run[mt][h];
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = ex2_fast(fmaf(x[e], p.scale_log2, -ref));
          sum += x[e];
        }
        l_run[mt][h] = l_run[mt][h] * alpha[mt][h] + sum;  // this thread's keys; the four lanes are added up at the end
        pa[mt][h] = pack_bf16x2(x[0], x[1]);
        pa[mt][2 + h] = pack_bf16x2(x[2], x[3]);
      }
    if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int n = 0; n < HDP / 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[mt][n][e] *= alpha[mt][e >> 1];
    }
    // a tile with places that not every row sees: look for V values that a zero would not cancel
    bool odd = false;
    if (masked) {
      for (int c = lane; c < kTile * chunks; c += 32) {
        const uint4 w = *reinterpret_cast<const uint4*>(vt + tile_at<HDP>(c / chunks, c % chunks));
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
              const uint32_t x = *reinterpret_cast<const uint32_t*>(vt + tile_at<HDP>(kl, n) + (lane & 3) * 4);
              if (sees) {
                o[mt][n][2 * h] = fmaf(pv, bf16_lo(x), o[mt][n][2 * h]);
                o[mt][n][2 * h + 1] = fmaf(pv, bf16_hi(x), o[mt][n][2 * h + 1]);
              }
            }
          }
        }
    }
    __syncwarp();  // the tile has been read before the next copies overwrite it
    if (++s == C::STAGES) {
      s = 0;
      phase ^= 1;
    }
  }

  // (a wait gave up: the copies that are still on their way land before the rings are written or left)
  for (; TMA && flying > 0; --flying) {
    mbar_wait(&full[s], phase, p.st, 97, nullptr);
    if (++s == C::STAGES) {
      s = 0;
      phase ^= 1;
    }
  }

  // ---- join the item's warps (their rings are free now), write this split's part of every row
  float* mo = reinterpret_cast<float*>(W == 1 ? ring : smem);  // [part][M][HDP]
  float* mml = mo + W * M * HDP;                               // [part][M][2]
  const auto join = [] {
    if (W == 1)
      __syncwarp();
    else
      __syncthreads();
  };
  join();
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = 16 * mt + 8 * h + (lane >> 2);
      float l = tiles > 0 ? l_run[mt][h] : 0.f;
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      if ((lane & 3) == 0)
        *reinterpret_cast<float2*>(mml + (part_w * M + r) * 2) = make_float2(tiles > 0 ? m_run[mt][h] : -INFINITY, l);
      if (tiles > 0 && r0 + r < r_end) {
#pragma unroll
        for (int n = 0; n < HDP / 8; ++n)
          *reinterpret_cast<float2*>(mo + (part_w * M + r) * HDP + ((n * 8 + (lane & 3) * 2) ^ ((r & 3) * 8))) =
              make_float2(o[mt][n][2 * h], o[mt][n][2 * h + 1]);
      }
    }
  join();
  const int slots = SPARE ? slots_of(p) : p.P + p.T;
  for (int r = part_w; r < M && r0 + r < r_end; r += W) {
    float m = -INFINITY, f[W], l = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) m = max_nan(m, mml[(w * M + r) * 2]);
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      f[w] = ex2_fast(mml[(w * M + r) * 2] - ref);
      l += f[w] * mml[(w * M + r) * 2 + 1];
    }
    const int gr = r0 + r, bt = gr / p.G;
    const long part = ((long)bt * p.H + hk * p.G + gr - bt * p.G) * slots + slot;
    for (int d = lane * 2; d < p.HD; d += 64) {
      float2 acc = make_float2(0.f, 0.f);
#pragma unroll
      for (int w = 0; w < W; ++w)
        if (f[w] != 0.f) {  // (a warp without keys holds nothing)
          const float2 x = *reinterpret_cast<const float2*>(mo + (w * M + r) * HDP + (d ^ ((r & 3) * 8)));
          acc.x += f[w] * x.x;
          acc.y += f[w] * x.y;
        }
      *reinterpret_cast<float2*>(p.part_o + part * p.HD + d) = acc;
    }
    if (lane == 0) *reinterpret_cast<float2*>(p.part_ml + part * 2) = make_float2(m, l);
  }
  wait_for_previous();
}

// The pool as [page][head][64-column half][slot][64]: a box is `rows` slots of `halves` halves.
CUtensorMap pool_map(const Params& p, const bf16* pool, int rows, int halves) {
  const uint64_t row = (uint64_t)p.Hkv * p.HD * 2;
  const uint64_t ext[5] = {64, (uint64_t)p.bs, (uint64_t)p.HD / 64, (uint64_t)p.Hkv, (uint64_t)p.num_pages};
  const uint64_t str[4] = {row, 128, (uint64_t)p.HD * 2, row * p.bs};
  const uint32_t bx[5] = {64, (uint32_t)rows, (uint32_t)halves, 1, 1};
  return make_tmap_bf16(pool, 5, ext, str, bx, CU_TENSOR_MAP_SWIZZLE_128B);
}

// W warps to an output row, which take every W-th part.
template <int W, bool SPARE>
__global__ void __launch_bounds__(128) combine_kernel(const Params p) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = blockIdx.x * (4 / W) + warp / W;
  if (row >= p.B * p.Q * p.H) return;
  __shared__ float4 acc_s[4][32];
  __shared__ float den_s[4];
  const int bt = row / p.H, h = row - bt * p.H, b = bt / p.Q, t = bt - b * p.Q;
  const int slots = SPARE ? slots_of(p) : p.P + p.T;
  const float* ml = p.part_ml + (long)row * slots * 2;
  const float* po = p.part_o + (long)row * slots * p.HD;
  const Seq s = seq_of(p, b);
  wait_for_previous();
  // a lane reads the maximum of one slot
  const float mine = lane < slots ? ml[2 * lane] : -INFINITY;
  // the slots that hold parts of this row: the prefix's, if the sequence takes part in it, and its tail's
  int np = 0, nt = 0, tail_at = p.P;
  if (t < s.ql) {
    if (s.start == p.L) {
      np = p.P;
      if (p.tc_share > 0) {
        // the CTAs whose blocks meet the row tile's
        const int hk = h / p.G, r = bt * p.G + h - hk * p.G;
        const int first = (hk * p.tc_tiles + r / p.tc_rows) * p.tc_blocks;
        np = ((first + p.tc_blocks - 1) / p.tc_share - first / p.tc_share + 1) * p.tc_streams;
      }
    }
    int parts = p.T;
    if (SPARE && ends_inside(p, s)) {
      parts += spare_parts(p, count_inside(p, lane));
      tail_at = spare_at(p);
    }
    const int n = tail_keys(s), share = tail_share(s, parts);
    if (n > 0) nt = (n + share - 1) / share;
  }
  const auto used = [&](int i) { return i < np || (i >= tail_at && i < tail_at + nt); };
  float m = used(lane) ? mine : -INFINITY;
  for (int i = lane + 32; i < slots; i += 32)
    if (used(i)) m = fmaxf(m, ml[2 * i]);
  m = warp_max(m);
  const float ref = m == -INFINITY ? 0.f : m;
  const auto slot_of = [&](int j) { return j < np ? j : tail_at + j - np; };
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float den = 0.f;
  const bool on = 4 * lane < p.HD;
#pragma unroll 4
  for (int j = warp % W; j < np + nt; j += W) {
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
  if (W > 1) {
    acc_s[warp][lane] = acc;
    if (lane == 0) den_s[warp] = den;
    __syncthreads();
    if (warp != 0) return;
#pragma unroll
    for (int w = 1; w < W; ++w) {
      const float4 o = acc_s[w][lane];
      acc.x += o.x;
      acc.y += o.y;
      acc.z += o.z;
      acc.w += o.w;
      den += den_s[w];
    }
  }
  if (!on) return;
  uint2 out = make_uint2(0u, 0u);
  if (den != 0.f) {
    const float inv = 1.f / den;
    out = make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
  }
  *reinterpret_cast<uint2*>(p.out + (long)row * p.HD + 4 * lane) = out;
}

}  // namespace prefix

// q [B, Q, H, HD] or [B, H, HD] (one query a sequence) bf16 -> the same shape, and the launches made. Pools
// [num_pages, block_size, Hkv, HD] bf16; tables int32 [B, max_pages] (each sequence's whole chain), lens int32 [B],
// pages int32 [>= ceil(L / block_size)] (the prefix's chain), qlens int32 [B] or none.
// tcgen05 takes the prefix from kTcKeys keys on if more than kTcRows rows share a cached head, and from kTcLong
// keys on always (8 cached heads of 128, tails of 128, mma.sync -> tcgen05: 24 rows, 1024 keys 15.8 -> 14.8 us,
// 8192 keys 37 -> 25 us; 16 rows, 8192 keys 21 -> 23 us, 65536 keys 66 -> 60 us; 16 rows of heads of 64, 1024 keys
// 10.8 -> 13.0 us).
constexpr int64_t kTcRows = 16, kTcKeys = 512, kTcLong = 32768;
// Keys of an item, at least (16 rows, 1024 keys of the prefix: 256 instead of 128 takes 12.8 us, not 10.8), and
// parts of a row's prefix, at most, where they fill the device (8192 keys in 32 parts instead of 64: 22 -> 15 us).
constexpr int64_t kMinKeys = 128, kParts = 32;
// Keys that a warp of a sequence that ends inside the prefix walks, at most, before spare items take parts of them
// (2048 take 0.15 ms). With one such sequence of 99990 tokens of 16 a call takes 181 us, without spare items 1484; 3 of
// 256 inside 32768 tokens 311 us, not 705; in tails of a warp 155, not 1616. Where no sequence ends inside, the kernels
// with spare items cost 0.3 to 1 % behind long prefixes, but 4 to 7 % where items are short or have 32 rows (1024
// sequences behind 2048 tokens 94 -> 101 us, 64 x 5 x 8 heads behind 4096 118 -> 123): those go without.
constexpr int64_t kWalk = 2048;
// Up to here a warp joins a row's parts, above four do (2048 rows of 20 parts: 9 us with four).
constexpr int kFewParts = 8;

std::tuple<torch::Tensor, int64_t> paged_prefix_attention(torch::Tensor q, torch::Tensor k_pool, torch::Tensor v_pool,
                                                          torch::Tensor tables, torch::Tensor lens,
                                                          torch::Tensor pages, int64_t L,
                                                          c10::optional<torch::Tensor> qlens, double scale) {
  CHECK_CUDA_TENSOR(q);
  CHECK_DTYPE(q, at::kBFloat16);
  CHECK_DTYPE(k_pool, at::kBFloat16);
  CHECK_DTYPE(v_pool, at::kBFloat16);
  TORCH_CHECK(q.dim() == 3 || q.dim() == 4, "q must be [B, H, HD] or [B, Q, H, HD]");
  const auto shape = q.sizes().vec();
  if (q.dim() == 3) q = q.unsqueeze(1);
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
  auto ints = [&](torch::Tensor& t, const char* what) {
    TORCH_CHECK(t.scalar_type() == at::kInt && t.device() == q.device(), what, ": int32 on q's device");
    if (!t.is_contiguous()) t = t.contiguous();
  };
  ints(tables, "block tables");
  ints(lens, "sequence lengths");
  ints(pages, "prefix pages");
  if (has_ql) ints(*qlens, "query lengths");
  TORCH_CHECK(k_pool.device() == q.device() && v_pool.device() == q.device(), "pools and q on different devices");
  TORCH_CHECK(tables.dim() == 2 && tables.size(0) == B && lens.numel() == B && (!has_ql || qlens->numel() == B),
              "one table row, length and query length per sequence");
  const int64_t max_pages = tables.size(1);
  TORCH_CHECK(num_pages > 0, "the pool has no pages");
  TORCH_CHECK(std::isfinite(scale) && scale * 1.4426950408889634 >= 1e-30, "scale must be positive and finite");
  TORCH_CHECK(L >= 0 && L <= pages.numel() * bs && L <= max_pages * bs, "a prefix of ", num(L),
              " tokens is longer than its pages or than a chain");
  TORCH_CHECK(max_pages * bs < (1LL << 30) && B * Q * H < (1LL << 30), "paged attention: too large");
  c10::cuda::CUDAGuard guard(q.get_device());
  auto out = at::empty(shape, q.options());
  if (out.numel() == 0) return {out, 0};
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
  p.max_pages = (int)max_pages;
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
  const bool tc = (L >= kTcKeys && rows > kTcRows) || L >= kTcLong;
  const int mt = std::max(L > 0 && !tc ? rows : 0, seq_rows) > 16 ? 2 : 1;
  p.rt_p = L > 0 && !tc ? (int)((rows + 16 * mt - 1) / (16 * mt)) : 0;
  p.rt_t = (int)((seq_rows + 16 * mt - 1) / (16 * mt));
  p.pages_max = (int)((L + bs - 1) / bs);
  p.bs_shift = 31;
  while ((1LL << (p.bs_shift - 31)) < bs) ++p.bs_shift;
  p.bs_mul = (uint32_t)(((1ULL << p.bs_shift) + bs - 1) / bs);
  // tails: two rounds of CTAs, of at least kMinKeys keys each
  const int64_t ctas = 2LL * sms * (HD <= 64 ? prefix::Cfg<64>::ctas(mt) : prefix::Cfg<128>::ctas(mt));
  const int64_t span = max_pages * bs - L;
  p.P = 0;
  if (p.rt_p > 0) {
    const int64_t n = std::min((L + kMinKeys - 1) / kMinKeys, std::max<int64_t>(kParts, 2 * sms / (Hkv * p.rt_p)));
    p.per_p = (int)(((L + n - 1) / n + prefix::kTile - 1) / prefix::kTile * prefix::kTile);
    p.P = (int)((L + p.per_p - 1) / p.per_p);
  }
  p.T = (int)std::max<int64_t>(1, std::min(ctas / (Hkv * B * p.rt_t), (span + kMinKeys - 1) / kMinKeys));
  // boxes of a power of two that divides the page size, at least the 8 rows of the swizzle
  const int run = p.bs & -p.bs;
  p.box = (HD == 64 || HD == 128) && run >= 8 ? std::min(run, prefix::kTile) : 0;
  if (tc) prefix::plan_prefix_tc(p, sms);
  const int64_t items = Hkv * ((int64_t)p.rt_p * p.P + B * p.rt_t * p.T);
  TORCH_CHECK(items < (1LL << 30), "paged attention: too large");
  p.items = (int)items;
  // many short tails (no longer than an item's smallest share, more than two rounds of CTAs): a warp each
  const bool solo = mt == 1 && p.rt_p == 0 && span <= kMinKeys && items > ctas;
  // a spare item for each SM where the T parts of a sequence that ends inside the prefix could have more than kWalk
  // keys a warp
  if (L > kWalk * p.T * (solo ? 1 : prefix::kWarps))
    p.spare = (int)(sms * (solo ? prefix::kWarps : 1) / Hkv * Hkv);
  const int slots = prefix::slots_of(p);
  auto parts = at::empty({B * Q * H * slots * (HD + 2)}, q.options().dtype(at::kFloat));
  p.part_o = parts.data_ptr<float>();
  p.part_ml = p.part_o + B * Q * H * slots * HD;
  if (tc) {
    prefix::launch_prefix_tc(p, cur_stream());
  }
  auto st = cur_stream();
  CUtensorMap map_k{}, map_v{};
  if (p.box > 0) {
    map_k = prefix::pool_map(p, p.k, p.box, p.box == prefix::kTile ? (int)HD / 64 : 1);
    map_v = prefix::pool_map(p, p.v, p.box, p.box == prefix::kTile ? (int)HD / 64 : 1);
  }
#define SCIRS_ITEMS(HDP_, MT_, TMA_, W_, SPARE_)                                                                     \
  {                                                                                                                  \
    auto kern = prefix::item_kernel<HDP_, MT_, TMA_, W_, SPARE_>;                                                    \
    constexpr int smem = prefix::Cfg<HDP_>::smem(MT_), each = prefix::kWarps / W_;                                   \
    set_max_smem((const void*)kern, smem);                                                                           \
    prefix::launch(kern, (unsigned)((items + p.spare + each - 1) / each), prefix::kThreads, smem, st, tc, map_k,     \
                   map_v, p);                                                                                        \
  }
#define SCIRS_ITEMS_MT(HDP_, TMA_, SPARE_)          \
  if (solo)                                         \
    SCIRS_ITEMS(HDP_, 1, TMA_, 1, SPARE_)           \
  else if (mt == 1)                                 \
    SCIRS_ITEMS(HDP_, 1, TMA_, 4, SPARE_)           \
  else                                              \
    SCIRS_ITEMS(HDP_, 2, TMA_, 4, SPARE_)
// four warps to a row where its parts are many, one where they are few
#define SCIRS_ATTEND(SPARE_)                                                                                   \
  if (p.box > 0) {                                                                                             \
    if (HD == 64) {                                                                                            \
      SCIRS_ITEMS_MT(64, true, SPARE_)                                                                         \
    } else {                                                                                                   \
      SCIRS_ITEMS_MT(128, true, SPARE_)                                                                        \
    }                                                                                                          \
  } else if (HD <= 64) {                                                                                       \
    SCIRS_ITEMS_MT(64, false, SPARE_)                                                                          \
  } else {                                                                                                     \
    SCIRS_ITEMS_MT(128, false, SPARE_)                                                                         \
  }                                                                                                            \
  if (p.P + p.T > kFewParts)                                                                                   \
    prefix::launch(prefix::combine_kernel<4, SPARE_>, (unsigned)(B * Q * H), 128, 0, st, true, p);             \
  else                                                                                                         \
    prefix::launch(prefix::combine_kernel<1, SPARE_>, (unsigned)((B * Q * H + 3) / 4), 128, 0, st, true, p);
  if (p.spare > 0) {
    SCIRS_ATTEND(true)
  } else {
    SCIRS_ATTEND(false)
  }
#undef SCIRS_ATTEND
#undef SCIRS_ITEMS_MT
#undef SCIRS_ITEMS
  return {out, tc ? 3 : 2};
}

}  // namespace scirs
