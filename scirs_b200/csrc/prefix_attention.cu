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
// An item belongs to one warp. It walks its keys 16 at a time, K and V rows of one head copied into a ring of
// its own: by TMA, a lane per box, where head_dim is 64 or 128 and the page size a multiple of 8, else by
// cp.async (16 bytes a lane, the same swizzle, free of bank conflicts for ldmatrix); S = Q K^T and
// O += P V by mma.sync m16n8k16 with the running max and sum in registers. No two warps ever wait for one
// another, and the copies run ahead over the end of an item into the next one, their page ids read a step
// before they are needed. Bound by memory as long as few rows share a key.
//
// Masked places (keys past a row's limit, slots past the length or before the item's first key) get P = 0
// by selection. Where a tile has any and one of its V values is infinite or NaN, P V is formed row by row
// without the masked keys, since 0 * NaN would reach the rows that do not see them.
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
  static constexpr int WARP = kStages * 2 * KV;      // a warp's ring
  static constexpr int SMEM = kWarps * WARP + 1024;
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

// What a warp works on: a run of tiles of one segment, that is of 16 MT rows of one cached head against the
// keys of the prefix or of a sequence's tail.
struct Item {
  bool is_prefix;
  int hk, r0, r_end, seg;  // seg: index into counts
  int b;                   // the sequence of a tail item
  int key0, k0, k1;        // tiles from key0; keys [k0, k1)
  int slot;
  bool ends;               // the segment's last tile is the item's
};

template <int HDP, int MT, bool TMA>
__global__ void __launch_bounds__(kThreads, Cfg<HDP>::ctas(MT)) item_kernel(const __grid_constant__ CUtensorMap map_k,
                                                                             const __grid_constant__ CUtensorMap map_v,
                                                                             const Params p) {
  using C = Cfg<HDP>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ Item queue_s[kWarps][4];  // items on their way
  __shared__ uint64_t full_s[kWarps][kStages];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint64_t* full = full_s[warp];
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(&full[s], 1);
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  __syncwarp();
  uint8_t* ring = smem + warp * C::WARP;
  const uint32_t ring_a = smem_u32(ring);
  Item* queue = queue_s[warp];
  const int chunks = p.HD / 8;  // 16-byte chunks that a row has; the rest of a padded row stays zero
  if (!TMA && chunks < HDP / 8) {
    for (int j = lane; j < C::WARP / 16; j += 32) reinterpret_cast<uint4*>(ring)[j] = make_uint4(0, 0, 0, 0);
    __syncwarp();
  }

  // ---- this warp's share of all tiles, laid end to end: the prefix's segments, then each sequence's
  const int nseg_p = p.Hkv * p.rt_p, per_b = p.Hkv * p.rt_t;  // segments of the prefix, of a sequence
  const int tiles_p = (p.L + kTile - 1) / kTile;
  auto tiles_of = [&](int b) { return b < p.B ? tail_tiles(seq_of(p, b)) : 0; };
  int total = 0, most = 0;
#pragma unroll 4
  for (int b = lane; b < p.B; b += 32) {
    const int n = tiles_of(b);
    total += n;
    most = max(most, n);
  }
  total = nseg_p * tiles_p + __reduce_add_sync(0xffffffffu, total) * per_b;
  most = __reduce_max_sync(0xffffffffu, most);
  const int nw = gridDim.x * kWarps;
  // (no tail may have more than T parts: sequences that end inside a long prefix can be longer than planned)
  const int share = max(max(p.share_min, (total + nw - 1) / nw), (most + p.T - 3) / (p.T - 2));
  // (few shares are spread over the SMs; of many, a CTA's warps take neighbours)
  const int w = share * nw - total >= share * (nw / 2) ? warp * gridDim.x + blockIdx.x : blockIdx.x * kWarps + warp;
  long u_at = (long)w * share;  // where the walk stands
  const int u_end = (int)min(u_at + share, (long)total);

  // ---- what is copied next; its page ids are read a step before they are used
  int lk = 0, lk1 = 0, lhk = 0, lmax = 0, q_tail = 0;
  const int* lpages = nullptr;
  bool more = u_at < u_end;
  // page and slot of key lk + lane * step for the lanes whose keys make up the tile (page -2: not read)
  int page = -2, at = 0;
  const int step = TMA ? p.box : 1;  // TMA: keys of a box; cp.async: single keys
  auto look_up = [&]() {
    const int key = lk + lane * step, pi = page_of(p, key);
    page = lane * step < kTile && key < lk1 && pi < lmax ? lpages[pi] : -2;
    at = key - pi * p.bs;
  };
  // the sequence that the walk is in, its first tile's place, and its tiles (from 32 read at a time)
  int cb = -1, c_at = nseg_p * tiles_p, c_tiles = 0, c_seg = 0;
  Seq cs{0, 0, 0};
  auto next_item = [&]() {
    if (u_at >= u_end) {
      more = false;
      return;
    }
    Item n;
    int seg_at, seg_tiles;  // the segment's first tile's place, and its tiles
    if (u_at < nseg_p * tiles_p) {
      const int g = (int)u_at / tiles_p;
      seg_at = g * tiles_p;
      seg_tiles = tiles_p;
      n.is_prefix = true;
      n.hk = g / p.rt_p;
      n.r0 = (g - n.hk * p.rt_p) * 16 * MT;
      n.r_end = p.B * p.Q * p.G;
      n.seg = g;
      n.b = 0;
      n.key0 = ((int)u_at - seg_at) * kTile;
      n.k0 = n.key0;
      lpages = p.pages;
      lmax = p.pages_max;
    } else {
      while ((int)u_at >= c_at + c_tiles * per_b) {
        c_at += c_tiles * per_b;
        if (cb + 1 >= p.B) {  // (lengths that change under the kernel: nothing is read past the batch)
          more = false;
          return;
        }
        // on to the sequence that holds u_at, 32 at a time
        const int b0 = cb + 1, mine = tiles_of(b0 + lane) * per_b;
        int inc = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int x = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += x;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, c_at + inc > (int)u_at);
        if (past == 0u) {
          cb = b0 + 31;
          c_at += __shfl_sync(0xffffffffu, inc, 31);
          c_tiles = 0;
        } else {
          const int j = __ffs(past) - 1;
          cb = b0 + j;
          c_at += __shfl_sync(0xffffffffu, inc - mine, j);
          cs = seq_of(p, cb);
          c_tiles = tail_tiles(cs);
          if (lane == 0 && p.lens[cb] > cs.len && cs.ql > 0) report_status(p.st, kStBounds, 95, (unsigned)p.lens[cb]);
        }
      }
      const int g = ((int)u_at - c_at) / c_tiles;
      seg_at = c_at + g * c_tiles;
      seg_tiles = c_tiles;
      n.is_prefix = false;
      n.hk = g / p.rt_t;
      n.b = cb;
      n.r0 = cb * p.Q * p.G + (g - n.hk * p.rt_t) * 16 * MT;
      n.r_end = (cb + 1) * p.Q * p.G;
      n.seg = nseg_p + cb * per_b + g;
      n.key0 = first_key(cs) + ((int)u_at - seg_at) * kTile;
      n.k0 = max(n.key0, cs.start);
      lpages = p.tables + (long)cb * p.table_stride;
      lmax = p.max_pages;
    }
    const int n_tiles = min(seg_at + seg_tiles, u_end) - (int)u_at;
    n.k1 = min(n.key0 + n_tiles * kTile, n.is_prefix ? p.L : cs.len);
    n.slot = w - seg_at / share + (n.is_prefix ? 0 : p.P);
    n.ends = (int)u_at + n_tiles == seg_at + seg_tiles;
    u_at += n_tiles;
    lk = n.key0;
    lk1 = n.k1;
    lhk = n.hk;
    if (lane == 0) queue[q_tail & 3] = n;
    ++q_tail;
  };
  // Copy the tile into a stage; returns which of its keys lie on pages of the pool (bit = key).
  auto copy = [&](int stage) -> uint32_t {
    uint32_t valid;
    const bool good = page != -2 && input_in_range(page, p.num_pages, p.st, 96);
    const uint32_t ok = __ballot_sync(0xffffffffu, good);
    uint8_t* dst = ring + stage * 2 * C::KV;
    if (TMA) {
      // a lane per box: K or V of the whole tile, or of 8 keys and one half of the columns; a box that is
      // not read is taken off the bytes to wait for
      if (lane == 0) mbar_arrive_expect_tx(&full[stage], __popc(ok) * 2 * HDP * 2 * p.box);
      __syncwarp();
      if (p.box == kTile) {
        const int pg = __shfl_sync(0xffffffffu, page, 0), slot = __shfl_sync(0xffffffffu, at, 0);
        if (lane < 2 && ok != 0u)
          tma_load_5d(dst + lane * C::KV, lane ? &map_v : &map_k, &full[stage], 0, slot, 0, lhk, pg);
        valid = ok != 0u ? 0xffffu : 0u;
      } else {
        const int i = lane & 1, h = lane >> 2;
        const int pg = __shfl_sync(0xffffffffu, page, i), slot = __shfl_sync(0xffffffffu, at, i);
        if (h < HDP / 64 && ((ok >> i) & 1u))
          tma_load_5d(dst + (lane >> 1 & 1) * C::KV + h * C::HALF + i * 1024, (lane & 2) ? &map_v : &map_k,
                      &full[stage], 0, slot, h, lhk, pg);
        valid = (ok & 1u ? 0xffu : 0u) | (ok & 2u ? 0xff00u : 0u);
      }
    } else {
      const long off = good ? (((long)page * p.bs + at) * p.Hkv + lhk) * p.HD : -1;
      constexpr int RPI = 32 / (HDP / 8);  // rows per instruction
      const int c = lane % (HDP / 8);
#pragma unroll
      for (int j = 0; j < kTile / RPI; ++j) {
        const int r = j * RPI + lane / (HDP / 8);
        const long ro = __shfl_sync(0xffffffffu, off, r);
        if (c < chunks) {
          const uint32_t d = smem_u32(dst) + tile_at<HDP>(r, c);
          const long e = (ro < 0 ? 0 : ro) + c * 8;
          cp_async16(d, p.k + e, ro >= 0);
          cp_async16(d + C::KV, p.v + e, ro >= 0);
        }
      }
      cp_commit();
      valid = ok;
    }
    return valid;
  };

  // ---- the item that is worked on
  Item it;
  int q_head = 0, key0 = 0, lo = 0;
  int limit[MT][2];  // keys that rows r0 + 16 mt + lane / 4 (+ 8) see
  uint32_t qf[MT][HDP / 16][4];
  float o[MT][HDP / 8][4];
  float m_run[MT][2], l_run[MT][2];
  // The queue's next item and its queries.
  auto begin = [&]() {
    __syncwarp();
    it = queue[q_head & 3];
    ++q_head;
    key0 = it.key0;
    Seq s{0, 0, 0};
    if (!it.is_prefix) s = seq_of(p, it.b);
    lo = 0x7fffffff;  // the smallest limit of a row that sees any of these keys
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = it.r0 + 16 * mt + 8 * h + (lane >> 2);
        const int bt = r / p.G, b = bt / p.Q, t = bt - b * p.Q;
        const bf16* src = p.q + b * p.q_sb + t * p.q_st + (long)(it.hk * p.G + r - bt * p.G) * p.q_sh;
#pragma unroll
        for (int kk = 0; kk < HDP / 16; ++kk)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int d = kk * 16 + e * 8 + (lane & 3) * 2;
            qf[mt][kk][e * 2 + h] = r < it.r_end && d < p.HD ? *reinterpret_cast<const uint32_t*>(src + d) : 0u;
          }
        int lim = 0;
        if (r < it.r_end) {
          if (it.is_prefix) s = seq_of(p, b);
          if (t < s.ql && (!it.is_prefix || s.start == p.L)) lim = max(s.len - s.ql + t + 1, 0);
        }
        limit[mt][h] = lim;
        if (lim > it.k0) lo = min(lo, lim);
        m_run[mt][h] = -INFINITY;
        l_run[mt][h] = 0.f;
#pragma unroll
        for (int d = 0; d < HDP / 8; ++d) o[mt][d][2 * h] = o[mt][d][2 * h + 1] = 0.f;
      }
    lo = __reduce_min_sync(0xffffffffu, lo);
  };

  // Every piece of code stands in the loop once: instructions that are fetched for the first time cost a
  // short call more than anything else here.
  bool primed = false, fresh = true;
  int flying = 0, s = 0, sw = 0;  // tiles on their way; stages to read and to write
  uint32_t phase = 0;
  uint64_t valid = 0;  // 16 bits a tile on its way
  while (true) {
    while (more && flying < kStages) {
      if (primed) {
        valid |= (uint64_t)copy(sw) << (16 * flying);
        ++flying;
        sw = sw + 1 == kStages ? 0 : sw + 1;
        lk += kTile;
      }
      primed = true;
      if (lk >= lk1) next_item();
      if (more) look_up();
    }
    if (flying == 0) break;
    if (fresh) begin();
    fresh = false;
    if (TMA) {
      if (!mbar_wait(&full[s], phase, p.st, 97, nullptr)) return;
    } else {
      if (flying > 2)
        cp_wait<2>();
      else if (flying == 2)
        cp_wait<1>();
      else
        cp_wait<0>();
    }
    __syncwarp();
    // the tile's keys that belong to the item and were read
    uint32_t vm = (uint32_t)valid & 0xffffu;
    valid >>= 16;
    --flying;
    if (key0 < it.k0) vm &= 0xffffu << (it.k0 - key0);
    if (key0 + kTile > it.k1) vm &= 0xffffu >> (key0 + kTile - it.k1);
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
        } else if (limit[mt][h] <= it.k0) {
          x[0] = x[1] = x[2] = x[3] = -INFINITY;  // a row that sees nothing here
        }
        float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        mx *= p.scale_log2;
        // the reference maximum is raised only when it grew by more than 2^8: P stays below 2^8
        alpha[mt][h] = 1.f;
        if (mx > m_run[mt][h] + kRaise) {
          alpha[mt][h] = ex2_fast(m_run[mt][h] - mx);  // 2^-inf = 0 before the first key
          m_run[mt][h] = mx;
          rescale = true;
        }
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
    __syncwarp();  // the tile has been read before the next step's copies overwrite it
    key0 += kTile;
    if (++s == kStages) {
      s = 0;
      phase ^= 1;
    }
    if (key0 < it.k1) continue;

    // ---- this split's part of every row
    const int slots = p.P + p.T;
    if (it.ends && lane == 0) p.counts[it.seg] = it.slot - (it.is_prefix ? 0 : p.P) + 1;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = it.r0 + 16 * mt + 8 * h + (lane >> 2);
        float l = l_run[mt][h];
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (r >= it.r_end) continue;
        const int bt = r / p.G;
        const long part = ((long)bt * p.H + it.hk * p.G + r - bt * p.G) * slots + it.slot;
        if ((lane & 3) == 0) *reinterpret_cast<float2*>(p.part_ml + part * 2) = make_float2(m_run[mt][h], l);
#pragma unroll
        for (int n = 0; n < HDP / 8; ++n)
          if (n < chunks)
            *reinterpret_cast<float2*>(p.part_o + part * p.HD + n * 8 + (lane & 3) * 2) =
                make_float2(o[mt][n][2 * h], o[mt][n][2 * h + 1]);
      }
    fresh = true;
  }
}

// The pool as [page][head][64-column half][slot][64]: a box is `rows` slots of `halves` halves.
CUtensorMap pool_map(const Params& p, const bf16* pool, int rows, int halves) {
  const uint64_t row = (uint64_t)p.Hkv * p.HD * 2;
  const uint64_t ext[5] = {64, (uint64_t)p.bs, (uint64_t)p.HD / 64, (uint64_t)p.Hkv, (uint64_t)p.num_pages};
  const uint64_t str[4] = {row, 128, (uint64_t)p.HD * 2, row * p.bs};
  const uint32_t bx[5] = {64, (uint32_t)rows, (uint32_t)halves, 1, 1};
  return make_tmap_bf16(pool, 5, ext, str, bx, CU_TENSOR_MAP_SWIZZLE_128B);
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
  // the slots that hold parts of this row: the prefix's, if the sequence takes part in it, and its tail's
  const int h = (int)(row % p.H), hk = h / p.G, r = (b * p.Q + t) * p.G + h % p.G;
  int np = 0, nt = 0;
  if (t < s.ql && s.start == p.L && p.L > 0) {
    if (p.tc_share > 0) {
      // the CTAs whose blocks meet the row tile's
      const int first = (hk * p.tc_tiles + r / p.tc_rows) * p.tc_blocks;
      np = ((first + p.tc_blocks - 1) / p.tc_share - first / p.tc_share + 1) * p.tc_streams;
    } else {
      np = p.counts[hk * p.rt_p + r / p.item_rows];
    }
  }
  if (t < s.ql && s.len > s.start)
    nt = p.counts[p.Hkv * p.rt_p + (b * p.Hkv + hk) * p.rt_t + (r - b * p.Q * p.G) / p.item_rows];
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
constexpr int64_t kMinTiles = 4;

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
  TORCH_CHECK(num_pages > 0, "the pool has no pages");
  TORCH_CHECK(std::isfinite(scale) && scale * 1.4426950408889634 >= 1e-30, "scale must be positive and finite");
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
  p.item_rows = 16 * mt;
  p.pages_max = (int)((L + bs - 1) / bs);
  p.bs_shift = 31;
  while ((1LL << (p.bs_shift - 31)) < bs) ++p.bs_shift;
  p.bs_mul = (uint32_t)(((1ULL << p.bs_shift) + bs - 1) / bs);
  // All tiles of 16 keys are cut into equal shares, one for each warp, by the lengths on the device. The
  // smallest share bounds the parts of a row: an eighth of what a warp gets if every chain is full, at least
  // kMinTiles.
  const int64_t ctas = (int64_t)sms * (HD <= 64 ? prefix::Cfg<64>::ctas(mt) : prefix::Cfg<128>::ctas(mt));
  const int64_t prefix_tiles = (L + prefix::kTile - 1) / prefix::kTile;
  const int64_t span_tiles = (max_pages * bs - L) / prefix::kTile + 2, chain_tiles = max_pages * bs / prefix::kTile + 2;
  const int64_t work = Hkv * (p.rt_p * prefix_tiles + B * p.rt_t * span_tiles);
  TORCH_CHECK(Hkv * (p.rt_p * prefix_tiles + B * p.rt_t * chain_tiles) < (1LL << 30), "paged attention: too large");
  p.share_min = (int)std::max<int64_t>(kMinTiles, work / (ctas * prefix::kWarps * 8));
  p.P = p.rt_p > 0 ? (int)((prefix_tiles - 1) / p.share_min + 2) : 0;
  p.T = (int)(span_tiles / p.share_min + 3);
  // boxes of a power of two that divides the page size, at least the 8 rows of the swizzle
  const int run = p.bs & -p.bs;
  p.box = (HD == 64 || HD == 128) && run >= 8 ? std::min(run, prefix::kTile) : 0;
  if (tc) prefix::plan_prefix_tc(p, sms);
  const int slots = p.P + p.T;
  auto part_o = at::empty({B * Q * H, slots, HD}, q.options().dtype(at::kFloat));
  auto part_ml = at::empty({B * Q * H, slots, 2}, q.options().dtype(at::kFloat));
  p.part_o = part_o.data_ptr<float>();
  p.part_ml = part_ml.data_ptr<float>();
  auto counts = at::empty({Hkv * (p.rt_p + B * p.rt_t)}, lens.options());
  p.counts = counts.data_ptr<int>();
  if (tc) {
    prefix::launch_prefix_tc(p, cur_stream());
    SCIRS_CHECK_LAUNCH();
  }
  auto st = cur_stream();
  CUtensorMap map_k{}, map_v{};
  if (p.box > 0) {
    map_k = prefix::pool_map(p, p.k, p.box, p.box == prefix::kTile ? (int)HD / 64 : 1);
    map_v = prefix::pool_map(p, p.v, p.box, p.box == prefix::kTile ? (int)HD / 64 : 1);
  }
#define SCIRS_ITEMS(HDP_, MT_, TMA_)                                                                                   \
  {                                                                                                                    \
    auto kern = prefix::item_kernel<HDP_, MT_, TMA_>;                                                                  \
    set_max_smem((const void*)kern, prefix::Cfg<HDP_>::SMEM);                                                          \
    kern<<<(unsigned)std::min<int64_t>(work, ctas), prefix::kThreads, prefix::Cfg<HDP_>::SMEM, st>>>(map_k, map_v, p); \
  }
#define SCIRS_ITEMS_MT(HDP_, TMA_) \
  if (mt == 1) SCIRS_ITEMS(HDP_, 1, TMA_) else SCIRS_ITEMS(HDP_, 2, TMA_)
  if (p.box > 0) {
    if (HD == 64) SCIRS_ITEMS_MT(64, true) else SCIRS_ITEMS_MT(128, true)
  } else {
    if (HD <= 64) SCIRS_ITEMS_MT(64, false) else SCIRS_ITEMS_MT(128, false)
  }
#undef SCIRS_ITEMS_MT
#undef SCIRS_ITEMS
  SCIRS_CHECK_LAUNCH();
  prefix::combine_kernel<<<(unsigned)(B * Q * H), 128, 0, st>>>(p);
  SCIRS_CHECK_LAUNCH();
  return out;
}

}  // namespace scirs
