// The shared prefix on tcgen05: all rows of the batch that share a cached head, in tiles, against the
// prefix's keys in blocks of 128.
//
// 512 threads, one CTA per SM:
//   warp 0        issues the MMAs (one thread) and owns TMEM
//   warps 4-7     producers: K and V blocks go through a ring of slots; unit 2 j is K of block j, 2 j + 1
//                 its V, and unit u belongs to warp 4 + u % 4. Where head_dim is 64 or 128 and the page size
//                 a multiple of 8, whole blocks come by TMA, one box per run of tc_box slots of a page (a
//                 lane each); the block that the prefix ends in, and everything else, by cp.async (16 bytes a
//                 lane, zeros past the end, written in the same 128-byte swizzle): the warp waits for its
//                 own copies, makes them visible to the asynchronous proxy and signals the slot full
//   warps 8-15    two softmax warpgroups, a thread per row: read the row's 128 scores from TMEM, raise the
//                 running maximum only when it grew by more than 2^8 (then O is rescaled in TMEM), write P
//                 back as packed bf16 over the scores, in two halves, so that P V of the first runs while the
//                 second is formed. (A block costs a tile about 2000 cycles here and 1450 in the MMAs, one after
//                 the other; the two tiles alternate. Moving 2 to 8 of 16 exponentials to the FMA pipe as
//                 polynomials made 256 sequences behind 32768 tokens slower, 134 -> 139 to 151 us: the warps are
//                 bound by issue and latency, not by the special-function unit.)
// S_t at TMEM columns [128 t, +128) (P_t aliases its first half), O_t at [256 + HDP t, + HDP). MMAs of one
// thread complete in order, so S_t of the next block may take the columns that P V_t reads, and S_t being
// full implies that P V_t before it is in O_t.
//
// Two schedules (template STREAMS):
//   1: a row tile is 256 rows, tile t its 128-row half; both use every key block (many rows: a K/V block is
//      read once for 256 rows, and one half's softmax runs during the other half's MMAs)
//   2: a row tile is 128 rows; tile t takes every other key block of the same rows (few rows: two
//      independent chains keep the loads and the tensor core busy), and writes a part of its own
//
// Measured: 1024 rows of each of 8 cached heads of 128 against 32768 keys (137 GFLOP) 134 us, 1.0 PFLOP/s, 0.62
// of the measured bf16 rate, the tensor pipe active 49 % of the time; 80 rows against 100003 keys (410 MB) 78 us,
// 5.2 TB/s; 256 rows against 8192 keys 22 us, of which about 10 are the start (lengths, queries, first block, code
// fetched for the first time) and the end of the four blocks that a CTA gets.
//
// Work is laid out evenly: the blocks of all row tiles end to end are cut into equal shares, one per CTA,
// so a CTA may finish one row tile and begin the next; its part of a row tile goes to the slot given by how
// many CTAs before it met that tile. Every wait is bounded (common.cuh).
//
// Reference parity: scirs2-neural/src/inference/paged_attention.rs:113-283.
#include "prefix_attention.cuh"

namespace scirs {
namespace prefix {

constexpr int kTcThreads = 512;
constexpr int kBlk = 128;  // keys of a block, rows of a tile
// warpgroups: MMA, producers, two of softmax; 512 x 128 registers at launch
constexpr int kRegsMma = 48, kRegsLoad = 56, kRegsSoftmax = 200;
static_assert(kRegsMma + kRegsLoad + 2 * kRegsSoftmax <= 4 * 128, "register split exceeds the launch");

template <int HDP>
struct Tc {
  static constexpr int TILE = kBlk * HDP * 2;  // a Q tile, or K or V of a block
  static constexpr int NS = HDP == 64 ? 8 : 4;  // ring slots
  static constexpr int OFF_Q = 0;               // two tiles
  static constexpr int OFF_RING = 2 * TILE;
  static constexpr int OFF_STAGE = OFF_RING + NS * TILE;  // 4 KB for each softmax warp's output
  static constexpr int OFF_BAR = OFF_STAGE + 8 * 4096;
  static constexpr int SMEM = OFF_BAR + 512 + 1024;
  static constexpr uint32_t IDESC_S = umma_idesc_bf16(kBlk, kBlk, 0, 0);
  static constexpr uint32_t IDESC_O = umma_idesc_bf16(kBlk, HDP, 0, 1);
};

// The MMAs are issued by a whole warp in uniform control flow with one lane predicated on: the compiler
// then keeps the descriptors in uniform registers instead of moving them there for every instruction.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc, uint32_t on) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(on)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc, uint32_t on) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(on)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t* bar, uint32_t on) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
      "r"(on)
      : "memory");
}

// A CTA's part of a row tile: blocks [j0, j0 + n).
struct TcItem {
  int hk, r0, j0, n, slot, tiles;
};

template <int STREAMS>
__device__ __forceinline__ TcItem tc_item(const Params& p, int u, int end) {
  TcItem i;
  const int g = u / p.tc_blocks;
  i.hk = g / p.tc_tiles;
  i.r0 = (g - i.hk * p.tc_tiles) * p.tc_rows;
  i.j0 = u - g * p.tc_blocks;
  i.n = min(p.tc_blocks - i.j0, end - u);
  i.slot = ((int)blockIdx.x - g * p.tc_blocks / p.tc_share) * STREAMS;
  i.tiles = STREAMS == 2 ? min(2, i.n) : (i.r0 + kBlk < p.B * p.Q * p.G ? 2 : 1);
  return i;
}

template <int HDP, int STREAMS>
__global__ void __launch_bounds__(kTcThreads, 1) prefix_tc_kernel(const __grid_constant__ CUtensorMap map_k,
                                                                     const __grid_constant__ CUtensorMap map_v,
                                                                     const Params p) {
  using C = Tc<HDP>;
  constexpr int NS = C::NS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);  // [NS]
  uint64_t* empty = full + NS;                                      // [NS]
  uint64_t* s_full = empty + NS;                                    // [2]
  uint64_t* p_full = s_full + 2;                                    // [2][2]: halves of P_t
  uint64_t* o_full = p_full + 4;                                    // [2]
  uint64_t* q_full = o_full + 2;
  uint64_t* q_empty = q_full + 1;
  uint64_t* drain = q_empty + 1;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  // a page of the prefix's chain was none of the pool's (at a fixed place: the softmax has no register for its address)
  __shared__ volatile int lost_flag;

  allow_next();
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int chunks = p.HD / 8;  // 16-byte chunks of a row; the rest of a padded row stays zero
  const int u_begin = blockIdx.x * p.tc_share;
  const int u_end = min(u_begin + p.tc_share, p.Hkv * p.tc_tiles * p.tc_blocks);

  if (threadIdx.x == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[2 * t], 4);
      mbar_init(&p_full[2 * t + 1], 4);
      mbar_init(&o_full[t], 1);
    }
    mbar_init(q_full, STREAMS == 2 ? 4 : 8);
    mbar_init(q_empty, 1);
    mbar_init(drain, 1);
    *abort_flag = 0;
    lost_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0) {
    tmem_alloc(tmem_holder, 512);
    tmem_relinquish();
  }
  if (chunks < HDP / 8) {
    for (int i = threadIdx.x; i < C::OFF_STAGE / 16; i += kTcThreads)
      reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;

  if (warp < 4) {
    setmaxnreg_dec<kRegsMma>();
    if (warp == 0) {
      const uint32_t on = elect_one_sync() ? 1u : 0u;
      // -------------------------------------------------------------- MMA
      const uint32_t q_addr = smem_u32(smem + C::OFF_Q), ring = smem_u32(smem + C::OFF_RING);
      int blk = 0;           // blocks of earlier items: unit 2 (blk + j) is K of block j
      int done[2] = {0, 0};  // phases of p_full
      bool ok = true;
      auto wait_unit = [&](int u) -> bool {
        if (!mbar_wait(&full[u % NS], (u / NS) & 1, p.st, 100, abort_flag)) return false;
        tc_fence_after();
        return true;
      };
      auto issue_s = [&](int t, int j) {
        const uint32_t ka = ring + ((2 * (blk + j)) % NS) * C::TILE;
        const uint32_t qa = q_addr + (STREAMS == 2 ? 0 : t * C::TILE);
#pragma unroll
        for (int kk = 0; kk < HDP / 16; ++kk) {
          const uint32_t off = (kk >> 2) * (kBlk * 128) + (kk & 3) * 32;
          mma_ss(tmem + t * kBlk, umma_desc_sw128(qa + off, 16, 1024), umma_desc_sw128(ka + off, 16, 1024),
                        C::IDESC_S, kk > 0 ? 1u : 0u, on);
        }
        mma_commit(&s_full[t], on);
      };
      auto issue_pv = [&](int t, int j, int half, bool first) {
        const uint32_t va = ring + ((2 * (blk + j) + 1) % NS) * C::TILE;
#pragma unroll
        for (int k2 = 0; k2 < kBlk / 32; ++k2) {
          const int kk = half * (kBlk / 32) + k2;
          // A = P_t from TMEM (16 keys = 8 packed columns a step), B = V [keys][HDP] MN-major
          mma_ts(tmem + 2 * kBlk + t * HDP, tmem + t * kBlk + kk * 8,
                 umma_desc_sw128(va + kk * 2048, kBlk * 128, 1024), C::IDESC_O, !first || kk > 0 ? 1u : 0u, on);
        }
      };
      // P_t V in two halves: the first runs while the softmax warps work on the second
      auto pv = [&](int t, int j, bool first, bool wait_v) -> bool {
        if (!mbar_wait(&p_full[2 * t], done[t] & 1, p.st, 102, abort_flag)) return false;
        if (wait_v && !wait_unit(2 * (blk + j) + 1)) return false;
        tc_fence_after();
        issue_pv(t, j, 0, first);
        if (!mbar_wait(&p_full[2 * t + 1], done[t] & 1, p.st, 102, abort_flag)) return false;
        ++done[t];
        tc_fence_after();
        issue_pv(t, j, 1, first);
        return true;
      };
      auto release = [&](int u) { mma_commit(&empty[u % NS], on); };
      int ii = 0;
      for (int u = u_begin; u < u_end && ok; ++ii) {
        const TcItem I = tc_item<STREAMS>(p, u, u_end);
        if (!mbar_wait(q_full, ii & 1, p.st, 101, abort_flag)) break;
        tc_fence_after();
        if (STREAMS == 1) {
          ok = wait_unit(2 * blk);
          if (!ok) break;
          for (int t = 0; t < I.tiles; ++t) issue_s(t, 0);
          release(2 * blk);
          if (I.n == 1) mma_commit(q_empty, on);
          for (int j = 0; j < I.n && ok; ++j) {
            for (int t = 0; t < I.tiles; ++t) {
              ok = pv(t, j, j == 0, t == 0);
              if (!ok) break;
              if (j + 1 < I.n) {
                if (t == 0) ok = wait_unit(2 * (blk + j + 1));
                if (!ok) break;
                issue_s(t, j + 1);
              } else {
                mma_commit(&o_full[t], on);
              }
            }
            if (!ok) break;
            release(2 * (blk + j) + 1);
            if (j + 1 < I.n) release(2 * (blk + j + 1));
            if (j == I.n - 2) mma_commit(q_empty, on);
          }
        } else {
          for (int t = 0; t < I.tiles && ok; ++t) {
            ok = wait_unit(2 * (blk + t));
            if (!ok) break;
            issue_s(t, t);
            release(2 * (blk + t));
          }
          if (ok && I.n <= 2) mma_commit(q_empty, on);
          for (int j = 0; j < I.n && ok; ++j) {
            const int t = j & 1;
            ok = pv(t, j, j < 2, true);
            if (!ok) break;
            release(2 * (blk + j) + 1);
            if (j + 2 < I.n) {
              ok = wait_unit(2 * (blk + j + 2));
              if (!ok) break;
              issue_s(t, j + 2);
              release(2 * (blk + j + 2));
              if (j + 3 == I.n) mma_commit(q_empty, on);
            } else {
              mma_commit(&o_full[t], on);
            }
          }
        }
        blk += I.n;
        u += I.n;
      }
      mma_commit(drain, on);
      mbar_wait(drain, 0, nullptr, 0, nullptr);
    }
  } else if (warp < 8) {
    setmaxnreg_dec<kRegsLoad>();
    // ---------------------------------------------------------------- producers
    const int w = warp - 4;
    const int box = p.tc_box;  // keys of a TMA box (0: cp.async only)
    constexpr int CPR = HDP / 8, RPI = 32 / CPR;  // chunks of a row, rows an instruction
    const int c = lane % CPR;
    const bf16* src = (w & 1) ? p.v : p.k;
    const uint32_t ring = smem_u32(smem + C::OFF_RING);
    const int max_pages = (p.L + p.bs - 1) / p.bs;
    int blk = 0, last = -1;  // (unit of the last copies by TMA)
    bool ok = true;
    for (int u = u_begin; u < u_end && ok;) {
      const TcItem I = tc_item<STREAMS>(p, u, u_end);
      for (int j = 0; j < I.n; ++j) {
        const int unit = 2 * (blk + j) + (w & 1);
        if ((unit & 3) != w) continue;
        const int key0 = (I.j0 + j) * kBlk;
        if (box > 0 && key0 + kBlk <= p.L) {
          const int key = key0 + lane * box;
          const int slot_in_page = key - page_of(p, key) * p.bs;
          const bool mine = lane * box < kBlk;
          const int page = mine ? p.pages[page_of(p, key)] : 0;
          const bool good = input_in_range(page, p.num_pages, p.st, 96);
          if (!mbar_wait(&empty[unit % NS], ((unit / NS) & 1) ^ 1, p.st, 103, abort_flag)) {
            ok = false;
            break;
          }
          uint64_t* bar = &full[unit % NS];
          uint8_t* dst = smem + C::OFF_RING + (unit % NS) * C::TILE + lane * box * 128;
          const uint32_t lost = __ballot_sync(0xffffffffu, !good);
          if (lost != 0u) {  // zeros in the box's place; the softmax leaves its keys out
            if (!good)
#pragma unroll 1
              for (int i = 0; i < box * 8; ++i)
#pragma unroll
                for (int h = 0; h < HDP / 64; ++h)
                  *reinterpret_cast<uint4*>(dst + h * (kBlk * 128) + i * 16) = make_uint4(0, 0, 0, 0);
            lost_flag = 1;
            fence_proxy_async_smem();
            __syncwarp();
          }
          if (lane == 0) mbar_arrive_expect_tx(bar, C::TILE - __popc(lost) * box * HDP * 2);
          __syncwarp();
          if (mine && good) {
#pragma unroll
            for (int h = 0; h < HDP / 64; ++h)
              tma_load_5d(dst + h * (kBlk * 128), (w & 1) ? &map_v : &map_k, bar, 0, slot_in_page, h, I.hk, page);
          }
          last = unit;
          continue;
        }
        // this lane looks four keys' rows up
        long row[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = key0 + i * 32 + lane;
          row[i] = key < p.L ? pool_row(p, p.pages, max_pages, key, I.hk) : -1;
          if (key < p.L && row[i] < 0) lost_flag = 1;
        }
        if (!mbar_wait(&empty[unit % NS], ((unit / NS) & 1) ^ 1, p.st, 103, abort_flag)) {
          ok = false;
          break;
        }
        const uint32_t slot = ring + (unit % NS) * C::TILE + (c >> 3) * (kBlk * 128);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll 8
          for (int k = 0; k < 32; k += RPI) {
            const int r = k + lane / CPR;
            const long e = __shfl_sync(0xffffffffu, row[i], r);
            if (c < chunks)
              cp_async16(slot + (i * 32 + r) * 128 + (((c ^ r) & 7) << 4), src + (e < 0 ? 0 : e) + c * 8, e >= 0);
          }
        cp_commit();
        cp_wait<0>();
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[unit % NS]);
      }
      blk += I.n;
      u += I.n;
    }
    // (a wait gave up: the copies that are still on their way land before the ring is left)
    if (!ok)
      for (int unit = last; unit >= 0 && unit > last - NS; unit -= 4)
        mbar_wait(&full[unit % NS], (unit / NS) & 1, p.st, 107, nullptr);
  } else {
    setmaxnreg_inc<kRegsSoftmax>();
    // ---------------------------------------------------------------- softmax
    const int t = (warp - 8) >> 2;
    const int r = (warp & 3) * 32 + lane;  // row of the tile = TMEM lane
    const uint32_t lane_off = uint32_t((warp & 3) * 32) << 16;
    const uint32_t s_base = tmem + lane_off + t * kBlk;
    const uint32_t o_base = tmem + lane_off + 2 * kBlk + t * HDP;
    const int slots = p.P + p.T;
    int cnt = 0, fin = 0, ii = 0;  // phases of s_full and o_full
    bool ok = true;
    for (int u = u_begin; u < u_end && ok; ++ii) {
      const TcItem I = tc_item<STREAMS>(p, u, u_end);
      const int gr = I.r0 + (STREAMS == 2 ? 0 : t * kBlk) + r;
      const bf16* q = prefix_query(p, gr, I.hk);
      if (STREAMS == 1 || t == 0) {
        // Q of this row (zeros for a row that takes no part)
        if (!mbar_wait(q_empty, (ii & 1) ^ 1, p.st, 104, abort_flag)) break;
        // the warp's 32 rows, a whole row (or two, four) per instruction; all loads before the first store
        constexpr int CPR = HDP / 8, RPI = 32 / CPR;
        const int c = lane % CPR;
        uint4 x[32 / RPI];
#pragma unroll
        for (int i = 0; i < 32 / RPI; ++i) {
          const uint64_t src = __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(q), i * RPI + lane / CPR);
          x[i] = src != 0 && c < chunks ? __ldg(reinterpret_cast<const uint4*>(src) + c) : make_uint4(0, 0, 0, 0);
        }
        uint8_t* dst = smem + C::OFF_Q + t * C::TILE + (warp & 3) * 32 * 128 + (c >> 3) * (kBlk * 128);
#pragma unroll
        for (int i = 0; i < 32 / RPI; ++i) {
          const int row = i * RPI + lane / CPR;
          *reinterpret_cast<uint4*>(dst + row * 128 + (((c ^ row) & 7) << 4)) = x[i];
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);
      }
      const int n = t >= I.tiles ? 0 : (STREAMS == 2 ? (I.n - t + 1) / 2 : I.n);
      float m_ref = -INFINITY, l = 0.f;
      for (int j = 0; j < n && ok; ++j, ++cnt) {
        if (!mbar_wait(&s_full[t], cnt & 1, p.st, 105, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        // the row's 128 scores; the maximum of one half is taken while the other comes
        float sv[kBlk];
        uint32_t* x = reinterpret_cast<uint32_t*>(sv);
        tmem_ld_32x32b_x32(s_base, x);
        tmem_ld_32x32b_x32(s_base + 32, x + 32);
        tc_wait_ld_regs(x);
        tc_wait_ld_regs(x + 32);
        tmem_ld_32x32b_x32(s_base + 64, x + 64);
        tmem_ld_32x32b_x32(s_base + 96, x + 96);
        // keys that are not there: behind the prefix's end, or of a page that is none of the pool's
        const int key0 = (I.j0 + (STREAMS == 2 ? 2 * j + t : j)) * kBlk;
        const bool partial = p.L - key0 < kBlk || lost_flag != 0;
        const auto leave_out = [&](float* v, int first) {
          const int key = first + lane;
          const uint32_t there =
              __ballot_sync(0xffffffffu, key < p.L && (unsigned)p.pages[page_of(p, key)] < (unsigned)p.num_pages);
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = (there >> e) & 1u ? v[e] : -INFINITY;
        };
        if (partial) {
          leave_out(sv, key0);
          leave_out(sv + 32, key0 + 32);
        }
        float m4[4] = {sv[0], sv[1], sv[2], sv[3]};
#pragma unroll
        for (int i = 0; i < 4; ++i) m4[i] = max_nan(m4[i], sv[4 + i]);
#pragma unroll
        for (int e = 8; e < kBlk / 2; e += 8) {
#pragma unroll
          for (int i = 0; i < 4; ++i) m4[i] = max_nan(m4[i], sv[e + i], sv[e + 4 + i]);
        }
        tc_wait_ld_regs(x + 64);
        tc_wait_ld_regs(x + 96);
        if (partial) {
          leave_out(sv + 64, key0 + 64);
          leave_out(sv + 96, key0 + 96);
        }
#pragma unroll
        for (int e = kBlk / 2; e < kBlk; e += 8) {
#pragma unroll
          for (int i = 0; i < 4; ++i) m4[i] = max_nan(m4[i], sv[e + i], sv[e + 4 + i]);
        }
        const float mx = max_nan(max_nan(m4[0], m4[1]), m4[2], m4[3]) * p.scale_log2;
        const bool raise = mx > m_ref + kRaise;
        float alpha = 1.f;
        if (raise) {
          alpha = ex2_fast(m_ref - mx);  // 0 before the first block
          m_ref = mx;
          l *= alpha;
        }
        if (j > 0 && __any_sync(0xffffffffu, raise)) {
#pragma unroll 1
          for (int c = 0; c < HDP; c += 32) {
            uint32_t ov[32];
            tmem_ld_32x32b_x32(o_base + c, ov);
            tc_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * alpha);
            tmem_st_32x32b_x16(o_base + c, ov);
            tmem_st_32x32b_x16(o_base + c + 16, ov + 16);
          }
          tc_wait_st();
        }
        // (a score that is NaN or infinite makes the row NaN)
        if (!(mx < INFINITY)) m_ref = NAN;
        const float ref = m_ref == -INFINITY ? 0.f : m_ref;
        const uint64_t sc2 = f2_pack(p.scale_log2, p.scale_log2), nref2 = f2_pack(-ref, -ref);
        uint64_t sum2[2] = {0ull, 0ull};
#pragma unroll
        for (int c = 0; c < kBlk; c += 32) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            float x0, x1;
            f2_unpack(f2_fma(f2_pack(sv[c + e], sv[c + e + 1]), sc2, nref2), x0, x1);
            x0 = ex2_fast(x0);
            x1 = ex2_fast(x1);
            sum2[(e >> 1) & 1] = f2_add(sum2[(e >> 1) & 1], f2_pack(x0, x1));
            pk[e >> 1] = pack_bf16x2(x0, x1);
          }
          tmem_st_32x32b_x16(s_base + (c >> 1), pk);
          if (c == kBlk / 2 - 32) {
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[2 * t]);
          }
        }
        float l0, l1;
        f2_unpack(f2_add(sum2[0], sum2[1]), l0, l1);
        l += l0 + l1;
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * t + 1]);
      }
      if (!ok) break;
      // this CTA's part of the row
      const int bt = gr / p.G;
      const long at = ((long)bt * p.H + I.hk * p.G + gr % p.G) * slots + I.slot + (STREAMS == 2 ? t : 0);
      const bool live = q != nullptr && n > 0;
      if (n > 0) {
        if (!mbar_wait(&o_full[t], fin & 1, p.st, 106, abort_flag)) break;
        ++fin;
        tc_fence_after();
        // 32 columns at a time through shared memory, so that a store writes four rows' whole lines
        uint8_t* stage = smem + C::OFF_STAGE + (warp - 8) * 4096;
        long to[8];  // the rows that this lane stores, four lanes' rows apart
#pragma unroll
        for (int i = 0; i < 8; ++i)
          to[i] = __shfl_sync(0xffffffffu, live ? at * p.HD : -1L, i * 4 + (lane >> 3));
#pragma unroll 1
        for (int c = 0; c < HDP; c += 32) {
          uint32_t ov[32];
          tmem_ld_32x32b_x32(o_base + c, ov);
          tc_wait_ld();
          __syncwarp();
#pragma unroll
          for (int e = 0; e < 8; ++e)
            *reinterpret_cast<uint4*>(stage + lane * 128 + ((e ^ lane) & 7) * 16) =
                make_uint4(ov[4 * e], ov[4 * e + 1], ov[4 * e + 2], ov[4 * e + 3]);
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int row = i * 4 + (lane >> 3), e = lane & 7;
            if (to[i] >= 0 && c + 4 * e < p.HD)
              *reinterpret_cast<uint4*>(p.part_o + to[i] + c + 4 * e) =
                  *reinterpret_cast<const uint4*>(stage + row * 128 + ((e ^ row) & 7) * 16);
          }
        }
        tc_fence_before();
      }
      if (q != nullptr) {
        p.part_ml[at * 2] = live ? m_ref : -INFINITY;
        p.part_ml[at * 2 + 1] = live ? l : 0.f;
      }
      u += I.n;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

void plan_prefix_tc(Params& p, int sms) {
  const int rows = p.B * p.Q * p.G;
  p.tc_streams = rows > kBlk ? 1 : 2;
  p.tc_rows = rows > kBlk ? 2 * kBlk : kBlk;
  p.tc_tiles = (rows + p.tc_rows - 1) / p.tc_rows;
  p.tc_blocks = (p.L + kBlk - 1) / kBlk;
  const int64_t units = (int64_t)p.Hkv * p.tc_tiles * p.tc_blocks;
  TORCH_CHECK(units < (1LL << 30), "paged attention: too large");
  p.tc_share = (int)std::max<int64_t>(2, (units + sms - 1) / sms);
  p.P = (int)((p.tc_blocks - 1) / p.tc_share + 2) * p.tc_streams;
  // boxes of the largest power of two that divides the page size: at least the 8 rows of the swizzle
  const int box = std::min(p.bs & -p.bs, kBlk);
  p.tc_box = (p.HD == 64 || p.HD == 128) && box >= 8 ? box : 0;
}

template <int HDP, int STREAMS>
static void launch_tc(const Params& p, cudaStream_t st) {
  auto kern = prefix_tc_kernel<HDP, STREAMS>;
  set_max_smem((const void*)kern, Tc<HDP>::SMEM);
  const int units = p.Hkv * p.tc_tiles * p.tc_blocks;
  CUtensorMap mk{}, mv{};
  if (p.tc_box > 0) {
    mk = pool_map(p, p.k, p.tc_box, 1);
    mv = pool_map(p, p.v, p.tc_box, 1);
  }
  launch(kern, (unsigned)((units + p.tc_share - 1) / p.tc_share), kTcThreads, Tc<HDP>::SMEM, st, false, mk, mv, p);
}

void launch_prefix_tc(const Params& p, cudaStream_t st) {
  if (p.HD <= 64) {
    p.tc_streams == 1 ? launch_tc<64, 1>(p, st) : launch_tc<64, 2>(p, st);
  } else {
    p.tc_streams == 1 ? launch_tc<128, 1>(p, st) : launch_tc<128, 2>(p, st);
  }
}

}  // namespace prefix
}  // namespace scirs
