// tree_attn.cu — attention of a tree of drafted tokens over the paged cache on
// the tcgen05 tensor cores (head dims 64 and 128).
//
// What it computes: see cie_tree_attn. The rows of a kv head (its G = Hq / Hkv
// query heads times the T nodes) are packed into groups of up to 128, so that
// every K and V byte is read once for all rows of a group:
//   S = Q K^T            M = 128 rows, N = 64 keys, fp32 in TMEM
//   P = 2^(S scale - m)  one thread per row (= TMEM lane), no shuffles
//   O += P V             A = P from TMEM as two halves of 16 bits, fp32 in TMEM
//   warp 0  loader of K, warp 2 of V, into rings of 64-key tiles: by TMA, one box of
//           8 or 16 tokens per page lookup, a lane each, or, for pages that such boxes
//           do not divide, by cp.async row by row
//   warp 1  issues the MMAs, S two tiles ahead of PV in two TMEM buffers
//   warps 4..7  softmax; a warp whose 32 rows are all padding does nothing
// The history needs no mask. Only tiles that reach past it (the last T keys) are
// masked, by a window per row out of the bitmap of the row's ancestors.
//
// Work split: lengths are only known on the device and differ widely in a batch,
// so each CTA takes an equal run of key tiles out of the list of all sequences laid
// end to end, whatever the sequences' borders. A sequence that lies in one run is
// written to the output; one cut by a border leaves partial results, at most two
// per CTA, that the merge kernel joins. (Equal partitions of the table's width, the
// split of paged_attn.cu, took 171 us against 131 us for trees of 12 over 64
// contexts of up to 8K at d = 64.) Batches of short sequences are dealt out whole
// and need no merge.
//
// Precision: scores, the softmax's maximum and sum, O and the merge are fp32. P goes
// to the tensor cores as hi + lo (2^-15 relative in bf16, 2^-22 in fp16), so that of
// the roundings to 16 bits only the output's own is left, and q's behind its rotation,
// where the model rounds it too. Rounded once to bf16 P costs the output as much again
// as its own rounding (2.3e-3 against 1.7e-3 off in the 2-norm).
//
// Bound: K/V bytes. A 64-key tile is 32 KB at d = 128, about 1400 cycles of one
// SM's share of HBM; its MMAs take 960 and its exponentials 512 cycles (MUFU). Two
// CTAs share an SM (256 TMEM columns, ~100 KB each), so one's hand-offs hide behind
// the other's. More than 128 rows take another pass over K/V, which comes from L2.
// Measured on B200 (2.2 GB of K/V, 32 contexts of 1K-32K, d = 128, bf16; on two GPUs):
// trees of 5 340-357 us (6.2-6.5 TB/s), of 16 371-394 us (5.6-6.0), of 32 422-449 us
// (5.0-5.3); with P rounded once 328-336, 346-356 and 375-390 us. For seconds on end,
// under the power cap, trees of 16 take 451 us, with P rounded once 396. Trees of 64 over
// 8 contexts of up to 16K (256 rows) 112-115 us, with P rounded once 98; so measured, a
// form with two 128-row tiles in one CTA that fills the SM by itself took 103.
//
// The choices below were measured with P rounded once to bf16.
#include <cuda.h>
#include <cuda_runtime.h>

#include <cfloat>
#include <cstdint>
#include <type_traits>

#include "cie_common.cuh"
#include "sm100_ptx.cuh"

namespace cie {

constexpr int kTcMaxTree = 256;  // nodes whose parents and bitmaps a CTA holds
constexpr int kTcKeys = 64;      // keys of a tile
constexpr int kTcBufs = 2;       // S buffers
constexpr int kTcThreads = 256;
// Tiles of the longest sequence up to which sequences stay whole: cutting 16 tiles
// of one sequence in four and joining them takes 14 us, leaving them whole 21 us.
constexpr int kTcWhole = 8;
// Shortest run of tiles worth a CTA of its own (with 6 instead of 4 one context of 1K
// took 20 against 17 us), and the tiles that one more piece costs a CTA (trees of 24
// over 4 contexts of up to 4K, 16 heads: 32, 29, 26 and 25 us with 4, 5, 8 and 12;
// trees of 12 over 64 contexts of up to 8K, d = 64: 133 us with 8, 136 with 12).
constexpr int kTcMinRun = 4;
constexpr int kTcOpen = 8;

template <int D>
struct TcCfg {
  static constexpr int KCH = D / 64;  // 128-byte swizzle slices along d
  static constexpr int Q_BYTES = 128 * D * 2;
  static constexpr int KV_BYTES = kTcKeys * D * 2;
  static constexpr int ST = D == 128 ? 2 : 4;  // stages of the K and of the V ring
  static constexpr int BAR_OFF = Q_BYTES + 2 * ST * KV_BYTES;
  static constexpr int NBARS = 4 * ST + 2 * kTcBufs + 6;
  // + slot, flag; the parents of two pieces; alignment
  static constexpr int PAR_OFF = BAR_OFF + NBARS * 8 + 8;
  static constexpr int SMEM = PAR_OFF + 2 * kTcMaxTree * 4 + 1024;
  static_assert(2 * (SMEM + 1024) <= 228 * 1024, "two CTAs must fit on an SM");
  static constexpr uint32_t TM_O = kTcBufs * kTcKeys;  // S(buf) at buf * 64, O behind them
  static constexpr uint32_t TM_COLS = 256;
};

// ------------------------------------------------------------------ work split
// CTA c works for head group c % groups (groups = kv heads * row groups) and takes
// part c / groups of that group's list: the key tiles of all sequences end to end,
// with kTcOpen idle places between two sequences that stand for what one more piece
// costs a CTA. The CTAs of one part thus read the same token rows, one head each,
// at about the same time: at d = 64 two heads share a 256-byte fetch, and lists that
// ran through the heads one after the other took twice as long.
__device__ __forceinline__ int tc_len(const PagedParams& p, int b) {
  return min(max(p.kv_lens[b], 0), p.max_blocks * p.block_size);
}

// The split as every warp of both kernels finds it for itself from the lengths.
struct TcPlan {
  int run;     // places of a CTA
  bool whole;  // sequences dealt out whole
};

__device__ __forceinline__ int tc_places(int tiles) { return tiles > 0 ? tiles + kTcOpen : 0; }

// len: the length of sequence `lane` (0 past the last), loaded early; mine: its places.
__device__ __forceinline__ TcPlan tc_plan(const PagedParams& p, int keys, int parts, int lane,
                                          int len, int& mine) {
  int most = (len + keys - 1) / keys;
  mine = tc_places(most);
  int sum = mine;
  for (int b = lane + 32; b < p.B; b += 32) {
    const int tiles = (tc_len(p, b) + keys - 1) / keys;
    sum += tc_places(tiles);
    most = max(most, tiles);
  }
  sum = __reduce_add_sync(0xffffffffu, sum);
  most = __reduce_max_sync(0xffffffffu, most);
  TcPlan plan;
  plan.run = max((sum - kTcOpen + parts - 1) / parts, p.min_run);
  plan.whole = most <= p.whole;
  return plan;
}

// The first sequence with keys among b, b + by, b + 2 by, .., B when there is none: 32 at a
// time, as a padded batch may have hundreds of idle sequences in a row. Not inlined: the
// roles' code, which all CTAs fetch, stays short (inlined, 1 us of 29 in a batch without any).
__device__ __noinline__ int tc_skip_idle(const int32_t* kv_lens, int B, int b, int by) {
  const int lane = threadIdx.x & 31;
  for (; b < B; b += 32 * by) {
    const int i = b + lane * by;
    const uint32_t hit = __ballot_sync(0xffffffffu, i < B && kv_lens[i] > 0);
    if (hit) return b + (__ffs(hit) - 1) * by;
  }
  return B;
}

// A CTA's walk over its pieces of sequences. All members are warp-uniform.
struct TcWalk {
  int b, kv_len, tiles;  // sequence, its length and key tiles
  int first, n;          // tiles [first, first + n) of it are this piece
  int at, lo, hi;        // the sequence's place in the list, the run's places
  bool whole, more;      // more: this piece exists

  __device__ __forceinline__ void seq(const PagedParams& p, int keys) {
    kv_len = tc_len(p, b);
    tiles = (kv_len + keys - 1) / keys;
  }
  // the first sequence with keys from b on, in steps of `by`
  __device__ __forceinline__ bool busy(const PagedParams& p, int keys, int by) {
    while (b < p.B) {
      seq(p, keys);
      if (tiles > 0) return true;
      b = tc_skip_idle(p.kv_lens, p.B, b + by, by);
    }
    return false;
  }
  // the first piece of the run in sequence b or behind it
  __device__ __forceinline__ void find(const PagedParams& p, int keys) {
    for (; at < hi && busy(p, keys, 1); ++b) {
      first = max(lo - at - kTcOpen, 0);
      n = min(hi - at - kTcOpen, tiles) - first;
      if (n > 0) return;
      at += tc_places(tiles);
    }
    more = false;
  }
  // whole sequences: the first with keys from b on, in steps of the parts
  __device__ __forceinline__ void deal(const PagedParams& p, int keys) {
    more = busy(p, keys, hi);
    n = tiles;
  }
  __device__ __forceinline__ void start(const PagedParams& p, int keys, int groups, int lane,
                                        int len) {
    const int parts = gridDim.x / groups, part = blockIdx.x / groups;
    int mine;
    const TcPlan plan = tc_plan(p, keys, parts, lane, len, mine);
    whole = plan.whole;
    more = true;
    first = 0;
    if (whole) {
      b = part;
      hi = parts;
      deal(p, keys);
      return;
    }
    lo = part * plan.run + kTcOpen;  // the list begins with a tile: every CTA opens one piece
    hi = lo + plan.run;
    at = 0;
    b = 0;
    for (; b < p.B; b += 32) {  // the sequence that holds place lo
      if (b > 0) mine = b + lane < p.B ? tc_places((tc_len(p, b + lane) + keys - 1) / keys) : 0;
      int inc = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int z = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += z;
      }
      const uint32_t over = __ballot_sync(0xffffffffu, at + inc > lo);
      if (over) {
        const int src = __ffs(over) - 1;
        at += __shfl_sync(0xffffffffu, inc - mine, src);
        b += src;
        break;
      }
      at += __shfl_sync(0xffffffffu, inc, 31);
    }
    find(p, keys);
  }
  __device__ __forceinline__ void next(const PagedParams& p, int keys) {
    if (whole) {
      b += hi;
      deal(p, keys);
    } else {
      at += tc_places(tiles);
      ++b;
      find(p, keys);
    }
  }
};

// One asynchronous 4-byte copy to shared memory.
__device__ __forceinline__ void cp_async_4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src)
               : "memory");
}
// 32 bytes in one store: a whole sector of a row that one thread owns.
__device__ __forceinline__ void store_f32x8(float* dst, const float (&x)[8]) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "f"(x[0]),
               "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7])
               : "memory");
}

// TMA = false: pages that no 8-token box divides; the loaders copy rows with cp.async.
template <int D, bool BF16, bool TMA>
__global__ void __launch_bounds__(kTcThreads, 2)
    tree_attn_kernel(const __grid_constant__ CUtensorMap tm_k,
                     const __grid_constant__ CUtensorMap tm_v, const PagedParams p) {
  using C = TcCfg<D>;
  constexpr int KEYS = kTcKeys, NBUF = kTcBufs;
  using elem_t = typename std::conditional<BF16, __nv_bfloat16, __half>::type;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int groups = p.Hkv * p.row_groups;
  const int R = p.G * p.M;

  const int len = lane < p.B ? tc_len(p, lane) : 0;  // on its way during the set-up

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                      // [KCH][128][128B]
  uint8_t* sK = sQ + C::Q_BYTES;           // [ST][KCH][KEYS][128B]
  uint8_t* sV = sK + C::ST * C::KV_BYTES;  // [ST][KCH][KEYS][128B]
  // g counts the CTA's tiles over all its pieces
  uint64_t* bar_k_full = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);
  uint64_t* bar_v_full = bar_k_full + C::ST;
  uint64_t* bar_k_free = bar_v_full + C::ST;  // S of the stage's tile complete
  uint64_t* bar_v_free = bar_k_free + C::ST;  // PV of the stage's tile complete
  uint64_t* bar_s_full = bar_v_free + C::ST;  // [NBUF] S(g % NBUF) complete
  uint64_t* bar_p_full = bar_s_full + NBUF;   // [NBUF] P(g % NBUF) written
  uint64_t* bar_q = bar_p_full + NBUF;        // a piece's Q is in sQ
  uint64_t* bar_go = bar_q + 1;               // the first Q is
  uint64_t* bar_pv = bar_go + 1;              // PV complete, but a piece's last
  uint64_t* bar_o = bar_pv + 1;               // a piece's last PV complete
  uint64_t* bar_seen = bar_o + 1;             // bad V rows: every warp has read V
  uint64_t* bar_drain = bar_seen + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::BAR_OFF + C::NBARS * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* s_par = reinterpret_cast<int*>(smem + C::PAR_OFF);  // [2][kTcMaxTree]

  const int y = blockIdx.x % groups;  // head group: kv head, row group
  const int kvh = y / p.row_groups, row0 = (y % p.row_groups) * p.rg_rows;
  const int active = p.rg_rows / 32;  // softmax warps

  // the merge kernel may be set up while this one runs; it waits for its end by itself
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 0) {
    for (int s = 0; s < 4 * C::ST + NBUF; ++s) mbar_init(bar_k_full + s, 1);
    for (int i = 0; i < NBUF; ++i) mbar_init(bar_p_full + i, active);
    mbar_init(bar_q, active);
    mbar_init(bar_go, active);
    mbar_init(bar_pv, 1);
    mbar_init(bar_o, 1);
    mbar_init(bar_seen, active);
    mbar_init(bar_drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::TM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  int copies = 0;  // loader warps: TMA tiles issued

  if (warp < 4) {
    TcWalk w;
    if (warp != 3) w.start(p, KEYS, groups, lane, len);
    if (warp == 0 || warp == 2) {
      // ---------------------------------------------- loaders
      const bool is_k = warp == 0;
      const CUtensorMap* map = is_k ? &tm_k : &tm_v;
      uint8_t* ring = is_k ? sK : sV;
      uint64_t* full = is_k ? bar_k_full : bar_v_full;
      uint64_t* free_ = is_k ? bar_k_free : bar_v_free;
      constexpr int stages = C::ST;
      const int32_t* tables = p.block_tables;
      // pool token of position t of the piece's sequence, `none` past its end or for a
      // refused page
      auto token = [&](int t, int none) -> int {
        if (t >= w.kv_len) return none;
        const int lb = p.bs_log2 >= 0 ? t >> p.bs_log2 : t / p.block_size;
        const int blk = tables[static_cast<int64_t>(w.b) * p.max_blocks + lb];
        if (blk < 0 || blk >= p.num_blocks) {
          raise_status(CIE_DEV_BAD_BLOCK_ID);
          return none;
        }
        return blk * p.block_size + (p.bs_log2 >= 0 ? t & (p.block_size - 1) : t % p.block_size);
      };
      // wait for tile g's stage; the first Q goes ahead of all but the first K tile:
      // behind the full rings of every SM its loads would wait for several microseconds
      auto wait_stage = [&](int g) -> bool {
        bool ok = true;
        if (g == (is_k ? 1 : 0))
          ok = __all_sync(0xffffffffu,
                          mbar_wait_bounded(bar_go, 0, abort_flag, &g_wait_limit_ns));
        if (ok && g >= stages)
          ok = __all_sync(0xffffffffu,
                          mbar_wait_bounded(free_ + g % stages, (g / stages - 1) & 1, abort_flag,
                                            &g_wait_limit_ns));
        return ok;
      };
      int g = 0, j = w.first;
      auto advance = [&]() {  // to the run's next tile
        if (++j == w.first + w.n) {
          w.next(p, KEYS);
          j = w.first;
        }
      };
      if constexpr (TMA) {
        const int per_slice = KEYS / p.box_rows;  // boxes along the tile's keys
        const int box = lane % per_slice, slice = lane / per_slice;
        if (lane == 0) tma_prefetch_desc(map);
        // a token outside the map is filled with zeros
        auto coord = [&]() {
          return slice < C::KCH ? token(j * KEYS + box * p.box_rows, p.pool_tokens) : 0;
        };
        int at = w.more ? coord() : 0;
        while (w.more) {
          const int now = at, st = g % stages;
          // the next tile's lookup is in flight during the wait for a stage
          auto look_up = [&]() {
            advance();
            if (w.more) at = coord();
          };
          if (g >= stages) look_up();
          if (!wait_stage(g)) break;
          if (lane == 0) mbar_arrive_expect_tx(full + st, C::KV_BYTES);
          __syncwarp();
          if (slice < C::KCH)
            tma_load_4d(ring + st * C::KV_BYTES + slice * KEYS * 128 + box * p.box_rows * 128, map,
                        full + st, slice * 64, kvh, now, 0);
          if (g < stages) look_up();
          copies = ++g;
        }
      } else {
        constexpr int CPR = D / 8, RPI = 32 / CPR;  // 16-byte chunks of a row, rows at a time
        const elem_t* pool = reinterpret_cast<const elem_t*>(is_k ? p.k_pool : p.v_pool) +
                             kvh * D + (lane % CPR) * 8;
        const int64_t tok_stride = static_cast<int64_t>(p.Hkv) * D;
        const int ch = lane % CPR;
        int row[2] = {-1, -1};  // pool tokens of the tile's keys lane and lane + 32
        auto look_up = [&]() {
#pragma unroll
          for (int h = 0; h < 2; ++h) row[h] = token(j * KEYS + h * 32 + lane, -1);
        };
        int told = 0;  // tiles announced to the MMA warp
        auto announce = [&]() {  // the last tile copied is there: its waits are over
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(full + told % stages);
          ++told;
        };
        if (w.more) look_up();
        while (w.more) {
          if (told < g && g >= stages &&
              !__all_sync(0xffffffffu, mbar_test(free_ + g % stages, (g / stages - 1) & 1))) {
            cp_async_wait<0>();
            announce();
          }
          if (!wait_stage(g)) break;
          uint8_t* dst = ring + (g % stages) * C::KV_BYTES + (ch / 8) * KEYS * 128;
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll 4
            for (int i = 0; i < 32; i += RPI) {
              const int r = i + lane / CPR, key = h * 32 + r;
              const int tok = __shfl_sync(0xffffffffu, row[h], r);
              cp_async_16(dst + key * 128 + (((ch % 8) ^ (key & 7)) * 16),
                          pool + max(tok, 0) * tok_stride, tok >= 0);
            }
          cp_async_commit();
          ++g;
          advance();
          if (w.more) look_up();
          if (told < g - 1) {
            cp_async_wait<1>();
            announce();
          }
        }
        cp_async_wait<0>();
        if (told < g) announce();
      }
    } else if (warp == 1) {
      // ---------------------------------------------- MMA issuer (one elected lane)
      constexpr int fmt = BF16 ? 1 : 0;
      constexpr uint32_t idesc_s = umma_idesc_f16(128, KEYS, fmt, 0, 0);
      constexpr uint32_t idesc_o = umma_idesc_f16(128, D, fmt, 0, 1);
      const uint64_t dq = umma_smem_desc(smem_u32(sQ), 16, 1024);
      const uint64_t dk = umma_smem_desc(smem_u32(sK), 16, 1024);
      const uint64_t dv = umma_smem_desc(smem_u32(sV), KEYS * 128, 1024);
      auto commit = [](uint64_t* bar) {
        if (elect_one_sync()) umma_commit(bar);
      };
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        return __all_sync(0xffffffffu,
                          mbar_wait_bounded(bar, parity, abort_flag, &g_wait_limit_ns));
      };
      auto issue_s = [&](int i) {  // S of the CTA's tile i, once K is there
        if (!wait(bar_k_full + i % C::ST, (i / C::ST) & 1)) return false;
        tc_fence_after();
        const uint64_t bk = dk + static_cast<uint64_t>(((i % C::ST) * C::KV_BYTES) >> 4);
        const uint32_t s_col = tmem + (i % NBUF) * KEYS;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t qo = ((kk >> 2) * 128 * 128 + (kk & 3) * 32) >> 4;
          const uint32_t ko = ((kk >> 2) * KEYS * 128 + (kk & 3) * 32) >> 4;
          if (elect_one_sync()) umma_ss(s_col, dq + qo, bk + ko, idesc_s, kk > 0 ? 1u : 0u);
        }
        commit(bar_s_full + i % NBUF);
        commit(bar_k_free + i % C::ST);
        return true;
      };
      bool ok = true;
      int g = 0;
      for (int piece = 0; ok && w.more; w.next(p, KEYS), ++piece) {
        const int hist = w.kv_len - p.M;
        // S runs NBUF tiles ahead of PV within a piece. Never into the next one: its Q
        // comes after this piece's output, behind the last PV.
        ok = wait(bar_q, piece & 1);
        for (int i = 0; ok && i < NBUF && i < w.n; ++i) ok = issue_s(g + i);
        for (int j = 0; ok && j < w.n; ++j, ++g) {
          const int st = g % C::ST;
          if (!(ok = wait(bar_v_full + st, (g / C::ST) & 1) &&
                     wait(bar_p_full + g % NBUF, (g / NBUF) & 1)))
            break;
          tc_fence_after();
          const uint64_t bv = dv + static_cast<uint64_t>((st * C::KV_BYTES) >> 4);
          // a masked first tile finds O zeroed by the softmax warps
          const uint32_t acc0 = j > 0 || (w.first + 1) * KEYS > hist ? 1u : 0u;
          const uint32_t p_col = tmem + (g % NBUF) * KEYS;
#pragma unroll
          for (int half = 0; half < 2; ++half)  // P's upper and lower halves
#pragma unroll
            for (int kk = 0; kk < KEYS / 16; ++kk)
              if (elect_one_sync())
                umma_ts(tmem + C::TM_O, p_col + half * (KEYS / 2) + kk * 8,
                        bv + ((kk * 16 * 128) >> 4), idesc_o, half > 0 || kk > 0 ? 1u : acc0);
          // a barrier of its own for a piece's last one: a warp that comes late to the
          // wait for it must not find bar_pv two phases on
          commit(j == w.n - 1 ? bar_o : bar_pv);
          commit(bar_v_free + st);
          // S of two tiles on goes to the buffer whose P the PV just issued reads: MMAs
          // of a CTA execute in issue order
          if (j + NBUF < w.n) ok = issue_s(g + NBUF);
        }
      }
      if (!ok && lane == 0) raise_status(CIE_DEV_TIMEOUT);
      // every MMA and commit has landed before TMEM and shared memory are released
      commit(bar_drain);
      mbar_wait_timeout(bar_drain, 0, kWaitLimitNs);
    } else {
      // ---------------------------------------------- warp 3: what has no tiles
      if (blockIdx.x == 0)
        for (int b = lane; b < p.B; b += 32)
          if (p.kv_lens[b] > p.max_blocks * p.block_size) raise_status(CIE_DEV_BAD_BLOCK_ID);
      for (int b = blockIdx.x; b < p.B; b += gridDim.x)
        if (tc_len(p, b) == 0)  // an empty sequence: zeros, 8 elements at a time
          for (int i = lane; i < p.Hq * p.M * (D / 8); i += 32) {
            const int r = i / (D / 8);
            elem_t* o = reinterpret_cast<elem_t*>(p.o) + b * p.o_sb + (r / p.M) * p.o_sh +
                        (r % p.M) * p.o_sm + (i % (D / 8)) * 8;
            if (p.o_vec) {
              *reinterpret_cast<uint4*>(o) = make_uint4(0, 0, 0, 0);
            } else {
              for (int e = 0; e < 8; ++e) o[e] = elem_t(0.f);
            }
          }
    }
  } else {
    if (warp - 4 < active) {
      // ---------------------------------------------- softmax warps
      const int wq = warp - 4;
      const int row = wq * 32 + lane;  // row of the group == TMEM lane
      const uint32_t lanes = static_cast<uint32_t>(wq * 32) << 16;
      const uint32_t o_col = tmem + lanes + C::TM_O;
      const int words = tree_words(p.M);
      const int gr = row0 + row;
      const bool live_row = gr < R;
      const int node = live_row ? gr % p.M : 0;
      const int head = kvh * p.G + (live_row ? gr / p.M : 0);
      const int64_t q_off = head * p.q_sh + node * p.q_sm;  // of this lane's row
      const uint32_t live_rows = __ballot_sync(0xffffffffu, live_row);
      TcWalk w, ahead;
      w.start(p, KEYS, groups, lane, len);

      // Q rows and parents of piece number k, `x`, on their way to shared memory: a warp
      // copies its 32 rows, whole rows at a time (a row per lane would touch 32 lines
      // with every instruction), and all parents, as the other warps do, the same values
      // to the same place.
      auto fetch = [&](const TcWalk& x, int k) {
        constexpr int CPR = D / 8, RPI = 32 / CPR;  // 16-byte chunks of a row, rows at a time
        const int ch = lane % CPR;
        const elem_t* src = reinterpret_cast<const elem_t*>(p.q) + x.b * p.q_sb + ch * 8;
        uint8_t* dst = sQ + (ch / 8) * 128 * 128 + wq * 32 * 128;
#pragma unroll 2
        for (int i = 0; i < 32; i += RPI) {
          const int r = i + lane / CPR;
          const int64_t off = __shfl_sync(0xffffffffu, q_off, r);
          if ((live_rows >> r) & 1u)
            cp_async_16(dst + r * 128 + (((ch % 8) ^ (r & 7)) * 16), src + off, true);
        }
        for (int i = lane; i < p.M; i += 32)
          cp_async_4(s_par + (k & 1) * kTcMaxTree + i, p.parents + x.b * p.par_sb + i);
        cp_async_commit();
      };
      auto parent = [&](int k, int i) { return tree_parent(s_par + (k & 1) * kTcMaxTree, i); };
      // ... and once there, Q rotated and handed to the MMA warp
      auto hand_over = [&](const TcWalk& x, int k) {
        cp_async_wait<0>();
        __syncwarp();
        if (p.cos != nullptr && live_row) {
          int pos = x.kv_len - p.M;
          for (int a = parent(k, node); a >= 0; a = parent(k, a)) ++pos;  // indices only fall: ends
          if (pos < 0 || pos >= p.rope_max_pos) {
            raise_status(CIE_DEV_BAD_POSITION);
            pos = pos < 0 ? 0 : p.rope_max_pos - 1;
          }
          rope_q_row<D, BF16>(sQ, row, pos, p.cos, p.sin);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_q);
      };

      bool ok = true;
      int g = 0, pieces = 0, pvs = 0, events = 0;  // tiles, pieces, phases of bar_pv, bar_seen
      if (w.more) {
        fetch(w, 0);
        hand_over(w, 0);
        if (lane == 0) mbar_arrive(bar_go);
      }
      for (; ok && w.more; w = ahead) {
        const int hist = w.kv_len - p.M;
        const int n = w.n;
        // first tile of the piece that reaches past the history
        const int first_masked = hist <= w.first * KEYS ? 0 : hist / KEYS - w.first;
        uint32_t anc[kTcMaxTree / 32 + 1];  // ancestors of the node; in local memory
        if (first_masked < n) {
          for (int i = 0; i < words; ++i) anc[i] = 0;
          if (live_row)
            for (int a = node; a >= 0; a = parent(pieces, a)) anc[a >> 5] |= 1u << (a & 31);
        }
        ahead = w;
        ahead.next(p, KEYS);

        float m_run = -INFINITY, l_run = 0.f;  // running max (log2 domain), sum
        for (int j = 0; j < n; ++j, ++g) {
          const int buf = g % NBUF;
          const uint32_t s_col = tmem + lanes + buf * KEYS;
          ok = __all_sync(0xffffffffu, mbar_wait_bounded(bar_s_full + buf,
                                                         (g / NBUF) & 1, abort_flag,
                                                         &g_wait_limit_ns));
          if (!ok) break;
          tc_fence_after();
          // the piece's last S is done with Q: fetch the next piece's
          if (j == n - 1 && ahead.more) fetch(ahead, pieces + 1);
          float sv[KEYS];
#pragma unroll
          for (int c = 0; c < KEYS; c += 32)
            tmem_ld32(s_col + c, reinterpret_cast<uint32_t*>(sv) + c);
          tmem_wait_ld();
          const bool masked = j >= first_masked;
          const int t0 = (w.first + j) * KEYS;
          uint32_t win[KEYS / 32];  // bit c of word h: key t0 + 32 h + c is visible to this row
          if (masked) {
#pragma unroll
            for (int h = 0; h < KEYS / 32; ++h) {
              const int j0 = t0 + h * 32 - hist;  // node of the word's first key
              auto word = [&](int i) -> uint32_t { return i >= 0 && i < words ? anc[i] : 0u; };
              uint32_t x = ~0u;
              if (j0 >= 0)
                x = __funnelshift_r(word(j0 >> 5), word((j0 >> 5) + 1), j0 & 31);
              else if (j0 > -32)  // its first -j0 keys are history
                x = (word(0) << -j0) | ((1u << -j0) - 1u);
              win[h] = x;
#pragma unroll
              for (int c = 0; c < 32; ++c)
                if (!(x & (1u << c))) sv[h * 32 + c] = -INFINITY;
            }
          }
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int c = 0; c < KEYS; c += 2)
            mx[(c >> 1) & 3] = fmax3(mx[(c >> 1) & 3], sv[c], sv[c + 1]);
          const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
          const float m_new = fmaxf(m_run, top * p.scale_log2);
          if (j == 0) {
            m_run = m_new;
            if (masked) {  // O starts at zero, so that the first PV may add to it
              uint32_t z[16];
#pragma unroll
              for (int e = 0; e < 16; ++e) z[e] = 0;
#pragma unroll
              for (int c = 0; c < D / 16; ++c) tmem_st16(o_col + c * 16, z);
            }
          } else {
            // rows whose max grew by more than 2^8 move their reference and rescale O; O
            // and the sum share the old one otherwise, which stays exact
            const bool need = m_new > m_run + 8.0f;
            if (__any_sync(0xffffffffu, need)) {
              ok = __all_sync(0xffffffffu, mbar_wait_bounded(bar_pv, (pvs + j - 1) & 1,
                                                             abort_flag, &g_wait_limit_ns));
              if (!ok) break;
              tc_fence_after();
              const float alpha = need ? ex2(m_run - m_new) : 1.0f;
#pragma unroll
              for (int c = 0; c < D / 16; ++c) {
                uint32_t ov[16];
                tmem_ld16(o_col + c * 16, ov);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 16; ++e)
                  ov[e] = __float_as_uint(__uint_as_float(ov[e]) * alpha);
                tmem_st16(o_col + c * 16, ov);
              }
              if (need) {
                l_run *= alpha;
                m_run = m_new;
              }
            }
          }
          const float m_use = m_run == -INFINITY ? 0.f : m_run;

          if (masked) {
            // V of a masked tile: rows past the sequence are zeroed (their P is 0, but
            // 0 x NaN is not), and rows of drafted nodes that hold NaN or infinity, none
            // as a rule, are added here for the rows that see them and zeroed as well.
            const int st = g % C::ST;
            uint8_t* v = sV + st * C::KV_BYTES;
            ok = __all_sync(0xffffffffu, mbar_wait_bounded(bar_v_full + st, (g / C::ST) & 1,
                                                           abort_flag, &g_wait_limit_ns));
            if (!ok) break;
            auto chunk = [&](int key, int ch) {
              return reinterpret_cast<uint4*>(v + (ch / 8) * KEYS * 128 + key * 128 +
                                              (((ch % 8) ^ (key & 7)) * 16));
            };
            auto clear = [&](int key) {  // this warp's share; PV waits for all warps
              for (int ch = wq; ch < D / 8; ch += active) *chunk(key, ch) = make_uint4(0, 0, 0, 0);
            };
            uint32_t bad[KEYS / 32];  // bit c of word h: key 32 h + c holds NaN or infinity
            bool any_bad = false;
            const int drafted = hist - t0;  // keys from here on are no history
#pragma unroll
            for (int h = 0; h < KEYS / 32; ++h) {  // a key per lane
              const int key = h * 32 + lane;
              bad[h] = 0;
              if (h * 32 + 31 < drafted) continue;
              bool nf = false;
              if (t0 + key >= w.kv_len) {
                clear(key);
              } else if (key >= drafted) {
                using elem2_t = typename std::conditional<BF16, __nv_bfloat162, __half2>::type;
                elem2_t z, acc;  // 0 x value: NaN once a value is not finite
                *reinterpret_cast<uint32_t*>(&z) = 0;
                acc = z;
#pragma unroll 4
                for (int ch = 0; ch < D / 8; ++ch) {
                  const uint4 x = *chunk(key, ch);
                  const elem2_t* e = reinterpret_cast<const elem2_t*>(&x);
                  acc = __hfma2(e[0], z, acc);
                  acc = __hfma2(e[1], z, acc);
                  acc = __hfma2(e[2], z, acc);
                  acc = __hfma2(e[3], z, acc);
                }
                const float2 f = unpack2<BF16>(*reinterpret_cast<uint32_t*>(&acc));
                nf = f.x != f.x || f.y != f.y;
              }
              bad[h] = __ballot_sync(0xffffffffu, nf);
              any_bad |= bad[h] != 0;
            }
            if (any_bad) {
              if (j > 0) {
                ok = __all_sync(0xffffffffu, mbar_wait_bounded(bar_pv, (pvs + j - 1) & 1,
                                                               abort_flag, &g_wait_limit_ns));
                if (!ok) break;
                tc_fence_after();
              }
              tmem_wait_st();  // O as rescaled or zeroed above
#pragma unroll 1
              for (int key = 0; key < KEYS; ++key) {
                uint32_t theirs = bad[0], mine = win[0];
#pragma unroll
                for (int h = 1; h < KEYS / 32; ++h)
                  if (key >= 32 * h) {
                    theirs = bad[h];
                    mine = win[h];
                  }
                if (!((theirs >> (key & 31)) & 1u)) continue;
                uint32_t raw;
                asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];"
                             : "=r"(raw)
                             : "r"(s_col + key));
                tmem_wait_ld();
                const bool sees = (mine >> (key & 31)) & 1u;
                const float s = sees ? __uint_as_float(raw) : -INFINITY;
                const float pj = ex2(s * p.scale_log2 - m_use);
#pragma unroll 1
                for (int c = 0; c < D / 16; ++c) {
                  uint32_t ov[16];
                  tmem_ld16(o_col + c * 16, ov);
                  tmem_wait_ld();
                  if (sees) {
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                      const uint4 x = *chunk(key, 2 * c + hf);
                      const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                      for (int e = 0; e < 4; ++e) {
                        const float2 f = unpack2<BF16>(u[e]);
                        uint32_t& a0 = ov[hf * 8 + 2 * e];
                        uint32_t& a1 = ov[hf * 8 + 2 * e + 1];
                        a0 = __float_as_uint(__uint_as_float(a0) + pj * f.x);
                        a1 = __float_as_uint(__uint_as_float(a1) + pj * f.y);
                      }
                    }
                  }
                  tmem_st16(o_col + c * 16, ov);
                }
                tmem_wait_st();
              }
              // every warp has read V before the rows are cleared
              __syncwarp();
              if (lane == 0) mbar_arrive(bar_seen);
              ok = __all_sync(0xffffffffu, mbar_wait_bounded(bar_seen, events & 1, abort_flag,
                                                             &g_wait_limit_ns));
              if (!ok) break;
              ++events;
#pragma unroll
              for (int h = 0; h < KEYS / 32; ++h)
                if ((bad[h] >> lane) & 1u) clear(h * 32 + lane);
            }
            fence_proxy_async_smem();
          }

          // p = 2^(s * scale - m) in groups of 8 pairs, as two halves of 16 bits
          const uint64_t sc2 = f2_pack(p.scale_log2, p.scale_log2);
          const uint64_t nm2 = f2_pack(-m_use, -m_use);
          uint64_t sum_a = f2_pack(0.f, 0.f), sum_b = sum_a;
#pragma unroll
          for (int h = 0; h < KEYS / 32; ++h) {  // 32 keys = 16 columns of P
            uint32_t pk[16], pl[16];
#pragma unroll
            for (int g0 = 0; g0 < 16; g0 += 8) {
              float e[16];
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const int c = h * 32 + 2 * (g0 + i);
                f2_unpack(ffma2(f2_pack(sv[c], sv[c + 1]), sc2, nm2), e[2 * i], e[2 * i + 1]);
              }
#pragma unroll
              for (int i = 0; i < 16; ++i) e[i] = ex2(e[i]);
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const uint64_t p2 = f2_pack(e[2 * i], e[2 * i + 1]);
                if (i & 1) sum_b = fadd2(sum_b, p2);
                else sum_a = fadd2(sum_a, p2);
                split2<BF16>(e[2 * i], e[2 * i + 1], pk[g0 + i], pl[g0 + i]);
              }
            }
            tmem_st16(s_col + h * 16, pk);
            tmem_st16(s_col + KEYS / 2 + h * 16, pl);
          }
          float s0, s1;
          f2_unpack(fadd2(sum_a, sum_b), s0, s1);
          l_run += s0 + s1;
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_p_full + buf);
        }
        if (!ok) break;
        pvs += n - 1;

        ok = __all_sync(0xffffffffu, mbar_wait_bounded(bar_o, pieces & 1, abort_flag,
                                                       &g_wait_limit_ns));
        if (!ok) break;
        tc_fence_after();
        const bool direct = n == w.tiles;
        const float inv = l_run > 0.f ? 1.0f / l_run : __int_as_float(0x7fc00000);
        // partials: a row that saw nothing has weight 0; a NaN sum stays NaN
        const bool live = !(l_run <= 0.f);
        // a CTA leaves at most one piece that does not open its sequence and one that does
        const int64_t pr =
            static_cast<int64_t>(2 * blockIdx.x + (w.first == 0 ? 1 : 0)) * p.rg_rows + row;
        elem_t* o = reinterpret_cast<elem_t*>(p.o) + w.b * p.o_sb + head * p.o_sh + node * p.o_sm;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          uint32_t ov[16];
          tmem_ld16(o_col + c * 16, ov);
          tmem_wait_ld();
          if (!live_row) continue;
          if (direct) {
            uint32_t pk[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
              pk[e] = pack2<BF16>(__uint_as_float(ov[2 * e]) * inv,
                                  __uint_as_float(ov[2 * e + 1]) * inv);
            if (p.o_vec) {
              *reinterpret_cast<uint4*>(o + c * 16) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
              *reinterpret_cast<uint4*>(o + c * 16 + 8) = make_uint4(pk[4], pk[5], pk[6], pk[7]);
            } else {
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                const uint16_t u = static_cast<uint16_t>(pk[e / 2] >> (16 * (e & 1)));
                o[c * 16 + e] = *reinterpret_cast<const elem_t*>(&u);
              }
            }
          } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float x[8];
#pragma unroll
              for (int e = 0; e < 8; ++e)
                x[e] = live ? __uint_as_float(ov[8 * h + e]) * inv : 0.f;
              store_f32x8(p.part_o + pr * D + c * 16 + 8 * h, x);
            }
          }
        }
        if (!direct && live_row) p.part_lse[pr] = live ? m_run + __log2f(l_run) : -INFINITY;
        tc_fence_before();  // the next piece's first PV overwrites O, behind this warp's next P
        ++pieces;
        if (ahead.more) hand_over(ahead, pieces);
      }
      cp_async_wait<0>();  // a role gave up: the next piece's Q and parents may be on their way
      if (!ok) raise_status(CIE_DEV_TIMEOUT);
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, C::TM_COLS);
  // a role gave up: copies still in flight land before the shared memory is released
  if (*abort_flag && copies > 0 && lane == 0) {
    uint64_t* full = warp == 0 ? bar_k_full : bar_v_full;
    for (int i = copies - 1; i >= 0 && i >= copies - C::ST; --i)
      mbar_wait_timeout(full + i % C::ST, (i / C::ST) & 1, kWaitLimitNs);
  }
}

// Joins the partial results of the units that the runs' borders cut: piece i of a
// unit weighs 2^(lse_i - max lse). One CTA per unit and slice of rows, one thread
// per float4 column of a row; a CTA whose unit was not cut returns at once.
constexpr int kTcMergeThreads = 128;
template <int D, bool BF16>
__global__ void __launch_bounds__(kTcMergeThreads)
    tree_merge_kernel(const PagedParams p, int ctas) {
  constexpr int keys = kTcKeys;
  constexpr int D4 = D / 4, ROWS = kTcMergeThreads / D4;
  const int lane = threadIdx.x & 31;
  const int groups = p.Hkv * p.row_groups;
  const int b = blockIdx.x / groups, y = blockIdx.x % groups;
  const int tiles = (tc_len(p, b) + keys - 1) / keys;
  if (tiles == 0) {  // idle: nothing to plan for
    asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }
  int mine;
  const TcPlan plan =
      tc_plan(p, keys, ctas / groups, lane, lane < p.B ? tc_len(p, lane) : 0, mine);
  int at = 0;  // the sequence's place in the list
  if (lane < b) at = mine;
  for (int i = lane + 32; i < b; i += 32) at += tc_places((tc_len(p, i) + keys - 1) / keys);
  at = __reduce_add_sync(0xffffffffu, at);
  const int c0 = at / plan.run, c1 = (at + tiles - 1) / plan.run;  // parts that share it
  // The partial results are there. Every CTA waits, also one without work: what
  // follows this kernel on the stream may count on the whole call being done.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (plan.whole || c0 == c1) return;
  const int r = blockIdx.y * ROWS + threadIdx.x / D4, c = threadIdx.x % D4;
  const int gr = (y % p.row_groups) * p.rg_rows + r;
  if (r >= p.rg_rows || gr >= p.G * p.M) return;
  auto row_of = [&](int part) {
    return static_cast<int64_t>(2 * (part * groups + y) + (part == c0 ? 1 : 0)) * p.rg_rows + r;
  };
  // eight pieces at a time, their loads in flight together; a NaN weight stays NaN
  float mx = -INFINITY, sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = c0; i0 <= c1; i0 += 8) {
    float lse[8];
    float4 v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool there = i0 + i <= c1;
      lse[i] = there ? __ldg(p.part_lse + row_of(i0 + i)) : -INFINITY;
      v[i] = there ? __ldg(reinterpret_cast<const float4*>(p.part_o + row_of(i0 + i) * D) + c)
                   : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float top = mx;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, lse[i]);
    if (top == -INFINITY) top = 0.f;  // nothing so far: all weights 0 (or NaN)
    const float old = ex2(mx - top);
    sum *= old;
    acc.x *= old;
    acc.y *= old;
    acc.z *= old;
    acc.w *= old;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float wt = ex2(lse[i] - top);
      sum += wt;
      acc.x += wt * v[i].x;
      acc.y += wt * v[i].y;
      acc.z += wt * v[i].z;
      acc.w += wt * v[i].w;
    }
    mx = top;
  }
  const float inv = sum > 0.f ? 1.0f / sum : __int_as_float(0x7fc00000);
  using elem_t = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  elem_t* dst = reinterpret_cast<elem_t*>(p.o) + b * p.o_sb +
                ((y / p.row_groups) * p.G + gr / p.M) * p.o_sh + (gr % p.M) * p.o_sm + c * 4;
  const uint32_t lo2 = pack2<BF16>(acc.x * inv, acc.y * inv), hi2 = pack2<BF16>(acc.z * inv, acc.w * inv);
  if (p.o_vec) {
    *reinterpret_cast<uint2*>(dst) = make_uint2(lo2, hi2);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint16_t u = static_cast<uint16_t>((e < 2 ? lo2 : hi2) >> (16 * (e & 1)));
      dst[e] = *reinterpret_cast<const elem_t*>(&u);
    }
  }
}

// ------------------------------------------------------------------ host
struct TreePlan {
  MmaPlan pl;  // the mma.sync kernel's plan, or the row groups and buffers of tcgen05
  int ctas;    // CTAs of the tcgen05 kernel; 0: the mma.sync kernel serves the call
  int min_run, whole;
};

// The tcgen05 kernel takes head dims 64 and 128 and trees whose bitmaps it holds (and
// lists and grids whose counts fit in an int), from a single row on: even trees of 5 over 2.2 GB of K/V take 340 us there and took 403 us in
// the mma.sync kernel, which serves everything else.
static TreePlan tree_plan(int B, int Hq, int Hkv, int T, int d, int block_size, int max_blocks,
                          int split_tokens) {
  const int max_len = max_blocks * block_size;
  const int64_t R = static_cast<int64_t>(Hq / Hkv) * T;
  TreePlan tp{};
  if ((d != 64 && d != 128) || T > kTcMaxTree ||
      static_cast<int64_t>(B) * (max_len / kTcKeys + 1 + kTcOpen) >= (1 << 30) ||
      static_cast<int64_t>(Hkv) * ((R + 127) / 128) > 4096) {
    tp.pl = make_plan(B, Hq, Hkv, T, d, max_len, split_tokens);
    return tp;
  }
  MmaPlan& pl = tp.pl;
  pl.row_groups = static_cast<int>((R + 127) / 128);
  pl.rg_rows = static_cast<int>((R + pl.row_groups - 1) / pl.row_groups + 31) / 32 * 32;
  const int groups = Hkv * pl.row_groups;
  const int max_tiles = (max_len + kTcKeys - 1) / kTcKeys;
  const int slots = num_sms() * 2;  // CTAs that run at once
  tp.min_run = kTcMinRun;
  tp.whole = kTcWhole;
  // parts of a head group's list: as many as run at once. With so many groups that more
  // than a tenth of the slots would idle, two to four rounds of CTAs, whichever leaves a
  // slot the smallest share of a list (rounds / parts). 8 contexts of 4K-8K, d = 64, one, two
  // and three rounds: 64 groups 186, 173 and 182 us; 80 groups 243, 214 and 215; 100 groups
  // 356, 292 and 281. One part more is a round more: 200, 243 and 309 us.
  int64_t parts = slots / groups;
  if (parts == 0 || (slots - parts * groups) * 10 > slots) {
    int64_t rounds = 1;
    for (int r = 2; r <= 4; ++r) {
      const int64_t n = static_cast<int64_t>(r) * slots / groups;
      if (n > 0 && (parts == 0 || r * parts < rounds * n)) {
        parts = n;
        rounds = r;
      }
    }
  }
  if (split_tokens > 0) {  // runs of that many tokens
    tp.min_run = (split_tokens + kTcKeys - 1) / kTcKeys;
    tp.whole = tp.min_run;
    parts = (static_cast<int64_t>(B) * (max_tiles + kTcOpen) + tp.min_run - 1) / tp.min_run;
    if (parts * groups > (1 << 20)) parts = (1 << 20) / groups;
  }
  // no more than there can be whole sequences, or runs
  const int64_t most = max_tiles <= tp.whole ? B : (static_cast<int64_t>(B) * (max_tiles + kTcOpen) + tp.min_run - 1) / tp.min_run;
  if (parts > most) parts = most;
  if (parts < 1) parts = 1;
  tp.ctas = static_cast<int>(parts) * groups;
  // sequences that cannot be longer than a whole one need no partial results
  pl.max_splits = max_tiles > tp.whole ? 2 : 1;
  const size_t part = static_cast<size_t>(2) * tp.ctas * pl.rg_rows;
  pl.part_o_bytes = (part * d * sizeof(float) + 255) & ~size_t(255);
  pl.part_lse_bytes = part * sizeof(float);
  return tp;
}

template <int D, bool BF16, bool TMA>
static int launch_tree_tc(const CUtensorMap& mk, const CUtensorMap& mv, const PagedParams& prm,
                          const TreePlan& tp, cudaStream_t st) {
  constexpr int smem = TcCfg<D>::SMEM;
  auto kern = tree_attn_kernel<D, BF16, TMA>;
  cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  kern<<<tp.ctas, kTcThreads, smem, st>>>(mk, mv, prm);
  CIE_CHECK_LAUNCH("tree_attn_kernel");
  if (prm.max_splits > 1) {
    constexpr int ROWS = kTcMergeThreads / (D / 4);
    const dim3 grid(prm.B * prm.Hkv * prm.row_groups, (prm.rg_rows + ROWS - 1) / ROWS);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kTcMergeThreads);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const cudaError_t e =
        cudaLaunchKernelEx(&cfg, tree_merge_kernel<D, BF16>, prm, tp.ctas);
    if (e != cudaSuccess) {
      cudaGetLastError();
      set_error("tree_merge_kernel: launch failed: %s", cudaGetErrorString(e));
      return CIE_ERR_LAUNCH;
    }
  }
  return CIE_OK;
}

template <int D, bool BF16>
static int dispatch_tree_tc(const PagedParams& prm, const TreePlan& tp, cudaStream_t st) {
  CUtensorMap mk{}, mv{};
  if (prm.box_rows == 0) return launch_tree_tc<D, BF16, false>(mk, mv, prm, tp, st);
  // (d, head, pool token, 1) with a (64, 1, 8 or 16, 1) box, 128-byte swizzle
  const cuuint64_t tokens = static_cast<cuuint64_t>(prm.pool_tokens);
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)prm.Hkv, tokens, 1};
  const cuuint64_t strides[3] = {(cuuint64_t)D * 2, (cuuint64_t)prm.Hkv * D * 2,
                                 tokens * prm.Hkv * D * 2};
  const cuuint32_t box[4] = {64, 1, (cuuint32_t)prm.box_rows, 1};
  if (!make_kv_map(&mk, prm.k_pool, D, dims, strides, box, BF16) ||
      !make_kv_map(&mv, prm.v_pool, D, dims, strides, box, BF16)) {
    set_error("cie_tree_attn: cuTensorMapEncodeTiled failed for the pools");
    return CIE_ERR_LAUNCH;
  }
  return launch_tree_tc<D, BF16, true>(mk, mv, prm, tp, st);
}

}  // namespace cie

using namespace cie;

extern "C" size_t cie_tree_attn_workspace(int B, int Hq, int Hkv, int T, int d, int block_size,
                                          int max_blocks, int split_tokens) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || T <= 0 || Hq % Hkv != 0 || !mma_head_dim_ok(d) ||
      block_size <= 0 || max_blocks < 0 ||
      static_cast<int64_t>(max_blocks) * block_size >= (int64_t(1) << 31) - 4096)
    return 0;
  return tree_plan(B, Hq, Hkv, T, d, block_size, max_blocks, split_tokens).pl.workspace();
}

extern "C" int cie_tree_attn(const void* q, const void* k_pool, const void* v_pool,
                             const int32_t* block_tables, const int32_t* kv_lens,
                             const int32_t* parents, int64_t parents_stride_b, void* o, int B,
                             int Hq, int Hkv, int T, int d, int num_blocks, int block_size,
                             int max_blocks, const int64_t* q_strides, const int64_t* o_strides,
                             float scale, int dtype, const float* rope_cos, const float* rope_sin,
                             int rope_max_pos, int split_tokens, void* workspace,
                             size_t workspace_bytes, void* stream) {
  CIE_CHECK_ARG(q && k_pool && v_pool && block_tables && kv_lens && parents && o,
                "cie_tree_attn: null tensor pointer");
  CIE_CHECK_ARG(B >= 0 && Hq > 0 && Hkv > 0 && T >= 0, "cie_tree_attn: bad shape");
  CIE_CHECK_ARG(Hq % Hkv == 0, "cie_tree_attn: Hq (%d) must be a multiple of Hkv (%d)", Hq, Hkv);
  CIE_CHECK_ARG(T <= CIE_MAX_TREE, "cie_tree_attn: %d nodes, at most %d", T, CIE_MAX_TREE);
  CIE_CHECK_ARG(parents_stride_b >= 0, "cie_tree_attn: negative parents stride");
  CIE_CHECK_ARG(dtype == CIE_DTYPE_BF16 || dtype == CIE_DTYPE_FP16, "cie_tree_attn: bad dtype %d",
                dtype);
  CIE_CHECK_ARG(num_blocks > 0 && block_size > 0 && max_blocks > 0,
                "cie_tree_attn: bad pool geometry");
  CIE_CHECK_ARG(static_cast<int64_t>(max_blocks) * block_size < (int64_t(1) << 31) - 4096,
                "cie_tree_attn: max_blocks * block_size too large");
  CIE_CHECK_ARG(q_strides && o_strides, "cie_tree_attn: null strides");
  // the kernels take the largest score for the largest exponent
  CIE_CHECK_ARG(scale > 0.f && scale <= FLT_MAX, "cie_tree_attn: scale must be positive and finite");
  CIE_CHECK_ARG(aligned16(q) && aligned16(k_pool) && aligned16(v_pool),
                "cie_tree_attn: q/k_pool/v_pool must be 16-byte aligned");
  CIE_CHECK_ARG(q_strides[0] % 8 == 0 && q_strides[1] % 8 == 0 && q_strides[2] % 8 == 0,
                "cie_tree_attn: q strides must be multiples of 8 elements");
  CIE_CHECK_ARG(split_tokens == 0 || (split_tokens > 0 && split_tokens % 16 == 0),
                "cie_tree_attn: split_tokens must be 0 or a positive multiple of 16");
  CIE_CHECK_ARG((rope_cos == nullptr) == (rope_sin == nullptr),
                "cie_tree_attn: rope_cos and rope_sin must both be given or both NULL");
  CIE_CHECK_ARG(rope_cos == nullptr || rope_max_pos > 0, "cie_tree_attn: rope_max_pos <= 0");
  if (!mma_head_dim_ok(d)) {
    set_error("cie_tree_attn: head_dim %d unsupported (16, 32, 64, 128 or 256)", d);
    return CIE_ERR_UNSUPPORTED;
  }
  if (B == 0 || T == 0) return CIE_OK;
  CIE_CHECK_ARG(static_cast<int64_t>(num_blocks) * block_size < (int64_t(1) << 31) - 16,
                "cie_tree_attn: pool too large");
  CIE_CHECK_ARG(rope_cos == nullptr || (aligned16(rope_cos) && aligned16(rope_sin)),
                "cie_tree_attn: rope tables must be 16-byte aligned");
  const TreePlan tp = tree_plan(B, Hq, Hkv, T, d, block_size, max_blocks, split_tokens);
  const MmaPlan& pl = tp.pl;
  if (pl.workspace() > 0 && (workspace == nullptr || workspace_bytes < pl.workspace())) {
    set_error("cie_tree_attn: workspace of %zu bytes required, got %zu", pl.workspace(),
              workspace_bytes);
    return CIE_ERR_WORKSPACE;
  }
  if (B > 65535 || static_cast<int64_t>(Hkv) * pl.row_groups > 65535 ||
      static_cast<int64_t>(B) * Hkv * pl.row_groups >= (int64_t(1) << 31)) {
    set_error("cie_tree_attn: grid too large (B=%d, Hkv*row_groups=%d)", B, Hkv * pl.row_groups);
    return CIE_ERR_UNSUPPORTED;
  }
  PagedParams prm{};
  fill_common(prm, pl, q, o, B, Hq, Hkv, T, q_strides, o_strides, scale, 0, rope_cos, rope_sin,
              rope_max_pos, workspace);
  prm.k_pool = k_pool;
  prm.v_pool = v_pool;
  prm.block_tables = block_tables;
  prm.kv_lens = kv_lens;
  prm.num_blocks = num_blocks;
  prm.block_size = block_size;
  prm.max_blocks = max_blocks;
  prm.bs_log2 = (block_size & (block_size - 1)) == 0 ? __builtin_ctz(block_size) : -1;
  prm.parents = parents;
  prm.par_sb = parents_stride_b;
  const bool bf16 = dtype == CIE_DTYPE_BF16;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (tp.ctas == 0) return dispatch_d<true, true>(prm, d, pl.mt, bf16, st);
  prm.pool_tokens = num_blocks * block_size;
  prm.o_vec = aligned16(o) && o_strides[0] % 8 == 0 && o_strides[1] % 8 == 0 &&
              o_strides[2] % 8 == 0;
  prm.box_rows = block_size % 16 == 0 ? 16 : block_size % 8 == 0 ? 8 : 0;
  prm.rg_rows = pl.rg_rows;
  prm.min_run = tp.min_run;
  prm.whole = tp.whole;
  if (d == 64)
    return bf16 ? dispatch_tree_tc<64, true>(prm, tp, st)
                : dispatch_tree_tc<64, false>(prm, tp, st);
  return bf16 ? dispatch_tree_tc<128, true>(prm, tp, st)
              : dispatch_tree_tc<128, false>(prm, tp, st);
}
