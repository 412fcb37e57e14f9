// tree_attn.cu — attention of a tree of drafted tokens over the paged cache on
// the tcgen05 tensor cores, for trees whose G * T query rows per kv head are too
// many for the mma.sync kernel of paged_attn.cu to stay at memory speed.
//
// What it computes: see cie_tree_attn. The rows of a kv head (its G = Hq / Hkv
// query heads times the T nodes) are packed into 128-row tiles, so every K and V
// byte of the history is read once for all of them:
//   S = Q K^T            M = 128 rows, N = 64 keys, fp32 in TMEM
//   P = 2^(S scale - m)  one thread per row (= TMEM lane), no shuffles
//   O += P V             A = P from TMEM, fp32 in TMEM
// One CTA takes one split-KV partition of one (sequence, kv head, row group):
//   warp 0  TMA loader of K, warp 2 of V: one 16-token box per page lookup, a lane
//           each, into rings of 64-key tiles
//   warp 1  issues the MMAs: S runs two tiles ahead of PV in two TMEM buffers
//   warps 4..  softmax, one warpgroup per 128-row tile (NT = 1 or 2). Warps whose
//           32 rows are all padding do nothing.
// The history needs no mask. Only tiles that reach past it (the last T keys) are
// masked, by a 64-bit window per row out of ancestor bitmaps that each row's
// thread builds once from the parents.
//
// Bound: K/V bytes. A 64-key tile is 32 KB at d = 128, about 1400 cycles of one
// SM's share of HBM; its MMAs take 640 and its exponentials 512 (MUFU) per 128-row
// tile. With NT = 1 two CTAs share an SM (256 TMEM columns and ~100 KB each), so
// one's hand-offs hide behind the other's; NT = 2 fills the SM by itself.
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "cie_common.cuh"
#include "sm100_ptx.cuh"

namespace cie {

constexpr int kTcKeys = 64;      // keys of a tile
constexpr int kTcMaxTree = 256;  // nodes whose bitmaps fit beside the rings

template <int D, int NT>
struct TcCfg {
  static constexpr int KCH = D / 64;  // 128-byte swizzle slices along d
  static constexpr int Q_BYTES = 128 * D * 2;
  static constexpr int KV_BYTES = kTcKeys * D * 2;
  static constexpr int KS = NT == 1 ? (D == 128 ? 2 : 4) : (D == 128 ? 5 : 8);
  static constexpr int VS = NT == 1 ? (D == 128 ? 2 : 4) : (D == 128 ? 4 : 8);
  static constexpr int THREADS = 128 + 128 * NT;
  static constexpr int BOXES = KCH * (kTcKeys / 16);  // TMA boxes of a tile
  static constexpr int BAR_OFF = NT * Q_BYTES + (KS + VS) * KV_BYTES;
  static constexpr int NBARS = 1 + 2 * (KS + VS) + 2 * NT + 2 * NT + 2 * NT + 2 + 1;
  static constexpr int ANC_OFF = BAR_OFF + NBARS * 8 + 32;
  // + parents and one bitmap per row, sized by T; 1024 for alignment
  static int smem(int T) { return ANC_OFF + 4 * T + NT * 128 * tree_words(T) * 4 + 1024; }
  static constexpr uint32_t TM_O = NT * 128;  // S(t, buf) at t * 128 + buf * 64
  static constexpr uint32_t TM_COLS = NT == 1 ? 256 : 512;
};

__device__ __forceinline__ void named_barrier(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

template <int D, int NT, bool BF16>
__global__ void __launch_bounds__(TcCfg<D, NT>::THREADS, NT == 1 ? 2 : 1)
    tree_attn_kernel(const __grid_constant__ CUtensorMap tm_k,
                     const __grid_constant__ CUtensorMap tm_v, const PagedParams p) {
  using C = TcCfg<D, NT>;
  constexpr int RG = NT * 128;
  // fp16: P as two halves (p_hi + p_lo), as in paged_attn.cu and for its reason
  constexpr bool kSplitP = !BF16;
  using elem_t = typename std::conditional<BF16, __nv_bfloat16, __half>::type;

  const int split = blockIdx.x;
  const int kvh = blockIdx.y / p.row_groups;
  const int rg = blockIdx.y % p.row_groups;
  const int b = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  int kv_len = p.kv_lens[b];
  if (kv_len < 0) kv_len = 0;
  const int cap = p.max_blocks * p.block_size;
  if (kv_len > cap) {
    if (split == 0 && blockIdx.y == 0 && threadIdx.x == 0) raise_status(CIE_DEV_BAD_BLOCK_ID);
    kv_len = cap;
  }
  const int nsplit = kv_len > 0 ? (kv_len + p.split_tokens - 1) / p.split_tokens : 1;
  if (split >= nsplit) return;
  const int R = p.G * p.M;
  const int row0 = rg * RG;
  const int tok_begin = split * p.split_tokens;
  const int tok_end = min(kv_len, tok_begin + p.split_tokens);
  const int n = (tok_end - tok_begin + kTcKeys - 1) / kTcKeys;  // key tiles
  const int hist = kv_len - p.M;
  // first tile that reaches past the history
  const int first_masked = hist <= tok_begin ? 0 : (hist - tok_begin) / kTcKeys;

  if (n == 0) {  // an empty sequence: zeros
    for (int i = threadIdx.x; i < RG * D; i += C::THREADS) {
      const int gr = row0 + i / D;
      if (gr < R)
        reinterpret_cast<elem_t*>(p.o)[b * p.o_sb + (kvh * p.G + gr / p.M) * p.o_sh +
                                       (gr % p.M) * p.o_sm + i % D] = elem_t(0.f);
    }
    return;
  }

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                      // [NT][KCH][128][128B]
  uint8_t* sK = sQ + NT * C::Q_BYTES;      // [KS][KCH][64][128B]
  uint8_t* sV = sK + C::KS * C::KV_BYTES;  // [VS][KCH][64][128B]
  uint64_t* bar_q = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);
  uint64_t* bar_k_full = bar_q + 1;
  uint64_t* bar_v_full = bar_k_full + C::KS;
  uint64_t* bar_k_free = bar_v_full + C::VS;   // S of the stage's tile complete
  uint64_t* bar_v_free = bar_k_free + C::KS;   // PV of the stage's tile complete
  uint64_t* bar_s_full = bar_v_free + C::VS;   // [NT][2] S(t, buf) complete
  uint64_t* bar_p_full = bar_s_full + 2 * NT;  // [NT][2] P(t, buf) written
  uint64_t* bar_pv = bar_p_full + 2 * NT;      // [NT] phase j: PV(t) of tile j < n - 1 complete
  uint64_t* bar_o = bar_pv + NT;               // [NT] the last PV(t) complete
  uint64_t* bar_seen = bar_o + NT;             // [2] masked tiles: V looked at / V read
  uint64_t* bar_drain = bar_seen + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::BAR_OFF + C::NBARS * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  unsigned long long* s_bad = reinterpret_cast<unsigned long long*>(tmem_slot + 2);  // [2]
  int* s_parent = reinterpret_cast<int*>(smem + C::ANC_OFF);                // [M]
  uint32_t* s_anc = reinterpret_cast<uint32_t*>(s_parent + p.M);            // [RG][words]

  const int rows = min(RG, R - row0);
  const int active = (rows + 31) / 32;  // softmax warps with rows

  if (threadIdx.x == 0) {
    mbar_init(bar_q, active);
    for (int s = 0; s < C::KS; ++s) {
      mbar_init(bar_k_full + s, 1);
      mbar_init(bar_k_free + s, 1);
    }
    for (int s = 0; s < C::VS; ++s) {
      mbar_init(bar_v_full + s, 1);
      mbar_init(bar_v_free + s, 1);
    }
    for (int t = 0; t < NT; ++t) {
      const int warps = min(4, active - 4 * t);
      for (int i = 0; i < 2; ++i) {
        mbar_init(bar_s_full + 2 * t + i, 1);
        mbar_init(bar_p_full + 2 * t + i, warps > 0 ? warps : 1);
      }
      mbar_init(bar_pv + t, 1);
      mbar_init(bar_o + t, 1);
    }
    mbar_init(bar_seen + 0, active);
    mbar_init(bar_seen + 1, active);
    mbar_init(bar_drain, 1);
    *abort_flag = 0;
    s_bad[0] = s_bad[1] = 0;
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
  const int nt = (rows + 127) / 128;  // row tiles with rows

  if (warp == 0 || warp == 2) {
    // ------------------------------------------------ loaders
    const bool is_k = warp == 0;
    const CUtensorMap* map = is_k ? &tm_k : &tm_v;
    uint8_t* ring = is_k ? sK : sV;
    uint64_t* full = is_k ? bar_k_full : bar_v_full;
    uint64_t* free_ = is_k ? bar_k_free : bar_v_free;
    const int stages = is_k ? C::KS : C::VS;
    const int32_t* table = p.block_tables + static_cast<int64_t>(b) * p.max_blocks;
    const int box = lane % (kTcKeys / 16), slice = lane / (kTcKeys / 16);
    if (lane == 0) tma_prefetch_desc(map);
    // pool token of this lane's 16-token box of tile j; past the sequence, or for a
    // refused page, a token outside the map, which TMA fills with zeros
    auto coord = [&](int j) -> int {
      const int t = tok_begin + j * kTcKeys + box * 16;
      if (lane >= C::BOXES || t >= kv_len) return p.pool_tokens;
      const int lb = p.bs_log2 >= 0 ? t >> p.bs_log2 : t / p.block_size;
      const int blk = table[lb];  // t < kv_len <= max_blocks * block_size
      if (blk < 0 || blk >= p.num_blocks) {
        raise_status(CIE_DEV_BAD_BLOCK_ID);
        return p.pool_tokens;
      }
      return blk * p.block_size + (p.bs_log2 >= 0 ? t & (p.block_size - 1) : t % p.block_size);
    };
    int next = coord(0);
    int issued = 0;
    for (int j = 0; j < n; ++j) {
      const int at = next;
      if (j + 1 < n) next = coord(j + 1);  // the next lookup is in flight during the wait
      const int st = j % stages;
      if (j >= stages &&
          !__all_sync(0xffffffffu, mbar_wait_bounded(free_ + st, (j / stages - 1) & 1, abort_flag,
                                                     &g_wait_limit_ns)))
        break;
      if (lane == 0) mbar_arrive_expect_tx(full + st, C::KV_BYTES);
      __syncwarp();
      if (lane < C::BOXES)
        tma_load_4d(ring + st * C::KV_BYTES + slice * kTcKeys * 128 + box * 16 * 128, map,
                    full + st, slice * 64, kvh, at, 0);
      issued = j + 1;
    }
    if (*abort_flag && lane == 0) {
      // copies still in flight land before the shared memory is released
      for (int j = issued - 1; j >= 0 && j >= issued - stages; --j)
        mbar_wait_timeout(full + j % stages, (j / stages) & 1, kWaitLimitNs);
    }
  } else if (warp == 1) {
    // ------------------------------------------------ MMA issuer (one elected lane)
    constexpr int fmt = BF16 ? 1 : 0;
    constexpr uint32_t idesc_s = umma_idesc_f16(128, kTcKeys, fmt, 0, 0);
    constexpr uint32_t idesc_o = umma_idesc_f16(128, D, fmt, 0, 1);
    const uint64_t dq = umma_smem_desc(smem_u32(sQ), 16, 1024);
    const uint64_t dk = umma_smem_desc(smem_u32(sK), 16, 1024);
    const uint64_t dv = umma_smem_desc(smem_u32(sV), kTcKeys * 128, 1024);
    auto commit = [](uint64_t* bar) {
      if (elect_one_sync()) umma_commit(bar);
    };
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      return __all_sync(0xffffffffu,
                        mbar_wait_bounded(bar, parity, abort_flag, &g_wait_limit_ns));
    };
    auto issue_s = [&](int j) -> bool {
      const int st = j % C::KS;
      if (!wait(bar_k_full + st, (j / C::KS) & 1)) return false;
      tc_fence_after();
      const uint64_t bk = dk + static_cast<uint64_t>((st * C::KV_BYTES) >> 4);
      for (int t = 0; t < nt; ++t) {
        const uint64_t aq = dq + static_cast<uint64_t>((t * C::Q_BYTES) >> 4);
        const uint32_t s_col = tmem + t * 128 + (j & 1) * 64;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t qo = ((kk >> 2) * 128 * 128 + (kk & 3) * 32) >> 4;
          const uint32_t ko = ((kk >> 2) * kTcKeys * 128 + (kk & 3) * 32) >> 4;
          if (elect_one_sync()) umma_ss(s_col, aq + qo, bk + ko, idesc_s, kk > 0 ? 1u : 0u);
        }
        commit(bar_s_full + 2 * t + (j & 1));
      }
      commit(bar_k_free + st);
      return true;
    };
    bool ok = wait(bar_q, 0);
    tc_fence_after();
    for (int j = 0; ok && j < 2 && j < n; ++j) ok = issue_s(j);
    for (int j = 0; ok && j < n; ++j) {
      const int st = j % C::VS;
      if (!(ok = wait(bar_v_full + st, (j / C::VS) & 1))) break;
      const uint64_t bv = dv + static_cast<uint64_t>((st * C::KV_BYTES) >> 4);
      // a masked first tile finds O zeroed by the softmax warps
      const uint32_t acc0 = j > 0 || first_masked == 0 ? 1u : 0u;
      for (int t = 0; ok && t < nt; ++t) {
        if (!(ok = wait(bar_p_full + 2 * t + (j & 1), (j >> 1) & 1))) break;
        tc_fence_after();
        const uint32_t p_col = tmem + t * 128 + (j & 1) * 64;
        const uint32_t o_col = tmem + C::TM_O + t * D;
#pragma unroll
        for (int half = 0; half < (kSplitP ? 2 : 1); ++half)
#pragma unroll
          for (int kk = 0; kk < kTcKeys / 16; ++kk)
            if (elect_one_sync())
              umma_ts(o_col, p_col + half * 32 + kk * 8, bv + ((kk * 16 * 128) >> 4), idesc_o,
                      half > 0 || kk > 0 ? 1u : acc0);
        // a barrier of its own for the last one: a warp that comes late to the wait
        // for it must not find bar_pv two phases on
        commit((j < n - 1 ? bar_pv : bar_o) + t);
      }
      if (!ok) break;
      if (j < n - 1) commit(bar_v_free + st);
      // S of tile j + 2 goes to the buffer whose P the PV just issued reads: MMAs of
      // a CTA execute in issue order
      if (j + 2 < n) ok = issue_s(j + 2);
    }
    if (!ok) {
      if (lane == 0) raise_status(CIE_DEV_TIMEOUT);
      commit(bar_drain);  // all MMAs issued so far finish before TMEM is freed
      mbar_wait_timeout(bar_drain, 0, kWaitLimitNs);
    }
  } else if (warp >= 4 && warp - 4 < active) {
    // ------------------------------------------------ softmax warps
    const int sw = warp - 4, t = sw >> 2, wq = sw & 3;
    const int row = wq * 32 + lane;  // row of tile t == TMEM lane
    const int gr = row0 + t * 128 + row;
    const bool live_row = gr < R;
    const int node = live_row ? gr % p.M : 0;
    const uint32_t lanes = static_cast<uint32_t>(wq * 32) << 16;
    const uint32_t o_col = tmem + lanes + C::TM_O + t * D;
    const int tid = threadIdx.x - 128;
    const int words = tree_words(p.M);
    uint32_t* anc = s_anc + (t * 128 + row) * words;

    // parents, then this row's ancestors and depth
    for (int i = tid; i < p.M; i += 32 * active)
      s_parent[i] = tree_parent(p.parents + b * p.par_sb, i);
    named_barrier(1, 32 * active);
    int depth = -1;
    for (int w = 0; w < words; ++w) anc[w] = 0;
    if (live_row)
      for (int a = node; a >= 0; a = s_parent[a]) {  // indices only fall: ends
        anc[a >> 5] |= 1u << (a & 31);
        ++depth;
      }

    // Q row of this thread, rotated, into the swizzled tile
    {
      const elem_t* src = reinterpret_cast<const elem_t*>(p.q) + b * p.q_sb +
                          (kvh * p.G + (live_row ? gr / p.M : 0)) * p.q_sh + node * p.q_sm;
      uint8_t* dst = sQ + t * C::Q_BYTES + row * 128;
#pragma unroll
      for (int ch = 0; ch < D / 8; ++ch) {
        uint4 x = make_uint4(0, 0, 0, 0);
        if (live_row) x = *reinterpret_cast<const uint4*>(src + ch * 8);
        *reinterpret_cast<uint4*>(dst + (ch / 8) * 128 * 128 + (((ch % 8) ^ (row & 7)) * 16)) = x;
      }
      if (p.cos != nullptr && live_row) {
        int pos = hist + depth;
        if (pos < 0 || pos >= p.rope_max_pos) {
          raise_status(CIE_DEV_BAD_POSITION);
          pos = pos < 0 ? 0 : p.rope_max_pos - 1;
        }
        rope_q_row<D, BF16>(sQ + t * C::Q_BYTES, row, pos, p.cos, p.sin);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_q);
    }

    float m_run = -INFINITY, l_run = 0.f;  // running max (log2 domain), sum
    bool ok = true;
    int events = 0;  // masked tiles so far
    for (int j = 0; j < n; ++j) {
      const int buf = j & 1;
      const uint32_t s_col = tmem + lanes + t * 128 + buf * 64;
      ok = __all_sync(0xffffffffu, mbar_wait_bounded(bar_s_full + 2 * t + buf, (j >> 1) & 1,
                                                     abort_flag, &g_wait_limit_ns));
      if (!ok) break;
      tc_fence_after();
      float sv[kTcKeys];
      tmem_ld32(s_col, reinterpret_cast<uint32_t*>(sv));
      tmem_ld32(s_col + 32, reinterpret_cast<uint32_t*>(sv) + 32);
      tmem_wait_ld();
      const bool masked = j >= first_masked;
      const int t0 = tok_begin + j * kTcKeys;
      unsigned long long win = ~0ull;  // bit c: key t0 + c is visible to this row
      if (masked) {
        const int j0 = t0 - hist;  // node of the tile's first key
        auto word = [&](int i) -> unsigned long long { return i >= 0 && i < words ? anc[i] : 0u; };
        if (j0 < 0) {  // > -64: the tile's first -j0 keys are history
          win = (((word(1) << 32) | word(0)) << -j0) | ((1ull << -j0) - 1ull);
        } else {
          const int i = j0 >> 5, sh = j0 & 31;
          win = ((word(i + 1) << 32) | word(i)) >> sh;
          if (sh) win |= word(i + 2) << (64 - sh);
        }
#pragma unroll
        for (int c = 0; c < kTcKeys; ++c)
          if (!((win >> c) & 1ull)) sv[c] = -INFINITY;
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < kTcKeys; c += 2)
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
          ok = __all_sync(0xffffffffu, mbar_wait_bounded(bar_pv + t, (j - 1) & 1, abort_flag,
                                                         &g_wait_limit_ns));
          if (!ok) break;
          tc_fence_after();
          const float alpha = need ? ex2(m_run - m_new) : 1.0f;
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            uint32_t ov[16];
            tmem_ld16(o_col + c * 16, ov);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * alpha);
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
        // 0 x NaN is not), and rows of drafted nodes that hold NaN or infinity, none as
        // a rule, are added here for the rows that see them and zeroed as well.
        const int st = j % C::VS;
        uint8_t* v = sV + st * C::KV_BYTES;
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(bar_v_full + st, (j / C::VS) & 1,
                                                       abort_flag, &g_wait_limit_ns));
        if (!ok) break;
        const int slot = events & 1;
        auto chunk = [&](int key, int ch) {
          return reinterpret_cast<uint4*>(v + (ch / 8) * kTcKeys * 128 + key * 128 +
                                          (((ch % 8) ^ (key & 7)) * 16));
        };
        unsigned long long mine = 0;
        for (int i = tid; i < kTcKeys * (D / 8); i += 32 * active) {
          const int key = i / (D / 8), ch = i % (D / 8);
          if (t0 + key >= kv_len) {
            *chunk(key, ch) = make_uint4(0, 0, 0, 0);
          } else if (t0 + key >= hist) {
            const uint4 x = *chunk(key, ch);
            constexpr uint32_t kExp = BF16 ? 0x7f80u : 0x7c00u;
            const uint32_t u[4] = {x.x, x.y, x.z, x.w};
            bool nf = false;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              nf |= (u[e] & kExp) == kExp || (u[e] & (kExp << 16)) == (kExp << 16);
            if (nf) mine |= 1ull << key;
          }
        }
        if (mine) atomicOr(s_bad + slot, mine);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_seen + 0);
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(bar_seen + 0, events & 1, abort_flag,
                                                       &g_wait_limit_ns));
        if (!ok) break;
        const unsigned long long bad =
            *reinterpret_cast<volatile unsigned long long*>(s_bad + slot);
        if (bad) {
          if (j > 0) {
            ok = __all_sync(0xffffffffu, mbar_wait_bounded(bar_pv + t, (j - 1) & 1, abort_flag,
                                                           &g_wait_limit_ns));
            if (!ok) break;
            tc_fence_after();
          }
          tmem_wait_st();  // O as rescaled or zeroed above
          for (unsigned long long left = bad; left; left &= left - 1) {
            const int key = __ffsll(left) - 1;
            float s = -INFINITY;
            uint32_t raw;
            asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];"
                         : "=r"(raw)
                         : "r"(s_col + key));
            tmem_wait_ld();
            const bool sees = (win >> key) & 1ull;
            if (sees) s = __uint_as_float(raw);
            const float pj = ex2(s * p.scale_log2 - m_use);
#pragma unroll
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
        }
        // second meeting: every row has read V (and this tile's s_bad)
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_seen + 1);
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(bar_seen + 1, events & 1, abort_flag,
                                                       &g_wait_limit_ns));
        if (!ok) break;
        if (bad) {
          for (int i = tid; i < kTcKeys * (D / 8); i += 32 * active)
            if ((bad >> (i / (D / 8))) & 1ull) *chunk(i / (D / 8), i % (D / 8)) = make_uint4(0, 0, 0, 0);
          fence_proxy_async_smem();
          if (tid == 0) s_bad[slot] = 0;  // next used two masked tiles on
        }
        ++events;
      }

      // p = 2^(s * scale - m) in groups of 8 pairs, packed to 16 bits
      const uint64_t sc2 = f2_pack(p.scale_log2, p.scale_log2);
      const uint64_t nm2 = f2_pack(-m_use, -m_use);
      uint64_t sum_a = f2_pack(0.f, 0.f), sum_b = sum_a;
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // 32 keys = 16 columns of P
        uint32_t pk[16], pl[kSplitP ? 16 : 1];
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
            pk[g0 + i] = pack2<BF16>(e[2 * i], e[2 * i + 1]);
            if constexpr (kSplitP) {
              const float2 hi = unpack2<BF16>(pk[g0 + i]);
              pl[g0 + i] = pack2<BF16>(e[2 * i] - hi.x, e[2 * i + 1] - hi.y);
            }
          }
        }
        tmem_st16(s_col + h * 16, pk);
        if constexpr (kSplitP) tmem_st16(s_col + 32 + h * 16, pl);
      }
      float s0, s1;
      f2_unpack(fadd2(sum_a, sum_b), s0, s1);
      l_run += s0 + s1;
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_p_full + 2 * t + buf);
    }

    if (ok)
      ok = __all_sync(0xffffffffu,
                      mbar_wait_bounded(bar_o + t, 0, abort_flag, &g_wait_limit_ns));
    if (ok) {
      tc_fence_after();
      const bool direct = nsplit == 1;
      const float inv = l_run > 0.f ? 1.0f / l_run : __int_as_float(0x7fc00000);
      // partials: a row that saw nothing has weight 0; a NaN sum stays NaN
      const bool live = !(l_run <= 0.f);
      const int64_t unit = (static_cast<int64_t>(b) * p.Hkv + kvh) * p.row_groups + rg;
      const int64_t pr = (unit * p.max_splits + split) * RG + t * 128 + row;
      elem_t* o = reinterpret_cast<elem_t*>(p.o) + b * p.o_sb +
                  (kvh * p.G + (live_row ? gr / p.M : 0)) * p.o_sh + node * p.o_sm;
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
          float4* dst = reinterpret_cast<float4*>(p.part_o + pr * D + c * 16);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float4 x;
            x.x = live ? __uint_as_float(ov[4 * e]) * inv : 0.f;
            x.y = live ? __uint_as_float(ov[4 * e + 1]) * inv : 0.f;
            x.z = live ? __uint_as_float(ov[4 * e + 2]) * inv : 0.f;
            x.w = live ? __uint_as_float(ov[4 * e + 3]) * inv : 0.f;
            dst[e] = x;
          }
        }
      }
      if (!direct && live_row)
        p.part_lse[pr] = live ? m_run + __log2f(l_run) : -INFINITY;
      tc_fence_before();
    } else {
      raise_status(CIE_DEV_TIMEOUT);
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, C::TM_COLS);
}

// ------------------------------------------------------------------ host
// Query rows per kv head from which the tcgen05 kernel serves a call.
#ifndef CIE_TREE_TC_ROWS
#define CIE_TREE_TC_ROWS 33
#endif
// Split-KV partitions per resident CTA if every sequence were full, and the
// shortest partition.
#ifndef CIE_TREE_WAVES
#define CIE_TREE_WAVES 3
#endif
#ifndef CIE_TREE_MIN_SPLIT
#define CIE_TREE_MIN_SPLIT 256
#endif

struct TreePlan {
  MmaPlan pl;
  int tiles;  // 128-row tiles of a CTA (tcgen05), 0: the mma.sync kernel
};

// The tcgen05 kernel takes head dims 64 and 128, pages of whole 16-token boxes
// and trees whose bitmaps fit in shared memory; everything else, and few rows,
// go to the mma.sync kernel.
static TreePlan tree_plan(int B, int Hq, int Hkv, int T, int d, int block_size, int max_blocks,
                          int split_tokens) {
  const int max_len = max_blocks * block_size;
  const int64_t R = static_cast<int64_t>(Hq / Hkv) * T;
  TreePlan tp{};
  if ((d != 64 && d != 128) || block_size % 16 != 0 || T > kTcMaxTree || R < CIE_TREE_TC_ROWS) {
    tp.pl = make_plan(B, Hq, Hkv, T, d, max_len, split_tokens);
    return tp;
  }
  MmaPlan& pl = tp.pl;
  tp.tiles = R <= 128 ? 1 : 2;
  pl.rg_rows = 128 * tp.tiles;
  pl.row_groups = static_cast<int>((R + pl.rg_rows - 1) / pl.rg_rows);
  const int64_t units = static_cast<int64_t>(B) * Hkv * pl.row_groups;
  int64_t split = split_tokens;
  if (split == 0) {
    const int64_t slots = static_cast<int64_t>(num_sms()) * (tp.tiles == 1 ? 2 : 1);
    split = units * max_len / (slots * CIE_TREE_WAVES);
    if (split < CIE_TREE_MIN_SPLIT) split = CIE_TREE_MIN_SPLIT;
    if (split > 4096) split = 4096;
  }
  pl.split_tokens = static_cast<int>((split + kTcKeys - 1) / kTcKeys * kTcKeys);
  pl.max_splits = max_len > 0 ? (max_len + pl.split_tokens - 1) / pl.split_tokens : 1;
  const size_t part_rows = static_cast<size_t>(units) * pl.max_splits * pl.rg_rows;
  pl.part_o_bytes = (part_rows * d * sizeof(float) + 255) & ~size_t(255);
  pl.part_lse_bytes = part_rows * sizeof(float);
  return tp;
}

template <int D, int NT, bool BF16>
static int launch_tree_tc(const CUtensorMap& mk, const CUtensorMap& mv, const PagedParams& prm,
                          cudaStream_t st) {
  const int smem = TcCfg<D, NT>::smem(prm.M);
  auto kern = tree_attn_kernel<D, NT, BF16>;
  cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  kern<<<dim3(prm.max_splits, prm.Hkv * prm.row_groups, prm.B), TcCfg<D, NT>::THREADS, smem, st>>>(
      mk, mv, prm);
  CIE_CHECK_LAUNCH("tree_attn_kernel");
  if (prm.max_splits > 1) {
    constexpr int RG = 128 * NT;
    const dim3 grid(prm.B * prm.Hkv * prm.row_groups,
                    (RG + merge_rows<D, RG>() - 1) / merge_rows<D, RG>());
    paged_merge_kernel<D, RG, BF16, true><<<grid, kMergeThreads, 0, st>>>(prm);
    CIE_CHECK_LAUNCH("paged_merge_kernel");
  }
  return CIE_OK;
}

template <int D, bool BF16>
static int dispatch_tree_tc(const PagedParams& prm, int tiles, cudaStream_t st) {
  // (d, head, pool token, 1) with a (64, 1, 16, 1) box, 128-byte swizzle
  const cuuint64_t tokens = static_cast<cuuint64_t>(prm.pool_tokens);
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)prm.Hkv, tokens, 1};
  const cuuint64_t strides[3] = {(cuuint64_t)D * 2, (cuuint64_t)prm.Hkv * D * 2,
                                 tokens * prm.Hkv * D * 2};
  const cuuint32_t box[4] = {64, 1, 16, 1};
  CUtensorMap mk, mv;
  if (!make_kv_map(&mk, prm.k_pool, D, dims, strides, box, BF16) ||
      !make_kv_map(&mv, prm.v_pool, D, dims, strides, box, BF16)) {
    set_error("cie_tree_attn: cuTensorMapEncodeTiled failed for the pools");
    return CIE_ERR_LAUNCH;
  }
  return tiles == 1 ? launch_tree_tc<D, 1, BF16>(mk, mv, prm, st)
                    : launch_tree_tc<D, 2, BF16>(mk, mv, prm, st);
}

}  // namespace cie

using namespace cie;

extern "C" size_t cie_tree_attn_workspace(int B, int Hq, int Hkv, int T, int d, int block_size,
                                          int max_blocks, int split_tokens) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || T <= 0 || Hq % Hkv != 0 || !mma_head_dim_ok(d) ||
      block_size <= 0 || max_blocks < 0)
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
  if (B > 65535 || static_cast<int64_t>(Hkv) * pl.row_groups > 65535) {
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
  if (tp.tiles == 0) return dispatch_d<true, true>(prm, d, pl.mt, bf16, st);
  prm.pool_tokens = num_blocks * block_size;
  prm.o_vec = aligned16(o) && o_strides[0] % 8 == 0 && o_strides[1] % 8 == 0 &&
              o_strides[2] % 8 == 0;
  if (d == 64)
    return bf16 ? dispatch_tree_tc<64, true>(prm, tp.tiles, st)
                : dispatch_tree_tc<64, false>(prm, tp.tiles, st);
  return bf16 ? dispatch_tree_tc<128, true>(prm, tp.tiles, st)
              : dispatch_tree_tc<128, false>(prm, tp.tiles, st);
}
