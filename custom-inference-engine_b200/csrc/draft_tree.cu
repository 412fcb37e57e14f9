// draft_tree.cu — the two steps that follow the attention over a tree of drafted
// tokens: which nodes are kept (verify_drafts) and the move of their K/V rows
// behind the history (keep_path). The attention itself is cie_tree_attn in
// tree_attn.cu. The reference decodes greedily on the host with one chain
// (engine/decode/speculative.py:88-123); here a whole batch of trees is decided
// on the device, without a host sync.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <memory>
#include <new>
#include <type_traits>

#include "cie_common.cuh"
#include "sm100_ptx.cuh"

namespace cie {

namespace cg = cooperative_groups;

// ------------------------------------------------------------------ verify
// Speculative sampling over a tree. At node `cur` with target row p (mass m = 1)
// and draft row q, its children x_1, x_2, .. are tested in index order:
//   keep x iff u q(x) m < r(x)          with r = p at first;
//   else r <- max(r - m q, 0), m <- sum_v r(v).
// As q is one row for all children of a node, r after k refusals is
// max(p - c q, 0) with c the sum of the masses so far, so no residual row is ever
// stored: a refusal costs one pass over p and q (read again from L2) and only if
// another child follows. Without draft probabilities a draft was chosen, not
// sampled: q is 1 at x, so a refusal zeroes r(x) and takes it off m, and no pass
// is needed. Where no child is kept, the last token is the first v with
//   cumsum(r)[v] > u_0 sum(r).
// The answers are whole numbers, so r, m and all sums are held in 64 bits: in
// fp32 a sum over 1e5 tokens is off by about as much as one token of a long tail
// weighs, and the drawn token would depend on the order of the additions.
//
// One cluster of up to 8 CTAs per sequence: every CTA reads the T nodes' p(x) and
// q(x) (one load each, all at once) and walks the tree by itself, and the CTAs
// meet only to add up a row, through distributed shared memory. Bound: the rows'
// bytes for large batches, and for one sequence four dependent memory latencies
// (entries, gathers, row, drawn segment). Measured on B200: 8.3 us for one chain of
// four drafts over 32000 tokens, 14.8 us for 32 chains over 128256 (33 MB of fp32
// rows, 5.1 us at the copy rate), 16.8 us for 8 greedy trees of 21. The drawn
// element is looked for by a whole CTA, one element a thread: with one warp walking
// a segment of 1024 the 32 chains took 24.4 us.
constexpr int kVfThreads = 512;
constexpr int kVfWarps = kVfThreads / 32;
constexpr int kSeg = 512;         // elements of a row summed by one warp at a time; one per
                                  // thread when the drawn token is looked for in it
constexpr int kVfMaxCluster = 8;  // portable cluster size
constexpr int kVfMaxRow = 1 << 23;  // elements of a row
// shared memory of a CTA for rows of `segs` segments of its own and T nodes
constexpr size_t vf_smem_bytes(int segs, int T) {
  return static_cast<size_t>(segs) * 8 + static_cast<size_t>(T) * (8 + 6 * 4);
}
static_assert(kSeg == kVfThreads, "the search gives every thread one element");

struct VerifyParams {
  const void* tokens;  // (B, T) int32 or int64
  int64_t tok_sb;
  int tok64;
  const int32_t* parents;
  int64_t par_sb;
  const void* p;  // (B, T, V)
  int64_t p_sb, p_st;
  const void* q;  // (B, Tq, V) or null
  int64_t q_sb, q_st;
  int Tq;
  const float* u;  // (B, T) or null: greedy
  int64_t u_sb;
  void* out_tokens;  // (B, T) contiguous, the type of tokens
  int32_t* path;     // (B, T)
  int32_t* n;        // (B,)
  int T, V;
  int segs;  // segments of a row per CTA
};

template <typename T>
__device__ __forceinline__ float to_f32(T x) {
  if constexpr (std::is_same<T, float>::value) return x;
  else if constexpr (std::is_same<T, __half>::value) return __half2float(x);
  else return __bfloat162float(x);
}

// VEC consecutive elements; VEC * sizeof(T) is 16 bytes (16-byte aligned rows) or one element.
template <typename T, int VEC>
__device__ __forceinline__ void load_row(const T* src, float (&x)[VEC]) {
  if constexpr (VEC == 1) {
    x[0] = to_f32(__ldg(src));
  } else {
    const uint4 w = __ldg(reinterpret_cast<const uint4*>(src));
    const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
    for (int i = 0; i < VEC; ++i) x[i] = to_f32(e[i]);
  }
}

// What is left of p at one element: max(p - c q, 0), NaN counting as nothing.
__device__ __forceinline__ double residual(float p, float q, double c) {
  const double d = static_cast<double>(p) - c * static_cast<double>(q);
  return d > 0.0 ? d : 0.0;
}
__device__ __forceinline__ double residual(float p) { return p > 0.f ? static_cast<double>(p) : 0.0; }

// 32-bit key whose unsigned order is the order of the floats, NaN above all (as
// torch.argmax has it) and -0 equal to +0.
__device__ __forceinline__ uint32_t order_key(float x) {
  x += 0.f;
  const uint32_t b = __float_as_uint(x);
  const uint32_t k = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return x != x ? 0xffffffffu : k;
}

template <typename T, int VEC, bool GREEDY>
__global__ void __launch_bounds__(kVfThreads) verify_kernel(const VerifyParams p) {
  extern __shared__ __align__(16) uint8_t vf_smem[];
  double* s_seg = reinterpret_cast<double*>(vf_smem);           // [segs]
  int64_t* s_tok = reinterpret_cast<int64_t*>(s_seg + p.segs);  // [T]
  int* s_par = reinterpret_cast<int*>(s_tok + p.T);             // [T]
  float* s_p = reinterpret_cast<float*>(s_par + p.T);           // [T] p(x) of each node
  float* s_q = s_p + p.T;                                       // [T] q(x)
  float* s_u = s_q + p.T;                                       // [T]
  int* s_path = reinterpret_cast<int*>(s_u + p.T);              // [T]
  int* s_gone = s_path + p.T;                                   // [T] refused children of the node
  __shared__ unsigned long long s_part[2];                      // this CTA's share of a row, two rounds
  __shared__ double s_cum[kVfMaxCluster + 1];                   // shares of the CTAs before each, and all
  __shared__ unsigned long long s_warp[kVfWarps];
  __shared__ double s_c;                                        // r = max(p - s_c q, 0)
  __shared__ double s_before;                                 // sum before the drawn segment
  __shared__ int s_cur, s_len, s_ngone, s_done, s_best;
  __shared__ int s_first, s_last, s_which;                      // the search for the last token

  cg::cluster_group cluster = cg::this_cluster();
  const int CL = static_cast<int>(cluster.num_blocks());
  const int rank = static_cast<int>(cluster.block_rank());
  const int b = blockIdx.x / CL;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const T* prow = static_cast<const T*>(p.p) + b * p.p_sb;
  const T* qrow = p.q ? static_cast<const T*>(p.q) + b * p.q_sb : nullptr;

  // the nodes' entries, then p(x) and q(x) at their parents' rows
  for (int i = tid; i < p.T; i += kVfThreads) {
    const int64_t at = b * p.tok_sb + i;
    const int64_t x = p.tok64 ? static_cast<const int64_t*>(p.tokens)[at]
                              : static_cast<const int32_t*>(p.tokens)[at];
    int a = p.parents[b * p.par_sb + i];
    if (a < -1 || a >= i || (a >= 0 && (x < 0 || x >= p.V))) {
      if (rank == 0) raise_status(CIE_DEV_BAD_TREE);
      if (a < -1 || a >= i) a = -1;
    }
    if (qrow != nullptr && a >= p.Tq) a = -1;  // no draft row: not a node that was expanded
    s_tok[i] = x;
    s_par[i] = a;
    if constexpr (!GREEDY) {
      const bool ok = a >= 0 && x >= 0 && x < p.V;
      s_p[i] = ok ? to_f32(prow[a * p.p_st + x]) : 0.f;
      s_q[i] = ok && qrow != nullptr ? to_f32(qrow[a * p.q_st + x]) : 0.f;
      s_u[i] = p.u[b * p.u_sb + i];
    }
  }
  if (tid == 0) {
    s_cur = 0;
    s_len = 1;
    s_path[0] = 0;
    s_ngone = 0;
    s_c = 0.0;
    s_done = 0;
  }
  __syncthreads();

  // first child of `node` with an index above `after`; T when there is none (warp 0)
  auto next_child = [&](int node, int after) -> int {
    for (int i0 = after + 1; i0 < p.T; i0 += 32) {
      const int i = i0 + lane;
      const uint32_t hit = __ballot_sync(0xffffffffu, i < p.T && s_par[i] == node);
      if (hit) return i0 + __ffs(hit) - 1;
    }
    return p.T;
  };
  // thread 0's 64-bit value of every CTA: CTA r's comes back in lane r of warp 0
  int round = 0;
  auto exchange = [&](unsigned long long mine) -> unsigned long long {
    unsigned long long* slot = s_part + (round++ & 1);  // two slots: one sync a round is enough
    if (tid == 0) *slot = mine;
    cluster.sync();
    return tid < CL ? *cluster.map_shared_rank(slot, tid) : 0ull;
  };

  const int seg0 = rank * p.segs;
  if constexpr (GREEDY) {
    // each round: the row's best token, then the child that drafted it
    while (true) {
      const T* row = prow + s_cur * p.p_st;
      unsigned long long best = 0;
      for (int s = warp; s < p.segs; s += kVfWarps) {
        const int64_t e0 = static_cast<int64_t>(seg0 + s) * kSeg;
#pragma unroll 4
        for (int j = 0; j < kSeg / (32 * VEC); ++j) {
          const int64_t at = e0 + (j * 32 + lane) * VEC;
          float x[VEC];
          if (VEC == 1 ? at < p.V : at + VEC <= p.V) {
            load_row<T, VEC>(row + at, x);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              const unsigned long long k =
                  (static_cast<unsigned long long>(order_key(x[e])) << 32) |
                  (0xffffffffu - static_cast<uint32_t>(at + e));
              best = k > best ? k : best;
            }
          } else if (VEC > 1) {
            for (int e = 0; e < VEC; ++e)
              if (at + e < p.V) {
                const unsigned long long k =
                    (static_cast<unsigned long long>(order_key(to_f32(row[at + e]))) << 32) |
                    (0xffffffffu - static_cast<uint32_t>(at + e));
                best = k > best ? k : best;
              }
          }
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long k = __shfl_xor_sync(0xffffffffu, best, o);
        best = k > best ? k : best;
      }
      if (lane == 0) s_warp[warp] = best;
      __syncthreads();
      if (tid == 0)
        for (int w = 1; w < kVfWarps; ++w) best = s_warp[w] > best ? s_warp[w] : best;
      unsigned long long all = exchange(best);
      if (warp == 0) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const unsigned long long k = __shfl_xor_sync(0xffffffffu, all, o);
          all = k > all ? k : all;
        }
        const int x = static_cast<int>(0xffffffffu - static_cast<uint32_t>(all));
        const int cur = s_cur;
        int child = next_child(cur, cur);
        while (child < p.T && s_tok[child] != x) child = next_child(cur, child);
        __syncwarp();
        if (lane == 0) {
          s_best = x;
          if (child < p.T) {
            s_cur = child;
            s_path[s_len++] = child;
          } else {
            s_done = 1;
          }
        }
      }
      __syncthreads();
      if (s_done) break;
    }
    if (rank == 0 && tid == 0) {
      const int64_t at = static_cast<int64_t>(b) * p.T + s_len - 1;
      if (p.tok64) static_cast<int64_t*>(p.out_tokens)[at] = s_best;
      else static_cast<int32_t*>(p.out_tokens)[at] = s_best;
    }
  } else {
    // r summed over one segment, the same value in every lane. `gone`: a refused
    // child's token lies in it (chosen drafts).
    auto left_at = [&](const T* pr, const T* qr, double c, int64_t at, bool gone) -> double {
      const float x = to_f32(pr[at]);
      double r = qr != nullptr ? residual(x, to_f32(qr[at]), c) : residual(x);
      if (gone)
        for (int i = 0; i < s_ngone; ++i)
          if (s_tok[s_gone[i]] == at) r = 0.0;
      return r;
    };
    auto gone_in = [&](int64_t e0) -> bool {
      bool hit = false;
      for (int i = lane; i < s_ngone; i += 32) {
        const int64_t x = s_tok[s_gone[i]];
        hit |= x >= e0 && x < e0 + kSeg;
      }
      return __any_sync(0xffffffffu, hit);
    };
    auto sum_row = [&](const T* pr, const T* qr, double c) {
      for (int s = warp; s < p.segs; s += kVfWarps) {
        const int64_t e0 = static_cast<int64_t>(seg0 + s) * kSeg;
        double sum = 0.0;
        if (e0 < p.V) {
          const bool gone = gone_in(e0);
          if (gone || e0 + kSeg > p.V) {  // an edge or an excluded token: one element at a time
            for (int64_t at = e0 + lane; at < e0 + kSeg && at < p.V; at += 32)
              sum += left_at(pr, qr, c, at, gone);
          } else {
            // all of the lane's loads first, then four chains of additions
            constexpr int kStep = kSeg / (32 * VEC) < 8 ? kSeg / (32 * VEC) : 8;
            double acc[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
            for (int j0 = 0; j0 < kSeg / (32 * VEC); j0 += kStep) {
              float x[kStep][VEC], y[kStep][VEC];
#pragma unroll
              for (int j = 0; j < kStep; ++j) {
                const int64_t at = e0 + ((j0 + j) * 32 + lane) * VEC;
                load_row<T, VEC>(pr + at, x[j]);
                if (qr != nullptr) load_row<T, VEC>(qr + at, y[j]);
              }
#pragma unroll
              for (int j = 0; j < kStep; ++j)
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                  acc[(j * VEC + e) & 3] +=
                      qr != nullptr ? residual(x[j][e], y[j][e], c) : residual(x[j][e]);
            }
            sum = (acc[0] + acc[1]) + (acc[2] + acc[3]);
          }
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        }
        if (lane == 0) s_seg[s] = sum;
      }
      __syncthreads();
      double mine = 0.0;
      if (warp == 0) {
        for (int s = lane; s < p.segs; s += 32) mine += s_seg[s];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
      }
      const unsigned long long got =
          exchange(static_cast<unsigned long long>(__double_as_longlong(mine)));
      if (warp == 0) {
        const double share = __longlong_as_double(static_cast<long long>(got));
        double cum = 0.0;  // every CTA adds the shares in the same order
        for (int r = 0; r < CL; ++r) {
          if (lane == 0) s_cum[r] = cum;
          cum += __shfl_sync(0xffffffffu, share, r);
        }
        if (lane == 0) s_cum[CL] = cum;
      }
      __syncthreads();
    };

    // the walk: warp 0 of every CTA, on the same numbers
    int at = 0;       // last child tested at s_cur
    double m = 1.0;   // mass left
    while (true) {
      if (warp == 0) {
        int cur = s_cur;
        double c = s_c;
        int ngone = s_ngone;
        bool sum = false;
        int child = next_child(cur, at);
        while (child < p.T) {
          at = child;
          const double qx = qrow != nullptr ? s_q[child] : 1.0;
          double r = qrow != nullptr && c > 0.0 ? residual(s_p[child], s_q[child], c)
                                                : residual(s_p[child]);
          if (qrow == nullptr) {  // an earlier sibling with the same token took it already
            bool same = false;
            for (int i = lane; i < ngone; i += 32) same |= s_tok[s_gone[i]] == s_tok[child];
            if (__any_sync(0xffffffffu, same)) r = 0.0;
          }
          if (static_cast<double>(s_u[child]) * qx * m < r) {
            cur = child;
            if (lane == 0) s_path[s_len++] = child;
            c = 0.0;
            m = 1.0;
            ngone = 0;
            child = next_child(cur, at);
            continue;
          }
          if (qrow != nullptr) {
            c += m;
            child = next_child(cur, at);
            if (child < p.T) {  // the next test needs the mass that is left
              sum = true;
              break;
            }
          } else {
            if (lane == 0) s_gone[ngone] = child;
            ++ngone;
            m -= r;
            __syncwarp();
            child = next_child(cur, at);
          }
        }
        __syncwarp();
        if (lane == 0) {
          s_cur = cur;
          s_c = c;
          s_ngone = ngone;
          s_done = sum ? 0 : 1;
        }
      }
      __syncthreads();
      const T* pr = prow + s_cur * p.p_st;
      const T* qr = s_c > 0.0 ? qrow + s_cur * p.q_st : nullptr;
      sum_row(pr, qr, s_c);
      m = s_cum[CL];
      if (s_done) break;
      __syncthreads();
    }

    // the last token; when nothing is left of the row, from the whole row
    if (!(s_cum[CL] > 0.0) && (s_c > 0.0 || s_ngone > 0)) {
      __syncthreads();
      if (tid == 0) {
        s_c = 0.0;
        s_ngone = 0;
      }
      __syncthreads();
      sum_row(prow + s_cur * p.p_st, nullptr, 0.0);
    }
    const double total = s_cum[CL];
    const int64_t out_at = static_cast<int64_t>(b) * p.T + s_len - 1;
    auto put = [&](int64_t x) {
      if (p.tok64) static_cast<int64_t*>(p.out_tokens)[out_at] = x;
      else static_cast<int32_t*>(p.out_tokens)[out_at] = static_cast<int32_t>(x);
    };
    if (!(total > 0.0) || isinf(total)) {
      if (rank == 0 && tid == 0) {
        raise_status(CIE_DEV_BAD_PROBS);
        put(-1);
      }
    } else {
      const double u0 = fmin(static_cast<double>(s_u[0]), 1.0 - 0x1p-24);
      const double want = (u0 > 0.0 ? u0 : 0.0) * total;
      int owner = CL - 1;
      for (int r = CL - 1; r >= 0; --r)
        if (s_cum[r + 1] > want) owner = r;
      if (owner == rank) {
        // warp 0: the segment where the running sum passes `want` (the last one with
        // mass if rounding leaves it just short), and the sum before it
        if (warp == 0) {
          double before = s_cum[rank];
          int seg = -1;
          double seg_before = before;
          for (int s0 = 0; s0 < p.segs; s0 += 32) {
            const double mass = s0 + lane < p.segs ? s_seg[s0 + lane] : 0.0;
            double inc = mass;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const double y = __shfl_up_sync(0xffffffffu, inc, o);
              if (lane >= o) inc += y;
            }
            const uint32_t some = __ballot_sync(0xffffffffu, mass > 0.0);
            const uint32_t over = __ballot_sync(0xffffffffu, mass > 0.0 && before + inc > want);
            if (some) {
              const int at = over ? __ffs(over) - 1 : 31 - __clz(some);
              seg = s0 + at;
              seg_before = before + __shfl_sync(0xffffffffu, inc - mass, at);
            }
            if (over) break;
            before += __shfl_sync(0xffffffffu, inc, 31);
          }
          if (lane == 0) {
            s_which = seg;
            s_before = seg_before;
            s_first = kSeg;
            s_last = -1;
          }
        }
        __syncthreads();
        // every thread one element of it: the first where the running sum passes
        const T* pr = prow + s_cur * p.p_st;
        const T* qr = s_c > 0.0 ? qrow + s_cur * p.q_st : nullptr;
        const int64_t e0 = static_cast<int64_t>(seg0 + s_which) * kSeg;
        const bool gone = gone_in(e0);
        const double r = e0 + tid < p.V ? left_at(pr, qr, s_c, e0 + tid, gone) : 0.0;
        double inc = r;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double y = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += y;
        }
        if (lane == 31) s_warp[warp] = static_cast<unsigned long long>(__double_as_longlong(inc));
        __syncthreads();
        double before = s_before;
        for (int w = 0; w < warp; ++w)
          before += __longlong_as_double(static_cast<long long>(s_warp[w]));
        if (r > 0.0) {
          atomicMax(&s_last, tid);
          if (before + inc > want) atomicMin(&s_first, tid);
        }
        __syncthreads();
        if (tid == 0) put(e0 + (s_first < kSeg ? s_first : s_last));
      }
    }
  }

  // the path and the kept drafts; -1 behind them
  if (rank == 0) {
    const int len = s_len;
    for (int i = tid; i < p.T; i += kVfThreads) {
      const int64_t at = static_cast<int64_t>(b) * p.T + i;
      p.path[at] = i < len ? s_path[i] : -1;
      if (i == len - 1) continue;  // the last token
      const int64_t x = i < len ? s_tok[s_path[i + 1]] : -1;
      if (p.tok64) static_cast<int64_t*>(p.out_tokens)[at] = x;
      else static_cast<int32_t*>(p.out_tokens)[at] = static_cast<int32_t>(x);
    }
    if (tid == 0) p.n[b] = len;
  }
  cluster.sync();  // no CTA leaves while another may still read its share
}

template <typename T, int VEC, bool GREEDY>
static int launch_verify(const VerifyParams& prm, int B, int cl, size_t smem, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(B) * cl);
  cfg.blockDim = dim3(kVfThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cl;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  // the limit belongs to the kernel, not to this call: one value for every caller, so
  // that no thread lowers it between another's setting and its launch
  if (smem > 40000)
    cudaFuncSetAttribute(
        verify_kernel<T, VEC, GREEDY>, cudaFuncAttributeMaxDynamicSharedMemorySize,
        static_cast<int>(vf_smem_bytes(kVfMaxRow / kSeg / kVfMaxCluster, CIE_MAX_TREE)));
  const cudaError_t e = cudaLaunchKernelEx(&cfg, verify_kernel<T, VEC, GREEDY>, prm);
  if (e != cudaSuccess) {
    cudaGetLastError();
    set_error("verify_kernel: launch failed: %s", cudaGetErrorString(e));
    return CIE_ERR_LAUNCH;
  }
  return CIE_OK;
}

template <typename T>
static int dispatch_verify(const VerifyParams& prm, int B, int cl, size_t smem, bool vec,
                           cudaStream_t st) {
  constexpr int VEC = 16 / sizeof(T);
  if (prm.u == nullptr)
    return vec ? launch_verify<T, VEC, true>(prm, B, cl, smem, st)
               : launch_verify<T, 1, true>(prm, B, cl, smem, st);
  return vec ? launch_verify<T, VEC, false>(prm, B, cl, smem, st)
             : launch_verify<T, 1, false>(prm, B, cl, smem, st);
}

// ------------------------------------------------------------------ kept path
// Slot base + i of every pool takes the K or V row of slot base + path[i], where
// base = kv_len - T is the length of the history. path rises from 0, so path[i]
// >= i, and a thread that copies its 16-byte column in the order i = 1, 2, .. never
// writes a slot that it has yet to read (slots read later are path[j] >= j > i):
// the move is in place, with no copy of the rows. Loads of up to 8 moves are in
// flight at once; that keeps the order, as all of them are read before the first
// is written. One launch serves all layers' pools: the latency of lengths, path
// and table, three dependent loads, is paid once per CTA, not once per layer.
// Bound: those latencies, then bytes. Measured on B200: 3.0 us for 3 rows in 32 pools
// (64 x 8 heads), 5.5 us for 160 rows of 2 KB in 32 pools (21 MB, 3.2 us at the copy
// rate).
constexpr int kMaxPools = 256;
constexpr int kKeepThreads = 128;

struct KeepParams {
  uint8_t* pools[kMaxPools];
  const int32_t* tables;
  const int32_t* kv_lens;
  const int32_t* path;
  const int32_t* n;
  int32_t* new_lens;
  int n_pools, pools_per_cta, T, num_blocks, block_size, max_blocks, row_chunks;
};

__global__ void __launch_bounds__(kKeepThreads) keep_path_kernel(const __grid_constant__ KeepParams p) {
  __shared__ int2 s_move[CIE_MAX_TREE];  // (from, to) pool rows; from < 0: nothing to do
  const int b = blockIdx.y;
  int n = p.n[b];
  const int len = max(p.kv_lens[b], 0);
  const int base = len - p.T;
  const int tid = threadIdx.x;
  if (n < 0 || n > p.T) {
    if (tid == 0) raise_status(CIE_DEV_BAD_TREE);
    n = n < 0 ? 0 : p.T;
  }
  if (len == 0) n = 0;  // an idle slot of a padded batch has no rows, whatever its verdict
  const int32_t* table = p.tables + static_cast<int64_t>(b) * p.max_blocks;
  auto row_of = [&](int pos) -> int {
    const int lb = pos / p.block_size;
    const int blk = pos >= 0 && lb < p.max_blocks ? table[lb] : -1;
    if (blk < 0 || blk >= p.num_blocks) {
      raise_status(CIE_DEV_BAD_BLOCK_ID);
      return -1;
    }
    return blk * p.block_size + pos % p.block_size;
  };
  for (int i = 1 + tid; i < n; i += kKeepThreads) {
    const int j = p.path[static_cast<int64_t>(b) * p.T + i];
    int2 mv = make_int2(-1, -1);
    if (j < i || j >= p.T) {
      raise_status(CIE_DEV_BAD_TREE);
    } else if (j > i) {
      const int from = row_of(base + j), to = row_of(base + i);
      if (from >= 0 && to >= 0) mv = make_int2(from, to);
    }
    s_move[i] = mv;
  }
  if (blockIdx.x == 0 && tid == 0 && p.new_lens != nullptr) p.new_lens[b] = max(0, base + n);
  __syncthreads();
  const int first = blockIdx.x * p.pools_per_cta;
  const int last = min(p.n_pools, first + p.pools_per_cta);
  const int64_t row_bytes = static_cast<int64_t>(p.row_chunks) * 16;
  for (int w = tid; w < (last - first) * p.row_chunks; w += kKeepThreads) {
    uint8_t* col = p.pools[first + w / p.row_chunks] + (w % p.row_chunks) * 16;
    for (int i0 = 1; i0 < n; i0 += 8) {
      uint4 v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (i0 + k < n && s_move[i0 + k].x >= 0)
          v[k] = *reinterpret_cast<const uint4*>(col + s_move[i0 + k].x * row_bytes);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (i0 + k < n && s_move[i0 + k].x >= 0)
          *reinterpret_cast<uint4*>(col + s_move[i0 + k].y * row_bytes) = v[k];
    }
  }
}

// The index in `pools` of a pool that shares memory with another, each `bytes` long; -1:
// none, -2: no host memory to look for it. The moves of two such pools would race.
static int shared_pool(void* const* pools, int n, uint64_t bytes) {
  uintptr_t few[kMaxPools];
  std::unique_ptr<uintptr_t[]> many;
  uintptr_t* at = few;
  if (n > kMaxPools) {
    many.reset(new (std::nothrow) uintptr_t[n]);
    at = many.get();
    if (at == nullptr) return -2;
  }
  for (int i = 0; i < n; ++i) at[i] = reinterpret_cast<uintptr_t>(pools[i]);
  std::sort(at, at + n);
  for (int i = 1; i < n; ++i)
    if (at[i] - at[i - 1] < bytes)
      for (int k = n - 1; k >= 0; --k)
        if (reinterpret_cast<uintptr_t>(pools[k]) == at[i]) return k;
  return -1;
}

}  // namespace cie

using namespace cie;

extern "C" int cie_verify_drafts(const void* tokens, int64_t tokens_stride_b, int tokens_64bit,
                                 const int32_t* parents, int64_t parents_stride_b,
                                 const void* target, const int64_t* target_strides,
                                 const void* draft, const int64_t* draft_strides, int draft_rows,
                                 const float* uniforms, int64_t uniforms_stride_b, int B, int T,
                                 int V, int dtype, void* out_tokens, int32_t* path, int32_t* n,
                                 void* stream) {
  CIE_CHECK_ARG(tokens && parents && target && target_strides && out_tokens && path && n,
                "cie_verify_drafts: null pointer");
  CIE_CHECK_ARG(B >= 0 && T > 0 && V > 0, "cie_verify_drafts: bad shape");
  CIE_CHECK_ARG(T <= CIE_MAX_TREE, "cie_verify_drafts: %d nodes, at most %d", T, CIE_MAX_TREE);
  CIE_CHECK_ARG(V <= kVfMaxRow, "cie_verify_drafts: %d tokens in a row, at most %d", V, kVfMaxRow);
  CIE_CHECK_ARG(dtype == CIE_DTYPE_BF16 || dtype == CIE_DTYPE_FP16 || dtype == CIE_DTYPE_FP32,
                "cie_verify_drafts: bad dtype %d", dtype);
  CIE_CHECK_ARG(draft == nullptr || (draft_strides && draft_rows > 0 && draft_rows <= T),
                "cie_verify_drafts: draft_rows must be in [1, T]");
  CIE_CHECK_ARG(uniforms != nullptr || draft == nullptr,
                "cie_verify_drafts: draft probabilities need uniforms");
  CIE_CHECK_ARG(tokens_stride_b >= 0 && parents_stride_b >= 0 && uniforms_stride_b >= 0,
                "cie_verify_drafts: negative stride");
  if (B == 0) return CIE_OK;
  CIE_CHECK_ARG(B <= (1 << 24), "cie_verify_drafts: batch too large");
  const int elem = dtype == CIE_DTYPE_FP32 ? 4 : 2;
  auto rows16 = [&](const void* base, const int64_t* s) {
    return aligned16(base) && (s[0] * elem) % 16 == 0 && (s[1] * elem) % 16 == 0;
  };
  const bool vec = rows16(target, target_strides) && (draft == nullptr || rows16(draft, draft_strides));
  // as many CTAs per sequence as give every one a few segments, up to a portable cluster
  const int nseg = (V + kSeg - 1) / kSeg;
  int cl = 1;
  while (cl < kVfMaxCluster && nseg >= 8 * cl) cl *= 2;
  VerifyParams prm{};
  prm.tokens = tokens;
  prm.tok_sb = tokens_stride_b;
  prm.tok64 = tokens_64bit ? 1 : 0;
  prm.parents = parents;
  prm.par_sb = parents_stride_b;
  prm.p = target;
  prm.p_sb = target_strides[0];
  prm.p_st = target_strides[1];
  prm.q = draft;
  if (draft != nullptr) {
    prm.q_sb = draft_strides[0];
    prm.q_st = draft_strides[1];
    prm.Tq = draft_rows;
  }
  prm.u = uniforms;
  prm.u_sb = uniforms_stride_b;
  prm.out_tokens = out_tokens;
  prm.path = path;
  prm.n = n;
  prm.T = T;
  prm.V = V;
  prm.segs = (nseg + cl - 1) / cl;
  const size_t smem = vf_smem_bytes(prm.segs, T);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case CIE_DTYPE_BF16: return dispatch_verify<__nv_bfloat16>(prm, B, cl, smem, vec, st);
    case CIE_DTYPE_FP16: return dispatch_verify<__half>(prm, B, cl, smem, vec, st);
    default: return dispatch_verify<float>(prm, B, cl, smem, vec, st);
  }
}

extern "C" int cie_keep_path(void* const* pools, int n_pools, const int32_t* block_tables,
                             const int32_t* kv_lens, const int32_t* path, const int32_t* n,
                             int32_t* new_lens, int B, int T, int num_blocks, int block_size,
                             int max_blocks, size_t row_bytes, void* stream) {
  CIE_CHECK_ARG((pools || n_pools == 0) && block_tables && kv_lens && path && n,
                "cie_keep_path: null pointer");
  CIE_CHECK_ARG(n_pools >= 0 && B >= 0 && T > 0, "cie_keep_path: bad shape");
  CIE_CHECK_ARG(T <= CIE_MAX_TREE, "cie_keep_path: %d nodes, at most %d", T, CIE_MAX_TREE);
  CIE_CHECK_ARG(num_blocks > 0 && block_size > 0 && max_blocks > 0,
                "cie_keep_path: bad pool geometry");
  CIE_CHECK_ARG(static_cast<int64_t>(num_blocks) * block_size < (int64_t(1) << 31) &&
                    static_cast<int64_t>(max_blocks) * block_size < (int64_t(1) << 31),
                "cie_keep_path: pool too large");
  CIE_CHECK_ARG(row_bytes > 0 && row_bytes % 16 == 0 && row_bytes <= (size_t(1) << 24),
                "cie_keep_path: row_bytes must be a positive multiple of 16");
  for (int i = 0; i < n_pools; ++i)
    CIE_CHECK_ARG(pools[i] != nullptr && aligned16(pools[i]),
                  "cie_keep_path: pool %d null or not 16-byte aligned", i);
  if (B == 0) return CIE_OK;
  CIE_CHECK_ARG(B <= 65535, "cie_keep_path: B must be <= 65535");
  const int twice =
      shared_pool(pools, n_pools, static_cast<uint64_t>(num_blocks) * block_size * row_bytes);
  CIE_CHECK_ARG(twice != -2, "cie_keep_path: no host memory for %d pools", n_pools);
  CIE_CHECK_ARG(twice == -1, "cie_keep_path: pool %d shares memory with another", twice);
  for (int p0 = 0; p0 == 0 || p0 < n_pools; p0 += kMaxPools) {
    KeepParams prm{};
    prm.n_pools = n_pools - p0 < kMaxPools ? n_pools - p0 : kMaxPools;
    for (int i = 0; i < prm.n_pools; ++i) prm.pools[i] = static_cast<uint8_t*>(pools[p0 + i]);
    prm.tables = block_tables;
    prm.kv_lens = kv_lens;
    prm.path = path;
    prm.n = n;
    prm.new_lens = p0 == 0 ? new_lens : nullptr;
    prm.T = T;
    prm.num_blocks = num_blocks;
    prm.block_size = block_size;
    prm.max_blocks = max_blocks;
    prm.row_chunks = static_cast<int>(row_bytes / 16);
    // one pool per CTA until the grid fills the GPU eight times over, then several
    const int64_t ctas = static_cast<int64_t>(B) * prm.n_pools;
    prm.pools_per_cta = static_cast<int>((ctas + 8 * num_sms() - 1) / (8 * num_sms()));
    if (prm.pools_per_cta < 1) prm.pools_per_cta = 1;
    const int gx = prm.n_pools > 0 ? (prm.n_pools + prm.pools_per_cta - 1) / prm.pools_per_cta : 1;
    keep_path_kernel<<<dim3(gx, B), kKeepThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(prm);
    CIE_CHECK_LAUNCH("keep_path_kernel");
  }
  return CIE_OK;
}
