// Tokens sorted by expert and back on one GPU: the way of a MoE layer's rows to the grouped GEMM and home, with its gradients.
//   slots[t, j] = rank of assignment (t, j) among all assignments ordered by expert, then by position (a stable counting sort);
//                 -1 for an assignment that names no expert (a dropped one)
//   permute     xp[slots[t, j]] = x[t]                      gradient: dx[t] = sum_j dxp[slots[t, j]]
//   unpermute   out[t] = sum_j gate[t, j] y[slots[t, j]]    gradient: dy[slots[t, j]] = gate[t, j] dout[t], dgate[t, j] = <dout[t], y[slots[t, j]]>
// The row kernels are memory bound. All of them walk the tokens, not the sorted rows: a token's row is read (or written) once for its
// top_k copies, which are scattered (or gathered) as whole rows; sums over a token's experts run in the order of j in fp32, so nothing
// depends on timing. Rows behind the last expert's (as many as there are dropped assignments) are written as zeros.
// 8192 tokens x 7168 bf16, top-8 of 256: sort 13 us, permute 168, unpermute 169, its gradient 313, the permutation's 164: 5.17 GB in 827 us, 95 % of
// the copy bandwidth. Small calls are bound by the host (11 us a call).
#include <cooperative_groups.h>

#include "pkb/api.h"
#include "pkb/host.h"
#include "pkb/ptx.cuh"

namespace pkb {

namespace {

namespace cg = cooperative_groups;

// ------------------------------------------------------------------------------------------------ sort
// One cluster of CTAs, one launch. A warp owns a contiguous run of assignments, 32 at a time. Pass 1 counts its experts in its own row of
// the CTA's table (lanes with the same expert find one another by votes; one of them adds for all, so the table needs no atomics);
// the table is then summed over warps, over CTAs (distributed shared memory) and over experts; pass 2 walks the assignments again and
// hands out the slots in order.
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortMaxExperts = 1024;
constexpr int kSortMaxBits = 10;
constexpr int kSortCluster = 16;

constexpr int kSortHeld = 8;       // rounds whose experts are held in registers between the passes

__global__ void __launch_bounds__(kSortThreads)
moe_sort_kernel(const int* __restrict__ idx, int n, int experts, int* __restrict__ offsets, int* __restrict__ order, int* __restrict__ slots) {
  extern __shared__ int table[];                        // [warps in use][experts]
  __shared__ int total[kSortMaxExperts], base[kSortMaxExperts], warp_sums[kSortWarps];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int all_rounds = (int)(((long long)n + 31) / 32);
  const int rounds = (all_rounds + kSortWarps * ctas - 1) / (kSortWarps * ctas);                // per warp
  const int warps = min(kSortWarps, (all_rounds + rounds - 1) / rounds);                        // that have any, in the first CTA
  const long long first = ((long long)rank * kSortWarps + warp) * rounds * 32;
  int* mine = table + warp * experts;
  // the experts of the first rounds, all loads in flight at once
  int held[kSortHeld];
#pragma unroll
  for (int r = 0; r < kSortHeld; ++r) {
    const long long i = first + r * 32 + lane;
    held[r] = r < rounds && i < n ? idx[i] : -1;
  }
  for (int e = threadIdx.x; e < warps * experts; e += kSortThreads) table[e] = 0;
  __syncthreads();
  const int bits = 32 - __clz(experts - 1);
  // lanes that name the same expert (of a lane that names one): a vote per bit of its number
  auto peers_of = [&](int e, bool ok) {
    unsigned peers = __ballot_sync(0xffffffffu, ok);
#pragma unroll
    for (int b = 0; b < kSortMaxBits; ++b) {
      if (b < bits) {
        const unsigned set = __ballot_sync(0xffffffffu, (e >> b) & 1);
        peers &= (e >> b) & 1 ? set : ~set;
      }
    }
    return peers;
  };
  auto count = [&](int e) {
    const bool ok = (unsigned)e < (unsigned)experts;
    const unsigned peers = peers_of(e, ok);
    if (ok && lane == __ffs(peers) - 1) mine[e] += __popc(peers);
    __syncwarp();
  };
#pragma unroll
  for (int r = 0; r < kSortHeld; ++r)
    if (r < rounds && first + r * 32 < n) count(held[r]);
  for (int r = kSortHeld; r < rounds && first + r * 32ll < n; ++r) {
    const long long i = first + r * 32ll + lane;
    count(i < n ? idx[i] : -1);
  }
  __syncthreads();
  const int e = threadIdx.x;
  if (e < experts) {
    int run = 0;
    for (int w = 0; w < warps; ++w) {
      const int c = table[w * experts + e];
      table[w * experts + e] = run;
      run += c;
    }
    total[e] = run;
  }
  int before = 0, all = 0;
  if (ctas > 1) {
    cluster.sync();
    if (e < experts) {
      for (int c = 0; c < ctas; ++c) {
        const int v = cluster.map_shared_rank(total, c)[e];
        if (c < rank) before += v;
        all += v;
      }
    }
  } else if (e < experts) {
    all = total[e];
  }
  // exclusive sum over the experts, one per thread
  int incl = all;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += v;
  }
  if (lane == 31) warp_sums[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    int s = warp_sums[lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, s, d);
      if (lane >= d) s += v;
    }
    warp_sums[lane] = s;
  }
  __syncthreads();
  const int start = incl - all + (warp > 0 ? warp_sums[warp - 1] : 0);
  const int kept = warp_sums[kSortWarps - 1];
  if (e < experts) {
    base[e] = start + before;
    if (rank == 0) {
      offsets[e] = start;
      if (e == experts - 1) offsets[experts] = kept;
    }
  }
  __syncthreads();
  auto place = [&](long long i, int x) {
    const bool ok = (unsigned)x < (unsigned)experts;
    const unsigned peers = peers_of(x, ok);
    const int slot = ok ? base[x] + mine[x] + __popc(peers & ((1u << lane) - 1u)) : -1;
    __syncwarp();
    if (ok && lane == __ffs(peers) - 1) mine[x] += __popc(peers);
    __syncwarp();
    if (i < n) slots[i] = slot;
    if (ok) order[slot] = (int)i;
  };
#pragma unroll
  for (int r = 0; r < kSortHeld; ++r)
    if (r < rounds && first + r * 32 < n) place(first + r * 32 + lane, held[r]);
  for (int r = kSortHeld; r < rounds && first + r * 32ll < n; ++r) {
    const long long i = first + r * 32ll + lane;
    place(i, i < n ? idx[i] : -1);
  }
  for (long long i = kept + (long long)rank * kSortThreads + threadIdx.x; i < n; i += (long long)ctas * kSortThreads) order[i] = -1;
  if (ctas > 1) cluster.sync();      // nobody leaves while its totals may still be read
}

// ------------------------------------------------------------------------------------------------ rows
// 16 bytes (VEC = 8 bf16 or 4 fp32 values) or one value of a row, as it is or as fp32
template <typename T, int VEC>
struct RowVec {
  using Raw = typename std::conditional<VEC == 1, T, U4>::type;
  static __device__ __forceinline__ Raw load(const T* p) {
    if constexpr (VEC == 1) return *p;
    else return ld_global_nc_v4(p);
  }
  static __device__ __forceinline__ void store(T* p, const Raw& v) {
    if constexpr (VEC == 1) *p = v;
    else st_global_v4(p, v);
  }
  static __device__ __forceinline__ Raw zero() {
    if constexpr (VEC == 1) return T(0.f);
    else return U4{0u, 0u, 0u, 0u};
  }
  static __device__ __forceinline__ void unpack(const Raw& v, float (&f)[VEC]) {
    if constexpr (VEC == 1) f[0] = static_cast<float>(v);
    else unpack16(v, f);
  }
  static __device__ __forceinline__ Raw pack(const float (&f)[VEC]) {
    if constexpr (VEC == 1) {
      if constexpr (sizeof(T) == 2) return __float2bfloat16_rn(f[0]);
      else return f[0];
    } else {
      return pack16(f);
    }
  }
};

constexpr int kRowThreads = 256;

// Where a thread works: blocks are split into teams of `team` threads (a power of two); a team takes one token and one piece of
// team * unroll accesses of its row.
struct RowGrid {
  int team_log2, pieces;
  __device__ __forceinline__ bool place(long long tokens, long long& token, int& first, int unroll = 1) const {
    const int team = 1 << team_log2;
    const long long unit = (long long)blockIdx.x * (kRowThreads >> team_log2) + (threadIdx.x >> team_log2);
    token = unit / pieces;
    first = (int)(unit - token * pieces) * team * unroll + (threadIdx.x & (team - 1));
    return token < tokens;
  }
};

// zeros into the rows from `kept` on, by all blocks
template <typename T, int VEC>
__device__ __forceinline__ void zero_rows(T* rows, long long n, int nvec, const int* kept) {
  const long long from = max(*kept, 0), count = (n - from) * nvec;
  for (long long i = (long long)blockIdx.x * kRowThreads + threadIdx.x; i < count; i += (long long)gridDim.x * kRowThreads) {
    const long long r = i / nvec;
    RowVec<T, VEC>::store(rows + ((from + r) * nvec + (i - r * nvec)) * VEC, RowVec<T, VEC>::zero());
  }
}

// accesses per thread of the permutation
constexpr int row_unroll(int vec) { return vec == 1 ? 4 : 2; }

template <typename T, int VEC>
__global__ void __launch_bounds__(kRowThreads)
moe_permute_kernel(const T* __restrict__ x, long long ldx, const int* __restrict__ slots, const int* __restrict__ kept, T* __restrict__ xp,
                   long long tokens, int top_k, int nvec, const RowGrid grid) {
  using V = RowVec<T, VEC>;
  constexpr int U = row_unroll(VEC);
  long long t;
  int first;
  if (grid.place(tokens, t, first, U)) {
    const int team = 1 << grid.team_log2;
    const unsigned n = (unsigned)(tokens * top_k);
    typename V::Raw v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (first + u * team < nvec) v[u] = V::load(x + t * ldx + (long long)(first + u * team) * VEC);
    for (int j = 0; j < top_k; ++j) {
      const unsigned s = (unsigned)slots[t * top_k + j];
      if (s < n) {
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (first + u * team < nvec) V::store(xp + ((long long)s * nvec + first + u * team) * VEC, v[u]);
      }
    }
  }
  zero_rows<T, VEC>(xp, tokens * top_k, nvec, kept);
}

// out[t] = sum_j gate[t, j] y[slots[t, j]]; GATED = false: weights of one. One access per row and thread, eight rows in flight: with two
// accesses per row the registers left two blocks per SM, too few to cover the way from a slot to its row (8192 tokens x 7168, top-8: 210 us).
constexpr int kGatherAhead = 8;   // accesses in flight per thread before the first of them is added
// single values: four columns of two rows (four bytes per access of eight rows leave a warp with half a line each)
constexpr int gather_unroll(int vec) { return vec == 1 ? 4 : 1; }

template <typename T, int VEC, bool GATED>
__global__ void __launch_bounds__(kRowThreads, 4)
moe_unpermute_kernel(const T* __restrict__ y, long long ldy, const int* __restrict__ slots, const float* __restrict__ gates, T* __restrict__ out,
                     long long tokens, int top_k, int nvec, const RowGrid grid) {
  using V = RowVec<T, VEC>;
  constexpr int U = gather_unroll(VEC), kAhead = kGatherAhead / U;
  long long t;
  int first;
  if (!grid.place(tokens, t, first, U) || first >= nvec) return;
  const int team = 1 << grid.team_log2;
  const unsigned n = (unsigned)(tokens * top_k);
  float acc[U][VEC] = {};
  for (int j0 = 0; j0 < top_k; j0 += kAhead) {
    typename V::Raw v[kAhead][U];
    unsigned s[kAhead];
    float g[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      s[a] = j0 + a < top_k ? (unsigned)slots[t * top_k + j0 + a] : n;
      g[a] = GATED && j0 + a < top_k ? gates[t * top_k + j0 + a] : 1.f;
    }
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      if (s[a] < n) {
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (U == 1 || first + u * team < nvec) v[a][u] = V::load(y + (long long)s[a] * ldy + (long long)(first + u * team) * VEC);
      }
    }
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      if (s[a] < n) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float f[VEC];
          V::unpack(v[a][u], f);
#pragma unroll
          for (int c = 0; c < VEC; ++c) acc[u][c] += GATED ? g[a] * f[c] : f[c];
        }
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (U == 1 || first + u * team < nvec) V::store(out + (t * nvec + first + u * team) * VEC, V::pack(acc[u]));
}

// A team of TEAM threads per token: dy rows and the dot products in one pass over dout and y.
constexpr int kBwdExperts = 8;    // experts of a token that a pass over its row handles at once

template <typename T, int VEC, int TEAM>
__global__ void __launch_bounds__(kRowThreads)
moe_unpermute_bwd_kernel(const T* __restrict__ dout, long long lddo, const T* __restrict__ y, long long ldy, const int* __restrict__ slots,
                         const float* __restrict__ gates, const int* __restrict__ kept, T* __restrict__ dy, float* __restrict__ dgates,
                         long long tokens, int top_k, int nvec) {
  using V = RowVec<T, VEC>;
  constexpr int kTeams = kRowThreads / TEAM, kWarps = TEAM / 32;
  __shared__ float red[kRowThreads / 32][kBwdExperts];
  const unsigned n = (unsigned)(tokens * top_k);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, in_team = threadIdx.x % TEAM;
  const long long t = (long long)blockIdx.x * kTeams + threadIdx.x / TEAM;
  // a team of one warp leaves when there is no token for it; larger teams are the whole block
  static_assert(TEAM == 32 || TEAM == kRowThreads, "teams are a warp or the block");
  for (int j0 = 0; j0 < top_k && t < tokens; j0 += kBwdExperts) {
    unsigned s[kBwdExperts];
    float g[kBwdExperts], dot[kBwdExperts] = {};
#pragma unroll
    for (int a = 0; a < kBwdExperts; ++a) {
      const bool in = j0 + a < top_k;
      s[a] = in ? (unsigned)slots[t * top_k + j0 + a] : n;
      g[a] = in ? gates[t * top_k + j0 + a] : 0.f;
    }
    constexpr int U = VEC == 1 ? 4 : 1;           // columns of a thread whose loads are in flight together
    for (int i0 = in_team; i0 < nvec; i0 += U * TEAM) {
      float d[U][VEC];
      typename V::Raw v[U][kBwdExperts];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * TEAM;
        if (U > 1 && i >= nvec) break;
        V::unpack(V::load(dout + t * lddo + (long long)i * VEC), d[u]);
#pragma unroll
        for (int a = 0; a < kBwdExperts; ++a)
          if (s[a] < n) v[u][a] = V::load(y + (long long)s[a] * ldy + (long long)i * VEC);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * TEAM;
        if (U > 1 && i >= nvec) break;
#pragma unroll
        for (int a = 0; a < kBwdExperts; ++a) {
          if (s[a] < n) {
            float f[VEC], o[VEC];
            V::unpack(v[u][a], f);
#pragma unroll
            for (int c = 0; c < VEC; ++c) {
              dot[a] += d[u][c] * f[c];
              o[c] = g[a] * d[u][c];
            }
            V::store(dy + ((long long)s[a] * nvec + i) * VEC, V::pack(o));
          }
        }
      }
    }
#pragma unroll
    for (int a = 0; a < kBwdExperts; ++a) {
      const float w = warp_sum(dot[a]);
      if (lane == 0) red[warp][a] = w;
    }
    if constexpr (TEAM > 32) __syncthreads();
    else __syncwarp();
    if (in_team < kBwdExperts && j0 + in_team < top_k) {
      const int w0 = TEAM > 32 ? 0 : warp;
      float w = 0.f;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) w += red[w0 + k][in_team];
      dgates[t * top_k + j0 + in_team] = w;
    }
    if constexpr (TEAM > 32) __syncthreads();
    else __syncwarp();
  }
  zero_rows<T, VEC>(dy, tokens * top_k, nvec, kept);
}

bool rows_aligned(const void* p, long long pitch_bytes) { return ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)pitch_bytes) & 15) == 0; }

// teams of the smallest power of two that covers a row with `unroll` accesses per thread, up to the whole block
RowGrid row_grid(long long tokens, int nvec, int unroll, unsigned* blocks) {
  RowGrid g{0, 1};
  while (g.team_log2 < 8 && (unroll << g.team_log2) < nvec) ++g.team_log2;
  const int per = unroll << g.team_log2;
  g.pieces = (nvec + per - 1) / per;
  const long long teams = kRowThreads >> g.team_log2;
  *blocks = (unsigned)((tokens * g.pieces + teams - 1) / teams);
  return g;
}

template <typename T, int VEC>
int permute_rows(const void* x, long long ldx, const int* slots, const int* kept, void* xp, long long tokens, int top_k, int hidden, cudaStream_t s) {
  unsigned blocks;
  const RowGrid g = row_grid(tokens, hidden / VEC, row_unroll(VEC), &blocks);
  moe_permute_kernel<T, VEC><<<blocks, kRowThreads, 0, s>>>(static_cast<const T*>(x), ldx, slots, kept, static_cast<T*>(xp), tokens, top_k, hidden / VEC, g);
  PKB_CHECK_CUDA(cudaGetLastError());
  return kApiOk;
}

template <typename T, int VEC>
int unpermute_rows(const void* y, long long ldy, const int* slots, const float* gates, void* out, long long tokens, int top_k, int hidden,
                   cudaStream_t s) {
  unsigned blocks;
  const RowGrid g = row_grid(tokens, hidden / VEC, gather_unroll(VEC), &blocks);
  const T* yp = static_cast<const T*>(y);
  T* op = static_cast<T*>(out);
  if (gates != nullptr) moe_unpermute_kernel<T, VEC, true><<<blocks, kRowThreads, 0, s>>>(yp, ldy, slots, gates, op, tokens, top_k, hidden / VEC, g);
  else moe_unpermute_kernel<T, VEC, false><<<blocks, kRowThreads, 0, s>>>(yp, ldy, slots, gates, op, tokens, top_k, hidden / VEC, g);
  PKB_CHECK_CUDA(cudaGetLastError());
  return kApiOk;
}

template <typename T, int VEC>
int unpermute_bwd_rows(const void* dout, long long lddo, const void* y, long long ldy, const int* slots, const float* gates, const int* kept,
                       void* dy, float* dgates, long long tokens, int top_k, int hidden, cudaStream_t s) {
  // a warp per token up to four accesses per lane (no barrier, eight tokens per block), else the block
  auto go = [&](auto kern, int teams) {
    kern<<<(unsigned)((tokens + teams - 1) / teams), kRowThreads, 0, s>>>(static_cast<const T*>(dout), lddo, static_cast<const T*>(y), ldy, slots, gates,
                                                                         kept, static_cast<T*>(dy), dgates, tokens, top_k, hidden / VEC);
  };
  if (hidden / VEC <= 128) go(moe_unpermute_bwd_kernel<T, VEC, 32>, kRowThreads / 32);
  else go(moe_unpermute_bwd_kernel<T, VEC, kRowThreads>, 1);
  PKB_CHECK_CUDA(cudaGetLastError());
  return kApiOk;
}

}  // namespace

}  // namespace pkb

using namespace pkb;

#define PKB_ROWS_ARGS()                                                                                                          \
  PKB_CHECK_ARG(tokens > 0 && top_k > 0 && hidden > 0 && tokens <= 0x7fffffffll / top_k, "1 .. 2^31 - 1 assignments of at least one column"); \
  PKB_CHECK_ARG(dtype == 0 || dtype == 1, "dtype must be 0 (bf16) or 1 (fp32)");                                                   \
  const int vec = dtype ? 4 : 8, esize = dtype ? 4 : 2;                                                                            \
  cudaStream_t s = static_cast<cudaStream_t>(stream)

// offsets [experts + 1], order [n], slots [n] (int32) of the n assignments idx (int32; values outside [0, experts) are dropped).
extern "C" int pkb_moe_sort(const void* idx, long long n, int experts, void* offsets, void* order, void* slots, void* stream) {
  PKB_CHECK_ARG(n > 0 && n <= 0x7fffffffll, "1 .. 2^31 - 1 assignments");
  PKB_CHECK_ARG(experts >= 1 && experts <= kSortMaxExperts, "1 .. 1024 experts");
  const long long rounds = (n + 31) / 32;
  const int smem = (int)(rounds < kSortWarps ? rounds : kSortWarps) * experts * (int)sizeof(int);
  if (const int rc = prepare_kernel<moe_sort_kernel>(kSortWarps * kSortMaxExperts * (int)sizeof(int), true)) return rc;
  const int ctas = n > 8192 ? kSortCluster : 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(kSortThreads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  PKB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, moe_sort_kernel, static_cast<const int*>(idx), (int)n, experts, static_cast<int*>(offsets),
                                    static_cast<int*>(order), static_cast<int*>(slots)));
  return kApiOk;
}

// xp [tokens * top_k, hidden] (contiguous) from x [tokens, hidden] (ldx elements between rows); kept: offsets[experts] on the device.
extern "C" int pkb_moe_permute(const void* x, long long ldx, const void* slots, const void* kept, void* xp, long long tokens, int top_k, int hidden,
                               int dtype, void* stream) {
  PKB_ROWS_ARGS();
  const bool v = hidden % vec == 0 && rows_aligned(x, ldx * esize) && rows_aligned(xp, 0);
  const int *sp = static_cast<const int*>(slots), *kp = static_cast<const int*>(kept);
  if (dtype) return v ? permute_rows<float, 4>(x, ldx, sp, kp, xp, tokens, top_k, hidden, s) : permute_rows<float, 1>(x, ldx, sp, kp, xp, tokens, top_k, hidden, s);
  return v ? permute_rows<__nv_bfloat16, 8>(x, ldx, sp, kp, xp, tokens, top_k, hidden, s)
           : permute_rows<__nv_bfloat16, 1>(x, ldx, sp, kp, xp, tokens, top_k, hidden, s);
}

// out [tokens, hidden] (contiguous) from y [tokens * top_k, hidden] (ldy elements between rows); gates fp32 [tokens, top_k] or null (ones).
extern "C" int pkb_moe_unpermute(const void* y, long long ldy, const void* slots, const void* gates, void* out, long long tokens, int top_k,
                                 int hidden, int dtype, void* stream) {
  PKB_ROWS_ARGS();
  const bool v = hidden % vec == 0 && rows_aligned(y, ldy * esize) && rows_aligned(out, 0);
  const int* sp = static_cast<const int*>(slots);
  const float* gp = static_cast<const float*>(gates);
  if (dtype) return v ? unpermute_rows<float, 4>(y, ldy, sp, gp, out, tokens, top_k, hidden, s) : unpermute_rows<float, 1>(y, ldy, sp, gp, out, tokens, top_k, hidden, s);
  return v ? unpermute_rows<__nv_bfloat16, 8>(y, ldy, sp, gp, out, tokens, top_k, hidden, s)
           : unpermute_rows<__nv_bfloat16, 1>(y, ldy, sp, gp, out, tokens, top_k, hidden, s);
}

// dy [tokens * top_k, hidden] (contiguous) and dgates fp32 [tokens, top_k] of pkb_moe_unpermute.
extern "C" int pkb_moe_unpermute_bwd(const void* dout, long long lddo, const void* y, long long ldy, const void* slots, const void* gates,
                                     const void* kept, void* dy, void* dgates, long long tokens, int top_k, int hidden, int dtype, void* stream) {
  PKB_ROWS_ARGS();
  PKB_CHECK_ARG(gates != nullptr, "the gradient of the weights needs the weights");
  const bool v = hidden % vec == 0 && rows_aligned(dout, lddo * esize) && rows_aligned(y, ldy * esize) && rows_aligned(dy, 0);
  const int *sp = static_cast<const int*>(slots), *kp = static_cast<const int*>(kept);
  const float* gp = static_cast<const float*>(gates);
  float* dg = static_cast<float*>(dgates);
  if (dtype)
    return v ? unpermute_bwd_rows<float, 4>(dout, lddo, y, ldy, sp, gp, kp, dy, dg, tokens, top_k, hidden, s)
             : unpermute_bwd_rows<float, 1>(dout, lddo, y, ldy, sp, gp, kp, dy, dg, tokens, top_k, hidden, s);
  return v ? unpermute_bwd_rows<__nv_bfloat16, 8>(dout, lddo, y, ldy, sp, gp, kp, dy, dg, tokens, top_k, hidden, s)
           : unpermute_bwd_rows<__nv_bfloat16, 1>(dout, lddo, y, ldy, sp, gp, kp, dy, dg, tokens, top_k, hidden, s);
}
