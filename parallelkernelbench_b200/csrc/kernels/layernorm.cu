// Layer norm, forward and backward (memory bound: a row is read once and stays in registers between its sums and its results).
//   mean = sum x / N, rstd = 1 / sqrt(sum (x - mean)^2 / N + eps), y = (x - mean) rstd gamma + beta
//   g = dy gamma, xhat = (x - mean) rstd, dx = rstd (g - mean(g) - xhat mean(g xhat)), dgamma = sum_rows dy xhat, dbeta = sum_rows dy
// Forward, a row's sum gives a first mean m0, rounded to fp32 like every value near it. From d = x - m0, which is small and nearly exact, come
// delta = sum d / N, mean = m0 + delta, variance = (sum d^2 - delta sum d) / N and y = (d - delta) rstd gamma + beta: with m0 alone a constant row of 1e5
// at 1000 columns (sum / N an ulp off) came out at -0.93 instead of 0. Never E[x^2] - mean^2.
// A row belongs to a team of TPR threads that holds VEC * CH of its values each: 16-byte accesses where base, row pitch and width
// allow them (VEC = 8 bf16 or 4 fp32), single values otherwise. All sums are fp32 (of rows in passes runs of 32, added in 64 bits).
// Forms, by width, alignment and number of rows (ln_fwd_any, ln_bwd_any): teams of 32 to 512 threads straight from global memory; from 1025 columns
// and a few hundred rows on, rings of rows in shared memory; rows that no team holds in passes; backward a few rows in one launch of a cluster.
// Measured, forward / backward with the weights' sums, us (of the copy bandwidth): 16384 x 8192 bf16 111 / 140 (74 % / 88 %), 8192 x 4096 33 / 45 (62 / 68),
// 16384 x 1000 19 / 25, 8192 x 4097 70 / 101, 8192 x 4097 fp32 73 / 104 (56 / 59). Of these 11 to 12 forward and 16 to 18 backward are start and end (launches,
// the first rows' way, the blocks' last rows, the weights' sums); what each further row adds at 4096 and 8192 columns is 89 and 82 % of the copy bandwidth
// forward and all of it backward (8192 to 65536 rows of 4096: 33, 57, 103, 195 us and 45, 75, 135, 254). A copy of 16384 x 8192 takes 84: what keeps the
// forward from it is not one thing (a warp per row without any barrier takes as long, prefetching further ahead takes longer).
#include "pkb/api.h"
#include "pkb/bulk_copy.cuh"
#include "pkb/host.h"
#include "pkb/ptx.cuh"

namespace pkb {

namespace {

// one row access: VEC values of type T at p as fp32, and back (rounded to nearest)
template <typename T, int VEC>
__device__ __forceinline__ void ln_load(const T* p, float (&f)[VEC]) {
  if constexpr (VEC == 1) f[0] = static_cast<float>(*p);
  else unpack16(ld_global_nc_v4(p), f);
}

// the same access as it is, for rows on their way
template <typename T, int VEC>
struct LnRaw {
  typename std::conditional<VEC == 1, T, U4>::type u;
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (VEC == 1) u = *p;
    else u = ld_global_nc_v4(p);
  }
  __device__ __forceinline__ void unpack(float (&f)[VEC]) const {
    if constexpr (VEC == 1) f[0] = static_cast<float>(u);
    else unpack16(u, f);
  }
};

template <typename T, int VEC>
__device__ __forceinline__ void ln_store(T* p, const float (&f)[VEC]) {
  if constexpr (VEC > 1) st_global_v4(p, pack16(f));
  else if constexpr (sizeof(T) == 2)
    *p = __float2bfloat16_rn(f[0]);
  else
    *p = f[0];
}

// The weights' kernel is launched while the last blocks of the backward still run (programmatic dependent launch) and waits for all of them.
__device__ __forceinline__ void ln_let_successor_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void ln_wait_for_predecessor() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// gain or bias: bf16 or fp32 whatever the rows are, or absent
struct LnParam {
  const void* p;
  int f32;
  float none;     // value where there is no tensor
  __device__ __forceinline__ float at(int c) const {
    if (p == nullptr) return none;
    return f32 ? static_cast<const float*>(p)[c] : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[c]);
  }
  // VEC consecutive ones from c on, c a multiple of VEC; 16-byte loads where VEC > 1 (the host checks the alignment)
  template <int VEC>
  __device__ __forceinline__ void load(int c, float (&f)[VEC]) const {
    if constexpr (VEC == 1) {
      f[0] = at(c);
    } else if (p == nullptr) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[j] = none;
    } else if (f32) {
#pragma unroll
      for (int j = 0; j < VEC; j += 4) {
        float q[4];
        unpack16(ld_global_v4(static_cast<const float*>(p) + c + j), q);
        f[j] = q[0]; f[j + 1] = q[1]; f[j + 2] = q[2]; f[j + 3] = q[3];
      }
    } else if constexpr (VEC == 8) {
      unpack16(ld_global_v4(static_cast<const __nv_bfloat16*>(p) + c), f);
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(p) + c);
      const float2 a = unpack_bf16x2(u.x), b = unpack_bf16x2(u.y);
      f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
    }
  }
};

// barrier of one team; a team of one warp needs none beyond the warp's own
template <int TPR, int NT>
__device__ __forceinline__ void team_sync(int team) {
  if constexpr (TPR == 32) __syncwarp();
  else if constexpr (TPR == NT) __syncthreads();
  else asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "n"(TPR) : "memory");
}

// Sums of K values over a team. `red` holds [K][NT / 32] floats; the caller alternates between two of them, so that a warp that is
// ahead never writes what another one still reads.
template <int K, int TPR, int NT>
__device__ __forceinline__ void team_sum(float (&v)[K], float* red, int team) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = warp_sum(v[k]);
  if constexpr (TPR > 32) {
    constexpr int W = TPR / 32;
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) red[k * (NT / 32) + warp] = v[k];
    }
    team_sync<TPR, NT>(team);
    // a lane takes one warp's sum and the lanes add them up: the same tree, and so the same bits, in every lane
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] = red[k * (NT / 32) + team * W + (threadIdx.x & (W - 1))];
#pragma unroll
      for (int o = W / 2; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
    }
  }
}

// The same for K = 2 or 4 with fewer shuffles (K = 4 over 16 warps: 13 instead of 36): the first exchanges halve the values that a lane still adds
// for, lane l ending up with value l / (32 / K), and a value's lanes share the warps' sums among them. 16384 x 8192 bf16 forward 121 us without, 111
// with, backward 143 and 140. (The backward kernels outside the aligned ring have no registers left for the exchanges: 8192 x 4097 bf16 101 and 113.)
template <int K, int TPR, int NT>
__device__ __forceinline__ void team_sum_shared(float (&v)[K], float* red, int team) {
  static_assert(K == 1 || K == 2 || K == 4, "values per lane");
  if constexpr (K == 1) {
    team_sum<1, TPR, NT>(v, red, team);
  } else {
    constexpr unsigned kAll = 0xffffffffu;
    constexpr int G = 32 / K;       // lanes per value
    const int lane = threadIdx.x & 31;
    const bool up = lane & 16;
    float s;
    if constexpr (K == 2) {
      s = (up ? v[1] : v[0]) + __shfl_xor_sync(kAll, up ? v[0] : v[1], 16);
      s += __shfl_xor_sync(kAll, s, 8);
    } else {
      const bool odd = lane & 8;
      const float a = (up ? v[2] : v[0]) + __shfl_xor_sync(kAll, up ? v[0] : v[2], 16);
      const float b = (up ? v[3] : v[1]) + __shfl_xor_sync(kAll, up ? v[1] : v[3], 16);
      s = (odd ? b : a) + __shfl_xor_sync(kAll, odd ? a : b, 8);
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) s += __shfl_xor_sync(kAll, s, o);
    if constexpr (TPR > 32) {
      constexpr int W = TPR / 32, S = W < G ? W : G;       // warps, lanes that add different warps' sums
      if (lane % G == 0) red[lane / G * (NT / 32) + (threadIdx.x >> 5)] = s;
      team_sync<TPR, NT>(team);
      const float* r = red + lane / G * (NT / 32) + team * W + lane % S;
      s = r[0];
#pragma unroll
      for (int i = S; i < W; i += S) s += r[i];
#pragma unroll
      for (int o = S / 2; o > 0; o >>= 1) s += __shfl_xor_sync(kAll, s, o);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = __shfl_sync(kAll, s, k * G);
  }
}

// A row's statistics from its first mean m0, the sum of its differences from it and the sum of their squares (see the top). The quotient is
// rounded once, so that it is exact where it can be: a constant row, whose differences are one number of a few bits, has no variance and nothing left
// of it. (With divisions here and for m0: 16384 x 8192 bf16 116 us instead of 111.)
struct LnStats {
  float delta, mean, rstd;
  __device__ __forceinline__ LnStats(float m0, float sum, float squares, int cols, float inv, float eps) {
    delta = div_rn_by(sum, (float)cols, inv);
    mean = m0 + delta;
    float q = fmaf(-sum, delta, squares);
    if (!(q >= 0.f)) q = isfinite(squares) ? 0.f : squares;      // rounding, or squares that left fp32
    rstd = rsqrtf(fmaf(q, inv, eps));
  }
};

template <typename T, int VEC, int TPR, int CH>
struct LnTeam {
  static constexpr int kThreads = TPR > 256 ? TPR : 256;
  static constexpr int kRows = kThreads / TPR;      // rows that a block has in hand
  static constexpr int kCols = TPR * VEC * CH;      // widest row
};

// (Single values: at most 64 registers, so that 1024 threads are resident: 16384 x 1001 bf16 38 us, 42 without.)
template <typename T, int VEC, int TPR, int CH>
__global__ void __launch_bounds__(LnTeam<T, VEC, TPR, CH>::kThreads, VEC == 1 ? 1024 / LnTeam<T, VEC, TPR, CH>::kThreads : 0)
ln_fwd_kernel(const T* __restrict__ x, long long ldx, const LnParam gamma, const LnParam beta, T* __restrict__ y,
              float* __restrict__ mean_out, float* __restrict__ rstd_out, long long rows, int cols, float eps) {
  using L = LnTeam<T, VEC, TPR, CH>;
  __shared__ float red[2][2 * (L::kThreads / 32)];
  const int team = threadIdx.x / TPR, t = threadIdx.x % TPR;
  const float inv = 1.f / (float)cols;
  for (long long row = (long long)blockIdx.x * L::kRows + team; row < rows; row += (long long)gridDim.x * L::kRows) {
    float v[CH][VEC];
    float s[1] = {0.f};
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) {
      const int c = (ch * TPR + t) * VEC;
      if (c < cols) {
        ln_load<T, VEC>(x + row * ldx + c, v[ch]);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[ch][j] = 0.f;
      }
    }
#pragma unroll
    for (int ch = 0; ch < CH; ++ch)
#pragma unroll
      for (int j = 0; j < VEC; ++j) s[0] += v[ch][j];
    team_sum<1, TPR, L::kThreads>(s, red[0], team);
    const float m0 = s[0] * inv;
    float q[2] = {0.f, 0.f};
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) {
      if ((ch * TPR + t) * VEC < cols) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          v[ch][j] -= m0;
          q[0] += v[ch][j];
          q[1] += v[ch][j] * v[ch][j];
        }
      }
    }
    team_sum_shared<2, TPR, L::kThreads>(q, red[1], team);
    const LnStats st(m0, q[0], q[1], cols, inv, eps);
    if (t == 0 && mean_out != nullptr) {
      mean_out[row] = st.mean;
      rstd_out[row] = st.rstd;
    }
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) {
      const int c = (ch * TPR + t) * VEC;
      if (c < cols) {
        float g[VEC], b[VEC];
        gamma.template load<VEC>(c, g);
        beta.template load<VEC>(c, b);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[ch][j] = (v[ch][j] - st.delta) * st.rstd * g[j] + b[j];
        ln_store<T, VEC>(y + row * cols + c, v[ch]);
      }
    }
  }
}

// Rows wider than a team holds: three passes over the row (the second and third come from L2), one block per row.
constexpr int kLnLongThreads = 512;
constexpr int kLnLongRun = 32;      // terms that a thread adds in fp32; runs are added in 64 bits, so that an error does not grow with the width

// sums of K terms per column over a row, by the whole block: add(column, sums) adds a column's. UNROLL > 1: that many columns at a time, each with its
// own check, which keeps more loads in flight where a column takes three of them (backward of 4096 x 15001 bf16 223 us, 265 with a loop up to the
// row's end; forward, with one load, 1000 x 50001 bf16 198 us as a loop, 209 with the checks).
template <int K, int UNROLL, typename F>
__device__ __forceinline__ void ln_long_sums(int cols, float (&sums)[K], float* red, F&& add) {
  double total[K] = {};
  for (int c0 = threadIdx.x; c0 < cols; c0 += kLnLongRun * kLnLongThreads) {
    float run[K] = {};
    if constexpr (UNROLL > 1) {
#pragma unroll UNROLL
      for (int j = 0; j < kLnLongRun; ++j) {
        const int c = c0 + j * kLnLongThreads;
        if (c < cols) add(c, run);
      }
    } else {
      const int end = min(cols, c0 + kLnLongRun * kLnLongThreads);
      for (int c = c0; c < end; c += kLnLongThreads) add(c, run);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) total[k] += (double)run[k];
  }
#pragma unroll
  for (int k = 0; k < K; ++k) sums[k] = (float)total[k];
  team_sum_shared<K, kLnLongThreads, kLnLongThreads>(sums, red, 0);
}

template <typename T>
__global__ void __launch_bounds__(kLnLongThreads)
ln_fwd_long_kernel(const T* __restrict__ x, long long ldx, const LnParam gamma, const LnParam beta, T* __restrict__ y,
                   float* __restrict__ mean_out, float* __restrict__ rstd_out, long long rows, int cols, float eps) {
  __shared__ float red[2][2 * (kLnLongThreads / 32)];
  const float inv = 1.f / (float)cols;
  for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + row * ldx;
    float s[1], q[2];
    ln_long_sums<1, 1>(cols, s, red[0], [&](int c, float (&run)[1]) { run[0] += static_cast<float>(xr[c]); });
    const float m0 = s[0] * inv;
    ln_long_sums<2, 1>(cols, q, red[1], [&](int c, float (&run)[2]) {
      const float d = static_cast<float>(xr[c]) - m0;
      run[0] += d;
      run[1] += d * d;
    });
    const LnStats st(m0, q[0], q[1], cols, inv, eps);
    if (threadIdx.x == 0 && mean_out != nullptr) {
      mean_out[row] = st.mean;
      rstd_out[row] = st.rstd;
    }
    for (int c = threadIdx.x; c < cols; c += kLnLongThreads) {
      const float f[1] = {((static_cast<float>(xr[c]) - m0) - st.delta) * st.rstd * gamma.at(c) + beta.at(c)};
      ln_store<T, 1>(y + row * cols + c, f);
    }
  }
}

constexpr int kLnCluster = 16;

// Backward. The blocks are persistent: a thread keeps its columns' sums of dy xhat and dy in registers over all rows of its block and
// writes them once, to part[block][2][cols]; ln_bwd_params_kernel adds the blocks' sums in a fixed order. The loads of a team's next
// row are issued before the sums of the current one.
// CLUSTER: all blocks are one cluster, which adds the blocks' sums itself through distributed shared memory and writes them to part[2][cols].
template <typename T, int VEC, int TPR, int CH, bool CLUSTER>
__global__ void __launch_bounds__(LnTeam<T, VEC, TPR, CH>::kThreads, 512 / LnTeam<T, VEC, TPR, CH>::kThreads)
ln_bwd_kernel(const T* __restrict__ x, long long ldx, const T* __restrict__ dy, long long lddy, const LnParam gamma,
              const float* __restrict__ mean_in, const float* __restrict__ rstd_in, T* __restrict__ dx, float* __restrict__ part,
              float* __restrict__ dgamma, float* __restrict__ dbeta, long long rows, int cols) {
  using L = LnTeam<T, VEC, TPR, CH>;
  __shared__ float red[2][2 * (L::kThreads / 32)];
  __shared__ float sums[L::kRows > 1 ? L::kRows * L::kCols : 1];
  const int team = threadIdx.x / TPR, t = threadIdx.x % TPR;
  const float inv = 1.f / (float)cols;
  float ag[CH][VEC] = {}, ab[CH][VEC] = {};
  float g[CH][VEC];
#pragma unroll
  for (int ch = 0; ch < CH; ++ch) {
    const int c = (ch * TPR + t) * VEC;
    if (c < cols) gamma.template load<VEC>(c, g[ch]);
  }
  LnRaw<T, VEC> xn[CH], dn[CH];
  float mean_n = 0.f, rstd_n = 0.f;
  auto fetch = [&](long long row) {
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) {
      const int c = (ch * TPR + t) * VEC;
      if (c < cols) {
        xn[ch].load(x + row * ldx + c);
        dn[ch].load(dy + row * lddy + c);
      }
    }
    mean_n = mean_in[row];
    rstd_n = rstd_in[row];
  };
  const long long step = (long long)gridDim.x * L::kRows;
  long long row = (long long)blockIdx.x * L::kRows + team;
  if (row < rows) fetch(row);
  for (int it = 0; row < rows; row += step, it ^= 1) {
    float xv[CH][VEC], dv[CH][VEC];
    const float mean = mean_n, rstd = rstd_n;
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) {
      xn[ch].unpack(xv[ch]);
      dn[ch].unpack(dv[ch]);
    }
    if (row + step < rows) fetch(row + step);
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) {
      if ((ch * TPR + t) * VEC < cols) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          xv[ch][j] = (xv[ch][j] - mean) * rstd;
          ag[ch][j] += dv[ch][j] * xv[ch][j];
          ab[ch][j] += dv[ch][j];
          dv[ch][j] *= g[ch][j];
          s[0] += dv[ch][j];
          s[1] += dv[ch][j] * xv[ch][j];
        }
      }
    }
    team_sum<2, TPR, L::kThreads>(s, red[it], team);
    const float c1 = s[0] * inv, c2 = s[1] * inv;
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) {
      const int c = (ch * TPR + t) * VEC;
      if (c < cols) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) dv[ch][j] = rstd * (dv[ch][j] - c1 - xv[ch][j] * c2);
        ln_store<T, VEC>(dx + row * cols + c, dv[ch]);
      }
    }
  }
  // the teams' sums, added in the order of the teams
  extern __shared__ float block_sums[];              // CLUSTER: [2][cols]
  if constexpr (!CLUSTER) ln_let_successor_launch();
  float* out = CLUSTER ? block_sums : part + (long long)blockIdx.x * 2 * cols;
  if constexpr (L::kRows == 1) {
#pragma unroll
    for (int ch = 0; ch < CH; ++ch)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int c = (ch * TPR + t) * VEC + j;
        if (c < cols) {
          out[c] = ag[ch][j];
          out[cols + c] = ab[ch][j];
        }
      }
  } else {
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int ch = 0; ch < CH; ++ch)
#pragma unroll
        for (int j = 0; j < VEC; ++j) sums[team * L::kCols + (ch * TPR + t) * VEC + j] = which == 0 ? ag[ch][j] : ab[ch][j];
      __syncthreads();
      for (int c = threadIdx.x; c < cols; c += L::kThreads) {
        float a = 0.f;
#pragma unroll
        for (int r = 0; r < L::kRows; ++r) a += sums[r * L::kCols + c];
        out[which * cols + c] = a;
      }
    }
  }
  if constexpr (CLUSTER) {
    cluster_sync_all();
    const int ctas = (int)cluster_nctaid();
    for (int i = (int)(cluster_ctarank() * L::kThreads + threadIdx.x); i < 2 * cols; i += ctas * L::kThreads) {
      const uint32_t at = smem_u32(block_sums + i);
      float v[kLnCluster];
#pragma unroll
      for (int c = 0; c < kLnCluster; ++c)
        if (c < ctas) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v[c]) : "r"(mapa_shared(at, (uint32_t)c)) : "memory");
      float a = 0.f;
#pragma unroll
      for (int c = 0; c < kLnCluster; ++c)
        if (c < ctas) a += v[c];
      if (i < cols) dgamma[i] = a;
      else dbeta[i - cols] = a;
    }
    cluster_sync_all();      // nobody leaves while its sums may still be read
  }
}

// ---- many wide rows: a ring of rows in shared memory --------------------------------------------
// A block of NT threads walks its rows with the next ones already on their way: thread 0 keeps bulk copies of up to kLnStages rows in flight
// (192 KB per SM over all blocks), so the memory system does not wait for a row's sums. With the loads in registers and one row ahead,
// 8192 x 4096 bf16 took 36 us forward and 59 backward, 16384 x 8192 took 142 and 237. A stage is free again once the block has passed the
// first barrier of its row: by then every thread holds its part in registers.
constexpr int kLnStages = 8;
constexpr int kLnRingBytes = 192 * 1024;                  // per SM
constexpr uint32_t kLnKernelId = 112;

struct LnRing {
  uint32_t base, bars, stage_bytes;
  int stages;
};

// Pairs of fp32 values in one register pair: Blackwell's packed adds, products and fused products halve the arithmetic, which with single
// values had the schedulers of 16 warps busy for 55 % (forward) and 67 % (backward) of the time at half of the memory bandwidth.
typedef unsigned long long F2;
__device__ __forceinline__ F2 f2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ F2 f2(float both) { return f2(both, both); }
__device__ __forceinline__ float2 f2_split(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
  return r;
}
__device__ __forceinline__ float f2_sum(F2 a) {
  const float2 r = f2_split(a);
  return r.x + r.y;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// 16 bytes as VEC / 2 pairs, and back (rounded to nearest)
template <int VEC>
__device__ __forceinline__ void ln_pairs(const U4& u, F2 (&f)[VEC / 2]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < VEC / 2; ++j)
    f[j] = VEC == 8 ? f2(__uint_as_float(w[j & 3] << 16), __uint_as_float(w[j & 3] & 0xffff0000u)) : f2(__uint_as_float(w[(2 * j) & 3]), __uint_as_float(w[(2 * j + 1) & 3]));
}
template <typename T, int VEC>
__device__ __forceinline__ void ln_store_pairs(T* p, const F2 (&f)[VEC / 2]) {
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < VEC / 2; ++j) {
    const float2 v = f2_split(f[j]);
    if constexpr (VEC == 8) {
      w[j] = pack_bf16x2(v.x, v.y);
    } else {
      w[2 * j] = __float_as_uint(v.x);
      w[2 * j + 1] = __float_as_uint(v.y);
    }
  }
  st_global_v4(p, U4{w[0], w[1], w[2], w[3]});
}
template <int VEC>
__device__ __forceinline__ void ln_param_pairs(const LnParam& p, int c, F2 (&f)[VEC / 2]) {
  float v[VEC];
  p.template load<VEC>(c, v);
#pragma unroll
  for (int j = 0; j < VEC / 2; ++j) f[j] = f2(v[2 * j], v[2 * j + 1]);
}
__device__ __forceinline__ U4 ln_shared(uint32_t a) {
  U4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}

__device__ __forceinline__ LnRing ln_ring_init(uint8_t* smem, int stages, uint32_t stage_bytes, int* abort_flag) {
  const LnRing r{smem_u32(smem) + 128, smem_u32(smem), stage_bytes, stages};
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int i = 0; i < stages; ++i) mbar_init(r.bars + 8 * i, 1);
    fence_mbar_init();
  }
  __syncthreads();
  return r;
}

// false once a row did not come within the budget. The block then walks its other rows without waiting (their results are of no use), so that
// nobody is missing at a barrier, copies nothing more, and leaves after what is in flight.
__device__ __forceinline__ bool ln_ring_wait(const LnRing& r, int stage, uint32_t parity, volatile int* abort_flag, uint32_t* status, long long row) {
  if (mbar_wait(r.bars + 8 * stage, parity, abort_flag)) return true;
  if (threadIdx.x == 0) record_status(status, kStatusMbarTimeout, kLnKernelId, 0, stage, 1, (uint32_t)row);
  return false;
}
__device__ __forceinline__ void ln_ring_leave(bool ok) {
  if (ok) return;
  const uint64_t t0 = globaltimer_ns();
  while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
}

// PER: values per thread; with 16 the gain and bias are held in registers, with 32 they are read again for every row. (Read for every row, from
// an L1 that the ring leaves little of, fp32 gains are twice the traffic of the rows: 8192 x 4096 took 40 us.)
// R rows at a time share the two barriers of their sums: with one, the latency of shuffles, shared memory and barriers left the schedulers idle
// for 56 % of the time (16384 x 8192: 116 us).
template <typename T, int NT, int PER, int R>
__global__ void __launch_bounds__(NT, 512 / NT)
ln_fwd_ring_kernel(const T* __restrict__ x, long long ldx, const LnParam gamma, const LnParam beta, T* __restrict__ y,
                   float* __restrict__ mean_out, float* __restrict__ rstd_out, long long rows, int cols, float eps, int stages, uint32_t* status) {
  constexpr int VEC = 16 / sizeof(T), CH = PER / VEC, P = VEC / 2;
  constexpr bool kHoldGain = PER <= 16;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float red[2][2 * R * (NT / 32)];
  __shared__ int abort_flag;
  const uint32_t bytes = (uint32_t)cols * sizeof(T);
  const LnRing ring = ln_ring_init(smem, stages, R * bytes, &abort_flag);
  const int t = threadIdx.x;
  const float inv = 1.f / (float)cols;
  const long long groups = (rows + R - 1) / R;        // of R rows, the last one maybe with fewer
  auto issue = [&](long long grp, int stage) {
    const uint32_t bar = ring.bars + 8 * stage;
    const int here = (int)min((long long)R, rows - grp * R);
    mbar_expect_tx(bar, here * bytes);
    for (int i = 0; i < here; ++i) bulk_load(ring.base + (stage * R + i) * bytes, x + (grp * R + i) * ldx, bytes, bar);
  };
  if (t == 0)
    for (int i = 0; i < stages; ++i)
      if (blockIdx.x + (long long)i * gridDim.x < groups) issue(blockIdx.x + (long long)i * gridDim.x, i);
  F2 g[kHoldGain ? CH : 1][P], b[kHoldGain ? CH : 1][P];
  if constexpr (kHoldGain) {
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) {
      const int c = (ch * NT + t) * VEC;
      if (c < cols) {
        ln_param_pairs<VEC>(gamma, c, g[ch]);
        ln_param_pairs<VEC>(beta, c, b[ch]);
      }
    }
  }
  int stage = 0;
  uint32_t parity = 0;
  bool ok = true;
  for (long long grp = blockIdx.x; grp < groups; grp += gridDim.x) {
    ok = ok && ln_ring_wait(ring, stage, parity, &abort_flag, status, grp);
    const int here = R == 1 ? 1 : (int)min((long long)R, rows - grp * R);
    F2 v[R][CH][P];
    float s[R], q[2 * R], rstd[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      F2 acc = 0;
#pragma unroll
      for (int ch = 0; ch < CH; ++ch) {
        const int c = (ch * NT + t) * VEC;
        if (c < cols) {       // (a row that is not there reads the stage's old bytes: they are not used)
          ln_pairs<VEC>(ln_shared(ring.base + (stage * R + i) * bytes + c * (int)sizeof(T)), v[i][ch]);
#pragma unroll
          for (int j = 0; j < P; ++j) acc = add2(acc, v[i][ch][j]);
        }
      }
      s[i] = f2_sum(acc);
    }
    team_sum_shared<R, NT, NT>(s, red[0], 0);
    if (t == 0 && ok && grp + (long long)stages * gridDim.x < groups) {
      fence_proxy_async_smem();
      issue(grp + (long long)stages * gridDim.x, stage);
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      s[i] *= inv;
      const F2 shift = f2(-s[i]);
      F2 sum = 0, squares = 0;
#pragma unroll
      for (int ch = 0; ch < CH; ++ch) {
        if ((ch * NT + t) * VEC < cols) {
#pragma unroll
          for (int j = 0; j < P; ++j) {
            v[i][ch][j] = add2(v[i][ch][j], shift);
            sum = add2(sum, v[i][ch][j]);
            squares = fma2(v[i][ch][j], v[i][ch][j], squares);
          }
        }
      }
      q[2 * i] = f2_sum(sum);
      q[2 * i + 1] = f2_sum(squares);
    }
    team_sum_shared<2 * R, NT, NT>(q, red[1], 0);
    F2 shift[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const LnStats st(s[i], q[2 * i], q[2 * i + 1], cols, inv, eps);
      rstd[i] = st.rstd;
      shift[i] = f2(-st.delta);
      if (t == 0 && i < here && mean_out != nullptr) {
        mean_out[grp * R + i] = st.mean;
        rstd_out[grp * R + i] = st.rstd;
      }
    }
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) {
      const int c = (ch * NT + t) * VEC;
      if (c < cols) {
        constexpr int kAt = kHoldGain ? 1 : 0;
        if constexpr (!kHoldGain) {
          ln_param_pairs<VEC>(gamma, c, g[0]);
          ln_param_pairs<VEC>(beta, c, b[0]);
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
          if (i < here) {
            const F2 r2 = f2(rstd[i]);
#pragma unroll
            for (int j = 0; j < P; ++j) v[i][ch][j] = fma2(mul2(add2(v[i][ch][j], shift[i]), r2), g[kAt * ch][j], b[kAt * ch][j]);
            ln_store_pairs<T, VEC>(y + (grp * R + i) * cols + c, v[i][ch]);
          }
        }
      }
    }
    if (++stage == stages) {
      stage = 0;
      parity ^= 1u;
    }
  }
  ln_ring_leave(ok);
}

// A stage holds a row of x and the same row of dy. PER as above; here only the gain is held.
template <typename T, int NT, int PER>
__global__ void __launch_bounds__(NT, 512 / NT)
ln_bwd_ring_kernel(const T* __restrict__ x, long long ldx, const T* __restrict__ dy, long long lddy, const LnParam gamma,
                   const float* __restrict__ mean_in, const float* __restrict__ rstd_in, T* __restrict__ dx, float* __restrict__ part,
                   long long rows, int cols, int stages, uint32_t* status) {
  constexpr int VEC = 16 / sizeof(T), CH = PER / VEC, P = VEC / 2;
  constexpr bool kHoldGain = PER <= 16;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float red[2][2 * (NT / 32)];
  __shared__ int abort_flag;
  const uint32_t bytes = (uint32_t)cols * sizeof(T);
  const LnRing ring = ln_ring_init(smem, stages, 2 * bytes, &abort_flag);
  const int t = threadIdx.x;
  const float inv = 1.f / (float)cols;
  auto issue = [&](long long row, int stage) {
    const uint32_t dst = ring.base + stage * 2 * bytes, bar = ring.bars + 8 * stage;
    mbar_expect_tx(bar, 2 * bytes);
    bulk_load(dst, x + row * ldx, bytes, bar);
    bulk_load(dst + bytes, dy + row * lddy, bytes, bar);
  };
  if (t == 0)
    for (int i = 0; i < stages; ++i)
      if (blockIdx.x + (long long)i * gridDim.x < rows) issue(blockIdx.x + (long long)i * gridDim.x, i);
  F2 ag[CH][P] = {}, ab[CH][P] = {};
  F2 g[kHoldGain ? CH : 1][P];
  if constexpr (kHoldGain) {
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) {
      const int c = (ch * NT + t) * VEC;
      if (c < cols) ln_param_pairs<VEC>(gamma, c, g[ch]);
    }
  }
  int stage = 0, it = 0;
  uint32_t parity = 0;
  bool ok = true;
  float mean_n = blockIdx.x < rows ? mean_in[blockIdx.x] : 0.f, rstd_n = blockIdx.x < rows ? rstd_in[blockIdx.x] : 0.f;
  for (long long row = blockIdx.x; row < rows; row += gridDim.x, it ^= 1) {
    const float mean = mean_n, rstd = rstd_n;
    if (row + gridDim.x < rows) {        // the next row's, a row ahead of their use
      mean_n = mean_in[row + gridDim.x];
      rstd_n = rstd_in[row + gridDim.x];
    }
    ok = ok && ln_ring_wait(ring, stage, parity, &abort_flag, status, row);
    const F2 shift = f2(-mean), r2 = f2(rstd);
    U4 xr[CH], dr[CH];
    F2 s1 = 0, s2 = 0;
    const uint32_t at = ring.base + stage * 2 * bytes;
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) {
      const int c = (ch * NT + t) * VEC;
      if (c < cols) {
        xr[ch] = ln_shared(at + c * (int)sizeof(T));
        dr[ch] = ln_shared(at + bytes + c * (int)sizeof(T));
        F2 xv[P], dv[P];
        ln_pairs<VEC>(xr[ch], xv);
        ln_pairs<VEC>(dr[ch], dv);
        if constexpr (!kHoldGain) ln_param_pairs<VEC>(gamma, c, g[0]);
#pragma unroll
        for (int j = 0; j < P; ++j) {
          const F2 xh = mul2(add2(xv[j], shift), r2), gd = mul2(dv[j], g[kHoldGain ? ch : 0][j]);
          ag[ch][j] = fma2(dv[j], xh, ag[ch][j]);
          ab[ch][j] = add2(dv[j], ab[ch][j]);
          s1 = add2(gd, s1);
          s2 = fma2(gd, xh, s2);
        }
      }
    }
    float s[2] = {f2_sum(s1), f2_sum(s2)};
    team_sum_shared<2, NT, NT>(s, red[it], 0);
    if (t == 0 && ok && row + (long long)stages * gridDim.x < rows) {
      fence_proxy_async_smem();
      issue(row + (long long)stages * gridDim.x, stage);
    }
    // rstd (g dy - c1 - xhat c2)
    const F2 c1 = f2(-s[0] * inv * rstd), c2 = f2(-s[1] * inv * rstd);
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) {
      const int c = (ch * NT + t) * VEC;
      if (c < cols) {
        F2 xv[P], dv[P];
        ln_pairs<VEC>(xr[ch], xv);
        ln_pairs<VEC>(dr[ch], dv);
        if constexpr (!kHoldGain) ln_param_pairs<VEC>(gamma, c, g[0]);
#pragma unroll
        for (int j = 0; j < P; ++j) {
          const F2 xh = mul2(add2(xv[j], shift), r2), gd = mul2(dv[j], g[kHoldGain ? ch : 0][j]);
          dv[j] = fma2(xh, c2, fma2(gd, r2, c1));
        }
        ln_store_pairs<T, VEC>(dx + row * cols + c, dv);
      }
    }
    if (++stage == stages) {
      stage = 0;
      parity ^= 1u;
    }
  }
  ln_let_successor_launch();
  float* out = part + (long long)blockIdx.x * 2 * cols;
#pragma unroll
  for (int ch = 0; ch < CH; ++ch) {
    const int c = (ch * NT + t) * VEC;
    if (c < cols) {
#pragma unroll
      for (int j = 0; j < P; j += 2) {
        *reinterpret_cast<ulonglong2*>(out + c + 2 * j) = make_ulonglong2(ag[ch][j], ag[ch][j + 1]);
        *reinterpret_cast<ulonglong2*>(out + cols + c + 2 * j) = make_ulonglong2(ab[ch][j], ab[ch][j + 1]);
      }
    }
  }
  ln_ring_leave(ok);
}

// ---- many wide rows that do not start on 16 bytes -------------------------------------------------
// The same ring for rows of any width, pitch and address. A bulk copy moves whole 16-byte pieces, so a row comes with up to 15 bytes of its
// neighbours on either side, and its values lie at their own address modulo 16. No piece is copied that reaches outside the tensor (from its first
// row's first to its last row's last value): the few values that this leaves out, in the first and last row, are read where they are used.
// A thread owns the columns t, t + NT, ...: 4- and 2-byte accesses of shared and global memory, 32 neighbours per warp. Against the team form,
// which takes such rows straight from global memory, us forward / backward: 8192 x 4097 bf16 93 / 191 there.
struct LnSpan {
  uintptr_t first, last;          // the tensor's bytes
  __device__ __forceinline__ LnSpan(const void* base, long long pitch_bytes, long long rows, uint32_t row_bytes)
      : first(reinterpret_cast<uintptr_t>(base)), last(first + (rows - 1) * pitch_bytes + row_bytes) {}
  // the part of a row's pieces that may be copied; `at`: the address that the stage's first byte stands for
  __device__ __forceinline__ void pieces(uintptr_t row, uint32_t row_bytes, uintptr_t& at, uintptr_t& lo, uintptr_t& hi) const {
    at = row & ~(uintptr_t)15;
    lo = at < first ? at + 16 : at;
    hi = (row + row_bytes + 15) & ~(uintptr_t)15;
    if (hi > last) hi -= 16;
  }
};

// one value at a shared-memory address
template <typename T>
__device__ __forceinline__ float odd_shared(uint32_t a) {
  if constexpr (sizeof(T) == 2) {
    uint16_t u;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(u) : "r"(a) : "memory");
    return __uint_as_float((uint32_t)u << 16);
  } else {
    float f;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(f) : "r"(a) : "memory");
    return f;
  }
}

// A row in its stage. Pair j of a thread is columns (2 j NT + t, (2 j + 1) NT + t), `none` where there is no column: the row's mean in the backward, so
// that xhat is zero there whatever the row's size and deviation (0 - mean may leave fp32 when it is multiplied with rstd).
template <typename T, int NT>
struct LnOddRow {
  const T* global;                // the row
  uint32_t shared;                // where its first value would be in the stage
  int from, to;                   // columns that are there
  __device__ __forceinline__ float one(int c) const { return c >= from && c < to ? odd_shared<T>(shared + c * (int)sizeof(T)) : static_cast<float>(global[c]); }
  template <int P>
  __device__ __forceinline__ void load(F2 (&v)[P], int cols, float none = 0.f) const {
    const int t = threadIdx.x;
    if (from == 0 && to >= cols) {          // all rows but the tensor's first and last
      const uint32_t at = shared + t * (int)sizeof(T);
#pragma unroll
      for (int j = 0; j < P; ++j) {
        float lo = none, hi = none;
        if ((2 * j + 1) * NT <= cols || 2 * j * NT + t < cols) lo = odd_shared<T>(at + 2 * j * NT * (int)sizeof(T));
        if ((2 * j + 2) * NT <= cols || (2 * j + 1) * NT + t < cols) hi = odd_shared<T>(at + (2 * j + 1) * NT * (int)sizeof(T));
        v[j] = f2(lo, hi);
      }
    } else {
#pragma unroll
      for (int j = 0; j < P; ++j) {
        const int c0 = 2 * j * NT + t, c1 = c0 + NT;
        v[j] = f2(c0 < cols ? one(c0) : none, c1 < cols ? one(c1) : none);
      }
    }
  }
};

// the pairs of a row, rounded to its type
template <typename T, int NT, int P>
__device__ __forceinline__ void odd_store(T* row, int j, F2 v, int cols) {
  const int t = threadIdx.x;
  const float2 w = f2_split(v);
  const float lo[1] = {w.x}, hi[1] = {w.y};
  if ((2 * j + 1) * NT <= cols || 2 * j * NT + t < cols) ln_store<T, 1>(row + t + 2 * j * NT, lo);
  if ((2 * j + 2) * NT <= cols || (2 * j + 1) * NT + t < cols) ln_store<T, 1>(row + t + (2 * j + 1) * NT, hi);
}

template <typename T>
__device__ __forceinline__ void odd_issue(const LnSpan& span, const T* row, uint32_t row_bytes, uint32_t dst, uint32_t bar) {
  uintptr_t at, lo, hi;
  span.pieces(reinterpret_cast<uintptr_t>(row), row_bytes, at, lo, hi);
  bulk_load(dst + (uint32_t)(lo - at), reinterpret_cast<const void*>(lo), (uint32_t)(hi - lo), bar);
}
template <typename T>
__device__ __forceinline__ uint32_t odd_bytes(const LnSpan& span, const T* row, uint32_t row_bytes) {
  uintptr_t at, lo, hi;
  span.pieces(reinterpret_cast<uintptr_t>(row), row_bytes, at, lo, hi);
  return (uint32_t)(hi - lo);
}
template <int NT, typename T>
__device__ __forceinline__ LnOddRow<T, NT> odd_row(const LnSpan& span, const T* row, uint32_t row_bytes, uint32_t stage) {
  uintptr_t at, lo, hi;
  const uintptr_t a = reinterpret_cast<uintptr_t>(row);
  span.pieces(a, row_bytes, at, lo, hi);
  return {row, stage + (uint32_t)(a - at), lo > a ? (int)((lo - a) / sizeof(T)) : 0, (int)((hi - a) / sizeof(T))};
}

template <typename T, int NT, int PER, int R>
__global__ void __launch_bounds__(NT, 512 / NT)
ln_fwd_odd_kernel(const T* __restrict__ x, long long ldx, const LnParam gamma, const LnParam beta, T* __restrict__ y,
                  float* __restrict__ mean_out, float* __restrict__ rstd_out, long long rows, int cols, float eps, int stages, uint32_t row_stage,
                  uint32_t* status) {
  constexpr int P = PER / 2;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float red[2][2 * R * (NT / 32)];
  __shared__ int abort_flag;
  const uint32_t bytes = (uint32_t)cols * sizeof(T);
  const LnRing ring = ln_ring_init(smem, stages, R * row_stage, &abort_flag);
  const LnSpan span(x, ldx * (long long)sizeof(T), rows, bytes);
  const int t = threadIdx.x;
  const float inv = 1.f / (float)cols;
  const long long groups = (rows + R - 1) / R;
  auto issue = [&](long long grp, int stage) {
    const uint32_t bar = ring.bars + 8 * stage;
    const int here = (int)min((long long)R, rows - grp * R);
    uint32_t all = 0;
    for (int i = 0; i < here; ++i) all += odd_bytes(span, x + (grp * R + i) * ldx, bytes);
    mbar_expect_tx(bar, all);
    for (int i = 0; i < here; ++i) odd_issue(span, x + (grp * R + i) * ldx, bytes, ring.base + (stage * R + i) * row_stage, bar);
  };
  if (t == 0)
    for (int i = 0; i < stages; ++i)
      if (blockIdx.x + (long long)i * gridDim.x < groups) issue(blockIdx.x + (long long)i * gridDim.x, i);
  auto col = [&](int k) { return k * NT + t; };
  auto gains = [&](const LnParam& p, int j) { return f2(col(2 * j) < cols ? p.at(col(2 * j)) : 0.f, col(2 * j + 1) < cols ? p.at(col(2 * j + 1)) : 0.f); };
  F2 g[P], b[P];
#pragma unroll
  for (int j = 0; j < P; ++j) {
    g[j] = gains(gamma, j);
    b[j] = gains(beta, j);
  }
  int stage = 0;
  uint32_t parity = 0;
  bool ok = true;
  for (long long grp = blockIdx.x; grp < groups; grp += gridDim.x) {
    ok = ok && ln_ring_wait(ring, stage, parity, &abort_flag, status, grp);
    const int here = R == 1 ? 1 : (int)min((long long)R, rows - grp * R);
    F2 v[R][P];
    float s[R] = {}, q[2 * R] = {};
#pragma unroll
    for (int i = 0; i < R; ++i) {
      F2 acc = 0;
      if (i < here) {
        odd_row<NT>(span, x + (grp * R + i) * ldx, bytes, ring.base + (stage * R + i) * row_stage).load(v[i], cols);
#pragma unroll
        for (int j = 0; j < P; ++j) acc = add2(acc, v[i][j]);
      }
      s[i] = f2_sum(acc);
    }
    team_sum_shared<R, NT, NT>(s, red[0], 0);
    if (t == 0 && ok && grp + (long long)stages * gridDim.x < groups) {
      fence_proxy_async_smem();
      issue(grp + (long long)stages * gridDim.x, stage);
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      s[i] *= inv;
      const F2 shift = f2(-s[i]);
      F2 sum = 0, squares = 0;
#pragma unroll
      for (int j = 0; j < P; ++j) {
        v[i][j] = add2(v[i][j], shift);
        if ((2 * j + 2) * NT > cols) {        // columns that are not there count nothing
          const float2 w = f2_split(v[i][j]);
          v[i][j] = f2(col(2 * j) < cols ? w.x : 0.f, col(2 * j + 1) < cols ? w.y : 0.f);
        }
        sum = add2(sum, v[i][j]);
        squares = fma2(v[i][j], v[i][j], squares);
      }
      q[2 * i] = f2_sum(sum);
      q[2 * i + 1] = f2_sum(squares);
    }
    team_sum_shared<2 * R, NT, NT>(q, red[1], 0);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (i >= here) break;
      const LnStats st(s[i], q[2 * i], q[2 * i + 1], cols, inv, eps);
      if (t == 0 && mean_out != nullptr) {
        mean_out[grp * R + i] = st.mean;
        rstd_out[grp * R + i] = st.rstd;
      }
      const F2 r2 = f2(st.rstd), shift = f2(-st.delta);
      T* yr = y + (grp * R + i) * cols;
#pragma unroll
      for (int j = 0; j < P; ++j) odd_store<T, NT, P>(yr, j, fma2(mul2(add2(v[i][j], shift), r2), g[j], b[j]), cols);
    }
    if (++stage == stages) {
      stage = 0;
      parity ^= 1u;
    }
  }
  ln_ring_leave(ok);
}

// Both passes over a row read it from its stage (the registers hold the weights' sums), which is therefore free only after the next row's barrier.
template <typename T, int NT, int PER>
__global__ void __launch_bounds__(NT, 512 / NT)
ln_bwd_odd_kernel(const T* __restrict__ x, long long ldx, const T* __restrict__ dy, long long lddy, const LnParam gamma,
                  const float* __restrict__ mean_in, const float* __restrict__ rstd_in, T* __restrict__ dx, float* __restrict__ part,
                  long long rows, int cols, int stages, uint32_t row_stage, uint32_t* status) {
  constexpr int P = PER / 2;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float red[2][2 * (NT / 32)];
  __shared__ int abort_flag;
  const uint32_t bytes = (uint32_t)cols * sizeof(T);
  const LnRing ring = ln_ring_init(smem, stages, 2 * row_stage, &abort_flag);
  const LnSpan span_x(x, ldx * (long long)sizeof(T), rows, bytes), span_d(dy, lddy * (long long)sizeof(T), rows, bytes);
  const int t = threadIdx.x;
  const float inv = 1.f / (float)cols;
  auto issue = [&](long long row, int stage) {
    const uint32_t dst = ring.base + stage * 2 * row_stage, bar = ring.bars + 8 * stage;
    mbar_expect_tx(bar, odd_bytes(span_x, x + row * ldx, bytes) + odd_bytes(span_d, dy + row * lddy, bytes));
    odd_issue(span_x, x + row * ldx, bytes, dst, bar);
    odd_issue(span_d, dy + row * lddy, bytes, dst + row_stage, bar);
  };
  if (t == 0)
    for (int i = 0; i < stages; ++i)
      if (blockIdx.x + (long long)i * gridDim.x < rows) issue(blockIdx.x + (long long)i * gridDim.x, i);
  auto col = [&](int k) { return k * NT + t; };
  auto gains = [&](int j) { return f2(col(2 * j) < cols ? gamma.at(col(2 * j)) : 0.f, col(2 * j + 1) < cols ? gamma.at(col(2 * j + 1)) : 0.f); };
  F2 ag[P] = {}, ab[P] = {};
  F2 g[P];
#pragma unroll
  for (int j = 0; j < P; ++j) g[j] = gains(j);
  int stage = 0, before = -1, it = 0;
  uint32_t parity = 0;
  bool ok = true;
  float mean_n = blockIdx.x < rows ? mean_in[blockIdx.x] : 0.f, rstd_n = blockIdx.x < rows ? rstd_in[blockIdx.x] : 0.f;
  for (long long row = blockIdx.x; row < rows; row += gridDim.x, it ^= 1) {
    const float mean = mean_n, rstd = rstd_n;
    if (row + gridDim.x < rows) {
      mean_n = mean_in[row + gridDim.x];
      rstd_n = rstd_in[row + gridDim.x];
    }
    ok = ok && ln_ring_wait(ring, stage, parity, &abort_flag, status, row);
    const uint32_t at = ring.base + stage * 2 * row_stage;
    const LnOddRow<T, NT> xr = odd_row<NT>(span_x, x + row * ldx, bytes, at), dr = odd_row<NT>(span_d, dy + row * lddy, bytes, at + row_stage);
    const F2 shift = f2(-mean), r2 = f2(rstd);
    F2 s1 = 0, s2 = 0, xv[P], dv[P];
    xr.load(xv, cols, mean);
    dr.load(dv, cols);
#pragma unroll
    for (int j = 0; j < P; ++j) {
      // (dy, the gain and xhat are zero where there is no column)
      const F2 xh = mul2(add2(xv[j], shift), r2), gd = mul2(dv[j], g[j]);
      ag[j] = fma2(dv[j], xh, ag[j]);
      ab[j] = add2(dv[j], ab[j]);
      s1 = add2(gd, s1);
      s2 = fma2(gd, xh, s2);
    }
    float s[2] = {f2_sum(s1), f2_sum(s2)};
    team_sum<2, NT, NT>(s, red[it], 0);
    const long long ahead = row + (long long)(stages - 1) * gridDim.x;
    if (t == 0 && ok && before >= 0 && ahead < rows) {
      fence_proxy_async_smem();
      issue(ahead, before);
    }
    const F2 c1 = f2(-s[0] * inv * rstd), c2 = f2(-s[1] * inv * rstd);
    T* out = dx + row * cols;
    xr.load(xv, cols, mean);
    dr.load(dv, cols);
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const F2 xh = mul2(add2(xv[j], shift), r2), gd = mul2(dv[j], g[j]);
      odd_store<T, NT, P>(out, j, fma2(xh, c2, fma2(gd, r2, c1)), cols);
    }
    before = stage;
    if (++stage == stages) {
      stage = 0;
      parity ^= 1u;
    }
  }
  ln_let_successor_launch();
  float* out = part + (long long)blockIdx.x * 2 * cols;
#pragma unroll
  for (int j = 0; j < P; ++j) {
    const float2 a = f2_split(ag[j]), b = f2_split(ab[j]);
    if (col(2 * j) < cols) {
      out[col(2 * j)] = a.x;
      out[cols + col(2 * j)] = b.x;
    }
    if (col(2 * j + 1) < cols) {
      out[col(2 * j + 1)] = a.y;
      out[cols + col(2 * j + 1)] = b.y;
    }
  }
  ln_ring_leave(ok);
}

// dgamma, dbeta [2][cols] = sum over the blocks of part[block][2][cols]: 32 columns and 32 strands of blocks per thread block
__global__ void __launch_bounds__(1024)
ln_bwd_params_kernel(const float* __restrict__ part, int blocks, long long width, float* __restrict__ dgamma, float* __restrict__ dbeta, int cols) {
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, strand = threadIdx.x >> 5;
  const long long i = (long long)blockIdx.x * 32 + lane;
  float a = 0.f;
  ln_wait_for_predecessor();
  if (i < width) {
#pragma unroll 8
    for (int b = strand; b < blocks; b += 32) a += part[b * width + i];
  }
  s[strand][lane] = a;
  __syncthreads();
  a = warp_sum(s[lane][strand]);           // warp w adds the strands of column w
  const long long o = (long long)blockIdx.x * 32 + strand;
  if (lane == 0 && o < width) {
    if (o < cols) dgamma[o] = a;
    else dbeta[o - cols] = a;
  }
}

// Rows wider than a team holds: dx from two passes over a row, and the weight's sums by blocks of 64 columns and a slice of the rows.
template <typename T>
__global__ void __launch_bounds__(kLnLongThreads)
ln_bwd_long_dx_kernel(const T* __restrict__ x, long long ldx, const T* __restrict__ dy, long long lddy, const LnParam gamma,
                      const float* __restrict__ mean_in, const float* __restrict__ rstd_in, T* __restrict__ dx, long long rows, int cols) {
  __shared__ float red[2][2 * (kLnLongThreads / 32)];
  const float inv = 1.f / (float)cols;
  int it = 0;
  for (long long row = blockIdx.x; row < rows; row += gridDim.x, it ^= 1) {
    const T *xr = x + row * ldx, *dr = dy + row * lddy;
    const float mean = mean_in[row], rstd = rstd_in[row];
    float s[2];
    ln_long_sums<2, 8>(cols, s, red[it], [&](int c, float (&run)[2]) {
      const float gd = static_cast<float>(dr[c]) * gamma.at(c);
      run[0] += gd;
      run[1] += gd * ((static_cast<float>(xr[c]) - mean) * rstd);
    });
    const float c1 = s[0] * inv, c2 = s[1] * inv;
    for (int c = threadIdx.x; c < cols; c += kLnLongThreads) {
      const float gd = static_cast<float>(dr[c]) * gamma.at(c), xh = (static_cast<float>(xr[c]) - mean) * rstd;
      const float f[1] = {rstd * (gd - c1 - xh * c2)};
      ln_store<T, 1>(dx + row * cols + c, f);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256)
ln_bwd_long_params_kernel(const T* __restrict__ x, long long ldx, const T* __restrict__ dy, long long lddy, const float* __restrict__ mean_in,
                          const float* __restrict__ rstd_in, float* __restrict__ part, long long rows, int cols) {
  __shared__ float s[2][4][64];
  const int lane = threadIdx.x & 63, strand = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + lane;
  float a = 0.f, b = 0.f;
  if (c < cols) {
    for (long long r = (long long)blockIdx.y * 4 + strand; r < rows; r += (long long)gridDim.y * 4) {
      const float d = static_cast<float>(dy[r * lddy + c]);
      a += d * ((static_cast<float>(x[r * ldx + c]) - mean_in[r]) * rstd_in[r]);
      b += d;
    }
  }
  s[0][strand][lane] = a;
  s[1][strand][lane] = b;
  __syncthreads();
  if (strand < 2 && c < cols) {
    const float t = s[strand][0][lane] + s[strand][1][lane] + s[strand][2][lane] + s[strand][3][lane];
    part[((long long)blockIdx.y * 2 + strand) * cols + c] = t;
  }
}

constexpr int kLnLongSlices = 64;    // row slices of the long form's weight sums

// the widest row of the team forms: 16 values per thread, 512 threads
constexpr int kLnTeamCols = 512 * 16;

bool ln_aligned(const void* p, long long pitch_bytes) { return ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)pitch_bytes) & 15) == 0; }

template <typename F, typename T, int VEC, bool BACKWARD>
int ln_by_width(int cols, F&& f) {
  // 16 values per thread, 2 (bf16) or 4 (fp32) accesses of 16 bytes or 16 single ones. Forward a warp takes rows of up to 1024 with twice as many;
  // backward the sums for the weights leave no registers for that.
  constexpr int CH = 16 / VEC;
  using One = std::integral_constant<int, CH>;
  if (cols <= 32 * 16) return f(std::integral_constant<int, 32>{}, One{});
  if constexpr (BACKWARD) {
    if (cols <= 64 * 16) return f(std::integral_constant<int, 64>{}, One{});
  } else if constexpr (VEC > 1) {
    if (cols <= 32 * 32) return f(std::integral_constant<int, 32>{}, std::integral_constant<int, 2 * CH>{});
  } else {
    if (cols <= 64 * 16) return f(std::integral_constant<int, 64>{}, One{});
  }
  if (cols <= 128 * 16) return f(std::integral_constant<int, 128>{}, One{});
  if (cols <= 256 * 16) return f(std::integral_constant<int, 256>{}, One{});
  return f(std::integral_constant<int, 512>{}, One{});
}

template <typename T, int VEC>
int ln_fwd_team(const T* x, long long ldx, LnParam g, LnParam b, T* y, float* mean, float* rstd, long long rows, int cols, float eps,
                cudaStream_t s) {
  auto go = [&](auto tpr, auto ch) -> int {
    using L = LnTeam<T, VEC, tpr.value, ch.value>;
    long long grid = (rows + L::kRows - 1) / L::kRows;
    const long long most = (long long)sm_count() * (2048 / L::kThreads);
    if (grid > most) grid = most;
    ln_fwd_kernel<T, VEC, tpr.value, ch.value><<<(unsigned)grid, L::kThreads, 0, s>>>(x, ldx, g, b, y, mean, rstd, rows, cols, eps);
    PKB_CHECK_CUDA(cudaGetLastError());
    return kApiOk;
  };
  return ln_by_width<decltype(go)&, T, VEC, false>(cols, go);
}

// The rings take over from 1025 columns on (teams of a warp have enough rows in flight) where every block has more than two rows: up to 16384
// columns, up to 8192 backward in fp32 and where rows start anywhere (with 32 single values per thread 4096 x 15001 bf16 took 222 us forward and
// 429 backward, the long form 212 and 231).
template <auto KERN>
struct KernelAt {
  static constexpr auto value = KERN;
};

struct LnRingPlan {
  int threads, per, together, blocks, stages, row_stage, smem;
};
// aligned: rows are whole multiples of 16 bytes that start on 16 bytes
bool ln_ring_plan(LnRingPlan& r, long long rows, int cols, int esize, bool backward, bool aligned, int sms) {
  if (cols <= 1024 || cols > (!aligned || (backward && esize == 4) ? 8192 : 16384)) return false;
  r.threads = cols <= 2048 ? 128 : cols <= 4096 ? 256 : 512;
  r.per = cols > 8192 ? 32 : !aligned && cols <= 10 * r.threads ? 10 : 16;
  const int per_sm = 512 / r.threads;
  r.blocks = sms * per_sm;
  r.together = !backward && r.per <= 16 ? 2 : 1;
  r.row_stage = aligned ? cols * esize : (cols * esize + 15) / 16 * 16 + 16;
  const int stage = r.row_stage * (backward ? 2 : r.together);
  r.stages = kLnRingBytes / per_sm / stage;
  if (r.stages > kLnStages) r.stages = kLnStages;
  r.smem = 128 + r.stages * stage;
  return r.stages >= 2 && rows > 2ll * r.blocks * r.together;
}

template <typename T>
int ln_fwd_ring(const LnRingPlan& r, const T* x, long long ldx, LnParam g, LnParam b, T* y, float* mean, float* rstd, long long rows, int cols,
                float eps, cudaStream_t s) {
  auto go = [&](auto at) -> int {
    constexpr auto kern = decltype(at)::value;
    if (const int rc = prepare_kernel<kern>(128 + kLnRingBytes)) return rc;
    kern<<<r.blocks, r.threads, r.smem, s>>>(x, ldx, g, b, y, mean, rstd, rows, cols, eps, r.stages, status_block_for_launch());
    PKB_CHECK_CUDA(cudaGetLastError());
    return kApiOk;
  };
  if (r.threads == 128) return go(KernelAt<ln_fwd_ring_kernel<T, 128, 16, 2>>{});
  if (r.threads == 256) return go(KernelAt<ln_fwd_ring_kernel<T, 256, 16, 2>>{});
  if (r.per == 16) return go(KernelAt<ln_fwd_ring_kernel<T, 512, 16, 2>>{});
  return go(KernelAt<ln_fwd_ring_kernel<T, 512, 32, 1>>{});
}

template <typename T>
int ln_fwd_odd(const LnRingPlan& r, const T* x, long long ldx, LnParam g, LnParam b, T* y, float* mean, float* rstd, long long rows, int cols,
               float eps, cudaStream_t s) {
  auto go = [&](auto at) -> int {
    constexpr auto kern = decltype(at)::value;
    if (const int rc = prepare_kernel<kern>(128 + kLnRingBytes)) return rc;
    kern<<<r.blocks, r.threads, r.smem, s>>>(x, ldx, g, b, y, mean, rstd, rows, cols, eps, r.stages, (uint32_t)r.row_stage, status_block_for_launch());
    PKB_CHECK_CUDA(cudaGetLastError());
    return kApiOk;
  };
  if (r.per == 10) {
    if (r.threads == 128) return go(KernelAt<ln_fwd_odd_kernel<T, 128, 10, 2>>{});
    if (r.threads == 256) return go(KernelAt<ln_fwd_odd_kernel<T, 256, 10, 2>>{});
    return go(KernelAt<ln_fwd_odd_kernel<T, 512, 10, 2>>{});
  }
  if (r.threads == 128) return go(KernelAt<ln_fwd_odd_kernel<T, 128, 16, 2>>{});
  if (r.threads == 256) return go(KernelAt<ln_fwd_odd_kernel<T, 256, 16, 2>>{});
  return go(KernelAt<ln_fwd_odd_kernel<T, 512, 16, 2>>{});
}

template <typename T>
int ln_bwd_odd(const LnRingPlan& r, const T* x, long long ldx, const T* dy, long long lddy, LnParam g, const float* mean, const float* rstd,
               T* dx, float* part, long long rows, int cols, cudaStream_t s) {
  auto go = [&](auto at) -> int {
    constexpr auto kern = decltype(at)::value;
    if (const int rc = prepare_kernel<kern>(128 + kLnRingBytes)) return rc;
    kern<<<r.blocks, r.threads, r.smem, s>>>(x, ldx, dy, lddy, g, mean, rstd, dx, part, rows, cols, r.stages, (uint32_t)r.row_stage,
                                             status_block_for_launch());
    PKB_CHECK_CUDA(cudaGetLastError());
    return kApiOk;
  };
  if (r.per == 10) {
    if (r.threads == 128) return go(KernelAt<ln_bwd_odd_kernel<T, 128, 10>>{});
    if (r.threads == 256) return go(KernelAt<ln_bwd_odd_kernel<T, 256, 10>>{});
    return go(KernelAt<ln_bwd_odd_kernel<T, 512, 10>>{});
  }
  if (r.threads == 128) return go(KernelAt<ln_bwd_odd_kernel<T, 128, 16>>{});
  if (r.threads == 256) return go(KernelAt<ln_bwd_odd_kernel<T, 256, 16>>{});
  return go(KernelAt<ln_bwd_odd_kernel<T, 512, 16>>{});
}

template <typename T>
int ln_bwd_ring(const LnRingPlan& r, const T* x, long long ldx, const T* dy, long long lddy, LnParam g, const float* mean, const float* rstd,
                T* dx, float* part, long long rows, int cols, cudaStream_t s) {
  auto go = [&](auto at) -> int {
    constexpr auto kern = decltype(at)::value;
    if (const int rc = prepare_kernel<kern>(128 + kLnRingBytes)) return rc;
    kern<<<r.blocks, r.threads, r.smem, s>>>(x, ldx, dy, lddy, g, mean, rstd, dx, part, rows, cols, r.stages, status_block_for_launch());
    PKB_CHECK_CUDA(cudaGetLastError());
    return kApiOk;
  };
  if (r.threads == 128) return go(KernelAt<ln_bwd_ring_kernel<T, 128, 16>>{});
  if (r.threads == 256) return go(KernelAt<ln_bwd_ring_kernel<T, 256, 16>>{});
  if constexpr (sizeof(T) == 2) {
    if (r.per == 32) return go(KernelAt<ln_bwd_ring_kernel<T, 512, 32>>{});
  }
  return go(KernelAt<ln_bwd_ring_kernel<T, 512, 16>>{});
}

template <typename T, int VEC16>
int ln_fwd_any(const void* xv, long long ldx, LnParam g, LnParam b, void* yv, float* mean, float* rstd, long long rows, int cols, float eps,
               cudaStream_t s) {
  const T* x = static_cast<const T*>(xv);
  T* y = static_cast<T*>(yv);
  const bool vec = cols % VEC16 == 0 && ln_aligned(x, ldx * (long long)sizeof(T)) && ln_aligned(y, 0) && ln_aligned(g.p, 0) && ln_aligned(b.p, 0);
  LnRingPlan ring;
  if (vec && ln_ring_plan(ring, rows, cols, sizeof(T), false, true, sm_count())) return ln_fwd_ring<T>(ring, x, ldx, g, b, y, mean, rstd, rows, cols, eps, s);
  if (!vec && ln_ring_plan(ring, rows, cols, sizeof(T), false, false, sm_count())) return ln_fwd_odd<T>(ring, x, ldx, g, b, y, mean, rstd, rows, cols, eps, s);
  if (cols > kLnTeamCols) {
    const long long most = (long long)sm_count() * 4;
    ln_fwd_long_kernel<T><<<(unsigned)(rows < most ? rows : most), kLnLongThreads, 0, s>>>(x, ldx, g, b, y, mean, rstd, rows, cols, eps);
    PKB_CHECK_CUDA(cudaGetLastError());
    return kApiOk;
  }
  return vec ? ln_fwd_team<T, VEC16>(x, ldx, g, b, y, mean, rstd, rows, cols, eps, s) : ln_fwd_team<T, 1>(x, ldx, g, b, y, mean, rstd, rows, cols, eps, s);
}

// threads of a row and rows of a block in the backward's team form
int ln_bwd_team_threads(int cols) { return cols <= 512 ? 32 : cols <= 1024 ? 64 : cols <= 2048 ? 128 : cols <= 4096 ? 256 : 512; }
int ln_bwd_team_rows(int cols) { return cols <= 4096 ? 256 / ln_bwd_team_threads(cols) : 1; }

// Small problems in one launch: a cluster of up to 16 blocks, which needs no partial sums in memory and no second kernel (5 us of the host's 19 per
// call), but has 16 SMs only: up to eight rows per team. Device us, one launch / two: 64 x 128 6.3 / 6.4, 512 x 512 (four rows) 8.4 / 6.4, 128 x 4096
// (eight) 12.5 / 12.5, 256 x 4096 (16) 16.6 / 18.4, 1000 x 1001 (16) 27.7 / 10.5, 4000 x 64 (32) 26.9 / 8.4.
bool ln_bwd_one_launch(long long rows, int cols) { return cols <= kLnTeamCols && rows <= 8ll * kLnCluster * ln_bwd_team_rows(cols); }

template <typename T, int VEC>
int ln_bwd_team(const T* x, long long ldx, const T* dy, long long lddy, LnParam g, const float* mean, const float* rstd, T* dx, float* dgamma,
                float* dbeta, float* part, int blocks, long long rows, int cols, cudaStream_t s) {
  auto go = [&](auto tpr, auto ch) -> int {
    using L = LnTeam<T, VEC, tpr.value, ch.value>;
    if (blocks > 0) {
      ln_bwd_kernel<T, VEC, tpr.value, ch.value, false><<<blocks, L::kThreads, 0, s>>>(x, ldx, dy, lddy, g, mean, rstd, dx, part, dgamma, dbeta, rows, cols);
      PKB_CHECK_CUDA(cudaGetLastError());
      return kApiOk;
    }
    constexpr auto kern = ln_bwd_kernel<T, VEC, tpr.value, ch.value, true>;
    if (const int rc = prepare_kernel<kern>(2 * L::kCols * (int)sizeof(float), true)) return rc;
    const long long want = (rows + L::kRows - 1) / L::kRows;
    const unsigned ctas = (unsigned)(want < kLnCluster ? want : kLnCluster);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(L::kThreads);
    cfg.dynamicSmemBytes = 2 * (size_t)cols * sizeof(float);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    PKB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kern, x, ldx, dy, lddy, g, mean, rstd, dx, (float*)nullptr, dgamma, dbeta, rows, cols));
    return kApiOk;
  };
  return ln_by_width<decltype(go)&, T, VEC, true>(cols, go);
}

// How the backward goes. What it writes (the blocks' partial sums) and what the caller is told to bring follow from this one decision.
struct LnBwdForm {
  enum Kind { kCluster, kRing, kOdd, kLong, kTeam } kind;
  LnRingPlan ring;
  int blocks;       // that write partial sums [2][cols] each; 0: none
  int launches() const { return kind == kCluster ? 1 : kind == kLong ? 3 : 2; }
};
LnBwdForm ln_bwd_form(long long rows, int cols, int esize, bool aligned, int sms) {
  LnBwdForm f = {};
  if (ln_bwd_one_launch(rows, cols)) {
    f.kind = LnBwdForm::kCluster;
  } else if (ln_ring_plan(f.ring, rows, cols, esize, true, aligned, sms)) {
    f.kind = aligned ? LnBwdForm::kRing : LnBwdForm::kOdd;
    f.blocks = f.ring.blocks;
  } else if (cols > kLnTeamCols) {      // row slices of the weights' sums
    f.kind = LnBwdForm::kLong;
    f.blocks = (int)(rows < 4 * kLnLongSlices ? (rows + 3) / 4 : kLnLongSlices);
  } else {                              // rows of a block at once, blocks per SM
    f.kind = LnBwdForm::kTeam;
    const int per = ln_bwd_team_rows(cols);
    const long long want = (rows + per - 1) / per, most = (long long)sms * (cols <= 4096 ? 2 : 1);
    f.blocks = (int)(want < most ? want : most);
  }
  return f;
}

template <typename T, int VEC16>
int ln_bwd_any(const void* xv, long long ldx, const void* dyv, long long lddy, LnParam g, const float* mean, const float* rstd, void* dxv,
               float* dgamma, float* dbeta, float* part, long long rows, int cols, cudaStream_t s) {
  const T *x = static_cast<const T*>(xv), *dy = static_cast<const T*>(dyv);
  T* dx = static_cast<T*>(dxv);
  const bool vec = cols % VEC16 == 0 && ln_aligned(x, ldx * (long long)sizeof(T)) && ln_aligned(dy, lddy * (long long)sizeof(T)) &&
                   ln_aligned(dx, 0) && ln_aligned(g.p, 0) && ln_aligned(part, 0);
  const LnBwdForm form = ln_bwd_form(rows, cols, sizeof(T), vec, sm_count());
  PKB_CHECK_ARG(part != nullptr || form.blocks == 0, "scratch for the partial sums");
  if (form.kind == LnBwdForm::kRing) {
    const int rc = ln_bwd_ring<T>(form.ring, x, ldx, dy, lddy, g, mean, rstd, dx, part, rows, cols, s);
    if (rc) return rc;
  } else if (form.kind == LnBwdForm::kOdd) {
    const int rc = ln_bwd_odd<T>(form.ring, x, ldx, dy, lddy, g, mean, rstd, dx, part, rows, cols, s);
    if (rc) return rc;
  } else if (form.kind == LnBwdForm::kLong) {
    const long long most = (long long)sm_count() * 4;
    ln_bwd_long_dx_kernel<T><<<(unsigned)(rows < most ? rows : most), kLnLongThreads, 0, s>>>(x, ldx, dy, lddy, g, mean, rstd, dx, rows, cols);
    ln_bwd_long_params_kernel<T><<<dim3((unsigned)((cols + 63) / 64), (unsigned)form.blocks), 256, 0, s>>>(x, ldx, dy, lddy, mean, rstd, part, rows, cols);
    PKB_CHECK_CUDA(cudaGetLastError());
  } else {
    const int rc = vec ? ln_bwd_team<T, VEC16>(x, ldx, dy, lddy, g, mean, rstd, dx, dgamma, dbeta, part, form.blocks, rows, cols, s)
                       : ln_bwd_team<T, 1>(x, ldx, dy, lddy, g, mean, rstd, dx, dgamma, dbeta, part, form.blocks, rows, cols, s);
    if (rc || form.kind == LnBwdForm::kCluster) return rc;
  }
  const long long width = 2ll * cols;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((width + 31) / 32));
  cfg.blockDim = dim3(1024);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  PKB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, ln_bwd_params_kernel, (const float*)part, form.blocks, width, dgamma, dbeta, cols));
  return kApiOk;
}

}  // namespace

}  // namespace pkb

using namespace pkb;

// y [rows, cols] (contiguous) = layer norm of x (ldx elements between rows, any value: rows may overlap or repeat). dtype: 0 bf16, 1 fp32.
// gamma, beta: cols values or null (1 and 0), bf16 (param_f32 = 0) or fp32. mean, rstd: fp32 [rows], both or neither null.
extern "C" int pkb_layer_norm_fwd(const void* x, long long ldx, const void* gamma, const void* beta, int param_f32, void* y, void* mean,
                                  void* rstd, long long rows, int cols, float eps, int dtype, void* stream) {
  PKB_CHECK_ARG(rows > 0 && cols > 0, "empty problem");
  PKB_CHECK_ARG(x != nullptr && y != nullptr && (mean == nullptr) == (rstd == nullptr), "x, y, and mean and rstd together");
  PKB_CHECK_ARG(dtype == 0 || dtype == 1, "dtype must be 0 (bf16) or 1 (fp32)");
  const LnParam g{gamma, param_f32, 1.f}, b{beta, param_f32, 0.f};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype ? ln_fwd_any<float, 4>(x, ldx, g, b, y, static_cast<float*>(mean), static_cast<float*>(rstd), rows, cols, eps, s)
               : ln_fwd_any<__nv_bfloat16, 8>(x, ldx, g, b, y, static_cast<float*>(mean), static_cast<float*>(rstd), rows, cols, eps, s);
}

// Blocks whose partial sums pkb_layer_norm_bwd writes on a GPU of `sms` SMs (0: the current device): its scratch is [this][2][cols] fp32.
// aligned: 1 where base, pitch and width of x and dy and the addresses of gamma, dx and the scratch are multiples of 16 bytes, else 0.
extern "C" int pkb_layer_norm_bwd_blocks(long long rows, int cols, int dtype, int aligned, int sms) {
  if (rows <= 0 || cols <= 0) return 0;
  return ln_bwd_form(rows, cols, dtype ? 4 : 2, aligned != 0, sms > 0 ? sms : sm_count()).blocks;
}

// The kernels that pkb_layer_norm_bwd launches, arguments as above.
extern "C" int pkb_layer_norm_bwd_launches(long long rows, int cols, int dtype, int aligned, int sms) {
  if (rows <= 0 || cols <= 0) return 0;
  return ln_bwd_form(rows, cols, dtype ? 4 : 2, aligned != 0, sms > 0 ? sms : sm_count()).launches();
}

// pkb_layer_norm_bwd_blocks whatever the alignment: the larger of the two. 0: one launch, no scratch.
extern "C" int pkb_layer_norm_bwd_partials(long long rows, int cols, int dtype) {
  const int a = pkb_layer_norm_bwd_blocks(rows, cols, dtype, 1, 0), b = pkb_layer_norm_bwd_blocks(rows, cols, dtype, 0, 0);
  return a > b ? a : b;
}

// dx [rows, cols] (contiguous, the type of x and dy), dgamma and dbeta fp32 [cols] from the saved statistics.
extern "C" int pkb_layer_norm_bwd(const void* x, long long ldx, const void* dy, long long lddy, const void* gamma, int param_f32, const void* mean,
                                  const void* rstd, void* dx, void* dgamma, void* dbeta, void* partial, long long rows, int cols, int dtype,
                                  void* stream) {
  PKB_CHECK_ARG(rows > 0 && cols > 0, "empty problem");
  PKB_CHECK_ARG(x && dy && mean && rstd && dx && dgamma && dbeta, "null pointer");
  PKB_CHECK_ARG(dtype == 0 || dtype == 1, "dtype must be 0 (bf16) or 1 (fp32)");
  const LnParam g{gamma, param_f32, 1.f};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto f = [](void* p) { return static_cast<float*>(p); };
  auto cf = [](const void* p) { return static_cast<const float*>(p); };
  return dtype ? ln_bwd_any<float, 4>(x, ldx, dy, lddy, g, cf(mean), cf(rstd), dx, f(dgamma), f(dbeta), f(partial), rows, cols, s)
               : ln_bwd_any<__nv_bfloat16, 8>(x, ldx, dy, lddy, g, cf(mean), cf(rstd), dx, f(dgamma), f(dbeta), f(partial), rows, cols, s);
}
