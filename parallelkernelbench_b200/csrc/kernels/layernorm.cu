// Layer norm, forward and backward (memory bound: a row is read once and stays in registers between its sums and its results).
//   mean = sum x / N, rstd = 1 / sqrt(sum (x - mean)^2 / N + eps), y = (x - mean) rstd gamma + beta
//   g = dy gamma, xhat = (x - mean) rstd, dx = rstd (g - mean(g) - xhat mean(g xhat)), dgamma = sum_rows dy xhat, dbeta = sum_rows dy
// The variance is the mean of squared differences from the mean, never E[x^2] - mean^2: a row far from zero loses nothing.
// A row belongs to a team of TPR threads that holds VEC * CH of its values each: 16-byte accesses where base, row pitch and width
// allow them (VEC = 8 bf16 or 4 fp32), single values otherwise. All sums are fp32.
#include "pkb/api.h"
#include "pkb/host.h"
#include "pkb/ptx.cuh"

namespace pkb {

namespace {

// one row access: VEC values of type T at p as fp32, and back (rounded to nearest)
template <typename T, int VEC>
__device__ __forceinline__ void ln_load(const T* p, float (&f)[VEC]) {
  if constexpr (VEC == 8) {
    const U4 u = ld_global_nc_v4(p);
    const float2 a = unpack_bf16x2(u.x), b = unpack_bf16x2(u.y), c = unpack_bf16x2(u.z), d = unpack_bf16x2(u.w);
    f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y; f[4] = c.x; f[5] = c.y; f[6] = d.x; f[7] = d.y;
  } else if constexpr (VEC == 4) {
    const U4 u = ld_global_nc_v4(p);
    f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
  } else {
    f[0] = static_cast<float>(*p);
  }
}

template <typename T, int VEC>
__device__ __forceinline__ void ln_store(T* p, const float (&f)[VEC]) {
  if constexpr (VEC == 8)
    st_global_v4(p, U4{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])});
  else if constexpr (VEC == 4)
    st_global_v4(p, U4{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])});
  else if constexpr (sizeof(T) == 2)
    *p = __float2bfloat16_rn(f[0]);
  else
    *p = f[0];
}

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
        const U4 u = ld_global_v4(static_cast<const float*>(p) + c + j);
        f[j] = __uint_as_float(u.x); f[j + 1] = __uint_as_float(u.y); f[j + 2] = __uint_as_float(u.z); f[j + 3] = __uint_as_float(u.w);
      }
    } else if constexpr (VEC == 8) {
      const U4 u = ld_global_v4(static_cast<const __nv_bfloat16*>(p) + c);
      const float2 a = unpack_bf16x2(u.x), b = unpack_bf16x2(u.y), g = unpack_bf16x2(u.z), d = unpack_bf16x2(u.w);
      f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y; f[4] = g.x; f[5] = g.y; f[6] = d.x; f[7] = d.y;
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
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) t += red[k * (NT / 32) + team * W + w];
      v[k] = t;
    }
  }
}

template <typename T, int VEC, int TPR, int CH>
struct LnTeam {
  static constexpr int kThreads = TPR > 256 ? TPR : 256;
  static constexpr int kRows = kThreads / TPR;      // rows that a block has in hand
  static constexpr int kCols = TPR * VEC * CH;      // widest row
};

template <typename T, int VEC, int TPR, int CH>
__global__ void __launch_bounds__(LnTeam<T, VEC, TPR, CH>::kThreads)
ln_fwd_kernel(const T* __restrict__ x, long long ldx, const LnParam gamma, const LnParam beta, T* __restrict__ y,
              float* __restrict__ mean_out, float* __restrict__ rstd_out, long long rows, int cols, float eps) {
  using L = LnTeam<T, VEC, TPR, CH>;
  __shared__ float red[2][L::kThreads / 32];
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
    const float mean = s[0] * inv;
    float q[1] = {0.f};
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) {
      if ((ch * TPR + t) * VEC < cols) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) q[0] += (v[ch][j] - mean) * (v[ch][j] - mean);
      }
    }
    team_sum<1, TPR, L::kThreads>(q, red[1], team);
    const float rstd = rsqrtf(q[0] * inv + eps);
    if (t == 0 && mean_out != nullptr) {
      mean_out[row] = mean;
      rstd_out[row] = rstd;
    }
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) {
      const int c = (ch * TPR + t) * VEC;
      if (c < cols) {
        float g[VEC], b[VEC];
        gamma.template load<VEC>(c, g);
        beta.template load<VEC>(c, b);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[ch][j] = (v[ch][j] - mean) * rstd * g[j] + b[j];
        ln_store<T, VEC>(y + row * cols + c, v[ch]);
      }
    }
  }
}

// Rows wider than a team holds: three passes over the row (the second and third come from L2), one block per row.
constexpr int kLnLongThreads = 512;

template <typename T>
__global__ void __launch_bounds__(kLnLongThreads)
ln_fwd_long_kernel(const T* __restrict__ x, long long ldx, const LnParam gamma, const LnParam beta, T* __restrict__ y,
                   float* __restrict__ mean_out, float* __restrict__ rstd_out, long long rows, int cols, float eps) {
  __shared__ float red[2][kLnLongThreads / 32];
  const float inv = 1.f / (float)cols;
  for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + row * ldx;
    float s[1] = {0.f}, q[1] = {0.f};
    for (int c = threadIdx.x; c < cols; c += kLnLongThreads) s[0] += static_cast<float>(xr[c]);
    team_sum<1, kLnLongThreads, kLnLongThreads>(s, red[0], 0);
    const float mean = s[0] * inv;
    for (int c = threadIdx.x; c < cols; c += kLnLongThreads) {
      const float d = static_cast<float>(xr[c]) - mean;
      q[0] += d * d;
    }
    team_sum<1, kLnLongThreads, kLnLongThreads>(q, red[1], 0);
    const float rstd = rsqrtf(q[0] * inv + eps);
    if (threadIdx.x == 0 && mean_out != nullptr) {
      mean_out[row] = mean;
      rstd_out[row] = rstd;
    }
    for (int c = threadIdx.x; c < cols; c += kLnLongThreads) {
      const float f[1] = {(static_cast<float>(xr[c]) - mean) * rstd * gamma.at(c) + beta.at(c)};
      ln_store<T, 1>(y + row * cols + c, f);
    }
  }
}

// Backward. The blocks are persistent: a thread keeps its columns' sums of dy xhat and dy in registers over all rows of its block and
// writes them once, to part[block][2][cols]; ln_bwd_params_kernel adds the blocks' sums in a fixed order. The loads of a team's next
// row are issued before the sums of the current one.
template <typename T, int VEC, int TPR, int CH>
__global__ void __launch_bounds__(LnTeam<T, VEC, TPR, CH>::kThreads, 512 / LnTeam<T, VEC, TPR, CH>::kThreads)
ln_bwd_kernel(const T* __restrict__ x, long long ldx, const T* __restrict__ dy, long long lddy, const LnParam gamma,
              const float* __restrict__ mean_in, const float* __restrict__ rstd_in, T* __restrict__ dx, float* __restrict__ part,
              long long rows, int cols) {
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
  float xn[CH][VEC], dn[CH][VEC];
  float mean_n = 0.f, rstd_n = 0.f;
  auto fetch = [&](long long row) {
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) {
      const int c = (ch * TPR + t) * VEC;
      if (c < cols) {
        ln_load<T, VEC>(x + row * ldx + c, xn[ch]);
        ln_load<T, VEC>(dy + row * lddy + c, dn[ch]);
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
    for (int ch = 0; ch < CH; ++ch)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        xv[ch][j] = xn[ch][j];
        dv[ch][j] = dn[ch][j];
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
  float* out = part + (long long)blockIdx.x * 2 * cols;
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
}

// dgamma, dbeta [2][cols] = sum over the blocks of part[block][2][cols]: 32 columns and 8 strands of blocks per thread block
__global__ void __launch_bounds__(256)
ln_bwd_params_kernel(const float* __restrict__ part, int blocks, long long width, float* __restrict__ dgamma, float* __restrict__ dbeta, int cols) {
  __shared__ float s[8][33];
  const int lane = threadIdx.x & 31, strand = threadIdx.x >> 5;
  const long long i = (long long)blockIdx.x * 32 + lane;
  float a = 0.f;
  if (i < width)
    for (int b = strand; b < blocks; b += 8) a += part[b * width + i];
  s[strand][lane] = a;
  __syncthreads();
  if (strand == 0 && i < width) {
    a = s[0][lane];
#pragma unroll
    for (int k = 1; k < 8; ++k) a += s[k][lane];
    if (i < cols) dgamma[i] = a;
    else dbeta[i - cols] = a;
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
    float s[2] = {0.f, 0.f};
    for (int c = threadIdx.x; c < cols; c += kLnLongThreads) {
      const float gd = static_cast<float>(dr[c]) * gamma.at(c);
      s[0] += gd;
      s[1] += gd * ((static_cast<float>(xr[c]) - mean) * rstd);
    }
    team_sum<2, kLnLongThreads, kLnLongThreads>(s, red[it], 0);
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

template <typename F, typename T, int VEC>
int ln_by_width(int cols, F&& f) {
  // 16 values per thread: 2 (bf16), 4 (fp32) accesses of 16 bytes, or 16 single ones
  constexpr int CH = 16 / VEC;
  if (cols <= 32 * 16) return f(std::integral_constant<int, 32>{}, std::integral_constant<int, CH>{});
  if (cols <= 64 * 16) return f(std::integral_constant<int, 64>{}, std::integral_constant<int, CH>{});
  if (cols <= 128 * 16) return f(std::integral_constant<int, 128>{}, std::integral_constant<int, CH>{});
  if (cols <= 256 * 16) return f(std::integral_constant<int, 256>{}, std::integral_constant<int, CH>{});
  return f(std::integral_constant<int, 512>{}, std::integral_constant<int, CH>{});
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
  return ln_by_width<decltype(go)&, T, VEC>(cols, go);
}

template <typename T, int VEC16>
int ln_fwd_any(const void* xv, long long ldx, LnParam g, LnParam b, void* yv, float* mean, float* rstd, long long rows, int cols, float eps,
               cudaStream_t s) {
  const T* x = static_cast<const T*>(xv);
  T* y = static_cast<T*>(yv);
  if (cols > kLnTeamCols) {
    const long long most = (long long)sm_count() * 4;
    ln_fwd_long_kernel<T><<<(unsigned)(rows < most ? rows : most), kLnLongThreads, 0, s>>>(x, ldx, g, b, y, mean, rstd, rows, cols, eps);
    PKB_CHECK_CUDA(cudaGetLastError());
    return kApiOk;
  }
  const bool vec = cols % VEC16 == 0 && ln_aligned(x, ldx * (long long)sizeof(T)) && ln_aligned(y, 0) && ln_aligned(g.p, 0) && ln_aligned(b.p, 0);
  return vec ? ln_fwd_team<T, VEC16>(x, ldx, g, b, y, mean, rstd, rows, cols, eps, s) : ln_fwd_team<T, 1>(x, ldx, g, b, y, mean, rstd, rows, cols, eps, s);
}

template <typename T, int VEC>
int ln_bwd_team(const T* x, long long ldx, const T* dy, long long lddy, LnParam g, const float* mean, const float* rstd, T* dx, float* part,
                int blocks, long long rows, int cols, cudaStream_t s) {
  auto go = [&](auto tpr, auto ch) -> int {
    using L = LnTeam<T, VEC, tpr.value, ch.value>;
    ln_bwd_kernel<T, VEC, tpr.value, ch.value><<<blocks, L::kThreads, 0, s>>>(x, ldx, dy, lddy, g, mean, rstd, dx, part, rows, cols);
    PKB_CHECK_CUDA(cudaGetLastError());
    return kApiOk;
  };
  return ln_by_width<decltype(go)&, T, VEC>(cols, go);
}

// rows of a block at once and blocks per SM of the backward's team forms
int ln_bwd_blocks(long long rows, int cols) {
  if (cols > kLnTeamCols) return (int)(rows < 4 * kLnLongSlices ? (rows + 3) / 4 : kLnLongSlices);
  const int tpr = cols <= 512 ? 32 : cols <= 1024 ? 64 : cols <= 2048 ? 128 : cols <= 4096 ? 256 : 512;
  const int threads = tpr > 256 ? tpr : 256, per = threads / tpr;
  const long long want = (rows + per - 1) / per, most = (long long)sm_count() * (512 / threads);
  return (int)(want < most ? want : most);
}

template <typename T, int VEC16>
int ln_bwd_any(const void* xv, long long ldx, const void* dyv, long long lddy, LnParam g, const float* mean, const float* rstd, void* dxv,
               float* dgamma, float* dbeta, float* part, long long rows, int cols, cudaStream_t s) {
  const T *x = static_cast<const T*>(xv), *dy = static_cast<const T*>(dyv);
  T* dx = static_cast<T*>(dxv);
  const int blocks = ln_bwd_blocks(rows, cols);
  if (cols > kLnTeamCols) {
    const long long most = (long long)sm_count() * 4;
    ln_bwd_long_dx_kernel<T><<<(unsigned)(rows < most ? rows : most), kLnLongThreads, 0, s>>>(x, ldx, dy, lddy, g, mean, rstd, dx, rows, cols);
    ln_bwd_long_params_kernel<T><<<dim3((unsigned)((cols + 63) / 64), (unsigned)blocks), 256, 0, s>>>(x, ldx, dy, lddy, mean, rstd, part, rows, cols);
    PKB_CHECK_CUDA(cudaGetLastError());
  } else {
    const bool vec = cols % VEC16 == 0 && ln_aligned(x, ldx * (long long)sizeof(T)) && ln_aligned(dy, lddy * (long long)sizeof(T)) &&
                     ln_aligned(dx, 0) && ln_aligned(g.p, 0);
    const int rc = vec ? ln_bwd_team<T, VEC16>(x, ldx, dy, lddy, g, mean, rstd, dx, part, blocks, rows, cols, s)
                       : ln_bwd_team<T, 1>(x, ldx, dy, lddy, g, mean, rstd, dx, part, blocks, rows, cols, s);
    if (rc) return rc;
  }
  const long long width = 2ll * cols;
  ln_bwd_params_kernel<<<(unsigned)((width + 31) / 32), 256, 0, s>>>(part, blocks, width, dgamma, dbeta, cols);
  PKB_CHECK_CUDA(cudaGetLastError());
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

// Blocks whose partial sums pkb_layer_norm_bwd writes: its scratch is [this][2][cols] fp32.
extern "C" int pkb_layer_norm_bwd_partials(long long rows, int cols) { return rows > 0 && cols > 0 ? ln_bwd_blocks(rows, cols) : 0; }

// dx [rows, cols] (contiguous, the type of x and dy), dgamma and dbeta fp32 [cols] from the saved statistics.
extern "C" int pkb_layer_norm_bwd(const void* x, long long ldx, const void* dy, long long lddy, const void* gamma, int param_f32, const void* mean,
                                  const void* rstd, void* dx, void* dgamma, void* dbeta, void* partial, long long rows, int cols, int dtype,
                                  void* stream) {
  PKB_CHECK_ARG(rows > 0 && cols > 0, "empty problem");
  PKB_CHECK_ARG(x && dy && mean && rstd && dx && dgamma && dbeta && partial, "null pointer");
  PKB_CHECK_ARG(dtype == 0 || dtype == 1, "dtype must be 0 (bf16) or 1 (fp32)");
  const LnParam g{gamma, param_f32, 1.f};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto f = [](void* p) { return static_cast<float*>(p); };
  auto cf = [](const void* p) { return static_cast<const float*>(p); };
  return dtype ? ln_bwd_any<float, 4>(x, ldx, dy, lddy, g, cf(mean), cf(rstd), dx, f(dgamma), f(dbeta), f(partial), rows, cols, s)
               : ln_bwd_any<__nv_bfloat16, 8>(x, ldx, dy, lddy, g, cf(mean), cf(rstd), dx, f(dgamma), f(dbeta), f(partial), rows, cols, s);
}
