// Orthogonalising a matrix by Newton-Schulz products, and the optimiser step around it.
//   X0 = U / (|U|_F + eps);  A = X X^T,  B = b A + c A^2,  X <- a X + B X  (steps times; X^T X and X B where X has more rows than columns)
// Every singular value s of X goes to a s + b s^3 + c s^5, so all of them approach 1 while the singular vectors stay.
//
// Numerics. The iterate is a state and is kept in fp32 (M = k X, k a power of two near the square root of the longer side, so that its
// entries are of the order of one); products run on the tensor cores from a copy of it rounded to fp16, with fp32 accumulation, and a X is
// added in fp32: what rounding adds to the small singular directions is not fed back through the linear term. fp16 because its 11 bits
// are 8 times as fine as bf16's at the same rate and nothing here leaves its range: |X|_2 <= 1 at the start and stays under the bound that the
// host checks for the coefficients, the Gram matrix A and B are O(1). Against 64 bits five steps are 1e-3 to 2e-3 off (2-norm) with fp16
// and 1e-2 to 2e-2 with bf16; with the iterate itself in fp16 a matrix of rank 16 in noise was 4e-2 off.
//
// Work: per step m (m + 1) n + m^2 (m + 1) + 2 m^2 n flops on the smaller side m: A and B are symmetric, so only the tiles on and below the
// diagonal are computed and each is stored twice.
// Three forms, by size: a short side (m <= 128) in one launch; few tiles, each shared by a cluster; tiles of CTA pairs that fill the GPU. A call in us:
// 16 x 16 19, 8 x 1024 x 128 53, 333 x 1000 114 (105 in a graph: 17 launches of about 6), 1024 x 1024 125, 2048 x 2048 254; with the optimiser step
// 4096 x 4096 1396 and 28672 x 4096 7281, 71 % and 75 % of what the tensor cores sustain under the power cap (the products' tensor pipe is active in
// 86 to 88 % of the cycles; the rest is the tail of their last tiles and the passes over momentum and weight).
#include <cuda_fp16.h>
#include <math.h>

#include "pkb/api.h"
#include "pkb/gemm_umma.cuh"
#include "pkb/host.h"

namespace pkb {

namespace {

constexpr int kNsTile = 256;                                  // rows and columns of a CTA pair's tile
constexpr int kNsStages = 6;
constexpr int kNsOperandBytes = 128 * kGemmBlockK * 2;        // a CTA's half of an operand
constexpr int kNsStageBytes = 2 * kNsOperandBytes;
constexpr int kNsThreads = 64 + 256;                          // loader, issuer, eight epilogue warps
constexpr int kNsStageOut = 8 * 4096;                         // a 32 x 32 fp32 chunk per epilogue warp
constexpr int kNsSmem = kNsStages * kNsStageBytes + kNsStageOut + 256 + 1024;
constexpr uint32_t kNsKernelId = 111;

enum NsEpilogue : int {
  kNsGram = 0,      // A = alpha acc, both triangles
  kNsPoly = 1,      // B = b A + c acc, both triangles
  kNsUpdate = 2,    // M = a M + acc, X16 = fp16(M)
  kNsResult = 3,    // out = bf16(scale (a M + acc))
  kNsStep = 4,      // p = decay p - scale (a M + acc), p_bf16 = bf16(p)
};

struct NsParams {
  int rows, cols, K, batch;     // output rows and columns of one matrix, inner extent
  __half* out16;                // fp16 result (A, B or the next X), pitch16 halves per row
  const __half* a16;            // A, read by kNsPoly
  long long pitch16;
  float* master;                // M, pitch_m floats per row
  long long pitch_m;
  void* final_out;              // kNsResult: bf16 [batch, rows, cols]; kNsStep: p, fp32 of that shape
  __nv_bfloat16* p_bf16;        // kNsStep: optional
  float alpha, beta;            // see NsEpilogue: (alpha, -), (c, b), (1, a), (scale, a), (scale, a)
  float decay;
  int vec_out;                  // the final result's rows start on 16 bytes
  uint32_t* status;
  uint64_t wait_budget_ns;
};

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_half2(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }

__device__ __forceinline__ void tma_load_3d_pair_p(uint32_t smem_dst, const CUtensorMap* desc, uint32_t bar, int32_t c0, int32_t c1, int32_t c2,
                                                   uint32_t lead) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %6, 0;\n\t"
      "@q cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];\n\t}\n"
      :
      : "r"(smem_dst), "l"(reinterpret_cast<uint64_t>(desc)), "r"(bar & kPeerBitMask), "r"(c0), "r"(c1), "r"(c2), "r"(lead)
      : "memory");
}

// The launches of a call depend on one another and are short where the matrices are: each one is launched while the one before it still
// runs (programmatic dependent launch), sets up its barriers and tensor memory, and waits here until everything before it has finished and is
// visible. Every thread waits before its first access to global memory.
__device__ __forceinline__ void wait_for_predecessor() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_successor_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// the row of the triangle's t-th element (rows of 1, 2, 3, ... elements)
__host__ __device__ inline int tri_row(int t) {
  int r = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
  while ((r + 1) * (r + 2) / 2 <= t) ++r;
  while (r * (r + 1) / 2 > t) --r;
  return r;
}

// Tile order: groups of eight tile rows, columns outermost inside a group, so that the tiles in flight share operand panels in L2. For the
// symmetric products only tiles with row >= column.
constexpr int kNsGroup = 8;
template <bool SYM>
__device__ __forceinline__ void ns_tile(int t, int num_m, int num_n, int& i, int& j) {
  if constexpr (SYM) {
    const int first = tri_row(t) / kNsGroup * kNsGroup;
    const int gm = min(kNsGroup, num_m - first);
    const int local = t - first * (first + 1) / 2;
    if (local < first * gm) {
      j = local / gm;
      i = first + local - j * gm;
    } else {
      const int rem = local - first * gm, r = tri_row(rem);
      i = first + r;
      j = first + rem - r * (r + 1) / 2;
    }
  } else {
    const int first = t / (kNsGroup * num_n) * kNsGroup;
    const int gm = min(kNsGroup, num_m - first);
    const int local = t - first * num_n;
    j = local / gm;
    i = first + local - j * gm;
  }
}

// ---- four columns of a result row: what the step adds to the product, and where the sum goes ----
// `at`: row in the stack of matrices, col: first of the four columns (a multiple of four, < p.cols). Rows of the scratch tensors are padded to
// eights, so there four columns never leave a row.
template <int EPI>
__device__ __forceinline__ uint4 ns_fetch4(const NsParams& p, long long at, int col) {
  if constexpr (EPI == kNsPoly) {
    const uint2 u = *reinterpret_cast<const uint2*>(p.a16 + at * p.pitch16 + col);
    return make_uint4(u.x, u.y, 0u, 0u);
  } else if constexpr (EPI != kNsGram) {
    const U4 u = ld_global_v4(p.master + at * p.pitch_m + col);
    return make_uint4(u.x, u.y, u.z, u.w);
  } else {
    return make_uint4(0u, 0u, 0u, 0u);
  }
}

template <int EPI>
__device__ __forceinline__ void ns_apply4(const NsParams& p, const uint4& in, float (&v)[4]) {
  if constexpr (EPI == kNsGram) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] *= p.alpha;
  } else if constexpr (EPI == kNsPoly) {
    const float2 f0 = unpack_half2(in.x), f1 = unpack_half2(in.y);
    v[0] = fmaf(p.alpha, v[0], p.beta * f0.x);
    v[1] = fmaf(p.alpha, v[1], p.beta * f0.y);
    v[2] = fmaf(p.alpha, v[2], p.beta * f1.x);
    v[3] = fmaf(p.alpha, v[3], p.beta * f1.y);
  } else {
    v[0] = fmaf(p.beta, __uint_as_float(in.x), v[0]);
    v[1] = fmaf(p.beta, __uint_as_float(in.y), v[1]);
    v[2] = fmaf(p.beta, __uint_as_float(in.z), v[2]);
    v[3] = fmaf(p.beta, __uint_as_float(in.w), v[3]);
  }
}

template <int EPI>
__device__ __forceinline__ void ns_put4(const NsParams& p, long long at, int col, float (&v)[4]) {
  if constexpr (EPI == kNsUpdate)
    st_global_v4(p.master + at * p.pitch_m + col, U4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])});
  if constexpr (EPI == kNsUpdate || EPI == kNsGram || EPI == kNsPoly)
    *reinterpret_cast<uint2*>(p.out16 + at * p.pitch16 + col) = make_uint2(pack_half2(v[0], v[1]), pack_half2(v[2], v[3]));
  if constexpr (EPI == kNsResult) {
    __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.final_out) + at * p.cols + col;
    if (p.vec_out) {
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(p.alpha * v[0], p.alpha * v[1]), pack_bf16x2(p.alpha * v[2], p.alpha * v[3]));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (col + j < p.cols) dst[j] = __float2bfloat16_rn(p.alpha * v[j]);
    }
  }
  if constexpr (EPI == kNsStep) {
    float* dst = static_cast<float*>(p.final_out) + at * p.cols + col;
    __nv_bfloat16* dst16 = p.p_bf16 != nullptr ? p.p_bf16 + at * p.cols + col : nullptr;
    if (p.vec_out) {
      const U4 u = ld_global_v4(dst);
      const uint32_t old[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = fmaf(-p.alpha, v[j], p.decay * __uint_as_float(old[j]));
      st_global_v4(dst, U4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])});
      if (dst16 != nullptr) *reinterpret_cast<uint2*>(dst16) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (col + j < p.cols) {
          const float np = fmaf(-p.alpha, v[j], p.decay * dst[j]);
          dst[j] = np;
          if (dst16 != nullptr) dst16[j] = __float2bfloat16_rn(np);
        }
    }
  }
}

__device__ __forceinline__ void st_shared_v4(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ U4 ld_shared_v4(uint32_t a) {
  U4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}

// Persistent GEMM on clusters of two CTAs, tiles of 256 x 256 (tcgen05.mma.cta_group::2, M = 256): warp 0 of both CTAs loads, warp 1 of
// the leader issues the products into two accumulators in tensor memory, warps 2 to 9 of both CTAs turn the finished one into results
// meanwhile. A_MN / B_MN: the operand is [K, rows] row-major and is described to the tensor core as MN-major.
template <bool A_MN, bool B_MN, int EPI>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kNsThreads, 1)
ns_gemm_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const NsParams p) {
  constexpr bool kSym = EPI == kNsGram || EPI == kNsPoly;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t bar_base = smem_base + kNsStages * kNsStageBytes + kNsStageOut;
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (kNsStages + s); };
  auto tfull_bar = [&](int a) { return bar_base + 8u * (2 * kNsStages + a); };
  auto tempty_bar = [&](int a) { return bar_base + 8u * (2 * kNsStages + 2 + a); };
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem_gen + kNsStages * kNsStageBytes + kNsStageOut + 8 * (2 * kNsStages + 4));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t cta_rank = cluster_ctarank();
  const bool leader = cta_rank == 0;
  const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
  const int num_m = (p.rows + kNsTile - 1) / kNsTile, num_n = (p.cols + kNsTile - 1) / kNsTile;
  const int num_k = (p.K + kGemmBlockK - 1) / kGemmBlockK;
  const int per_matrix = kSym ? num_m * (num_m + 1) / 2 : num_m * num_n;
  const int num_tiles = per_matrix * p.batch;

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < kNsStages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull_bar(a), 1);
      mbar_init(tempty_bar(a), 16);     // eight epilogue warps of each CTA
    }
    fence_mbar_init();
    tma_prefetch_desc(&tmap_a);
    tma_prefetch_desc(&tmap_b);
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(tmem_holder), 512);
    tmem_relinquish_pair();
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_holder;
  let_successor_launch();
  wait_for_predecessor();

  if (warp == 0) {
    const uint32_t lead = elect_one() ? 1u : 0u;
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int tile = pair; tile < num_tiles && ok; tile += num_pairs) {
      const int b = tile / per_matrix;
      int ti, tj;
      ns_tile<kSym>(tile - b * per_matrix, num_m, num_n, ti, tj);
      const int row0 = ti * kNsTile + (int)cta_rank * 128, col0 = tj * kNsTile + (int)cta_rank * 128;
      for (int kb = 0; kb < num_k; ++kb) {
        if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, p.wait_budget_ns)) {
          if (lane == 0) record_status(p.status, kStatusMbarTimeout, kNsKernelId, 0, stage, 11, tile);
          ok = false;
          break;
        }
        mbar_expect_tx_p(full_bar(stage), 2 * kNsStageBytes, leader ? lead : 0u);
        const uint32_t sa = smem_base + stage * kNsStageBytes, sb = sa + kNsOperandBytes;
        const int k0 = kb * kGemmBlockK;
        if constexpr (A_MN) {
          tma_load_3d_pair_p(sa, &tmap_a, full_bar(stage), row0, k0, b, lead);
          tma_load_3d_pair_p(sa + 8192, &tmap_a, full_bar(stage), row0 + 64, k0, b, lead);
        } else {
          tma_load_3d_pair_p(sa, &tmap_a, full_bar(stage), k0, row0, b, lead);
        }
        if constexpr (B_MN) {
          tma_load_3d_pair_p(sb, &tmap_b, full_bar(stage), col0, k0, b, lead);
          tma_load_3d_pair_p(sb + 8192, &tmap_b, full_bar(stage), col0 + 64, k0, b, lead);
        } else {
          tma_load_3d_pair_p(sb, &tmap_b, full_bar(stage), k0, col0, b, lead);
        }
        if (++stage == kNsStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (leader) {
      const uint32_t lead = elect_one() ? 1u : 0u;
      constexpr uint32_t idesc = make_idesc(kNsTile, kNsTile, 0, 0, A_MN ? 1 : 0, B_MN ? 1 : 0);
      const uint32_t a_lo0 = A_MN ? smem_desc_lo_mnmajor(smem_base, 8192u) : smem_desc_lo_kmajor(smem_base);
      const uint32_t b_lo0 = B_MN ? smem_desc_lo_mnmajor(smem_base + kNsOperandBytes, 8192u) : smem_desc_lo_kmajor(smem_base + kNsOperandBytes);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int tile = pair; tile < num_tiles && ok; tile += num_pairs) {
        if (!mbar_wait(tempty_bar(acc), acc_phase ^ 1u, abort_flag, p.wait_budget_ns)) {
          if (lane == 0) record_status(p.status, kStatusMbarTimeout, kNsKernelId, 0, acc, 20, tile);
          break;
        }
        tc_fence_after_sync();
        const uint32_t tmem_d = tmem_base + acc * 256;
        for (int kb = 0; kb < num_k; ++kb) {
          if (!mbar_wait(full_bar(stage), phase, abort_flag, p.wait_budget_ns)) {
            if (lane == 0) record_status(p.status, kStatusMbarTimeout, kNsKernelId, 0, stage, 21, tile);
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t a_lo = a_lo0 + stage * (kNsStageBytes >> 4), b_lo = b_lo0 + stage * (kNsStageBytes >> 4);
#pragma unroll
          for (int k = 0; k < kGemmBlockK / 16; ++k)
            umma_f16_ss_pair_p(tmem_d, smem_desc_join(a_lo + (A_MN ? 128u : 2u) * k), smem_desc_join(b_lo + (B_MN ? 128u : 2u) * k), idesc,
                               (kb | k) != 0 ? 1u : 0u, lead);
          umma_commit_pair_p(empty_bar(stage), 0x3, lead);
          if (++stage == kNsStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        umma_commit_pair_p(tfull_bar(acc), 0x3, lead);
        if (++acc == 2) {
          acc = 0;
          acc_phase ^= 1u;
        }
      }
    }
    __syncwarp();
  } else {
    // Two warps per quarter of a CTA's 128 rows, each with half of the tile's columns, 32 x 32 values at a time. The accumulator comes with a
    // row per lane; through 4 KB of shared memory (16-byte pieces swizzled by the row) it is turned so that eight lanes hold 128 bytes of a
    // row, and every access to global memory covers whole sectors. What the step adds (M, or A) is fetched one chunk ahead, for the first
    // chunk while the products still run. With a row per lane in global memory as well, 4096 x 4096 took 123 us per update, 62 per Gram matrix.
    const int q = warp & 3, half = (warp - 2) >> 2;
    const uint32_t stg = smem_base + kNsStages * kNsStageBytes + static_cast<uint32_t>(warp - 2) * 4096u;
    const int trow = lane >> 3, tcol = (lane & 7) * 4;       // place in the turned chunk: rows trow + 4 it, columns tcol .. tcol + 3
    int acc = 0;
    uint32_t acc_phase = 0;
    const uint32_t leader_tempty0 = mapa_shared(tempty_bar(0), 0), leader_tempty1 = mapa_shared(tempty_bar(1), 0);
    for (int tile = pair; tile < num_tiles; tile += num_pairs) {
      const int b = tile / per_matrix;
      int ti, tj;
      ns_tile<kSym>(tile - b * per_matrix, num_m, num_n, ti, tj);
      const int row0 = ti * kNsTile + (int)cta_rank * 128 + q * 32;
      const int colh = tj * kNsTile + half * 128;
      const int rows_here = p.rows - row0;                     // may be <= 0
      const long long grow = (long long)b * p.rows + row0;     // first row in the stack of matrices
      // the next chunk's M (four floats) or A (four halves) per row of the turned chunk
      uint4 in[8];
      auto fetch = [&](int c) {
        const int col = colh + c * 32 + tcol;
#pragma unroll
        for (int it = 0; it < 8; ++it)
          if (c < 4 && col < p.cols && trow + it * 4 < rows_here) in[it] = ns_fetch4<EPI>(p, grow + trow + it * 4, col);
      };
      fetch(0);
      bool ok = mbar_wait(tfull_bar(acc), acc_phase, abort_flag, p.wait_budget_ns);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) {
        if (lane == 0) record_status(p.status, kStatusMbarTimeout, kNsKernelId, 0, acc, 30, tile);
        break;
      }
      tc_fence_after_sync();
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        const int col0 = colh + c * 32;
        if (col0 >= p.cols || rows_here <= 0) break;
        uint32_t r[32];
        __syncwarp();                                           // the last chunk was read
        tmem_ld_32x32(tmem_base + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(acc * 256 + half * 128 + c * 32), r);
        tmem_ld_wait();
#pragma unroll
        for (int f = 0; f < 8; ++f) st_shared_v4(stg + lane * 128u + ((f ^ (lane & 7)) << 4), r[4 * f], r[4 * f + 1], r[4 * f + 2], r[4 * f + 3]);
        __syncwarp();
        float v[8][4];
#pragma unroll
        for (int it = 0; it < 8; ++it) {
          const int tr = trow + it * 4;
          const U4 u = ld_shared_v4(stg + tr * 128u + (((lane & 7) ^ (tr & 7)) << 4));
          v[it][0] = __uint_as_float(u.x); v[it][1] = __uint_as_float(u.y); v[it][2] = __uint_as_float(u.z); v[it][3] = __uint_as_float(u.w);
          ns_apply4<EPI>(p, in[it], v[it]);
        }
        fetch(c + 1);
        const int col = col0 + tcol;
        if constexpr (kSym) {
          if (ti != tj) {
            // the other triangle: turned back, a row per lane, 32 lanes write 32 consecutive columns of row col0 + j
            uint32_t w[32];
            if constexpr (EPI == kNsPoly) {
              __syncwarp();
#pragma unroll
              for (int it = 0; it < 8; ++it) {
                const int tr = trow + it * 4;
                st_shared_v4(stg + tr * 128u + (((lane & 7) ^ (tr & 7)) << 4), __float_as_uint(v[it][0]), __float_as_uint(v[it][1]),
                             __float_as_uint(v[it][2]), __float_as_uint(v[it][3]));
              }
              __syncwarp();
#pragma unroll
              for (int f = 0; f < 8; ++f) {
                const U4 u = ld_shared_v4(stg + lane * 128u + ((f ^ (lane & 7)) << 4));
                w[4 * f] = u.x; w[4 * f + 1] = u.y; w[4 * f + 2] = u.z; w[4 * f + 3] = u.w;
              }
            } else {
#pragma unroll
              for (int j = 0; j < 32; ++j) w[j] = __float_as_uint(p.alpha * __uint_as_float(r[j]));
            }
            if (lane < rows_here) {
              __half* dst = p.out16 + ((long long)b * p.rows + col0) * p.pitch16 + row0 + lane;
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (col0 + j < p.cols) dst[(long long)j * p.pitch16] = __float2half_rn(__uint_as_float(w[j]));
            }
          }
        }
#pragma unroll
        for (int it = 0; it < 8; ++it)
          if (col < p.cols && trow + it * 4 < rows_here) ns_put4<EPI>(p, grow + trow + it * 4, col, v[it]);
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(acc == 0 ? leader_tempty0 : leader_tempty1);
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1u;
      }
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag) {      // copies and products in flight end before the memory that they use goes away
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
    __syncthreads();
  }
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

// ------------------------------------------------------------------------------------------------ few tiles: one per cluster, K split over its CTAs
// Where a product has too few 256 x 256 tiles to occupy the GPU, its time is the way through K on the few SMs that have work: a CTA takes
// its 32 KB per 64 of K from L2 at about 0.27 us. Here a tile is 128 x 128 and belongs to a cluster of up to 16 CTAs that share its K range;
// each puts its partial sums into its shared memory, and after a cluster barrier sums its share of the rows over all of them (distributed
// shared memory, in the order of the CTAs) and finishes those rows. A call for 333 x 1000: 182 us with the pairs' tiles, 105 with these.
constexpr int kSplitTile = 128;
constexpr int kSplitStages = 4;
constexpr int kSplitStageBytes = 2 * kNsOperandBytes;         // 128 rows of A, 128 of B
constexpr int kSplitPartial = kSplitTile * kSplitTile * 4;
constexpr int kSplitSmem = kSplitStages * kSplitStageBytes + kSplitPartial + 256 + 1024;
constexpr int kSplitCluster = 16;

constexpr int kSplitRows = kSplitTile / 8;        // rows of a tile per epilogue warp, over all CTAs of its cluster

// The end of a tile on a cluster of S CTAs: this CTA's kSplitTile / S rows, a warp per row at a time, four columns per lane. All 16 reads of a
// thread (its rows times S CTAs) are in flight before the first sum: one row after the other took 3.6 us.
template <int EPI, int S>
__device__ __forceinline__ void split_finish(const NsParams& p, uint32_t partial, int rank, int et, int b, int row0, int col0, bool mirror,
                                             const uint4 (&in)[kSplitRows]) {
  constexpr int kShare = kSplitTile / S, kTurns = kSplitRows / S;
  const int lane = et & 31, col = col0 + lane * 4;
  auto place = [&](int row, int f) { return partial + row * 512u + ((uint32_t)(f ^ (row & 7)) << 4); };
  float4 part[kTurns][S];
#pragma unroll
  for (int i = 0; i < kTurns; ++i)
#pragma unroll
    for (int c = 0; c < S; ++c) part[i][c] = ld_shared_cluster_v4(mapa_shared(place(rank * kShare + (et >> 5) + i * 8, lane), (uint32_t)c));
#pragma unroll
  for (int i = 0; i < kTurns; ++i) {
    const int row = rank * kShare + (et >> 5) + i * 8;
    float v[4] = {part[i][0].x, part[i][0].y, part[i][0].z, part[i][0].w};
#pragma unroll
    for (int c = 1; c < S; ++c) {
      v[0] += part[i][c].x; v[1] += part[i][c].y; v[2] += part[i][c].z; v[3] += part[i][c].w;
    }
    ns_apply4<EPI>(p, in[i], v);
    if (mirror)      // kept for the other triangle: nobody else reads this CTA's copy of its own rows
      st_shared_v4(place(row, lane), __float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    if (row0 + row < p.rows && col < p.cols) ns_put4<EPI>(p, (long long)b * p.rows + row0 + row, col, v);
  }
  if (mirror) {
    asm volatile("bar.sync 1, 256;" ::: "memory");
#pragma unroll 8
    for (int i = et; i < kShare * kSplitTile; i += 256) {
      const int r = i % kShare, j = i / kShare, row = rank * kShare + r;
      float v;
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(place(row, j >> 2) + (j & 3) * 4u) : "memory");
      if (row0 + row < p.rows && col0 + j < p.cols) p.out16[((long long)b * p.rows + col0 + j) * p.pitch16 + row0 + row] = __float2half_rn(v);
    }
  }
}

template <bool A_MN, bool B_MN, int EPI>
__global__ void __launch_bounds__(kNsThreads, 1)
ns_split_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const NsParams p) {
  constexpr bool kSym = EPI == kNsGram || EPI == kNsPoly;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t partial = smem_base + kSplitStages * kSplitStageBytes;
  const uint32_t bar_base = partial + kSplitPartial;
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (kSplitStages + s); };
  const uint32_t done_bar = bar_base + 8u * 2 * kSplitStages;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem_gen + kSplitStages * kSplitStageBytes + kSplitPartial + 8 * (2 * kSplitStages + 1));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ctas = (int)cluster_nctaid(), rank = (int)cluster_ctarank();
  const int tile = (int)(blockIdx.x / ctas);
  const int num_m = (p.rows + kSplitTile - 1) / kSplitTile, num_n = (p.cols + kSplitTile - 1) / kSplitTile;
  const int per_matrix = kSym ? num_m * (num_m + 1) / 2 : num_m * num_n;
  const int b = tile / per_matrix;
  int ti, tj;
  ns_tile<kSym>(tile - b * per_matrix, num_m, num_n, ti, tj);
  const int row0 = ti * kSplitTile, col0 = tj * kSplitTile;
  const int num_k = (p.K + kGemmBlockK - 1) / kGemmBlockK, share_k = (num_k + ctas - 1) / ctas;
  const int kb0 = min(num_k, rank * share_k), kb1 = min(num_k, kb0 + share_k);     // may be empty

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < kSplitStages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    mbar_init(done_bar, 1);
    fence_mbar_init();
    tma_prefetch_desc(&tmap_a);
    tma_prefetch_desc(&tmap_b);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_holder), 128);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_holder;
  wait_for_predecessor();

  const int et = (int)threadIdx.x - 64;             // thread of the epilogue, < 0: not one
  const int share = kSplitTile / ctas;              // rows that this CTA finishes: four columns of a row per thread and turn
  uint4 in[kSplitRows];
  if (warp == 0) {
    const uint32_t lead = elect_one() ? 1u : 0u;
    int stage = 0;
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, p.wait_budget_ns)) {
        if (lane == 0) record_status(p.status, kStatusMbarTimeout, kNsKernelId + 2, 0, stage, 11, tile);
        break;
      }
      mbar_expect_tx_p(full_bar(stage), kSplitStageBytes, lead);
      const uint32_t sa = smem_base + stage * kSplitStageBytes, sb = sa + kNsOperandBytes;
      const int k0 = kb * kGemmBlockK;
      if constexpr (A_MN) {
        tma_load_3d_p(sa, &tmap_a, full_bar(stage), row0, k0, b, lead);
        tma_load_3d_p(sa + 8192, &tmap_a, full_bar(stage), row0 + 64, k0, b, lead);
      } else {
        tma_load_3d_p(sa, &tmap_a, full_bar(stage), k0, row0, b, lead);
      }
      if constexpr (B_MN) {
        tma_load_3d_p(sb, &tmap_b, full_bar(stage), col0, k0, b, lead);
        tma_load_3d_p(sb + 8192, &tmap_b, full_bar(stage), col0 + 64, k0, b, lead);
      } else {
        tma_load_3d_p(sb, &tmap_b, full_bar(stage), k0, col0, b, lead);
      }
      if (++stage == kSplitStages) {
        stage = 0;
        phase ^= 1u;
      }
    }
  } else if (warp == 1) {
    const uint32_t lead = elect_one() ? 1u : 0u;
    constexpr uint32_t idesc = make_idesc(kSplitTile, kSplitTile, 0, 0, A_MN ? 1 : 0, B_MN ? 1 : 0);
    const uint32_t a_lo0 = A_MN ? smem_desc_lo_mnmajor(smem_base, 8192u) : smem_desc_lo_kmajor(smem_base);
    const uint32_t b_lo0 = B_MN ? smem_desc_lo_mnmajor(smem_base + kNsOperandBytes, 8192u) : smem_desc_lo_kmajor(smem_base + kNsOperandBytes);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!mbar_wait(full_bar(stage), phase, abort_flag, p.wait_budget_ns)) {
        if (lane == 0) record_status(p.status, kStatusMbarTimeout, kNsKernelId + 2, 0, stage, 21, tile);
        ok = false;
        break;
      }
      tc_fence_after_sync();
      const uint32_t a_lo = a_lo0 + stage * (kSplitStageBytes >> 4), b_lo = b_lo0 + stage * (kSplitStageBytes >> 4);
#pragma unroll
      for (int k = 0; k < kGemmBlockK / 16; ++k)
        umma_f16_ss_p(tmem, smem_desc_join(a_lo + (A_MN ? 128u : 2u) * k), smem_desc_join(b_lo + (B_MN ? 128u : 2u) * k), idesc,
                      (kb != kb0 || k != 0) ? 1u : 0u, lead);
      umma_commit_p(empty_bar(stage), lead);
      if (++stage == kSplitStages) {
        stage = 0;
        phase ^= 1u;
      }
    }
    if (ok) umma_commit_p(done_bar, lead);
  } else {
    // what the step adds to this CTA's rows, fetched while the products run
#pragma unroll
    for (int i = 0; i < kSplitRows; ++i) {
      const int row = rank * share + (et >> 5) + i * 8, col = col0 + lane * 4;
      if (i * 8 + (et >> 5) < share && row0 + row < p.rows && col < p.cols) in[i] = ns_fetch4<EPI>(p, (long long)b * p.rows + row0 + row, col);
    }
    const int q = warp & 3, half = (warp - 2) >> 2, prow = q * 32 + lane;
    if (kb0 < kb1) {
      const bool ok = mbar_wait(done_bar, 0, abort_flag, p.wait_budget_ns);
      if (!__all_sync(0xffffffffu, ok) && lane == 0) record_status(p.status, kStatusMbarTimeout, kNsKernelId + 2, 0, 0, 30, tile);
      tc_fence_after_sync();
    }
#pragma unroll 1
    for (int c = half * 64; c < half * 64 + 64; c += 32) {
      uint32_t r[32];
      if (kb0 < kb1) {
        tmem_ld_32x32(tmem + (static_cast<uint32_t>(q * 32) << 16) + c, r);
        tmem_ld_wait();
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) r[j] = 0u;
      }
#pragma unroll
      for (int f = 0; f < 8; ++f)
        st_shared_v4(partial + prow * 512u + ((((uint32_t)(c >> 2) + f) ^ (prow & 7)) << 4), r[4 * f], r[4 * f + 1], r[4 * f + 2], r[4 * f + 3]);
    }
    tc_fence_before_sync();
  }
  __syncwarp();
  cluster_sync_all();
  if (et >= 0) {
    const bool mirror = kSym && ti != tj;
    switch (ctas) {
      case 1: split_finish<EPI, 1>(p, partial, rank, et, b, row0, col0, mirror, in); break;
      case 2: split_finish<EPI, 2>(p, partial, rank, et, b, row0, col0, mirror, in); break;
      case 4: split_finish<EPI, 4>(p, partial, rank, et, b, row0, col0, mirror, in); break;
      case 8: split_finish<EPI, 8>(p, partial, rank, et, b, row0, col0, mirror, in); break;
      default: split_finish<EPI, 16>(p, partial, rank, et, b, row0, col0, mirror, in); break;
    }
  }
  // Only now: CTAs that wait for their predecessor from its first microsecond on slow its reads of shared memory across the cluster (1024 x 1024:
  // 209 us a call against 180 with none).
  let_successor_launch();
  if (*abort_flag) {      // copies and products in flight end before the memory that they use goes away
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  __syncwarp();
  cluster_sync_all();     // nobody leaves while its partial sums may still be read
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, 128);
  }
}

// ------------------------------------------------------------------------------------------------ what goes before the products
// m <- momentum m + g, u = g + momentum m (Nesterov) or m; without momentum (m null) u = g. The sums of u^2 are 64-bit: squares of fp32 values
// neither overflow nor vanish there. part[matrix][block], added by every block of the next kernel in the same order.
struct NsInput {
  const void* g;
  int g_f32;
  float* m;
  float momentum;
  int nesterov;
  __device__ __forceinline__ float grad(long long i) const {
    return g_f32 ? static_cast<const float*>(g)[i] : __bfloat162float(static_cast<const __nv_bfloat16*>(g)[i]);
  }
  __device__ __forceinline__ float use(float gv, float mv) const { return m == nullptr ? gv : nesterov ? fmaf(momentum, mv, gv) : mv; }
};

constexpr int kNsPrepThreads = 256;
constexpr int kNsMaxParts = 1024;

// u * inv in fp32 for any |u| and inv whose product is in range (either alone may be far from one): inv = m 2^q is taken apart, u is moved half of
// the way by an exact power of two, and only the other factor rounds. Of a matrix of zeros nothing is divided: it stays zero for any eps.
struct NsScale {
  float first, second;
  __device__ __forceinline__ NsScale(double k, double square_sum, double eps) {
    int q = 0;
    const double m = square_sum == 0.0 ? 0.0 : frexp(k / (sqrt(square_sum) + eps), &q);
    const int half = q / 2;
    first = ldexpf(1.f, half);
    second = ldexpf((float)m, q - half);
  }
  __device__ __forceinline__ float operator()(float u) const { return u * first * second; }
};

// The sum of eight squares as a 64-bit number, formed in fp32 relative to the power of two of the largest: one conversion per eight values.
__device__ __forceinline__ double square_sum8(const float (&u)[8]) {
  float top = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(u[j]));
  const int e = min(max((int)(__float_as_uint(top) >> 23) - 127, -126), 126);       // (0 and denormal: 2^-126 will do)
  const float down = __uint_as_float((uint32_t)(127 - e) << 23);
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float v = u[j] * down;
    s = fmaf(v, v, s);
  }
  return (double)s * __longlong_as_double((long long)(1023 + 2 * e) << 52);
}

__device__ __forceinline__ double block_sum_double(double v, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0.0;
#pragma unroll
  for (int w = 0; w < kNsPrepThreads / 32; ++w) t += red[w];
  __syncthreads();
  return t;
}

// eight gradient values from i on (16 or 32 bytes, aligned)
__device__ __forceinline__ void load8(const NsInput& in, long long i, float (&g)[8]) {
  if (in.g_f32) {
    const U4 u = ld_global_nc_v4(static_cast<const float*>(in.g) + i), v = ld_global_nc_v4(static_cast<const float*>(in.g) + i + 4);
    const uint32_t w[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 8; ++j) g[j] = __uint_as_float(w[j]);
  } else {
    unpack16(ld_global_nc_v4(static_cast<const __nv_bfloat16*>(in.g) + i), g);
  }
}
__device__ __forceinline__ void load8(const float* p, float (&f)[8]) {
  const U4 u = ld_global_v4(p), v = ld_global_v4(p + 4);
  const uint32_t w[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = __uint_as_float(w[j]);
}
__device__ __forceinline__ void store8(float* p, const float (&f)[8]) {
  st_global_v4(p, U4{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])});
  st_global_v4(p + 4, U4{__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]), __float_as_uint(f[7])});
}

// VEC: a matrix is a multiple of eight values and the tensors start on 16 bytes. Two accesses of eight values in flight per thread.
template <bool VEC>
__global__ void __launch_bounds__(kNsPrepThreads)
ns_norm_kernel(const NsInput in, long long numel, double* __restrict__ part) {
  __shared__ double red[kNsPrepThreads / 32];
  const long long base = (long long)blockIdx.y * numel;
  double s = 0.0;
  if constexpr (VEC) {
    const long long step = (long long)gridDim.x * kNsPrepThreads * 8;
    for (long long i = ((long long)blockIdx.x * kNsPrepThreads + threadIdx.x) * 8; i < numel; i += 2 * step) {
      float g[2][8], m[2][8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (i + h * step < numel) {
          load8(in, base + i + h * step, g[h]);
          if (in.m != nullptr) load8(in.m + base + i + h * step, m[h]);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (i + h * step >= numel) break;
        if (in.m != nullptr) {
#pragma unroll
          for (int j = 0; j < 8; ++j) m[h][j] = fmaf(in.momentum, m[h][j], g[h][j]);
          store8(in.m + base + i + h * step, m[h]);
        }
        float u[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = in.use(g[h][j], m[h][j]);
        s += square_sum8(u);
      }
    }
  } else {
    for (long long i = (long long)blockIdx.x * kNsPrepThreads + threadIdx.x; i < numel; i += (long long)gridDim.x * kNsPrepThreads) {
      const float g = in.grad(base + i);
      float m = 0.f;
      if (in.m != nullptr) {
        m = fmaf(in.momentum, in.m[base + i], g);
        in.m[base + i] = m;
      }
      const double u = in.use(g, m);
      s += u * u;
    }
  }
  s = block_sum_double(s, red);
  if (threadIdx.x == 0) part[(long long)blockIdx.y * gridDim.x + blockIdx.x] = s;
  let_successor_launch();
}

// M = k u / (|u| + eps) and its fp16 copy, rows padded to their pitch with zeros
__global__ void __launch_bounds__(kNsPrepThreads)
ns_start_kernel(const NsInput in, int rows, int cols, int pitch, const double* __restrict__ part, int parts, double eps, double k, int vec,
                float* __restrict__ master, __half* __restrict__ x16) {
  __shared__ double red[kNsPrepThreads / 32];
  const long long b = blockIdx.y;
  wait_for_predecessor();
  double sum = 0.0;
  for (int i = threadIdx.x; i < parts; i += kNsPrepThreads) sum += part[b * parts + i];
  sum = block_sum_double(sum, red);
  const NsScale scale(k, sum, eps);
  const int vecs = pitch / 8;
  const long long total = (long long)rows * vecs, base = b * rows * cols;
  for (long long i = (long long)blockIdx.x * kNsPrepThreads + threadIdx.x; i < total; i += (long long)gridDim.x * kNsPrepThreads) {
    const long long r = i / vecs;
    const int c = (int)(i - r * vecs) * 8;
    float u[8];
    const long long at = base + r * cols + c;
    if (vec) {
      float g[8], m[8];
      load8(in, at, g);
      if (in.m != nullptr) load8(in.m + at, m);
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] = in.use(g[j], m[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] = c + j < cols ? in.use(in.grad(at + j), in.m != nullptr ? in.m[at + j] : 0.f) : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) u[j] = scale(u[j]);
    const long long dst = (b * rows + r) * pitch + c;
    store8(master + dst, u);
    st_global_v4(x16 + dst, U4{pack_half2(u[0], u[1]), pack_half2(u[2], u[3]), pack_half2(u[4], u[5]), pack_half2(u[6], u[7])});
  }
  let_successor_launch();
}

// ------------------------------------------------------------------------------------------------ a short side: one launch
// Matrices whose smaller side is at most 128 stay on the chip for the whole call: a cluster owns a matrix, each of its CTAs a slice of
// S <= 256 along the longer side. The iterate is in tensor memory in fp32, its fp16 copy in shared memory, where the same bytes serve the
// Gram product (K-major, over the slice) and the update (MN-major, the slice as columns). Only the Gram matrix crosses CTAs, through scratch that
// stays in L2: each writes its partial sums, adds its rows' share of all of them in the order of the CTAs, and reads the others' rounded rows; the
// polynomial is computed by every CTA for itself. B is kept as two fp16 numbers, which costs one more product: its rounding is the largest part of
// the error where the side is short (64 x 2048: 1.7e-3 off 64 bits with one, 1.2e-3 with two). (Distributed shared memory moved the 92 KB per CTA at about 17 bytes a cycle: 4 to 9 us a step.) What bounds it is latency: five rounds of three short products with two cluster barriers each.
constexpr int kSmallSide = 128;
constexpr int kSmallSlice = 256;
constexpr int kSmallCluster = 16;
constexpr int kSmallThreads = 256;
constexpr int kSmallX = kSmallSlice / 64 * 16384;              // X16: atoms of 64 columns, 128 rows of 128 bytes
constexpr int kSmallGram = kSmallSide * kSmallSide * 4;        // partial Gram sums, fp32
constexpr int kSmallA = kSmallSide * kSmallSide * 2;           // A and B, fp16
constexpr int kSmallStage = kSmallSide * kSmallSlice * 4;      // u, fp32; A and B take its place
constexpr int kSmallSmem = kSmallX + kSmallStage + 1024;
static_assert(3 * kSmallA <= kSmallStage, "A and B lie where u was staged");

constexpr int kSmallMaxSteps = 16;

struct NsSmallParams {
  NsInput in;
  long long matrix;          // values of one matrix
  int side, longer, tall, slice, steps;
  double eps, k;
  float co[3 * kSmallMaxSteps];
  int vec_in, vec_out;
  void* out;                 // bf16 result, or null
  float* p;
  __nv_bfloat16* p_bf16;
  float decay, scale;
  float* gram;               // scratch where a matrix has several CTAs: their partial Gram sums, kSmallGram bytes per CTA
  __half* rows;              // and the rounded Gram matrix, kSmallA bytes per matrix
  uint32_t* status;
  uint64_t wait_budget_ns;
};

// 16 bytes from L2: other SMs wrote them since this one may last have read the line
__device__ __forceinline__ U4 ld_global_l2(const void* p) {
  U4 v;
  asm volatile("ld.global.cg.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}

// byte of value (row, col) in atoms of 64 columns with the 128-byte swizzle
__device__ __forceinline__ uint32_t sw128_at(int row, int col) {
  return (uint32_t)(col >> 6) * 16384u + (uint32_t)row * 128u + ((((uint32_t)(col & 63) >> 3) ^ ((uint32_t)row & 7u)) << 4) + ((uint32_t)col & 7u) * 2u;
}
// eight values of row `row` from column `col` on (a multiple of eight) as fp16
__device__ __forceinline__ void put8(uint32_t base, int row, int col, const float* v) {
  st_shared_v4(base + sw128_at(row, col), pack_half2(v[0], v[1]), pack_half2(v[2], v[3]), pack_half2(v[4], v[5]), pack_half2(v[6], v[7]));
}

__global__ void __launch_bounds__(kSmallThreads, 1)
ns_small_kernel(const __grid_constant__ NsSmallParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ double red[kNsPrepThreads / 32];
  __shared__ double norm_part;
  __shared__ __align__(8) uint64_t bar_storage;
  __shared__ uint32_t tmem_holder;
  __shared__ int abort_storage;
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t x16 = smem_base, a16 = x16 + kSmallX, b16 = a16 + kSmallA, b16_low = b16 + kSmallA;
  float* u_stage = reinterpret_cast<float*>(smem_raw + (a16 - smem_u32(smem_raw)));
  volatile int* abort_flag = &abort_storage;
  const uint32_t bar = smem_u32(&bar_storage);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ctas = p.longer > p.slice ? (int)cluster_nctaid() : 1;
  const int rank = (int)cluster_ctarank();
  const long long matrix = blockIdx.x / cluster_nctaid();
  const int c0 = rank * p.slice;                                  // first column of the slice (along the longer side)
  const int width = max(0, min(p.slice, p.longer - c0));
  const long long base = matrix * p.matrix;

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    mbar_init(bar, 1);
    fence_mbar_init();
  }
  if (warp == 0) {
    tmem_alloc(smem_u32(&tmem_holder), 512);
    tmem_relinquish();
  }

  // ---- u of this slice into shared memory, u_stage[c][r], and its squares' sum. The rows are swizzled by the column so that eight columns of a row
  // (a wide matrix) as well as a column for all rows (the reader below) fall into different banks; a tall one has its rows side by side already.
  auto swz = [&](int c) { return p.tall ? 0 : (c ^ (c >> 3)) & 31; };
  double sum = 0.0;
  if (p.vec_in) {
    // eight values per access, four accesses per tensor in flight
    const int per = p.tall ? p.side / 8 : (width + 7) / 8, items = p.tall ? width * per : p.side * per;
    auto where = [&](int i, int& r, int& c) {
      const int o = i / per, w = (i - o * per) * 8;
      r = p.tall ? w : o;
      c = p.tall ? o : w;
      return base + (p.tall ? (long long)(c0 + c) * p.side + r : (long long)r * p.longer + c0 + c);
    };
    for (int i0 = threadIdx.x; i0 < items; i0 += 4 * kSmallThreads) {
      float g[4][8], m[4][8] = {};
      int r, c;
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        if (i0 + h * kSmallThreads < items) {
          const long long at = where(i0 + h * kSmallThreads, r, c);
          load8(p.in, at, g[h]);
          if (p.in.m != nullptr) load8(p.in.m + at, m[h]);
        }
      }
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        if (i0 + h * kSmallThreads >= items) break;
        const long long at = where(i0 + h * kSmallThreads, r, c);
        if (p.in.m != nullptr) {
#pragma unroll
          for (int j = 0; j < 8; ++j) m[h][j] = fmaf(p.in.momentum, m[h][j], g[h][j]);
          store8(p.in.m + at, m[h]);
        }
        float u[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = p.in.use(g[h][j], m[h][j]);
        sum += square_sum8(u);
        if (p.tall) {
          float4* dst = reinterpret_cast<float4*>(u_stage + c * kSmallSide + r);
          dst[0] = make_float4(u[0], u[1], u[2], u[3]);
          dst[1] = make_float4(u[4], u[5], u[6], u[7]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) u_stage[(c + j) * kSmallSide + (r ^ swz(c + j))] = u[j];
        }
      }
    }
  } else {
    const int inner = p.tall ? p.side : width, items = p.side * width;
#pragma unroll 8
    for (int i = threadIdx.x; i < items; i += kSmallThreads) {
      const int o = i / inner, w = i - o * inner;
      const int r = p.tall ? w : o, c = p.tall ? o : w;
      const long long at = base + (p.tall ? (long long)(c0 + c) * p.side + r : (long long)r * p.longer + c0 + c);
      const float g = p.in.grad(at);
      float m = 0.f;
      if (p.in.m != nullptr) {
        m = fmaf(p.in.momentum, p.in.m[at], g);
        p.in.m[at] = m;
      }
      const float u = p.in.use(g, m);
      u_stage[c * kSmallSide + (r ^ swz(c))] = u;
      sum += (double)u * (double)u;
    }
  }
  sum = block_sum_double(sum, red);
  if (ctas > 1) {
    if (threadIdx.x == 0) norm_part = sum;
    cluster_sync_all();
    double part[kSmallCluster];          // all reads in flight before the first sum
#pragma unroll
    for (int c = 0; c < kSmallCluster; ++c)
      if (c < ctas) asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(part[c]) : "r"(mapa_shared(smem_u32(&norm_part), (uint32_t)c)) : "memory");
    sum = 0.0;
#pragma unroll
    for (int c = 0; c < kSmallCluster; ++c)
      if (c < ctas) sum += part[c];
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const NsScale scale(p.k, sum, p.eps);
  const uint32_t tmem = tmem_holder, tm_acc = tmem + 256;
  // a warp's place in tensor memory: 32 rows, and half of the columns of what it walks
  const int q = warp & 3, half = warp >> 2, row = q * 32 + lane;
  const uint32_t lanes = (uint32_t)(q * 32) << 16;
  const int cols_half = p.slice / 2;
  for (int c = half * cols_half; c < (half + 1) * cols_half; c += 32) {
    float v[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      const bool in = row < p.side && c + j < width;
      v[j] = in ? scale(u_stage[(c + j) * kSmallSide + (row ^ swz(c + j))]) : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 32; j += 8) put8(x16, row, c + j, v + j);
    uint32_t w[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) w[j] = __float_as_uint(v[j]);
    tmem_st_32x32(tmem + lanes + c, w);
  }
  tmem_st_wait();
  fence_proxy_async_smem();
  tc_fence_before_sync();
  __syncthreads();

  uint32_t phase = 0;
  bool ok = true;
  auto wait_products = [&](int site) {
    if (ok && !mbar_wait(bar, phase, abort_flag, p.wait_budget_ns)) {
      if (threadIdx.x == 0) record_status(p.status, kStatusMbarTimeout, kNsKernelId + 1, 0, 0, site, (uint32_t)matrix);
      ok = false;
    }
    phase ^= 1u;
    __syncwarp();
    tc_fence_after_sync();
  };
  const float alpha = (float)(1.0 / (p.k * p.k));
  float* my_gram = p.gram + (matrix * ctas + rank) * (kSmallGram / 4);
  __half* my_rows = p.rows + matrix * (kSmallA / 2);
  constexpr uint32_t kSquare = make_idesc(kSmallSide, kSmallSide, 0, 0, 0, 0);
  const uint32_t idesc_update = make_idesc(kSmallSide, (uint32_t)p.slice, 0, 0, 0, 1);
#pragma unroll 1
  for (int step = 0; step < p.steps; ++step) {
    const float a = p.co[3 * step], b = p.co[3 * step + 1], cc = p.co[3 * step + 2];
    // ---- the slice's share of X X^T
    if (warp == 0) {
      const uint32_t lead = elect_one() ? 1u : 0u;
      tc_fence_after_sync();
      for (int kk = 0; kk < p.slice / 16; ++kk) {
        const uint32_t lo = smem_desc_lo_kmajor(x16 + (kk >> 2) * 16384u) + (kk & 3) * 2u;
        umma_f16_ss_p(tm_acc, smem_desc_join(lo), smem_desc_join(lo), kSquare, kk != 0 ? 1u : 0u, lead);
      }
      umma_commit_p(bar, lead);
    }
    wait_products(1);
#pragma unroll 1
    for (int c = half * 64; c < half * 64 + 64; c += 32) {
      uint32_t r[32];
      tmem_ld_32x32(tm_acc + lanes + c, r);
      tmem_ld_wait();
      if (ctas > 1) {
        // four columns of all rows side by side: a warp writes 512 bytes, and a CTA's rows below are contiguous as well
#pragma unroll
        for (int f = 0; f < 8; ++f)
          st_global_v4(my_gram + (((c >> 2) + f) * kSmallSide + row) * 4, U4{r[4 * f], r[4 * f + 1], r[4 * f + 2], r[4 * f + 3]});
      } else {
        float v[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = alpha * __uint_as_float(r[j]);
#pragma unroll
        for (int j = 0; j < 32; j += 8) put8(a16, row, c + j, v + j);
      }
    }
    if (ctas > 1) {
      cluster_sync_all();
      // this CTA's share of the rows, summed over all CTAs: four columns per thread and turn, all reads of a turn in flight at once
      const int share = kSmallSide / ctas;
      for (int i = (int)threadIdx.x; i < share * 32; i += kSmallThreads) {
        const int f = i / share, r = rank * share + i - f * share;
        const float* src = p.gram + matrix * ctas * (kSmallGram / 4) + (f * kSmallSide + r) * 4;
        U4 part[kSmallCluster];
#pragma unroll
        for (int c = 0; c < kSmallCluster; ++c)
          if (c < ctas) part[c] = ld_global_l2(src + c * (kSmallGram / 4));
        float t[4] = {};
#pragma unroll
        for (int c = 0; c < kSmallCluster; ++c) {
          if (c < ctas) {
            t[0] += __uint_as_float(part[c].x); t[1] += __uint_as_float(part[c].y); t[2] += __uint_as_float(part[c].z); t[3] += __uint_as_float(part[c].w);
          }
        }
        *reinterpret_cast<uint2*>(my_rows + r * kSmallSide + f * 4) = make_uint2(pack_half2(alpha * t[0], alpha * t[1]), pack_half2(alpha * t[2], alpha * t[3]));
      }
      cluster_sync_all();
      // all rows
      U4 got[8];
#pragma unroll
      for (int h = 0; h < 8; ++h) got[h] = ld_global_l2(my_rows + (h * kSmallThreads + threadIdx.x) * 8);
#pragma unroll
      for (int h = 0; h < 8; ++h) {
        const int i = h * kSmallThreads + (int)threadIdx.x;
        st_shared_v4(a16 + sw128_at(i >> 4, (i & 15) * 8), got[h].x, got[h].y, got[h].z, got[h].w);
      }
      fence_proxy_async_smem();
      tc_fence_before_sync();
      __syncthreads();
    } else {
      fence_proxy_async_smem();
      tc_fence_before_sync();
      __syncthreads();
    }
    // ---- A A, and B = b A + c A A
    if (warp == 0) {
      const uint32_t lead = elect_one() ? 1u : 0u;
      tc_fence_after_sync();
#pragma unroll
      for (int kk = 0; kk < kSmallSide / 16; ++kk) {
        const uint32_t lo = smem_desc_lo_kmajor(a16 + (kk >> 2) * 16384u) + (kk & 3) * 2u;
        umma_f16_ss_p(tm_acc, smem_desc_join(lo), smem_desc_join(lo), kSquare, kk != 0 ? 1u : 0u, lead);
      }
      umma_commit_p(bar, lead);
    }
    wait_products(2);
#pragma unroll 1
    for (int c = half * 64; c < half * 64 + 64; c += 32) {
      uint32_t r[32];
      tmem_ld_32x32(tm_acc + lanes + c, r);
      tmem_ld_wait();
      float v[32];
#pragma unroll
      for (int j = 0; j < 32; j += 8) {
        const U4 u = ld_shared_v4(a16 + sw128_at(row, c + j));
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const float2 f = unpack_half2(w[h]);
          v[j + 2 * h] = fmaf(cc, __uint_as_float(r[j + 2 * h]), b * f.x);
          v[j + 2 * h + 1] = fmaf(cc, __uint_as_float(r[j + 2 * h + 1]), b * f.y);
        }
        put8(b16, row, c + j, v + j);
#pragma unroll
        for (int h = 0; h < 8; ++h) v[j + h] -= __half2float(__float2half_rn(v[j + h]));
        put8(b16_low, row, c + j, v + j);
      }
    }
    fence_proxy_async_smem();
    tc_fence_before_sync();
    __syncthreads();
    // ---- X <- a X + B X
    if (warp == 0) {
      const uint32_t lead = elect_one() ? 1u : 0u;
      tc_fence_after_sync();
#pragma unroll
      for (int kk = 0; kk < 2 * kSmallSide / 16; ++kk) {
        const int k = kk & 7;
        const uint32_t alo = smem_desc_lo_kmajor((kk < 8 ? b16 : b16_low) + (k >> 2) * 16384u) + (k & 3) * 2u;
        const uint32_t blo = smem_desc_lo_mnmajor(x16, 16384u) + k * 128u;
        umma_f16_ss_p(tm_acc, smem_desc_join(alo), smem_desc_join(blo), idesc_update, kk != 0 ? 1u : 0u, lead);
      }
      umma_commit_p(bar, lead);
    }
    wait_products(3);
    const bool last = step + 1 == p.steps;
#pragma unroll 1
    for (int c = half * cols_half; c < (half + 1) * cols_half; c += 32) {
      uint32_t r[32], m[32];
      tmem_ld_32x32(tm_acc + lanes + c, r);
      tmem_ld_32x32(tmem + lanes + c, m);
      tmem_ld_wait();
      float v[32];
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = fmaf(a, __uint_as_float(m[j]), __uint_as_float(r[j]));
      if (!last) {
#pragma unroll
        for (int j = 0; j < 32; ++j) m[j] = __float_as_uint(v[j]);
        tmem_st_32x32(tmem + lanes + c, m);
#pragma unroll
        for (int j = 0; j < 32; j += 8) put8(x16, row, c + j, v + j);
      } else if (row < p.side) {
        const long long stride = p.tall ? p.side : 1;
        const long long at = base + (p.tall ? (long long)(c0 + c) * p.side + row : (long long)row * p.longer + c0 + c);
        if (p.out != nullptr) {
          __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.out) + at;
          if (p.vec_out) {
#pragma unroll
            for (int j = 0; j < 32; j += 8)
              if (c + j < width)
                st_global_v4(dst + j, U4{pack_bf16x2(p.scale * v[j], p.scale * v[j + 1]), pack_bf16x2(p.scale * v[j + 2], p.scale * v[j + 3]),
                                         pack_bf16x2(p.scale * v[j + 4], p.scale * v[j + 5]), pack_bf16x2(p.scale * v[j + 6], p.scale * v[j + 7])});
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (c + j < width) dst[j * stride] = __float2bfloat16_rn(p.scale * v[j]);
          }
        } else if (p.vec_out) {
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            if (c + j < width) {
              float o[8];
              load8(p.p + at + j, o);
#pragma unroll
              for (int i = 0; i < 8; ++i) o[i] = fmaf(-p.scale, v[j + i], p.decay * o[i]);
              store8(p.p + at + j, o);
              if (p.p_bf16 != nullptr)
                st_global_v4(p.p_bf16 + at + j, U4{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]), pack_bf16x2(o[4], o[5]), pack_bf16x2(o[6], o[7])});
            }
          }
        } else {
          float o[32];
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (c + j < width) o[j] = p.p[at + j * stride];
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            if (c + j < width) {
              const float np = fmaf(-p.scale, v[j], p.decay * o[j]);
              p.p[at + j * stride] = np;
              if (p.p_bf16 != nullptr) p.p_bf16[at + j * stride] = __float2bfloat16_rn(np);
            }
          }
        }
      }
      __syncwarp();
    }
    tmem_st_wait();
    fence_proxy_async_smem();
    tc_fence_before_sync();
    __syncthreads();
  }
  if (*abort_flag) {      // products in flight end before their memory goes away
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  __syncthreads();
  if (warp == 0) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
}

// cluster: CTAs of a cluster where the kernel does not fix them itself, else 0
template <typename... Params, typename... Args>
cudaError_t launch_dependent(void (*kern)(Params...), dim3 grid, int threads, int smem, cudaStream_t s, int cluster, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 0 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

// [i]: clusters of 2^i CTAs of a kernel that are resident at once (a cluster stays inside a group of SMs: 148, 74, 33, 15 and 7 on a whole GPU, which
// is also the answer where there is no device to ask).
using NsResident = std::array<int, 5>;
template <auto KERN>
const NsResident& ns_resident(int threads, int smem) {
  static const NsResident table = [&] {
    NsResident t = {148, 74, 33, 15, 7};
    if (prepare_kernel<KERN>(smem, true) != kApiOk) {
      (void)cudaGetLastError();
      return t;
    }
    for (int i = 0; i < 5; ++i) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(1u << i);
      cfg.blockDim = dim3((unsigned)threads);
      cfg.dynamicSmemBytes = (size_t)smem;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = 1u << i;
      attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&t[i], KERN, &cfg) != cudaSuccess) {
        (void)cudaGetLastError();
        t[i] = 0;
      }
    }
    return t;
  }();
  return table;
}

// CTAs that share a tile of the split form, 0 where the pairs' form is taken: that one's tiles are four times as large, so it needs the GPU
// filled, which 128 x 128 tiles in one wave say it is not.
int split_ctas(long long tiles, int num_k) {
  if (tiles > sm_count()) return 0;
  // the largest cluster of which all are resident at once, with at least two blocks of K for each CTA
  const NsResident& resident = ns_resident<ns_split_kernel<false, false, kNsPoly>>(kNsThreads, kSplitSmem);
  for (int i = 4; i > 0; --i)
    if (tiles <= resident[i] && num_k >= 2 << i) return 1 << i;
  return 1;
}

long long ns_tiles(long long batch, int rows, int cols, int size, bool symmetric) {
  const long long num_m = (rows + size - 1) / size, num_n = (cols + size - 1) / size;
  return (symmetric ? num_m * (num_m + 1) / 2 : num_m * num_n) * batch;
}

// One product. launch = false: only what can fail before a launch does (the kernel's limits), so that a call fails before it has changed anything.
template <bool A_MN, bool B_MN, int EPI>
int ns_gemm(const CUtensorMap& ta, const CUtensorMap& tb, NsParams p, cudaStream_t s, bool launch) {
  constexpr bool kSym = EPI == kNsGram || EPI == kNsPoly;
  const long long small_tiles = ns_tiles(p.batch, p.rows, p.cols, kSplitTile, kSym), tiles = ns_tiles(p.batch, p.rows, p.cols, kNsTile, kSym);
  if (const int ctas = split_ctas(small_tiles, (p.K + kGemmBlockK - 1) / kGemmBlockK)) {
    if (const int rc = prepare_kernel<ns_split_kernel<A_MN, B_MN, EPI>>(kSplitSmem, true)) return rc;
    if (!launch) return kApiOk;
    PKB_CHECK_CUDA(launch_dependent(ns_split_kernel<A_MN, B_MN, EPI>, dim3((unsigned)(small_tiles * ctas)), kNsThreads, kSplitSmem, s, ctas, ta, tb, p));
    return kApiOk;
  }
  int ctas = sm_count() & ~1;
  if (ctas > 2 * tiles) ctas = (int)(2 * tiles);
  if (const int rc = prepare_kernel<ns_gemm_kernel<A_MN, B_MN, EPI>>(kNsSmem)) return rc;
  if (!launch) return kApiOk;
  PKB_CHECK_CUDA(launch_dependent(ns_gemm_kernel<A_MN, B_MN, EPI>, dim3((unsigned)ctas), kNsThreads, kNsSmem, s, 0, ta, tb, p));
  return kApiOk;
}

// CTAs per matrix: as few as hold it, then more (down to slices of 64) while the clusters of all matrices are resident at once.
int small_cluster(long long batch, int longer) {
  const NsResident& resident = ns_resident<ns_small_kernel>(kSmallThreads, kSmallSmem);
  int i = 0;
  while ((kSmallSlice << i) < longer) ++i;
  while (i < 4 && (64 << i) < longer && batch <= resident[i + 1]) ++i;
  return 1 << i;
}

// (clusters of more than eight CTAs are not to be had everywhere)
bool small_fits(int side, int longer, int steps) {
  if (side > kSmallSide || longer > kSmallCluster * kSmallSlice || steps > kSmallMaxSteps) return false;
  return longer <= 8 * kSmallSlice || ns_resident<ns_small_kernel>(kSmallThreads, kSmallSmem)[4] > 0;
}

int launch_small(const NsSmallParams& p, int cluster, long long batch, cudaStream_t s) {
  if (const int rc = prepare_kernel<ns_small_kernel>(kSmallSmem, true)) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(batch * cluster));
  cfg.blockDim = dim3(kSmallThreads);
  cfg.dynamicSmemBytes = kSmallSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  PKB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, ns_small_kernel, p));
  return kApiOk;
}

long long pad8(long long n) { return (n + 7) / 8 * 8; }
long long pad256(long long n) { return (n + 255) / 256 * 256; }

// scratch: M [batch, rows, pitch] fp32, X twice the same in fp16, A and B [batch, m, pitch of m] in fp16, the norm's partial sums
struct NsScratch {
  long long master, x0, x1, a, b, part, total;
  NsScratch(long long batch, long long rows, long long cols) {
    const long long m = rows < cols ? rows : cols, x = batch * rows * pad8(cols), g = batch * m * pad8(m);
    master = 0;
    x0 = master + pad256(4 * x);
    x1 = x0 + pad256(2 * x);
    a = x1 + pad256(2 * x);
    b = a + pad256(2 * g);
    part = b + pad256(2 * g);
    total = part + pad256(8 * batch * kNsMaxParts);
  }
};

}  // namespace

}  // namespace pkb

using namespace pkb;

// bytes of scratch that pkb_newton_schulz wants (0: none) and, in *launches, the kernels that it launches
extern "C" long long pkb_newton_schulz_scratch(long long batch, int rows, int cols, int steps, int* launches) {
  if (batch <= 0 || rows <= 0 || cols <= 0) return 0;
  const int side = rows < cols ? rows : cols, longer = rows < cols ? cols : rows;
  const bool small = small_fits(side, longer, steps);
  if (launches != nullptr) *launches = small ? 1 : 2 + 3 * steps;
  if (!small) return NsScratch(batch, rows, cols).total;
  const int cluster = small_cluster(batch, longer);
  return cluster > 1 ? batch * ((long long)cluster * kSmallGram + kSmallA) : 0;
}

// Orthogonalises `batch` matrices [rows, cols] u (see NsInput: g bf16 or fp32, with the momentum m fp32 updated in place where it is not null).
// coeff: HOST array of steps triples (a, b, c). Result, by p: null -> out bf16 [batch, rows, cols]; else p (fp32) <- decay p - scale o,
// with a bf16 copy in p_bf16 where that is not null. scratch: pkb_newton_schulz_scratch bytes on a 256-byte boundary.
extern "C" int pkb_newton_schulz(const void* g, int g_f32, void* m, float momentum, int nesterov, long long batch, int rows, int cols,
                                 const float* coeff, int steps, double eps, void* out, void* p, float decay, float scale, void* p_bf16,
                                 void* scratch, void* stream) {
  PKB_CHECK_ARG(batch > 0 && batch <= 65535 && rows > 0 && cols > 0, "1 .. 65535 matrices of at least one row and column");
  PKB_CHECK_ARG(steps >= 1 && coeff != nullptr, "at least one step");
  PKB_CHECK_ARG(g != nullptr && ((out != nullptr) != (p != nullptr)), "g, scratch and one of out and p");
  const bool tall = rows > cols;
  const int side = tall ? cols : rows, longer = tall ? rows : cols;
  PKB_CHECK_ARG(small_fits(side, longer, steps) || ns_tiles(batch, rows, cols, kNsTile, false) < (1ll << 24), "too many tiles of 256 x 256");
  uint32_t* status = status_block_for_launch();
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const long long pitch = pad8(cols), pitch_a = pad8(side), numel = (long long)rows * cols;
  const double k = ldexp(1.0, (int)lrint(log2((double)longer) / 2));
  const NsInput in{g, g_f32, static_cast<float*>(m), momentum, nesterov};
  const bool aligned_out = ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(p_bf16)) & 15) == 0;
  const bool aligned = ((reinterpret_cast<uintptr_t>(g) | reinterpret_cast<uintptr_t>(m)) & 15) == 0, vec = aligned && numel % 8 == 0;
  if (small_fits(side, longer, steps)) {
    NsSmallParams q = {};
    q.in = in;
    q.matrix = numel;
    q.side = side;
    q.longer = longer;
    q.tall = tall;
    const int cluster = small_cluster(batch, longer);
    q.slice = ((longer + cluster - 1) / cluster + 63) / 64 * 64;
    q.steps = steps;
    q.eps = eps;
    q.k = k;
    for (int i = 0; i < 3 * steps; ++i) q.co[i] = coeff[i];
    q.vec_in = aligned && cols % 8 == 0;
    q.vec_out = !tall && aligned_out && cols % 8 == 0;
    q.out = out;
    q.p = static_cast<float*>(p);
    q.p_bf16 = static_cast<__nv_bfloat16*>(p_bf16);
    q.decay = decay;
    q.scale = (float)((p == nullptr ? 1.0 : (double)scale) / k);
    if (cluster > 1) {
      PKB_CHECK_ARG(scratch != nullptr && (reinterpret_cast<uintptr_t>(scratch) & 255) == 0, "scratch must start on 256 bytes");
      q.gram = static_cast<float*>(scratch);
      q.rows = reinterpret_cast<__half*>(static_cast<uint8_t*>(scratch) + batch * cluster * kSmallGram);
    }
    q.status = status;
    q.wait_budget_ns = kDefaultWaitBudgetNs;
    return launch_small(q, cluster, batch, s);
  }

  PKB_CHECK_ARG(scratch != nullptr && (reinterpret_cast<uintptr_t>(scratch) & 255) == 0, "scratch must start on 256 bytes");
  const NsScratch at(batch, rows, cols);
  uint8_t* base = static_cast<uint8_t*>(scratch);
  float* master = reinterpret_cast<float*>(base + at.master);
  __half *x[2] = {reinterpret_cast<__half*>(base + at.x0), reinterpret_cast<__half*>(base + at.x1)};
  __half *a16 = reinterpret_cast<__half*>(base + at.a), *b16 = reinterpret_cast<__half*>(base + at.b);
  double* part = reinterpret_cast<double*>(base + at.part);
  const long long most = ((long long)sm_count() * 8 + batch - 1) / batch;          // blocks per matrix that fill the GPU
  auto blocks_for = [&](long long items, long long cap) {
    long long n = (items + kNsPrepThreads - 1) / kNsPrepThreads;
    if (n > most) n = most;
    if (n > cap) n = cap;
    return (int)(n < 1 ? 1 : n);
  };
  // maps of X as an operand whose rows lie along K (boxes of 64 columns x 128 rows) and as one whose rows are K (64 x 64), and of A and B
  CUtensorMap xk[2], xm[2], ak, bk;
  int rc;
  for (int i = 0; i < 2; ++i) {
    rc = encode_tmap_3d(&xk[i], kTmapFp16, x[i], cols, rows, batch, pitch * 2, rows * pitch * 2, kGemmBlockK, 128, 1, kSwizzle128);
    if (rc) return rc;
    rc = encode_tmap_3d(&xm[i], kTmapFp16, x[i], cols, rows, batch, pitch * 2, rows * pitch * 2, 64, kGemmBlockK, 1, kSwizzle128);
    if (rc) return rc;
  }
  rc = encode_tmap_3d(&ak, kTmapFp16, a16, side, side, batch, pitch_a * 2, side * pitch_a * 2, kGemmBlockK, 128, 1, kSwizzle128);
  if (rc) return rc;
  rc = encode_tmap_3d(&bk, kTmapFp16, b16, side, side, batch, pitch_a * 2, side * pitch_a * 2, kGemmBlockK, 128, 1, kSwizzle128);
  if (rc) return rc;

  NsParams q = {};
  q.batch = (int)batch;
  q.vec_out = cols % 4 == 0 && aligned_out;
  q.status = status;
  q.wait_budget_ns = kDefaultWaitBudgetNs;
  auto step_products = [&](int step, bool launch) -> int {
    const float* co = coeff + 3 * step;
    const int cur = step & 1;
    NsParams e = q;
    e.rows = e.cols = side;
    e.pitch16 = pitch_a;
    e.K = longer;
    e.out16 = a16;
    e.alpha = (float)(1.0 / (k * k));
    int rc = tall ? ns_gemm<true, true, kNsGram>(xm[cur], xm[cur], e, s, launch) : ns_gemm<false, false, kNsGram>(xk[cur], xk[cur], e, s, launch);
    if (rc) return rc;
    e.K = side;
    e.a16 = a16;
    e.out16 = b16;
    e.alpha = co[2];
    e.beta = co[1];
    rc = ns_gemm<false, false, kNsPoly>(ak, ak, e, s, launch);
    if (rc) return rc;
    NsParams u = q;
    u.rows = rows;
    u.cols = cols;
    u.K = side;
    u.out16 = x[cur ^ 1];
    u.pitch16 = u.pitch_m = pitch;
    u.master = master;
    u.beta = co[0];
    if (step + 1 < steps) {
      rc = tall ? ns_gemm<false, false, kNsUpdate>(xk[cur], bk, u, s, launch) : ns_gemm<false, true, kNsUpdate>(bk, xm[cur], u, s, launch);
    } else if (p == nullptr) {
      u.final_out = out;
      u.alpha = (float)(1.0 / k);
      rc = tall ? ns_gemm<false, false, kNsResult>(xk[cur], bk, u, s, launch) : ns_gemm<false, true, kNsResult>(bk, xm[cur], u, s, launch);
    } else {
      u.final_out = p;
      u.p_bf16 = static_cast<__nv_bfloat16*>(p_bf16);
      u.alpha = (float)(scale / k);
      u.decay = decay;
      rc = tall ? ns_gemm<false, false, kNsStep>(xk[cur], bk, u, s, launch) : ns_gemm<false, true, kNsStep>(bk, xm[cur], u, s, launch);
    }
    return rc;
  };
  // whatever can fail without a launch fails here: the first launch updates the momentum
  for (const int step : {0, steps - 1}) {
    rc = step_products(step, false);
    if (rc) return rc;
  }
  const int parts = blocks_for(vec ? numel / 16 : numel, kNsMaxParts);
  if (vec) ns_norm_kernel<true><<<dim3((unsigned)parts, (unsigned)batch), kNsPrepThreads, 0, s>>>(in, numel, part);
  else ns_norm_kernel<false><<<dim3((unsigned)parts, (unsigned)batch), kNsPrepThreads, 0, s>>>(in, numel, part);
  PKB_CHECK_CUDA(cudaGetLastError());
  const int start_blocks = blocks_for((long long)rows * (pitch / 8), 1 << 20);
  PKB_CHECK_CUDA(launch_dependent(ns_start_kernel, dim3((unsigned)start_blocks, (unsigned)batch), kNsPrepThreads, 0, s, 0, in, rows, cols, (int)pitch,
                                  part, parts, eps, k, (int)(aligned && cols % 8 == 0), master, x[0]));
  for (int step = 0; step < steps; ++step) {
    rc = step_products(step, true);
    if (rc) return rc;
  }
  return kApiOk;
}
