// C API of libpkb200_cuda.so. Every function returns 0 on success or a pkb::ApiCode; the message
// of the last failure on the calling thread is available from pkb_last_error(). Pointers are raw
// device pointers, `stream` is a cudaStream_t passed as void*. Nothing here allocates device
// memory unless its comment says so.
#pragma once
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

const char* pkb_last_error();
int pkb_version();

// Per-device status block (16 uint32 words): word 0 is the first error code a kernel recorded.
int pkb_status_read(uint32_t* out_words);
int pkb_status_clear();
// Launch a one-thread kernel that waits (at most budget_ns) for *flag >= target.
int pkb_wait_selftest(const void* flag, uint32_t target, uint64_t budget_ns, void* out_elapsed_us,
                      void* stream);

// ---- dense GEMM (tcgen05): C[M,N] = epi(alpha * A[M,K] @ B[N,K]^T + bias) -------------------
// a, b: bf16 row-major with leading dimensions lda, ldb (elements, multiples of 8).
// out_f32: 0 -> C is bf16, 1 -> C is fp32. epilogue: 0 none, 1 SiLU, 2 bias, 3 bias + SiLU.
// block_n: 128 or 256 (0 = choose). num_ctas: 0 = one per SM.
int pkb_gemm_bf16(const void* a, long long lda, const void* b, long long ldb, void* c,
                  long long ldc, int M, int N, int K, const void* bias, float alpha, int epilogue,
                  int out_f32, int block_n, int num_ctas, void* stream);

// ---- normalisation / elementwise ------------------------------------------------------------
// y = x * rsqrt(mean(x^2) + eps) * gamma; x, y, gamma bf16; rows x cols (cols % 8 == 0).
int pkb_rmsnorm_bf16(const void* x, const void* gamma, void* y, int rows, int cols, float eps,
                     void* stream);
// sums `nsrc` row-major bf16 (or fp32) partial buffers (src + i*src_stride_elems), optionally
// scales by `scale`, applies RMSNorm with gamma, writes bf16.
int pkb_sum_rmsnorm(const void* src, long long src_stride_elems, int nsrc, int src_is_f32,
                    const void* gamma, void* y, int rows, int cols, float scale, float eps,
                    void* stream);
// Layer norm of rows x (ldx elements apart, any value) into y [rows, cols]; dtype 0 bf16, 1 fp32; gamma, beta [cols] or null, bf16 or
// (param_f32) fp32; mean, rstd fp32 [rows], both or neither null.
int pkb_layer_norm_fwd(const void* x, long long ldx, const void* gamma, const void* beta, int param_f32, void* y, void* mean, void* rstd,
                       long long rows, int cols, float eps, int dtype, void* stream);
// Its backward: dx, and dgamma, dbeta fp32 [cols]; partial: pkb_layer_norm_bwd_partials(rows, cols, dtype) x 2 x cols fp32 values.
int pkb_layer_norm_bwd_partials(long long rows, int cols, int dtype);
// What it writes of that on a GPU of `sms` SMs (0: the current device), for tensors on 16 bytes throughout or not, and its number of launches.
int pkb_layer_norm_bwd_blocks(long long rows, int cols, int dtype, int aligned, int sms);
int pkb_layer_norm_bwd_launches(long long rows, int cols, int dtype, int aligned, int sms);
int pkb_layer_norm_bwd(const void* x, long long ldx, const void* dy, long long lddy, const void* gamma, int param_f32, const void* mean,
                       const void* rstd, void* dx, void* dgamma, void* dbeta, void* partial, long long rows, int cols, int dtype, void* stream);

// ---- tokens sorted by expert and back, one GPU -----------------------------------------------
// idx int32 [n], values outside [0, experts) are dropped; offsets [experts + 1], order [n], slots [n] int32. experts <= 1024.
int pkb_moe_sort(const void* idx, long long n, int experts, void* offsets, void* order, void* slots, void* stream);
// kept: address of offsets[experts] (device). dtype 0 bf16, 1 fp32. See kernels/moe_sort.cu for the formulas.
int pkb_moe_permute(const void* x, long long ldx, const void* slots, const void* kept, void* xp, long long tokens, int top_k, int hidden, int dtype,
                    void* stream);
int pkb_moe_unpermute(const void* y, long long ldy, const void* slots, const void* gates, void* out, long long tokens, int top_k, int hidden,
                      int dtype, void* stream);
int pkb_moe_unpermute_bwd(const void* dout, long long lddo, const void* y, long long ldy, const void* slots, const void* gates, const void* kept,
                          void* dy, void* dgates, long long tokens, int top_k, int hidden, int dtype, void* stream);

// ---- orthogonalised updates ------------------------------------------------------------------
// Bytes of scratch (256-byte aligned) that pkb_newton_schulz wants for this problem and, where launches is not null, its number of launches.
long long pkb_newton_schulz_scratch(long long batch, int rows, int cols, int steps, int* launches);
// coeff: HOST array of `steps` triples. m (fp32 momentum, updated) may be null. One of out (bf16) and p (fp32, updated; p_bf16 its copy or null).
int pkb_newton_schulz(const void* g, int g_f32, void* m, float momentum, int nesterov, long long batch, int rows, int cols, const float* coeff,
                      int steps, double eps, void* out, void* p, float decay, float scale, void* p_bf16, void* scratch, void* stream);

#ifdef __cplusplus
}
#endif
