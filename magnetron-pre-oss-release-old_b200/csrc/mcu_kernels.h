/*
 * mcu_kernels.h - C-callable launchers of the sm_100a kernels.
 *
 * Every launcher enqueues on the given stream and returns a cudaError_t value
 * (0 on success).  Tensors are f32, strides are in elements, dim 0 is the
 * fastest dimension, exactly as in the magnetron core.
 */
#ifndef MCU_KERNELS_H
#define MCU_KERNELS_H
#include <stdint.h>
#include <stddef.h>
#include <cuda_runtime_api.h>
#include "magnetron_cuda.h"

#ifdef __cplusplus
extern "C" {
#endif

/* k_elementwise.cu */
int mcu_launch_unary(int op, float* r, const float* x, int64_t rows, int64_t cols, int64_t r_s1, int64_t x_s1,
                     float xi, cudaStream_t st);
int mcu_launch_binary(int op, float* r, const float* x, const float* y, const int64_t* x_dims,
                      const int64_t* x_strides, const int64_t* r_strides, const int64_t* y_dims,
                      const int64_t* y_strides, cudaStream_t st);
int mcu_launch_bcast2(int op, float* r, const float* x, const float* y, const int64_t* r_dims,
                      const int64_t* x_dims, const int64_t* y_dims, cudaStream_t st);

/* k_reduce.cu: scratch needs mcu_reduce_scratch_bytes() bytes of device memory. */
size_t mcu_reduce_scratch_bytes(void);
int mcu_launch_reduce(int op, float* r, const float* x, const int64_t* x_dims, const int64_t* x_strides,
                      void* scratch, cudaStream_t st);
/* One shard's full-reduction record (a sharded SUM/MEAN/MIN/MAX exchanges these). */
typedef struct McuReducePart {
    double sum;
    float min, max;
    uint64_t count;
} McuReducePart;
int mcu_launch_reduce_partial(McuReducePart* part, const float* x, const int64_t* x_dims, const int64_t* x_strides,
                              void* scratch, cudaStream_t st);
int mcu_launch_reduce_combine(int op, float* r, const McuReducePart* parts, int nparts, cudaStream_t st);
int mcu_launch_reduce_rows(int op, float* r, const float* x, int64_t rows, int64_t cols, cudaStream_t st);
/* Normalised row softmax; scratch needs mcu_softmax_rows_scratch_bytes(rows, cols) bytes
 * (nonzero only for rows wider than 65536, whose fallback, when their cluster shape cannot be
 * scheduled, takes two passes over slice statistics and a per-row combine). */
size_t mcu_softmax_rows_scratch_bytes(int64_t rows, int64_t cols);
int mcu_softmax_rows_kernels(int64_t rows, int64_t cols); /* kernel launches of one call */
int mcu_launch_softmax_rows(float* r, const float* x, int64_t rows, int64_t cols, void* scratch, cudaStream_t st);

/* k_fill.cu: PCG stream fills (normal != 0: Box-Muller pairs; p0, p1 = mean, stddev,
 * else p0, p1 = min, max - min) and constant fills. */
uint64_t mcu_pcg_advance(uint64_t state, uint64_t inc, uint64_t n);
int mcu_launch_fill_pcg(float* r, int64_t n, int normal, float p0, float p1, uint64_t state, uint64_t inc,
                        cudaStream_t st);
int mcu_launch_fill_const(float* r, int64_t n, float x, cudaStream_t st);
/* k_fill_mt.cu: fills from the Mersenne-twister stream of st = {remaining, next, state[624]},
 * which is left as the host generator leaves it (the call waits when it draws past the current
 * block).  *launches = kernels launched. */
size_t mcu_fill_mt_scratch_bytes(int64_t n, uint32_t remaining, uint32_t next);
int mcu_launch_fill_mt(float* r, int64_t n, int normal, float p0, float p1, uint32_t* st, void* scratch,
                       cudaStream_t stream, int* launches);
int mcu_mt19937_degree(void);
int mcu_mt19937_jump_host(const uint32_t* win, uint64_t d, uint32_t* out);

/* k_image.cu: planar f32 [c][h][w] <-> interleaved u8 [h][w][c] (resized to rw x rh when both
 * are nonzero, with ws = (w-1)/(rw-1), hs = (h-1)/(rh-1) rounded to f32), box and text drawing
 * on 3-channel images; glyphs holds (x, y, glyph index) triples. */
int mcu_launch_img_from_u8(float* dst, const uint8_t* src, uint32_t w, uint32_t h, uint32_t c, uint32_t rw,
                           uint32_t rh, float ws, float hs, cudaStream_t st);
int mcu_launch_img_to_u8(uint8_t* dst, const float* src, uint32_t w, uint32_t h, uint32_t c, cudaStream_t st);
int mcu_launch_img_draw_box(float* img, int32_t w, int32_t h, int32_t x1, int32_t y1, int32_t x2, int32_t y2,
                            int32_t wi, float r, float g, float b, cudaStream_t st);
int mcu_launch_img_draw_text(float* img, int32_t w, int32_t h, const int32_t* glyphs, int32_t n, float r, float g,
                             float b, cudaStream_t st);

/* k_matmul_exact.cu: R[b][i*r_ld + j] = (accumulate ? R : 0) + sum_k X[b][i*K+k]*Y[b][k*N+j],
 * summed k = 0..K-1 in order with separately rounded multiply and add. */
int mcu_launch_matmul_exact(float* r, const float* x, const float* y, int64_t batch, int64_t M, int64_t K,
                            int64_t N, int64_t r_ld, int accumulate, cudaStream_t st);
/* A single bit-exact product with a fused dense-layer epilogue: r = act(xy + bias), the bias
 * read at the flat result index (bias_mod = 0) or at that index mod bias_mod (a bias broadcast
 * along dim 0), act 0 none, 1 GELU, 2 SIGMOID (their vector-lane formulas).  At most 1048560
 * rows. */
int mcu_launch_matmul_exact_ep(float* r, const float* x, const float* y, int64_t M, int64_t K, int64_t N,
                               const float* bias, int64_t bias_mod, int act, cudaStream_t st);
/* Kernels one exact product launches: a single product of more than 1048560 rows runs in slices. */
int mcu_matmul_exact_kernels(int64_t batch, int64_t M);
/* Largest K the tensor-core product takes (its padded K indexes a grid dimension); beyond it the
 * CUDA-core paths, which have no K limit, run the product. */
#define MCU_TC_MAX_K (((int64_t)1 << 21) - 32)

size_t mcu_matmul_skinny_scratch_bytes(int64_t M, int64_t K, int64_t N);
int mcu_launch_matmul_skinny(float* r, const float* x, const float* y, int64_t M, int64_t K, int64_t N,
                             int64_t r_ld, void* scratch, cudaStream_t st);

/* Allocation-free skinny product: scratch is a fixed device array of this library. */
size_t mcu_skinny_noalloc_limit(void);
int mcu_skinny_noalloc_scratch(void** out);

/* k_matmul_tc.cu: tcgen05 GEMM with a three-product split, R[M,N] = X[M,K] Y[K,N] (row-major);
 * f16 = 0: tf32 hi/lo split (kind::tf32), f16 = 1: scaled f16 hi/lo split (kind::f16).
 * scratch needs mcu_matmul_tc_scratch_bytes(M, K, N) bytes (either split). */
size_t mcu_matmul_tc_scratch_bytes(int64_t M, int64_t K, int64_t N);
/* Kernels one single (unbatched) product launches: operand splits, the GEMM, and the part sum
 * when K is split (for few tiles, or for the tiles of a mostly empty last wave); flags bit 0:
 * X arrives split by the previous layer's epilogue (tf32), bit 1: fused dense-layer epilogue. */
int mcu_matmul_tc_kernels(int64_t M, int64_t K, int64_t N, int f16, int flags);
int mcu_launch_matmul_tc(float* r, const float* x, const float* y, int64_t M, int64_t K, int64_t N,
                         void* scratch, int* status, cudaStream_t st, int f16);
int mcu_matmul_tc_supported(void);

/* Fused dense-layer epilogue for the tensor-core GEMM: out = act(X Y + bias) with
 * bias at the result's row-major index (or NULL), act 0 = none, 1 = GELU; when
 * out_hi/out_lo are set the tf32 hi/lo split of out is also written in the
 * [M][kp_out] layout the next product reads (kp_out = N rounded up to 32, N % 32 == 0).
 * a_hi/a_lo, when set, are X already split in that layout (no split pass).  The split
 * fields apply to the tf32 split only; the f16 split always splits X itself. */
typedef struct mcu_tc_epilogue {
    const float* a_hi;
    const float* a_lo;
    const float* bias;
    float* out_hi;
    float* out_lo;
    int64_t kp_out;
    int act;
    int bias_zero; /* the bias is known to be zero: add +0.0f (which maps -0 to +0) and read nothing */
} mcu_tc_epilogue;
size_t mcu_matmul_tc_batched_scratch_bytes(int64_t B, int64_t M, int64_t K, int64_t N);
int mcu_matmul_tc_batched_kernels(int64_t B, int64_t M, int64_t K, int64_t N, int f16);
int mcu_launch_matmul_tc_batched(float* r, const float* x, const float* y, int64_t B, int64_t M, int64_t K,
                                 int64_t N, void* scratch, int* status, cudaStream_t st, int f16);
int mcu_launch_matmul_tc_ex(float* r, const float* x, const float* y, int64_t M, int64_t K, int64_t N,
                            void* scratch, int* status, cudaStream_t st, const mcu_tc_epilogue* ep, int f16);

/* The language-model row operators: arguments as in magnetron_cuda.h, already checked, rows (M, N) > 0.
 * *launches = kernels launched. */
/* k_rmsnorm.cu: the backward pass needs mcu_rmsnorm_backward_scratch_bytes of scratch when dw is set. */
int mcu_launch_rmsnorm(float* y, uint8_t* q, float* s, float* h, float* rstd, const float* x, const float* res,
                       const float* w, float eps, int64_t rows, int64_t cols, cudaStream_t st, int* launches);
size_t mcu_rmsnorm_backward_scratch_bytes(int64_t rows, int64_t cols);
int mcu_launch_rmsnorm_backward(float* dx, float* dw, const float* dy, const float* h, const float* w,
                                const float* rstd, const float* dh, int64_t rows, int64_t cols, void* scratch, int* status,
                                cudaStream_t st, int* launches);
/* k_quantize_e4m3.cu */
int mcu_launch_quantize_e4m3(uint8_t* q, float* s, const float* x, int64_t rows, int64_t cols, int block,
                             int transpose, cudaStream_t st, int* launches);
/* k_matmul_e4m3.cu */
int mcu_launch_matmul_e4m3(float* r, const uint8_t* xq, const float* xs, const uint8_t* yq, const float* ys, int64_t M,
                           int64_t K, int64_t N, int y_block, int* status, cudaStream_t st, int* launches);
/* k_logprobs.cu */
int mcu_launch_logprobs(float* logp, float* lse, float* entropy, float* top_logp, int32_t* top_id, const float* x,
                        const int32_t* id, int64_t rows, int64_t cols, int64_t x_s1, int top, cudaStream_t st,
                        int* launches);
int mcu_launch_logprobs_backward(float* dx, const float* x, const int32_t* id, const float* lse, const float* entropy,
                                 const float* g_logp, const float* g_entropy, int64_t rows, int64_t cols, int64_t x_s1,
                                 int64_t dx_s1, cudaStream_t st, int* launches);

/* k_heads.cu: the rotation's rot is 0 where there is none; the backward pass needs
 * mcu_rotate_heads_backward_scratch_bytes of scratch when dw is set.  q_heads = 0: no queries. */
int mcu_launch_rotate_heads(float* y, float* rstd, const float* x, const float* w, float eps, const mag_cuda_rotation* rot,
                            int64_t rows, int64_t heads, int64_t head_dim, int64_t x_s1, int64_t y_s1, cudaStream_t st,
                            int* launches);
size_t mcu_rotate_heads_backward_scratch_bytes(int64_t rows, int64_t heads, int64_t head_dim);
int mcu_launch_rotate_heads_backward(float* dx, float* dw, const float* dy, const float* x, const float* w, const float* rstd,
                                     const mag_cuda_rotation* rot, int64_t rows, int64_t heads, int64_t head_dim,
                                     int64_t dx_s1, int64_t dy_s1, int64_t x_s1, void* scratch, cudaStream_t st,
                                     int* launches);
int mcu_launch_kv_write(const mag_cuda_kv_cache* cache, const int32_t* slot, const float* k, const float* v, const float* k_w,
                        float* q_out, const float* q, const float* q_w, float eps, const mag_cuda_rotation* rot, int64_t rows,
                        int64_t q_heads, int64_t k_s1, int64_t v_s1, int64_t q_s1, int64_t q_out_s1, cudaStream_t st,
                        int* launches);
int mcu_launch_kv_read(const mag_cuda_kv_cache* cache, float* k, float* v, const int32_t* slot, int64_t rows, int64_t k_s1,
                       int64_t v_s1, cudaStream_t st, int* launches);
/* k_attention.cu: one call's arguments as in magnetron_cuda.h (window below 2^31 + 1). */
typedef struct mcu_attention {
    float* out;
    float* lse;
    const float* q;
    mag_cuda_kv_cache cache;
    const int32_t* table;
    const int32_t* start;
    const int32_t* length;
    int64_t seqs, table_s1, rows, max_new, q_heads;
    float scale;
    int64_t window, q_s1, out_s1;
} mcu_attention;
size_t mcu_attention_scratch_bytes(const mcu_attention* a);
/* joins: MCU_COUNTERS words, zero, which the call leaves zero; null: words of the scratch, cleared on the stream first (3 us). */
int mcu_launch_attention(const mcu_attention* a, void* scratch, uint32_t* joins, int* status, cudaStream_t st, int* launches);

#ifdef __cplusplus
}
#endif
#endif
