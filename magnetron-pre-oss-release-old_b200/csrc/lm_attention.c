/*
 * lm_attention.c - entry points of the attention operators (host side, C): argument checks, buffer bookkeeping and
 * launch of the head norm and rotation, the paged cache's write and read, and attention over the cache.
 * Nothing of the device is touched before the arguments have been checked.
 */
#include "magnetron_cuda.h"
#include "mcu_args.h"
#include "mcu_device.h"
#include "mcu_kernels.h"

#include <math.h>

#define MCU_MAX_HEADS 65535

/* Rows of `heads` head rows each, stride s1 apart. */
static int bad_heads(int64_t rows, int64_t heads, int64_t head_dim, int64_t s1) {
    return heads < 1 || heads > MCU_MAX_HEADS || s1 < heads * head_dim || s1 >= MCU_MAX_DIM || bad_matrix(rows, s1);
}

static int bad_eps(float eps) { return !(eps >= 0.0f) || isinf(eps); }

static int bad_rotation(const mag_cuda_rotation* r, int64_t head_dim) {
    if (!r || !r->rot) return 0;
    return r->rot < 0 || r->rot > head_dim || r->rot % 8 || !r->pos || !r->inv_freq || odd4(r->pos) || odd4(r->inv_freq) ||
           !isfinite(r->magnitude);
}

static mag_cuda_rotation rotation_of(const mag_cuda_rotation* r) {
    const mag_cuda_rotation none = {0};
    return r && r->rot ? *r : none;
}

static int bad_cache(const mag_cuda_kv_cache* c) {
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale || odd16(c->k) || odd16(c->v) || odd16(c->k_scale) || odd16(c->v_scale))
        return 1;
    if (c->pages < 1 || c->heads < 1 || c->heads > MCU_MAX_HEADS || c->head_dim < 16 || c->head_dim > 128 || c->head_dim % 16) return 1;
    if (c->page_size < 16 || c->page_size > 1024 || (c->page_size & (c->page_size - 1))) return 1;
    const int64_t slots = (int64_t)c->pages * c->page_size;
    return slots >= ((int64_t)1 << 31) || slots * c->heads > (((int64_t)1 << 42) / c->head_dim);
}

/* Rows that fill their stride are written whole; of padded rows the padding keeps what it holds. */
static size_t out_bytes(int64_t rows, int64_t width, int64_t s1) { return width == s1 ? (size_t)(rows * s1) * 4 : 4; }

int mag_cuda_rotate_heads_f32(mag_compute_device_t* dvc, float* y, float* rstd, const float* x, const float* w, float eps,
                              const mag_cuda_rotation* rotation, int64_t rows, int64_t heads, int64_t head_dim, int64_t x_s1,
                              int64_t y_s1) {
    if (!dvc || !y || !x || (rstd && !w) || head_dim < 8 || head_dim > 256 || head_dim % 8 || bad_heads(rows, heads, head_dim, x_s1) ||
        bad_heads(rows, heads, head_dim, y_s1) || bad_eps(eps) || bad_rotation(rotation, head_dim) || (y == x && x_s1 != y_s1) ||
        odd4(y) || odd4(rstd) || odd4(x) || odd4(w))
        return MAG_CUDA_E_INVALID;
    if (!rows) return 0;
    const mag_cuda_rotation rot = rotation_of(rotation);
    const mcu_buf bufs[] = {{x, 0, 0}, {w, 0, 0}, {rot.pos, 0, 0}, {rot.inv_freq, 0, 0},
                            {y, out_bytes(rows, heads * head_dim, y_s1), 1}, {rstd, (size_t)(rows * heads) * 4, 1}};
    mcu_call c;
    int k = 0, rc = mcu_call_begin(&c, dvc, bufs, 6, 0);
    if (rc) return rc;
    rc = mcu_launch_rotate_heads(y, rstd, x, w, eps, &rot, rows, heads, head_dim, x_s1, y_s1, c.stream, &k);
    return mcu_call_end(&c, rc, k);
}

int mag_cuda_rotate_heads_backward_f32(mag_compute_device_t* dvc, float* dx, float* dw, const float* dy, const float* x,
                                       const float* w, const float* rstd, const mag_cuda_rotation* rotation, int64_t rows,
                                       int64_t heads, int64_t head_dim, int64_t dx_s1, int64_t dy_s1, int64_t x_s1) {
    if (!dvc || !dx || !dy || (w ? !x || !rstd : x || rstd || dw) || head_dim < 8 || head_dim > 256 || head_dim % 8 ||
        bad_heads(rows, heads, head_dim, dx_s1) || bad_heads(rows, heads, head_dim, dy_s1) ||
        (x && bad_heads(rows, heads, head_dim, x_s1)) || bad_rotation(rotation, head_dim) || (dx == dy && dx_s1 != dy_s1) ||
        (dx == x && dx_s1 != x_s1) || odd4(dx) || odd4(dw) || odd4(dy) || odd4(x) || odd4(w) || odd4(rstd))
        return MAG_CUDA_E_INVALID;
    const mag_cuda_rotation rot = rotation_of(rotation);
    const mcu_buf bufs[] = {{dy, 0, 0}, {x, 0, 0}, {w, 0, 0}, {rstd, 0, 0}, {rot.pos, 0, 0}, {rot.inv_freq, 0, 0},
                            {dx, out_bytes(rows, heads * head_dim, dx_s1), 1}, {dw, (size_t)head_dim * 4, 1}};
    mcu_call c;
    int k = 0, rc;
    if (!rows) {
        if (!dw) return 0;
        if ((rc = mcu_call_begin(&c, dvc, bufs + 7, 1, 0))) return rc;
        return mcu_call_end(&c, (int)cudaMemsetAsync(dw, 0, (size_t)head_dim * 4, c.stream), 0);
    }
    rc = mcu_call_begin(&c, dvc, bufs, 8, dw ? mcu_rotate_heads_backward_scratch_bytes(rows, heads, head_dim) : 0);
    if (rc) return rc;
    rc = mcu_launch_rotate_heads_backward(dx, dw, dy, x, w, rstd, &rot, rows, heads, head_dim, dx_s1, dy_s1, x_s1, c.scratch,
                                          c.stream, &k);
    return mcu_call_end(&c, rc, k);
}

int mag_cuda_kv_write(mag_compute_device_t* dvc, const mag_cuda_kv_cache* cache, const int32_t* slot, const float* k,
                      const float* v, const float* k_w, float* q_out, const float* q, const float* q_w, float eps,
                      const mag_cuda_rotation* rotation, int64_t rows, int64_t q_heads, int64_t k_s1, int64_t v_s1,
                      int64_t q_s1, int64_t q_out_s1) {
    if (!dvc || bad_cache(cache) || !slot || !k || !v || !q != !q_out || (q_w && !q) || bad_heads(rows, cache->heads, cache->head_dim, k_s1) ||
        bad_heads(rows, cache->heads, cache->head_dim, v_s1) || bad_eps(eps) || bad_rotation(rotation, cache->head_dim) ||
        odd4(slot) || odd4(k) || odd4(v) || odd4(k_w) || odd4(q) || odd4(q_out) || odd4(q_w))
        return MAG_CUDA_E_INVALID;
    if (q && (bad_heads(rows, q_heads, cache->head_dim, q_s1) || bad_heads(rows, q_heads, cache->head_dim, q_out_s1) ||
              (q == q_out && q_s1 != q_out_s1)))
        return MAG_CUDA_E_INVALID;
    if (!rows) return 0;
    const mag_cuda_rotation rot = rotation_of(rotation);
    const mcu_buf bufs[] = {{slot, 0, 0}, {k, 0, 0}, {v, 0, 0}, {k_w, 0, 0}, {q, 0, 0}, {q_w, 0, 0}, {rot.pos, 0, 0}, {rot.inv_freq, 0, 0},
                            {cache->k, 1, 1}, {cache->v, 1, 1}, {cache->k_scale, 1, 1}, {cache->v_scale, 1, 1},
                            {q_out, q ? out_bytes(rows, q_heads * cache->head_dim, q_out_s1) : 0, 1}};
    mcu_call c;
    int n = 0, rc = mcu_call_begin(&c, dvc, bufs, 13, 0);
    if (rc) return rc;
    rc = mcu_launch_kv_write(cache, slot, k, v, k_w, q_out, q, q_w, eps, &rot, rows, q ? q_heads : 0, k_s1, v_s1, q_s1, q_out_s1,
                             c.stream, &n);
    return mcu_call_end(&c, rc, n);
}

int mag_cuda_kv_read(mag_compute_device_t* dvc, const mag_cuda_kv_cache* cache, float* k, float* v, const int32_t* slot,
                     int64_t rows, int64_t k_s1, int64_t v_s1) {
    if (!dvc || bad_cache(cache) || !slot || (!k && !v) || rows < 0 || (k && bad_heads(rows, cache->heads, cache->head_dim, k_s1)) ||
        (v && bad_heads(rows, cache->heads, cache->head_dim, v_s1)) || k == v || odd4(slot) || odd4(k) || odd4(v))
        return MAG_CUDA_E_INVALID;
    if (!rows) return 0;
    const int64_t width = (int64_t)cache->heads * cache->head_dim;
    const mcu_buf bufs[] = {{slot, 0, 0}, {cache->k, 0, 0}, {cache->v, 0, 0}, {cache->k_scale, 0, 0}, {cache->v_scale, 0, 0},
                            {k, out_bytes(rows, width, k_s1), 1}, {v, out_bytes(rows, width, v_s1), 1}};
    mcu_call c;
    int n = 0, rc = mcu_call_begin(&c, dvc, bufs, 7, 0);
    if (rc) return rc;
    rc = mcu_launch_kv_read(cache, k, v, slot, rows, k_s1, v_s1, c.stream, &n);
    return mcu_call_end(&c, rc, n);
}

int mag_cuda_attention_paged_f32(mag_compute_device_t* dvc, float* out, float* lse, const float* q,
                                 const mag_cuda_kv_cache* cache, const int32_t* table, const int32_t* start,
                                 const int32_t* length, int64_t seqs, int64_t table_s1, int64_t rows, int64_t max_new,
                                 int64_t q_heads, float scale, int64_t window, int64_t q_s1, int64_t out_s1) {
    if (!dvc || !out || !q || bad_cache(cache) || !table || !start || !length || bad_matrix(seqs, table_s1) ||
        table_s1 * cache->page_size >= MCU_MAX_DIM || max_new < 0 || max_new >= MCU_MAX_DIM || q_heads % cache->heads ||
        bad_heads(rows, q_heads, cache->head_dim, q_s1) || bad_heads(rows, q_heads, cache->head_dim, out_s1) || !(scale >= 0.0f) ||
        isinf(scale) || window < 0 || out == q || odd4(out) || odd4(lse) || odd4(q) || odd4(table) || odd4(start) || odd4(length))
        return MAG_CUDA_E_INVALID;
    if (!rows || !seqs || !max_new) return 0;
    /* rows behind the last sequence are left as they were */
    const mcu_buf bufs[] = {{q, 0, 0}, {cache->k, 0, 0}, {cache->v, 0, 0}, {cache->k_scale, 0, 0}, {cache->v_scale, 0, 0},
                            {table, 0, 0}, {start, 0, 0}, {length, 0, 0}, {out, 1, 1}, {lse, 1, 1}};
    if (window > ((int64_t)1 << 31)) window = 0; /* longer than any sequence */
    const mcu_attention a = {out, lse, q, *cache, table, start, length, seqs, table_s1, rows, max_new, q_heads, scale, window, q_s1, out_s1};
    mcu_call c;
    int n = 0, rc = mcu_call_begin(&c, dvc, bufs, 10, mcu_attention_scratch_bytes(&a));
    if (rc) return rc;
    rc = mcu_launch_attention(&a, c.scratch, mcu_call_counters(&c), c.status, c.stream, &n);
    return mcu_call_end(&c, rc, n);
}
