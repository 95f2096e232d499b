/* Argument checks that the language-model entry points share (lm_rows.c, lm_attention.c). */
#ifndef MCU_ARGS_H
#define MCU_ARGS_H
#include <stdint.h>

#define MCU_MAX_DIM (((int64_t)1 << 31) - 256)

static int odd4(const void* p) { return ((uintptr_t)p & 3) != 0; }
static int odd16(const void* p) { return ((uintptr_t)p & 15) != 0; }

/* Row counts and widths that the kernels index (their product stays far below 2^63). */
static int bad_matrix(int64_t rows, int64_t cols) {
    return rows < 0 || rows >= MCU_MAX_DIM || cols < 1 || cols >= MCU_MAX_DIM || rows * cols > ((int64_t)1 << 42);
}

#endif
