/* Device state that host modules other than device.c use (storage.c, lm_rows.c). */
#ifndef MCU_DEVICE_H
#define MCU_DEVICE_H

#include "mag_cuda_abi.h"

#include <cuda_runtime_api.h>
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

int mcu_dev_ordinal(mag_compute_device_t* dvc);
/* Waits for the device stream; returns a CUDA error or a kernel status code. */
int mcu_dev_sync(mag_compute_device_t* dvc);
/* Buffer bookkeeping for data read (p) or written (bytes at p) outside the device stream's ops. */
void mcu_dev_in(mag_compute_device_t* dvc, const void* p);
void mcu_dev_out(mag_compute_device_t* dvc, void* p, size_t bytes);

/* The buffers of one call, checked and booked together.  Null pointers are skipped. */
typedef struct mcu_buf {
    const void* p;
    size_t bytes; /* outputs: the bytes written */
    int out;
} mcu_buf;
/* One call on the device's stream: makes the device current, books the buffers and finds scratch.
 * While the stream is being captured the scratch is the graph's own (allocated and freed by nodes of
 * it), buffers that need a clear or a wait first are refused, and the buffers' later clears and
 * asynchronous copies are put on the stream at once, since a replay does not look for them.  mcu_call_end undoes both and
 * returns rc, or the error that ending met. */
typedef struct mcu_call {
    mag_compute_device_t* dvc;
    cudaStream_t stream;
    int* status; /* the device's status word of bounded waits */
    void* scratch;
    int prev_device;
    int own_scratch;
    int captured;
} mcu_call;
/* MCU_COUNTERS words of device memory that are zero between the launches of kernels that count on them.  Eager calls, which the
 * stream puts in order, share a set; each captured graph has one of its own, so that replays may run beside others.  Null
 * once MCU_COUNTER_SETS graphs have had theirs: the call then needs words of its own. */
enum { MCU_COUNTERS = 512, MCU_COUNTER_SETS = 512 };
uint32_t* mcu_call_counters(mcu_call* c);
int mcu_call_begin(mcu_call* c, mag_compute_device_t* dvc, const mcu_buf* bufs, int n, size_t scratch_bytes);
int mcu_call_end(mcu_call* c, int rc, int kernels);

#ifdef __cplusplus
}
#endif
#endif
