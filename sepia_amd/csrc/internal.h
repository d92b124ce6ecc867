/* internal.h -- what the other host files of libsepia_hip.so (store.c,
 * serve.c) use of sepia_hip.c. Not exported. */
#ifndef SEPIA_INTERNAL_H
#define SEPIA_INTERNAL_H

#define __HIP_PLATFORM_AMD__ 1
#include <hip/hip_runtime_api.h>

#include <stddef.h>
#include <stdint.h>

#include "../../include/sepia_gpu.h"

#define SEPIA_HIDDEN __attribute__((visibility("hidden")))

/* One "sepia: hip: ..." line on stderr. */
SEPIA_HIDDEN void sepia_log(const char *fmt, ...) __attribute__((format(printf, 1, 2)));
/* 1 if sepia_gpu_init succeeded (else logs for op). */
SEPIA_HIDDEN int sepia_ready(const char *op);
/* The library's stream. */
SEPIA_HIDDEN hipStream_t sepia_stream(void);
/* A buffer's device address and length. */
SEPIA_HIDDEN uint8_t *sepia_buf_dev(SepiaGpuBuf *b);
SEPIA_HIDDEN size_t sepia_buf_len(const SepiaGpuBuf *b);
/* Bytes of a row of n elements of a ggml type; -1 for an unknown type or an
 * n that is not a whole number of blocks (reference quants_row_bytes,
 * src/quants.c:45-56). */
SEPIA_HIDDEN int64_t sepia_row_bytes(int ggml_type, int64_t n);
/* Count one device or pinned-host allocation (sepia_hip_alloc_count). */
SEPIA_HIDDEN void sepia_count_alloc(void);
/* An op's checks and preparations (serve.c), as sepia_hip.c's own ops make
 * them: an open batch; [off, off + n) inside a buffer; an input's host-written
 * parts of a range uploaded; an output's device copy current, and downloaded
 * at sepia_gpu_end. Each logs and returns 0 on failure. */
SEPIA_HIDDEN int sepia_need_batch(const char *op);
SEPIA_HIDDEN int sepia_chk(const SepiaGpuBuf *b, size_t off, size_t n, const char *op, const char *what);
SEPIA_HIDDEN int sepia_prep_in(SepiaGpuBuf *b, size_t off, size_t n, const char *op);
SEPIA_HIDDEN int sepia_prep_out(SepiaGpuBuf *b, const char *op);
/* The scratch's data region of at least `need` bytes (NULL: logged), and how
 * many a call may ask for: what there is while the stream is being captured,
 * else any number. */
SEPIA_HIDDEN void *sepia_scratch(size_t need, const char *op);
/* Once there is scratch: SEPIA_COUNTERS arrival counters in front of it, zero
 * between launches (a kernel that uses one leaves it so). */
#define SEPIA_COUNTERS 16384
SEPIA_HIDDEN uint32_t *sepia_counters(void);
SEPIA_HIDDEN size_t sepia_scratch_limit(void);

/* Kernels of the second code object (kernels/sepia_serve.hip), and a launch
 * of one on the library's stream, timed when the profiler is on. */
enum { SK_KV8_APPEND, SK_KV8_READ, SK_KV8_ATTN, SK_KV8_ROWS = SK_KV8_ATTN + 4,   /* head dims 128, up to 128, 64, up to 64 */
       SK_SAMPLE_MAX = SK_KV8_ROWS + 4, SK_SAMPLE_BINS, SK_SAMPLE_PICK, SK_SAMPLE, SK_COUNT };
SEPIA_HIDDEN int sepia_serve_launch(int k, uint64_t gx, unsigned gy, unsigned gz, unsigned block, void **args,
                                    const char *op);

/* Release store.c's pinned staging buffers (sepia_gpu_shutdown calls it). */
SEPIA_HIDDEN void sepia_store_shutdown(void);

#endif
