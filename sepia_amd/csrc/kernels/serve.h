// serve.h -- what the serving kernels share.
#pragma once

// Kernel entry: the first BYTES of the arguments, a scalar load a 64-byte line,
// waited for at once; else each group of them that a branch reads is a memory
// round trip of its own. BYTES is at most the kernel's argument segment.
template <int BYTES>
__device__ __forceinline__ void serve_args() {
    const __attribute__((address_space(4))) uint32_t *ka =
        (const __attribute__((address_space(4))) uint32_t *)__builtin_amdgcn_kernarg_segment_ptr();
    uint32_t acc = 0;
#pragma unroll
    for (int o = 0; o < BYTES; o += 64) acc ^= ka[o / 4];
    asm volatile("" : : "s"(acc));
}
