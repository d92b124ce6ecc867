// sepia_serve.hip -- the serving operators' gfx950 kernels, a code object of
// their own (sepia_serve.hsaco), so that the kernels of sepia_kernels.hsaco
// keep their places: some of those measured differently when moved.
#include "common.h"
#include "kv8.h"
#include "kv8_attn.h"
#include "sample.h"

// The device error word's address (common.h); the host writes it right after
// loading this code object.
extern "C" __constant__ uint32_t *sepia_err_word = nullptr;
