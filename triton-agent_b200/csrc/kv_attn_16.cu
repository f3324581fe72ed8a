// Streaming decode attention and shared-prefix attention over 16-bit caches (kernels:
// kv_attn.cuh, prefix_attn.cuh).
#include "common.cuh"

B200_DEVICE_ERROR_WORD()

#include "prefix_attn.cuh"

B200_DEFINE_PIECE_LAUNCHERS(16, scalar_t)
B200_DEFINE_PREFIX_LAUNCHER(16, scalar_t)
