// Streaming decode attention and shared-prefix attention over int8 caches (kernels:
// kv_attn.cuh, prefix_attn.cuh).
#include "common.cuh"

B200_DEVICE_ERROR_WORD()

#include "prefix_attn.cuh"

B200_DEFINE_PIECE_LAUNCHERS(i8, int8_t)
B200_DEFINE_PREFIX_LAUNCHER(i8, int8_t)
