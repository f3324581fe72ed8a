// Streaming decode attention and shared-prefix attention over e4m3 caches (kernels:
// kv_attn.cuh, prefix_attn.cuh).
#include "common.cuh"

B200_DEVICE_ERROR_WORD()

#include "prefix_attn.cuh"

B200_DEFINE_PIECE_LAUNCHERS(e4m3, e4m3_t)
B200_DEFINE_PREFIX_LAUNCHER(e4m3, e4m3_t)
