// Streaming decode attention over 16-bit caches (kernels: kv_attn.cuh).
#include "common.cuh"

B200_DEVICE_ERROR_WORD()

#include "kv_attn.cuh"

B200_DEFINE_PIECE_LAUNCHERS(16, scalar_t)
