// Streaming decode attention over int8 caches (kernels: kv_attn.cuh).
#include "common.cuh"

B200_DEVICE_ERROR_WORD()

#include "kv_attn.cuh"

B200_DEFINE_PIECE_LAUNCHERS(i8, int8_t)
