// Streaming decode attention over e4m3 caches (kernels: kv_attn.cuh).
#include "common.cuh"

B200_DEVICE_ERROR_WORD()

#include "kv_attn.cuh"

B200_DEFINE_PIECE_LAUNCHERS(e4m3, e4m3_t)
