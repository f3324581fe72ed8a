// The 8-bit paged KV cache: rows quantised as they are appended, and whole
// contexts read back.
//
// A cached row (the D values of one token and one kv head) is D 8-bit codes
// and one fp32 scale:
//   amax = max|x|,  s = max(amax / qmax, 1e-12)
//   int8 (qmax 127): code = clamp(round_half_even(x / s), -127, 127)
//   e4m3 (qmax 448): code = nearest e4m3 value to x / s (half to even)
//   value read back: code * s
// with x in fp32 -- for K the rotated row before any rounding to 16 bits, so
// the only rounding a cached key sees is that of its code.  Every product,
// sum and quotient is rounded on its own (no FMA contraction; the quotients
// by a correction step), so codes and scales are bit-identical to the same
// formula evaluated in fp32 by any IEEE host.  A row that holds an infinity or a NaN gets a NaN
// scale and reads back as NaN.
//
// Layouts: codes [num_blocks, block_size, Hkv, D], as the 16-bit cache;
// scales [num_blocks, Hkv, block_size], so that the scales of consecutive heads of a page
// are contiguous (one bulk copy for the attention kernel that reads them).
#include "common.cuh"
#include "kv8.cuh"
#include "sm100.cuh"

namespace b200 {
namespace {

constexpr float kScaleFloor = 1e-12f;
// Appends of at most this many tokens find colliding slots by a scan of the later
// slots (one or two loads a thread); larger ones by the table below.
constexpr int64_t kScanTokens = 512;

// ---------------------------------------------------------------------------
// Colliding slots.  The last token that names a slot is the one written, as in
// the 16-bit append.  For many tokens an open-addressing table (twice as many
// entries as tokens or more, cleared by each call, so calls share no state)
// maps a slot to 1 + the last token naming it: O(T) against O(T^2) for the scan.
// ---------------------------------------------------------------------------
struct ClaimTable {
  unsigned long long* keys;  // slot + 1; 0 = empty
  int* owner;                // 1 + last token
  uint32_t mask;             // entries - 1
};

inline int64_t claim_entries(int64_t n_tok) {
  if (n_tok <= kScanTokens) return 0;
  int64_t n = 2;
  while (n < 2 * n_tok) n *= 2;
  return n;
}

__device__ __forceinline__ uint32_t claim_hash(int64_t slot) {
  uint64_t h = (uint64_t)slot * 0x9E3779B97F4A7C15ull;  // Fibonacci hashing (Knuth)
  return (uint32_t)(h >> 32);
}

__device__ __forceinline__ bool token_writes(const int64_t* __restrict__ slots, const int64_t* __restrict__ positions,
                                             int64_t t, int64_t slot_hi, int64_t cs_rows) {
  const int64_t slot = slots[t], pos = positions[t];
  return slot >= 0 && slot < slot_hi && pos >= 0 && pos < cs_rows;
}

__global__ void slot_claim_kernel(const int64_t* __restrict__ slots, const int64_t* __restrict__ positions,
                                  int64_t n_tok, int64_t slot_hi, int64_t cs_rows, ClaimTable tab) {
  const int64_t t = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (t >= n_tok || !token_writes(slots, positions, t, slot_hi, cs_rows)) return;
  const unsigned long long key = (unsigned long long)slots[t] + 1;
  uint32_t h = claim_hash(slots[t]) & tab.mask;
  // at most half the entries are ever taken: the probe ends
  for (uint32_t i = 0; i <= tab.mask; ++i, h = (h + 1) & tab.mask) {
    const unsigned long long old = atomicCAS(&tab.keys[h], 0ull, key);
    if (old == 0ull || old == key) {
      atomicMax(&tab.owner[h], (int)(t + 1));
      return;
    }
  }
}

__device__ __forceinline__ bool claimed_by(const ClaimTable& tab, int64_t slot, int64_t t) {
  const unsigned long long key = (unsigned long long)slot + 1;
  uint32_t h = claim_hash(slot) & tab.mask;
  for (uint32_t i = 0; i <= tab.mask; ++i, h = (h + 1) & tab.mask) {
    const unsigned long long k = tab.keys[h];
    if (k == key) return tab.owner[h] == (int)(t + 1);
    if (k == 0ull) return false;
  }
  return false;
}

// ---------------------------------------------------------------------------
// Row scale from the bits of max|x|: as unsigned integers the bit patterns of
// |x| order finite < infinity < NaN, so one integer maximum also finds the
// non-finite rows.
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

template <typename KV>
__device__ __forceinline__ float row_scale(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  return fmaxf(__fdiv_rn(__uint_as_float(amax_bits), kv8_max<KV>()), kScaleFloor);
}

// x / s correctly rounded by one correction step from r = 1 / s (P. Markstein,
// IBM J. Res. Dev. 1990): s is normal and at least 1e-12, and where the residual
// would underflow the quotient is far below the smallest code.
__device__ __forceinline__ float quotient(float x, float s, float r) {
  const float q0 = __fmul_rn(x, r);
  const float e = __fmaf_rn(-q0, s, x);
  return __fmaf_rn(e, r, q0);
}

// Codes of four values, one byte each (lowest address first).
template <typename KV>
__device__ __forceinline__ uint32_t codes4(const float* x, float s, float r) {
  if constexpr (std::is_same<KV, int8_t>::value) {
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // integer rounding (half to even) by adding 1.5 * 2^23: |x / s| < 128
      const int c = __float_as_int(__fadd_rn(quotient(x[j], s, r), 12582912.0f)) - 0x4B400000;
      w |= (uint32_t)(uint8_t)max(-127, min(127, c)) << (8 * j);
    }
    return w;
  } else {
    const __nv_fp8x2_storage_t lo =
        __nv_cvt_float2_to_fp8x2(make_float2(quotient(x[0], s, r), quotient(x[1], s, r)), __NV_SATFINITE, __NV_E4M3);
    const __nv_fp8x2_storage_t hi =
        __nv_cvt_float2_to_fp8x2(make_float2(quotient(x[2], s, r), quotient(x[3], s, r)), __NV_SATFINITE, __NV_E4M3);
    return (uint32_t)lo | ((uint32_t)hi << 16);
  }
}

struct AppendParams {
  int64_t n_tok, D, slot_hi, cs_rows, block_size;
  int nq, Hkv;  // query heads (0 without q), kv heads
  ClaimTable claim;  // keys == nullptr: scan
};

// Whether token t is the one written at its slot, for the whole CTA (every
// thread calls it with the same t).
__device__ __forceinline__ bool cta_owns_slot(const int64_t* __restrict__ slots, const int64_t* __restrict__ positions,
                                              int64_t t, int64_t slot, const AppendParams& p) {
  int lost = 0;
  if (p.claim.keys != nullptr) {
    if (threadIdx.x == 0) lost = !claimed_by(p.claim, slot, t);
  } else {
    for (int64_t j = t + 1 + threadIdx.x; j < p.n_tok; j += blockDim.x)
      if (__ldg(&slots[j]) == slot) lost |= token_writes(slots, positions, j, p.slot_hi, p.cs_rows);
  }
  return __syncthreads_or(lost) == 0;
}

// ---------------------------------------------------------------------------
// Fast kernel, D = 128.  One CTA a token; 16 lanes a row, a lane holding the
// four values 4l..4l+3 of each half (the rotation pairs).  A thread covers
// RPT rows g, g + groups, ... with all their loads issued first: RPT = 1 for
// decode sizes (a token's 48 rows in one pass of 768 threads: latency), more
// for prefill sizes (cos/sin and the slot are then fetched once for RPT rows).
// ---------------------------------------------------------------------------
__device__ __forceinline__ void load4(const float* p, float* f) {
  const float4 v = __ldg(reinterpret_cast<const float4*>(p));
  f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
}
template <typename T>
__device__ __forceinline__ void unpack8(const uint2& raw, float* f) {
  const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = to_f32(e[i]);
}
template <typename T>
__device__ __forceinline__ void load4(const T* p, float* f) {
  unpack8<T>(__ldg(reinterpret_cast<const uint2*>(p)), f);
}
template <typename T>
__device__ __forceinline__ uint2 pack8(const float* f) {
  uint2 raw;
  T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) e[i] = from_f32<T>(f[i]);
  return raw;
}

template <typename T, typename CS, typename KV, int RPT>
__global__ void __launch_bounds__(RPT == 1 ? 1024 : 256)
    kv_quant_append_kernel(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
                           const int64_t* __restrict__ positions, const CS* __restrict__ cos,
                           const CS* __restrict__ sin, const int64_t* __restrict__ slots, T* __restrict__ q_out,
                           uint8_t* __restrict__ k_cache, uint8_t* __restrict__ v_cache, float* __restrict__ k_scale,
                           float* __restrict__ v_scale, AppendParams p) {
  // a dependent launched with programmatic serialisation (the decode that
  // reads this cache) may start its prologue
  asm volatile("griddepcontrol.launch_dependents;");
  constexpr int kDim = 128, kHalf = 64;
  const int64_t t = blockIdx.x;
  const int c = (threadIdx.x & 15) * 4, g = threadIdx.x >> 4, groups = blockDim.x >> 4;
  const int rows = p.nq + 2 * p.Hkv;
  int64_t pos = __ldg(&positions[t]);
  const int64_t slot = __ldg(&slots[t]);
  const bool pos_ok = pos >= 0 && pos < p.cs_rows;
  if (!pos_ok) pos = 0;
  for (int r0 = g; r0 - g < rows; r0 += groups * RPT) {
    uint2 a[RPT], b[RPT];
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      const int row = r0 + groups * i;
      a[i] = b[i] = make_uint2(0, 0);
      if (row < rows) {
        const T* src = row < p.nq ? q + (t * p.nq + row) * kDim
                                  : (row < p.nq + p.Hkv ? k + (t * p.Hkv + (row - p.nq)) * kDim
                                                        : v + (t * p.Hkv + (row - p.nq - p.Hkv)) * kDim);
        a[i] = __ldg(reinterpret_cast<const uint2*>(src + c));
        b[i] = __ldg(reinterpret_cast<const uint2*>(src + kHalf + c));
      }
    }
    float cv[4], sv[4];
    load4(cos + pos * kDim + c, cv);
    load4(sin + pos * kDim + c, sv);
    const bool write_kv = pos_ok && slot >= 0 && slot < p.slot_hi;
    const bool owns = cta_owns_slot(slots, positions, t, slot, p);  // barrier: every thread gets here
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      const int row = r0 + groups * i;
      float x1[4], x2[4], y1[4], y2[4];
      unpack8<T>(a[i], x1);
      unpack8<T>(b[i], x2);
      if (row < p.nq + p.Hkv) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          y1[j] = __fsub_rn(__fmul_rn(x1[j], cv[j]), __fmul_rn(x2[j], sv[j]));
          y2[j] = __fadd_rn(__fmul_rn(x2[j], cv[j]), __fmul_rn(x1[j], sv[j]));
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) y1[j] = x1[j], y2[j] = x2[j];
      }
      // the row's maximum, over its 16 lanes (rows past the end hold zeros)
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) m = max(m, max(abs_bits(y1[j]), abs_bits(y2[j])));
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
      if (row >= rows) continue;
      if (row < p.nq) {
        if (!pos_ok) {
#pragma unroll
          for (int j = 0; j < 4; ++j) y1[j] = y2[j] = 0.f;
        }
        T* dst = q_out + (t * p.nq + row) * kDim;
        *reinterpret_cast<uint2*>(dst + c) = pack8<T>(y1);
        *reinterpret_cast<uint2*>(dst + kHalf + c) = pack8<T>(y2);
      } else if (write_kv && owns) {
        const bool is_k = row < p.nq + p.Hkv;
        const int h = is_k ? row - p.nq : row - p.nq - p.Hkv;
        const float s = row_scale<KV>(m), r = __frcp_rn(s);
        uint8_t* dst = (is_k ? k_cache : v_cache) + (slot * p.Hkv + h) * kDim;
        *reinterpret_cast<uint32_t*>(dst + c) = codes4<KV>(y1, s, r);
        *reinterpret_cast<uint32_t*>(dst + kHalf + c) = codes4<KV>(y2, s, r);
        if (c == 0) {
          const int64_t blk = slot / p.block_size, off = slot - blk * p.block_size;
          (is_k ? k_scale : v_scale)[(blk * p.Hkv + h) * p.block_size + off] = s;
        }
      }
    }
  }
}

// Any even D, any alignment: one warp a row, the row read twice.
template <typename T, typename CS, typename KV>
__global__ void __launch_bounds__(256)
    kv_quant_append_generic_kernel(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
                                   const int64_t* __restrict__ positions, const CS* __restrict__ cos,
                                   const CS* __restrict__ sin, const int64_t* __restrict__ slots,
                                   T* __restrict__ q_out, uint8_t* __restrict__ k_cache,
                                   uint8_t* __restrict__ v_cache, float* __restrict__ k_scale,
                                   float* __restrict__ v_scale, AppendParams p) {
  const int64_t t = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int rows = p.nq + 2 * p.Hkv;
  const int64_t half = p.D / 2;
  int64_t pos = positions[t];
  const int64_t slot = slots[t];
  const bool pos_ok = pos >= 0 && pos < p.cs_rows;
  if (!pos_ok) pos = 0;
  const bool write_kv = pos_ok && slot >= 0 && slot < p.slot_hi;
  const bool owns = cta_owns_slot(slots, positions, t, slot, p);
  for (int row = warp; row < rows; row += warps) {
    const bool is_q = row < p.nq, is_k = !is_q && row < p.nq + p.Hkv;
    if (!is_q && !(write_kv && owns)) continue;
    const int h = is_q ? row : (is_k ? row - p.nq : row - p.nq - p.Hkv);
    const T* src = is_q ? q + (t * p.nq + h) * p.D : (is_k ? k : v) + (t * p.Hkv + h) * p.D;
    auto pair = [&](int64_t i, float& y1, float& y2) {
      const float x1 = to_f32(src[i]), x2 = to_f32(src[half + i]);
      y1 = x1, y2 = x2;
      if (is_q || is_k) {
        const float cv = to_f32(cos[pos * p.D + i]), sv = to_f32(sin[pos * p.D + i]);
        y1 = __fsub_rn(__fmul_rn(x1, cv), __fmul_rn(x2, sv));
        y2 = __fadd_rn(__fmul_rn(x2, cv), __fmul_rn(x1, sv));
      }
    };
    if (is_q) {
      T* dst = q_out + (t * p.nq + h) * p.D;
      for (int64_t i = lane; i < half; i += 32) {
        float y1 = 0.f, y2 = 0.f;
        if (pos_ok) pair(i, y1, y2);
        dst[i] = from_f32<T>(y1);
        dst[half + i] = from_f32<T>(y2);
      }
      continue;
    }
    uint32_t m = 0;
    for (int64_t i = lane; i < half; i += 32) {
      float y1, y2;
      pair(i, y1, y2);
      m = max(m, max(abs_bits(y1), abs_bits(y2)));
    }
    m = __reduce_max_sync(0xffffffffu, m);
    const float s = row_scale<KV>(m), r = __frcp_rn(s);
    uint8_t* dst = (is_k ? k_cache : v_cache) + (slot * p.Hkv + h) * p.D;
    for (int64_t i = lane; i < half; i += 32) {
      float y[4] = {0.f, 0.f, 0.f, 0.f};
      pair(i, y[0], y[1]);
      const uint32_t w = codes4<KV>(y, s, r);
      dst[i] = (uint8_t)w;
      dst[half + i] = (uint8_t)(w >> 8);
    }
    if (lane == 0) {
      const int64_t blk = slot / p.block_size, off = slot - blk * p.block_size;
      (is_k ? k_scale : v_scale)[(blk * p.Hkv + h) * p.block_size + off] = s;
    }
  }
}

template <typename T, typename CS, typename KV>
int launch_append(const void* q, const void* k, const void* v, const int64_t* positions, const void* cos,
                  const void* sin, const int64_t* slots, void* q_out, void* k_cache, void* v_cache, float* k_scale,
                  float* v_scale, const AppendParams& p, const b200_launch_cfg* cfg, cudaStream_t s) {
  auto* qp = static_cast<const T*>(q);
  auto* kp = static_cast<const T*>(k);
  auto* vp = static_cast<const T*>(v);
  auto* cp = static_cast<const CS*>(cos);
  auto* sp = static_cast<const CS*>(sin);
  auto* qo = static_cast<T*>(q_out);
  auto* kc = static_cast<uint8_t*>(k_cache);
  auto* vc = static_cast<uint8_t*>(v_cache);
  const void* ptrs[] = {q, k, v, cos, sin, q_out, k_cache, v_cache};
  bool fast = p.D == 128;
  for (const void* x : ptrs)
    if (!aligned16(x)) fast = false;  // (a null q passes)
  const unsigned grid = (unsigned)p.n_tok;
  if (!fast) {
    kv_quant_append_generic_kernel<T, CS, KV><<<grid, 256, 0, s>>>(qp, kp, vp, positions, cp, sp, slots, qo, kc, vc,
                                                                  k_scale, v_scale, p);
    return launch_status(cudaGetLastError());
  }
  const int rows = p.nq + 2 * p.Hkv;
  const int rpt = (cfg && cfg->rows_per_cta > 0) ? cfg->rows_per_cta : (p.n_tok <= kScanTokens ? 1 : 3);
  // threads: the token's rows in one pass where they fit
  auto threads = [&](int per, int most) {
    const int n = ((rows + per - 1) / per * 16 + 31) / 32 * 32;
    return n < most ? n : most;
  };
  if (rpt == 1)
    kv_quant_append_kernel<T, CS, KV, 1><<<grid, threads(1, 1024), 0, s>>>(qp, kp, vp, positions, cp, sp, slots, qo,
                                                                          kc, vc, k_scale, v_scale, p);
  else if (rpt == 2)
    kv_quant_append_kernel<T, CS, KV, 2><<<grid, threads(2, 256), 0, s>>>(qp, kp, vp, positions, cp, sp, slots, qo,
                                                                         kc, vc, k_scale, v_scale, p);
  else if (rpt == 3)
    kv_quant_append_kernel<T, CS, KV, 3><<<grid, threads(3, 256), 0, s>>>(qp, kp, vp, positions, cp, sp, slots, qo,
                                                                         kc, vc, k_scale, v_scale, p);
  else
    kv_quant_append_kernel<T, CS, KV, 6><<<grid, threads(6, 256), 0, s>>>(qp, kp, vp, positions, cp, sp, slots, qo,
                                                                         kc, vc, k_scale, v_scale, p);
  return launch_status(cudaGetLastError());
}

// ---------------------------------------------------------------------------
// Read back.  Output rows [b, h, s, :] for s < max_len: token s of sequence b
// is token s % bs of its (s / bs)-th valid block (ids outside [0, num_blocks)
// are dropped and later blocks move up, as in the attention kernels); rows at
// or past the context are zero.  HBM-bound: 1 byte read and 2 written a
// value.  A CTA covers kPages output pages of one sequence; a thread keeps
// four 16-code loads of K and four of V in flight.
// ---------------------------------------------------------------------------
constexpr int kPages = 4;

struct DequantParams {
  int64_t B, Hkv, D, num_blocks, block_size, max_blocks, max_len;
};

template <typename IDX>
__device__ __forceinline__ bool in_pool(IDX id, int64_t nb) {
  return id >= 0 && (int64_t)id < nb;
}

// ids[i] = block of rank first + i among the valid ones of bt[0, n), -1 past the last.
template <typename IDX>
__device__ __forceinline__ void warp_find_blocks(const IDX* __restrict__ bt, int64_t n, int64_t nb, int64_t first,
                                                 int64_t* ids, int lane) {
  for (int i = lane; i < kPages; i += 32) ids[i] = -1;
  __syncwarp();
  int64_t rank0 = 0;
  for (int64_t j0 = 0; j0 < n && rank0 < first + kPages; j0 += 128) {
    IDX v[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = j0 + r * 32 + lane < n ? __ldg(&bt[j0 + r * 32 + lane]) : (IDX)-1;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const bool ok = in_pool(v[r], nb);
      const unsigned ballot = __ballot_sync(0xffffffffu, ok);
      const int64_t rank = rank0 + __popc(ballot & ((1u << lane) - 1u));
      if (ok && rank >= first && rank < first + kPages) ids[rank - first] = (int64_t)v[r];
      rank0 += __popc(ballot);
    }
  }
  __syncwarp();
}

template <typename T, typename KV, typename IDX, bool VEC>
__global__ void __launch_bounds__(256)
    kv_dequant_kernel(const uint8_t* __restrict__ k_cache, const uint8_t* __restrict__ v_cache,
                      const float* __restrict__ k_scale, const float* __restrict__ v_scale,
                      const IDX* __restrict__ block_table, const IDX* __restrict__ context_len,
                      T* __restrict__ k_out, T* __restrict__ v_out, DequantParams p, int64_t chunks) {
  __shared__ int64_t s_id[kPages];
  const int64_t b = blockIdx.x / chunks, first = (blockIdx.x - b * chunks) * kPages;
  const int64_t bs = p.block_size;
  int64_t ctx = (int64_t)context_len[b];
  ctx = ctx < 0 ? 0 : (ctx < p.max_len ? ctx : p.max_len);
  if (threadIdx.x < 32) {
    const int64_t full = (int64_t)context_len[b];
    const int64_t nvb = full > 0 ? min((full + bs - 1) / bs, p.max_blocks) : 0;
    warp_find_blocks(block_table + b * p.max_blocks, nvb, p.num_blocks, first, s_id, threadIdx.x);
  }
  __syncthreads();
  constexpr int W = VEC ? 16 : 1;  // codes a thread takes at a time
  const int cpr = (int)(p.D / W);
  const int per_page = (int)bs * (int)p.Hkv * cpr;
  for (int i = 0; i < kPages; ++i) {
    const int64_t row0 = (first + i) * bs;
    if (row0 >= p.max_len) break;
    const int64_t id = s_id[i];
    const int rows = (int)min(bs, p.max_len - row0);
    const int live = id < 0 ? 0 : (int)max((int64_t)0, min((int64_t)rows, ctx - row0));
    for (int x0 = threadIdx.x; x0 < per_page; x0 += blockDim.x * 4) {
      uint4 raw[2][4];
      float sc[2][4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int x = x0 + u * (int)blockDim.x;
        const int th = x / cpr, t = th / (int)p.Hkv, h = th - t * (int)p.Hkv;
        raw[0][u] = raw[1][u] = make_uint4(0, 0, 0, 0);
        sc[0][u] = sc[1][u] = 0.f;
        if (x < per_page && t < live) {
          const int64_t at = id * bs * p.Hkv * p.D + (int64_t)x * W;
          if constexpr (VEC) {
            raw[0][u] = ldg_stream16(k_cache + at);
            raw[1][u] = ldg_stream16(v_cache + at);
          } else {
            raw[0][u].x = k_cache[at];
            raw[1][u].x = v_cache[at];
          }
          const int64_t sat = (id * p.Hkv + h) * bs + t;
          sc[0][u] = __ldg(&k_scale[sat]);
          sc[1][u] = __ldg(&v_scale[sat]);
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int x = x0 + u * (int)blockDim.x;
        const int th = x / cpr, t = th / (int)p.Hkv, h = th - t * (int)p.Hkv;
        if (x >= per_page || t >= rows) continue;
        const int64_t at = ((b * p.Hkv + h) * p.max_len + row0 + t) * p.D + (int64_t)(x - th * cpr) * W;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          T* out = (w ? v_out : k_out) + at;
          if constexpr (VEC) {
            const uint32_t src[4] = {raw[w][u].x, raw[w][u].y, raw[w][u].z, raw[w][u].w};
            float f[16];
#pragma unroll
            for (int j = 0; j < 4; ++j) kv8_to_f32x4<KV>(src[j], f + 4 * j);
#pragma unroll
            for (int j = 0; j < 16; ++j) f[j] = __fmul_rn(f[j], sc[w][u]);
            *reinterpret_cast<uint4*>(out) = pack16<T>(f);
            *reinterpret_cast<uint4*>(out + 8) = pack16<T>(f + 8);
          } else {
            float f[4];
            kv8_to_f32x4<KV>(raw[w][u].x, f);
            out[0] = from_f32<T>(__fmul_rn(f[0], sc[w][u]));
          }
        }
      }
    }
  }
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" size_t b200_rope_kv_append_paged_quant_workspace_size(int64_t T) {
  if (T <= 0 || T > 0x3fffffffLL) return 0;
  return (size_t)claim_entries(T) * 12;
}

extern "C" int b200_rope_kv_append_paged_quant(const void* q, const void* k, const void* v, const int64_t* positions,
                                               const void* cos, const void* sin, int64_t cs_rows,
                                               const int64_t* slot_mapping, void* q_out, void* k_cache, void* v_cache,
                                               float* k_scale, float* v_scale, int64_t T, int64_t Hq, int64_t Hkv,
                                               int64_t D, int64_t num_blocks, int64_t block_size, int32_t dtype,
                                               int32_t cs_dtype, int32_t cache_dtype, void* workspace,
                                               size_t workspace_bytes, const b200_launch_cfg* cfg, void* stream) {
  if (int e = injected_error("rope_kv_append_paged_quant")) return e;
  if (T < 0 || Hkv <= 0 || D <= 0 || D % 2 != 0 || num_blocks <= 0 || block_size <= 0 || cs_rows <= 0)
    return B200_ERR_BAD_ARG;
  if ((q == nullptr) != (q_out == nullptr) && T > 0) return B200_ERR_BAD_ARG;
  if (q && Hq <= 0) return B200_ERR_BAD_ARG;
  if (T == 0) return B200_OK;
  if (!k || !v || !positions || !cos || !sin || !slot_mapping || !k_cache || !v_cache || !k_scale || !v_scale)
    return B200_ERR_BAD_ARG;
  if (T > 0x3fffffffLL || Hq > 4096 || Hkv > 4096 || block_size > 65536) return B200_ERR_UNSUPPORTED;
  if (cache_dtype != B200_I8 && cache_dtype != B200_F8E4M3) return B200_ERR_UNSUPPORTED;
  if (cs_dtype != dtype && cs_dtype != B200_F32) return B200_ERR_UNSUPPORTED;
  const size_t need = b200_rope_kv_append_paged_quant_workspace_size(T);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return B200_ERR_WORKSPACE;
  if (need > 0 && !aligned16(workspace)) return B200_ERR_ALIGNMENT;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  AppendParams p{T, D, num_blocks * block_size, cs_rows, block_size, q ? (int)Hq : 0, (int)Hkv, {nullptr, nullptr, 0}};
  return B200_DISPATCH_HALF(dtype, [&]() -> int {
    if (need > 0) {
      const int64_t n = claim_entries(T);
      p.claim.keys = static_cast<unsigned long long*>(workspace);
      p.claim.owner = reinterpret_cast<int*>(p.claim.keys + n);
      p.claim.mask = (uint32_t)(n - 1);
      cudaError_t e = cudaMemsetAsync(workspace, 0, need, s);
      if (e != cudaSuccess) return launch_status(e);
      slot_claim_kernel<<<(unsigned)((T + 255) / 256), 256, 0, s>>>(slot_mapping, positions, T, p.slot_hi, cs_rows,
                                                                  p.claim);
      e = cudaGetLastError();
      if (e != cudaSuccess) return launch_status(e);
    }
    auto run = [&](auto kv_tag) -> int {
      using KV = decltype(kv_tag);
      if (cs_dtype == B200_F32)
        return launch_append<scalar_t, float, KV>(q, k, v, positions, cos, sin, slot_mapping, q_out, k_cache, v_cache,
                                                  k_scale, v_scale, p, cfg, s);
      return launch_append<scalar_t, scalar_t, KV>(q, k, v, positions, cos, sin, slot_mapping, q_out, k_cache,
                                                   v_cache, k_scale, v_scale, p, cfg, s);
    };
    return cache_dtype == B200_I8 ? run(int8_t{}) : run(e4m3_t{});
  });
}

extern "C" int b200_paged_kv_dequant(const void* k_cache, const void* v_cache, const float* k_scale,
                                     const float* v_scale, const void* block_table, const void* context_len,
                                     void* k_out, void* v_out, int64_t B, int64_t Hkv, int64_t D, int64_t num_blocks,
                                     int64_t block_size, int64_t max_blocks, int64_t max_len, int32_t dtype,
                                     int32_t cache_dtype, int32_t index_dtype, const b200_launch_cfg* cfg,
                                     void* stream) {
  (void)cfg;
  if (int e = injected_error("paged_kv_dequant")) return e;
  if (B < 0 || Hkv <= 0 || D <= 0 || num_blocks <= 0 || block_size <= 0 || max_blocks <= 0 || max_len < 0)
    return B200_ERR_BAD_ARG;
  if (B == 0 || max_len == 0) return B200_OK;
  if (!k_cache || !v_cache || !k_scale || !v_scale || !block_table || !context_len || !k_out || !v_out)
    return B200_ERR_BAD_ARG;
  if (index_dtype != B200_I32 && index_dtype != B200_I64) return B200_ERR_UNSUPPORTED;
  if (cache_dtype != B200_I8 && cache_dtype != B200_F8E4M3) return B200_ERR_UNSUPPORTED;
  const int64_t chunks = ((max_len + block_size - 1) / block_size + kPages - 1) / kPages;
  if (chunks * B > 0x7fffffffLL || block_size * Hkv * D > (1 << 28)) return B200_ERR_UNSUPPORTED;
  const bool vec = D % 16 == 0 && aligned16(k_cache) && aligned16(v_cache) && aligned16(k_out) && aligned16(v_out);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  DequantParams p{B, Hkv, D, num_blocks, block_size, max_blocks, max_len};
  return B200_DISPATCH_HALF(dtype, [&]() -> int {
    auto run = [&](auto kv_tag, auto idx_tag) -> int {
      using KV = decltype(kv_tag);
      using IDX = decltype(idx_tag);
      auto kern = vec ? kv_dequant_kernel<scalar_t, KV, IDX, true> : kv_dequant_kernel<scalar_t, KV, IDX, false>;
      kern<<<(unsigned)(chunks * B), 256, 0, s>>>(
          static_cast<const uint8_t*>(k_cache), static_cast<const uint8_t*>(v_cache), k_scale, v_scale,
          static_cast<const IDX*>(block_table), static_cast<const IDX*>(context_len), static_cast<scalar_t*>(k_out),
          static_cast<scalar_t*>(v_out), p, chunks);
      return launch_status(cudaGetLastError());
    };
    auto by_index = [&](auto kv_tag) -> int {
      return index_dtype == B200_I32 ? run(kv_tag, int32_t{}) : run(kv_tag, int64_t{});
    };
    return cache_dtype == B200_I8 ? by_index(int8_t{}) : by_index(e4m3_t{});
  });
}
