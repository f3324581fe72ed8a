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
// the 16-bit append.  For many tokens, three launches: the claim kernel finds the
// slots that several tokens write and the last token of each, in an
// open-addressing table (twice as many entries as tokens or more, cleared by
// each call, so calls share no state; O(T) against O(T^2) for the scan); the
// append runs beside it and writes every token; the repair kernel, after both,
// writes the last tokens of the shared slots once more -- usually none.  (The
// append waiting for the claims instead cost their 13 us each time.)
// ---------------------------------------------------------------------------
struct ClaimTable {
  unsigned long long* keys;  // slot + 1; 0 = empty
  int* owner;                // 1 + last token
  int* shared;               // [0] number of shared slots, [1..] their last tokens
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

// One cluster of eight CTAs clears the table, fills it and reads it back, with
// cluster barriers between: one launch on eight SMs beside the append.
constexpr int kClaimCtas = 8, kClaimThreads = 1024, kClaimStep = kClaimCtas * kClaimThreads;
__global__ void __cluster_dims__(kClaimCtas, 1, 1) __launch_bounds__(kClaimThreads)
    slot_claim_kernel(const int64_t* __restrict__ slots, const int64_t* __restrict__ positions, int64_t n_tok,
                      int64_t slot_hi, int64_t cs_rows, ClaimTable tab) {
  asm volatile("griddepcontrol.launch_dependents;");
  constexpr unsigned long long kMark = 1ull << 63;  // on a key: a second token named the slot
  const int me = blockIdx.x * kClaimThreads + threadIdx.x;
  for (int64_t i = me; i <= (int64_t)tab.mask; i += kClaimStep) {
    __stcg(&tab.keys[i], 0ull);
    __stcg(&tab.owner[i], 0);
  }
  if (me == 0) __stcg(&tab.shared[0], 0);
  __threadfence();
  sm100::cluster_sync();
  // at most half the entries are ever taken: the probes end.  Four tokens a
  // thread in flight: their first probes go out together.
  for (int64_t t0 = me; t0 < n_tok; t0 += 4 * kClaimStep) {
    unsigned long long key[4], old[4];
    uint32_t h[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t t = t0 + u * kClaimStep;
      key[u] = t < n_tok && token_writes(slots, positions, t, slot_hi, cs_rows) ? (unsigned long long)slots[t] + 1 : 0ull;
      h[u] = key[u] ? claim_hash((int64_t)key[u] - 1) & tab.mask : 0u;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) old[u] = key[u] ? atomicCAS(&tab.keys[h[u]], 0ull, key[u]) : 0ull;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (!key[u]) continue;
      for (uint32_t i = 0; i <= tab.mask && old[u] != 0ull && (old[u] & ~kMark) != key[u]; ++i) {
        h[u] = (h[u] + 1) & tab.mask;
        old[u] = atomicCAS(&tab.keys[h[u]], 0ull, key[u]);
      }
      const int t = (int)(t0 + u * kClaimStep);
      if (atomicMax(&tab.owner[h[u]], t + 1) != 0) atomicOr(&tab.keys[h[u]], kMark);
    }
  }
  __threadfence();
  sm100::cluster_sync();
  // the last token of each marked slot
  for (int64_t i0 = me; i0 <= (int64_t)tab.mask; i0 += 4 * kClaimStep) {
    unsigned long long k[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      k[u] = i0 + u * kClaimStep <= (int64_t)tab.mask ? __ldcg(&tab.keys[i0 + u * kClaimStep]) : 0ull;
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (k[u] & kMark) tab.shared[1 + atomicAdd(&tab.shared[0], 1)] = __ldcg(&tab.owner[i0 + u * kClaimStep]) - 1;
  }
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

// Pairs of x / s, correctly rounded by one correction step from r = 1 / s (P.
// Markstein, IBM J. Res. Dev. 1990), two at a time: s is normal and at least
// 1e-12, and where the residual would underflow the quotient is far below the
// smallest code.
__device__ __forceinline__ void quotient2(float& a, float& b, float x0, float x1, float s, float r) {
  float q0, q1, e0, e1;
  sm100::fmul2_bcast(q0, q1, x0, x1, r);
  sm100::ffma2(e0, e1, q0, q1, -s, -s, x0, x1);
  sm100::ffma2(a, b, e0, e1, r, r, q0, q1);
}

// Codes of four values, one byte each (lowest address first).  int8: the
// quotient plus 1.5 * 2^23 is the integer rounded half to even in the low bits;
// |x| <= qmax s (1 + 2^-23), so the code needs no clamp (a NaN scale leaves any byte).
template <typename KV>
__device__ __forceinline__ uint32_t codes4(const float* x, float s, float r) {
  float q[4];
  quotient2(q[0], q[1], x[0], x[1], s, r);
  quotient2(q[2], q[3], x[2], x[3], s, r);
  if constexpr (std::is_same<KV, int8_t>::value) {
    uint32_t b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) b[j] = __float_as_uint(__fadd_rn(q[j], 12582912.0f));
    return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
  } else {
    const __nv_fp8x2_storage_t lo = __nv_cvt_float2_to_fp8x2(make_float2(q[0], q[1]), __NV_SATFINITE, __NV_E4M3);
    const __nv_fp8x2_storage_t hi = __nv_cvt_float2_to_fp8x2(make_float2(q[2], q[3]), __NV_SATFINITE, __NV_E4M3);
    return (uint32_t)lo | ((uint32_t)hi << 16);
  }
}

// max(|a|, |b|, |c|) with a NaN winning: of the bit patterns of magnitudes NaN is
// then the largest, infinity the next.
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Rotation of eight pairs; every product and sum rounded on its own (packed
// products feeding scalar sums, which nothing contracts).
__device__ __forceinline__ void rotate8(float (&x1)[8], float (&x2)[8], const float (&c)[8], const float (&s)[8]) {
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    float ac0, ac1, bs0, bs1, bc0, bc1, as0, as1;
    sm100::fmul2(ac0, ac1, x1[j], x1[j + 1], c[j], c[j + 1]);
    sm100::fmul2(bs0, bs1, x2[j], x2[j + 1], s[j], s[j + 1]);
    sm100::fmul2(bc0, bc1, x2[j], x2[j + 1], c[j], c[j + 1]);
    sm100::fmul2(as0, as1, x1[j], x1[j + 1], s[j], s[j + 1]);
    x1[j] = __fsub_rn(ac0, bs0), x1[j + 1] = __fsub_rn(ac1, bs1);
    x2[j] = __fadd_rn(bc0, as0), x2[j + 1] = __fadd_rn(bc1, as1);
  }
}

struct AppendParams {
  int64_t n_tok, D, slot_hi, cs_rows, block_size;
  int nq, Hkv;  // query heads (0 without q), kv heads
  int lg_bs;    // log2 of the block size, -1 if it is no power of two
  ClaimTable claim;  // keys == nullptr: scan
};

// Token t's slot if t writes it, else -1, for the whole CTA (every thread
// calls it with the same t): small appends scan the later slots; with the
// table every token writes, and the repair kernel comes after.
__device__ __forceinline__ int64_t cta_target(const int64_t* __restrict__ slots, const int64_t* __restrict__ positions,
                                              int64_t t, int64_t slot, bool writes, const AppendParams& p) {
  if (p.claim.keys != nullptr) return writes ? slot : -1;
  int lost = 0;
  for (int64_t j = t + 1 + threadIdx.x; j < p.n_tok; j += blockDim.x)
    if (__ldg(&slots[j]) == slot) lost |= token_writes(slots, positions, j, p.slot_hi, p.cs_rows);
  return __syncthreads_or(lost) == 0 && writes ? slot : -1;
}

// ---------------------------------------------------------------------------
// Fast kernels, D = 128.  Eight lanes a row, a lane holding the eight values
// 8l.. of each half (the rotation pairs) as one 16-byte load each.  A rotated
// row is about 90 instructions a lane and its codes 70 more, which weighs
// beside the bytes: roundings, maxima and quotients are packed or three-input forms.
// ---------------------------------------------------------------------------
__device__ __forceinline__ void load8(const float* p, float* f) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
}
template <typename T>
__device__ __forceinline__ void load8(const T* p, float* f) {
  unpack16<T>(__ldg(reinterpret_cast<const uint4*>(p)), f);
}

// Where the tensors of a call are.
template <typename T, typename CS>
struct AppendPtrs {
  const T *q, *k, *v;
  const CS *cos, *sin;
  const int64_t *positions, *slots;
  T* q_out;
  uint8_t *k_cache, *v_cache;
  float *k_scale, *v_scale;
};

template <typename T, typename CS>
__device__ __forceinline__ const T* row_source(const AppendPtrs<T, CS>& x, const AppendParams& p, int64_t t, int row) {
  return row < p.nq ? x.q + (t * p.nq + row) * 128
                    : (row < p.nq + p.Hkv ? x.k + (t * p.Hkv + (row - p.nq)) * 128
                                          : x.v + (t * p.Hkv + (row - p.nq - p.Hkv)) * 128);
}

// Block and offset of a slot.
__device__ __forceinline__ void split_slot(int64_t slot, int64_t bs, int lg_bs, int64_t& blk, int64_t& off) {
  blk = lg_bs >= 0 ? slot >> lg_bs : slot / bs;
  off = slot - blk * bs;
}

// One row (its eight values a lane of each half in a, b): rotated and written,
// or quantised and written.
template <typename T, typename CS, typename KV>
__device__ __forceinline__ void append_row(const AppendPtrs<T, CS>& x, const AppendParams& p, int64_t t, int row, int c,
                                           const uint4& a, const uint4& b, const float (&cv)[8], const float (&sv)[8],
                                           bool pos_ok, int64_t slot, int64_t blk, int64_t off) {
  float y1[8], y2[8];
  unpack16<T>(a, y1);
  unpack16<T>(b, y2);
  if (row < p.nq + p.Hkv) rotate8(y1, y2, cv, sv);
  if (row < p.nq) {
    if (!pos_ok) {
#pragma unroll
      for (int j = 0; j < 8; ++j) y1[j] = y2[j] = 0.f;
    }
    T* dst = x.q_out + (t * p.nq + row) * 128;
    *reinterpret_cast<uint4*>(dst + c) = pack16<T>(y1);
    *reinterpret_cast<uint4*>(dst + 64 + c) = pack16<T>(y2);
  } else if (slot >= 0) {
    // the row's maximum, over its eight lanes (which take this branch together)
    float mf = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) mf = max3_abs(mf, y1[j], y2[j]);
    uint32_t m = __float_as_uint(mf);
    const unsigned lanes = 0xffu << (threadIdx.x & 24);
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(lanes, m, o));
    const bool is_k = row < p.nq + p.Hkv;
    const int h = is_k ? row - p.nq : row - p.nq - p.Hkv;
    const float s = row_scale<KV>(m), r = __frcp_rn(s);
    uint8_t* dst = (is_k ? x.k_cache : x.v_cache) + (slot * p.Hkv + h) * 128;
    *reinterpret_cast<uint2*>(dst + c) = make_uint2(codes4<KV>(y1, s, r), codes4<KV>(y1 + 4, s, r));
    *reinterpret_cast<uint2*>(dst + 64 + c) = make_uint2(codes4<KV>(y2, s, r), codes4<KV>(y2 + 4, s, r));
    if (c == 0) (is_k ? x.k_scale : x.v_scale)[(blk * p.Hkv + h) * p.block_size + off] = s;
  }
}

// Decode sizes: one CTA a token, its rows in passes of blockDim / 8.
template <typename T, typename CS, typename KV>
__global__ void __launch_bounds__(1024) kv_quant_append_kernel(AppendPtrs<T, CS> x, AppendParams p) {
  // a dependent launched with programmatic serialisation (the decode that
  // reads this cache) may start its prologue
  asm volatile("griddepcontrol.launch_dependents;");
  const int64_t t = blockIdx.x;
  const int c = (threadIdx.x & 7) * 8, groups = blockDim.x >> 3;
  const int rows = p.nq + 2 * p.Hkv;
  int64_t pos = __ldg(&x.positions[t]);
  const int64_t named = __ldg(&x.slots[t]);
  const bool pos_ok = pos >= 0 && pos < p.cs_rows;
  if (!pos_ok) pos = 0;
  int row = threadIdx.x >> 3;
  uint4 a = make_uint4(0, 0, 0, 0), b = a;
  if (row < rows) {
    const T* src = row_source(x, p, t, row);
    a = ldg_stream16(src + c);
    b = ldg_stream16(src + 64 + c);
  }
  float cv[8], sv[8];
  load8(x.cos + pos * 128 + c, cv);
  load8(x.sin + pos * 128 + c, sv);
  const bool writes = pos_ok && named >= 0 && named < p.slot_hi;
  const int64_t slot = cta_target(x.slots, x.positions, t, named, writes, p);
  int64_t blk, off;
  split_slot(slot, p.block_size, p.lg_bs, blk, off);
  while (row < rows) {
    append_row<T, CS, KV>(x, p, t, row, c, a, b, cv, sv, pos_ok, slot, blk, off);
    row += groups;
    if (row < rows) {
      const T* src = row_source(x, p, t, row);
      a = ldg_stream16(src + c);
      b = ldg_stream16(src + 64 + c);
    }
  }
}

// Prefill sizes: a token's rows take `groups` groups of eight lanes, RPT rows a
// lane (g, g + groups, ...), all their loads issued first; as many tokens a
// CTA as fit 256 threads, each on its own (no barrier).  Launched beside the claim
// kernel; every token is written.  16384 tokens of 32 + 8 + 8 rows: 68 us,
// 5.5 TB/s of the 370 MB it must move.
template <typename T, typename CS, typename KV, int RPT>
__global__ void __launch_bounds__(256) kv_quant_append_stream_kernel(AppendPtrs<T, CS> x, AppendParams p, int groups) {
  asm volatile("griddepcontrol.launch_dependents;");
  const int tpt = groups * 8, lt = threadIdx.x / tpt;  // threads a token, token of the CTA
  const int c = (threadIdx.x & 7) * 8, g = (threadIdx.x - lt * tpt) >> 3;
  const int rows = p.nq + 2 * p.Hkv;
  const int64_t t = (int64_t)blockIdx.x * (blockDim.x / tpt) + lt;
  if (t < p.n_tok) {
    int64_t pos = __ldg(&x.positions[t]), slot = __ldg(&x.slots[t]);
    uint4 a[RPT], b[RPT];
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      const int row = g + groups * i;
      a[i] = b[i] = make_uint4(0, 0, 0, 0);
      if (row < rows) {
        const T* src = row_source(x, p, t, row);
        a[i] = ldg_stream16(src + c);
        b[i] = ldg_stream16(src + 64 + c);
      }
    }
    const bool pos_ok = pos >= 0 && pos < p.cs_rows;
    if (!pos_ok) pos = 0;
    if (!pos_ok || slot >= p.slot_hi) slot = -1;
    float cv[8], sv[8];
    load8(x.cos + pos * 128 + c, cv);
    load8(x.sin + pos * 128 + c, sv);
    int64_t blk, off;
    split_slot(slot, p.block_size, p.lg_bs, blk, off);
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      const int row = g + groups * i;
      if (row < rows) append_row<T, CS, KV>(x, p, t, row, c, a[i], b[i], cv, sv, pos_ok, slot, blk, off);
    }
  }
  // the grid counts as done only when the claims are (one CTA waits: all of
  // them would hold the SMs that the later ones need)
  if (blockIdx.x == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
}

// The last tokens of shared slots, written once more after all others: a warp
// a token, four K and V rows at a time.
template <typename T, typename CS, typename KV>
__global__ void __launch_bounds__(256) kv_quant_repair_kernel(AppendPtrs<T, CS> x, AppendParams p) {
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int n = __ldcg(&p.claim.shared[0]);
  const int c = (threadIdx.x & 7) * 8, rows = p.nq + 2 * p.Hkv;
  for (int i = blockIdx.x * 8 + (threadIdx.x >> 5); i < n; i += gridDim.x * 8) {
    const int64_t t = __ldcg(&p.claim.shared[1 + i]);
    const int64_t pos = x.positions[t], slot = x.slots[t];
    float cv[8], sv[8];
    load8(x.cos + pos * 128 + c, cv);
    load8(x.sin + pos * 128 + c, sv);
    int64_t blk, off;
    split_slot(slot, p.block_size, p.lg_bs, blk, off);
    for (int row = p.nq + ((threadIdx.x & 31) >> 3); row < rows; row += 4) {
      const T* src = row_source(x, p, t, row);
      append_row<T, CS, KV>(x, p, t, row, c, ldg_stream16(src + c), ldg_stream16(src + 64 + c), cv, sv, true, slot,
                            blk, off);
    }
  }
}

// Any even D, any alignment: one warp a row, the row read twice.  With `repair`
// a CTA writes the K and V rows of the shared slots' last tokens.
template <typename T, typename CS, typename KV>
__global__ void __launch_bounds__(256)
    kv_quant_append_generic_kernel(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
                                   const int64_t* __restrict__ positions, const CS* __restrict__ cos,
                                   const CS* __restrict__ sin, const int64_t* __restrict__ slots,
                                   T* __restrict__ q_out, uint8_t* __restrict__ k_cache,
                                   uint8_t* __restrict__ v_cache, float* __restrict__ k_scale,
                                   float* __restrict__ v_scale, AppendParams p, bool repair) {
  if (repair && (int)blockIdx.x >= __ldcg(&p.claim.shared[0])) return;
  const int64_t t = repair ? __ldcg(&p.claim.shared[1 + blockIdx.x]) : blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int rows = p.nq + 2 * p.Hkv;
  const int64_t half = p.D / 2;
  int64_t pos = positions[t];
  const int64_t slot = slots[t];
  const bool pos_ok = pos >= 0 && pos < p.cs_rows;
  if (!pos_ok) pos = 0;
  const bool write_kv = pos_ok && slot >= 0 && slot < p.slot_hi;
  const int64_t target = cta_target(slots, positions, t, slot, write_kv, p);
  for (int row = warp; row < rows; row += warps) {
    const bool is_q = row < p.nq, is_k = !is_q && row < p.nq + p.Hkv;
    if (is_q ? repair : target < 0) continue;
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
    for (int repair = 0; repair <= (p.claim.keys != nullptr ? 1 : 0); ++repair) {
      kv_quant_append_generic_kernel<T, CS, KV><<<grid, 256, 0, s>>>(qp, kp, vp, positions, cp, sp, slots, qo, kc, vc,
                                                                    k_scale, v_scale, p, repair != 0);
      if (cudaError_t e = cudaGetLastError(); e != cudaSuccess) return launch_status(e);
    }
    return B200_OK;
  }
  const int rows = p.nq + 2 * p.Hkv;
  const AppendPtrs<T, CS> x{qp, kp, vp, cp, sp, positions, slots, qo, kc, vc, k_scale, v_scale};
  if (p.claim.keys == nullptr) {
    int threads = (rows * 8 + 31) / 32 * 32;  // the token's rows in one pass where they fit
    if (threads > 1024) threads = 1024;
    kv_quant_append_kernel<T, CS, KV><<<grid, threads, 0, s>>>(x, p);
    return launch_status(cudaGetLastError());
  }
  // rows a lane: as few as let a token fit the CTA, at least two
  int rpt = (cfg && cfg->rows_per_cta > 0) ? cfg->rows_per_cta : 2;
  while (rpt < 8 && (rows + rpt - 1) / rpt > 32) ++rpt;
  rpt = rpt <= 4 ? rpt : (rpt <= 6 ? 6 : 8);
  int groups = ((rows + rpt - 1) / rpt + 3) / 4 * 4;
  cudaLaunchConfig_t lc = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  lc.attrs = attr;
  lc.numAttrs = 1;
  lc.stream = s;
  auto go = [&](auto rows_per_lane) {
    const int tpc = 256 / (groups * 8);
    lc.gridDim = dim3((unsigned)((p.n_tok + tpc - 1) / tpc));
    lc.blockDim = dim3((unsigned)(tpc * groups * 8));
    return cudaLaunchKernelEx(&lc, kv_quant_append_stream_kernel<T, CS, KV, decltype(rows_per_lane)::value>, x, p,
                              groups);
  };
  cudaError_t e;
  if (groups > 32) {
    // more rows than a CTA holds: a CTA a token, in passes (an ordinary launch)
    kv_quant_append_kernel<T, CS, KV><<<grid, 1024, 0, s>>>(x, p);
    e = cudaGetLastError();
  } else {
    e = rpt == 1   ? go(std::integral_constant<int, 1>{})
        : rpt == 2 ? go(std::integral_constant<int, 2>{})
        : rpt == 3 ? go(std::integral_constant<int, 3>{})
        : rpt == 4 ? go(std::integral_constant<int, 4>{})
        : rpt == 6 ? go(std::integral_constant<int, 6>{})
                   : go(std::integral_constant<int, 8>{});
  }
  if (e != cudaSuccess) return launch_status(e);
  lc.gridDim = dim3((unsigned)device_sm_count());
  lc.blockDim = dim3(256);
  return launch_status(cudaLaunchKernelEx(&lc, kv_quant_repair_kernel<T, CS, KV>, x, p));
}

// ---------------------------------------------------------------------------
// Read back.  Output rows [b, h, s, :] for s < max_len: token s of sequence b
// is token s % bs of its (s / bs)-th valid block (ids outside [0, num_blocks)
// are dropped and later blocks move up, as in the attention kernels); rows at
// or past the context are zero.  HBM-bound: 1 byte read and 2 written a
// value.  A CTA covers `pages` output pages of one sequence; a thread keeps
// two 16-code loads of K and two of V in flight, so that four CTAs fit an SM.
// ---------------------------------------------------------------------------
constexpr int kPages = 4;  // output pages of a CTA, at most

struct DequantParams {
  int64_t B, Hkv, D, num_blocks, block_size, max_blocks, max_len;
  int pages;
};

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  T e[2] = {from_f32<T>(lo), from_f32<T>(hi)};
  return *reinterpret_cast<uint32_t*>(e);
}

template <typename IDX>
__device__ __forceinline__ bool in_pool(IDX id, int64_t nb) {
  return id >= 0 && (int64_t)id < nb;
}

// ids[i] = block of rank first + i among the valid ones of bt[0, n), -1 past
// the last, i < pages.  With nothing dropped up to there (counted by the whole
// CTA) the rank is the index; else one warp walks the table.
template <typename IDX>
__device__ __forceinline__ void cta_find_blocks(const IDX* __restrict__ bt, int64_t n, int64_t nb, int64_t first,
                                                int pages, int64_t* ids) {
  const int lane = threadIdx.x & 31;
  const int64_t upto = min(n, first + pages);
  int dropped = 0;
#pragma unroll 4
  for (int64_t j = threadIdx.x; j < upto; j += blockDim.x) dropped |= !in_pool(__ldg(&bt[j]), nb);
  if ((int)threadIdx.x < pages) {
    const int64_t j = first + threadIdx.x;
    ids[threadIdx.x] = j < n ? (int64_t)__ldg(&bt[j]) : -1;
  }
  if (__syncthreads_or(dropped) == 0) return;
  if ((int)threadIdx.x < pages) ids[threadIdx.x] = -1;
  __syncwarp();
  if (threadIdx.x < 32) {
    int64_t rank0 = 0;
    for (int64_t j0 = 0; j0 < n && rank0 < first + pages; j0 += 32) {
      const IDX v = j0 + lane < n ? __ldg(&bt[j0 + lane]) : (IDX)-1;
      const bool ok = in_pool(v, nb);
      const unsigned ballot = __ballot_sync(0xffffffffu, ok);
      const int64_t rank = rank0 + __popc(ballot & ((1u << lane) - 1u));
      if (ok && rank >= first && rank < first + pages) ids[rank - first] = (int64_t)v;
      rank0 += __popc(ballot);
    }
  }
  __syncthreads();
}

template <typename T, typename KV, typename IDX, bool VEC>
__global__ void __launch_bounds__(256, 4)
    kv_dequant_kernel(const uint8_t* __restrict__ k_cache, const uint8_t* __restrict__ v_cache,
                      const float* __restrict__ k_scale, const float* __restrict__ v_scale,
                      const IDX* __restrict__ block_table, const IDX* __restrict__ context_len,
                      T* __restrict__ k_out, T* __restrict__ v_out, DequantParams p, int64_t chunks) {
  __shared__ int64_t s_id[kPages];
  const int64_t b = blockIdx.x / chunks, first = (blockIdx.x - b * chunks) * p.pages;
  const int64_t bs = p.block_size;
  int64_t ctx = (int64_t)context_len[b];
  const int64_t nvb = ctx > 0 ? min((ctx - 1) / bs + 1, p.max_blocks) : 0;
  ctx = ctx < 0 ? 0 : (ctx < p.max_len ? ctx : p.max_len);
  cta_find_blocks(block_table + b * p.max_blocks, nvb, p.num_blocks, first, p.pages, s_id);
  constexpr int W = VEC ? 16 : 1;  // codes a thread takes at a time
  constexpr int U = 2;             // times in flight, K and V each
  const int Hkv = (int)p.Hkv, cpr = (int)(p.D / W);
  const int per_page = (int)bs * Hkv * cpr;
  for (int i = 0; i < p.pages; ++i) {
    const int64_t row0 = (first + i) * bs;
    if (row0 >= p.max_len) break;
    const int64_t id = s_id[i];
    const int rows = (int)min(bs, p.max_len - row0);
    const int live = id < 0 ? 0 : (int)max((int64_t)0, min((int64_t)rows, ctx - row0));
    const int64_t src0 = id * bs * Hkv * p.D, sc0 = id * Hkv * bs;
    const int64_t dst0 = (b * Hkv * p.max_len + row0) * p.D;
    for (int x0 = threadIdx.x; x0 < per_page; x0 += blockDim.x * U) {
      uint4 raw[2][U];
      float sc[2][U];
      int64_t dst[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int x = x0 + u * (int)blockDim.x;
        const int th = x / cpr, t = th / Hkv, h = th - t * Hkv;
        raw[0][u] = raw[1][u] = make_uint4(0, 0, 0, 0);
        sc[0][u] = sc[1][u] = 0.f;
        dst[u] = x < per_page && t < rows ? dst0 + ((int64_t)h * p.max_len + t) * p.D + (x - th * cpr) * W : -1;
        if (x < per_page && t < live) {
          const int64_t at = src0 + (int64_t)x * W;
          if constexpr (VEC) {
            raw[0][u] = ldg_stream16(k_cache + at);
            raw[1][u] = ldg_stream16(v_cache + at);
          } else {
            raw[0][u].x = k_cache[at];
            raw[1][u].x = v_cache[at];
          }
          sc[0][u] = __ldg(&k_scale[sc0 + h * bs + t]);
          sc[1][u] = __ldg(&v_scale[sc0 + h * bs + t]);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (dst[u] < 0) continue;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          T* out = (w ? v_out : k_out) + dst[u];
          if constexpr (VEC) {
            const uint32_t src[4] = {raw[w][u].x, raw[w][u].y, raw[w][u].z, raw[w][u].w};
            uint32_t o[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              float f[4];
              kv8_to_f32x4<KV>(src[j], f);
              o[2 * j] = pack2<T>(__fmul_rn(f[0], sc[w][u]), __fmul_rn(f[1], sc[w][u]));
              o[2 * j + 1] = pack2<T>(__fmul_rn(f[2], sc[w][u]), __fmul_rn(f[3], sc[w][u]));
            }
            stg256(out, o);
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
  const size_t n = (size_t)claim_entries(T);
  return n == 0 ? 0 : n * 12 + (size_t)(T / 2 + 1) * 4;  // (a shared slot has two tokens at least)
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
  AppendParams p{T,         D, num_blocks * block_size, cs_rows, block_size, q ? (int)Hq : 0,
                 (int)Hkv, -1, {nullptr, nullptr, nullptr, 0}};
  for (int i = 0; i < 17; ++i)
    if (block_size == (1ll << i)) p.lg_bs = i;
  return B200_DISPATCH_HALF(dtype, [&]() -> int {
    if (need > 0) {
      const int64_t n = claim_entries(T);
      p.claim.keys = static_cast<unsigned long long*>(workspace);
      p.claim.owner = reinterpret_cast<int*>(p.claim.keys + n);
      p.claim.shared = p.claim.owner + n;
      p.claim.mask = (uint32_t)(n - 1);
      slot_claim_kernel<<<kClaimCtas, kClaimThreads, 0, s>>>(slot_mapping, positions, T, p.slot_hi, cs_rows, p.claim);
      cudaError_t e = cudaGetLastError();
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
  // one page a CTA until every SM has eight CTAs
  const int64_t out_pages = (max_len + block_size - 1) / block_size;
  int pages = 1;
  while (pages < kPages && B * out_pages > (int64_t)pages * 8 * device_sm_count()) pages *= 2;
  const int64_t chunks = (out_pages + pages - 1) / pages;
  if (chunks * B > 0x7fffffffLL || block_size * Hkv * D > (1 << 28)) return B200_ERR_UNSUPPORTED;
  const bool vec = D % 16 == 0 && aligned16(k_cache) && aligned16(v_cache) && aligned32(k_out) && aligned32(v_out);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  DequantParams p{B, Hkv, D, num_blocks, block_size, max_blocks, max_len, pages};
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
