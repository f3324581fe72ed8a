// Decode attention over 16-bit or 8-bit paged caches whose result is joined
// from pieces: the kernel that streams each sequence's own pages, the kernel
// that joins pieces, and a general kernel for shapes outside the fast path.
//
// A piece is what one stretch of the keys of one query row leaves behind:
// (m, l, o) with o[d] = sum_t 2^(x_t - m) v_t[d], l = sum_t 2^(x_t - m), x_t
// the logits in log2 units (no tokens: m = -1e30 or -inf, l = 0).  Pieces of one row join exactly:
//   M = max m_i,  out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i.
//
// 8-bit caches.  With codes c and scales s (k_t = ks_t ck_t, v_t = vs_t cv_t)
//   x_t = scale log2(e) ks_t (q . ck_t)
//   out = sum_t 2^(x_t) vs_t cv_t / sum_t 2^(x_t)
// so the codes go to the tensor cores as they are and the scales meet fp32
// values only: the kernels keep y_t = x_t + log2 vs_t, take maxima over y,
// feed weights w_t = 2^(y_t - m) to the second product with the bare codes, and sum
// l = sum_t w_t / vs_t in fp32.  Taking maxima over y rather than x keeps the largest
// weight at 1 however the value scales of the tokens differ.
// The streaming kernel multiplies int8 codes by bytes of the queries and weights.
// e4m3 codes there, and all codes in the prefix kernel, are widened to f16 (exact),
// with q in f16 after an exact power-of-two scaling of each row, and the weights
// rounded to f16: off by 2^-11 of themselves, or by 2^-32 of the largest where
// that is more (m sits 2^7 below the largest weight, see ref_below).
#pragma once

#include <math.h>

#include "common.cuh"
#include "decode_mma.cuh"
#include "kv8.cuh"
#include "sm100.cuh"

namespace b200 {

constexpr int kPieceDim = 128;
constexpr int kChunk = 16;  // tokens of a chunk
constexpr int kPiecePitch = kPieceDim + 8;  // floats of a piece row: o[128], m, l, pad to whole 32-byte sectors
constexpr int kMaxSeg = 2048;               // (sequence, head group) segments a launch takes

// One attention call, as the C entries take it (host side).
struct AttnCall {
  const void *q, *k_cache, *v_cache;
  const float *k_scale, *v_scale;  // null for 16-bit caches
  const void *prefix_table, *prefix_len;  // null without a shared prefix
  const void *block_table, *context_len;
  void* out;
  int64_t B, Hq, Hkv, D, num_blocks, block_size, max_blocks, max_prefix_blocks;
  float scale;  // logits = scale * q . k
  int32_t dtype, cache_dtype, index_dtype;
};

// Launch geometry of the fast path.
struct PieceGeom {
  bool fast;
  bool whole;             // short tables: a CTA a segment, and nothing to join
  int G, HG, n_hg, sub;   // query heads a kv head, kv heads a CTA, head groups, warps a kv head
  int stages, grid;
  int64_t seqs;           // sequences a launch takes (the batch runs in slices of this many)
  uint32_t entry_bytes;
  size_t smem;
  bool pdl;
};

// Workspace: [spans | pieces of the own pages | pieces of the prefix].  A segment's
// span: its first range, and how many ranges left a piece (-1: the row itself is written).
struct PieceSpace {
  int2* spans;    // nseg
  float* rows;    // piece segment + range, heads_cta rows each
  float* prefix;  // split-major: [splits][seqs * Hq] rows
  int prefix_splits;
};

int launch_pieces_i8(const AttnCall& a, const PieceGeom& g, const PieceSpace& w, bool overlap, cudaStream_t s);
int launch_pieces_e4m3(const AttnCall& a, const PieceGeom& g, const PieceSpace& w, bool overlap, cudaStream_t s);
int launch_pieces_16(const AttnCall& a, const PieceGeom& g, const PieceSpace& w, bool overlap, cudaStream_t s);
int launch_attn_generic_i8(const AttnCall& a, cudaStream_t s);
int launch_attn_generic_e4m3(const AttnCall& a, cudaStream_t s);
int launch_attn_generic_16(const AttnCall& a, cudaStream_t s);

// Ids outside [0, num_blocks) among a table's n, this thread's share: sixteen loads in flight.
template <typename I>
__device__ __forceinline__ int dropped_ids(const I* __restrict__ ids, int n, int64_t num_blocks) {
  int drop = 0;
#pragma unroll 1
  for (int j = threadIdx.x; j < n; j += 16 * blockDim.x) {
    I v[16];
#pragma unroll
    for (int u = 0; u < 16; ++u) {
      const int k = j + u * (int)blockDim.x;
      v[u] = k < n ? __ldg(ids + k) : 0;
    }
#pragma unroll
    for (int u = 0; u < 16; ++u) drop += v[u] < 0 || (int64_t)v[u] >= num_blocks;
  }
  return drop;
}

// Block ids and lengths are int32 or int64 by a flag (uniform; read by one warp).
struct IndexPtr {
  const void* p;
  int wide;
  __device__ __forceinline__ int64_t at(int64_t i) const {
    return wide ? __ldg(static_cast<const long long*>(p) + i) : (int64_t)__ldg(static_cast<const int*>(p) + i);
  }
  __device__ __forceinline__ int dropped(int64_t first, int n, int64_t num_blocks) const {
    return wide ? dropped_ids(static_cast<const long long*>(p) + first, n, num_blocks)
                : dropped_ids(static_cast<const int*>(p) + first, n, num_blocks);
  }
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Shared memory by 32-bit address (the kernels' base is aligned at run time,
// which hides its address space from the compiler: plain accesses would be generic).
__device__ __forceinline__ float lds_f32(uint32_t a) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float4 lds_f32x4(uint32_t a) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(a)
               : "memory");
  return v;
}
__device__ __forceinline__ int lds_s32(uint32_t a) {
  int v;
  asm volatile("ld.shared.s32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void sts_f32(uint32_t a, float v) {
  asm volatile("st.shared.f32 [%0], %1;" ::"r"(a), "f"(v) : "memory");
}
__device__ __forceinline__ void sts128(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

namespace {

// ---------------------------------------------------------------------------
// General kernel: any D <= 256, block size, head ratio and alignment.  One
// CTA of four warps a (sequence, query head); tokens dealt round-robin to the warps, lanes
// over the head dim; the prefix's pages first, then the sequence's own.
// ---------------------------------------------------------------------------
template <typename T, typename KV>
__global__ void __launch_bounds__(128)
    paged_attn_pieces_generic_kernel(const T* __restrict__ q, const KV* __restrict__ kc, const KV* __restrict__ vc,
                                     const float* __restrict__ ks, const float* __restrict__ vs, IndexPtr ptab,
                                     IndexPtr plen, IndexPtr btab, IndexPtr clen, T* __restrict__ out, int64_t Hq,
                                     int64_t Hkv, int64_t D, int64_t num_blocks, int64_t bs, int64_t max_blocks,
                                     int64_t max_prefix, float qscale) {
  __shared__ float s_m[4], s_l[4], s_o[4][256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t hq = blockIdx.x, b = blockIdx.y;
  const int64_t kvh = hq / (Hq / Hkv);
  const T* qr = q + (b * Hq + hq) * D;
  float qv[8], ov[8];
  for (int i = 0; i < 8; ++i) {
    const int64_t d = lane + 32 * i;
    qv[i] = d < D ? to_f32(qr[d]) : 0.f;
    ov[i] = 0.f;
  }
  float mrun = -INFINITY, lrun = 0.f;
  for (int part = ptab.p != nullptr ? 0 : 1; part < 2; ++part) {
    const IndexPtr tab = part ? btab : ptab;
    const int64_t at0 = part ? b * max_blocks : 0;
    const int64_t ctx = part ? clen.at(b) : plen.at(0);
    const int64_t nvb = ctx > 0 ? min((ctx - 1) / bs + 1, part ? max_blocks : max_prefix) : 0;
    int64_t rank = 0;
    for (int64_t j = 0; j < nvb; ++j) {
      const int64_t id = tab.at(at0 + j);
      if (id < 0 || id >= num_blocks) continue;
      int64_t nt = ctx - rank * bs;
      ++rank;
      nt = nt < 0 ? 0 : (nt > bs ? bs : nt);
      for (int64_t t = warp; t < nt; t += 4) {
        const int64_t row = ((id * bs + t) * Hkv + kvh) * D;
        float part_sum = 0.f;
        for (int i = 0; i < 8; ++i) {
          const int64_t d = lane + 32 * i;
          if (d < D) part_sum = fmaf(qv[i], (float)kc[row + d], part_sum);
        }
        float sc = warp_sum(part_sum) * qscale, vscale = 1.f;
        if constexpr (sizeof(KV) == 1) {
          const int64_t sat = (id * Hkv + kvh) * bs + t;
          sc *= ks[sat];
          vscale = vs[sat];
        }
        const float mn = fmaxf(mrun, sc);
        const float a = (mrun == -INFINITY) ? 0.f : exp2f(mrun - mn);
        const float pw = sc == -INFINITY ? 0.f : exp2f(sc - mn);
        lrun = lrun * a + pw;
        for (int i = 0; i < 8; ++i) {
          const int64_t d = lane + 32 * i;
          ov[i] = ov[i] * a + (d < D ? pw * ((float)vc[row + d] * vscale) : 0.f);
        }
        mrun = mn;
      }
    }
  }
  if (lane == 0) {
    s_m[warp] = mrun;
    s_l[warp] = lrun;
  }
  for (int i = 0; i < 8; ++i) {
    const int64_t d = lane + 32 * i;
    if (d < D) s_o[warp][d] = ov[i];
  }
  __syncthreads();
  float M = -INFINITY;
  for (int w = 0; w < 4; ++w) M = fmaxf(M, s_m[w]);
  float L = 0.f, wts[4];
  for (int w = 0; w < 4; ++w) {
    wts[w] = (s_m[w] == -INFINITY) ? s_l[w] : exp2f(s_m[w] - M);  // (no tokens: 0; NaN logits only: NaN)
    L += wts[w] * s_l[w];
  }
  for (int64_t d = threadIdx.x; d < D; d += blockDim.x) {
    float acc = 0.f;
    for (int w = 0; w < 4; ++w) acc += wts[w] * s_o[w][d];
    out[(b * Hq + hq) * D + d] = from_f32<T>(L == 0.f ? 0.f : acc / L);
  }
}

// ---------------------------------------------------------------------------
// 8-bit pages on the tensor cores.  As in the 16-bit tiles tokens (S^T = K Q^T)
// and head dims (O^T = V^T P^T) are the M side and the G query heads the N side.
// K comes by ldmatrix (lane (r, q) holds codes 4q.. of token r), V by the
// byte-transposing ldmatrix (codes of four tokens of dim r), whose row order makes
// a lane's four tokens {2q, 2q + 1, 8 + 2q, 9 + 2q}: those a movmatrix of the weights delivers.
// int8: m16n8k32 tiles of bytes, so that codes need no widening (which was half
// of the instructions: 64 sequences 121 us with codes widened to f16, 114 us
// so).  The other operand is a sum of byte terms, a product each:
//   q   the row scaled by a power of two to [2^30, 2^31) and rounded to an integer,
//       its four bytes (the top one signed): off by 2^-31 of the row's largest.  The
//       last byte is zero but for elements below 2^-15 of the largest (fp16: 2^-12);
//       its products run where a warp's rows have such elements (without it one
//       element 2^18 above the others, over a key channel of zeros, left them 6 bits)
//   w   relative to the largest of its 32 tokens (so that a long flat tail behind
//       one large weight keeps its bits), as a 16-bit integer, two unsigned bytes:
//       off by 2^-17 of that largest
// e4m3: widened to f16, m16n8k16 tiles (the m16n8k32 tiles of e4m3 are no
// hardware form here: ten instructions each); w in f16.
// ---------------------------------------------------------------------------
// Power-of-two factors that take a row with this largest magnitude to [2^X,
// 2^(X + 1)) and back; zero and non-finite rows stay.
template <int X>
__device__ __forceinline__ void pow2_scale(float amax, float& up, float& down) {
  int e = (int)(__float_as_uint(amax) >> 23) - 127;
  e = (amax == 0.f || e > 127) ? X : (e < -100 ? -100 : e);
  up = __uint_as_float((uint32_t)(X - e + 127) << 23);
  down = __uint_as_float((uint32_t)(e - X + 127) << 23);
}

// This warp's query rows as B fragments; slA, slB: logit factors of heads 2q, 2q + 1.
// int8: qf[8t + i], t = 0 the top byte, holds dims 16i + 4q + {0..3} of head r
// (zero for r >= G); true where a last byte (t = 3) of the warp is not zero.
// e4m3: qf[2i + {0, 1}] those dims in f16; false.
template <typename KV>
constexpr int q_words() { return std::is_same<KV, int8_t>::value ? 32 : 16; }
template <typename T, typename KV, int G>
__device__ __forceinline__ bool load_q_frags8(const T* __restrict__ qrow0, int lane, float qscale,
                                              uint32_t (&qf)[q_words<KV>()], float& slA, float& slB) {
  const int qh = lane >> 2, qc = (lane & 3) * 4;
  const T* qr = qrow0 + (qh < G ? qh : 0) * kD;
  float f[8][4];
  float amax = 0.f;
  bool bad = false;  // an infinity or a NaN: the row's logits are NaN
  uint32_t low = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint2 raw = *reinterpret_cast<const uint2*>(qr + 16 * i + qc);
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      f[i][u] = qh < G ? to_f32(e[u]) : 0.f;
      amax = fmaxf(amax, fabsf(f[i][u]));
      bad |= !(fabsf(f[i][u]) < INFINITY);
    }
  }
  amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
  amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
  float up, down;
  if constexpr (std::is_same<KV, int8_t>::value) {
    pow2_scale<22>(amax, up, down);  // (units of the third byte)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        v[u] = (uint32_t)__float2int_rn(f[i][u] * up * 256.0f);
        low |= v[u];
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int sel = 3 - t;
        const uint32_t lo = __byte_perm(v[0], v[1], sel | ((4 + sel) << 4));
        const uint32_t hi = __byte_perm(v[2], v[3], sel | ((4 + sel) << 4));
        qf[8 * t + i] = __byte_perm(lo, hi, 0x5410);
      }
    }
  } else {
    pow2_scale<13>(amax, up, down);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      qf[2 * i] = pack_pair<__half>(f[i][0] * up, f[i][1] * up);
      qf[2 * i + 1] = pack_pair<__half>(f[i][2] * up, f[i][3] * up);
    }
  }
  const unsigned any = __ballot_sync(0xffffffffu, bad);
  const float sl = any & (0xfu << (lane & ~3)) ? __uint_as_float(0x7fc00000u) : qscale * down;
  slA = __shfl_sync(0xffffffffu, sl, (lane & 3) * 8);
  slB = __shfl_sync(0xffffffffu, sl, (lane & 3) * 8 + 4);
  return std::is_same<KV, int8_t>::value && __any_sync(0xffffffffu, (low & 0xffu) != 0);
}

// Running maximum of a head without tokens: so low that any logit raises it
// and nothing scaled by it survives, and finite, so that differences are.
constexpr float kNoMax = -1e30f;

// How far below the largest logit the reference mu is set.  Weights that go to f16 are
// 2^7 where it is set and, as it may lag by 2^8, 2^15 at most: the range of f16 then
// holds weights down to 2^-21 of the largest in full, and to 2^-32 as
// subnormals (set at the largest itself 2^-14 and 2^-25: a long flat tail
// behind one loud key lost its bits).  bf16 has the range of fp32.
template <typename M>
constexpr float ref_below() { return std::is_same<M, __half>::value ? 7.0f : 0.0f; }

// Sets the references of this thread's two heads `below` m where that raises them.
__device__ __forceinline__ void raise_to(const float (&m)[2], float below, float (&mu)[2], float (&lp)[2],
                                         float (&o)[8][4]) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const float ref = m[c] - below;
    if (!(ref > mu[c])) continue;
    const float alpha = ex2(mu[c] - ref);
    mu[c] = ref;
    lp[c] *= alpha;
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) {
      o[mt][c] *= alpha;
      o[mt][c + 2] *= alpha;
    }
  }
}

// The same to the largest logits in the warp (of this thread: top), when one
// exceeds that place by more than 2^8 (exact: O and l share the reference).  Most
// entries need one vote here and no exchange.
template <typename M>
__device__ __forceinline__ void raise_max_lazy(const float (&top)[2], float (&mu)[2], float (&lp)[2],
                                               float (&o)[8][4]) {
  constexpr float kBelow = ref_below<M>();
  float m[2] = {top[0], top[1]};
  if (!__any_sync(0xffffffffu, m[0] - mu[0] > 8.0f + kBelow || m[1] - mu[1] > 8.0f + kBelow)) return;
#pragma unroll
  for (int off = 4; off <= 16; off <<= 1) {
    m[0] = fmaxf(m[0], __shfl_xor_sync(0xffffffffu, m[0], off));
    m[1] = fmaxf(m[1], __shfl_xor_sync(0xffffffffu, m[1], off));
  }
  raise_to(m, kBelow, mu, lp, o);
}

// Where a lane reads an entry's two chunks: its ldmatrix row of K with its first
// 16 bytes (16 bytes 2j + k of the row are 32 j on, in the swizzle an exclusive
// or), its row of V, its token's key scale, the head's rows of V; bytes of a chunk.
struct Lane8 {
  uint32_t k_at, v_at, scale_at, v_rows, chunk;
  __device__ __forceinline__ Lane8(int w, uint32_t box, int lane) {
    chunk = 2 * box + 1024;
    const int mat = lane >> 3, krow = w * 16 + (mat & 1) * 8 + (lane & 7);
    k_at = krow * 128 + (((mat >> 1) ^ (krow & 7)) << 4);
    // V: lanes 0-15 the first chunk's tokens in the order 0, 1, 8, 9, 2, 3, 10, 11, ...
    const int vrow = w * 16 + ((lane >> 2) & 3) * 2 + (lane & 1) + ((lane & 2) << 2);
    v_at = (lane >> 4) * chunk + box + vrow * 128 + ((vrow & 7) << 4);
    v_rows = box + (uint32_t)(w * 16) * 128;
    scale_at = 2 * box + (uint32_t)(w * 16 + (lane >> 2)) * 4;
  }
};

// Two chunks of sixteen tokens (nt[c] of them live) of one kv head, folded into
// the running (o, mu, lp): codes as [head][token][128] rows, 128-byte
// swizzled, scales as [head][token], the entry at `at`.
template <typename KV>
__device__ __forceinline__ void mma_pair8(uint32_t at, const Lane8& x, const int (&nt)[2], int lane, float slA,
                                          float slB, const uint32_t (&qf)[q_words<KV>()], bool last_byte,
                                          float (&o)[8][4], float (&mu)[2], float (&lp)[2]) {
  constexpr bool kInt = std::is_same<KV, int8_t>::value;
  const int tr = lane >> 2;
  float y[2][4], iv[2][2];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const uint32_t ka = at + c * x.chunk + x.k_at, sa = at + c * x.chunk + x.scale_at;
    // products of tokens tr and tr + 8 with heads 2(lane%4), +1
    float s[4];
    if constexpr (kInt) {
      int32_t d[3][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t kr[4];
        ldsm_x4(ka ^ (j << 5), kr[0], kr[1], kr[2], kr[3]);
        if (j == 0) {
          mma8_start<false>(d[0], kr, qf[0], qf[1], kAccStart);
          mma8_start<true>(d[1], kr, qf[8], qf[9], kAccStart);
          mma8_start<true>(d[2], kr, qf[16], qf[17], kAccStart);
        } else {
          mma8_add<false>(d[0], kr, qf[2 * j], qf[2 * j + 1]);
          mma8_add<true>(d[1], kr, qf[8 + 2 * j], qf[9 + 2 * j]);
          mma8_add<true>(d[2], kr, qf[16 + 2 * j], qf[17 + 2 * j]);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        float m0, m1, b0, b1;
        acc_values(d[0][i], d[0][i + 1], s[i], s[i + 1]);
        acc_values(d[1][i], d[1][i + 1], m0, m1);
        acc_values(d[2][i], d[2][i + 1], b0, b1);
        sm100::ffma2(m0, m1, s[i], s[i + 1], 256.0f, 256.0f, m0, m1);
        sm100::ffma2(s[i], s[i + 1], m0, m1, 256.0f, 256.0f, b0, b1);
      }
      if (last_byte) {  // (uniform; the rows of K once more rather than held)
        int32_t e[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t kr[4];
          ldsm_x4(ka ^ (j << 5), kr[0], kr[1], kr[2], kr[3]);
          if (j == 0) mma8_start<true>(e, kr, qf[24], qf[25], kAccStart);
          else mma8_add<true>(e, kr, qf[24 + 2 * j], qf[25 + 2 * j]);
        }
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          float e0, e1;
          acc_values(e[i], e[i + 1], e0, e1);
          sm100::ffma2(s[i], s[i + 1], e0, e1, 1.0f / 256.0f, 1.0f / 256.0f, s[i], s[i + 1]);
        }
      }
    } else {
      float s1[4] = {0.f, 0.f, 0.f, 0.f};
      s[0] = s[1] = s[2] = s[3] = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t kr[4], a[4][2];
        ldsm_x4(ka ^ (j << 5), kr[0], kr[1], kr[2], kr[3]);
#pragma unroll
        for (int i = 0; i < 4; ++i) kv8_in_order<KV>(kr[i], a[i][0], a[i][1]);
        mma16816<__half>(s, a[0][0], a[1][0], a[0][1], a[1][1], qf[4 * j], qf[4 * j + 1]);
        mma16816<__half>(s1, a[2][0], a[3][0], a[2][1], a[3][1], qf[4 * j + 2], qf[4 * j + 3]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] += s1[i];
    }
    const float k0 = lds_f32(sa), k1 = lds_f32(sa + 32);
    float lv0, lv1;
    kv8_value_scale(lds_f32(sa + 512), lv0, iv[c][0]);
    kv8_value_scale(lds_f32(sa + 544), lv1, iv[c][1]);
    sm100::ffma2(y[c][0], y[c][1], s[0], s[1], k0 * slA, k0 * slB, lv0, lv0);
    sm100::ffma2(y[c][2], y[c][3], s[2], s[3], k1 * slA, k1 * slB, lv1, lv1);
    if (nt[c] < 16) {
      // tokens past the end may hold any code and any scale: no weight, and no V
      // (an e4m3 NaN times a weight of 0 is NaN: their rows are zeroed)
      if (tr >= nt[c]) y[c][0] = y[c][1] = -INFINITY, iv[c][0] = 0.f;
      if (tr + 8 >= nt[c]) y[c][2] = y[c][3] = -INFINITY, iv[c][1] = 0.f;
      if (!kInt) {
        for (int i = nt[c] * 8 + lane; i < 128; i += 32)
          sts128(at + c * x.chunk + x.v_rows + i * 16, make_uint4(0, 0, 0, 0));
        sm100::fence_proxy_async_smem();  // (before the entry's next filling)
        __syncwarp();
      }
    }
  }
  float m[2] = {fmaxf(sm100::fmax3(y[0][0], y[0][2], y[1][0]), y[1][2]),
                fmaxf(sm100::fmax3(y[0][1], y[0][3], y[1][1]), y[1][3])};
  const uint32_t va = at + x.v_at;
  if constexpr (kInt) {
    // the pair's largest y of the two heads, over the eight lanes that hold its tokens
#pragma unroll
    for (int off = 4; off <= 16; off <<= 1) {
      m[0] = fmaxf(m[0], __shfl_xor_sync(0xffffffffu, m[0], off));
      m[1] = fmaxf(m[1], __shfl_xor_sync(0xffffffffu, m[1], off));
    }
    m[0] = fmaxf(m[0], kNoMax), m[1] = fmaxf(m[1], kNoMax);
    if (__any_sync(0xffffffffu, m[0] - mu[0] > 8.0f || m[1] - mu[1] > 8.0f)) raise_to(m, 0.f, mu, lp, o);
    const float f[2] = {ex2(m[0] - mu[0]), ex2(m[1] - mu[1])};
    // weights relative to the pair's largest, as B fragments: pb[t][c], t = 0 the high byte
    uint32_t pb[2][2];
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      // 16-bit integers by 2^23 + 65535 w; a 16-bit cell of the transposed matrix is one weight
      uint32_t u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float w = ex2(y[c][i] - m[i & 1]);
        sum[i & 1] = fmaf(w, iv[c][i >> 1], sum[i & 1]);
        u[i] = __float_as_uint(fmaf(w, 65535.0f, 8388608.0f));
      }
      const uint32_t t0 = movm_t(__byte_perm(u[0], u[1], 0x5410)), t1 = movm_t(__byte_perm(u[2], u[3], 0x5410));
      pb[0][c] = __byte_perm(t0, t1, 0x7531);
      pb[1][c] = __byte_perm(t0, t1, 0x6420);
    }
    lp[0] = fmaf(f[0], sum[0], lp[0]);
    lp[1] = fmaf(f[1], sum[1], lp[1]);
    const float fo[2] = {f[0] * (1.0f / 65535.0f), f[1] * (1.0f / 65535.0f)};
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) {
      uint32_t a[4];
      int32_t d[4], e[4];
      ldsm_x2_t8(va ^ (mt << 4), a);
      mma8_start<true>(d, a, pb[0][0], pb[0][1], kAccStart);
      mma8_start<true>(e, a, pb[1][0], pb[1][1], kAccStart);
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        float x0, x1, z0, z1;
        acc_values(d[i], d[i + 1], x0, x1);
        acc_values(e[i], e[i + 1], z0, z1);
        sm100::ffma2(x0, x1, x0, x1, 256.0f, 256.0f, z0, z1);
        sm100::ffma2(o[mt][i], o[mt][i + 1], x0, x1, fo[0], fo[1], o[mt][i], o[mt][i + 1]);
      }
    }
  } else {
    raise_max_lazy<__half>(m, mu, lp, o);
    uint32_t pb[2][2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const float p0 = ex2(y[c][0] - mu[0]), p2 = ex2(y[c][2] - mu[0]);
      const float p1 = ex2(y[c][1] - mu[1]), p3 = ex2(y[c][3] - mu[1]);
      lp[0] = fmaf(p0, iv[c][0], fmaf(p2, iv[c][1], lp[0]));
      lp[1] = fmaf(p1, iv[c][0], fmaf(p3, iv[c][1], lp[1]));
      pb[c][0] = movm_t(pack_pair<__half>(p0, p1));
      pb[c][1] = movm_t(pack_pair<__half>(p2, p3));
    }
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) {
      uint32_t v[4], a[4][2];
      ldsm_x2_t8(va ^ (mt << 4), v);
#pragma unroll
      for (int i = 0; i < 4; ++i) kv8_in_order<KV>(v[i], a[i][0], a[i][1]);
      mma16816<__half>(o[mt], a[0][0], a[1][0], a[0][1], a[1][1], pb[0][0], pb[0][1]);
      mma16816<__half>(o[mt], a[2][0], a[3][0], a[2][1], a[3][1], pb[1][0], pb[1][1]);
    }
  }
}

// One chunk of a 16-bit cache: K and V as [half of the dims][token][64] rows.
template <typename T>
__device__ __forceinline__ void mma_chunk16(uint32_t kb, uint32_t vb, int ntok, int lane, float sl,
                                            const uint32_t (&qb)[8][2], float (&o)[8][4], float (&mu)[2], float (&lp)[2]) {
  constexpr uint32_t kHalf = kChunk * 128;
  const int mat = lane >> 3, mrow = lane & 7;
  const int tr = lane >> 2, tq = (lane & 3) * 2;
  float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
  {
    // A = K rows: matrix `mat` = (token half mat&1, dim-chunk parity mat>>1)
    const int row = (mat & 1) * 8 + mrow;
    const uint32_t at = kb + row * 128, sw = ((mat >> 1) ^ (row & 7)) << 4;
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) {
      uint32_t a0, a1, a2, a3;
      ldsm_x4(at + (ks >> 2) * kHalf + (sw ^ ((ks & 3) << 5)), a0, a1, a2, a3);
      mma16816<T>((ks & 1) ? s1 : s0, a0, a1, a2, a3, qb[ks][0], qb[ks][1]);
    }
  }
  // A = V^T by ldmatrix.trans: matrix `mat` = (token half mat>>1, dim-chunk parity mat&1)
  uint32_t va[8][4];
  {
    const int row = (mat >> 1) * 8 + mrow;
    const uint32_t at = vb + row * 128, sw = ((mat & 1) ^ (row & 7)) << 4;
#pragma unroll
    for (int mt = 0; mt < 8; ++mt)
      ldsm_x4_t(at + (mt >> 2) * kHalf + (sw ^ ((mt & 3) << 5)), va[mt][0], va[mt][1], va[mt][2], va[mt][3]);
  }
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = (s0[i] + s1[i]) * sl;
  if (ntok < 16) {
    if (tr >= ntok) y[0] = y[1] = -INFINITY;
    if (tr + 8 >= ntok) y[2] = y[3] = -INFINITY;
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) {
      va[mt][0] = mask_pair(va[mt][0], tq, ntok);
      va[mt][1] = mask_pair(va[mt][1], tq, ntok);
      va[mt][2] = mask_pair(va[mt][2], 8 + tq, ntok);
      va[mt][3] = mask_pair(va[mt][3], 8 + tq, ntok);
    }
  }
  const float top[2] = {fmaxf(y[0], y[2]), fmaxf(y[1], y[3])};
  raise_max_lazy<T>(top, mu, lp, o);
  const float p0 = ex2(y[0] - mu[0]), p2 = ex2(y[2] - mu[0]);
  const float p1 = ex2(y[1] - mu[1]), p3 = ex2(y[3] - mu[1]);
  lp[0] += p0 + p2;
  lp[1] += p1 + p3;
  const uint32_t b0 = movm_t(pack_pair<T>(p0, p1));
  const uint32_t b1 = movm_t(pack_pair<T>(p2, p3));
#pragma unroll
  for (int mt = 0; mt < 8; ++mt) mma16816<T>(o[mt], va[mt][0], va[mt][1], va[mt][2], va[mt][3], b0, b1);
}

// store_rows with a NaN sum reaching the output (it has no value for l > 0 to fail).
template <typename T, int G>
__device__ __forceinline__ void store_rows_nan(T* __restrict__ orow0, const float (&o)[8][4], float lA, float lB,
                                               int lane) {
  const float iA = lA == 0.f ? 0.f : 1.f / lA, iB = lB == 0.f ? 0.f : 1.f / lB;
  const int h = lane >> 2, tq = (lane & 3) * 2;
  T* orow = orow0 + (h < G ? h : 0) * kD;
#pragma unroll
  for (int mt = 0; mt < 8; ++mt) {
    const uint32_t r0 = movm_t(pack_pair<T>(o[mt][0] * iA, o[mt][1] * iB));
    const uint32_t r1 = movm_t(pack_pair<T>(o[mt][2] * iA, o[mt][3] * iB));
    if (h < G) {
      *reinterpret_cast<uint32_t*>(orow + 16 * mt + tq) = r0;
      *reinterpret_cast<uint32_t*>(orow + 16 * mt + 8 + tq) = r1;
    }
  }
}

// ---------------------------------------------------------------------------
// Streaming kernel.  All segments' block-table entries (segment s = hg * B + b)
// laid end to end are cut into one equal contiguous range a CTA, one CTA an
// SM.  The producer warp walks its range and fills a ring with TMA; an entry is
// one chunk of sixteen tokens of a page (16-bit caches) or two (8-bit): K and V boxes of
// HG heads, and for 8-bit caches the tokens' scales.  sub consumer warps share
// a kv head: entry i goes to the HG warps of slot i % sub, so that eight
// warps have work whatever Hkv is.  End
// markers, one for each slot, close a segment: the warps of a head add up their (m,
// l, o) in shared memory, and the first writes the normalised row when the
// range holds the whole segment, else the range's piece at row segment +
// range -- the (segment, range) pairs of a call, taken in order, have distinct sums, so
// a piece's place needs no counters.  No state is kept between calls.
// Where the table bounds every segment to a few entries, a CTA takes a segment
// whole and there are no pieces.
// ---------------------------------------------------------------------------
struct PiecesParams {
  int64_t B, Hq, Hkv, num_blocks, max_blocks;
  int bs, HG, n_hg, sub, stages, nseg;
  int scale_maps;  // scales by tensor maps (pages of more than 16 tokens), else one copy a page
  int always;   // write every segment as pieces (a prefix joins them)
  int whole;    // range c is segment c
  int overlap;  // launched beside the previous grid of the call: wait for it at the end
  uint32_t entry_bytes;
  float qscale;  // scale * log2(e)
};

constexpr int kConsumers = 8;  // consumer warps, at most
struct EntryMeta {
  int kind;  // 0 tokens, 1 end of segment, 2 end of stream
  int seg;
  int ntok;   // live tokens of the first chunk
  int piece;  // live tokens of the second; end of segment: row of the piece, -1: the segment's only one
};
constexpr int kXchPitch = 36 * 32;  // floats a warp hands over: 32 o, 2 m, 2 l a lane

__device__ __forceinline__ int64_t range_lo(int64_t c, int64_t E, int64_t R) { return c * E / R; }
__device__ __forceinline__ int range_of(int64_t e, int64_t E, int64_t R) {
  return (int)(((e + 1) * R + E - 1) / E - 1);
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
      "r"(bytes), "r"(bar)
      : "memory");
}

template <typename T, typename KV, int G>
__global__ void __launch_bounds__((kConsumers + 1) * 32, 1)
    paged_attn_pieces_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                             const __grid_constant__ CUtensorMap tm_ks, const __grid_constant__ CUtensorMap tm_vs,
                             const float* __restrict__ k_scale, const float* __restrict__ v_scale,
                             const T* __restrict__ q, IndexPtr btab, IndexPtr clen, T* __restrict__ out,
                             float* __restrict__ ws_rows, int2* __restrict__ ws_spans, PiecesParams p) {
  constexpr bool k8 = sizeof(KV) == 1;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int HG = p.HG, bs = p.bs, sub = p.sub, consumers = HG * sub;
  const int heads_cta = HG * G;
  const int64_t B = p.B;
  float* xch = reinterpret_cast<float*>(smem + p.stages * p.entry_bytes);  // [sub - 1][HG][kXchPitch]
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(xch + (sub - 1) * HG * kXchPitch);
  uint64_t* empty_bar = full_bar + p.stages;
  uint64_t* xch_full = empty_bar + p.stages;  // [8]
  uint64_t* xch_empty = xch_full + 8;         // [8]
  static_assert(sizeof(EntryMeta) == 16, "read as one vector");
  EntryMeta* meta = reinterpret_cast<EntryMeta*>(xch_empty + 8);
  int* s_cum = reinterpret_cast<int*>(meta + p.stages);
  int* s_ctx = s_cum + (p.nseg + 1);
  int* chunk_id = s_ctx + B;
  int* chunk_ntok = chunk_id + 32;
  int* s_abort = chunk_ntok + 32;
  int* s_drop = s_abort + 1;  // dropped entries of the first segment before this range

  // the join kernel may be scheduled; it waits for this grid
  asm volatile("griddepcontrol.launch_dependents;");
  // ---- prologue: contexts, entries before each segment, barriers
  {
    const int64_t most = p.max_blocks * bs;
    for (int64_t b = threadIdx.x; b < B; b += blockDim.x) {
      const int64_t c = clen.at(b);
      s_ctx[b] = (int)(c < 0 ? 0 : (c < most ? c : most));
    }
    __syncthreads();
  }
  if (warp == consumers) {
    int run = 0;
    for (int s0 = 0; s0 < p.nseg; s0 += 32) {
      const int s = s0 + lane;
      const int e = s < p.nseg ? (s_ctx[s % (int)B] + bs - 1) / bs : 0;
      int incl = e;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      if (s < p.nseg) s_cum[s + 1] = run + incl;
      run += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) {
      s_cum[0] = 0;
      *s_abort = 0;
      *s_drop = 0;
    }
  } else if (warp == 0 && lane == 0) {
    for (int s = 0; s < p.stages; ++s) {
      sm100::mbar_init(sm100::smem_u32(&full_bar[s]), 1);
      sm100::mbar_init(sm100::smem_u32(&empty_bar[s]), HG);
    }
    for (int w = 0; w < HG; ++w) {
      sm100::mbar_init(sm100::smem_u32(&xch_full[w]), sub > 1 ? sub - 1 : 1);
      sm100::mbar_init(sm100::smem_u32(&xch_empty[w]), 1);
    }
    sm100::fence_barrier_init();
  }
  __syncthreads();
  const int64_t E = s_cum[p.nseg];
  const int64_t R = p.whole || E > (int64_t)gridDim.x ? (int64_t)gridDim.x : E;  // ranges
  const int c = blockIdx.x;
  int64_t lo = c < R ? range_lo(c, E, R) : 0, hi = c < R ? range_lo(c + 1, E, R) : 0;
  int seg0 = 0;  // segment of the range's first entry
  if (p.whole) {
    seg0 = c;
    lo = s_cum[c], hi = s_cum[c + 1];
  } else if (c < R) {
    int r = p.nseg;  // cum[seg0] <= lo < cum[r]
    while (r - seg0 > 1) {
      const int mid = (seg0 + r) >> 1;
      if (s_cum[mid] <= lo) seg0 = mid;
      else r = mid;
    }
    // Dropped entries before the range shift the token ranks of its pages:
    // counted by the whole CTA (over 8192 entries a warp alone takes 20 us, the
    // CTA with a load at a time 12; 3 sequences of 90001..131072 tokens: 131 us, so 124).
    const int j0 = (int)(lo - s_cum[seg0]);
    if (j0 > 0) {
      int drop = btab.dropped((seg0 % B) * p.max_blocks, j0, p.num_blocks);
      drop = __reduce_add_sync(0xffffffffu, drop);
      if (lane == 0 && drop) atomicAdd(s_drop, drop);
      __syncthreads();
    }
  }

  // Programmatic launch (cfg flags bit 3): what is above and the producer's
  // walk of the block table up to its first copy overlap the previous kernel,
  // whose caller guarantees that it writes neither context_len nor block_table.  No
  // q, page, output or workspace byte is touched before the wait.  A no-op for an
  // ordinary launch.  `overlap`: the previous kernel is the same call's prefix
  // grid, which shares nothing with this one; the wait comes at the end.
  if (warp < consumers && !p.overlap) asm volatile("griddepcontrol.wait;" ::: "memory");
  if (c == 0 && warp < consumers && !p.whole) {
    for (int s = threadIdx.x; s < p.nseg; s += consumers * 32) {
      const int64_t s0 = s_cum[s], s1 = s_cum[s + 1];
      int2 span = make_int2(0, 0);
      if (s1 > s0) {
        const int c1 = range_of(s0, E, R), c2 = range_of(s1 - 1, E, R);
        span = make_int2(c1, c1 == c2 && !p.always ? -1 : c2 - c1 + 1);
      }
      ws_spans[s] = span;
    }
  }

  if (c < R && warp == consumers) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      sm100::tma_prefetch_desc(&tm_k);
      sm100::tma_prefetch_desc(&tm_v);
    }
    const uint32_t base = sm100::smem_u32(smem);
    const uint32_t box = (uint32_t)(HG * kChunk * 128);  // 128 bytes wide: all of an 8-bit tile, half of a 16-bit one
    const uint32_t sbox = (uint32_t)(HG * kChunk * 4);
    const uint32_t chunk_tx = k8 ? 2 * box + 2 * sbox : 4 * box;
    const uint32_t chunk_bytes = k8 ? 2 * box + 1024 : 4 * box;
    const unsigned lt_mask = (1u << lane) - 1u;
    int it = 0, st = 0;
    uint32_t ph = 1;  // parity of the empty barriers in this round
    bool ok = true, waited = p.overlap != 0;
    // the next ring entry, free to fill; false when the wait gave up
    auto acquire = [&]() -> bool {
      const bool got = !*(volatile int*)s_abort && sm100::mbar_wait(sm100::smem_u32(&empty_bar[st]), ph);
      return __all_sync(0xffffffffu, got);
    };
    auto advance = [&]() {
      ++it;
      if (++st == p.stages) {
        st = 0;
        ph ^= 1u;
      }
    };
    auto markers = [&](int kind, int seg, int piece) -> bool {  // one for each slot
      for (int i = 0; i < sub; ++i) {
        if (!acquire()) return false;
        if (lane == 0) {
          meta[st] = EntryMeta{kind, seg, 0, piece};
          sm100::mbar_arrive(sm100::smem_u32(&full_bar[st]));
        }
        advance();
      }
      return true;
    };
    // The open entry's chunks: page, first token, live tokens.  Its copies are
    // issued by a lane each: as one lane's instructions in turn they took about 350
    // cycles each and bounded small boxes (48 sequences of 4 kv heads: 61 us, so 55).
    int fill = 0, c_id[2] = {0, 0}, c_t0[2] = {0, 0}, c_live[2] = {0, 0};
    auto issue_entry = [&](int seg, int h0) -> bool {
      if (!acquire()) return false;
      if (!waited) {  // programmatic launch: the first copy waits for the previous kernel
        asm volatile("griddepcontrol.wait;" ::: "memory");
        waited = true;
      }
      const uint32_t fb = sm100::smem_u32(&full_bar[st]), dst = base + st * p.entry_bytes;
      if (lane == 0) {
        meta[st] = EntryMeta{0, seg, c_live[0], fill > 1 ? c_live[1] : 0};
        sm100::mbar_arrive_expect_tx(fb, fill * chunk_tx);
      }
      __syncwarp();
      const int odd = lane & 1;
      if constexpr (k8) {
        const int ch = lane >> 2;  // lanes of a chunk: K, V, and their scales
        if (ch < fill) {
          const uint32_t cd = dst + ch * chunk_bytes;
          const int id = ch ? c_id[1] : c_id[0], t0 = ch ? c_t0[1] : c_t0[0];
          if ((lane & 2) == 0) {
            sm100::tma_load_3d(cd + odd * box, odd ? &tm_v : &tm_k, fb, 0, id * bs + t0, h0);
          } else if (p.scale_maps) {
            sm100::tma_load_2d(cd + 2 * box + odd * 512, odd ? &tm_vs : &tm_ks, fb, t0, id * (int32_t)p.Hkv + h0);
          } else {
            const int64_t sat = ((int64_t)id * p.Hkv + h0) * kChunk;
            bulk_load(cd + 2 * box + odd * 512, (odd ? v_scale : k_scale) + sat, sbox, fb);
          }
        }
      } else {
        if (lane < 2)
          sm100::tma_load_3d(dst + odd * 2 * box, odd ? &tm_v : &tm_k, fb, 0, c_id[0] * bs + c_t0[0], 2 * h0);
      }
      fill = 0;
      advance();
      return true;
    };
    int s = seg0;
    int64_t e = lo;
    if (lo == hi) ok = markers(1, s, -1);  // (whole: a sequence without tokens)
    while (e < hi && ok) {
      while (s_cum[s + 1] == s_cum[s]) ++s;
      const int64_t b = s % B;
      const int hg = s / (int)B;
      const int64_t segs = s_cum[s], sege = s_cum[s + 1];
      const int j0 = (int)(e - segs), j1 = (int)((hi < sege ? hi : sege) - segs);
      const int ctx = s_ctx[b];
      const int64_t bt0 = b * p.max_blocks;
      int inval = e == lo ? *s_drop : 0;
      for (int jj = j0; jj < j1 && ok; jj += 32) {
        const int j = jj + lane;
        const bool in = j < j1;
        const int64_t id = in ? btab.at(bt0 + j) : -1;
        const bool valid = in && id >= 0 && id < p.num_blocks;
        const unsigned ib = __ballot_sync(0xffffffffu, in && !valid);
        const int rank = j - (inval + __popc(ib & lt_mask));
        int64_t left = (int64_t)ctx - (int64_t)rank * bs;
        const int nt = (int)(left < 0 ? 0 : (left > bs ? bs : left));
        const bool use = valid && nt > 0;
        const unsigned ub = __ballot_sync(0xffffffffu, use);
        if (use) {
          const int k = __popc(ub & lt_mask);
          chunk_id[k] = (int)id;
          chunk_ntok[k] = nt;
        }
        inval += __popc(ib);
        __syncwarp();
        const int n = __popc(ub);
        for (int u = 0; u < n && ok; ++u) {
          const int page = chunk_id[u], nt_page = chunk_ntok[u];
          for (int t0 = 0; t0 < nt_page && ok; t0 += kChunk) {
            const int live = nt_page - t0 < kChunk ? nt_page - t0 : kChunk;
            if (fill == 0) c_id[0] = page, c_t0[0] = t0, c_live[0] = live;
            else c_id[1] = page, c_t0[1] = t0, c_live[1] = live;
            ++fill;
            if (!k8 || fill == 2) ok = issue_entry(s, hg * HG);
          }
        }
        __syncwarp();
      }
      if (ok && fill > 0) ok = issue_entry(s, hg * HG);  // the segment ends in the first chunk of an entry
      if (ok) {
        const bool one = p.whole || range_of(segs, E, R) == range_of(sege - 1, E, R);
        ok = markers(1, s, one && !p.always ? -1 : s + c);
      }
      e = segs + j1;
      if (e == sege) ++s;
    }
    if (ok) ok = markers(2, 0, 0);
    if (lane == 0) {
      if (!ok) {
        b200_dev_error(kDevErrTimeoutEmpty);
        atomicExch(s_abort, 1);
      }
      // never leave with copies landing in shared memory
      for (int i = it - 1; i >= 0 && i >= it - p.stages; --i)
        if (!sm100::mbar_wait(sm100::smem_u32(&full_bar[i % p.stages]), (i / p.stages) & 1))
          b200_dev_error(kDevErrTimeoutFull);
    }
  } else if (c < R && warp < consumers) {
    // ------------------------------------------------------------ consumers
    const int w = warp % HG, slot = warp / HG;
    const uint32_t base = sm100::smem_u32(smem), meta_at = sm100::smem_u32(meta);
    const uint32_t xch_at = sm100::smem_u32(xch) + (uint32_t)(w * kXchPitch + lane) * 4;
    const uint32_t box = (uint32_t)(HG * kChunk * 128);
    const Lane8 lane8(w, box, lane);
    uint32_t qb[8][2], qf[q_words<KV>()];
    float o[8][4];
    float mu[2] = {kNoMax, kNoMax}, lp[2] = {0.f, 0.f};
    float slA = p.qscale, slB = p.qscale;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    bool last_byte = false;
    int cur = -1;
    uint32_t xph = 0;
    int st = slot % p.stages;
    uint32_t ph = (slot / p.stages) & 1;
    for (;;) {
      if (!sm100::mbar_wait_warp(sm100::smem_u32(&full_bar[st]), ph)) {
        if (lane == 0) {
          b200_dev_error(kDevErrTimeoutFull);
          atomicExch(s_abort, 1);
        }
        break;
      }
      const uint4 mw = lds128(meta_at + st * (int)sizeof(EntryMeta));
      const EntryMeta m{(int)mw.x, (int)mw.y, (int)mw.z, (int)mw.w};
      if (m.kind == 0) {
        if (m.seg != cur) {
          cur = m.seg;
          const int64_t b = m.seg % B, kvh = (int64_t)(m.seg / B) * HG + w;
          const T* qrow = q + (b * p.Hq + kvh * G) * kD;
          if constexpr (k8) last_byte = load_q_frags8<T, KV, G>(qrow, lane, p.qscale, qf, slA, slB);
          else load_q_frags<T, G>(qrow, lane, qb);
        }
        const uint32_t pg = base + st * p.entry_bytes;
        if constexpr (k8) {
          const int nt[2] = {m.ntok, m.piece};
          mma_pair8<KV>(pg, lane8, nt, lane, slA, slB, qf, last_byte, o, mu, lp);
        } else {
          mma_chunk16<T>(pg + w * kChunk * 256, pg + 2 * box + w * kChunk * 256, m.ntok, lane, p.qscale, qb, o, mu, lp);
        }
      } else if (m.kind == 1) {
        bool write = true;
        if (sub > 1) {
          // the head's other warps hand over their state; slot 0 adds it up
          const uint32_t x = xch_at + (uint32_t)((slot - 1) * HG * kXchPitch) * 4;
          if (slot > 0) {
            write = false;
            if (!sm100::mbar_wait_warp(sm100::smem_u32(&xch_empty[w]), xph ^ 1u)) {
              if (lane == 0) {
                b200_dev_error(kDevErrTimeoutCombine);
                atomicExch(s_abort, 1);
              }
              break;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
              for (int k = 0; k < 4; ++k) sts_f32(x + (4 * i + k) * 128, o[i][k]);
            sts_f32(x + 32 * 128, mu[0]);
            sts_f32(x + 33 * 128, mu[1]);
            sts_f32(x + 34 * 128, lp[0]);
            sts_f32(x + 35 * 128, lp[1]);
            __syncwarp();
            if (lane == 0) sm100::mbar_arrive(sm100::smem_u32(&xch_full[w]));
          } else {
            if (!sm100::mbar_wait_warp(sm100::smem_u32(&xch_full[w]), xph)) {
              if (lane == 0) {
                b200_dev_error(kDevErrTimeoutCombine);
                atomicExch(s_abort, 1);
              }
              break;
            }
            for (int v = 1; v < sub; ++v) {
              const uint32_t y = xch_at + (uint32_t)((v - 1) * HG * kXchPitch) * 4;
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                // (no tokens: m = kNoMax with l and o zero)
                const float mo = lds_f32(y + (32 + k) * 128), lo2 = lds_f32(y + (34 + k) * 128);
                const float mn = fmaxf(mu[k], mo);
                const float fa = ex2(mu[k] - mn), fb = ex2(mo - mn);
                mu[k] = mn;
                lp[k] = lp[k] * fa + lo2 * fb;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  o[i][k] = o[i][k] * fa + lds_f32(y + (4 * i + k) * 128) * fb;
                  o[i][k + 2] = o[i][k + 2] * fa + lds_f32(y + (4 * i + k + 2) * 128) * fb;
                }
              }
            }
            __syncwarp();
            if (lane == 0) sm100::mbar_arrive(sm100::smem_u32(&xch_empty[w]));
          }
          xph ^= 1u;
        }
        if (write) {
          const float lA = head_sum(lp[0]), lB = head_sum(lp[1]);
          const int64_t b = m.seg % B, hg = m.seg / B;
          if (m.piece < 0) {
            T* orow = out + (b * p.Hq + hg * heads_cta + w * G) * kD;
            store_rows_nan<T, G>(orow, o, lA, lB, lane);
          } else {
            float* row0 = ws_rows + ((int64_t)m.piece * heads_cta + w * G) * kPiecePitch;
            store_partial<G>(row0, kPiecePitch, row0 + kD, kPiecePitch, o, mu, lA, lB, lane);
          }
        }
        mu[0] = mu[1] = kNoMax;
        lp[0] = lp[1] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        cur = -1;
      }
      __syncwarp();
      if (lane == 0) sm100::mbar_arrive(sm100::smem_u32(&empty_bar[st]));
      if (m.kind == 2) break;
      st += sub;
      while (st >= p.stages) {
        st -= p.stages;
        ph ^= 1u;
      }
    }
  }
  // this grid counts as done only when the previous one is (the other CTAs
  // may leave their SMs)
  if (blockIdx.x == 0 && threadIdx.x == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
}

// ---------------------------------------------------------------------------
// Host: tensor maps and launch of one slice of the batch (a.B <= kMaxSeg / n_hg).
// ---------------------------------------------------------------------------
template <typename T, typename KV, int G>
int launch_pieces(const AttnCall& a, const PieceGeom& g, const PieceSpace& w, bool overlap, cudaStream_t stream) {
  CUtensorMap tk, tv, tks{}, tvs{};
  constexpr bool k8 = sizeof(KV) == 1;
  constexpr uint64_t el = sizeof(KV);
  const CUtensorMapDataType dt = k8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                    : (std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                      : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16);
  // dims (128 bytes of dims, token slot, head or half of its dims): a box of 16
  // tokens x HG heads lands as [head][half][token] rows of 128 bytes, swizzled in 8-row atoms
  const uint64_t dims[3] = {128 / el, (uint64_t)(a.num_blocks * a.block_size), (uint64_t)a.Hkv * el};
  const uint64_t strides[2] = {(uint64_t)a.Hkv * kD * el, 128};
  const uint32_t box[3] = {(uint32_t)(128 / el), (uint32_t)kChunk, (uint32_t)(g.HG * el)};
  int st = encode_tensor_map(&tk, dt, 3, a.k_cache, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  if (st) return st;
  st = encode_tensor_map(&tv, dt, 3, a.v_cache, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  if (st) return st;
  const bool scale_maps = k8 && a.block_size != kChunk;
  if (scale_maps) {
    // scales [num_blocks * Hkv rows][block_size]: a box of 16 tokens x HG heads
    const uint64_t sdims[2] = {(uint64_t)a.block_size, (uint64_t)(a.num_blocks * a.Hkv)};
    const uint64_t sstride[1] = {(uint64_t)a.block_size * 4};
    const uint32_t sbox[2] = {(uint32_t)kChunk, (uint32_t)g.HG};
    st = encode_tensor_map(&tks, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, a.k_scale, sdims, sstride, sbox,
                           CU_TENSOR_MAP_SWIZZLE_NONE);
    if (st) return st;
    st = encode_tensor_map(&tvs, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, a.v_scale, sdims, sstride, sbox,
                           CU_TENSOR_MAP_SWIZZLE_NONE);
    if (st) return st;
  }
  PiecesParams p{};
  p.scale_maps = scale_maps;
  p.B = a.B, p.Hq = a.Hq, p.Hkv = a.Hkv, p.num_blocks = a.num_blocks, p.max_blocks = a.max_blocks;
  p.bs = (int)a.block_size, p.HG = g.HG, p.n_hg = g.n_hg, p.sub = g.sub, p.stages = g.stages;
  p.nseg = (int)(g.n_hg * a.B);
  p.always = a.prefix_table != nullptr;
  p.whole = g.whole;
  p.overlap = overlap;
  p.entry_bytes = g.entry_bytes;
  p.qscale = a.scale * 1.4426950408889634f;
  auto kern = paged_attn_pieces_kernel<T, KV, G>;
  static SmemGrant grant;
  cudaError_t e = grant(kern, g.smem);
  if (e != cudaSuccess) return launch_status(e);
  cudaLaunchConfig_t lc = {};
  lc.gridDim = dim3((unsigned)(g.whole ? p.nseg : g.grid));
  lc.blockDim = dim3((unsigned)((g.HG * g.sub + 1) * 32));
  lc.dynamicSmemBytes = g.smem;
  lc.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  lc.attrs = attr;
  lc.numAttrs = (overlap || g.pdl) ? 1 : 0;
  const int wide = a.index_dtype == B200_I64;
  e = cudaLaunchKernelEx(&lc, kern, tk, tv, tks, tvs, a.k_scale, a.v_scale, static_cast<const T*>(a.q),
                         IndexPtr{a.block_table, wide}, IndexPtr{a.context_len, wide}, static_cast<T*>(a.out), w.rows,
                         w.spans, p);
  return launch_status(e);
}

template <typename T, typename KV>
int launch_pieces_by_group(const AttnCall& a, const PieceGeom& g, const PieceSpace& w, bool overlap, cudaStream_t s) {
  switch (g.G) {
    case 1: return launch_pieces<T, KV, 1>(a, g, w, overlap, s);
    case 2: return launch_pieces<T, KV, 2>(a, g, w, overlap, s);
    case 4: return launch_pieces<T, KV, 4>(a, g, w, overlap, s);
    default: return launch_pieces<T, KV, 8>(a, g, w, overlap, s);
  }
}

template <typename T, typename KV>
int launch_generic(const AttnCall& a, cudaStream_t s) {
  const int wide = a.index_dtype == B200_I64;
  for (int64_t b0 = 0; b0 < a.B; b0 += 65535) {
    const int64_t n = a.B - b0 < 65535 ? a.B - b0 : 65535;
    const size_t isz = wide ? 8 : 4;
    auto at = [&](const void* p, int64_t i) {
      return static_cast<const void*>(static_cast<const char*>(p) + (size_t)i * isz);
    };
    paged_attn_pieces_generic_kernel<T, KV><<<dim3((unsigned)a.Hq, (unsigned)n), 128, 0, s>>>(
        static_cast<const T*>(a.q) + b0 * a.Hq * a.D, static_cast<const KV*>(a.k_cache),
        static_cast<const KV*>(a.v_cache), a.k_scale, a.v_scale, IndexPtr{a.prefix_table, wide},
        IndexPtr{a.prefix_len, wide}, IndexPtr{at(a.block_table, b0 * a.max_blocks), wide},
        IndexPtr{at(a.context_len, b0), wide}, static_cast<T*>(a.out) + b0 * a.Hq * a.D, a.Hq, a.Hkv, a.D,
        a.num_blocks, a.block_size, a.max_blocks, a.max_prefix_blocks, a.scale * 1.4426950408889634f);
    if (cudaError_t e = cudaGetLastError(); e != cudaSuccess) return launch_status(e);
  }
  return B200_OK;
}

}  // namespace
}  // namespace b200

#define B200_DEFINE_PIECE_LAUNCHERS(NAME, KVT)                                                                  \
  namespace b200 {                                                                                              \
  int launch_pieces_##NAME(const AttnCall& a, const PieceGeom& g, const PieceSpace& w, bool overlap,            \
                           cudaStream_t s) {                                                                    \
    return B200_DISPATCH_HALF(a.dtype, [&] { return launch_pieces_by_group<scalar_t, KVT>(a, g, w, overlap, s); }); \
  }                                                                                                             \
  int launch_attn_generic_##NAME(const AttnCall& a, cudaStream_t s) {                                           \
    return B200_DISPATCH_HALF(a.dtype, [&] { return launch_generic<scalar_t, KVT>(a, s); });                    \
  }                                                                                                             \
  }
