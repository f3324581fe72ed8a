// Device helpers of the paged decode kernels: the transposed m16n8k16 tiles
// (tokens or head dims on the M side, query heads on the N side), their
// online softmax and the stores of rows and partial rows.
#pragma once

#include <math.h>

#include "common.cuh"
#include "sm100.cuh"

namespace b200 {
namespace {

constexpr int kD = 128;  // head dim of the TMA path

__device__ __forceinline__ void named_bar_sync(int id, int n) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory");
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr));
  return v;
}

template <typename T>
__device__ __forceinline__ void widen8(const uint4& raw, float* f) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
    unpack16<T>(raw, f);
  }
}

template <typename IDX>
__device__ __forceinline__ bool bad_block(IDX id, int64_t nb) {
  return id < 0 || (int64_t)id >= nb;
}

// ---------------------------------------------------------------------------
// Tensor-core consumer (block size a multiple of 16), transposed form.  Warp
// w owns kv head h0 + w and its G query heads.  Tokens are the M dimension of
// the m16n8k16 tiles and query heads the N dimension (8 columns, heads >= G
// are zero), so a 16-token chunk of a page costs 8 + 8 mma.sync:
//   S^T[16 tok x 8 heads] = K[16 x 128] Q^T  -- 8 k-steps, K as the A operand
//                                              by ldmatrix (rows = tokens), two
//                                              independent accumulator chains
//   online softmax on the C fragments: a thread holds tokens lane/4 and
//   lane/4 + 8 of heads 2(lane%4) and 2(lane%4)+1; a head's max over the 16
//   tokens needs 3 xor-shuffles
//   O^T[128 x 8 heads] += V^T[128 x 16 tok] P^T  -- 8 m-tiles of 16 dims, V as
//                                              the A operand by ldmatrix.trans;
//                                              P^T's B fragments are the packed
//                                              S^T fragments transposed in
//                                              registers by movmatrix
// The accumulator is 8 tiles x 4 floats per thread, and the V fragments are
// loaded before the softmax so their latency overlaps it.  Shared-memory
// tiles are SWIZZLE_128B with rows = (head, token), so the 8 rows of every
// ldmatrix matrix hit 8 distinct 16-byte bank groups.  Each head's running
// max is raised only when it grows by more than 2^8 (exact: O and l share the
// offset).
// ---------------------------------------------------------------------------
__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr));
}
// 8x8 b16 matrix transpose across the warp (fragment layout: row lane/4,
// columns 2(lane%4) and 2(lane%4)+1 in one register).
__device__ __forceinline__ uint32_t movm_t(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <typename T>
__device__ __forceinline__ void mma16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}

template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  } else {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
}

// Zeroes the 16-bit halves of a fragment register whose token is >= ntok.
__device__ __forceinline__ uint32_t mask_pair(uint32_t v, int tok, int ntok) {
  const uint32_t lo = tok < ntok ? 0x0000ffffu : 0u;
  const uint32_t hi = tok + 1 < ntok ? 0xffff0000u : 0u;
  return v & (lo | hi);
}

// Q^T B fragments of this warp's query heads: head lane/4 (zero if >= G),
// dims 16ks + 2(lane%4) + {0,1} and +8.
template <typename T, int G>
__device__ __forceinline__ void load_q_frags(const T* __restrict__ qrow0, int lane, uint32_t (&qb)[8][2]) {
  const int qh = lane >> 2, qc = (lane & 3) * 2;
  const T* qr = qrow0 + (qh < G ? qh : 0) * kD;
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) {
    qb[ks][0] = qh < G ? *reinterpret_cast<const uint32_t*>(qr + 16 * ks + qc) : 0u;
    qb[ks][1] = qh < G ? *reinterpret_cast<const uint32_t*>(qr + 16 * ks + 8 + qc) : 0u;
  }
}

// Raises head c's running max to mx when it grew by more than 2^8; o entries
// of that head are columns c and c + 2 of every tile.
__device__ __forceinline__ void raise_max(float& mu, float mx, float& lp, float (&o)[8][4], int c) {
  if (mu == -INFINITY) {
    mu = mx;
  } else if (mx > mu + 8.0f) {
    const float alpha = exp2f(mu - mx);
    mu = mx;
    lp *= alpha;
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) {
      o[mt][c] *= alpha;
      o[mt][c + 2] *= alpha;
    }
  }
}

// One page (ntok tokens of one kv head, K tile at kb, V tile at vb in the
// swizzled [d-half][head][token][64] layout) folded into this warp's running
// (o, mu, lp): mu/lp[0] for head 2(lane%4), [1] for head 2(lane%4)+1.
template <typename T>
__device__ __forceinline__ void mma_page(uint32_t kb, uint32_t vb, int ntok, int w, int bs, int lane,
                                         uint32_t hbytes, float sl2, const uint32_t (&qb)[8][2],
                                         float (&o)[8][4], float (&mu)[2], float (&lp)[2]) {
  const int mat = lane >> 3, mrow = lane & 7;
  const int tr = lane >> 2, tq = (lane & 3) * 2;
  for (int t0 = 0; t0 < ntok; t0 += 16) {
    float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
    {
      // A = K rows: matrix `mat` = (token half mat&1, dim-chunk parity mat>>1)
      const int row = w * bs + t0 + (mat & 1) * 8 + mrow;
      const uint32_t rbase = kb + row * 128;
      const int sw = row & 7;
      uint32_t ka[8][4];
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) {
        const int chunk = ((ks & 3) << 1) | (mat >> 1);
        ldsm_x4(rbase + (ks >> 2) * hbytes + ((chunk ^ sw) << 4), ka[ks][0], ka[ks][1], ka[ks][2], ka[ks][3]);
      }
#pragma unroll
      for (int ks = 0; ks < 8; ++ks)
        mma16816<T>((ks & 1) ? s1 : s0, ka[ks][0], ka[ks][1], ka[ks][2], ka[ks][3], qb[ks][0], qb[ks][1]);
    }
    // A = V^T by ldmatrix.trans: matrix `mat` = (token half mat>>1, dim-chunk parity mat&1)
    uint32_t va[8][4];
    {
      const int row = w * bs + t0 + (mat >> 1) * 8 + mrow;
      const uint32_t rbase = vb + row * 128;
      const int sw = row & 7;
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) {
        const int chunk = ((mt & 3) << 1) | (mat & 1);
        ldsm_x4_t(rbase + (mt >> 2) * hbytes + ((chunk ^ sw) << 4), va[mt][0], va[mt][1], va[mt][2], va[mt][3]);
      }
    }
    // x[0]/x[1]: token tr of heads 2(lane%4), +1; x[2]/x[3]: token tr + 8
    const bool ok0 = t0 + tr < ntok, ok1 = t0 + tr + 8 < ntok;
    float x[4];
    x[0] = ok0 ? (s0[0] + s1[0]) * sl2 : -INFINITY;
    x[1] = ok0 ? (s0[1] + s1[1]) * sl2 : -INFINITY;
    x[2] = ok1 ? (s0[2] + s1[2]) * sl2 : -INFINITY;
    x[3] = ok1 ? (s0[3] + s1[3]) * sl2 : -INFINITY;
    float mA = fmaxf(x[0], x[2]), mB = fmaxf(x[1], x[3]);
#pragma unroll
    for (int off = 4; off <= 16; off <<= 1) {
      mA = fmaxf(mA, __shfl_xor_sync(0xffffffffu, mA, off));
      mB = fmaxf(mB, __shfl_xor_sync(0xffffffffu, mB, off));
    }
    raise_max(mu[0], mA, lp[0], o, 0);
    raise_max(mu[1], mB, lp[1], o, 1);
    const float p0 = exp2f(x[0] - mu[0]), p2 = exp2f(x[2] - mu[0]);
    const float p1 = exp2f(x[1] - mu[1]), p3 = exp2f(x[3] - mu[1]);
    lp[0] += p0 + p2;
    lp[1] += p1 + p3;
    // P^T B fragments: tokens tq + {0,1} (b0) and 8 + tq + {0,1} (b1) of head lane/4
    const uint32_t b0 = movm_t(pack_pair<T>(p0, p1));
    const uint32_t b1 = movm_t(pack_pair<T>(p2, p3));
    if (t0 + 16 > ntok) {
      // tokens past the end may hold anything (NaN included): zero their V
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) {
        va[mt][0] = mask_pair(va[mt][0], t0 + tq, ntok);
        va[mt][1] = mask_pair(va[mt][1], t0 + tq, ntok);
        va[mt][2] = mask_pair(va[mt][2], t0 + 8 + tq, ntok);
        va[mt][3] = mask_pair(va[mt][3], t0 + 8 + tq, ntok);
      }
    }
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) mma16816<T>(o[mt], va[mt][0], va[mt][1], va[mt][2], va[mt][3], b0, b1);
  }
}

// Sum of a head's l over the 8 lanes that share it.
__device__ __forceinline__ float head_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 4);
  v += __shfl_xor_sync(0xffffffffu, v, 8);
  v += __shfl_xor_sync(0xffffffffu, v, 16);
  return v;
}

// Normalised output rows of this warp's heads: orow0 = row of head 0; the
// O^T fragments are transposed back by movmatrix into 4-byte stores of two
// dims of head lane/4.
template <typename T, int G>
__device__ __forceinline__ void store_rows(T* __restrict__ orow0, const float (&o)[8][4], float lA, float lB,
                                           int lane) {
  const float iA = lA > 0.f ? 1.f / lA : 0.f, iB = lB > 0.f ? 1.f / lB : 0.f;
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

// Unnormalised fp32 partial of this warp's heads: row(h) = base + h * pitch
// floats holds o[0..127]; (m, l) go to mpos(h), mpos(h) + 1 via ml_base +
// h * ml_pitch.
template <int G>
__device__ __forceinline__ void store_partial(float* __restrict__ base, int64_t pitch, float* __restrict__ ml_base,
                                              int64_t ml_pitch, const float (&o)[8][4], const float (&mu)[2],
                                              float lA, float lB, int lane) {
  const int hA = (lane & 3) * 2, hB = hA + 1, d = lane >> 2;
#pragma unroll
  for (int mt = 0; mt < 8; ++mt) {
    if (hA < G) {
      base[hA * pitch + 16 * mt + d] = o[mt][0];
      base[hA * pitch + 16 * mt + 8 + d] = o[mt][2];
    }
    if (hB < G) {
      base[hB * pitch + 16 * mt + d] = o[mt][1];
      base[hB * pitch + 16 * mt + 8 + d] = o[mt][3];
    }
  }
  if (d == 0) {
    if (hA < G) {
      ml_base[hA * ml_pitch] = mu[0];
      ml_base[hA * ml_pitch + 1] = lA;
    }
    if (hB < G) {
      ml_base[hB * ml_pitch] = mu[1];
      ml_base[hB * ml_pitch + 1] = lB;
    }
  }
}

}  // namespace
}  // namespace b200
