// The shared prefix of a batch: all query rows of a kv head against the
// prefix's keys, on the fifth-generation tensor cores.
//
// For kv head h the batch's query rows r = b * G + g form one matrix Q_h
// [B G, 128].  A CTA takes two 128-row tiles of it (one when there are no more) and one
// stretch of the prefix's block table, and leaves one piece (m, l, o) a row --
// the pieces the streaming kernel leaves for the own tokens, joined with them:
//   S = Q K^T    tcgen05.mma 128 x 128 x 16 (Q, K K-major in shared memory), fp32 in tensor memory
//   softmax      one thread a row: the row's 128 logits read twice from tensor memory (maximum,
//                then weights), so that a thread needs few registers; O rescaled only when the
//                maximum grew by more than 2^8
//   O += P V     P (16-bit) over S's columns in tensor memory, V MN-major
// With one row tile the two softmax warpgroups take its even and its odd key
// tiles, each with an O of its own, joined in shared memory at the end: the
// chain S -> softmax -> P V of one tile then runs beside the other's as with two row tiles.
//
// Reading the prefix costs its bytes once a CTA column instead of once a
// sequence: at 64 sequences of an 8192-token prefix 33.5 MB instead of 2.1 GB.
//
// Roles: warp 0 walks the block table and copies pages (TMA boxes of bs
// tokens; a tile is as many pages as fit 128 tokens), warp 1 issues the MMAs,
// warps 4-11 are the two tiles' softmax warpgroups.  16-bit caches: pages land
// in the K/V ring as the MMA reads them; warp 2 zeroes V rows behind the last
// token (a weight of 0 times a NaN left in the cache is NaN).  8-bit caches:
// pages land in a ring of code tiles, and warps 12-15 widen them to f16 tiles
// (codes are exact in f16; the scales go beside them in fp32 and meet
// the logits and weights as in the streaming kernel).
#pragma once

#include "kv_attn.cuh"

namespace b200 {

int launch_prefix_i8(const AttnCall& a, const PieceGeom& g, const PieceSpace& w, cudaStream_t s);
int launch_prefix_e4m3(const AttnCall& a, const PieceGeom& g, const PieceSpace& w, cudaStream_t s);
int launch_prefix_16(const AttnCall& a, const PieceGeom& g, const PieceSpace& w, cudaStream_t s);

namespace {

constexpr int kPM = 128;                   // rows of a query tile, keys of a key tile
constexpr uint32_t kPHalf = kPM * 128;     // 64 dims (16-bit) of 128 rows
constexpr uint32_t kPTile = 2 * kPHalf;    // a Q, K or V tile
constexpr uint32_t kPCodes = kPHalf;       // an 8-bit K or V tile
constexpr int kPRing16 = 5, kPRing8 = 3;   // K/V tiles in shared memory
constexpr int kPMaxCodes = 6;              // code tiles, at most
constexpr int kPMaxPages = 8;              // pages of a tile (block size 16)

struct PrefixParams {
  int64_t B, Hq, Hkv, num_blocks, max_prefix;
  int G, bs, ppt;  // pages a key tile
  int codes;       // ring depth of the code tiles (8-bit)
  int splits;
  float qscale;  // scale * log2(e)
};

template <bool k8>
struct PrefixSmem {
  static constexpr uint32_t oQ = 0;  // two Q tiles
  static constexpr uint32_t oRing = 2 * kPTile;
  static constexpr uint32_t oCodes = oRing + (k8 ? kPRing8 : kPRing16) * kPTile;
};

// One row of Q into the swizzled tile: 16-byte chunk c of row r sits at chunk
// c ^ (r & 7) of its 128-byte row, dims 64.. in the second half.  8-bit caches: f16, the
// row scaled to [2^13, 2^14) by a power of two; returns its logit factor.
template <typename T, bool k8>
__device__ __forceinline__ float stage_q_row(const T* __restrict__ src, bool live, uint8_t* tile, int r, float qscale) {
  uint4 raw[16];
#pragma unroll
  for (int c = 0; c < 16; ++c)
    raw[c] = live ? __ldg(reinterpret_cast<const uint4*>(src) + c) : make_uint4(0, 0, 0, 0);
  float factor = qscale;
  if constexpr (k8) {
    float amax = 0.f;
#pragma unroll
    for (int c = 0; c < 16; ++c) {
      float f[8];
      unpack16<T>(raw[c], f);
#pragma unroll
      for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(f[i]));
    }
    float up, down;
    pow2_scale(amax, up, down);
    factor *= down;
#pragma unroll
    for (int c = 0; c < 16; ++c) {
      float f[8];
      unpack16<T>(raw[c], f);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] *= up;
      raw[c] = pack16<__half>(f);
    }
  }
#pragma unroll
  for (int c = 0; c < 16; ++c)
    *reinterpret_cast<uint4*>(tile + (c >> 3) * kPHalf + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = raw[c];
  return factor;
}

template <typename T, typename KV>
__global__ void __launch_bounds__(sizeof(KV) == 1 ? 512 : 384, 1)
    prefix_attn_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                       const float* __restrict__ k_scale, const float* __restrict__ v_scale, const T* __restrict__ q,
                       IndexPtr ptab, IndexPtr plen, float* __restrict__ pieces, PrefixParams p) {
  constexpr bool k8 = sizeof(KV) == 1;
  using M = typename std::conditional<k8, __half, T>::type;  // type of the matrix operands
  using L = PrefixSmem<k8>;
  constexpr int kRing = k8 ? kPRing8 : kPRing16;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = sm100::smem_u32(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = blockIdx.x, h = blockIdx.z;
  const int64_t R = p.B * p.G, row0 = (int64_t)blockIdx.y * 2 * kPM;
  const int tiles = R - row0 > kPM ? 2 : 1;
  const int both = tiles == 2;  // else: streams 0 and 1 are the even and odd key tiles of one row tile
  const int bs = p.bs, tile_tok = p.ppt * bs;

  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::oCodes + (k8 ? p.codes * kPCodes : 0));
  uint64_t* q_full = bars;
  uint64_t* ring_full = bars + 1;               // [kRing]
  uint64_t* ring_empty = ring_full + kPRing16;  // [kRing]
  uint64_t* s_full = ring_empty + kPRing16;     // [2]
  uint64_t* p_full = s_full + 2;                // [2]
  uint64_t* o_done = p_full + 2;                // [2]
  uint64_t* v_fixed = o_done + 2;
  uint64_t* sc_full = v_fixed + 1;              // [2]
  uint64_t* sc_empty = sc_full + 2;             // [2]
  uint64_t* code_full = sc_empty + 2;           // [kPMaxCodes]
  uint64_t* code_empty = code_full + kPMaxCodes;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(code_empty + kPMaxCodes);
  int* s_misc = reinterpret_cast<int*>(tmem_slot + 1);  // [0] abort, [1] valid entries before the split, [2] in it
  int* s_ids = s_misc + 3;                              // [kPMaxCodes][kPMaxPages] page ids of a code tile
  float* s_sc = reinterpret_cast<float*>(s_ids + kPMaxCodes * kPMaxPages);  // [2][3][kPM]: ks, log2 vs, 1 / vs

  // the own-token kernel may run beside this one
  asm volatile("griddepcontrol.launch_dependents;");

  // ---- this split's entries [e0, e1), its first page's rank and its tokens
  int e0 = 0, e1 = 0;
  int64_t plen_tokens = plen.at(0);
  {
    const int64_t most = p.max_prefix * bs;
    plen_tokens = plen_tokens < 0 ? 0 : (plen_tokens < most ? plen_tokens : most);
    const int E = (int)((plen_tokens + bs - 1) / bs);
    int per = (E + p.splits - 1) / p.splits;
    per = (per + p.ppt - 1) / p.ppt * p.ppt;  // whole tiles
    const int64_t a = (int64_t)split * per, b = a + per;
    e0 = (int)(a < E ? a : E);
    e1 = (int)(b < E ? b : E);
    if (threadIdx.x < 3) s_misc[threadIdx.x] = 0;
    __syncthreads();
    // valid entries before the split and in it, counted by the whole CTA
    int before = 0, in = 0;
    for (int j = threadIdx.x; j < e1; j += blockDim.x) {
      const int64_t id = ptab.at(j);
      const int ok = id >= 0 && id < p.num_blocks;
      if (j < e0) before += ok;
      else in += ok;
    }
    before = __reduce_add_sync(0xffffffffu, before);
    in = __reduce_add_sync(0xffffffffu, in);
    if (lane == 0) {
      atomicAdd(&s_misc[1], before);
      atomicAdd(&s_misc[2], in);
    }
  }
  if (threadIdx.x == 32) {
    sm100::mbar_init(sm100::smem_u32(q_full), 4 * tiles);
    for (int i = 0; i < kRing; ++i) {
      sm100::mbar_init(sm100::smem_u32(&ring_full[i]), k8 ? 4 : 1);
      sm100::mbar_init(sm100::smem_u32(&ring_empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      sm100::mbar_init(sm100::smem_u32(&s_full[i]), 1);
      sm100::mbar_init(sm100::smem_u32(&p_full[i]), 4);
      sm100::mbar_init(sm100::smem_u32(&o_done[i]), 1);
      sm100::mbar_init(sm100::smem_u32(&sc_full[i]), 4);
      sm100::mbar_init(sm100::smem_u32(&sc_empty[i]), 4 * tiles);  // one stream's warps, or both's
    }
    sm100::mbar_init(sm100::smem_u32(v_fixed), 1);
    for (int i = 0; i < kPMaxCodes; ++i) {
      sm100::mbar_init(sm100::smem_u32(&code_full[i]), 1);
      sm100::mbar_init(sm100::smem_u32(&code_empty[i]), 4);
    }
    sm100::fence_barrier_init();
  }
  if (!k8 && tile_tok < kPM) {
    // rows no page reaches stay zero in every ring tile (both operands)
    for (int i = threadIdx.x; i < kRing * 2 * (kPM - tile_tok) * 8; i += blockDim.x) {
      const int c = i & 7, r = (i >> 3) % (kPM - tile_tok), half = (i >> 3) / (kPM - tile_tok);
      *reinterpret_cast<uint4*>(smem + L::oRing + half * kPHalf + (tile_tok + r) * 128 + c * 16) = make_uint4(0, 0, 0, 0);
    }
    sm100::fence_proxy_async_smem();
  }
  if (warp == 1) {
    sm100::tmem_alloc(sm100::smem_u32(tmem_slot), 512);
    sm100::tmem_relinquish();
  }
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  const uint32_t tmem = *tmem_slot;  // columns: S_t at 128 t, O_t at 256 + 128 t
  int* s_abort = &s_misc[0];
  int ntok;
  {
    const int64_t left = plen_tokens - (int64_t)s_misc[1] * bs, have = (int64_t)s_misc[2] * bs;
    ntok = (int)(left < 0 ? 0 : (left < have ? left : have));
  }
  const int nkt = (ntok + tile_tok - 1) / tile_tok;
  const int last_valid = ntok - (nkt - 1) * tile_tok;  // tokens of the last tile
  const bool fix_v = !k8 && nkt > 0 && last_valid < tile_tok;

  if (warp == 0) {
    // -------------------------------------------------------------- producer
    if (lane == 0) {
      sm100::tma_prefetch_desc(&tm_k);
      sm100::tma_prefetch_desc(&tm_v);
    }
    int left = (ntok + bs - 1) / bs;  // pages still to copy
    int issued = 0, np = 0;           // (lane 0) copies of tiles issued, pages of the open tile
    int ids[kPMaxPages];
    bool ok = true;
    auto copy_tile = [&](int which) -> bool {
      const int depth = k8 ? p.codes : kRing;
      const int slot = issued % depth;
      uint64_t* empty = k8 ? code_empty : ring_empty;
      if (*(volatile int*)s_abort) return false;
      if (!sm100::mbar_wait(sm100::smem_u32(&empty[slot]), ((issued / depth) & 1) ^ 1)) return false;
      const uint32_t fb = sm100::smem_u32(&(k8 ? code_full : ring_full)[slot]);
      const CUtensorMap* map = which ? &tm_v : &tm_k;
      if constexpr (k8) {
#pragma unroll
        for (int i = 0; i < kPMaxPages; ++i)
          if (i < np) s_ids[slot * kPMaxPages + i] = ids[i];
      }
      sm100::mbar_arrive_expect_tx(fb, (uint32_t)(np * bs * (k8 ? 128 : 256)));
      const uint32_t dst = sbase + (k8 ? L::oCodes + slot * kPCodes : L::oRing + slot * kPTile);
#pragma unroll
      for (int i = 0; i < kPMaxPages; ++i) {
        if (i < np) {
          sm100::tma_load_3d(dst + i * bs * 128, map, fb, 0, ids[i] * bs, h);
          if constexpr (!k8) sm100::tma_load_3d(dst + kPHalf + i * bs * 128, map, fb, 64, ids[i] * bs, h);
        }
      }
      ++issued;
      return true;
    };
    for (int j0 = e0; j0 < e1 && left > 0 && ok; j0 += 32) {
      const int64_t id = j0 + lane < e1 ? ptab.at(j0 + lane) : -1;
      unsigned use = __ballot_sync(0xffffffffu, id >= 0 && id < p.num_blocks);
      while (use != 0 && left > 0 && ok) {
        const int src = __ffs(use) - 1;
        use &= use - 1;
        const int page = (int)__shfl_sync(0xffffffffu, (int)id, src);
        --left;
#pragma unroll
        for (int i = 0; i < kPMaxPages; ++i)
          if (i == np) ids[i] = page;
        ++np;
        if (np == p.ppt || left == 0) {
          if (lane == 0) ok = copy_tile(0) && copy_tile(1);
          ok = __shfl_sync(0xffffffffu, ok, 0);
          np = 0;
        }
      }
    }
    if (lane == 0) {
      if (!ok) {
        b200_dev_error(kDevErrTimeoutEmpty);
        atomicExch(s_abort, 1);
      }
      // no copy may still be writing shared memory when the CTA exits
      const int depth = k8 ? p.codes : kRing;
      for (int i = issued - 1; i >= 0 && i >= issued - depth; --i)
        if (!sm100::mbar_wait(sm100::smem_u32(&(k8 ? code_full : ring_full)[i % depth]), (i / depth) & 1))
          b200_dev_error(kDevErrTimeoutFull);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------- MMA issue
    constexpr uint32_t fmt = std::is_same<M, __nv_bfloat16>::value ? 1u : 0u;
    constexpr uint32_t idesc_s = sm100::make_idesc(1, fmt, fmt, 0, 0, kPM, kPM);
    constexpr uint32_t idesc_o = sm100::make_idesc(1, fmt, fmt, 0, 1, kPM, kPieceDim);
    const uint32_t leader = sm100::elect_one();
    const uint64_t dq = sm100::make_smem_desc(sbase + L::oQ, 16, 1024, sm100::kSwizzle128B);
    const uint64_t dk = sm100::make_smem_desc(sbase + L::oRing, 16, 1024, sm100::kSwizzle128B);
    const uint64_t dv = sm100::make_smem_desc(sbase + L::oRing, kPHalf, 1024, sm100::kSwizzle128B);
    bool ok = nkt > 0 && sm100::mbar_wait_warp(sm100::smem_u32(q_full), 0);
    auto full = [&](int it) -> bool {
      return sm100::mbar_wait_warp(sm100::smem_u32(&ring_full[it % kRing]), (it / kRing) & 1);
    };
    auto release = [&](int it) { sm100::tc_commit(sm100::smem_u32(&ring_empty[it % kRing]), leader); };
    // stream t's n-th key tile: j = n with two row tiles, 2n + t with one
    auto issue_s = [&](int t, int j) -> bool {
      if (!full(2 * j)) return false;
      sm100::tc_fence_after();
      const uint64_t ad = dq + (uint64_t)((both * t * kPTile) >> 4);
      const uint64_t bd = dk + (uint64_t)((((2 * j) % kRing) * kPTile) >> 4);
#pragma unroll
      for (int kk = 0; kk < kPieceDim / 16; ++kk) {
        const uint32_t off = ((kk >> 2) * kPHalf + (kk & 3) * 32) >> 4;
        sm100::mma_f16_ss(tmem + t * 128, ad + off, bd + off, idesc_s, kk > 0 ? 1u : 0u, leader);
      }
      sm100::tc_commit(sm100::smem_u32(&s_full[t]), leader);
      return true;
    };
    auto issue_pv = [&](int t, int n, int j) -> bool {
      if (!sm100::mbar_wait_warp(sm100::smem_u32(&p_full[t]), n & 1) || !full(2 * j + 1)) return false;
      if (fix_v && j == nkt - 1 && !sm100::mbar_wait_warp(sm100::smem_u32(v_fixed), 0)) return false;
      sm100::tc_fence_after();
      const uint64_t bd = dv + (uint64_t)((((2 * j + 1) % kRing) * kPTile) >> 4);
#pragma unroll
      for (int kk = 0; kk < kPM / 16; ++kk)
        sm100::mma_f16_ts(tmem + 256 + t * 128, tmem + t * 128 + kk * 8, bd + (uint64_t)((kk * 2048) >> 4), idesc_o,
                          (n > 0 || kk > 0) ? 1u : 0u, leader);
      return true;
    };
    if (both) {
      for (int t = 0; t < 2 && ok; ++t) ok = issue_s(t, 0);
      if (ok) release(0);
      for (int j = 0; ok && j < nkt; ++j) {
        if (*(volatile int*)s_abort) ok = false;
        for (int t = 0; t < 2 && ok; ++t) {
          ok = issue_pv(t, j, j);
          if (ok && t == 1) release(2 * j + 1);
          if (ok && j + 1 < nkt) ok = issue_s(t, j + 1);
          if (ok && j + 1 == nkt) sm100::tc_commit(sm100::smem_u32(&o_done[t]), leader);
        }
        if (ok && j + 1 < nkt) release(2 * (j + 1));
      }
    } else {
      // S of tile j + 1 is issued before P V of tile j, which it runs beside
      if (ok) ok = issue_s(0, 0);
      if (ok) release(0);
      for (int j = 0; ok && j < nkt; ++j) {
        if (*(volatile int*)s_abort) ok = false;
        if (ok && j + 1 < nkt) {
          // (the stream's last P was read by its last P V, issued before)
          ok = issue_s((j + 1) & 1, j + 1);
          if (ok) release(2 * (j + 1));
        }
        if (ok) ok = issue_pv(j & 1, j >> 1, j);
        if (ok) release(2 * j + 1);
        if (ok && j + 2 >= nkt) sm100::tc_commit(sm100::smem_u32(&o_done[j & 1]), leader);
      }
    }
    if (!ok && nkt > 0) {
      if (leader) {
        b200_dev_error(kDevErrTimeoutFull);
        atomicExch(s_abort, 1);
      }
      for (int t = 0; t < 2; ++t) sm100::tc_commit(sm100::smem_u32(&o_done[t]), leader);
    }
  } else if (warp == 2) {
    // ---------------------------------- V rows behind the last token are zero
    if (fix_v) {
      const int it = 2 * nkt - 1, slot = it % kRing;
      if (sm100::mbar_wait_warp(sm100::smem_u32(&ring_full[slot]), (it / kRing) & 1)) {
        for (int i = lane; i < 2 * (tile_tok - last_valid) * 8; i += 32) {
          const int c = i & 7, r = (i >> 3) % (tile_tok - last_valid), half = (i >> 3) / (tile_tok - last_valid);
          *reinterpret_cast<uint4*>(smem + L::oRing + slot * kPTile + half * kPHalf + (last_valid + r) * 128 + c * 16) =
              make_uint4(0, 0, 0, 0);
        }
        sm100::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive(sm100::smem_u32(v_fixed));
      } else if (lane == 0) {
        b200_dev_error(kDevErrTimeoutFull);
        atomicExch(s_abort, 1);
      }
    }
  } else if (k8 && warp >= 12) {
    // ------------------------------------------------- code tiles to f16 tiles
    if constexpr (k8) {
      const int r = threadIdx.x - 384;  // this thread's key of every tile
      const int page = r / bs, off = r - page * bs;
      bool ok = true;
      for (int it = 0; it < 2 * nkt && ok; ++it) {
        const int cs = it % p.codes, slot = it % kRing, j = it >> 1, which = it & 1;
        const int valid = j == nkt - 1 ? last_valid : tile_tok;
        const bool live = r < valid;
        ok = sm100::mbar_wait_warp(sm100::smem_u32(&code_full[cs]), (it / p.codes) & 1);
        float ks = 0.f, vs = 1.f;
        if (ok && which == 0 && live) {
          const int64_t at = ((int64_t)s_ids[cs * kPMaxPages + page] * p.Hkv + h) * bs + off;
          ks = __ldg(&k_scale[at]);
          vs = __ldg(&v_scale[at]);
        }
        ok = ok && sm100::mbar_wait_warp(sm100::smem_u32(&ring_empty[slot]), ((it / kRing) & 1) ^ 1);
        if (!ok) break;
        const uint8_t* src = smem + L::oCodes + cs * kPCodes + r * 128;
        uint8_t* dst = smem + L::oRing + slot * kPTile + r * 128;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          uint4 w = make_uint4(0, 0, 0, 0), a = w, b = w;
          if (live) {
            w = *reinterpret_cast<const uint4*>(src + ((c ^ (r & 7)) << 4));
            a = make_uint4(kv8_pair<KV, 0, 1>(w.x), kv8_pair<KV, 2, 3>(w.x), kv8_pair<KV, 0, 1>(w.y),
                           kv8_pair<KV, 2, 3>(w.y));
            b = make_uint4(kv8_pair<KV, 0, 1>(w.z), kv8_pair<KV, 2, 3>(w.z), kv8_pair<KV, 0, 1>(w.w),
                           kv8_pair<KV, 2, 3>(w.w));
          }
          uint8_t* d = dst + (c >> 2) * kPHalf;
          *reinterpret_cast<uint4*>(d + ((((2 * c) & 7) ^ (r & 7)) << 4)) = a;
          *reinterpret_cast<uint4*>(d + ((((2 * c + 1) & 7) ^ (r & 7)) << 4)) = b;
        }
        sm100::fence_proxy_async_smem();
        if (which == 0) {
          // scales of the tile; a key behind the last token has log2 weight -inf
          ok = sm100::mbar_wait_warp(sm100::smem_u32(&sc_empty[j & 1]), ((j >> 1) & 1) ^ 1);
          float lv = -INFINITY, iv = 0.f;
          if (live) kv8_value_scale(vs, lv, iv);
          float* sc = s_sc + (j & 1) * 3 * kPM;
          sc[r] = ks;
          sc[kPM + r] = lv;
          sc[2 * kPM + r] = iv;
        }
        __syncwarp();
        if (lane == 0) {
          sm100::mbar_arrive(sm100::smem_u32(&ring_full[slot]));
          sm100::mbar_arrive(sm100::smem_u32(&code_empty[cs]));
          if (which == 0) sm100::mbar_arrive(sm100::smem_u32(&sc_full[j & 1]));
        }
      }
      if (!ok && lane == 0) {
        b200_dev_error(kDevErrTimeoutFull);
        atomicExch(s_abort, 1);
      }
    }
  } else if (warp >= 4 && warp < 12) {
    // --------------------------------------------------------------- softmax
    const int t = (warp >> 2) - 1, quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const int64_t qr = row0 + both * t * kPM + r;  // row of Q_h
    const bool live = qr < R;
    const int64_t b = live ? qr / p.G : 0;
    const int64_t qrow = b * p.Hq + (int64_t)h * p.G + (live ? qr - b * p.G : 0);
    // (with one row tile the second stream stages it too, into the unused tile, for the row's factor)
    const float sl = stage_q_row<T, k8>(q + qrow * kPieceDim, live, smem + L::oQ + t * kPTile, r, p.qscale);
    sm100::fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0 && (both || t == 0)) sm100::mbar_arrive(sm100::smem_u32(q_full));

    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const uint32_t tS = tmem + t * 128 + lane_off, tO = tmem + 256 + t * 128 + lane_off;
    float m_used = -INFINITY, l = 0.f;
    bool ok = true;
    const int n_tiles = both ? nkt : (nkt - t + 1) / 2;  // key tiles of this stream
    for (int n = 0; n < n_tiles; ++n) {
      const int j = both ? n : 2 * n + t;
      ok = sm100::mbar_wait_warp(sm100::smem_u32(&s_full[t]), n & 1);
      if (k8 && ok) ok = sm100::mbar_wait_warp(sm100::smem_u32(&sc_full[j & 1]), (j >> 1) & 1);
      if (!ok) break;
      sm100::tc_fence_after();
      const int valid = j == nkt - 1 ? last_valid : tile_tok;
      const float* sc = s_sc + (j & 1) * 3 * kPM;
      // logits (log2 units; 8-bit: plus log2 of the value's scale) of 32 keys
      auto logits = [&](int c, float* y) {
        uint32_t v[32];
        sm100::tmem_ld_32x32b_x32(tS + c * 32, v);
        sm100::tmem_wait_ld_regs(v);
        if constexpr (k8) {
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 k4 = *reinterpret_cast<const float4*>(sc + c * 32 + i);
            const float4 l4 = *reinterpret_cast<const float4*>(sc + kPM + c * 32 + i);
            y[i] = fmaf(__uint_as_float(v[i]) * sl, k4.x, l4.x);
            y[i + 1] = fmaf(__uint_as_float(v[i + 1]) * sl, k4.y, l4.y);
            y[i + 2] = fmaf(__uint_as_float(v[i + 2]) * sl, k4.z, l4.z);
            y[i + 3] = fmaf(__uint_as_float(v[i + 3]) * sl, k4.w, l4.w);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) y[i] = c * 32 + i < valid ? __uint_as_float(v[i]) * sl : -INFINITY;
        }
      };
      float mx = -INFINITY;
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        float y[32];
        logits(c, y);
#pragma unroll
        for (int i = 0; i < 32; i += 2) mx = sm100::fmax3(mx, y[i], y[i + 1]);
      }
      float alpha = 1.f;
      bool rescale = false;
      if (m_used == -INFINITY) {
        m_used = mx;
      } else if (mx > m_used + 8.0f) {
        alpha = ex2(m_used - mx);
        m_used = mx;
        rescale = true;
      }
      const float m0 = m_used == -INFINITY ? 0.f : m_used;
      // O holds the products of the tiles before this one (complete: S of this tile is)
      if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll 1
        for (int c = 0; c < kPieceDim; c += 32) {
          uint32_t o[32];
          sm100::tmem_ld_32x32b_x32(tO + c, o);
          sm100::tmem_wait_ld_regs(o);
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
          sm100::tmem_st_32x32b_x32(tO + c, o);
        }
      }
      float sum = 0.f;
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        float y[32];
        logits(c, y);
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          float w0 = ex2(y[i] - m0), w1 = ex2(y[i + 1] - m0), w2 = ex2(y[i + 2] - m0), w3 = ex2(y[i + 3] - m0);
          pk[i / 2] = pack_pair<M>(w0, w1);
          pk[i / 2 + 1] = pack_pair<M>(w2, w3);
          if constexpr (k8) {
            const float4 i4 = *reinterpret_cast<const float4*>(sc + 2 * kPM + c * 32 + i);
            sum = fmaf(w0, i4.x, fmaf(w1, i4.y, fmaf(w2, i4.z, fmaf(w3, i4.w, sum))));
          } else {
            sum += (w0 + w1) + (w2 + w3);
          }
        }
        // P's 16 columns overwrite logits this thread has read already
        sm100::tmem_st_32x32b_x16(tS + c * 16, pk);
      }
      l = l * alpha + sum;
      sm100::tmem_wait_st();
      sm100::tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        sm100::mbar_arrive(sm100::smem_u32(&p_full[t]));
        if (k8) sm100::mbar_arrive(sm100::smem_u32(&sc_empty[j & 1]));
      }
    }
    // ---- the row's piece
    if (ok && n_tiles > 0) ok = sm100::mbar_wait_warp(sm100::smem_u32(&o_done[t]), 0);
    if (!ok) {
      b200_dev_error(kDevErrTimeoutMma);
      atomicExch(s_abort, 1);
    }
    sm100::tc_fence_after();
    // With one row tile stream 1 hands its state to stream 0 through the K/V
    // ring, which nothing reads any more once both streams' products are done.
    // (Every path leads both warpgroups to the barrier.)
    float* hand = reinterpret_cast<float*>(smem + L::oRing);  // [130][128]
    const bool join = !both && nkt > 1;
    float f0 = 1.f, f1 = 0.f;
    if (join) {
      if (t == 1) {
        if (ok && !sm100::mbar_wait_warp(sm100::smem_u32(&o_done[0]), 0)) ok = false;
        sm100::tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < kPieceDim; c += 32) {
          uint32_t o[32];
          sm100::tmem_ld_32x32b_x32(tO + c, o);
          sm100::tmem_wait_ld_regs(o);
#pragma unroll
          for (int i = 0; i < 32; ++i) hand[(c + i) * kPM + r] = __uint_as_float(o[i]);
        }
        hand[128 * kPM + r] = m_used;
        hand[129 * kPM + r] = l;
      }
      named_bar_sync(1, 256);
      if (t == 0) {
        const float m1 = hand[128 * kPM + r], mn = fmaxf(m_used, m1);
        f0 = m_used == mn || m_used == -INFINITY ? 1.f : ex2(m_used - mn);
        f1 = m1 == mn || m1 == -INFINITY ? 1.f : ex2(m1 - mn);
        m_used = mn;
        l = l * f0 + hand[129 * kPM + r] * f1;
      }
    }
    if (both || t == 0) {
      float* dst = pieces + ((int64_t)split * p.B * p.Hq + qrow) * kPiecePitch;
      if (live) *reinterpret_cast<float2*>(dst + kPieceDim) = make_float2(m_used, l);
      if (n_tiles > 0) {
#pragma unroll 1
        for (int c = 0; c < kPieceDim; c += 32) {
          uint32_t o[32];
          sm100::tmem_ld_32x32b_x32(tO + c, o);
          sm100::tmem_wait_ld_regs(o);
          if (join) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              o[i] = __float_as_uint(__uint_as_float(o[i]) * f0 + hand[(c + i) * kPM + r] * f1);
          }
          if (live) {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              *reinterpret_cast<uint4*>(dst + c + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          }
        }
      }
    }
    sm100::tc_fence_before();
  }
  __syncthreads();
  if (warp == 1) {
    sm100::tc_fence_after();
    sm100::tmem_dealloc(tmem, 512);
  }
}

template <typename T, typename KV>
int launch_prefix(const AttnCall& a, const PieceGeom& g, const PieceSpace& w, cudaStream_t stream) {
  constexpr bool k8 = sizeof(KV) == 1;
  constexpr uint64_t el = sizeof(KV);
  const CUtensorMapDataType dt = k8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                    : (std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                      : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16);
  // a box: 128 bytes of dims x one page's tokens x one head, as 128-byte rows swizzled in 8-row atoms
  CUtensorMap tk, tv;
  const uint64_t dims[3] = {(uint64_t)kPieceDim, (uint64_t)(a.num_blocks * a.block_size), (uint64_t)a.Hkv};
  const uint64_t strides[2] = {(uint64_t)a.Hkv * kPieceDim * el, (uint64_t)kPieceDim * el};
  const uint32_t box[3] = {(uint32_t)(128 / el), (uint32_t)a.block_size, 1};
  int st = encode_tensor_map(&tk, dt, 3, a.k_cache, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  if (st) return st;
  st = encode_tensor_map(&tv, dt, 3, a.v_cache, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  if (st) return st;
  PrefixParams p{};
  p.B = a.B, p.Hq = a.Hq, p.Hkv = a.Hkv, p.num_blocks = a.num_blocks, p.max_prefix = a.max_prefix_blocks;
  p.G = g.G, p.bs = (int)a.block_size, p.ppt = kPM / (int)a.block_size;
  p.codes = 3;
  p.splits = w.prefix_splits;
  p.qscale = a.scale * 1.4426950408889634f;
  const size_t smem = 1024 + PrefixSmem<k8>::oCodes + (k8 ? p.codes * kPCodes : 0) +
                      8 * (1 + 2 * kPRing16 + 6 + 1 + 4 + 2 * kPMaxCodes) + 16 + 4 * kPMaxCodes * kPMaxPages +
                      (k8 ? 2 * 3 * kPM * 4 : 0);
  auto kern = prefix_attn_kernel<T, KV>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return launch_status(e);
  const int64_t pairs = (a.B * g.G + 2 * kPM - 1) / (2 * kPM);
  kern<<<dim3((unsigned)p.splits, (unsigned)pairs, (unsigned)a.Hkv), k8 ? 512 : 384, smem, stream>>>(
      tk, tv, a.k_scale, a.v_scale, static_cast<const T*>(a.q), IndexPtr{a.prefix_table, a.index_dtype == B200_I64},
      IndexPtr{a.prefix_len, a.index_dtype == B200_I64}, w.prefix, p);
  return launch_status(cudaGetLastError());
}

}  // namespace
}  // namespace b200

#define B200_DEFINE_PREFIX_LAUNCHER(NAME, KVT)                                                           \
  namespace b200 {                                                                                       \
  int launch_prefix_##NAME(const AttnCall& a, const PieceGeom& g, const PieceSpace& w, cudaStream_t s) { \
    return B200_DISPATCH_HALF(a.dtype, [&] { return launch_prefix<scalar_t, KVT>(a, g, w, s); });        \
  }                                                                                                      \
  }
