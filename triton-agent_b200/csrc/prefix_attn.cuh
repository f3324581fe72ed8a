// The shared prefix of a batch: all query rows of a kv head against the
// prefix's keys, on the fifth-generation tensor cores.
//
// For kv head h the batch's query rows r = b * G + g form one matrix Q_h
// [B G, 128].  A CTA takes two 128-row tiles of it (one when there are no more) and one
// stretch of the prefix's block table, and leaves one piece (m, l, o) a row --
// the pieces the streaming kernel leaves for the own tokens, joined with them:
//   S = Q K^T    tcgen05.mma 128 x 128 x 16 (Q, K K-major in shared memory), fp32 in tensor memory
//   softmax      one thread a row, the row's 128 logits in registers; O rescaled only
//                when the maximum grew by more than 2^8
//   O += P V     P (16-bit) over S's columns in tensor memory, V MN-major
// With one row tile the two softmax warpgroups take its even and its odd key
// tiles, each with an O of its own, joined in shared memory at the end: the
// chain S -> softmax -> P V of one tile then runs beside the other's as with two row tiles.
//
// Reading the prefix costs its bytes once a CTA column instead of once a
// sequence: at 64 sequences of an 8192-token prefix 33.5 MB instead of 2.1 GB.
//
// Roles: warps 0 and 2 walk the block table and copy the pages of K and V (one TMA
// box a page; a tile is as many pages as fit 128 tokens), warp 1 issues the MMAs,
// warps 4-11 are the two streams' softmax warpgroups.  16-bit caches: pages land
// in the K/V ring as the MMA reads them; warp 2 zeroes V rows behind the last
// token (a weight of 0 times a NaN left in the cache is NaN).  8-bit caches:
// pages land in a ring of code tiles, and warps 12-15 widen them to f16 tiles
// (codes are exact in f16) and load the scales, a tile ahead; the scales meet the
// logits and weights in fp32 as in the streaming kernel.
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
constexpr int kPRing16 = 5, kPRing8 = 3;   // K/V tiles in shared memory; one more with one row tile
constexpr int kPCodeRing = 3;              // code tiles (8-bit)
constexpr int kPScaleRing = 4;             // key tiles whose scales wait for the softmax (8-bit), and page ids
constexpr int kPMaxPages = 8;              // pages of a tile (block size 16)
constexpr int kPList = 32 + kPMaxPages;    // pages a producer holds

struct PrefixParams {
  int64_t B, Hq, Hkv, num_blocks, max_prefix;
  int lgG, bs, ppt;  // log2 of the query heads a kv head, block size, pages a key tile
  int splits;
  float qscale;  // scale * log2(e)
};

template <bool k8>
struct PrefixSmem {
  static constexpr uint32_t oQ = 0;  // two Q tiles
  static constexpr uint32_t oRing = 2 * kPTile;
  static constexpr uint32_t oCodes = oRing + (k8 ? kPRing8 : kPRing16) * kPTile;
  static constexpr uint32_t oScales = oCodes + (k8 ? kPCodeRing * kPCodes : 0);  // [tile][ks, log2 vs, 1 / vs][128]
  static constexpr uint32_t oRaw = oScales + (k8 ? kPScaleRing * 3 * kPM * 4 : 0);  // [ks, vs][128] of the next tile
  static constexpr uint32_t oBars = oRaw + (k8 ? 2 * kPM * 4 : 0);
};

// A warp's 32 rows of Q (row r of the batch's matrix: sequence r / G, head h G +
// r % G) into the swizzled tile at `tile`: 16-byte chunk c of row r sits at
// chunk c ^ (r & 7) of its 128-byte row, dims 64.. in the second half.  Sixteen
// lanes a row, so that the loads are whole rows.  8-bit caches: f16, each row scaled
// to [2^13, 2^14) by a power of two.  Returns the logit factor of row `lane`; a
// tile of 0 stages nothing else.
template <typename T, bool k8>
__device__ __forceinline__ float stage_q_rows(const T* __restrict__ q, int r0, int R, int64_t Hq, int h, int lgG,
                                              uint32_t tile, int r_tile, int lane, float qscale) {
  const int c = lane & 15, odd = lane >> 4;
  float factor = qscale;
  uint4 raw[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int r = r0 + 2 * i + odd;
    raw[i] = make_uint4(0, 0, 0, 0);
    if (r < R) {
      const int64_t row = (int64_t)(r >> lgG) * Hq + (h << lgG) + (r & ((1 << lgG) - 1));
      raw[i] = __ldg(reinterpret_cast<const uint4*>(q + row * kPieceDim) + c);
    }
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    if constexpr (k8) {
      float f[8], amax = 0.f, up, down;
      unpack16<T>(raw[i], f);
#pragma unroll
      for (int k = 0; k < 8; ++k) amax = fmaxf(amax, fabsf(f[k]));
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      pow2_scale<13>(amax, up, down);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] *= up;
      raw[i] = pack16<__half>(f);
      const float d = __shfl_sync(0xffffffffu, down, (lane & 1) * 16);
      if (i == lane >> 1) factor = qscale * d;
    }
    const int r = r_tile + 2 * i + odd;
    if (tile != 0) sts128(tile + (c >> 3) * kPHalf + r * 128 + (((c & 7) ^ (r & 7)) << 4), raw[i]);
  }
  return factor;
}

// A K or V tile: groups of eight tokens, each with dims 0..63 and then 64..127
// as an atom of eight swizzled 128-byte rows, so that a page is one contiguous
// box whatever its size.  Where 16-byte chunk c of token r sits:
__device__ __forceinline__ uint32_t kv_at(int r, int c) {
  return (uint32_t)((r >> 3) * 2048 + (c >> 3) * 1024 + (r & 7) * 128 + (((c & 7) ^ (r & 7)) << 4));
}

// Registers a thread, softmax warps and the others: 128 at launch with 8-bit caches (8 warps each), 168
// with 16-bit ones (8 and 4).  The split hands out what the kernel has at launch; build.py holds the
// compiler's choice against `launch`.
template <bool k8>
struct PrefixRegs {
  static constexpr int low = 72, high = k8 ? 184 : 216, threads = k8 ? 512 : 384, launch = k8 ? 128 : 168;
  static_assert(launch * threads >= 256 * high + (threads - 256) * low, "more registers than at launch");
};

template <typename T, typename KV>
__global__ void __launch_bounds__(PrefixRegs<sizeof(KV) == 1>::threads, 1)
    prefix_attn_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                       const float* __restrict__ k_scale, const float* __restrict__ v_scale, const T* __restrict__ q,
                       IndexPtr ptab, IndexPtr plen, float* __restrict__ pieces, PrefixParams p) {
  constexpr bool k8 = sizeof(KV) == 1;
  using M = typename std::conditional<k8, __half, T>::type;  // type of the matrix operands
  using L = PrefixSmem<k8>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = sm100::smem_u32(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = blockIdx.x, h = blockIdx.z;
  const int R = (int)p.B << p.lgG, row0 = (int)blockIdx.y * 2 * kPM;
  const int tiles = R - row0 > kPM ? 2 : 1;
  const int both = tiles == 2;  // else: streams 0 and 1 are the even and odd key tiles of one row tile
  const int bs = p.bs, tile_tok = p.ppt * bs;

  // with one row tile the second Q tile's place belongs to the ring
  const int depth = (k8 ? kPRing8 : kPRing16) + (both ? 0 : 1);
  const uint32_t ring = sbase + L::oRing - (both ? 0 : kPTile);
  const uint32_t depth_inv = 0xffffffffu / (uint32_t)depth + 1;  // i / depth for i < 2^29
  auto round_of = [&](int i) { return (int)__umulhi((uint32_t)i, depth_inv); };
  auto slot_of = [&](int i) { return i - round_of(i) * depth; };

  uint64_t* ring_full = reinterpret_cast<uint64_t*>(smem + L::oBars);  // [depth]
  uint64_t* ring_empty = ring_full + kPRing16 + 1;  // [depth]
  uint64_t* s_full = ring_empty + kPRing16 + 1;  // [2]
  uint64_t* p_full = s_full + 2;                // [2]
  uint64_t* o_done = p_full + 2;                // [2]
  uint64_t* v_fixed = o_done + 2;
  uint64_t* q_full = v_fixed + 1;
  uint64_t* sc_full = q_full + 1;                // [kPScaleRing]
  uint64_t* sc_empty = sc_full + kPScaleRing;    // [kPScaleRing]
  uint64_t* ids_full = sc_empty + kPScaleRing;   // [kPScaleRing]
  uint64_t* code_full = ids_full + kPScaleRing;  // [kPCodeRing]
  uint64_t* code_empty = code_full + kPCodeRing;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(code_empty + kPCodeRing);
  int* s_abort = reinterpret_cast<int*>(tmem_slot + 1);
  int* s_count = s_abort + 1;  // [2][16] dropped entries before the split and in it, by warp
  int* s_ids = s_count + 32;   // [kPScaleRing][kPMaxPages] page ids of a key tile
  int* s_list = s_ids + kPScaleRing * kPMaxPages;  // [K, V][kPList] pages to copy

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
    // dropped entries before the split and in it
    const int before = __reduce_add_sync(0xffffffffu, ptab.dropped(0, e0, p.num_blocks));
    const int in = __reduce_add_sync(0xffffffffu, ptab.dropped(e0, e1 - e0, p.num_blocks));
    if (lane == 0) {
      s_count[warp] = before;
      s_count[16 + warp] = in;
    }
  }
  if (threadIdx.x == 32) {
    *s_abort = 0;
    for (int i = 0; i < depth; ++i) {
      sm100::mbar_init(sm100::smem_u32(&ring_full[i]), k8 ? 4 : 1);
      sm100::mbar_init(sm100::smem_u32(&ring_empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      sm100::mbar_init(sm100::smem_u32(&s_full[i]), 1);
      sm100::mbar_init(sm100::smem_u32(&p_full[i]), 4);
      sm100::mbar_init(sm100::smem_u32(&o_done[i]), 1);
    }
    sm100::mbar_init(sm100::smem_u32(v_fixed), 1);
    sm100::mbar_init(sm100::smem_u32(q_full), 8);
    for (int i = 0; i < kPScaleRing; ++i) {
      sm100::mbar_init(sm100::smem_u32(&sc_full[i]), 4);
      sm100::mbar_init(sm100::smem_u32(&ids_full[i]), 1);
      sm100::mbar_init(sm100::smem_u32(&sc_empty[i]), 4 * tiles);  // one stream's warps, or both's
    }
    for (int i = 0; i < kPCodeRing; ++i) {
      sm100::mbar_init(sm100::smem_u32(&code_full[i]), 1);
      sm100::mbar_init(sm100::smem_u32(&code_empty[i]), 4);
    }
    sm100::fence_barrier_init();
  }
  if (!k8 && tile_tok < kPM) {
    // rows no page reaches stay zero in every ring tile (both operands)
    const int dead = kPM - tile_tok;
    for (int i = threadIdx.x; i < depth * dead * 16; i += blockDim.x) {
      const int c = i & 15, r = (i >> 4) % dead, slot = (i >> 4) / dead;
      sts128(ring + slot * kPTile + kv_at(tile_tok + r, c), make_uint4(0, 0, 0, 0));
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
  int ntok;
  {
    int before = e0, in = e1 - e0;
    for (int w = 0; w < (int)(blockDim.x >> 5); ++w) {
      before -= s_count[w];
      in -= s_count[16 + w];
    }
    const int64_t left = plen_tokens - (int64_t)before * bs, have = (int64_t)in * bs;
    ntok = (int)(left < 0 ? 0 : (left < have ? left : have));
  }
  const int nkt = (ntok + tile_tok - 1) / tile_tok;
  const int last_valid = ntok - (nkt - 1) * tile_tok;  // tokens of the last tile
  const bool fix_v = !k8 && nkt > 0 && last_valid < tile_tok;

  if (warp < 4) sm100::setmaxnreg_dec<PrefixRegs<k8>::low>();
  if (warp == 0 || warp == 2) {
    // ------------------------------------- producers: K tiles and V tiles, in turn in one ring
    const int which = warp >> 1;
    const CUtensorMap* map = which ? &tm_v : &tm_k;
    if (lane == 0) sm100::tma_prefetch_desc(map);
    const int slots = k8 ? kPCodeRing : depth;
    uint64_t* fulls = k8 ? code_full : ring_full;
    uint64_t* empties = k8 ? code_empty : ring_empty;
    const uint32_t page_bytes = (uint32_t)(bs * kPieceDim * (int)sizeof(KV));
    int* list = s_list + which * kPList;
    int left = (ntok + bs - 1) / bs;  // pages still to copy
    int have = 0, issued = 0;         // pages in the list, tiles copied
    int slot = which;
    uint32_t ph = 1;  // parity of the empty barriers in this round
    bool ok = true;
    int64_t next = e0 + lane < e1 ? ptab.at(e0 + lane) : -1;
    for (int j0 = e0; j0 < e1 && left > 0 && ok; j0 += 32) {
      const int64_t id = next;
      next = j0 + 32 + lane < e1 ? ptab.at(j0 + 32 + lane) : -1;
      const bool valid = id >= 0 && id < p.num_blocks;
      const unsigned use = __ballot_sync(0xffffffffu, valid);
      if (valid) list[have + __popc(use & ((1u << lane) - 1u))] = (int)id;
      have += __popc(use);
      __syncwarp();
      int at = 0;
      while (left > 0 && (have - at >= p.ppt || have - at >= left)) {
        const int np = left < p.ppt ? left : p.ppt;
        ok = !*(volatile int*)s_abort && sm100::mbar_wait(sm100::smem_u32(&empties[slot]), ph);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const uint32_t fb = sm100::smem_u32(&fulls[slot]);
        const int page = lane < np ? list[at + lane] : 0;
        if (lane == 0) sm100::mbar_arrive_expect_tx(fb, np * page_bytes);
        if (k8 && which == 0 && lane < np) s_ids[issued % kPScaleRing * kPMaxPages + lane] = page;
        __syncwarp();
        if (lane < np) {
          if constexpr (k8)
            sm100::tma_load_3d(sbase + L::oCodes + slot * kPCodes + lane * page_bytes, map, fb, 0, page * bs, h);
          else
            sm100::tma_load_4d(ring + slot * kPTile + lane * page_bytes, map, fb, 0, 0, 2 * h,
                               page * (bs >> 3));
        }
        if (k8 && which == 0 && lane == 0) sm100::mbar_arrive(sm100::smem_u32(&ids_full[issued % kPScaleRing]));
        at += np;
        left -= np;
        ++issued;
        slot += 2;
        if (slot >= slots) {
          slot -= slots;
          ph ^= 1u;
        }
      }
      have -= at;  // (fewer than a tile's pages are left)
      const int rest = lane < have ? list[at + lane] : 0;
      __syncwarp();
      if (lane < have) list[lane] = rest;
    }
    if (lane == 0) {
      if (!ok) {
        b200_dev_error(kDevErrTimeoutEmpty);
        atomicExch(s_abort, 1);
      }
      // no copy may still be writing shared memory when the CTA exits
      for (int i = 2 * issued - 2 + which; i >= 0 && i >= 2 * issued - slots; i -= 2)
        if (!sm100::mbar_wait(sm100::smem_u32(&fulls[i % slots]), (i / slots) & 1)) b200_dev_error(kDevErrTimeoutFull);
    }
    __syncwarp();
    if (warp == 2 && fix_v) {
      // V rows behind the last token are zero
      const int it = 2 * nkt - 1, vslot = slot_of(it);
      if (sm100::mbar_wait_warp(sm100::smem_u32(&ring_full[vslot]), round_of(it) & 1)) {
        for (int i = lane; i < (tile_tok - last_valid) * 16; i += 32)
          sts128(ring + vslot * kPTile + kv_at(last_valid + (i >> 4), i & 15), make_uint4(0, 0, 0, 0));
        sm100::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive(sm100::smem_u32(v_fixed));
      } else if (lane == 0) {
        b200_dev_error(kDevErrTimeoutFull);
        atomicExch(s_abort, 1);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------- MMA issue
    constexpr uint32_t fmt = std::is_same<M, __nv_bfloat16>::value ? 1u : 0u;
    constexpr uint32_t idesc_s = sm100::make_idesc(1, fmt, fmt, 0, 0, kPM, kPM);
    constexpr uint32_t idesc_o = sm100::make_idesc(1, fmt, fmt, 0, 1, kPM, kPieceDim);
    const uint32_t leader = sm100::elect_one();
    const uint64_t dq = sm100::make_smem_desc(sbase + L::oQ, 16, 1024, sm100::kSwizzle128B);
    const uint64_t dk = sm100::make_smem_desc(ring, 16, 2048, sm100::kSwizzle128B);
    const uint64_t dv = sm100::make_smem_desc(ring, 1024, 2048, sm100::kSwizzle128B);
    bool ok = nkt > 0 && sm100::mbar_wait_warp(sm100::smem_u32(q_full), 0);
    auto full = [&](int it) -> bool {
      return sm100::mbar_wait_warp(sm100::smem_u32(&ring_full[slot_of(it)]), round_of(it) & 1);
    };
    auto release = [&](int it) { sm100::tc_commit(sm100::smem_u32(&ring_empty[slot_of(it)]), leader); };
    // stream t's n-th key tile: j = n with two row tiles, 2n + t with one
    auto issue_s = [&](int t, int j) -> bool {
      if (!full(2 * j)) return false;
      sm100::tc_fence_after();
      const uint64_t ad = dq + (uint64_t)((both * t * kPTile) >> 4);
      const uint64_t bd = dk + (uint64_t)((slot_of(2 * j) * kPTile) >> 4);
#pragma unroll
      for (int kk = 0; kk < kPieceDim / 16; ++kk) {
        const uint32_t offa = ((kk >> 2) * kPHalf + (kk & 3) * 32) >> 4;
        const uint32_t offb = ((kk >> 2) * 1024 + (kk & 3) * 32) >> 4;
        sm100::mma_f16_ss(tmem + t * 128, ad + offa, bd + offb, idesc_s, kk > 0 ? 1u : 0u, leader);
      }
      sm100::tc_commit(sm100::smem_u32(&s_full[t]), leader);
      return true;
    };
    auto issue_pv = [&](int t, int n, int j) -> bool {
      if (!sm100::mbar_wait_warp(sm100::smem_u32(&p_full[t]), n & 1) || !full(2 * j + 1)) return false;
      if (fix_v && j == nkt - 1 && !sm100::mbar_wait_warp(sm100::smem_u32(v_fixed), 0)) return false;
      sm100::tc_fence_after();
      const uint64_t bd = dv + (uint64_t)((slot_of(2 * j + 1) * kPTile) >> 4);
#pragma unroll
      for (int kk = 0; kk < kPM / 16; ++kk)
        sm100::mma_f16_ts(tmem + 256 + t * 128, tmem + t * 128 + kk * 8, bd + (uint64_t)((kk * 4096) >> 4), idesc_o,
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
  } else if (k8 && warp >= 12) {
    // ------------------------------------------------- code tiles to f16 tiles
    if constexpr (k8) {
      sm100::setmaxnreg_dec<PrefixRegs<k8>::low>();
      const int r = threadIdx.x - 384;  // this thread's key of every tile
      const int page = r / bs, off = r - page * bs;
      bool ok = true;
      int cs = 0;
      uint32_t cph = 0;
      // scales of this thread's key of tile j on their way to its own places in
      // shared memory (its page ids are there: a code ring of three tiles or more
      // holds K of the next tile)
      const uint32_t raw = sbase + L::oRaw + r * 4;
      auto load_scales = [&](int j) {
        if (!sm100::mbar_wait_warp(sm100::smem_u32(&ids_full[j % kPScaleRing]), (j / kPScaleRing) & 1)) return false;
        if (r < (j == nkt - 1 ? last_valid : tile_tok)) {
          const int id = lds_s32(sm100::smem_u32(s_ids + (j % kPScaleRing) * kPMaxPages + page));
          const int64_t at = ((int64_t)id * p.Hkv + h) * bs + off;
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(raw), "l"(k_scale + at) : "memory");
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(raw + kPM * 4), "l"(v_scale + at) : "memory");
        }
        return true;
      };
      if (nkt > 0) ok = load_scales(0);
      for (int it = 0; it < 2 * nkt && ok; ++it) {
        const int slot = slot_of(it), j = it >> 1, which = it & 1;
        const int valid = j == nkt - 1 ? last_valid : tile_tok;
        const bool live = r < valid;
        ok = sm100::mbar_wait_warp(sm100::smem_u32(&code_full[cs]), cph);
        if (!ok) break;
        const uint32_t src = sbase + L::oCodes + cs * kPCodes + r * 128;
        uint4 w[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) w[c] = lds128(src + ((c ^ (r & 7)) << 4));
        ok = sm100::mbar_wait_warp(sm100::smem_u32(&ring_empty[slot]), (round_of(it) & 1) ^ 1);
        if (!ok) break;
        const uint32_t dst = ring + slot * kPTile;
        if (live) {
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            uint4 a, b;
            kv8_in_order<KV>(w[c].x, a.x, a.y);
            kv8_in_order<KV>(w[c].y, a.z, a.w);
            kv8_in_order<KV>(w[c].z, b.x, b.y);
            kv8_in_order<KV>(w[c].w, b.z, b.w);
            sts128(dst + kv_at(r, 2 * c), a);
            sts128(dst + kv_at(r, 2 * c + 1), b);
          }
        } else {
          for (int c = 0; c < 16; ++c) sts128(dst + kv_at(r, c), make_uint4(0, 0, 0, 0));
        }
        sm100::fence_proxy_async_smem();
        if (which == 0) {
          // scales of the tile; a key behind the last token has log2 weight -inf
          const int ss = j % kPScaleRing;
          ok = sm100::mbar_wait_warp(sm100::smem_u32(&sc_empty[ss]), ((j / kPScaleRing) & 1) ^ 1);
          float ks = 0.f, lv = -INFINITY, iv = 0.f;
          asm volatile("cp.async.wait_all;" ::: "memory");
          if (live) {
            ks = lds_f32(raw);
            kv8_value_scale(lds_f32(raw + kPM * 4), lv, iv);
          }
          const uint32_t sc = sbase + L::oScales + (uint32_t)(ss * 3 * kPM + r) * 4;
          sts_f32(sc, ks);
          sts_f32(sc + kPM * 4, lv);
          sts_f32(sc + 2 * kPM * 4, iv);
          if (ok && j + 1 < nkt) ok = load_scales(j + 1);
        }
        __syncwarp();
        if (lane == 0) {
          sm100::mbar_arrive(sm100::smem_u32(&ring_full[slot]));
          sm100::mbar_arrive(sm100::smem_u32(&code_empty[cs]));
          if (which == 0) sm100::mbar_arrive(sm100::smem_u32(&sc_full[j % kPScaleRing]));
        }
        if (++cs == kPCodeRing) {
          cs = 0;
          cph ^= 1u;
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      if (!ok && lane == 0) {
        b200_dev_error(kDevErrTimeoutFull);
        atomicExch(s_abort, 1);
      }
    }
  } else if (warp >= 4 && warp < 12) {
    // --------------------------------------------------------------- softmax
    sm100::setmaxnreg_inc<PrefixRegs<k8>::high>();
    const int t = (warp >> 2) - 1, quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const int qr = row0 + both * t * kPM + r;  // row of Q_h
    const bool live = qr < R;
    const int64_t qrow = live ? (int64_t)(qr >> p.lgG) * p.Hq + (h << p.lgG) + (qr & ((1 << p.lgG) - 1)) : 0;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const uint32_t tS = tmem + t * 128 + lane_off, tO = tmem + 256 + t * 128 + lane_off;
    // Q, while the first pages are on their way (with one row tile the second
    // warpgroup only takes its rows' factors)
    const uint32_t q_tile = t == 0 || both ? sbase + L::oQ + t * kPTile : 0;
    float sl = p.qscale;
    if (k8 || q_tile != 0)
      sl = stage_q_rows<T, k8>(q, row0 + both * t * kPM + quarter * 32, R, p.Hq, h, p.lgG, q_tile, quarter * 32, lane,
                               p.qscale);
    sm100::fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) sm100::mbar_arrive(sm100::smem_u32(q_full));
    float m_used = -INFINITY, l = 0.f;
    bool ok = true;
    const int n_tiles = both ? nkt : (nkt - t + 1) / 2;  // key tiles of this stream
    for (int n = 0; n < n_tiles; ++n) {
      const int j = both ? n : 2 * n + t, ss = j % kPScaleRing;
      ok = sm100::mbar_wait_warp(sm100::smem_u32(&s_full[t]), n & 1);
      if (k8 && ok) ok = sm100::mbar_wait_warp(sm100::smem_u32(&sc_full[ss]), (j / kPScaleRing) & 1);
      if (!ok) break;
      sm100::tc_fence_after();
      uint32_t v[kPM];
      sm100::tmem_ld_32x32b_x64(tS, v);
      sm100::tmem_ld_32x32b_x64(tS + 64, v + 64);
      sm100::tmem_wait_ld_regs(v);
      sm100::tmem_wait_ld_regs(v + 32);
      sm100::tmem_wait_ld_regs(v + 64);
      sm100::tmem_wait_ld_regs(v + 96);
      const uint32_t sc = sbase + L::oScales + (uint32_t)(ss * 3 * kPM) * 4;
      float f = sl;  // logits in log2 units: f times v (16-bit), or v itself
      if constexpr (k8) {
        // y = (S sl) ks + log2 vs; a key behind the last token has log2 vs = -inf
#pragma unroll
        for (int i = 0; i < kPM; i += 4) {
          const float4 k4 = lds_f32x4(sc + i * 4), l4 = lds_f32x4(sc + (kPM + i) * 4);
          float y[4];
          sm100::fmul2_bcast(y[0], y[1], __uint_as_float(v[i]), __uint_as_float(v[i + 1]), sl);
          sm100::fmul2_bcast(y[2], y[3], __uint_as_float(v[i + 2]), __uint_as_float(v[i + 3]), sl);
          sm100::ffma2(y[0], y[1], y[0], y[1], k4.x, k4.y, l4.x, l4.y);
          sm100::ffma2(y[2], y[3], y[2], y[3], k4.z, k4.w, l4.z, l4.w);
#pragma unroll
          for (int u = 0; u < 4; ++u) v[i + u] = __float_as_uint(y[u]);
        }
        f = 1.f;
      } else {
        const int valid = j == nkt - 1 ? last_valid : tile_tok;
        if (valid < kPM) {
#pragma unroll
          for (int i = 0; i < kPM; ++i)
            if (i >= valid) v[i] = 0xff800000u;
        }
      }
      float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < kPM; i += 8) {
#pragma unroll
        for (int u = 0; u < 4; ++u)
          mx4[u] = sm100::fmax3(mx4[u], __uint_as_float(v[i + 2 * u]), __uint_as_float(v[i + 2 * u + 1]));
      }
      const float mx = sm100::fmax3(mx4[0], mx4[1], fmaxf(mx4[2], mx4[3])) * f;
      float alpha = 1.f;
      bool rescale = false;
      constexpr float kBelow = ref_below<M>();  // (f16 weights: the largest between 2^7 and 2^15)
      if (m_used == -INFINITY) {
        m_used = mx - kBelow;
      } else if (mx > m_used + (8.0f + kBelow)) {
        alpha = ex2(m_used - (mx - kBelow));
        m_used = mx - kBelow;
        rescale = true;
      }
      const float neg = m_used == -INFINITY ? 0.f : -m_used;
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < kPM; i += 4) {
        float w[4];
        if constexpr (k8) {
#pragma unroll
          for (int u = 0; u < 4; ++u) w[u] = ex2(__uint_as_float(v[i + u]) + neg);
          const float4 i4 = lds_f32x4(sc + (2 * kPM + i) * 4);
          sm100::ffma2(sum[0], sum[1], w[0], w[1], i4.x, i4.y, sum[0], sum[1]);
          sm100::ffma2(sum[2], sum[3], w[2], w[3], i4.z, i4.w, sum[2], sum[3]);
        } else {
          sm100::ffma2_bcast(w[0], w[1], __uint_as_float(v[i]), __uint_as_float(v[i + 1]), f, neg);
          sm100::ffma2_bcast(w[2], w[3], __uint_as_float(v[i + 2]), __uint_as_float(v[i + 3]), f, neg);
#pragma unroll
          for (int u = 0; u < 4; ++u) w[u] = ex2(w[u]);
          sm100::fadd2_acc(sum[0], sum[1], w[0], w[1]);
          sm100::fadd2_acc(sum[2], sum[3], w[2], w[3]);
        }
        v[i / 2] = pack_pair<M>(w[0], w[1]);
        v[i / 2 + 1] = pack_pair<M>(w[2], w[3]);
      }
      sm100::tmem_st_32x32b_x64(tS, v);  // P over the logits' columns
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
      l = l * alpha + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
      sm100::tmem_wait_st();
      sm100::tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        sm100::mbar_arrive(sm100::smem_u32(&p_full[t]));
        if (k8) sm100::mbar_arrive(sm100::smem_u32(&sc_empty[ss]));
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
    const uint32_t hand = ring + r * 4;  // [130][128] floats
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
          for (int i = 0; i < 32; ++i) sts_f32(hand + (c + i) * kPM * 4, __uint_as_float(o[i]));
        }
        sts_f32(hand + 128 * kPM * 4, m_used);
        sts_f32(hand + 129 * kPM * 4, l);
      }
      named_bar_sync(1, 256);
      if (t == 0) {
        const float m1 = lds_f32(hand + 128 * kPM * 4), mn = fmaxf(m_used, m1);
        f0 = m_used == mn || m_used == -INFINITY ? 1.f : ex2(m_used - mn);
        f1 = m1 == mn || m1 == -INFINITY ? 1.f : ex2(m1 - mn);
        m_used = mn;
        l = l * f0 + lds_f32(hand + 129 * kPM * 4) * f1;
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
              o[i] = __float_as_uint(__uint_as_float(o[i]) * f0 + lds_f32(hand + (c + i) * kPM * 4) * f1);
          }
          if (live) {
#pragma unroll
            for (int i = 0; i < 32; i += 8) stg256(dst + c + i, o + i);
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
  // a box is a page of one head.  8-bit: its tokens' rows of 128 bytes, swizzled in
  // 8-row atoms; 16-bit: (64 dims, 8 tokens, 2 halves of the dims, groups of 8 tokens)
  CUtensorMap tk, tv;
  const uint64_t tokens = (uint64_t)(a.num_blocks * a.block_size), row = (uint64_t)a.Hkv * kPieceDim * el;
  const uint64_t dims8[3] = {(uint64_t)kPieceDim, tokens, (uint64_t)a.Hkv};
  const uint64_t strides8[2] = {row, (uint64_t)kPieceDim};
  const uint32_t box8[3] = {(uint32_t)kPieceDim, (uint32_t)a.block_size, 1};
  const uint64_t dims16[4] = {64, 8, (uint64_t)(2 * a.Hkv), tokens / 8};
  const uint64_t strides16[3] = {row, 128, 8 * row};
  const uint32_t box16[4] = {64, 8, 2, (uint32_t)(a.block_size / 8)};
  auto encode = [&](CUtensorMap* m, const void* base) {
    return encode_tensor_map(m, dt, k8 ? 3 : 4, base, k8 ? dims8 : dims16, k8 ? strides8 : strides16,
                             k8 ? box8 : box16, CU_TENSOR_MAP_SWIZZLE_128B);
  };
  int st = encode(&tk, a.k_cache);
  if (st) return st;
  st = encode(&tv, a.v_cache);
  if (st) return st;
  PrefixParams p{};
  p.B = a.B, p.Hq = a.Hq, p.Hkv = a.Hkv, p.num_blocks = a.num_blocks, p.max_prefix = a.max_prefix_blocks;
  while ((1 << p.lgG) < g.G) ++p.lgG;
  p.bs = (int)a.block_size, p.ppt = kPM / (int)a.block_size;
  p.splits = w.prefix_splits;
  p.qscale = a.scale * 1.4426950408889634f;
  const size_t smem = 1024 + PrefixSmem<k8>::oBars +
                      8 * (2 * (kPRing16 + 1) + 6 + 2 + 3 * kPScaleRing + 2 * kPCodeRing) + 8 + 128 +
                      4 * (kPScaleRing * kPMaxPages + 2 * kPList);
  static_assert(PrefixSmem<k8>::oBars + 1024 + 1024 <= 227 * 1024, "shared memory of a CTA");
  auto kern = prefix_attn_kernel<T, KV>;
  using Regs = PrefixRegs<k8>;
  // (without the registers the split hands out its warps would wait for good; a
  // failed query is asked again by the next call)
  static std::atomic<bool> checked{false};
  if (!checked.load(std::memory_order_relaxed)) {
    cudaFuncAttributes at{};
    const cudaError_t qe = cudaFuncGetAttributes(&at, kern);
    if (qe != cudaSuccess) return launch_status(qe);
    if (at.numRegs < Regs::launch) {
      set_last_error_detail("prefix_attn_kernel: too few registers at launch for its split");
      return B200_ERR_LAUNCH;
    }
    checked.store(true, std::memory_order_relaxed);
  }
  static SmemGrant grant;
  cudaError_t e = grant(kern, smem);
  if (e != cudaSuccess) return launch_status(e);
  const int64_t pairs = (a.B * g.G + 2 * kPM - 1) / (2 * kPM);
  kern<<<dim3((unsigned)p.splits, (unsigned)pairs, (unsigned)a.Hkv), Regs::threads, smem, stream>>>(
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
