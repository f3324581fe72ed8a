// Decode attention over the 8-bit paged cache, and of batches that share a
// prefix: argument checks, launch geometry, and the kernel that joins pieces.
// The streaming kernel and its mathematics: kv_attn.cuh.
#include "common.cuh"

B200_DEVICE_ERROR_WORD()

#include "prefix_attn.cuh"

namespace b200 {
namespace {

// ---------------------------------------------------------------------------
// Join: W warps a query row (1, 2, 4 or 8: as many as keep a GPU's worth of
// warps busy when rows are few and their pieces many).  The row's pieces are those
// of its segment's ranges and those of the prefix's splits; every warp folds the (m) of
// all of them, then adds the weighted rows of its share, four dims a lane,
// and the first warp adds up the shares.  A row that the streaming kernel
// wrote itself is skipped; a row without any token is zero.  What bounds it is the chain of
// loads behind the wait -- span, sums, rows -- so spans come ready from the streaming kernel
// and the first kAhead rows are fetched beside the sums (with divisions
// for the spans and rows after the weights: 250 sequences behind a prefix 65 us, so 58).
// ---------------------------------------------------------------------------
struct JoinParams {
  int64_t B, Hq;
  int heads_cta, splits, W;
};

constexpr int kAhead = 4;
template <typename T>
__global__ void __launch_bounds__(256)
    paged_attn_join_kernel(const int2* __restrict__ spans, const float* __restrict__ rows,
                           const float* __restrict__ prefix, T* __restrict__ out, JoinParams p) {
  __shared__ float s_part[8][kD];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int W = p.W, share = warp % W;
  const uint32_t row = blockIdx.x * (uint32_t)(8 / W) + warp / W;
  const bool live = row < (uint32_t)(p.B * p.Hq);
  const uint32_t b = live ? row / (uint32_t)p.Hq : 0;
  const int h = live ? (int)(row - b * (uint32_t)p.Hq) : 0, hg = h / p.heads_cta, hh = h - hg * p.heads_cta;
  const int seg = (int)(hg * p.B + b);
  const float* own = rows + ((int64_t)seg * p.heads_cta + hh) * kPiecePitch;
  const float* const pre = prefix + row * (int64_t)kPiecePitch;
  const int64_t own_step = (int64_t)p.heads_cta * kPiecePitch, pre_step = p.B * p.Hq * kPiecePitch;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int2 span = live ? __ldcg(&spans[seg]) : make_int2(0, -1);
  own += span.x * own_step;
  const int n = span.y < 0 ? 0 : span.y + p.splits;
  auto piece = [&](int i) -> const float* {
    return i < span.y ? own + i * own_step : pre + (i - span.y) * pre_step;
  };
  // this warp's share: pieces share, share + W, ...
  const int mine = n > share ? (n - share + W - 1) / W : 0;
  float4 v[kAhead];
  auto fetch = [&](int i0) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (i0 + u < mine) v[u] = __ldcg(reinterpret_cast<const float4*>(piece(share + (i0 + u) * W) + 4 * lane));
  };
  auto sums = [&](int i) {
    return i < n ? __ldcg(reinterpret_cast<const float2*>(piece(i) + kD)) : make_float2(-INFINITY, 0.f);
  };
  float2 ml = sums(lane);
  fetch(0);
  float M = ml.x;
  for (int i = lane + 32; i < n; i += 32) M = fmaxf(M, sums(i).x);
  M = warp_max(M);
  float L = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  // pieces in runs of 32, a weight a lane
  for (int i0 = 0; i0 < n; i0 += 32) {
    if (i0 > 0) ml = sums(i0 + lane);
    // no weight without tokens (l = 0); NaN logits only leave m without a value and l = NaN
    const float w = ml.y == 0.f ? 0.f : (ml.x > -1e29f ? ex2(ml.x - M) : ml.y);
    if (w != 0.f) L = fmaf(w, ml.y, L);
    const int k1 = i0 + 32 < n ? i0 + 32 : n;
    const int j0 = (i0 + W - 1 - share) / W, j1 = (k1 + W - 1 - share) / W;  // of this share
    for (int j = j0; j < j1; j += kAhead) {
      if (j > 0) fetch(j);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const float wu = __shfl_sync(0xffffffffu, w, (share + (j + u) * W) & 31);
        if (j + u >= j1 || wu == 0.f) continue;  // (its row may never have been written)
        acc.x = fmaf(wu, v[u].x, acc.x);
        acc.y = fmaf(wu, v[u].y, acc.y);
        acc.z = fmaf(wu, v[u].z, acc.z);
        acc.w = fmaf(wu, v[u].w, acc.w);
      }
    }
  }
  L = warp_sum(L);
  if (W > 1) {
    // (every warp has the whole sum)
    *reinterpret_cast<float4*>(&s_part[warp][4 * lane]) = acc;
    __syncthreads();
    if (share == 0) {
      for (int u = 1; u < W; ++u) {
        const float4 x = *reinterpret_cast<const float4*>(&s_part[warp + u][4 * lane]);
        acc.x += x.x, acc.y += x.y, acc.z += x.z, acc.w += x.w;
      }
    }
  }
  if (span.y < 0 || share != 0) return;
  const float inv = L == 0.f ? 0.f : 1.f / L;
  uint2 pk;
  pk.x = pack_pair<T>(acc.x * inv, acc.y * inv);
  pk.y = pack_pair<T>(acc.z * inv, acc.w * inv);
  *reinterpret_cast<uint2*>(out + row * (int64_t)kD + 4 * lane) = pk;
}

// ---------------------------------------------------------------------------
// Geometry.  HG: the largest divisor of Hkv up to 8; sub warps share a head.
// The fast path covers head dim 128, blocks of a multiple of 16 tokens up to 256 and
// 1, 2, 4 or 8 query heads a kv head.
// ---------------------------------------------------------------------------
PieceGeom piece_geometry(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t bs, int64_t num_blocks,
                         int64_t max_blocks, int elem, const b200_launch_cfg* cfg) {
  PieceGeom g{};
  const int64_t G = Hq / Hkv;
  if (D != kD || !(G == 1 || G == 2 || G == 4 || G == 8) || bs % 16 != 0 || bs > 256) return g;
  // 32-bit token slots and scale rows (TMA coordinates) and entry counts
  if (num_blocks * bs >= (1ll << 31) || num_blocks * Hkv >= (1ll << 31) || max_blocks * bs >= (1ll << 31)) return g;
  g.G = (int)G;
  g.HG = (cfg && cfg->rows_per_cta > 0 && cfg->rows_per_cta <= 8) ? cfg->rows_per_cta : 8;
  while (Hkv % g.HG) --g.HG;
  g.sub = kConsumers / g.HG;
  const int box = g.HG * kChunk * 128;
  g.entry_bytes = (uint32_t)(elem == 1 ? 2 * (2 * box + 1024) : 4 * box);
  g.n_hg = (int)(Hkv / g.HG);
  g.seqs = kMaxSeg / g.n_hg < B ? kMaxSeg / g.n_hg : B;
  if (g.seqs < 1 || g.n_hg * g.seqs * max_blocks >= (1ll << 31)) return g;
  g.grid = device_sm_count();
  g.pdl = cfg && (cfg->flags & 8);
  // A CTA a segment while the table bounds it to a few entries: no pieces, no join,
  // one launch less (1 sequence: of 64 tokens 8.2 us instead of 10.7, of 128 10.3 / 11.0, of 256
  // 14.3 / 11.8; 64 sequences: 64 tokens 8.7 / 17.2, 384 19.0 / 21.8, 512 23.2 / 24.4).
  const int64_t nseg = g.n_hg * B, most = 160 + 8 * nseg;
  g.whole = nseg <= g.grid && max_blocks * bs <= (most < 384 ? most : 384);
  const size_t per = g.entry_bytes + 16 + sizeof(EntryMeta);
  const size_t fixed = 1024 + 16 * 8 + (size_t)(g.n_hg * g.seqs + 1) * 4 + (size_t)g.seqs * 4 + 66 * 4 +
                       (size_t)(g.sub - 1) * g.HG * kXchPitch * 4;
  // The ring holds a multiple of sub entries, so that an entry belongs to one
  // slot: its warps have then seen each earlier filling of the entry they wait
  // for (copies complete out of order, and a wait tells only two fillings apart).
  const int unit = g.sub;
  int stages = (cfg && cfg->stages > 0) ? cfg->stages : (int)(204 * 1024 / g.entry_bytes);
  if (stages > 64) stages = 64;
  stages = stages / unit * unit;
  while (stages > unit && stages * per + fixed > kSmemMost) stages -= unit;
  if (stages < unit) stages = unit;
  if (stages < 2) stages = 2;
  g.stages = stages;
  g.smem = stages * per + fixed;
  g.fast = g.smem <= kSmemMost;
  return g;
}

// Splits of the prefix, and the SMs that stream the own pages beside it (g.grid).
// A CTA of either kernel holds its SM alone.  Measured, in us: a prefix CTA --
// (split, pair of 128-row tiles, kv head) -- takes 2.5 for a key tile (2.0 with one row
// tile) and 13 to start and end; the own pages 1.1 (8-bit: 0.8) for 128 tokens of a
// kv head and 2 a segment, over their SMs, and 10 to start and end.
// Both kernels mostly wait at their starts and ends, so side by side on an SM each
// is best where it fits (64 sequences, prefix 8192: one after the other on
// all SMs 53 us, 10 splits beside 68 SMs 40 us, 6 beside 100 48 us, 16 beside 20 67 us).
// One after the other remains where the prefix alone fills the GPU, or the own
// pages outweigh it.  Lengths live on the device: the prefix counts with its table's
// size, the own tokens with half of theirs (an own table eight times as wide as the contexts:
// 65 us instead of 38), and the streaming kernel keeps a sixteenth of the SMs.  Fewest
// splits within the minimum: each leaves a piece a row to join.
int share_sms(PieceGeom& g, int64_t Hkv, int64_t bs, int64_t max_prefix_blocks, int64_t max_blocks,
              int elem) {
  const int64_t ppt = 128 / bs, tiles = (max_prefix_blocks + ppt - 1) / ppt;
  const int64_t units = (g.seqs * g.G + 255) / 256 * Hkv;
  const int sms = g.grid;
  const double unit = elem == 1 ? 0.8 : 1.1, tile = g.seqs * g.G > 128 ? 2.5 : 2.0;
  const double own = unit / 256 * (double)(g.seqs * max_blocks * bs) * (double)Hkv + 2.0 * (double)(g.seqs * g.n_hg);
  int64_t best = 1;
  double best_cost = 1e300;
  for (int64_t s = 1; s <= tiles && s <= sms; ++s) {
    const double prefix = (double)((units * s + sms - 1) / sms) * ((double)((tiles + s - 1) / s) * tile + 13);
    const int64_t left = sms - units * s;
    const double after = prefix + own / sms + 10;
    const double beside = left * 16 >= sms ? fmax(prefix, own / (double)left + 10) : 1e300;
    const double cost = fmin(after, beside);
    if (cost < best_cost) {
      best = s, best_cost = cost;
      g.grid = beside < after ? (int)left : sms;
    }
  }
  return (int)best;
}

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// Bytes of the workspace's parts for one slice.
struct SpaceBytes {
  size_t spans, rows, prefix;
};
SpaceBytes space_bytes(const PieceGeom& g, int64_t Hq, int prefix_splits) {
  const int64_t nseg = g.n_hg * g.seqs;
  SpaceBytes s;
  s.spans = up256((size_t)nseg * sizeof(int2));
  s.rows = up256((size_t)(nseg + g.grid) * g.HG * g.G * kPiecePitch * 4);
  s.prefix = up256((size_t)prefix_splits * g.seqs * Hq * kPiecePitch * 4);
  return s;
}

template <typename T>
int launch_join(const AttnCall& a, const PieceGeom& g, const PieceSpace& w, cudaStream_t s) {
  JoinParams p{a.B, a.Hq, g.HG * g.G, w.prefix_splits, 1};
  // pieces a row, about: the grid's ranges over the segments, and the splits;
  // two or three a warp while the rows alone would not fill the SMs
  const int64_t rows = a.B * a.Hq, pieces = g.grid / (g.n_hg * a.B) + 1 + w.prefix_splits;
  while (p.W < 8 && p.W * 3 <= pieces && rows * p.W < 16 * (int64_t)device_sm_count()) p.W *= 2;
  cudaLaunchConfig_t lc = {};
  lc.gridDim = dim3((unsigned)((rows * p.W + 7) / 8));
  lc.blockDim = dim3(256);
  lc.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  lc.attrs = attr;
  lc.numAttrs = 1;
  return launch_status(cudaLaunchKernelEx(&lc, paged_attn_join_kernel<T>, (const int2*)w.spans, (const float*)w.rows,
                                          (const float*)w.prefix, static_cast<T*>(a.out), p));
}

int elem_of(const AttnCall& a) { return a.cache_dtype == B200_I8 || a.cache_dtype == B200_F8E4M3 ? 1 : 2; }

// Slice [b0, b0 + n) of a call.
AttnCall slice_of(const AttnCall& a, int64_t b0, int64_t n) {
  AttnCall c = a;
  const size_t isz = a.index_dtype == B200_I64 ? 8 : 4;
  c.B = n;
  c.q = static_cast<const char*>(a.q) + (size_t)(b0 * a.Hq * a.D) * 2;
  c.out = static_cast<char*>(a.out) + (size_t)(b0 * a.Hq * a.D) * 2;
  c.block_table = static_cast<const char*>(a.block_table) + (size_t)(b0 * a.max_blocks) * isz;
  c.context_len = static_cast<const char*>(a.context_len) + (size_t)b0 * isz;
  return c;
}

// The prefix kernel's tiles: whole pages within 128 keys.
bool prefix_fits(const PieceGeom& g, int64_t Hkv, int64_t bs, int64_t max_prefix_blocks) {
  return g.fast && bs <= 128 && Hkv <= 65535 && max_prefix_blocks * bs < (1ll << 31);
}

int attend(const AttnCall& a, const b200_launch_cfg* cfg, void* workspace, size_t workspace_bytes, cudaStream_t s) {
  PieceGeom g = piece_geometry(a.B, a.Hq, a.Hkv, a.D, a.block_size, a.num_blocks, a.max_blocks, elem_of(a), cfg);
  const bool aligned = aligned16(a.q) && aligned16(a.out) && aligned16(a.k_cache) && aligned16(a.v_cache) &&
                       aligned16(a.k_scale) && aligned16(a.v_scale);
  const bool prefix = a.prefix_table != nullptr;
  const bool fast = g.fast && aligned && (!prefix || prefix_fits(g, a.Hkv, a.block_size, a.max_prefix_blocks)) &&
                    !(cfg && (cfg->flags & 1));
  if (!fast) {
    if (a.D > 256) return B200_ERR_UNSUPPORTED;
    if (a.cache_dtype == B200_I8) return launch_attn_generic_i8(a, s);
    if (a.cache_dtype == B200_F8E4M3) return launch_attn_generic_e4m3(a, s);
    return launch_attn_generic_16(a, s);
  }
  if (prefix) g.whole = false;
  const int splits = prefix ? share_sms(g, a.Hkv, a.block_size, a.max_prefix_blocks, a.max_blocks, elem_of(a)) : 0;
  const SpaceBytes sb = space_bytes(g, a.Hq, splits);
  if (!g.whole && (workspace == nullptr || workspace_bytes < sb.spans + sb.rows + sb.prefix)) return B200_ERR_WORKSPACE;
  // (the prefix kernel stores 32 bytes of a piece row at a time; its parts and rows keep the base's alignment)
  if (prefix ? !aligned32(workspace) : !aligned16(workspace)) return B200_ERR_ALIGNMENT;
  PieceSpace w{};
  w.spans = static_cast<int2*>(workspace);
  w.rows = reinterpret_cast<float*>(static_cast<char*>(workspace) + sb.spans);
  w.prefix = reinterpret_cast<float*>(static_cast<char*>(workspace) + sb.spans + sb.rows);
  for (int64_t b0 = 0; b0 < a.B; b0 += g.seqs) {
    const AttnCall c = slice_of(a, b0, a.B - b0 < g.seqs ? a.B - b0 : g.seqs);
    PieceGeom gs = g;
    if (b0 > 0) gs.pdl = false;  // the kernel before is this call's join, which reads the workspace
    w.prefix_splits = splits;
    int st = B200_OK;
    if (prefix) {
      st = a.cache_dtype == B200_I8       ? launch_prefix_i8(c, gs, w, s)
           : a.cache_dtype == B200_F8E4M3 ? launch_prefix_e4m3(c, gs, w, s)
                                          : launch_prefix_16(c, gs, w, s);
      if (st) return st;
    }
    st = a.cache_dtype == B200_I8       ? launch_pieces_i8(c, gs, w, prefix, s)
             : a.cache_dtype == B200_F8E4M3 ? launch_pieces_e4m3(c, gs, w, prefix, s)
                                            : launch_pieces_16(c, gs, w, prefix, s);
    if (st || g.whole) return st;
    st = B200_DISPATCH_HALF(a.dtype, [&] { return launch_join<scalar_t>(c, gs, w, s); });
    if (st) return st;
  }
  return B200_OK;
}

// Checks the two entries share.
int check_call(const AttnCall& a) {
  if (a.B < 0 || a.Hq <= 0 || a.Hkv <= 0 || a.D <= 0 || a.num_blocks <= 0 || a.block_size <= 0 || a.max_blocks < 0 ||
      a.Hq % a.Hkv != 0)
    return B200_ERR_BAD_ARG;
  if (a.B == 0) return B200_OK;
  if (!a.q || !a.k_cache || !a.v_cache || !a.out || !a.context_len || (!a.block_table && a.max_blocks > 0))
    return B200_ERR_BAD_ARG;
  if (a.index_dtype != B200_I32 && a.index_dtype != B200_I64) return B200_ERR_UNSUPPORTED;
  if (a.dtype != B200_F16 && a.dtype != B200_BF16) return B200_ERR_UNSUPPORTED;
  if (a.cache_dtype == B200_I8 || a.cache_dtype == B200_F8E4M3) {
    if (!a.k_scale || !a.v_scale) return B200_ERR_BAD_ARG;
  } else if (a.cache_dtype != a.dtype) {
    return B200_ERR_UNSUPPORTED;
  }
  if (a.Hq > 65535 || a.B > (1 << 24)) return B200_ERR_UNSUPPORTED;
  return B200_OK;
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" size_t b200_paged_attention_quant_workspace_size(int64_t B, int64_t Hq, int64_t Hkv, int64_t D,
                                                            int64_t num_blocks, int64_t block_size,
                                                            int64_t max_blocks, const b200_launch_cfg* cfg) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || num_blocks <= 0 || block_size <= 0 || max_blocks <= 0 || Hq % Hkv)
    return 0;
  const PieceGeom g = piece_geometry(B, Hq, Hkv, D, block_size, num_blocks, max_blocks, 1, cfg);
  if (!g.fast || g.whole) return 0;
  const SpaceBytes sb = space_bytes(g, Hq, 0);
  return sb.spans + sb.rows + sb.prefix;
}

extern "C" int b200_paged_attention_quant(const void* q, const void* k_cache, const void* v_cache,
                                          const float* k_scale, const float* v_scale, const void* block_table,
                                          const void* context_len, void* out, int64_t B, int64_t Hq, int64_t Hkv,
                                          int64_t D, int64_t num_blocks, int64_t block_size, int64_t max_blocks,
                                          float scale, int32_t dtype, int32_t cache_dtype, int32_t index_dtype,
                                          void* workspace, size_t workspace_bytes, const b200_launch_cfg* cfg,
                                          void* stream) {
  if (int e = injected_error("paged_attention_quant")) return e;
  if (scale <= 0.f && D > 0) scale = 1.0f / sqrtf((float)D);
  const AttnCall a{q,  k_cache, v_cache, k_scale,    v_scale,    nullptr,    nullptr, block_table, context_len, out,
                   B,  Hq,      Hkv,     D,          num_blocks, block_size, max_blocks, 0,        scale,       dtype,
                   cache_dtype, index_dtype};
  if (cache_dtype != B200_I8 && cache_dtype != B200_F8E4M3) return B200_ERR_UNSUPPORTED;
  if (max_blocks <= 0) return B200_ERR_BAD_ARG;
  if (int e = check_call(a)) return e;
  if (B == 0) return B200_OK;
  return attend(a, cfg, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

extern "C" size_t b200_paged_attention_prefix_workspace_size(int64_t B, int64_t Hq, int64_t Hkv, int64_t D,
                                                             int64_t num_blocks, int64_t block_size,
                                                             int64_t max_prefix_blocks, int64_t max_blocks,
                                                             int32_t cache_dtype, const b200_launch_cfg* cfg) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || num_blocks <= 0 || block_size <= 0 || max_prefix_blocks <= 0 ||
      max_blocks < 0 || Hq % Hkv)
    return 0;
  const int elem = cache_dtype == B200_I8 || cache_dtype == B200_F8E4M3 ? 1 : 2;
  PieceGeom g = piece_geometry(B, Hq, Hkv, D, block_size, num_blocks, max_blocks, elem, cfg);
  if (!prefix_fits(g, Hkv, block_size, max_prefix_blocks)) return 0;
  const int splits = share_sms(g, Hkv, block_size, max_prefix_blocks, max_blocks, elem);
  const SpaceBytes sb = space_bytes(g, Hq, splits);
  return sb.spans + sb.rows + sb.prefix;
}

extern "C" int b200_paged_attention_prefix(const void* q, const void* k_cache, const void* v_cache,
                                           const float* k_scale, const float* v_scale, const void* prefix_table,
                                           const void* prefix_len, const void* block_table, const void* context_len,
                                           void* out, int64_t B, int64_t Hq, int64_t Hkv, int64_t D,
                                           int64_t num_blocks, int64_t block_size, int64_t max_prefix_blocks,
                                           int64_t max_blocks, float scale, int32_t dtype, int32_t cache_dtype,
                                           int32_t index_dtype, void* workspace, size_t workspace_bytes,
                                           const b200_launch_cfg* cfg, void* stream) {
  if (int e = injected_error("paged_attention_prefix")) return e;
  if (scale <= 0.f && D > 0) scale = 1.0f / sqrtf((float)D);
  const AttnCall a{q,  k_cache, v_cache, k_scale,    v_scale,    prefix_table, prefix_len, block_table, context_len,
                   out, B,      Hq,      Hkv,        D,          num_blocks,   block_size, max_blocks,
                   max_prefix_blocks, scale, dtype, cache_dtype, index_dtype};
  if (max_prefix_blocks <= 0) return B200_ERR_BAD_ARG;
  if (int e = check_call(a)) return e;
  if (B == 0) return B200_OK;
  if (!prefix_table || !prefix_len) return B200_ERR_BAD_ARG;
  return attend(a, cfg, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}
