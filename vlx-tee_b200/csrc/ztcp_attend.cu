// ztcp_attend.cu -- attention of the newest tokens over a paged cache (ztcp_attend_pages), general kernel.
//
// Mathematics.  For one row (token, head) with scores s_j = scale * q.k_j over its visible tokens j: with the
// running maximum m, p_j = 2^((s_j - m) log2 e), l = sum p_j, o = sum p_j v_j / l and lse = ln l + m.  One pass over
// K and V; a larger maximum rescales l and o.  m, l and o are fp32; p is rounded to the pool's 16-bit type for the
// second product only (l sums the unrounded p), the same half step that the output's own rounding takes.
//
// Work.  A row tile is up to 16 (token, head-of-the-group) rows of one KV head, so that a group's heads share one
// read of K and V; an item is a row tile of one sequence and KV head, a tile BK keys of it.  Items of all sequences
// form one line of tiles that the grid's CTAs share evenly (SplitSpan): a CTA's share begins and ends inside items,
// which leave partial (o, m, l) in the workspace -- at most two per CTA, whatever the lengths -- and
// attend_merge_kernel joins them in CTA order.  The split depends on the lengths and the grid alone, so results
// repeat bit for bit.
//
// A CTA is 8 warps.  K and V tiles arrive by 16-byte cp.async through a ring of stages (any page size, rows of
// masked tokens zero-filled so that whatever lies in unused rows of a page never enters a product).  QK^T: each warp
// takes 8 of the tile's keys; scores cross shared memory; each warp then holds the softmax of all keys (one quad per
// row pair) and multiplies P with its own slice of V's columns, so that no accumulator crosses warps.
#include "../../include/ztcp_kvcache.h"
#include "ztcp_kvcache.cuh"

namespace ztcp {

namespace {

constexpr int kThreads = 256;
constexpr int kRows = 16;  // rows of a row tile: one MMA row block

// ---- items and tiles ------------------------------------------------------------------------------
// Tiles of a sequence's items: every item of a sequence counts the tiles of its whole length (a row tile that sees
// fewer skips the rest), at least one, so that rows that see nothing are written too.
__device__ __forceinline__ int seq_tiles(const Seq& s, int bk) { return s.kv_len > 0 ? (s.kv_len + bk - 1) / bk : 1; }
__device__ __forceinline__ int seq_items(const CacheParams& c, const Seq& s) {
  return (int)(((int64_t)s.q_len * c.group + kRows - 1) / kRows) * c.kv_heads;
}
__device__ __forceinline__ int64_t seq_work(const CacheParams& c, int b, int bk) {
  const Seq s = load_seq(c, b);
  return (int64_t)seq_items(c, s) * seq_tiles(s, bk);
}

// A position on the line: item `item` of sequence b, tile `tile` of it, with `left` tiles to go.
struct Cursor {
  Seq s;
  int64_t left;
  int32_t b, items, tiles, item, tile;
  __device__ __forceinline__ void load(const CacheParams& c, int seq, int bk) {
    b = seq;
    s = load_seq(c, seq);
    items = seq_items(c, s);
    tiles = seq_tiles(s, bk);
  }
  __device__ __forceinline__ void next(const CacheParams& c, int bk) {
    --left;
    if (++tile < tiles) return;
    tile = 0;
    if (++item < items || left <= 0) return;
    item = 0;
    do load(c, b + 1, bk);
    while (items == 0);  // left > 0: a later sequence has tiles
  }
  // The item's KV head, first packed row and its number of rows; packed row r is token r / group, head r % group.
  __device__ __forceinline__ int head(const CacheParams& c) const { return item % c.kv_heads; }
  __device__ __forceinline__ int row(const CacheParams& c) const { return item / c.kv_heads * kRows; }
  __device__ __forceinline__ int rows(const CacheParams& c) const {
    const int n = s.q_len * c.group - row(c);
    return n < kRows ? n : kRows;
  }
  __device__ __forceinline__ int visible(const CacheParams& c) const {  // keys that any row of the item sees
    return visible_keys(c, s, (row(c) + rows(c) - 1) / c.group);
  }
};

// ---- kernel ---------------------------------------------------------------------------------------
// Shared-memory rows are padded to a multiple of 64 columns and their 16-byte chunks permuted by the row's low three
// bits, so that the eight rows of an ldmatrix lie in different banks.
__device__ __forceinline__ uint32_t chunk_at(uint32_t base, int row, int chunk, int pitch) {
  return base + row * pitch + ((chunk ^ (row & 7)) << 4);
}

// NB: 8-column blocks of V per warp (V has up to 64 * NB columns).  KSPLIT: warps that share a key block's product,
// each over a part of head_dim; a tile is 64 / KSPLIT keys.
template <bool BF16, int NB, int KSPLIT, int STAGES>
__global__ void __launch_bounds__(kThreads, NB <= 2 ? 2 : 1) attend_kernel(const __grid_constant__ AttendParams P) {
  constexpr int BK = 64 / KSPLIT;
  constexpr int SP = BK + 8;  // floats per row of the score buffer: rows 8 banks apart
  constexpr int KS = BK / 16;
  extern __shared__ __align__(128) uint8_t smem[];
  const CacheParams& c = P.c;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t4 = lane & 3;

  int64_t at;
  Spot spot;
  const SplitSpan S = locate(c.n_seqs, P.grid, [&](int b) { return seq_work(c, b, BK); }, &at, &spot);
  if (at < 0) {
    if (tid == 0) P.cuts[blockIdx.x] = Cut{};
    return;
  }
  Cursor cons;
  cons.load(c, spot.seq, BK);
  cons.item = (int32_t)((at - spot.first) / cons.tiles);
  cons.tile = (int32_t)((at - spot.first) % cons.tiles);
  cons.left = S.begin(blockIdx.x + 1) - at;
  Cursor prod = cons;

  const int pitch = (c.head_dim + 63) / 64 * 128;
  const int kbytes = BK * pitch;
  const int sbytes = c.v ? 2 * kbytes : kbytes;
  const uint32_t ring = smem_u32(smem);
  const uint32_t qbase = ring + STAGES * sbytes;
  float* const sbuf = reinterpret_cast<float*>(smem + STAGES * sbytes + kRows * pitch);
  uint8_t* const there = reinterpret_cast<uint8_t*>(sbuf + KSPLIT * kRows * SP);  // [STAGES][BK]: key in a pool page
  const uint32_t voff = c.v ? kbytes : 0;
  const int vchunk = c.v ? 0 : c.v_col / 8;
  const int chunks = c.head_dim / 8;

  // Loads the producer's tile into `stage`: 16 lanes per key, each key's pool row looked up by its lanes.
  auto issue = [&](int stage) {
    const int vis = prod.visible(c), j0 = prod.tile * BK;
    if (j0 < vis) {
      const int h = prod.head(c);
      const uint32_t base = ring + stage * sbytes;
      for (int r = tid >> 4; r < BK; r += kThreads / 16) {
        const int64_t row = j0 + r < vis ? pool_row(c, prod.b, j0 + r) : -1;
        const int64_t off = (row < 0 ? 0 : (row * c.kv_heads + h) * c.head_dim);
        if ((tid & 15) == 0) there[stage * BK + r] = row >= 0;
        for (int ch = tid & 15; ch < chunks; ch += 16) {
          cp_async16(chunk_at(base, r, ch, pitch), c.k + off + ch * 8, row >= 0);
          if (c.v) cp_async16(chunk_at(base + kbytes, r, ch, pitch), c.v + off + ch * 8, row >= 0);
        }
      }
    }
    prod.next(c, BK);
  };

  for (int i = 0; i < STAGES - 1; ++i) {
    if (prod.left > 0) issue(i);
    cp_async_commit();
  }

  float acc[NB][4], m0, m1, l0, l1;
  int lim0 = 0, lim1 = 0, vis = 0, rows = 0;
  const int nks = c.head_dim / 16;
  const int nblk = c.v_dim / 8;
  const int kb = KSPLIT == 1 ? warp : warp & (BK / 8 - 1);
  const int half = KSPLIT == 1 ? 0 : warp / (BK / 8);
  const int mid = ((nks + 1) / 2 + 1) & ~1;
  const int ks0 = half ? mid : 0, ks1 = (KSPLIT == 1 || half) ? nks : mid;

  bool fresh = true;
  bool whole = cons.tile == 0;  // the item's first tile is this CTA's
  int stage = 0;
  Cut cut = {};
  if (cons.tile > 0) cut.tiles[0] = (int32_t)(cons.left < cons.tiles - cons.tile ? cons.left : cons.tiles - cons.tile);
  while (cons.left > 0) {
    cp_async_wait<STAGES - 2>();
    __syncthreads();  // the tile has arrived; everyone is done with the stage that is refilled next
    if (prod.left > 0) issue(stage == 0 ? STAGES - 1 : stage - 1);
    cp_async_commit();

    if (fresh) {
      fresh = false;
      rows = cons.rows(c);
      vis = cons.visible(c);
      const int row = cons.row(c), h = cons.head(c);
      for (int i = tid; i < rows * chunks; i += kThreads) {
        const int r = i / chunks, ch = i - r * chunks;
        const int tok = (row + r) / c.group, gh = (row + r) - tok * c.group;
        const uint4 x = __ldg(reinterpret_cast<const uint4*>(c.q + (cons.s.row0 + tok) * c.q_token_stride +
                                                             (int64_t)(h * c.group + gh) * c.q_head_stride + ch * 8));
        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(chunk_at(qbase, r, ch, pitch)), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w) : "memory");
      }
      lim0 = g < rows ? visible_keys(c, cons.s, (row + g) / c.group) : 0;
      lim1 = g + 8 < rows ? visible_keys(c, cons.s, (row + g + 8) / c.group) : 0;
      m0 = m1 = -INFINITY;
      l0 = l1 = 0.f;
#pragma unroll
      for (int i = 0; i < NB; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
      __syncthreads();
    }

    const int j0 = cons.tile * BK;
    if (j0 < vis) {
      const uint32_t kbase = ring + stage * sbytes;
      float sc[4] = {0.f, 0.f, 0.f, 0.f};
      for (int ks = ks0; ks < ks1; ks += 2) {
        uint32_t b[4], a[4];
        ldmatrix4(b, chunk_at(kbase, kb * 8 + (lane & 7), ks * 2 + (lane >> 3), pitch));
        ldmatrix4(a, chunk_at(qbase, (lane & 7) + (lane & 8), ks * 2 + (lane >> 4), pitch));
        mma16816<BF16>(sc, a, b[0], b[1]);
        if (ks + 1 < ks1) {
          ldmatrix4(a, chunk_at(qbase, (lane & 7) + (lane & 8), ks * 2 + 2 + (lane >> 4), pitch));
          mma16816<BF16>(sc, a, b[2], b[3]);
        }
      }
      const uint8_t* const ok = there + stage * BK + kb * 8 + 2 * t4;
      if (!ok[0]) sc[0] = sc[2] = -INFINITY;
      if (!ok[1]) sc[1] = sc[3] = -INFINITY;
      float* const sw = sbuf + half * kRows * SP + kb * 8 + 2 * t4;
      *reinterpret_cast<float2*>(sw + g * SP) = make_float2(sc[0], sc[1]);
      *reinterpret_cast<float2*>(sw + (g + 8) * SP) = make_float2(sc[2], sc[3]);
      __syncthreads();

      float x0[KS][4], x1[KS][4], t0 = -INFINITY, t1 = -INFINITY;
      const float* const sr = sbuf + 2 * t4;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int col = ks * 16 + e * 8;
          float2 u = *reinterpret_cast<const float2*>(sr + g * SP + col);
          float2 w = *reinterpret_cast<const float2*>(sr + (g + 8) * SP + col);
          if constexpr (KSPLIT == 2) {
            const float2 u2 = *reinterpret_cast<const float2*>(sr + (kRows + g) * SP + col);
            const float2 w2 = *reinterpret_cast<const float2*>(sr + (kRows + g + 8) * SP + col);
            u.x += u2.x, u.y += u2.y, w.x += w2.x, w.y += w2.y;
          }
          const int j = j0 + col + 2 * t4;
          x0[ks][2 * e] = j < lim0 ? u.x * c.scale_log2 : -INFINITY;
          x0[ks][2 * e + 1] = j + 1 < lim0 ? u.y * c.scale_log2 : -INFINITY;
          x1[ks][2 * e] = j < lim1 ? w.x * c.scale_log2 : -INFINITY;
          x1[ks][2 * e + 1] = j + 1 < lim1 ? w.y * c.scale_log2 : -INFINITY;
          t0 = fmaxf(t0, fmaxf(x0[ks][2 * e], x0[ks][2 * e + 1]));
          t1 = fmaxf(t1, fmaxf(x1[ks][2 * e], x1[ks][2 * e + 1]));
        }
      t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 1));
      t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 2));
      t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 1));
      t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 2));
      t0 = fmaxf(t0, m0);
      t1 = fmaxf(t1, m1);
      const float z0 = t0 == -INFINITY ? 0.f : t0, z1 = t1 == -INFINITY ? 0.f : t1;
      const float f0 = fast_exp2(m0 - z0), f1 = fast_exp2(m1 - z1);
      m0 = t0;
      m1 = t1;
      l0 *= f0;
      l1 *= f1;
#pragma unroll
      for (int i = 0; i < NB; ++i) acc[i][0] *= f0, acc[i][1] *= f0, acc[i][2] *= f1, acc[i][3] *= f1;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x0[ks][e] = fast_exp2(x0[ks][e] - z0);
          x1[ks][e] = fast_exp2(x1[ks][e] - z1);
          l0 += x0[ks][e];
          l1 += x1[ks][e];
        }
        const uint32_t a[4] = {pack2<BF16>(x0[ks][0], x0[ks][1]), pack2<BF16>(x1[ks][0], x1[ks][1]),
                               pack2<BF16>(x0[ks][2], x0[ks][3]), pack2<BF16>(x1[ks][2], x1[ks][3])};
#pragma unroll
        for (int i = 0; i < NB; i += 2) {
          const int blk = warp * NB + i;  // value columns [8 blk, 8 blk + 16): v_dim is a multiple of 16
          if (blk < nblk) {
            uint32_t b[4];
            ldmatrix4_trans(b, chunk_at(kbase + voff, ks * 16 + (lane & 15), vchunk + blk + (lane >> 4), pitch));
            mma16816<BF16>(acc[i], a, b[0], b[1]);
            mma16816<BF16>(acc[i + 1], a, b[2], b[3]);
          }
        }
      }
    }

    const bool last = cons.tile + 1 == cons.tiles;
    if (last || cons.left == 1) {  // end of the item, or of this CTA's part of it
      l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
      l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
      l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
      l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
      const int row = cons.row(c), h = cons.head(c);
      const bool full = whole && last;
      float* const part = P.part + (int64_t)(2 * blockIdx.x + (whole ? 1 : 0)) * P.part_floats;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = g + 8 * e;
        const float m = e ? m1 : m0, l = e ? l1 : l0;
        if (r >= rows) continue;
        const int tok = (row + r) / c.group, gh = (row + r) - tok * c.group;
        const int64_t o = (cons.s.row0 + tok) * (int64_t)(c.kv_heads * c.group) + h * c.group + gh;
        const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // a NaN stays one
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          const int col = (warp * NB + i) * 8 + 2 * t4;
          if (warp * NB + i >= nblk) break;
          if (full)
            *reinterpret_cast<uint32_t*>(P.out + o * c.v_dim + col) = pack2<BF16>(acc[i][2 * e] * inv, acc[i][2 * e + 1] * inv);
          else
            *reinterpret_cast<float2*>(part + r * c.v_dim + col) = make_float2(acc[i][2 * e], acc[i][2 * e + 1]);
        }
        if (warp == 0 && t4 == 0) {
          if (!full) {
            part[P.part_rows * c.v_dim + r] = m;
            part[P.part_rows * (c.v_dim + 1) + r] = l;
          } else if (P.lse) {
            P.lse[o] = l == 0.f ? -INFINITY : fmaf(m, 0.693147180559945f, logf(l));
          }
        }
      }
      if (whole && !last) {  // the share ends inside the item
        const int64_t end = S.begin(blockIdx.x + 1), start = end - cons.tile - 1;
        cut.row0 = cons.s.row0;
        cut.row = row;
        cut.rows = rows;
        cut.head = h;
        cut.last = S.owner(start + cons.tiles - 1);
        cut.tiles[1] = cons.tile + 1;
      }
      fresh = true;
      whole = true;
    }
    cons.next(c, BK);
    stage = stage + 1 == STAGES ? 0 : stage + 1;
  }
  cp_async_wait<0>();
  if (tid == 0) P.cuts[blockIdx.x] = cut;
}

// Joins the partial results of the item that CTA x's share began and did not end (Cut): partial 1 of CTA x and
// partial 0 of the CTAs behind it.  Blocks y share its rows.  A thread holds four value columns of one row.  An item cut
// into few (a chunk's: two or three) has a thread for each, which adds up all partials; of one cut into many, the
// block's four groups of 64 threads take every fourth partial each, so that their loads are in flight together, and add
// up in shared memory in a fixed order.  (Measured, attention and join: groups for all, 281 us for five ragged chunks
// and 65.5 for the latent cache of 32 sequences cut into four to eight; a thread for all, 244 and 62; but one sequence
// of 1,021 keys cut into 19 per item 16.8 us, with groups 13.2.)
constexpr int kMergeThreads = 256, kMergeQuads = 64, kMergeFew = 16;

template <bool BF16>
__global__ void __launch_bounds__(kMergeThreads) attend_merge_kernel(const __grid_constant__ AttendParams P) {
  const CacheParams& c = P.c;
  __shared__ float s_m[4][kMergeQuads], s_l[4][kMergeQuads];
  __shared__ float4 s_o[4][kMergeQuads];
  __shared__ int s_late;
  const int tid = threadIdx.x, quad = tid & (kMergeQuads - 1), grp = tid / kMergeQuads;
  const int x = blockIdx.x;
  cudaGridDependencySynchronize();
  if (blockIdx.y == 0) {
    if (tid == 0) s_late = 0;
    __syncthreads();
    for (int i = tid; i < P.grid; i += kMergeThreads)
      if (__ldcg(&P.cuts[i].error)) s_late = 1;
    __syncthreads();
    for (int b = x * (kMergeThreads / 32) + (tid >> 5); b < c.n_seqs; b += gridDim.x * (kMergeThreads / 32)) {
      if (!s_late) write_seq_status(c, b, tid & 31);
      else if (tid % 32 == 0) c.status[b] = ZTCP_SEQ_TIMEOUT;
    }
  }
  const int rows = __ldcg(&P.cuts[x].rows);
  if (rows == 0) return;
  const Cut cut = P.cuts[x];
  const int n = cut.last - x + 1;
  auto tiles = [&](int i) { return i == 0 ? cut.tiles[1] : __ldcg(&P.cuts[x + i].tiles[0]); };
  // rounding to tiles may have left the whole item to one CTA, which has then written the result
  int some = 0;
  for (int i = tid; i < n; i += kMergeThreads) some += tiles(i) > 0;
  if (__syncthreads_count(some > 0) < 2 && __syncthreads_count(some > 1) == 0) return;
  const int64_t mo = (int64_t)P.part_rows * c.v_dim, lo = mo + P.part_rows;
  auto part = [&](int i) { return P.part + (int64_t)(2 * (x + i) + (i == 0 ? 1 : 0)) * P.part_floats; };
  const int quads = c.v_dim / 4;
  const int count = (P.tiled ? (rows + 7) / 8 * 8 : rows) * quads;
  const bool few = n <= kMergeFew;
  const int across_block = few ? kMergeThreads : kMergeQuads, first = few ? 0 : grp, by = few ? 1 : 4;
  for (int base = blockIdx.y * across_block; base < count; base += gridDim.y * across_block) {
    // rows by quads; tiled partials are read as 8 rows by 4 quads a warp, whole sectors on both sides
    const int i = base + (few ? tid : quad);
    int r, col;
    if (P.tiled) {
      const int blk = i >> 5, across = quads >> 2;
      r = blk / across * 8 + (i & 7);
      col = (blk % across * 4 + (i >> 3 & 3)) * 4;
    } else {
      r = i / quads;
      col = (i - r * quads) * 4;
    }
    const bool live = r < rows;
    if (!live) r = 0;
    float m = -INFINITY, l = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k0 = first; k0 < n; k0 += 4 * by) {  // four partials in flight
      float pm[4], pl[4];
      float4 po[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int k = k0 + by * u;
        pm[u] = -INFINITY;
        pl[u] = 0.f;
        po[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (live && k < n && tiles(k) > 0) {
          const float* const p = part(k);
          pm[u] = __ldcg(p + mo + r);
          pl[u] = __ldcg(p + lo + r);
          po[u] = __ldcg(reinterpret_cast<const float4*>(p + (P.tiled ? (int64_t)(col / 4 * P.part_rows + r) * 4 : (int64_t)r * c.v_dim + col)));
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float t = fmaxf(m, pm[u]);
        const float z = t == -INFINITY ? 0.f : t;
        const float f = fast_exp2(m - z), e = fast_exp2(pm[u] - z);
        m = t;
        l = l * f + pl[u] * e;
        a.x = a.x * f + po[u].x * e;
        a.y = a.y * f + po[u].y * e;
        a.z = a.z * f + po[u].z * e;
        a.w = a.w * f + po[u].w * e;
      }
    }
    if (!few) {
      s_m[grp][quad] = m;
      s_l[grp][quad] = l;
      s_o[grp][quad] = a;
      __syncthreads();
      if (grp == 0) {
#pragma unroll
        for (int u = 1; u < 4; ++u) m = fmaxf(m, s_m[u][quad]);
        const float z = m == -INFINITY ? 0.f : m;
        l = 0.f;
        a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float f = fast_exp2(s_m[u][quad] - z);
          const float4 o = s_o[u][quad];
          l = fmaf(s_l[u][quad], f, l);
          a.x = fmaf(o.x, f, a.x);
          a.y = fmaf(o.y, f, a.y);
          a.z = fmaf(o.z, f, a.z);
          a.w = fmaf(o.w, f, a.w);
        }
      }
      __syncthreads();
    }
    if ((few || grp == 0) && live) {
      const int tok = (cut.row + r) / c.group, gh = (cut.row + r) - tok * c.group;
      const int64_t o = (cut.row0 + tok) * (int64_t)(c.kv_heads * c.group) + cut.head * c.group + gh;
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
      *reinterpret_cast<uint2*>(P.out + o * c.v_dim + col) = make_uint2(pack2<BF16>(a.x * inv, a.y * inv), pack2<BF16>(a.z * inv, a.w * inv));
      if (col == 0 && P.lse) P.lse[o] = l == 0.f ? -INFINITY : fmaf(m, 0.693147180559945f, logf(l));
    }
  }
}

// ---- variants -------------------------------------------------------------------------------------
struct Variant {
  int bk, stages, per_sm, smem;
};

template <int NB, int KSPLIT, int STAGES>
Variant variant(const CacheParams& c) {
  const int bk = 64 / KSPLIT, pitch = (c.head_dim + 63) / 64 * 128;
  return {bk, STAGES, NB <= 2 ? 2 : 1,
          STAGES * bk * pitch * (c.v ? 2 : 1) + kRows * pitch + KSPLIT * kRows * (bk + 8) * (int)sizeof(float) + STAGES * bk};
}

// Head dims up to 128 leave room for two CTAs per SM, so that one's softmax runs under the other's products and
// loads; up to 256 for one; wider ones (single-buffer pools only) halve the tile and split head_dim between warps.
Variant pick(const CacheParams& c) {
  if (c.head_dim <= 128) return variant<2, 1, 3>(c);
  if (c.head_dim <= 256) return variant<4, 1, 3>(c);
  return variant<8, 2, 5>(c);
}

template <bool BF16, int NB, int KSPLIT, int STAGES>
void launch_kernel(const AttendParams& P, const Variant& v, cudaStream_t s) {
  auto* const k = attend_kernel<BF16, NB, KSPLIT, STAGES>;
  cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, v.smem);
  k<<<P.grid, kThreads, v.smem, s>>>(P);
}

}  // namespace

AttendShape attend_shape(const CacheParams& c, int sms) { return {sms * pick(c).per_sm, kRows, kRows * (c.v_dim + 2), 0}; }

void launch_attend(const AttendParams& P, bool bf16, cudaStream_t s) {
  const Variant v = pick(P.c);
  if (P.c.head_dim <= 128) bf16 ? launch_kernel<true, 2, 1, 3>(P, v, s) : launch_kernel<false, 2, 1, 3>(P, v, s);
  else if (P.c.head_dim <= 256) bf16 ? launch_kernel<true, 4, 1, 3>(P, v, s) : launch_kernel<false, 4, 1, 3>(P, v, s);
  else bf16 ? launch_kernel<true, 8, 2, 5>(P, v, s) : launch_kernel<false, 8, 2, 5>(P, v, s);
}

void launch_attend_merge(const AttendParams& P, bool bf16, int64_t rows, cudaStream_t s) {
  // One block per border and 64 quads of columns, at most 12 blocks a border (with 32, four ragged waves: five chunks
  // took 245 us instead of 240).  The launch overlaps the end of the kernel before it (programmatic dependent launch).
  const int64_t quads = (rows < P.part_rows ? rows : P.part_rows) * (P.c.v_dim / 4);
  int64_t y = (quads + kMergeQuads - 1) / kMergeQuads;
  if (y > 12) y = 12;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(P.grid, (unsigned)y);
  cfg.blockDim = dim3(kMergeThreads);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (bf16) cudaLaunchKernelEx(&cfg, attend_merge_kernel<true>, P);
  else cudaLaunchKernelEx(&cfg, attend_merge_kernel<false>, P);
}

}  // namespace ztcp
