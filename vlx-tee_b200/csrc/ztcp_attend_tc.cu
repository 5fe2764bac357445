// ztcp_attend_tc.cu -- attention of the newest tokens over a paged cache (ztcp_attend_pages) on the 5th-generation
// tensor cores, for items of more than one MMA row block: prefill chunks, wide groups.
//
// The mathematics is that of ztcp_attend.cu.  An item is up to 256 (token, head-of-the-group) rows of one sequence
// and KV head, as two row tiles of 128: S = Q K^T and O += P V are tcgen05.mma of 128 x 128 x 16, K and V tiles of
// 128 keys arrive by TMA page by page (boxes of one page's rows, 128-byte swizzle), and S, P and O live in TMEM:
// S0 S1 O0 O1 fill its 512 columns, P overwrites the first half of its S.
//
// Warps.  0-3 and 4-7: the softmax of row tiles 0 and 1, a thread per row; 8: one thread issues the products; 9: TMA.
// The products of one row tile run under the softmax of the other:
//   tensor core   PV0(j-1) QK0(j) | PV1(j-1) QK1(j) | PV0(j) QK0(j+1) | ...
//   softmax 0                       ---- S0(j) ----
//   softmax 1                                         ---- S1(j) ----
// S_q(j) is committed after PV_q(j-1), so whoever sees S_q(j) may also change O_q.  O is rescaled only when a row's
// maximum has grown by more than 2^8 over the one in use (the weights then stay below 2^8, which the 16-bit types
// hold without loss); m, l and O are fp32.
//
// Bound.  Per 128 x 128 scores the tensor core needs 2 x 512 cycles (head_dim 128) and the exponentials 1,024 of the
// 16-per-cycle unit, so the two take turns at being the limit; a share of the exponentials is computed by a
// polynomial on the FMA pipes instead (exp2_poly).
//
// Work.  As in ztcp_attend.cu the items form one line that the CTAs (one per SM) share evenly, in units of
// keys x group: an item's length is what its last row sees plus its own rows, which sums over row tiles in closed
// form.  Shares are rounded to tiles.  attend_tc_merge_kernel joins items that several CTAs share.
//
// Waits are bounded: a wait that does not end within about two seconds sets the CTA's error word, every role leaves
// its loop, copies and products in flight are waited for (bounded again), TMEM is freed, and the merge kernel
// reports ZTCP_SEQ_TIMEOUT for every sequence.
#include <cuda.h>

#include "../../include/ztcp_kvcache.h"
#include "ztcp_kvcache.cuh"

namespace ztcp {

namespace {

constexpr int kRowTile = 128;
constexpr int kItemRows = 256;
constexpr int kKeys = 128;  // keys per tile
constexpr int kThreads = 320;
constexpr int kMmaWarp = 8, kTmaWarp = 9;
constexpr long long kWaitCycles = 4000000000ll;  // about two seconds

struct TcParams {
  AttendParams a;
  int32_t box_rows;   // rows of one TMA box: a page, or 128 of a larger one (8 to 128, a power of two)
  int32_t box_shift;  // its logarithm
  int64_t pool_rows;  // rows of the tensor maps; a load at this row is filled with zeros
};

// ---- PTX ------------------------------------------------------------------------------------------
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok;
}
// False when the wait ran out, here or (dead set) elsewhere in the CTA.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* dead) {
  if (mbar_try(bar, parity)) return true;
  const long long start = clock64();
  while (!mbar_try(bar, parity)) {
    if (*dead) return false;
    if (clock64() - start > kWaitCycles) {
      *dead = 1;
      return false;
    }
  }
  return true;
}
// The same for a whole warp: all lanes go on, or none.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* dead) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, dead));
}
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
               "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
__device__ __forceinline__ void tc_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a),
               "l"(b), "r"(idesc), "r"((uint32_t)acc) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a),
               "l"(b), "r"(idesc), "r"((uint32_t)acc) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,"
      "%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
        "=r"(r[31])
      : "r"(addr) : "memory");
}
// Waits for the thread's TMEM loads; the values pass through, so that no use of them can move above the wait.
__device__ __forceinline__ void tmem_ready32(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), 
               "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]) : : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,"
      "%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
      "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

// Shared-memory matrix descriptor, 128-byte swizzle, descriptor version 1.  K-major operands (Q, K: 64 columns per
// 128-byte row): 8-row groups 1,024 bytes apart.  MN-major operand (V: 64 output columns per row of a key): 8-key
// groups 1,024 bytes apart, the next 64 columns one half tile (16 KB) on.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  return (uint64_t)((addr & 0x3ffff) >> 4) | (uint64_t)(lbo >> 4) << 16 | (uint64_t)(sbo >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// Instruction descriptor: fp32 accumulators, both operands of the pool's type, M = 128.
__device__ __forceinline__ uint32_t inst_desc(bool bf16, int n, bool b_mn_major) {
  const uint32_t t = bf16 ? 1 : 0;
  return 1u << 4 | t << 7 | t << 10 | (b_mn_major ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 | (uint32_t)(kRowTile >> 4) << 24;
}

// ---- the line of items ----------------------------------------------------------------------------
struct Line {
  int64_t head;  // units of row tile 0's items, without the rows' share
  int64_t step;  // what each further row tile adds
  int32_t row_tiles, heads;
  __device__ __forceinline__ int64_t cost(int rt) const { return head + (rt + 1) * step + kItemRows; }
  __device__ __forceinline__ int64_t before(int rt) const {  // units of one head's row tiles [0, rt)
    return rt * (head + kItemRows) + step * ((int64_t)rt * (rt + 1) / 2);
  }
  __device__ __forceinline__ int64_t total() const { return before(row_tiles) * heads; }
};
__device__ __forceinline__ Line line_of(const CacheParams& c, const Seq& s) {
  Line l;
  l.row_tiles = (int)(((int64_t)s.q_len * c.group + kItemRows - 1) / kItemRows);
  l.heads = c.kv_heads;
  const int64_t seen = c.causal ? (s.kv_len > s.q_len ? s.kv_len - s.q_len : 0) : s.kv_len;
  l.head = seen * c.group;
  l.step = c.causal ? kItemRows : 0;
  return l;
}
__device__ __forceinline__ int64_t seq_work(const CacheParams& c, int b) { return line_of(c, load_seq(c, b)).total(); }

// An item and the tiles [ta, tb) of its `nt` that a share [pos, end) of the line covers.
struct Item {
  Seq s;
  Line line;
  int64_t seq_start, start, cost;
  int32_t b, rt, h, nt, ta, tb, rows, row;
  bool inside;  // the share begins inside the item
  __device__ __forceinline__ void load_seq_at(const CacheParams& c, int seq, int64_t first) {
    b = seq;
    seq_start = first;
    s = load_seq(c, seq);
    line = line_of(c, s);
  }
  __device__ __forceinline__ void find(const CacheParams& c, int64_t pos) {  // pos lies in sequence b
    const int64_t x = pos - seq_start;
    int lo = 0, hi = line.row_tiles - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (line.before(mid) * line.heads <= x) lo = mid;
      else hi = mid - 1;
    }
    rt = lo;
    cost = line.cost(rt);
    h = (int)((x - line.before(rt) * line.heads) / cost);
    start = seq_start + line.before(rt) * line.heads + h * cost;
    row = rt * kItemRows;
    rows = min(s.q_len * c.group - row, kItemRows);
    const int vis = visible_keys(c, s, (row + rows - 1) / c.group);
    nt = vis > 0 ? (vis + kKeys - 1) / kKeys : 1;
  }
  __device__ __forceinline__ int tile_at(int64_t pos) const { return (int)((pos - start) * nt / cost); }
  __device__ __forceinline__ void clip(int64_t pos, int64_t end) {
    inside = pos > start;
    ta = tile_at(pos);
    tb = end >= start + cost ? nt : tile_at(end);
  }
};

// Walks the items of a share; every role of the CTA walks the same ones.
struct Walk {
  Item it;
  int64_t pos, end;
  __device__ __forceinline__ void begin(const CacheParams& c, const Spot& spot, int64_t p, int64_t e) {
    pos = p;
    end = e;
    it.load_seq_at(c, spot.seq, spot.first);
  }
  __device__ __forceinline__ bool next(const CacheParams& c) {  // the next item with tiles, in `it`
    while (pos < end) {
      while (pos >= it.seq_start + it.line.total()) it.load_seq_at(c, it.b + 1, it.seq_start + it.line.total());
      it.find(c, pos);
      it.clip(pos, end);
      pos = min(end, it.start + it.cost);
      if (it.ta < it.tb) return true;
    }
    return false;
  }
};

// ---- softmax arithmetic ---------------------------------------------------------------------------
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t r, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

constexpr int kMaxGrid = 1024;
constexpr int kBars = 32;  // barrier slots at the start of shared memory

template <bool BF16, int HALVES, int SLOTS>
__global__ void __launch_bounds__(kThreads, 1)
attend_tc_kernel(const __grid_constant__ TcParams P, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  constexpr int kHalf = kKeys * 128;           // bytes of 128 rows x 64 columns
  constexpr int kTile = HALVES * kHalf;        // a K or V tile, or a Q row tile
  constexpr int kCols = HALVES * 64;           // head_dim rounded up
  extern __shared__ uint8_t smem_raw[];
  __shared__ int dead_s;
  __shared__ uint32_t tmem_s;
  const CacheParams& c = P.a.c;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  volatile int* const dead = &dead_s;

  // barriers first, then the 1,024-byte aligned tiles
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t bars = raw;
  const uint32_t tiles = (raw + kBars * 8 + 1023) & ~1023u;
  const uint32_t qtile = tiles, ring = tiles + 2 * kTile;
  auto full = [&](int s) { return bars + s * 8; };
  auto empty = [&](int s) { return bars + (SLOTS + s) * 8; };
  const uint32_t q_full = bars + 2 * SLOTS * 8, s_full = q_full + 16, p_full = s_full + 16, o_full = p_full + 16, drain = o_full + 16;
  static_assert(2 * SLOTS + 9 <= kBars, "barrier slots");

  int64_t at;
  Spot spot;
  const SplitSpan S = locate(c.n_seqs, P.a.grid, [&](int b) { return seq_work(c, b); },
                             [&](const SplitSpan& s) { return blockIdx.x < s.n ? s.begin(blockIdx.x) : (int64_t)-1; }, &at, &spot);
  int32_t* const err = reinterpret_cast<int32_t*>(P.a.part) + blockIdx.x;
  if (at < 0) {
    if (tid == 0) *err = 0;
    return;
  }
  if (tid == 0) {
    dead_s = 0;
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int q = 0; q < 2; ++q) {
      mbar_init(q_full + 8 * q, 128);
      mbar_init(s_full + 8 * q, 1);
      mbar_init(p_full + 8 * q, 128);
      mbar_init(o_full + 8 * q, 1);
    }
    mbar_init(drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_s)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_s;

  Walk walk;
  walk.begin(c, spot, at, S.begin(blockIdx.x + 1));

  if (warp == kTmaWarp) {
    // ---- TMA: K and V tiles in turn through the ring; lane p fetches page p of the tile ------------
    const int per_tile = kKeys / P.box_rows;
    uint32_t pos = 0;  // tiles so far: K of step t is 2 t, V is 2 t + 1
    bool ok = true;
    while (ok && walk.next(c)) {
      const Item& it = walk.it;
      for (int t = it.ta; ok && t < it.tb; ++t) {
        const int j = t * kKeys + lane * P.box_rows;
        int64_t row = P.pool_rows;  // past the sequence's end, or a bad page: zeros
        if (lane < per_tile && j < it.s.kv_len) {
          const int64_t r = pool_row(c, it.b, j);
          if (r >= 0) row = r;
        }
#pragma unroll
        for (int kv = 0; kv < 2; ++kv, ++pos) {
          const int slot = pos % SLOTS;
          ok = ok && (pos < SLOTS || mbar_wait(empty(slot), (pos / SLOTS - 1) & 1, dead));
          if (!__all_sync(0xffffffffu, ok)) {
            ok = false;
            break;
          }
          if (lane == 0) mbar_expect(full(slot), kTile);
          __syncwarp();
          if (lane < per_tile)
#pragma unroll
            for (int x = 0; x < HALVES; ++x)
              tma_load(ring + slot * kTile + x * kHalf + lane * P.box_rows * 128, kv ? &vmap : &kmap, x * 64, it.h, (int)row, full(slot));
        }
      }
    }
    // after a timeout: no copy may be in flight when the CTA ends
    if (*dead) {
      int none = 0;
      for (uint32_t p = pos > SLOTS ? pos - SLOTS : 0; p < pos; ++p) mbar_wait(full(p % SLOTS), (p / SLOTS) & 1, &none);
    }
  } else if (warp == kMmaWarp) {
    // ---- products ----------------------------------------------------------------------------------
    if (lane == 0) {
      const uint32_t qk = inst_desc(BF16, kKeys, false), pv = inst_desc(BF16, kCols, true);
      const int ksteps = (c.head_dim + 15) / 16;
      uint32_t step = 0;                      // tiles so far
      uint32_t items0 = 0, items1 = 0;        // items so far, per row tile
      uint32_t softs0 = 0, softs1 = 0;        // tiles so far, per row tile
      bool ok = true, have = walk.next(c);
      int nq = 0;
      auto scores = [&](int q, uint32_t st) {  // S_q = Q_q K^T of step st
        const uint32_t kb = ring + (2 * st % SLOTS) * kTile, qb = qtile + q * kTile;
        for (int k = 0; k < ksteps; ++k) {
          const uint32_t off = (k >> 2) * kHalf + (k & 3) * 32;
          mma_ss(tmem + q * 128, smem_desc(qb + off, 16, 1024), smem_desc(kb + off, 16, 1024), qk, k > 0);
        }
        tc_commit(s_full + 8 * q);
      };
      auto wait = [&](uint32_t bar, uint32_t n) {  // the n-th completion (from 0)
        ok = ok && mbar_wait(bar, n & 1, dead);
        return ok;
      };
      if (have) {  // the first step's scores
        nq = walk.it.rows > kRowTile ? 2 : 1;
        if (wait(full(0), 0)) {
          for (int q = 0; q < nq; ++q)
            if (wait(q_full + 8 * q, 0)) {
              tc_fence_after();
              scores(q, 0);
            }
          tc_commit(empty(0));
        }
      }
      while (ok && have) {
        const int n = walk.it.tb - walk.it.ta;
        const int cur = nq;
        bool more = false;
        for (int t = 0; ok && t < n; ++t, ++step) {
          const bool last = t + 1 == n;
          if (last) {
            more = walk.next(c);
            nq = more ? (walk.it.rows > kRowTile ? 2 : 1) : 0;
          }
          const bool nxt = !last || more;
          const uint32_t vp = 2 * step + 1, kp = vp + 1;
          if (!wait(full(vp % SLOTS), vp / SLOTS)) break;
          bool k_there = false;
          for (int q = 0; ok && q < 2; ++q) {
            if (q < cur) {
              if (!wait(p_full + 8 * q, q ? softs1 : softs0)) break;
              if (q) ++softs1;
              else ++softs0;
              tc_fence_after();
              const uint32_t vb = ring + (vp % SLOTS) * kTile;
              for (int k = 0; k < kKeys / 16; ++k)
                mma_ts(tmem + 256 + q * 128, tmem + q * 128 + k * 8, smem_desc(vb + k * 2048, kHalf, 1024), pv, t > 0 || k > 0);
              if (last) {
                tc_commit(o_full + 8 * q);
                if (q) ++items1;
                else ++items0;
              }
            }
            if (nxt && q < nq) {
              if (!k_there) {
                if (!wait(full(kp % SLOTS), kp / SLOTS)) break;
                k_there = true;
              }
              if (last && !wait(q_full + 8 * q, q ? items1 : items0)) break;
              tc_fence_after();
              scores(q, step + 1);
            }
          }
          if (!ok) break;
          tc_commit(empty(vp % SLOTS));
          if (nxt) tc_commit(empty(kp % SLOTS));
        }
        have = more;
      }
      if (*dead) {  // no product may be in flight when TMEM is freed
        int none = 0;
        tc_commit(drain);
        mbar_wait(drain, 0, &none);
      }
    }
    __syncwarp();
  } else {
    // ---- softmax of row tile q: a thread per row -----------------------------------------------------
    const int q = warp >> 2, wg = tid & 127;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;
    const uint32_t ts = tmem + lanes + q * 128, to = tmem + lanes + 256 + q * 128;
    const uint32_t qdst = qtile + q * kTile + wg * 128;
    const int chunks = c.head_dim / 8;
    uint32_t step = 0, mine = 0, done = 0;  // tiles of the CTA, tiles and items of this row tile
    // Item's row of this thread -> shared memory (rows past the item's end: the last one, results unused)
    auto load_q = [&](const Item& it) {
      const int r = it.row + min(q * kRowTile + wg, it.rows - 1);
      const int tok = r / c.group, gh = r - tok * c.group;
      const uint16_t* const src = c.q + (it.s.row0 + tok) * c.q_token_stride + (int64_t)(it.h * c.group + gh) * c.q_head_stride;
      for (int x = 0; x < kCols / 8; ++x) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (x < chunks) v = __ldg(reinterpret_cast<const uint4*>(src) + x);
        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(qdst + (x >> 3) * kHalf + (((x & 7) ^ (wg & 7)) << 4)), "r"(v.x), "r"(v.y),
                     "r"(v.z), "r"(v.w) : "memory");
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(q_full + 8 * q);
    };
    bool have = walk.next(c), ok = true;
    if (have && (q == 0 || walk.it.rows > kRowTile)) load_q(walk.it);
    while (ok && have) {
      Item it = walk.it;
      const int n = it.tb - it.ta;
      if (q == 1 && it.rows <= kRowTile) {  // nothing in this row tile
        step += n;
        have = walk.next(c);
        if (have && walk.it.rows > kRowTile) load_q(walk.it);
        continue;
      }
      const int r = q * kRowTile + wg;
      const int lim = r < it.rows ? visible_keys(c, it.s, (it.row + r) / c.group) : 0;
      float m = -INFINITY, l = 0.f;
      for (int t = it.ta; t < it.tb; ++t, ++step, ++mine) {
        const int j0 = t * kKeys;
        // pages of this tile outside the pool count as masked
        unsigned bad = 0;
        {
          const int j = j0 + lane * P.box_rows;
          const bool b = lane < kKeys / P.box_rows && j < it.s.kv_len && pool_row(c, it.b, j) < 0;
          bad = __ballot_sync(0xffffffffu, b);
        }
        if (!(ok = warp_wait(s_full + 8 * q, mine & 1, dead))) break;
        tc_fence_after();
        uint32_t x[128];
#pragma unroll
        for (int i = 0; i < 4; ++i) tmem_ld32(ts + i * 32, x + i * 32);
#pragma unroll
        for (int i = 0; i < 4; ++i) tmem_ready32(x + i * 32);
        if (!__all_sync(0xffffffffu, lim >= j0 + kKeys) || bad) {
#pragma unroll
          for (int i = 0; i < 128; ++i)
            if (j0 + i >= lim || (bad >> (i >> P.box_shift) & 1)) x[i] = 0xff800000u;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 128; i += 2) mx = fmaxf(mx, fmaxf(__uint_as_float(x[i]), __uint_as_float(x[i + 1])));
        mx *= c.scale_log2;
        const bool grow = mx > m + 8.f || (m == -INFINITY && mx > -INFINITY);
        if (__any_sync(0xffffffffu, grow)) {
          const float mn = grow ? mx : m;
          const float f = grow ? fast_exp2(m - mn) : 1.f;  // 0 for the first maximum
          if (t > it.ta) {
            uint32_t o[32];
#pragma unroll 1
            for (int i = 0; i < HALVES * 2; ++i) {
              tmem_ld32(to + i * 32, o);
              tmem_ready32(o);
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st32(to + i * 32, o);
            }
          }
          l *= f;
          m = mn;
        }
        const float z = m == -INFINITY ? 0.f : -m;
        const uint64_t sc2 = pair(c.scale_log2, c.scale_log2), z2 = pair(z, z);
        uint64_t sum = pair(0.f, 0.f), sum1 = pair(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < 128; i += 4) {
          float a, b, d, e;
          unpair(fma2(pair(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), sc2, z2), a, b);
          unpair(fma2(pair(__uint_as_float(x[i + 2]), __uint_as_float(x[i + 3])), sc2, z2), d, e);
          a = fast_exp2(a);
          b = fast_exp2(b);
          d = fast_exp2(d);
          e = fast_exp2(e);
          sum = add2(sum, pair(a, b));
          sum1 = add2(sum1, pair(d, e));
          x[i / 2] = pack2<BF16>(a, b);
          x[i / 2 + 1] = pack2<BF16>(d, e);
        }
        tmem_st32(ts, x);
        tmem_st32(ts + 32, x + 32);
        float s0, s1, s2, s3;
        unpair(sum, s0, s1);
        unpair(sum1, s2, s3);
        l += (s0 + s1) + (s2 + s3);
        // rows of V past the sequence's end lie in its last page and may hold anything: zero them for 0 * V
        const int end = it.s.kv_len - j0;
        if (q == 0 && end < kKeys && it.s.kv_len % c.page_tokens != 0) {
          const uint32_t vp = 2 * step + 1;
          if (!(ok = warp_wait(full(vp % SLOTS), (vp / SLOTS) & 1, dead))) break;
          if (wg >= end)
#pragma unroll
            for (int i = 0; i < HALVES * 8; ++i)
              asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(ring + (vp % SLOTS) * kTile + (i >> 3) * kHalf + wg * 128 + (i & 7) * 16),
                           "r"(0) : "memory");
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        tc_wait_st();
        tc_fence_before();
        mbar_arrive(p_full + 8 * q);
      }
      if (!ok) break;
      have = walk.next(c);
      if (have && (q == 0 || walk.it.rows > kRowTile)) load_q(walk.it);  // the item's last QK^T has been seen

      if (!(ok = warp_wait(o_full + 8 * q, done & 1, dead))) break;
      ++done;
      tc_fence_after();
      const bool whole = it.ta == 0 && it.tb == it.nt;
      const int tok = (it.row + r) / c.group, gh = (it.row + r) - tok * c.group;
      const int64_t o = (it.s.row0 + tok) * (int64_t)(c.kv_heads * c.group) + it.h * c.group + gh;
      float* const part = P.a.part + gridDim.x + (int64_t)(2 * blockIdx.x + (it.inside ? 0 : 1)) * P.a.part_floats;
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
#pragma unroll 1
      for (int i = 0; i < HALVES * 2; ++i) {
        uint32_t v[32];
        tmem_ld32(to + i * 32, v);
        tmem_ready32(v);
        if (r < it.rows) {
          if (whole) {
#pragma unroll
            for (int e = 0; e < 32; e += 8)
              if (i * 32 + e < c.v_dim) {
                uint4 w;
                w.x = pack2<BF16>(__uint_as_float(v[e]) * inv, __uint_as_float(v[e + 1]) * inv);
                w.y = pack2<BF16>(__uint_as_float(v[e + 2]) * inv, __uint_as_float(v[e + 3]) * inv);
                w.z = pack2<BF16>(__uint_as_float(v[e + 4]) * inv, __uint_as_float(v[e + 5]) * inv);
                w.w = pack2<BF16>(__uint_as_float(v[e + 6]) * inv, __uint_as_float(v[e + 7]) * inv);
                *reinterpret_cast<uint4*>(P.a.out + o * c.v_dim + i * 32 + e) = w;
              }
          } else {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              if (i * 32 + e < c.v_dim) *reinterpret_cast<uint4*>(part + r * c.v_dim + i * 32 + e) = make_uint4(v[e], v[e + 1], v[e + 2], v[e + 3]);
          }
        }
      }
      tc_fence_before();
      if (r < it.rows) {
        if (!whole) {
          part[kItemRows * c.v_dim + r] = m;
          part[kItemRows * (c.v_dim + 1) + r] = l;
        } else if (P.a.lse) {
          P.a.lse[o] = l == 0.f ? -INFINITY : fmaf(m, 0.693147180559945f, logf(l));
        }
      }
    }
  }
  __syncthreads();
  if (tid == 0) *err = *dead;
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// Joins the partial results of each item that several CTAs share, and writes the sequences' status.  Block x looks
// at the border between CTAs x and x + 1 and takes the item cut there if this is its first border; blocks y share
// its rows.
template <bool BF16>
__global__ void __launch_bounds__(256) attend_tc_merge_kernel(const __grid_constant__ TcParams P) {
  const CacheParams& c = P.a.c;
  __shared__ int late;
  int64_t w;
  Spot spot;
  if (threadIdx.x == 0) late = 0;
  const SplitSpan S = locate(c.n_seqs, P.a.grid, [&](int b) { return seq_work(c, b); },
                             [&](const SplitSpan& s) { return (int)blockIdx.x + 1 < s.n ? s.begin(blockIdx.x + 1) : (int64_t)-1; }, &w, &spot);
  cudaGridDependencySynchronize();
  if (blockIdx.y == 0) {
    for (int i = threadIdx.x; i < P.a.grid; i += blockDim.x)
      if (__ldcg(reinterpret_cast<const int32_t*>(P.a.part) + i)) late = 1;
    __syncthreads();
    for (int b = blockIdx.x * 8 + (threadIdx.x >> 5); b < c.n_seqs; b += gridDim.x * 8) {
      if (!late) write_seq_status(c, b, threadIdx.x & 31);
      else if (threadIdx.x % 32 == 0) c.status[b] = ZTCP_SEQ_TIMEOUT;
    }
  }
  if (w < 0) return;
  Item it;
  it.load_seq_at(c, spot.seq, spot.first);
  it.find(c, w);
  if (w == it.start || S.begin(blockIdx.x) > it.start) return;
  const int c0 = blockIdx.x, c1 = S.owner(it.start + it.cost - 1);
  const int64_t mo = (int64_t)kItemRows * c.v_dim, lo = mo + kItemRows;  // m, then l, behind the rows
  const float* const base = P.a.part + P.a.grid;
  auto part = [&](int cta) { return base + (int64_t)(2 * cta + (S.begin(cta) > it.start ? 0 : 1)) * P.a.part_floats; };
  auto tiles = [&](int cta) {  // of the item, in the CTA's share
    Item x = it;
    x.clip(max(S.begin(cta), it.start), S.begin(cta + 1));
    return x.tb - x.ta;
  };
  __shared__ uint8_t has[kMaxGrid];
  __shared__ int single;
  if (threadIdx.x == 0) single = 0;
  __syncthreads();
  for (int k = c0 + threadIdx.x; k <= c1; k += blockDim.x) {
    const int n = tiles(k);
    has[k - c0] = n > 0;
    if (n == it.nt) single = 1;
  }
  __syncthreads();
  if (single) return;  // rounding left all tiles to one CTA, which has written the result
  const int rows = it.rows, row = it.row, h = it.h;
  const int quarter = c.v_dim / 4;
  for (int i = blockIdx.y * blockDim.x + threadIdx.x; i < rows * quarter; i += gridDim.y * blockDim.x) {
    const int r = i / quarter, col = (i - r * quarter) * 4;
    float m = -INFINITY;
    for (int k = c0; k <= c1; ++k)
      if (has[k - c0]) m = fmaxf(m, __ldcg(part(k) + mo + r));
    const float z = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = c0; k <= c1; ++k) {
      if (!has[k - c0]) continue;
      const float* const p = part(k);
      const float f = fast_exp2(__ldcg(p + mo + r) - z);
      const float4 o = __ldcg(reinterpret_cast<const float4*>(p + (int64_t)r * c.v_dim + col));
      l = fmaf(__ldcg(p + lo + r), f, l);
      a.x = fmaf(o.x, f, a.x);
      a.y = fmaf(o.y, f, a.y);
      a.z = fmaf(o.z, f, a.z);
      a.w = fmaf(o.w, f, a.w);
    }
    const int tok = (row + r) / c.group, gh = (row + r) - tok * c.group;
    const int64_t o = (it.s.row0 + tok) * (int64_t)(c.kv_heads * c.group) + h * c.group + gh;
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
    *reinterpret_cast<uint2*>(P.a.out + o * c.v_dim + col) = make_uint2(pack2<BF16>(a.x * inv, a.y * inv), pack2<BF16>(a.z * inv, a.w * inv));
    if (col == 0 && P.a.lse) P.a.lse[o] = l == 0.f ? -INFINITY : fmaf(m, 0.693147180559945f, logf(l));
  }
}

// ---- host -----------------------------------------------------------------------------------------
using EncodeTiled = decltype(&cuTensorMapEncodeTiled);

EncodeTiled encode_tiled() {  // the driver's entry point, looked up once (the library links no libcuda)
  static const EncodeTiled f = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &r) != cudaSuccess ||
        r != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return f;
}

// The pool as [rows][heads][head_dim], boxes of box_rows rows x one head x 64 columns.
bool pool_map(CUtensorMap* map, const void* pool, const CacheParams& c, bool bf16, int box_rows, int64_t pool_rows) {
  const cuuint64_t dims[3] = {(cuuint64_t)c.head_dim, (cuuint64_t)c.kv_heads, (cuuint64_t)pool_rows};
  const cuuint64_t strides[2] = {(cuuint64_t)c.head_dim * 2, (cuuint64_t)c.kv_heads * c.head_dim * 2};
  const cuuint32_t box[3] = {64, 1, (cuuint32_t)box_rows}, elem[3] = {1, 1, 1};
  return encode_tiled()(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(pool), dims, strides,
                        box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool BF16, int HALVES, int SLOTS>
void launch_kernel(const TcParams& P, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t s) {
  auto* const f = attend_tc_kernel<BF16, HALVES, SLOTS>;
  const int smem = kBars * 8 + 1024 + (2 + SLOTS) * HALVES * kKeys * 128;
  cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  f<<<P.a.grid, kThreads, smem, s>>>(P, k, v);
}

}  // namespace

// Pages must fill TMA boxes of whole swizzle groups (8 rows) that fit a tile of 128 keys evenly.
bool attend_tc_fits(const CacheParams& c) {
  const int T = c.page_tokens;
  return c.v && c.head_dim <= 128 && T % 8 == 0 && (T <= kKeys ? kKeys % T == 0 : T % kKeys == 0) && c.pool_pages * T < ((int64_t)1 << 31) &&
         encode_tiled() != nullptr;
}

int64_t attend_tc_workspace(const CacheParams& c, AttendParams* P) {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  P->grid = (sms < kMaxGrid ? sms : kMaxGrid) / 4 * 4;  // the error words in front of the partials keep these 16-byte aligned
  P->part_rows = kItemRows;
  P->part_floats = kItemRows * (c.v_dim + 2);
  return ((int64_t)P->grid + (int64_t)P->grid * 2 * P->part_floats) * (int64_t)sizeof(float);
}

bool launch_attend_tc(const AttendParams& A, bool bf16, cudaStream_t s) {
  TcParams P;
  P.a = A;
  P.box_rows = A.c.page_tokens < kKeys ? A.c.page_tokens : kKeys;
  P.box_shift = 0;
  while (1 << P.box_shift < P.box_rows) ++P.box_shift;
  P.pool_rows = A.c.pool_pages * A.c.page_tokens;
  CUtensorMap k, v;
  if (!pool_map(&k, A.c.k, A.c, bf16, P.box_rows, P.pool_rows) || !pool_map(&v, A.c.v, A.c, bf16, P.box_rows, P.pool_rows)) return false;
  if (A.c.head_dim <= 64) bf16 ? launch_kernel<true, 1, 8>(P, k, v, s) : launch_kernel<false, 1, 8>(P, k, v, s);
  else bf16 ? launch_kernel<true, 2, 5>(P, k, v, s) : launch_kernel<false, 2, 5>(P, k, v, s);
  if (cudaPeekAtLastError() != cudaSuccess) return true;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(P.a.grid > 1 ? P.a.grid - 1 : 1, 8);
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (bf16) cudaLaunchKernelEx(&cfg, attend_tc_merge_kernel<true>, P);
  else cudaLaunchKernelEx(&cfg, attend_tc_merge_kernel<false>, P);
  return true;
}

}  // namespace ztcp
