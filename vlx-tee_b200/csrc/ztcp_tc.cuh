// ztcp_tc.cuh -- what the tensor-core kernels of the paged cache share: PTX wrappers, shared-memory and instruction
// descriptors, the line of items that CTAs share, and the pool's tensor maps.
#pragma once
#include <cuda.h>

#include "ztcp_kvcache.cuh"

namespace ztcp {

constexpr int kKeys = 128;                           // keys per tile
constexpr int kGroupBytes = kKeys * 128;             // a tile's 64-column group: 128 rows of 128 bytes

// Boxes of the pool's TMA loads.
struct PoolBoxes {
  int32_t rows;       // rows of one box: a page, or a tile's keys of a larger one (8 to 128, a power of two)
  int32_t shift;      // its logarithm
  int32_t pool_rows;  // rows of the tensor maps; a load at this row is filled with zeros
};

#if defined(__CUDACC__)

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
      "{\n\t.reg .pred P;\n\tmbarrier.try_wait.parity.shared.b64 P, [%1], %2;\n\tselp.u32 %0, 1, 0, P;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok;
}
// The bound of a CTA's waits, in cycles, and whether one has run out.
struct Waits {
  long long limit;
  int dead;
};
// Waits for the phase of this parity.  False when the wait ran out: here, which sets the CTA's dead flag, or in another
// role.  (A single attempt may be suspended by the hardware for tens of microseconds, so the bound is one of time.)
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile Waits* waits) {
  if (mbar_try(bar, parity)) return true;
  const long long start = clock64();
  while (!mbar_try(bar, parity)) {
    if (waits->dead) return false;
    if (clock64() - start > waits->limit) {
      waits->dead = 1;
      return false;
    }
  }
  return true;
}
// Waits for `n` fills of a ring's slots, the last ones of `pos`, whatever the other roles have come to.  A copy still in
// flight when its CTA ends would write into the next one's shared memory.
__device__ __forceinline__ void drain_fills(uint32_t bars, uint32_t slots, uint32_t pos) {
  Waits none = {kWaitCycles, 0};
  for (uint32_t p = pos > slots ? pos - slots : 0; p < pos; ++p) mbar_wait(bars + p % slots * 8, (p / slots) & 1, &none);
}
// One lane of a converged warp, always the same.  The compiler keeps the operands of what it guards in uniform
// registers, which tcgen05 instructions read (measured: 39 cycles per small product, against 44 to 53 under lane == 0).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred P;\n\telect.sync _|P, 0xffffffff;\n\tselp.u32 %0, 1, 0, P;\n\t}" : "=r"(p));
  return p;
}
// The same for a whole warp: all lanes go on, or none.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile Waits* waits) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, waits));
}
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
               "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
__device__ __forceinline__ void tma_load4(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
               "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar) : "memory");
}
__device__ __forceinline__ void tc_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// Waits for every product that this thread has issued: none may be in flight when TMEM is freed.
__device__ __forceinline__ void drain_products(uint32_t bar) {
  Waits none = {kWaitCycles, 0};
  tc_commit(bar);
  mbar_wait(bar, 0, &none);
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Matrix descriptors as their two words: the low one holds the address (in 16 bytes) and lbo and takes offsets by
// plain addition, the high one is a constant of the layout.
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.u32 p, %6, 0;\n\tmov.b64 a, {%1, %2};\n\tmov.b64 b, {%3, %4};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %5, p;\n\t}" ::"r"(d), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"((uint32_t)acc)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.u32 p, %5, 0;\n\tmov.b64 b, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d), "r"(a), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"((uint32_t)acc)
      : "memory");
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
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr) : "memory");
}
// Wait for the thread's TMEM loads; the values pass through, so that no use of them can move above the wait.
__device__ __forceinline__ void tmem_ready16(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]) : : "memory");
}
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
// groups 1,024 bytes apart, the next 64 columns `lbo` bytes on.
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo) { return ((addr & 0x3ffff) >> 4) | (lbo >> 4) << 16; }
__host__ __device__ constexpr uint32_t desc_hi(uint32_t sbo, uint32_t swizzle) { return (sbo >> 4) | 1u << 14 | swizzle << 29; }
constexpr uint32_t kSwizzle128 = 2, kSwizzle32 = 6;
// Instruction descriptor: fp32 accumulators, both operands of the pool's type.
__device__ __forceinline__ uint32_t inst_desc(bool bf16, int m, int n, bool a_mn_major, bool b_mn_major) {
  const uint32_t t = bf16 ? 1 : 0;
  return 1u << 4 | t << 7 | t << 10 | (a_mn_major ? 1u << 15 : 0u) | (b_mn_major ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24;
}

// ---- pages of the tiles to come ---------------------------------------------------------------------
// The pool rows of the next 32 boxes of a sequence, a lane each: one look at the page table serves 32 / per_tile tiles.
// (A look per tile costs the loading warp 600 to 900 cycles of a tile's 1,800 to 3,000.)
struct PageRows {
  int32_t row, t0;
  __device__ __forceinline__ void start(int t) { t0 = t - 32; }  // a new item that begins with tile t
  // Lane p, p + per_tile, ..: the row of tile t's box p; pool_rows past the sequence's end and for a page outside the pool.
  __device__ __forceinline__ int32_t at(const CacheParams& c, const PoolBoxes& box, int per_tile, int b, int kv_len, int t, int lane) {
    if ((t - t0) * per_tile >= 32) {
      t0 = t;
      const int64_t j = ((int64_t)t * per_tile + lane) << box.shift;
      row = box.pool_rows;
      if (j < kv_len) {
        const int64_t r = pool_row(c, b, (int)j);
        if (r >= 0) row = (int32_t)r;
      }
    }
    return __shfl_sync(0xffffffffu, row, (t - t0) * per_tile + (lane & (per_tile - 1)));
  }
};

// ---- the line of items ----------------------------------------------------------------------------
// Items of up to `rows` (token, head-of-the-group) rows of one sequence and KV head form one line, sequence by
// sequence, row tile by row tile, head by head, that the CTAs share evenly, in units of keys x group: an item's
// length is what its last row sees plus its own rows, which sums over row tiles in closed form.  Shares are rounded
// to tiles of KEYS keys.
struct Line {
  int64_t head;  // units of row tile 0's items, without the rows' share
  int64_t step;  // what each further row tile adds
  int32_t row_tiles, heads, rows;
  __device__ __forceinline__ int64_t cost(int rt) const { return head + (rt + 1) * step + rows; }
  __device__ __forceinline__ int64_t before(int rt) const {  // units of one head's row tiles [0, rt)
    return rt * (head + rows) + step * ((int64_t)rt * (rt + 1) / 2);
  }
  __device__ __forceinline__ int64_t total() const { return before(row_tiles) * heads; }
};
__device__ __forceinline__ Line line_of(const CacheParams& c, int rows, const Seq& s) {
  Line l;
  l.rows = rows;
  l.row_tiles = (int)div_pos((int64_t)s.q_len * c.group + rows - 1, rows);
  l.heads = c.kv_heads;
  const int64_t seen = c.causal ? (s.kv_len > s.q_len ? s.kv_len - s.q_len : 0) : s.kv_len;
  l.head = seen * c.group;
  l.step = c.causal ? rows : 0;
  return l;
}
__device__ __forceinline__ int64_t seq_work(const CacheParams& c, int rows, int b) { return line_of(c, rows, load_seq(c, b)).total(); }

// An item and the tiles [ta, tb) of its `nt` that a share [pos, end) of the line covers.
template <int KEYS>
struct Item {
  Seq s;
  Line line;
  int64_t seq_start, start, cost;
  int32_t b, rt, h, nt, ta, tb, rows, row, snap;
  bool inside;  // the share begins inside the item
  __device__ __forceinline__ void load_seq_at(const CacheParams& c, int rows_max, int seq, int64_t first) {
    b = seq;
    seq_start = first;
    s = load_seq(c, seq);
    line = line_of(c, rows_max, s);
  }
  __device__ __forceinline__ void find(const CacheParams& c, int64_t pos) {  // pos lies in sequence b
    const int64_t x = pos - seq_start;
    int lo = 0, hi = line.row_tiles - 1;  // one token per sequence: no search
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (line.before(mid) * line.heads <= x) lo = mid;
      else hi = mid - 1;
    }
    rt = lo;
    cost = line.cost(rt);
    h = (int)div_pos(x - line.before(rt) * line.heads, cost);
    start = seq_start + line.before(rt) * line.heads + h * cost;
    row = rt * line.rows;
    rows = min(s.q_len * c.group - row, line.rows);
    const int vis = visible_keys(c, s, (row + rows - 1) / c.group);
    nt = vis > 0 ? (vis + KEYS - 1) / KEYS : 1;
  }
  // The first tile of a share that begins at pos: whole tiles of keys x group before it, rounded down -- and a cut
  // that would leave fewer than `snap` tiles on a side moves to the item's end (joining a part costs as much).
  __device__ __forceinline__ int tile_at(const CacheParams& c, int64_t pos) const {
    const int64_t t = div_pos(pos - start, (int64_t)c.group * KEYS);
    return t < snap ? 0 : t > nt - snap ? nt : (int)t;
  }
  __device__ __forceinline__ void clip(const CacheParams& c, int64_t pos, int64_t end) {
    inside = pos > start;
    ta = inside ? tile_at(c, pos) : 0;
    tb = end >= start + cost ? nt : tile_at(c, end);
  }
};

// Walks the items of a share; every role of the CTA walks the same ones.
template <int KEYS>
struct Walk {
  Item<KEYS> it;
  int64_t pos, end;
  __device__ __forceinline__ void begin(const CacheParams& c, int rows, int snap, const Spot& spot, int64_t p, int64_t e) {
    pos = p;
    end = e;
    it.load_seq_at(c, rows, spot.seq, spot.first);
    it.start = it.cost = 0;  // no item yet
    it.rt = it.h = it.nt = it.ta = it.tb = it.rows = it.row = 0;
    it.inside = false;
    it.snap = snap;
  }
  __device__ __forceinline__ bool next(const CacheParams& c) {  // the next item with tiles, in `it`
    while (pos < end) {
      while (pos >= it.seq_start + it.line.total()) it.load_seq_at(c, it.line.rows, it.b + 1, it.seq_start + it.line.total());
      it.find(c, pos);
      it.clip(c, pos, end);
      pos = min(end, it.start + it.cost);
      if (it.ta < it.tb) return true;
    }
    return false;
  }
};


// The share of a CTA, found by one warp: sums every sequence's units, 32 sequences at a time, and finds the sequence
// that holds the share's first unit (-1: the share is empty).
template <class Count>
__device__ __forceinline__ SplitSpan locate_warp(int n_seqs, int grid, int lane, Count count, int64_t* want, Spot* spot) {
  auto sums = [&](int base) {  // inclusive, over the 32 sequences from `base`
    int64_t x = base + lane < n_seqs ? count(base + lane) : 0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t o = __shfl_up_sync(0xffffffffu, x, d);
      if (lane >= d) x += o;
    }
    return x;
  };
  SplitSpan S;
  S.total = 0;
  int64_t x = 0;
  for (int base = 0; base < n_seqs; base += 32) {
    x = sums(base);
    S.total += __shfl_sync(0xffffffffu, x, 31);
  }
  S.share = div_pos(S.total + grid - 1, grid);
  if (S.share == 0) S.share = 1;
  *want = S.own_begin();
  spot->seq = 0;
  spot->first = 0;
  if (*want >= 0)
    for (int base = 0; base < n_seqs; base += 32) {
      if (n_seqs > 32) x = sums(base);
      const unsigned m = __ballot_sync(0xffffffffu, *want < spot->first + x);
      if (m) {
        const int l = __ffs(m) - 1;
        const int64_t before = __shfl_sync(0xffffffffu, x, l > 0 ? l - 1 : 0);
        spot->seq = base + l;
        spot->first += l > 0 ? before : 0;
        break;
      }
      spot->first += __shfl_sync(0xffffffffu, x, 31);
    }
  return S;
}

// What the roles of a CTA need to know of an item.  The TMA warp walks the share and publishes its items through a
// small ring in shared memory, so that the walk's divisions run once and, as that warp is a ring of tiles ahead, off
// the other roles' path.
struct Job {
  int64_t row0;                          // the sequence's first row
  int32_t b, kv_len, q_len, row, rows, head;
  int32_t ta, tb;                        // tiles; ta == tb: no more items
  int32_t whole, inside;                 // all of the item's tiles; the item began before this share
};
constexpr int kJobs = 4;

template <int KEYS>
struct Publisher {
  Walk<KEYS> walk;
  Cut cut;
  uint32_t n;  // published so far
  // Publishes the next item (lane 0 of the warp writes) and keeps it in `job`; false after a timeout.
  __device__ __forceinline__ bool next(const CacheParams& c, const SplitSpan& S, Job* jobs, uint32_t full, uint32_t empty, int lane, volatile Waits* waits,
                                       Job* job) {
    Item<KEYS>& it = walk.it;
    const int64_t begin = S.begin(blockIdx.x);
    const bool have = walk.next(c);
    job->row0 = it.s.row0;
    job->b = it.b;
    job->kv_len = it.s.kv_len;
    job->q_len = it.s.q_len;
    job->row = it.row;
    job->rows = it.rows;
    job->head = it.h;
    job->ta = have ? it.ta : 0;
    job->tb = have ? it.tb : 0;
    job->whole = it.ta == 0 && it.tb == it.nt;
    job->inside = it.inside;
    if (have && it.inside) cut.tiles[0] = it.tb - it.ta;
    if (walk.pos >= walk.end && it.start >= begin && it.start + it.cost > walk.end) {  // the share ends inside the item
      cut.row0 = it.s.row0;
      cut.row = it.row;
      cut.rows = it.rows;
      cut.head = it.h;
      cut.last = S.owner(it.start + it.cost - 1);
      cut.tiles[1] = it.tb;
    }
    const uint32_t e = n % kJobs;
    if (n >= kJobs && !__all_sync(0xffffffffu, mbar_wait(empty + 8 * e, (n / kJobs - 1) & 1, waits))) return false;
    if (lane == 0) {
      jobs[e] = *job;
      mbar_arrive(full + 8 * e);
    }
    ++n;
    return true;
  }
};

// The other side, for one thread that stands for its warp.
__device__ __forceinline__ bool take_job_alone(const Job* jobs, uint32_t full, uint32_t empty, uint32_t& n, volatile Waits* waits, Job* job) {
  const uint32_t e = n % kJobs;
  if (!mbar_wait(full + 8 * e, (n / kJobs) & 1, waits)) return false;
  *job = jobs[e];
  mbar_arrive(empty + 8 * e);
  ++n;
  return true;
}
// The other side: a warp takes the next item (false after a timeout) and frees its place at once.
__device__ __forceinline__ bool take_job(const Job* jobs, uint32_t full, uint32_t empty, uint32_t& n, int lane, volatile Waits* waits, Job* job) {
  const uint32_t e = n % kJobs;
  if (!warp_wait(full + 8 * e, (n / kJobs) & 1, waits)) return false;
  *job = jobs[e];
  __syncwarp();
  if (lane == 0) mbar_arrive(empty + 8 * e);
  ++n;
  return true;
}

#endif  // __CUDACC__

// ---- host -----------------------------------------------------------------------------------------
using EncodeTiled = decltype(&cuTensorMapEncodeTiled);

inline EncodeTiled encode_tiled() {  // the driver's entry point, looked up once (the library links no libcuda)
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

// The pool as [rows][heads][head_dim], boxes of b.rows rows x one head x 64 columns.
inline bool pool_map(CUtensorMap* map, const void* pool, const CacheParams& c, bool bf16, const PoolBoxes& b) {
  const cuuint64_t dims[3] = {(cuuint64_t)c.head_dim, (cuuint64_t)c.kv_heads, (cuuint64_t)b.pool_rows};
  const cuuint64_t strides[2] = {(cuuint64_t)c.head_dim * 2, (cuuint64_t)c.kv_heads * c.head_dim * 2};
  const cuuint32_t box[3] = {64, 1, (cuuint32_t)b.rows}, elem[3] = {1, 1, 1};
  return encode_tiled()(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(pool), dims, strides,
                        box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}


// Q as [token][KV head][head of the group][head_dim], boxes of `tokens` tokens x `heads` of a group x 64 columns.
inline bool query_map(CUtensorMap* map, const CacheParams& c, bool bf16, int tokens, int heads) {
  const cuuint64_t dims[4] = {(cuuint64_t)c.head_dim, (cuuint64_t)c.group, (cuuint64_t)c.kv_heads, (cuuint64_t)c.total_rows};
  const cuuint64_t strides[3] = {(cuuint64_t)c.q_head_stride * 2, (cuuint64_t)c.q_head_stride * 2 * c.group, (cuuint64_t)c.q_token_stride * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)heads, 1, (cuuint32_t)tokens}, elem[4] = {1, 1, 1, 1};
  return encode_tiled()(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<uint16_t*>(c.q), dims, strides,
                        box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Pages must fill TMA boxes of whole swizzle groups (8 rows) that fit a tile of `keys` evenly.
inline bool pages_fit(const CacheParams& c, int keys) {
  const int T = c.page_tokens;
  return T % 8 == 0 && (T <= keys ? keys % T == 0 : T % keys == 0) && c.pool_pages * T < ((int64_t)1 << 31) && encode_tiled() != nullptr;
}
inline PoolBoxes pool_boxes(const CacheParams& c, int keys) {
  PoolBoxes b;
  b.rows = c.page_tokens < keys ? c.page_tokens : keys;
  b.shift = 0;
  while (1 << b.shift < b.rows) ++b.shift;
  b.pool_rows = (int32_t)(c.pool_pages * c.page_tokens);
  return b;
}

}  // namespace ztcp
