// ztcp_mass_tc.cu -- attention weight per page (ztcp_page_mass) on the 5th-generation tensor cores.
//
// The mathematics is that of ztcp_mass.cu: weights exp(scale * q.k - lse) summed over rows, heads and a page's keys.
//   S^T[128 keys, N rows] = K Q^T   (tcgen05.mma, keys on the 128 lanes)
// puts a key's weights into one thread, which adds them up over the columns; a warp's 32 keys (or a smaller page's)
// are then one segment, whose sum goes to the workspace per KV head.  With 256 rows the product is turned over,
//   S[2 x 128 rows, 128 keys] = Q K^T   (rows on the lanes)
// so that a thread's lse is a register (read from shared memory for every column it took the bandwidth that the
// products need: 87 us against 80, before the join got faster, for windows of 64 tokens of four sequences, 32 heads over
// 84,800 keys); a warp adds its 32 rows up by shuffles, segment by segment.  page_mass_join_kernel adds a page's segments
// and heads in a fixed order, so there are no atomics and results repeat bit for bit.
//
// Accuracy.  The exponent is formed as fma(s, scale, -lse) -- one rounding of a value that is small wherever the
// weight is not -- and only then multiplied by log2 e: folding log2 e into the scale would round s * scale * log2 e
// and lse * log2 e, both of tens, apart from each other.  The tensor cores' accumulator drops what lies below its last
// bit, for every product of 16 columns that enters it, so that a long chain makes a score small by as much as the data
// has bits to drop (8 products: nothing where they are exact, 2.6 units of 2^-24 of the score on normally distributed
// queries and keys, 8.6 where all are positive; 36 products: 0, 10 and 54).  So an accumulator takes one column group,
// four products (two groups where TMEM has no more room: head_dim beyond 256 with 32 rows), and the groups add up in
// fp32: 0, 1.5 and 3.4 units at any head_dim, and page weights within 6e-7 of 64-bit ones in the cases below instead of
// 1.2e-6.  It costs a second reading of TMEM: windows of 64 tokens 92 us instead of 75, one token each nothing.
//
// Work.  An item is one KV head of one sequence, a tile 128 of its keys times as many chunks of N rows as its queries
// need (N = 16 for one token's group, up to 256 for a window of them); the line of tiles x chunks is shared evenly.
// Bound: for few rows the reading of K (48 sequences of 1,024 to 8,192 keys, 8 heads, one token each: 94 us, 5.3 TB/s, of
// which 8 us are start and join); for an observation window the threads' chains of score loads, exponentials and sums
// (92 us, of which the special-function units need 27 and the join 13: neither they nor the issue of instructions is
// half busy).  Measured for windows: steps of two row tiles and 64 keys instead of one and 128 the same time (with up to 128
// rows, 187 us instead of 128: half of the warps have none); loads of the next 16 scores under the arithmetic of these
// 1 us less; before, with one accumulator a score, a quarter or 3/8 of the exponentials as a polynomial on the FMA pipes
// or a second warp of products 2 to 8 us more.
//
// Warps.  Groups of four: sums of every other step, a thread per key, no warp waiting for another; then one for the
// products and one for TMA (K tiles page by page through a ring, Q chunks as boxes of tokens x group).  Waits are bounded as in
// ztcp_attend_tc.cu.
#include "../../include/ztcp_kvcache.h"
#include "ztcp_tc.cuh"

namespace ztcp {

namespace {

constexpr int kBars = 40;

struct MassTcParams {
  MassParams m;
  PoolBoxes box;
  // A chunk's rows, at most N: whole tokens of a group each, or (groups wider than N) a part of one token's group.
  int32_t chunk_tokens;  // tokens of a chunk
  int32_t parts;         // chunks that share a token: 1, or ceil(group / N)
  int32_t part_heads;    // heads of the group in a chunk
  int32_t seg_shift;     // log2 of the keys of a segment: 32, or a smaller page's
  int32_t segs;          // segments of a sequence in the workspace
  int32_t sums;          // sums of a segment that a step leaves in the workspace
  int32_t halves;        // a step is one row tile of a chunk
};

template <int KG, int N>
struct Shape {
  static constexpr bool kRows = N == 256;                   // rows on the lanes
  // Warps of the sums: two groups by turns, of as many warps as a step has lanes' quarters.
  static constexpr int kSumWarps = kRows ? 16 : 8;
  static constexpr int kThreads = (kSumWarps + 2) * 32;
  static constexpr int kGroups = KG == 1 ? 1 : 2;           // column groups of a slot
  static constexpr int kSlotBytes = kGroups * kGroupBytes;
  static constexpr int kTileSlots = (KG + kGroups - 1) / kGroups;
  static constexpr int kQBytes = KG * N * 128;
  static constexpr int kQSlots = kQBytes > 32 * 1024 ? 1 : 2;
  static constexpr int kNegBytes = kRows ? 0 : 8 * N * 4;    // every warp its copy of its columns' -lse
  static constexpr int kRoom = (232448 - 4096 - kQSlots * kQBytes - kNegBytes) / kSlotBytes;
  static constexpr int kSlots = kRoom < 8 ? kRoom : 8;
  static constexpr int kSmem = kBars * 8 + 1024 + kSlots * kSlotBytes + kQSlots * kQBytes + kNegBytes;
  // Accumulators of a step: one per column group (two groups where TMEM has no room for more).
  static constexpr int kPer = !kRows && 2 * N * KG > 512 ? 2 : 1;
  static constexpr int kAccs = (KG + kPer - 1) / kPer;
  // With rows on the lanes a second accumulator takes the columns of the second row tile: a step is one row tile then,
  // and the warps that have the other one where there is one accumulator have the other 64 keys.
  static constexpr bool kHalves = kRows && kAccs == 2;
  static constexpr int kBuf = kRows ? 256 : kAccs * N;      // columns of a step's scores; TMEM holds two steps'
  static constexpr int kCols = 2 * kBuf <= 32 ? 32 : 2 * kBuf <= 64 ? 64 : 2 * kBuf <= 128 ? 128 : 2 * kBuf <= 256 ? 256 : 512;
  static_assert(kSlots >= kTileSlots && 2 * kSlots + 9 + 2 * kJobs <= kBars && 2 * kBuf <= kCols, "shape");
};

// Tiles and chunks of a sequence.
struct MassSeq {
  Seq s;
  int32_t tiles, chunks;
  __device__ __forceinline__ int64_t cost() const { return (int64_t)tiles * chunks; }
};
__device__ __forceinline__ MassSeq mass_seq(const MassTcParams& P, int b) {
  const CacheParams& c = P.m.c;
  MassSeq m;
  m.s = load_seq(c, b);
  m.tiles = m.s.q_len > 0 ? (m.s.kv_len + kKeys - 1) / kKeys : 0;
  m.chunks = (m.s.q_len + P.chunk_tokens - 1) / P.chunk_tokens * P.parts;
  return m;
}
// Whether chunk ch's rows fill more than one row tile.
__device__ __forceinline__ bool two_row_tiles(const MassTcParams& P, int N, int q_len, int ch) {
  return (P.parts == 1 ? (q_len - ch * P.chunk_tokens) * (int64_t)P.m.c.group : P.m.c.group - ch % P.parts * N) > 128;
}

template <int N>
__device__ __forceinline__ void tmem_load(uint32_t addr, uint32_t* r) {
  if constexpr (N == 32) tmem_ld32(addr, r);
  else tmem_ld16(addr, r);
}
template <int N>
__device__ __forceinline__ void tmem_ready(uint32_t* r) {
  if constexpr (N == 32) tmem_ready32(r);
  else tmem_ready16(r);
}
// x += y, columns of fp32.
template <int N>
__device__ __forceinline__ void add_columns(uint32_t* x, const uint32_t* y) {
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    float a, b;
    unpair(add2(pair(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), pair(__uint_as_float(y[i]), __uint_as_float(y[i + 1]))), a, b);
    x[i] = __float_as_uint(a);
    x[i + 1] = __float_as_uint(b);
  }
}

template <bool BF16, int KG, int N>
__global__ void __launch_bounds__((Shape<KG, N>::kThreads), 1)
page_mass_tc_kernel(const __grid_constant__ MassTcParams P, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap qmap) {
  using Sh = Shape<KG, N>;
  constexpr int kSlots = Sh::kSlots, kTS = Sh::kTileSlots, kQS = Sh::kQSlots, kMmaWarp = Sh::kSumWarps, kTmaWarp = kMmaWarp + 1;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Waits waits_s;
  __shared__ uint32_t tmem_s;
  __shared__ Job s_jobs[kJobs];  // row: chunks of the item; whole, inside: not used
  __shared__ unsigned s_bad[16];  // a tile's boxes that lie outside the pool
  const CacheParams& c = P.m.c;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  volatile Waits* const waits = &waits_s;
  const uint32_t bars = smem_u32(smem_raw);
  const uint32_t ring = (bars + kBars * 8 + 1023) & ~1023u;
  const uint32_t qbuf = ring + kSlots * Sh::kSlotBytes;
  float* const negs = reinterpret_cast<float*>(smem_raw + (qbuf - bars) + kQS * Sh::kQBytes);
  auto full = [&](uint32_t s) { return bars + s * 8; };
  auto empty = [&](uint32_t s) { return bars + (kSlots + s) * 8; };
  const uint32_t q_full = bars + 2 * kSlots * 8, q_empty = q_full + 16, s_full = q_empty + 16, s_read = s_full + 16, job_full = s_read + 16,
                 job_empty = job_full + 8 * kJobs, drain = job_empty + 8 * kJobs;
  if (tid == 0) {
    waits_s.limit = c.wait_cycles;
    waits_s.dead = 0;
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_full + 8 * i, 1);
      mbar_init(q_empty + 8 * i, 1);
      mbar_init(s_full + 8 * i, 1);
      mbar_init(s_read + 8 * i, Sh::kSumWarps / 2);
    }
    for (int e = 0; e < kJobs; ++e) {
      mbar_init(job_full + 8 * e, 1);
      mbar_init(job_empty + 8 * e, Sh::kSumWarps + 1);
    }
    mbar_init(drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_s)), "n"(Sh::kCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_s;
  cudaTriggerProgrammaticLaunchCompletion();

  if (warp == kTmaWarp) {
    // ---- TMA -------------------------------------------------------------------------------------------
    int64_t at;
    Spot spot;
    const SplitSpan S = locate_warp(c.n_seqs, P.m.grid, lane, [&](int b) { return mass_seq(P, b).cost() * c.kv_heads; }, &at, &spot);
    int64_t pos = at < 0 ? 0 : at;
    const int64_t end = at < 0 ? 0 : S.begin(blockIdx.x + 1);
    int64_t first = spot.first;
    int b = spot.seq;
    const int per_tile = kKeys / P.box.rows;
    uint32_t kpos = 0, qpos = 0, n = 0, tile = 0;
    bool ok = true;
    auto next = [&](Job* job) {  // publishes the share's next item (none: ta == tb)
      *job = Job{};
      while (pos < end && job->ta == job->tb) {
        MassSeq m = mass_seq(P, b);
        while (pos >= first + m.cost() * c.kv_heads) {
          first += m.cost() * c.kv_heads;
          m = mass_seq(P, ++b);
        }
        const int64_t x = pos - first, h = div_pos(x, m.cost()), start = first + h * m.cost();
        job->row0 = m.s.row0;
        job->b = b;
        job->kv_len = m.s.kv_len;
        job->q_len = m.s.q_len;
        job->row = m.chunks;
        job->head = (int32_t)h;
        job->ta = (int32_t)div_pos(pos - start, m.chunks);
        pos = min(end, start + m.cost());
        job->tb = (int32_t)div_pos(pos - start, m.chunks);
      }
      const uint32_t e = n % kJobs;
      if (n >= kJobs && !warp_wait(job_empty + 8 * e, (n / kJobs - 1) & 1, waits)) return false;
      if (lane == 0) {
        s_jobs[e] = *job;
        mbar_arrive(job_full + 8 * e);
      }
      ++n;
      return true;
    };
    Job job;
    PageRows pages;
    while (ok && (ok = next(&job)) && job.ta < job.tb) {
      auto load_q = [&](int ch) {
        const uint32_t slot = qpos % kQS;
        if (qpos >= kQS && !warp_wait(q_empty + 8 * slot, (qpos / kQS - 1) & 1, waits)) return false;
        if (lane == 0) mbar_expect(q_full + 8 * slot, KG * P.chunk_tokens * P.part_heads * 128);
        const int first_tok = ch / P.parts * P.chunk_tokens;
        __syncwarp();
        if (lane < KG)
          tma_load4(qbuf + slot * Sh::kQBytes + lane * N * 128, &qmap, lane * 64, ch % P.parts * N, job.head, (int)job.row0 + first_tok,
                    q_full + 8 * slot);
        ++qpos;
        return true;
      };
      if (job.row == 1) ok = load_q(0);
      pages.start(job.ta);
      for (int t = job.ta; ok && t < job.tb; ++t) {
        const int32_t row = pages.at(c, P.box, per_tile, job.b, job.kv_len, t, lane);  // pool_rows: zeros
        // (16 tiles back everyone has read theirs: at most 8 are in the ring and 2 more in TMEM)
        const unsigned bad = __ballot_sync(0xffffffffu, lane < per_tile && row == P.box.pool_rows && t * kKeys + (lane << P.box.shift) < job.kv_len);
        if (lane == 0) s_bad[tile & 15] = bad;
        ++tile;
#pragma unroll
        for (int s = 0; s < kTS; ++s, ++kpos) {
          const uint32_t slot = kpos % kSlots;
          if (kpos >= kSlots && !(ok = warp_wait(empty(slot), (kpos / kSlots - 1) & 1, waits))) break;
          const int groups = KG - s * Sh::kGroups < Sh::kGroups ? KG - s * Sh::kGroups : Sh::kGroups;
          if (lane == 0) mbar_expect(full(slot), groups * kGroupBytes);
          __syncwarp();
          if (lane < per_tile)
            for (int g = 0; g < groups; ++g)
              tma_load(ring + slot * Sh::kSlotBytes + g * kGroupBytes + lane * P.box.rows * 128, &kmap, (s * Sh::kGroups + g) * 64, job.head, row, full(slot));
        }
        if (job.row > 1)
          for (int ch = 0; ok && ch < job.row; ++ch) ok = load_q(ch);
      }
    }
    drain_fills(full(0), kSlots, kpos);
    drain_fills(q_full, kQS, qpos);
  } else if (warp == kMmaWarp) {
    // ---- products: one thread ---------------------------------------------------------------------------
    if (elect_one()) {
      constexpr uint32_t kHi = desc_hi(1024, kSwizzle128);
      const uint32_t qk = inst_desc(BF16, 128, Sh::kRows ? kKeys : N, false, false);
      const uint32_t k_lo = desc_lo(ring, 16), q_lo = desc_lo(qbuf, 16);
      uint32_t kpos = 0, qpos = 0, step = 0, jobs = 0;
      bool ok = true;
      auto wait = [&](uint32_t bar, uint32_t n) {  // the n-th completion (from 0)
        ok = ok && mbar_wait(bar, n & 1, waits);
        return ok;
      };
      Job job;
      while (ok && (ok = take_job_alone(s_jobs, job_full, job_empty, jobs, waits, &job)) && job.ta < job.tb) {
        const int chunks = job.row;
        const int tiles = job.tb - job.ta;
        for (int t = 0; ok && t < tiles; ++t) {
          for (int ch = 0; ok && ch < chunks; ++ch) {
            const bool fresh = chunks > 1 || t == 0;             // this step's Q is a new one,
            const bool spent = chunks > 1 || t + 1 == tiles;     // and not used again
            const uint32_t qslot = qpos % kQS;
            if (fresh && !wait(q_full + 8 * qslot, qpos / kQS)) break;
            const bool two = Sh::kRows && two_row_tiles(P, N, job.q_len, ch);
            const int row_steps = Sh::kHalves && two ? 2 : 1;
            for (int half = 0; ok && half < row_steps; ++half, ++step) {
              const uint32_t buf = step & 1, d = tmem + buf * Sh::kBuf, q = q_lo + qslot * (Sh::kQBytes >> 4);
              if (step > 1 && !wait(s_read + 8 * buf, (step >> 1) - 1)) break;
#pragma unroll
              for (int s = 0; s < kTS; ++s) {
                const uint32_t pos = kpos + s, slot = pos % kSlots;
                if (ch == 0 && half == 0 && !wait(full(slot), pos / kSlots)) break;
                tc_fence_after();
                const uint32_t a = k_lo + slot * (Sh::kSlotBytes >> 4);
#pragma unroll
                for (int i = 0; i < Sh::kGroups; ++i) {
                  const int g = s * Sh::kGroups + i;
                  if (g >= KG) continue;
                  if constexpr (Sh::kHalves) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                      mma_ss(d + g * kKeys, q + ((g * N * 128 + k * 32) >> 4) + half * (128 * 128 >> 4), kHi, a + ((i * kGroupBytes + k * 32) >> 4), kHi, qk, k > 0);
                  } else if constexpr (Sh::kRows) {
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                      if (h == 0 || two)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                          mma_ss(d + h * kKeys, q + ((h * 128 * 128 + k * 32) >> 4), kHi, a + (k * 32 >> 4), kHi, qk, k > 0);
                  } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                      mma_ss(d + g / Sh::kPer * N, a + ((i * kGroupBytes + k * 32) >> 4), kHi, q + ((g * N * 128 + k * 32) >> 4), kHi, qk,
                             g % Sh::kPer > 0 || k > 0);
                  }
                }
                if (ch + 1 == chunks && half + 1 == row_steps) tc_commit(empty(slot));
              }
              if (ok) tc_commit(s_full + 8 * buf);
            }
            if (ok && spent) {
              tc_commit(q_empty + 8 * qslot);
              ++qpos;
            }
          }
          kpos += kTS;
        }
      }
      drain_products(drain);
    }
    __syncwarp();
  } else if constexpr (Sh::kRows) {
    // ---- sums: a thread per row -------------------------------------------------------------------------
    const int wg = (warp >> 2) & 1, other = warp >> 3;  // 1: the second row tile's warps, or the second 64 keys'
    const uint32_t ts = tmem + ((uint32_t)(warp & 3) << 21) + wg * Sh::kBuf + other * (Sh::kHalves ? 64 : kKeys);
    const int from = Sh::kHalves ? other * 64 : 0, keys = Sh::kHalves ? 64 : kKeys;  // this warp's, of a tile
    const uint64_t scale2 = pair(c.scale, c.scale), log2e = pair(1.44269504088896f, 1.44269504088896f);
    uint32_t step = 0, mine = 0, jobs = 0, tile = 0;
    Job job;
    bool ok = true;
    while (ok && (ok = take_job(s_jobs, job_full, job_empty, jobs, lane, waits, &job)) && job.ta < job.tb) {
      const int chunks = job.row;
      float neg = -INFINITY;  // -lse; -inf where the row adds nothing
      int lim = 0, clear = 0;  // keys that the row sees, and that all of the warp's rows see
      bool any = false;        // a row of the warp adds something
      auto load_row = [&](int ch, int half) {
        const int r = half * 128 + (tid & 127), tok_in = r / P.part_heads, head_in = r - tok_in * P.part_heads;
        const int tok = ch / P.parts * P.chunk_tokens + tok_in, g = ch % P.parts * N + head_in;
        neg = -INFINITY;
        if (tok_in < P.chunk_tokens && tok < job.q_len && g < c.group) {
          neg = -__ldg(P.m.lse + (job.row0 + tok) * (int64_t)(c.kv_heads * c.group) + job.head * c.group + g);
          if (neg == INFINITY) neg = -INFINITY;
        }
        lim = neg == -INFINITY ? INT_MAX : visible_keys(c, Seq{job.kv_len, job.q_len, job.row0}, tok);
        clear = __reduce_min_sync(0xffffffffu, lim);
        any = __any_sync(0xffffffffu, neg != -INFINITY);
      };
      const bool two = two_row_tiles(P, N, job.q_len, 0);
      const bool several = chunks > 1 || (Sh::kHalves && two);  // steps a tile
      // (an only chunk's two row tiles go to the groups by turns, from whichever the item's first step falls to)
      if (chunks == 1) load_row(0, !Sh::kHalves ? other : two ? (int)(step & 1) ^ wg : 0);
      for (int t = job.ta; ok && t < job.tb; ++t, ++tile) {
        const int j0 = t * kKeys;
        unsigned bad = 0;
        float total = 0.f;  // lane i: the tile's segment i
        bool some = false;
        int ch = 0, half = 0;
        for (; ch < chunks; ++step) {
          const int ch_now = ch, half_now = half;
          if (Sh::kHalves && half == 0 && (ch == 0 ? two : two_row_tiles(P, N, job.q_len, ch))) half = 1;
          else half = 0, ++ch;
          if ((step & 1) != wg) continue;
          some = true;
          if (chunks > 1) load_row(ch_now, Sh::kHalves ? half_now : other);
          if (!(ok = warp_wait(s_full + 8 * wg, mine & 1, waits))) break;
          ++mine;
          tc_fence_after();
          bad = s_bad[tile & 15];
          const uint64_t neg2 = pair(neg, neg);
          auto add_block = [&](uint32_t* x, int n0) {
            if (j0 + n0 + 32 > clear) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (j0 + n0 + i >= lim) x[i] = 0xff800000u;
            }
            uint64_t acc[4];
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const uint64_t s = pair(__uint_as_float(x[i]), __uint_as_float(x[i + 1]));
              uint64_t u = mul2(fma2(s, scale2, neg2), log2e);
              float a, b2;
              unpair(u, a, b2);
              u = pair(fast_exp2(a), fast_exp2(b2));
              acc[i / 8] = i % 8 == 0 ? u : add2(acc[i / 8], u);
            }
            auto put = [&](uint64_t pr, int seg) {
              float a, b2;
              unpair(pr, a, b2);
              float v = neg == -INFINITY ? 0.f : a + b2;
#pragma unroll
              for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
              if (lane == seg) total += v;
            };
            if (P.seg_shift == 5) {
              put(add2(add2(acc[0], acc[1]), add2(acc[2], acc[3])), n0 >> 5);
            } else if (P.seg_shift == 4) {
              put(add2(acc[0], acc[1]), n0 >> 4);
              put(add2(acc[2], acc[3]), (n0 >> 4) + 1);
            } else {
#pragma unroll
              for (int k = 0; k < 4; ++k) put(acc[k], (n0 >> 3) + k);
            }
          };
          if (any) {
#pragma unroll 1
            for (int n0 = 0; n0 < keys; n0 += 32) {
              uint32_t x[32];
              tmem_ld32(ts + n0, x);
              if constexpr (Sh::kHalves) {
                uint32_t y[32];
                tmem_ld32(ts + kKeys + n0, y);
                tmem_ready32(x);
                tmem_ready32(y);
                add_columns<32>(x, y);
              } else {
                tmem_ready32(x);
              }
              if (n0 + 32 == keys) {  // S has been read
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(s_read + 8 * wg);
              }
              add_block(x, from + n0);
            }
          } else {
            __syncwarp();
            if (lane == 0) mbar_arrive(s_read + 8 * wg);
          }
        }
        if (!ok) break;
        const int seg = (j0 >> P.seg_shift) + lane;
        const int at = lane << P.seg_shift;  // the segment's first key, of the tile's
        if (some && at >= from && at < from + keys && seg << P.seg_shift < job.kv_len) {
          if (bad >> (lane << P.seg_shift >> P.box.shift) & 1) total = 0.f;
          P.m.part[(((int64_t)((several ? P.sums * wg : 0) + (Sh::kHalves ? 0 : other * 4) + (warp & 3)) * c.n_seqs + job.b) * c.kv_heads + job.head) * P.segs + seg] = total;
        }
      }
    }
  } else {
    // ---- sums: a thread per key -------------------------------------------------------------------------
    const int wg = warp >> 2, key = tid & 127;
    const uint32_t ts = tmem + ((uint32_t)(warp & 3) << 21) + wg * Sh::kBuf;
    float* const neg = negs + warp * N;
    const uint64_t scale2 = pair(c.scale, c.scale), log2e = pair(1.44269504088896f, 1.44269504088896f);
    uint32_t step = 0, mine = 0, jobs = 0, tile = 0;
    Job job;
    bool ok = true;
    while (ok && (ok = take_job(s_jobs, job_full, job_empty, jobs, lane, waits, &job)) && job.ta < job.tb) {
      const int chunks = job.row;
      bool none = false;  // a row of the chunk adds nothing
      // -lse of a chunk's rows, -inf where a row adds nothing
      auto load_neg = [&](int ch) {
        __syncwarp();
        bool inf = false;
#pragma unroll 1
        for (int i = lane; i < N; i += 32) {
          const int r = i, t = r / P.part_heads, tok = ch / P.parts * P.chunk_tokens + t, g = ch % P.parts * N + r - t * P.part_heads;
          float x = -INFINITY;
          if (t < P.chunk_tokens && tok < job.q_len && g < c.group) {
            x = -__ldg(P.m.lse + (job.row0 + tok) * (int64_t)(c.kv_heads * c.group) + job.head * c.group + g);
            if (x == INFINITY) x = -INFINITY;
            inf = inf || x == -INFINITY;
          }
          neg[i] = x;
        }
        none = __any_sync(0xffffffffu, inf);
      };
      if (chunks == 1) load_neg(0);
      for (int t = job.ta; ok && t < job.tb; ++t, ++tile) {
        const int j = t * kKeys + key;
        bool there = false;
        float sum = 0.f;
        bool some = false;
        for (int ch = 0; ch < chunks; ++ch, ++step) {
          if ((step & 1) != wg) continue;
          some = true;
          if (chunks > 1) load_neg(ch);
          const int tok0 = ch / P.parts * P.chunk_tokens;
          const int valid = P.parts == 1 ? min(P.chunk_tokens, job.q_len - tok0) * c.group : min(N, c.group - ch % P.parts * N);  // the chunk's rows
          // token i of the chunk sees key j when j < kv_len - q_len + tok0 + i + 1: rows from `from` on.  (Clamped to the
          // chunk's tokens first: a key far before the window times a wide group does not fit 32 bits.)
          const int unseen = c.causal ? min(max(j - (job.kv_len - job.q_len + tok0), 0), P.chunk_tokens) : 0;
          const int from = unseen * c.group;
          if (!(ok = warp_wait(s_full + 8 * wg, mine & 1, waits))) break;
          ++mine;
          tc_fence_after();
          there = j < job.kv_len && !(s_bad[tile & 15] >> (key >> P.box.shift) & 1);
          uint64_t acc0 = pair(0.f, 0.f), acc1 = acc0;
          constexpr int kBlock = N < 32 ? N : 32;
          auto add_block = [&](const uint32_t* x, int n0) {  // columns [n0, n0 + kBlock)
            if (n0 >= valid) return;
            const bool whole = !none && n0 + kBlock <= valid && __all_sync(0xffffffffu, from <= n0);
#pragma unroll
            for (int i = 0; i < kBlock; i += 4) {
              if (N < 32 && i >= valid) break;
              const float4 w = *reinterpret_cast<const float4*>(neg + n0 + i);
              float a, b2, d, e;
              const uint64_t s = pair(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), s1 = pair(__uint_as_float(x[i + 2]), __uint_as_float(x[i + 3]));
              unpair(mul2(fma2(s, scale2, pair(w.x, w.y)), log2e), a, b2);
              unpair(mul2(fma2(s1, scale2, pair(w.z, w.w)), log2e), d, e);
              a = fast_exp2(a);
              b2 = fast_exp2(b2);
              d = fast_exp2(d);
              e = fast_exp2(e);
              if (!whole) {
                const int r = n0 + i;
                a = r >= from && r < valid ? a : 0.f;
                b2 = r + 1 >= from && r + 1 < valid ? b2 : 0.f;
                d = r + 2 >= from && r + 2 < valid ? d : 0.f;
                e = r + 3 >= from && r + 3 < valid ? e : 0.f;
              }
              acc0 = add2(acc0, pair(a, b2));
              acc1 = add2(acc1, pair(d, e));
            }
          };
          auto release = [&] {  // S^T has been read
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(s_read + 8 * wg);
          };
          // Columns [n0, n0 + kBlock) of all accumulators, added up; two more of them are loaded at a time.
          auto load_block = [&](uint32_t* x, int n0) {
            tmem_load<kBlock>(ts + n0, x);
            if constexpr (Sh::kAccs == 1) tmem_ready<kBlock>(x);
#pragma unroll
            for (int a = 1; a < Sh::kAccs; a += 2) {
              uint32_t y[kBlock], z[kBlock];
              tmem_load<kBlock>(ts + a * N + n0, y);
              if (a + 1 < Sh::kAccs) tmem_load<kBlock>(ts + (a + 1) * N + n0, z);
              if (a == 1) tmem_ready<kBlock>(x);
              tmem_ready<kBlock>(y);
              add_columns<kBlock>(x, y);
              if (a + 1 < Sh::kAccs) {
                tmem_ready<kBlock>(z);
                add_columns<kBlock>(x, z);
              }
            }
          };
          if constexpr (N < 64 || Sh::kAccs > 1) {
            uint32_t x[kBlock];
#pragma unroll 1
            for (int n0 = 0; n0 < N; n0 += kBlock) {
              load_block(x, n0);
              const bool more = n0 + kBlock < N && n0 + kBlock < valid;
              if (!more) release();
              add_block(x, n0);
              if (!more) break;
            }
          } else {  // one block's loads under the other's arithmetic
            uint32_t x[32], y[32];
            tmem_ld32(ts, x);
#pragma unroll 1
            for (int n0 = 0; n0 < N; n0 += 64) {
              tmem_ready32(x);
              tmem_ld32(ts + n0 + 32, y);
              add_block(x, n0);
              tmem_ready32(y);
              const bool more = n0 + 64 < N && n0 + 64 < valid;
              if (more) tmem_ld32(ts + n0 + 64, x);
              else release();
              add_block(y, n0 + 32);
              if (!more) break;
            }
          }
          float s0, s1, s2, s3;
          unpair(acc0, s0, s1);
          unpair(acc1, s2, s3);
          sum += (s0 + s1) + (s2 + s3);
        }
        if (!ok) break;
        if (some) {
          if (!there) sum = 0.f;
          const int seg = 1 << P.seg_shift;
          for (int d = seg >> 1; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
          if ((lane & (seg - 1)) == 0 && j < job.kv_len)
            P.m.part[(((int64_t)(chunks > 1 ? wg : 0) * c.n_seqs + job.b) * c.kv_heads + job.head) * P.segs + (j >> P.seg_shift)] = sum;
        }
      }
    }
  }
  __syncthreads();
  if (tid == 0) P.m.errors[blockIdx.x] = waits->dead;
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(Sh::kCols) : "memory");
  }
}

// A page's weight: its segments' sums in a fixed order.  A warp per page, a lane with every 32nd sum, then a tree (eight
// threads per page took 14 us for 2,048 pages of 128 sums); also the status.
__global__ void __launch_bounds__(256) page_mass_join_kernel(const __grid_constant__ MassTcParams P) {
  const CacheParams& c = P.m.c;
  const int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const int b = (int)(i / c.max_pages), p = (int)(i - (int64_t)b * c.max_pages);
  float before = 0.f;
  int n = 0, slots = 0;
  if (b < c.n_seqs) {
    const MassSeq m = mass_seq(P, b);
    const int64_t left = m.s.kv_len - (int64_t)p * c.page_tokens;
    if (left > 0) {
      if (P.m.mass) before = P.m.mass[i];
      if (m.chunks > 0) {
        n = (int)((min((int64_t)c.page_tokens, left) + (1 << P.seg_shift) - 1) >> P.seg_shift);
        slots = m.chunks > 1 || (P.halves && two_row_tiles(P, 256, m.s.q_len, 0)) ? 2 : 1;
      }
    }
  }
  cudaGridDependencySynchronize();
  for (int s = blockIdx.x * 8 + (threadIdx.x >> 5); s < c.n_seqs; s += gridDim.x * 8) {
    int late = 0;
    for (int e = threadIdx.x & 31; e < P.m.grid; e += 32) late |= __ldcg(P.m.errors + e);
    if (!__any_sync(0xffffffffu, late)) write_seq_status(c, s, threadIdx.x & 31);
    else if (threadIdx.x % 32 == 0) c.status[s] = ZTCP_SEQ_TIMEOUT;
  }
  float sum = 0.f;
  const float* const first = P.m.part + (int64_t)b * c.kv_heads * P.segs + ((int64_t)p * c.page_tokens >> P.seg_shift);
  const int64_t per_sum = (int64_t)c.n_seqs * c.kv_heads * P.segs;
  for (int x = lane; x < slots * P.sums * c.kv_heads * n; x += 32) {
    const int y = x / n, k = x - y * n, z = y / c.kv_heads, h = y - z * c.kv_heads;
    sum += __ldcg(first + z * per_sum + (int64_t)h * P.segs + k);
  }
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if (b < c.n_seqs && lane == 0) P.m.out[i] = P.m.mass ? fmaf(P.m.decay, before, sum) : sum;
}

// ---- host -----------------------------------------------------------------------------------------
template <bool BF16, int KG, int N>
void launch_kernel(const MassTcParams& P, const CUtensorMap& k, const CUtensorMap& q, cudaStream_t s) {
  auto* const f = page_mass_tc_kernel<BF16, KG, N>;
  constexpr int smem = Shape<KG, N>::kSmem;
  cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  f<<<P.m.grid, Shape<KG, N>::kThreads, smem, s>>>(P, k, q);
}

template <bool BF16>
void launch_any(const MassTcParams& P, int n, const CUtensorMap& k, const CUtensorMap& q, cudaStream_t s) {
  const int d = P.m.c.head_dim;
  if (d <= 64) n == 16 ? launch_kernel<BF16, 1, 16>(P, k, q, s) : n == 64 ? launch_kernel<BF16, 1, 64>(P, k, q, s) : launch_kernel<BF16, 1, 256>(P, k, q, s);
  else if (d <= 128) n == 16 ? launch_kernel<BF16, 2, 16>(P, k, q, s) : n == 64 ? launch_kernel<BF16, 2, 64>(P, k, q, s) : launch_kernel<BF16, 2, 256>(P, k, q, s);
  else if (d <= 256) n == 16 ? launch_kernel<BF16, 4, 16>(P, k, q, s) : launch_kernel<BF16, 4, 64>(P, k, q, s);
  else n == 16 ? launch_kernel<BF16, 9, 16>(P, k, q, s) : launch_kernel<BF16, 9, 32>(P, k, q, s);
}

// Rows of a chunk: the smallest of 16, 64 and 256 that holds a sequence's rows; wide heads leave less room for Q.
// Measured on 48 sequences of 1,024 to 8,192 tokens, 8 KV heads of 128, with 16 / 64 / 256: 4 rows 87.5 / 92.0 / 128 us,
// 32 rows 156 / 90 / 128, 64 rows 251 / 113 / 129, 128 rows 449 / 233 / 129.
int chunk_rows(const CacheParams& c, int64_t rows) {
  if (rows <= 16) return 16;
  if (c.head_dim > 256) return 32;
  return rows <= 64 || c.head_dim > 128 ? 64 : 256;
}
// Shape::kHalves, and the sums of a segment that a step leaves: one per warp with rows on the lanes, else one in all.
bool halves_of(const CacheParams& c, int n) { return n == 256 && c.head_dim > 64; }
int sums_of(const CacheParams& c, int n) { return n != 256 ? 1 : halves_of(c, n) ? 4 : 8; }
int seg_shift(const CacheParams& c) { return c.page_tokens >= 32 ? 5 : c.page_tokens == 16 ? 4 : 3; }
int64_t seg_count(const CacheParams& c) { return (int64_t)c.max_pages * c.page_tokens >> seg_shift(c); }

}  // namespace

int64_t page_mass_tc_workspace(const CacheParams& c, int64_t rows, int sms) {  // sums by step parity
  return (sms + 3) / 4 * 16 + 2 * sums_of(c, chunk_rows(c, rows)) * c.n_seqs * (int64_t)c.kv_heads * seg_count(c) * (int64_t)sizeof(float);
}

// A sequence's segments and a page's sums have to fit 32 bits (16 sums a segment at most), and all sums a GPU's memory
// (whose size is formed here in floating point: in 64 bits it could wrap).
bool page_mass_tc_fits(const CacheParams& c) {
  const int64_t page_sums = 16 * (int64_t)c.kv_heads * ((c.page_tokens >> seg_shift(c)) + 1);
  return pages_fit(c, kKeys) && seg_count(c) < ((int64_t)1 << 31) && page_sums < ((int64_t)1 << 31) &&
         64.0 * c.n_seqs * c.kv_heads * (double)seg_count(c) < 0x1p37;
}

bool launch_page_mass_tc(MassParams m, int64_t rows, int sms, void* workspace, bool bf16, cudaStream_t s) {
  MassTcParams P;
  P.m = m;
  P.m.grid = sms;
  P.m.errors = static_cast<int32_t*>(workspace);
  P.m.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + (sms + 3) / 4 * 16);
  P.box = pool_boxes(m.c, kKeys);
  const int n = chunk_rows(m.c, rows);
  P.chunk_tokens = m.c.group < n ? n / m.c.group : 1;
  P.parts = (m.c.group + n - 1) / n;
  P.part_heads = m.c.group < n ? m.c.group : n;
  P.seg_shift = seg_shift(m.c);
  P.segs = (int32_t)seg_count(m.c);
  P.sums = sums_of(m.c, n);
  P.halves = halves_of(m.c, n);
  CUtensorMap k, q;
  if (!pool_map(&k, m.c.k, m.c, bf16, P.box) || !query_map(&q, m.c, bf16, P.chunk_tokens, P.part_heads)) return false;
  if (bf16) launch_any<true>(P, n, k, q, s);
  else launch_any<false>(P, n, k, q, s);
  if (cudaPeekAtLastError() != cudaSuccess) return true;
  cudaLaunchConfig_t cfg = {};
  const int64_t pages = (int64_t)m.c.n_seqs * m.c.max_pages;
  cfg.gridDim = dim3((unsigned)((pages + 7) / 8));
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, page_mass_join_kernel, P);
  return true;
}

}  // namespace ztcp
