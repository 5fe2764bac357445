// ztcp_attend_decode.cu -- attention of the newest tokens over a paged cache (ztcp_attend_pages) for items of few
// rows: one token per sequence, or a few, times a group of heads.
//
// The mathematics is that of ztcp_attend.cu.  Bound: a K and V row serves at most N rows here, so the time is that
// of reading K and V once, and the kernel's one job is to keep that many bytes in flight with little else to do.
// The products are turned over, so that the keys fill the tensor core's 128 lanes and the few rows its N columns:
//   S^T[128 keys, N]   = K Q^T        (K, Q K-major)
//   O^T[128 columns, N] += V^T P^T    (V as it lies, MN-major; P^T from shared memory)
// A tile of 128 keys is then one thread per key in the softmax, which touches N scores, and a handful of
// tcgen05.mma by one thread: about 500 instructions per warp where a 16-row mma.sync tile needed 4,000 (measured:
// 359 us for 48 sequences of up to 8,192 tokens, 32/8 heads of 128, against 144 us to read K and V once).
//
// Warps.  0-3 and 4-7: softmax of every other tile, a thread per key, each group with its own O^T, maxima and sums (a
// tile's softmax takes longer than its products and its share of the memory's time; two of them side by side do not);
// 8: one thread issues the products; 9: TMA.  K and V tiles pass a ring of slots of up to 128 columns, one box per
// page.  A row's maximum over the tile is a redux per warp and an exchange through shared memory; sums stay per
// thread until the item ends.  O^T is rescaled only when a maximum has grown by more than 2^8 over the one in use.
// For single-buffer pools V's columns are those of the K tile itself.
//
// Measured: 48 sequences of 1,024 to 8,192 tokens, 32/8 heads of 128: 165 us, 5.7 TB/s, of which 8 us are start and join;
// 32 sequences of 1,000 to 8,100 over a latent cache, 16 heads of 576: 63 us, 2.8 TB/s (48 us of them without any load:
// 15 tiles a CTA, of 52 products that take 39 cycles each to issue, do not hide the start, two items' ends and the
// join); one sequence of 1,021 tokens: 16 us, two launches.  Chunks that have no kernel of their own come here too, a
// reading of K and V per 16 rows (latent pages: 32): 512 tokens over 8,192, 16 latent heads of 576 531 us, 32/8 heads of
// 256 826.
//
// Work, joining of shared items and bounded waits as in ztcp_attend_tc.cu.
#include "ztcp_tc.cuh"

namespace ztcp {

namespace {

constexpr int kThreads = 320;
constexpr int kMmaWarp = 8, kTmaWarp = 9;
constexpr int kTurns = 4;
constexpr int kBars = 40;  // barrier slots at the start of shared memory

struct DecodeParams {
  AttendParams a;
  PoolBoxes box;
};

// KG: 64-column groups of K; MB: 128-column blocks of V; N: rows of an item.
template <int KG, int MB, int N, bool SHARED>
struct Shape {
  // Keys of a tile.  A single-buffer pool's rows are wide: 64 keys, so that two tiles fit the ring; S^T then has 64
  // rows, 16 in the first lanes of each warp's 32.
  static constexpr int kTileKeys = SHARED ? 64 : kKeys;
  static constexpr int kGroupBytes = kTileKeys * 128;                   // one column group of a tile
  static constexpr int kGroups = KG == 1 ? 1 : 2;                       // column groups of a slot
  static constexpr int kSlotBytes = kGroups * kGroupBytes;
  static constexpr int kKSlots = SHARED ? 1 + MB : (KG + 1) / 2;        // slots of a tile's K (shared: group 0, then V's pairs)
  static constexpr int kTileSlots = SHARED ? kKSlots : 2 * kKSlots;
  static constexpr int kQBytes = KG * N * 128;
  static constexpr int kPBlock = kTileKeys * 32;                        // P^T of 16 rows
  static constexpr int kPBytes = N / 16 * kPBlock;
  static constexpr int kTail = 2 * kPBytes + kQBytes;
  static constexpr int kRoom = (232448 - 8192 - kTail) / kSlotBytes;
  static constexpr int kSlots = kRoom < 3 * kTileSlots ? kRoom : 3 * kTileSlots;  // fewer than four tiles: see s_full
  static constexpr int kSmem = kBars * 8 + 1024 + kSlots * kSlotBytes + kTail;
  static constexpr int kCols = (2 + 2 * MB) * N <= 64 ? 64 : ((2 + 2 * MB) * N <= 128 ? 128 : ((2 + 2 * MB) * N <= 256 ? 256 : 512));
  // the next tile's K and this tile's V share the ring
  static_assert(kSlots >= (SHARED ? 2 * kTileSlots : kTileSlots + kKSlots) && kSlots + 16 + 2 * kJobs <= kBars && (2 + 2 * MB) * N <= kCols, "shape");
  // first column group, and number of groups, of slot s of a tile's K
  static __device__ __forceinline__ constexpr int group(int s) { return SHARED ? (s == 0 ? 0 : 2 * s - 1) : s * kGroups; }
  static __device__ __forceinline__ constexpr int groups(int s) { return SHARED && s == 0 ? 1 : kGroups; }
};

__device__ __forceinline__ float warp_max(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}

// Lane n gets the sum of v[n] over the warp.
template <int N>
__device__ __forceinline__ float lane_sums(float (&v)[N], int lane) {
#pragma unroll
  for (int d = N / 2; d > 0; d >>= 1)
#pragma unroll
    for (int i = 0; i < d; ++i) {
      const bool up = lane & d;
      const float keep = up ? v[i + d] : v[i], send = up ? v[i] : v[i + d];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, d);
    }
  return N == 32 ? v[0] : v[0] + __shfl_xor_sync(0xffffffffu, v[0], 16);
}

template <int N>
__device__ __forceinline__ void tmem_ld_cols(uint32_t addr, uint32_t* r) {
  if constexpr (N == 32) {
    tmem_ld32(addr, r);
    tmem_ready32(r);
  } else {
    tmem_ld16(addr, r);
    tmem_ready16(r);
  }
}
template <int N>
__device__ __forceinline__ void tmem_st_cols(uint32_t addr, const uint32_t* r) {
  if constexpr (N == 32) tmem_st32(addr, r);
  else
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
                 "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
template <bool BF16, int KG, int MB, int N, bool SHARED>
__global__ void __launch_bounds__(kThreads, 1)
attend_decode_kernel(const __grid_constant__ DecodeParams P, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using Sh = Shape<KG, MB, N, SHARED>;
  constexpr int kSlots = Sh::kSlots, kTS = Sh::kTileSlots, kKS = Sh::kKSlots, kTileKeys = Sh::kTileKeys;
  constexpr int kGroupBytes = Sh::kGroupBytes, kKGroups = Sh::kGroups;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Waits waits_s;
  __shared__ uint32_t tmem_s;
  __shared__ unsigned s_bad[16];  // a tile's boxes that lie outside the pool
  __shared__ float4 s_max[2][2][N], s_sum[2][N];  // per group (and tile, by turns) and row: one value of each warp
  __shared__ float s_top[2][N];                   // per group and row: the maximum in use
  __shared__ float2 s_mix[2][N];                     // per row: what the groups' O count
  __shared__ int64_t s_row[2][kTurns][N];         // per group, item (by turns) and row: the row of the output,
  __shared__ int32_t s_lim[2][kTurns][N];         // and the keys that it sees
  __shared__ Job s_jobs[kJobs];
  const CacheParams& c = P.a.c;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  volatile Waits* const waits = &waits_s;

  const uint32_t bars = smem_u32(smem_raw);
  const uint32_t ring = (bars + kBars * 8 + 1023) & ~1023u;
  const uint32_t qbuf = ring + kSlots * Sh::kSlotBytes, pbuf = qbuf + Sh::kQBytes;
  auto full = [&](uint32_t s) { return bars + s * 8; };
  // s_full, pv_done: a tile's scores and products are done, four barriers by turns -- the TMA warp, which waits for the
  // tiles whose slots it refills, may find up to three later ones done as well, and a barrier tells a phase only from
  // the next one.  q_full: Q is there; p_full, meet: per group; summed, read: at an item's end, both groups' sums are
  // there and both have read O
  const uint32_t q_full = bars + kSlots * 8, s_full = q_full + 8, p_full = s_full + 32, pv_done = p_full + 16, meet = pv_done + 32,
                 summed = meet + 16, read = summed + 8, job_full = read + 8, job_empty = job_full + 8 * kJobs, drain = job_empty + 8 * kJobs;

  if (tid == 0) {
    waits_s.limit = c.wait_cycles;
    waits_s.dead = 0;
    for (int s = 0; s < kSlots; ++s) mbar_init(full(s), 1);
    mbar_init(q_full, 256);
    for (int i = 0; i < 4; ++i) {
      mbar_init(s_full + 8 * i, 1);
      mbar_init(pv_done + 8 * i, 1);
    }
    for (int g = 0; g < 2; ++g) {
      mbar_init(p_full + 8 * g, 128);
      mbar_init(meet + 8 * g, 4);
    }
    mbar_init(summed, 8);
    mbar_init(read, 8);
    for (int e = 0; e < kJobs; ++e) {
      mbar_init(job_full + 8 * e, 1);
      mbar_init(job_empty + 8 * e, 9);
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
  cudaTriggerProgrammaticLaunchCompletion();  // the joining kernel may be set up meanwhile; it waits for this one's end

  if (warp == kTmaWarp) {
    // ---- TMA: a tile's slots in turn through the ring; lane p fetches page p of the tile ------------
    const int per_tile = kTileKeys / P.box.rows;
    uint32_t pos = 0, tile = 0;
    int64_t at;
    Spot spot;
    const SplitSpan S = locate_warp(c.n_seqs, P.a.grid, lane, [&](int b) { return seq_work(c, N, b); }, &at, &spot);
    Publisher<kTileKeys> pub;
    pub.walk.begin(c, N, 0, spot, at < 0 ? 0 : at, at < 0 ? 0 : S.begin(blockIdx.x + 1));
    pub.cut = Cut{};
    pub.n = 0;
    Job job;
    PageRows pages;
    bool ok = true;
    while (ok && (ok = pub.next(c, S, s_jobs, job_full, job_empty, lane, waits, &job)) && job.ta < job.tb) {
      pages.start(job.ta);
      for (int t = job.ta; ok && t < job.tb; ++t) {
        const int32_t row = pages.at(c, P.box, per_tile, job.b, job.kv_len, t, lane);  // pool_rows: zeros
        // (16 tiles back everyone has read theirs: fewer than four are in the ring and two more in TMEM)
        const unsigned bad = __ballot_sync(0xffffffffu, lane < per_tile && row == P.box.pool_rows && t * kTileKeys + (lane << P.box.shift) < job.kv_len);
        if (lane == 0) s_bad[tile & 15] = bad;
        ++tile;
#pragma unroll
        for (int s = 0; s < kTS; ++s, ++pos) {
          const uint32_t slot = pos % kSlots;
          if (pos >= kSlots) {  // the slot's last tile: its K is done with its scores, its V (or shared K) with its products
            const uint32_t was = pos - kSlots, tile = was / kTS;
            ok = ok && mbar_wait((SHARED || was % kTS >= kKS ? pv_done : s_full) + 8 * (tile & 3), (tile >> 2) & 1, waits);
          }
          if (!__all_sync(0xffffffffu, ok)) {
            ok = false;
            break;
          }
          const bool isv = !SHARED && s >= kKS;
          const int ks = isv ? s - kKS : s;
          const int g0 = Sh::group(ks), n = Sh::groups(ks);
          if (lane == 0) mbar_expect(full(slot), n * kGroupBytes);
          __syncwarp();
          if (lane < per_tile)
            for (int g = 0; g < n; ++g)
              tma_load(ring + slot * Sh::kSlotBytes + g * kGroupBytes + lane * P.box.rows * 128, isv ? &vmap : &kmap, (g0 + g) * 64, job.head, row,
                       full(slot));
        }
      }
    }
    if (lane == 0) P.a.cuts[blockIdx.x] = pub.cut;
    drain_fills(full(0), kSlots, pos);
  } else if (warp == kMmaWarp) {
    // ---- products: one thread ------------------------------------------------------------------------
    if (elect_one()) {
      // P^T: 32-byte swizzle, rows of the product contiguous per key, 8-key groups 256 bytes apart, the next 16 rows
      // one block on.  V: the next 64 columns one group on (KG = 1: the block's upper half repeats rows nobody reads).
      constexpr uint32_t kHi = desc_hi(1024, kSwizzle128), kPHi = desc_hi(256, kSwizzle32);
      constexpr uint32_t kVLbo = KG == 1 ? 1024 : kGroupBytes;
      const uint32_t qk = inst_desc(BF16, kTileKeys, N, false, false), pv = inst_desc(BF16, 128, N, true, true);
      const uint32_t k_lo = desc_lo(ring, 16), v_lo = desc_lo(ring, kVLbo), q_lo = desc_lo(qbuf, 16), p_lo = desc_lo(pbuf, Sh::kPBlock);
      bool ok = true;
      auto wait = [&](uint32_t bar, uint32_t n) {  // the n-th completion (from 0)
        ok = ok && mbar_wait(bar, n & 1, waits);
        return ok;
      };
      auto scores = [&](uint32_t step) {  // S^T of the CTA's tile `step`
#pragma unroll
        for (int s = 0; s < kKS; ++s) {
          const uint32_t pos = step * kTS + s, slot = pos % kSlots;
          if (!wait(full(slot), pos / kSlots)) return;
          tc_fence_after();
          const uint32_t a = k_lo + slot * (Sh::kSlotBytes >> 4), d = tmem + (step & 1) * N;
#pragma unroll
          for (int g = 0; g < Sh::groups(s); ++g)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              mma_ss(d, a + ((g * kGroupBytes + k * 32) >> 4), kHi, q_lo + (((Sh::group(s) + g) * N * 128 + k * 32) >> 4), kHi, qk,
                     Sh::group(s) + g > 0 || k > 0);
        }
        tc_commit(s_full + 8 * (step & 3));
      };
      auto values = [&](uint32_t step, bool acc) {  // O^T += V^T P^T
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
          const uint32_t pos = step * kTS + (SHARED ? 1 : kKS) + mb, slot = pos % kSlots;
          if (!SHARED) {  // a shared tile has been waited for by its scores
            if (!wait(full(slot), pos / kSlots)) return;
            tc_fence_after();
          }
          const uint32_t a = v_lo + slot * (Sh::kSlotBytes >> 4), d = tmem + (2 + (step & 1) * MB + mb) * N,
                         p = p_lo + (step & 1) * (Sh::kPBytes >> 4);
#pragma unroll
          for (int k = 0; k < kTileKeys / 16; ++k)
            mma_ss(d, a + (k * 2048 >> 4), kHi, p + (k * 512 >> 4), kPHi, pv, acc || k > 0);
        }
        tc_commit(pv_done + 8 * (step & 3));
      };
      uint32_t step = 0, items = 0;
      Job job;
      while (ok && (ok = take_job_alone(s_jobs, job_full, job_empty, items, waits, &job)) && job.ta < job.tb) {
        const int n = job.tb - job.ta;
        if (!wait(q_full, items - 1)) break;
        tc_fence_after();
        for (int t = 0; ok && t <= n; ++t) {  // a tile's scores run under the softmax of the one before
          if (t < n) scores(step + t);
          if (t > 0) {
            const uint32_t s = step + t - 1;
            if (!wait(p_full + 8 * (s & 1), s >> 1)) break;
            tc_fence_after();
            values(s, t > 2);
          }
        }
        step += n;
      }
      drain_products(drain);
    }
    __syncwarp();
  } else {
    // ---- softmax: a thread per key, the CTA's tiles by turns to two groups of four warps -------------
    const int wg = warp >> 2, wt = tid & 127, ww = warp & 3;
    const uint32_t lanes = (uint32_t)ww << 21;
    const uint32_t ts = tmem + lanes + wg * N, to = tmem + lanes + (2 + wg * MB) * N;  // this group's S^T and O^T
    const int key = kTileKeys == 128 ? wt : ww * 16 + (lane & 15);  // the thread's key of a tile
    const bool holds = kTileKeys == 128 || lane < 16;
    const uint32_t pdst = pbuf + wg * Sh::kPBytes + key * 32;
    const int chunks = c.head_dim / 8;
    uint32_t step = 0, mine = 0, meets = 0, nitem = 0;  // tiles of the CTA, of this group, meetings, items
    auto tile_wait = [&](uint32_t bars, uint32_t tile) { return warp_wait(bars + 8 * (tile & 3), (tile >> 2) & 1, waits); };
    // The group's four warps meet.  Not a bar.sync, which no bound could end if a warp had left after a timeout.
    auto meet_warps = [&] {
      __syncwarp();
      if (lane == 0) mbar_arrive(meet + 8 * wg);
      return warp_wait(meet + 8 * wg, meets++ & 1, waits);
    };
    // The next item: its rows' places and limits (tables of kTurns items, by turns: a warp may be two items ahead of
    // another), and Q into shared memory.
    Job job;
    uint32_t jobs = 0;
    auto open = [&] {
      if (!take_job(s_jobs, job_full, job_empty, jobs, lane, waits, &job)) return false;
      if (job.ta == job.tb) return true;
      if (wt < job.rows) {
        const int tok = (job.row + wt) / c.group, gh = job.row + wt - tok * c.group;
        s_row[wg][jobs % kTurns][wt] = (job.row0 + tok) * (int64_t)(c.kv_heads * c.group) + job.head * c.group + gh;
        s_lim[wg][jobs % kTurns][wt] = visible_keys(c, Seq{job.kv_len, job.q_len, job.row0}, tok);
      }
      constexpr int kAhead = KG > 2 ? 4 : 1;  // chunks of 16 bytes in flight per thread
#pragma unroll 1
      for (int i0 = tid; i0 < job.rows * KG * 8; i0 += 256 * kAhead) {
        uint4 v[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int i = i0 + u * 256, r = i / (KG * 8), x = i - r * (KG * 8);
          v[u] = make_uint4(0, 0, 0, 0);
          if (r < job.rows && x < chunks) {
            const int tok = (job.row + r) / c.group, gh = (job.row + r) - tok * c.group;
            v[u] = __ldg(reinterpret_cast<const uint4*>(c.q + (job.row0 + tok) * c.q_token_stride + (int64_t)(job.head * c.group + gh) * c.q_head_stride) + x);
          }
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int i = i0 + u * 256, r = i / (KG * 8), x = i - r * (KG * 8);
          if (r < job.rows)
            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(qbuf + (x >> 3) * N * 128 + r * 128 + (((x & 7) ^ (r & 7)) << 4)), "r"(v[u].x),
                         "r"(v[u].y), "r"(v[u].z), "r"(v[u].w) : "memory");
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(q_full);
      return true;
    };
    bool ok = open();
    while (ok && job.ta < job.tb) {
      const Job it = job;
      const uint32_t turn = jobs % kTurns;
      const int rows = it.rows;
      bool fresh = true;  // no tile of this item yet
      float top = -INFINITY;  // the maximum in use of row `lane`
      float l[N];             // this thread's share of each row's sum
#pragma unroll
      for (int n = 0; n < N; ++n) l[n] = 0.f;
      const uint32_t last = step + it.tb - it.ta - 1;
      for (int t = it.ta + ((int)(step & 1) ^ wg); t < it.tb; t += 2, ++mine) {
        const int j0 = t * kTileKeys, j = j0 + key;
        const uint32_t g = 2 * mine + wg;  // the CTA's tile
        if (!(ok = tile_wait(s_full, g))) break;
        tc_fence_after();
        const bool there = holds && j < it.kv_len && !(s_bad[g & 15] >> (key >> P.box.shift) & 1);
        uint32_t x[N];
        tmem_ld_cols<N>(ts, x);
        if (fresh && !(ok = meet_warps())) break;  // the item's tables are written
        if (!holds) {
#pragma unroll
          for (int n = 0; n < N; ++n) x[n] = 0xff800000u;
        }
        // the first row sees the least
        if (j0 + kTileKeys > s_lim[wg][turn][0] || !__all_sync(0xffffffffu, there || !holds)) {
#pragma unroll
          for (int n = 0; n < N; ++n)
            if (n < rows && !(there && j < s_lim[wg][turn][n])) x[n] = 0xff800000u;
        }
        float4* const peak = s_max[wg][mine & 1];
#pragma unroll
        for (int n = 0; n < N; n += 4)
          if (n < rows) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float w = warp_max(__uint_as_float(x[n + e]));
              if (lane == n + e) reinterpret_cast<float*>(peak)[4 * (n + e) + ww] = w;
            }
          }
        if (!(ok = meet_warps())) break;
        const float4 w = peak[lane & (N - 1)];
        const float mx = fmaxf(fmaxf(w.x, w.y), fmaxf(w.z, w.w)) * c.scale_log2;
        const bool grows = lane < rows && (mx > top + 8.f || (top == -INFINITY && mx > -INFINITY));
        const float f = grows ? fast_exp2(top - mx) : 1.f;  // 0 for the first maximum
        if (grows) top = mx;
        const float zero = top == -INFINITY ? 0.f : top;
        const bool grow = __any_sync(0xffffffffu, grows);
        // the group's product before has read P and written O; at an item's start, O has been read as well
        if (mine > 0 && !(ok = tile_wait(pv_done, g - 2))) break;
        if (fresh && nitem > 0 && !(ok = warp_wait(read, (nitem - 1) & 1, waits))) break;
        if (!fresh && grow) {  // the same in every thread of the group
          tc_fence_after();
#pragma unroll
          for (int n = 0; n < N; ++n) l[n] *= __shfl_sync(0xffffffffu, f, n);
#pragma unroll 1
          for (int mb = 0; mb < MB; ++mb) {
            uint32_t o[N];
            tmem_ld_cols<N>(to + mb * N, o);
#pragma unroll
            for (int n = 0; n < N; ++n) o[n] = __float_as_uint(__uint_as_float(o[n]) * __shfl_sync(0xffffffffu, f, n));
            tmem_st_cols<N>(to + mb * N, o);
          }
          tc_wait_st();
        }
        fresh = false;
#pragma unroll
        for (int n = 0; n < N; n += 4)
          if (n < rows) {
            float p[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              p[e] = fast_exp2(fmaf(__uint_as_float(x[n + e]), c.scale_log2, -__shfl_sync(0xffffffffu, zero, n + e)));
              l[n + e] += p[e];
            }
            if (holds)
              asm volatile("st.shared.v2.b32 [%0], {%1,%2};" ::"r"(pdst + (n >> 4) * Sh::kPBlock + ((((n >> 3) & 1) ^ ((key >> 2) & 1)) << 4) + (n & 4) * 2),
                           "r"(pack2<BF16>(p[0], p[1])), "r"(pack2<BF16>(p[2], p[3])) : "memory");
          }
        // rows of V past the sequence's end lie in its last page and may hold anything: zero them for 0 * V
        if (j0 + kTileKeys > it.kv_len && it.kv_len % c.page_tokens != 0) {
          for (int s = SHARED ? 1 : kKS; s < kTS; ++s) {
            const uint32_t pos = g * kTS + s, slot = pos % kSlots;
            if (!(ok = warp_wait(full(slot), (pos / kSlots) & 1, waits))) break;
            if (j >= it.kv_len && holds)
              for (int i = 0; i < kKGroups * 8; ++i)
                asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(ring + slot * Sh::kSlotBytes + (i >> 3) * kGroupBytes + key * 128 + (i & 7) * 16),
                             "r"(0) : "memory");
          }
          if (!ok) break;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        tc_fence_before();
        mbar_arrive(p_full + 8 * wg);
      }
      if (!ok) break;
      // the item's last QK^T is done: the next one's Q may come
      if (!(ok = tile_wait(s_full, last)) || !(ok = open())) break;

      // The groups' maxima and sums meet in shared memory; each group then joins and writes its share of the columns
      // (one block of columns: its share of the rows).
      if (fresh && nitem > 0 && !(ok = warp_wait(read, (nitem - 1) & 1, waits))) break;
      {
        const float sum = lane_sums<N>(l, lane);
        if (lane < N) reinterpret_cast<float*>(s_sum[wg])[4 * lane + ww] = sum;
        if (wt < N) s_top[wg][lane] = top;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(summed);
      if (!(ok = warp_wait(summed, nitem & 1, waits))) break;
      float* const part = P.a.part + (int64_t)(2 * blockIdx.x + (it.inside ? 0 : 1)) * P.a.part_floats;
      if (wt < rows) {
        const float4 u = s_sum[0][wt], v = s_sum[1][wt];
        const float m0 = s_top[0][wt], m1 = s_top[1][wt];
        const float mm = fmaxf(m0, m1), z = mm == -INFINITY ? 0.f : mm;
        const float f0 = fast_exp2(m0 - z), f1 = fast_exp2(m1 - z);
        const float sum = ((u.x + u.y) + (u.z + u.w)) * f0 + ((v.x + v.y) + (v.z + v.w)) * f1;
        const float inv = it.whole ? (sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum)) : 1.f;
        s_mix[wg][wt] = make_float2(f0 * inv, f1 * inv);
        if (wg == 0) {
          if (!it.whole) {
            part[P.a.part_rows * c.v_dim + wt] = mm;
            part[P.a.part_rows * (c.v_dim + 1) + wt] = sum;
          } else if (P.a.lse) {
            P.a.lse[s_row[wg][turn][wt]] = sum == 0.f ? -INFINITY : fmaf(mm, 0.693147180559945f, logf(sum));
          }
        }
      }
      if (!(ok = meet_warps())) break;
      if (!(ok = tile_wait(pv_done, last))) break;
      if (last != step && !(ok = tile_wait(pv_done, last - 1))) break;
      tc_fence_after();
#pragma unroll 1
      for (int mb = MB > 1 ? wg : 0; mb < MB; mb += 2) {
        uint32_t o[N], o1[N];
        tmem_ld_cols<N>(tmem + lanes + (2 + mb) * N, o);
        tmem_ld_cols<N>(tmem + lanes + (2 + MB + mb) * N, o1);
        const int col = mb * 128 + wt;
        if (col < c.v_dim) {
#pragma unroll
          for (int n = 0; n < N; n += 4)
            if (n < rows && (MB > 1 || (n / 4 & 1) == wg)) {
              float v[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 w = s_mix[wg][n + e];  // a group without tiles has weight 0 and an O that holds anything
                v[e] = (w.x != 0.f ? __uint_as_float(o[n + e]) * w.x : 0.f) + (w.y != 0.f ? __uint_as_float(o1[n + e]) * w.y : 0.f);
              }
              if (it.whole) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (n + e < rows) P.a.out[s_row[wg][turn][n + e] * c.v_dim + col] = (uint16_t)(pack2<BF16>(v[e], 0.f) & 0xffff);
              } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) part[(n + e) * c.v_dim + col] = v[e];  // rows up to N have room
              }
            }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(read);
      step = last + 1;
      ++nitem;
    }
  }
  __syncthreads();
  if (tid == 0 && waits->dead) P.a.cuts[blockIdx.x].error = 1;
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(Sh::kCols) : "memory");
  }
}

// ---- host -----------------------------------------------------------------------------------------
template <bool BF16, int KG, int MB, int N, bool SHARED>
void launch_kernel(const DecodeParams& P, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t s) {
  auto* const f = attend_decode_kernel<BF16, KG, MB, N, SHARED>;
  constexpr int smem = Shape<KG, MB, N, SHARED>::kSmem;
  cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  f<<<P.a.grid, kThreads, smem, s>>>(P, k, v);
}

template <bool BF16>
void launch_any(const DecodeParams& P, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t s) {
  const CacheParams& c = P.a.c;
  if (!c.v) P.a.part_rows == 16 ? launch_kernel<BF16, 9, 4, 16, true>(P, k, v, s) : launch_kernel<BF16, 9, 4, 32, true>(P, k, v, s);
  else if (c.head_dim <= 64) launch_kernel<BF16, 1, 1, 16, false>(P, k, v, s);
  else if (c.head_dim <= 128) launch_kernel<BF16, 2, 1, 16, false>(P, k, v, s);
  else launch_kernel<BF16, 4, 2, 16, false>(P, k, v, s);
}

}  // namespace

// Single-buffer pools need V to begin at the second column group.
bool attend_decode_fits(const CacheParams& c) { return (c.v ? c.head_dim <= 256 : c.v_col == 64) && pages_fit(c, c.v ? kKeys : 64); }

// Single-buffer pools often have more than 16 heads per KV head: 32 rows an item then, so that K and V are read
// half as often.
AttendShape attend_decode_shape(const CacheParams& c, int sms, int64_t rows) {
  const int n = !c.v && rows > 16 ? 32 : 16;
  return {sms, n, n * (c.v_dim + 2), 0};
}

bool launch_attend_decode(const AttendParams& A, bool bf16, cudaStream_t s) {
  DecodeParams P;
  P.a = A;
  P.box = pool_boxes(A.c, A.c.v ? kKeys : 64);
  CUtensorMap k, v;
  if (!pool_map(&k, A.c.k, A.c, bf16, P.box)) return false;
  v = k;
  if (A.c.v && !pool_map(&v, A.c.v, A.c, bf16, P.box)) return false;
  if (bf16) launch_any<true>(P, k, v, s);
  else launch_any<false>(P, k, v, s);
  return true;
}

}  // namespace ztcp
