// ztcp_select.cu -- choice of the coldest pages and compaction of the block tables (ztcp_select_cold_pages).
//
// Per sequence: of the pages that may leave, the `count` with the least weight, ties to the lower page.  The
// count-th smallest weight is found digit by digit among the bits in which the weights differ (of their
// order-preserving 32-bit images, with a histogram in shared memory, a bin per thread), until the digits so far tell
// the cold pages from the others: two passes for most weights, four at most.  Pages below it are cold, and of the pages
// equal to it the first ones that are still wanted.  Counts are integers, so the order of atomics changes nothing.  One
// CTA per sequence; a thread holds four neighbouring pages, so that up to 4,096 pages are read once and placed by one
// scan.  A few bytes per page, so the time is that of the passes' barriers, not of memory.
// Measured in a graph of calls: one sequence of 256 pages 4.7 us (an empty kernel takes 2.5), 64 sequences of up to 4,096
// pages 10.5 (6.2 and 12.3 as calls in a stream); with four passes of 8-bit digits that each read the weights again, and
// a scan per 1,024 pages, 5.3 and 16.3.
#include "ztcp_kvcache.cuh"
#include "../../include/ztcp_kvcache.h"

namespace ztcp {

namespace {

// Order-preserving image of a weight: -0 equals 0, a NaN is above every number.
__device__ __forceinline__ uint32_t image(float x) {
  if (isnan(x)) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct Pages {
  int32_t n, count, lo, hi, kv_len;  // pages, cold ones, and the range that they come from
};
__device__ __forceinline__ Pages pages_of(const ztcp_cold_selection& S, int64_t b) {
  Pages p;
  const int64_t cap = S.max_pages * S.page_tokens;
  int64_t len = S.kv_lens[b];
  len = len < 0 ? 0 : (len > cap ? cap : len);
  p.kv_len = (int32_t)len;
  const int64_t n = (len + S.page_tokens - 1) / S.page_tokens;
  int64_t lo = S.sink, hi = n - S.recent, c = n - S.keep;
  if (hi < lo) hi = lo;
  if (c > hi - lo) c = hi - lo;
  p.n = (int32_t)n;
  p.count = c > 0 ? (int32_t)c : 0;
  p.lo = (int32_t)(lo < n ? lo : n);
  p.hi = (int32_t)(hi < n ? hi : n);
  return p;
}

constexpr int kPer = 4;  // pages of a thread

// Sum of x over the threads before this one; *total over all.  `sums`: one int per warp, free again after the caller's
// next barrier.
__device__ __forceinline__ int sum_before(int x, int* sums, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int inc = x;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += o;
  }
  if (lane == 31) sums[warp] = inc;
  __syncthreads();
  const int y = lane < warps ? sums[lane] : 0;
  const int before = __reduce_add_sync(0xffffffffu, lane < warp ? y : 0);
  *total = __reduce_add_sync(0xffffffffu, y);
  return before + inc - x;
}

// Where every sequence's cold pages begin, found beforehand for large batches: each CTA adding up all counts itself takes
// time in proportion to the batch's square.  Measured with 256 pages a sequence, by each CTA / beforehand: 256 sequences
// 6.2 / 7.5 us, 512 8.2 / 8.8, 1,024 15.5 / 13.3, 4,096 79 / 38; 262,144 of 4 pages 180 / 2.3 ms.
constexpr int kManySeqs = 512;

__global__ void __launch_bounds__(1024) select_starts_kernel(const __grid_constant__ ztcp_cold_selection S) {
  __shared__ int sums[2][32];  // by turns, so that one barrier a step is enough
  int run = 0;                 // fewer than 2^31 pages in all
  for (int64_t b0 = 0, turn = 0; b0 < S.n_seqs; b0 += 1024, turn ^= 1) {
    const int64_t b = b0 + threadIdx.x;
    const int c = b < S.n_seqs ? pages_of(S, b).count : 0;
    int total;
    const int before = sum_before(c, sums[turn], &total);
    if (b < S.n_seqs) S.cold_starts[b + 1] = run + before + c;
    run += total;
  }
  if (threadIdx.x == 0) S.cold_starts[0] = 0;
}

template <int BITS>  // of a digit: as many bins as threads
__global__ void __launch_bounds__(1 << BITS) select_kernel(const __grid_constant__ ztcp_cold_selection S) {
  constexpr int nt = 1 << BITS, kChunk = nt * kPer;
  __shared__ int hist[nt];
  __shared__ int sums[2][32];
  __shared__ long long offs[2];
  __shared__ uint32_t least_s, most_s;
  __shared__ int digit_s, below_s, in_s;
  const int tid = threadIdx.x;
  const int b = blockIdx.x, P = (int)S.max_pages;
  const Pages me = pages_of(S, b);
  const float* const mass = S.mass + (int64_t)b * P;
  const int32_t* const table = S.block_tables + (int64_t)b * P;
  const bool held = P <= kChunk;  // the pages are read once

  float w[kPer];
  int32_t blk[kPer];
  auto load = [&](int p0, bool blocks) {
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int p = p0 + tid * kPer + e;
      w[e] = p < me.n ? mass[p] : 0.f;
      if (blocks) blk[e] = p < me.n ? table[p] : -1;
    }
  };
  load(0, held);

  // where this sequence's cold pages go, and where the last one's end
  if (tid < 2) offs[tid] = 0;
  if (tid == 0) least_s = 0xffffffffu, most_s = 0;
  hist[tid] = 0;
  __syncthreads();
  const bool many = S.n_seqs > kManySeqs;
  if (many && tid < 2) offs[tid] = S.cold_starts[tid == 0 ? b : S.n_seqs];
  long long before = 0, all = 0;
  for (int i = tid; !many && i < S.n_seqs; i += nt) {
    const int c = pages_of(S, i).count;
    all += c;
    if (i < b) before += c;
  }
  if (!many && tid - (tid & 31) < S.n_seqs) {  // one 64-bit atomic a warp: from every thread they took 4 us (64 sequences)
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
      all += __shfl_xor_sync(0xffffffffu, all, d);
      before += __shfl_xor_sync(0xffffffffu, before, d);
    }
    if ((tid & 31) == 0) {
      atomicAdd((unsigned long long*)&offs[1], (unsigned long long)all);
      atomicAdd((unsigned long long*)&offs[0], (unsigned long long)before);
    }
  }

  // f(image) of the pages that may leave
  auto each = [&](auto f) {
    for (int p0 = 0; p0 < me.hi; p0 += kChunk) {
      if (!held) load(p0, false);
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const int p = p0 + tid * kPer + e;
        if (p >= me.lo && p < me.hi) f(image(w[e]));
      }
    }
  };
  uint32_t prefix = 0, mask = 0;  // the wanted weight's image, as far as it is known
  int want = me.count;            // how many of the pages with this prefix are cold
  bool whole = false;             // all of them
  if (me.count > 0) {
    uint32_t least = 0xffffffffu, most = 0;
    each([&](uint32_t u) { least = min(least, u), most = max(most, u); });
    least = __reduce_min_sync(0xffffffffu, least);
    most = __reduce_max_sync(0xffffffffu, most);
    if ((tid & 31) == 0) {
      atomicMin(&least_s, least);
      atomicMax(&most_s, most);
    }
    __syncthreads();
    int bits = 32 - __clz(least_s ^ most_s);  // 0: all alike
    mask = bits == 32 ? 0 : 0xffffffffu << bits;
    prefix = least_s & mask;
    while (bits > 0 && !whole) {
      const int shift = bits > BITS ? bits - BITS : 0;
      const uint32_t low = (1u << (bits - shift)) - 1;
      each([&](uint32_t u) {
        if ((u & mask) == prefix) atomicAdd(&hist[(u >> shift) & low], 1);
      });
      __syncthreads();
      const int n = hist[tid];
      int total;
      const int run = sum_before(n, sums[0], &total);
      if (want > run && want <= run + n) {  // the bin of the want-th smallest
        digit_s = tid;
        below_s = run;
        in_s = n;
      }
      hist[tid] = 0;
      __syncthreads();
      prefix |= (uint32_t)digit_s << shift;
      mask |= low << shift;
      want -= below_s;
      whole = want == in_s;
      bits = shift;
    }
  }

  __syncthreads();
  const int64_t base = offs[0], end = offs[1];
  int below_run = 0, tie_run = 0;
  for (int p0 = 0; p0 < P; p0 += kChunk) {
    if (!held) load(p0, true);
    int count = 0;  // pages below the prefix, and those with it << 16 (a chunk has at most 4,096)
    bool below[kPer], tie[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int p = p0 + tid * kPer + e;
      const bool may = me.count > 0 && p >= me.lo && p < me.hi;
      const uint32_t u = image(w[e]) & mask;
      below[e] = may && u < prefix;
      tie[e] = may && u == prefix;
      count += (int)below[e] + ((int)tie[e] << 16);
    }
    int total;
    const int at = sum_before(count, sums[1], &total);
    int belows = below_run + (at & 0xffff), ties = tie_run + (at >> 16);
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int p = p0 + tid * kPer + e;
      const bool cold = below[e] || (tie[e] && ties < want);
      const int cold_at = belows + min(ties, want);  // cold pages before this one
      if (p < me.n) {
        if (cold) {
          S.cold_blocks[base + cold_at] = blk[e];
          S.cold_index[base + cold_at] = (int32_t)((int64_t)b * P + p);
        } else {
          S.kept_tables[(int64_t)b * P + p - cold_at] = blk[e];
          S.kept_mass[(int64_t)b * P + p - cold_at] = w[e];
        }
      }
      if (p < P && p >= me.n - me.count) {  // behind the kept pages
        S.kept_tables[(int64_t)b * P + p] = -1;
        S.kept_mass[(int64_t)b * P + p] = 0.f;
      }
      belows += below[e];
      ties += tie[e];
    }
    below_run += total & 0xffff;
    tie_run += total >> 16;
    __syncthreads();
  }

  const int64_t room = S.n_seqs * S.max_pages - end;  // the cold lists' unused tail, shared by the CTAs
  for (int64_t i = end + room * b / S.n_seqs + tid, z = end + room * (b + 1) / S.n_seqs; i < z; i += nt) {
    S.cold_blocks[i] = -1;
    S.cold_index[i] = -1;
  }
  if (tid == 0) {
    if (!many) {
      if (b == 0) S.cold_starts[0] = 0;
      S.cold_starts[b + 1] = (int32_t)(base + me.count);
    }
    S.kept_lens[b] = (int32_t)(me.kv_len - me.count * S.page_tokens);
    S.status[b] = S.kv_lens[b] == me.kv_len ? ZTCP_SEQ_OK : ZTCP_SEQ_BAD_LENGTH;
  }
}

}  // namespace

void launch_select(const ztcp_cold_selection& S, cudaStream_t s) {
  const unsigned n = (unsigned)S.n_seqs;
  if (S.n_seqs > kManySeqs) select_starts_kernel<<<1, 1024, 0, s>>>(S);
  if (S.max_pages <= 256 * kPer) select_kernel<8><<<n, 256, 0, s>>>(S);
  else if (S.max_pages <= 512 * kPer) select_kernel<9><<<n, 512, 0, s>>>(S);
  else select_kernel<10><<<n, 1024, 0, s>>>(S);
}

}  // namespace ztcp
