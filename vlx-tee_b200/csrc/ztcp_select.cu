// ztcp_select.cu -- choice of the coldest pages and compaction of the block tables (ztcp_select_cold_pages).
//
// Per sequence: of the pages that may leave, the `count` with the least weight, ties to the lower page.  The
// count-th smallest weight is found digit by digit (four passes over 8-bit digits of the weights' order-preserving
// 32-bit images, with histograms in shared memory); pages below it are cold, and of the pages equal to it the first
// ones that are still wanted.  Counts are integers, so the order of atomics changes nothing.  One CTA per sequence;
// a few bytes per page, so the time is that of the passes' barriers, not of memory.
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

// Sum of x over the threads before this one, in warp order; *total over all.  `sums`: one int per warp, free again
// after the caller's next barrier.
__device__ __forceinline__ int flags_before(bool flag, int* sums, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const unsigned m = __ballot_sync(0xffffffffu, flag);
  if (lane == 0) sums[warp] = __popc(m);
  __syncthreads();
  const int x = lane < warps ? sums[lane] : 0;
  const int before = __reduce_add_sync(0xffffffffu, lane < warp ? x : 0);
  *total = __reduce_add_sync(0xffffffffu, x);
  return before + __popc(m & ((1u << lane) - 1));
}

__global__ void __launch_bounds__(1024) select_kernel(const __grid_constant__ ztcp_cold_selection S) {
  __shared__ int hist[256];
  __shared__ int sums[2][32];
  __shared__ long long offs[2];
  __shared__ int digit_s, below_s;
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31;
  const int b = blockIdx.x, P = (int)S.max_pages;
  const Pages me = pages_of(S, b);
  const float* const mass = S.mass + (int64_t)b * P;
  const int32_t* const table = S.block_tables + (int64_t)b * P;

  // where this sequence's cold pages go, and where the last one's end
  if (tid < 2) offs[tid] = 0;
  __syncthreads();
  long long before = 0, all = 0;
  for (int i = tid; i < S.n_seqs; i += nt) {
    const int c = pages_of(S, i).count;
    all += c;
    if (i < b) before += c;
  }
  if (all) {
    atomicAdd((unsigned long long*)&offs[1], (unsigned long long)all);
    if (before) atomicAdd((unsigned long long*)&offs[0], (unsigned long long)before);
  }

  uint32_t prefix = 0, mask = 0;  // the wanted weight's image, as far as it is known
  int want = me.count;            // how many of the pages with this prefix are cold
  if (me.count > 0)
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += nt) hist[i] = 0;
      __syncthreads();
      for (int p = me.lo + tid; p < me.hi; p += nt) {
        const uint32_t u = image(mass[p]);
        if ((u & mask) == prefix) atomicAdd(&hist[(u >> shift) & 255], 1);
      }
      __syncthreads();
      if (tid < 32) {  // the digit in whose bin the want-th smallest lies
        int s = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += hist[lane * 8 + i];
        int inc = s;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int o = __shfl_up_sync(0xffffffffu, inc, d);
          if (lane >= d) inc += o;
        }
        int run = inc - s;
        if (want > run && want <= inc)
          for (int i = 0; i < 8; ++i) {
            const int n = hist[lane * 8 + i];
            if (want <= run + n) {
              digit_s = lane * 8 + i;
              below_s = run;
              break;
            }
            run += n;
          }
      }
      __syncthreads();
      prefix |= (uint32_t)digit_s << shift;
      mask |= 255u << shift;
      want -= below_s;
    }

  __syncthreads();
  const int64_t base = offs[0], end = offs[1];
  int cold_run = 0, tie_run = 0;
  for (int p0 = 0; p0 < P; p0 += nt) {
    const int p = p0 + tid;
    const bool free_page = me.count > 0 && p >= me.lo && p < me.hi;
    const float w = p < me.n ? mass[p] : 0.f;
    const int32_t blk = p < me.n ? table[p] : -1;
    const uint32_t u = image(w);
    const bool tie = free_page && u == prefix;
    int ties, colds;
    const int tie_at = flags_before(tie, sums[0], &ties) + tie_run;
    const bool cold = (free_page && u < prefix) || (tie && tie_at < want);
    const int cold_at = flags_before(cold, sums[1], &colds) + cold_run;
    if (p < me.n) {
      if (cold) {
        S.cold_blocks[base + cold_at] = blk;
        S.cold_index[base + cold_at] = (int32_t)((int64_t)b * P + p);
      } else {
        S.kept_tables[(int64_t)b * P + p - cold_at] = blk;
        S.kept_mass[(int64_t)b * P + p - cold_at] = w;
      }
    }
    if (p < P && p >= me.n - me.count) {  // behind the kept pages
      S.kept_tables[(int64_t)b * P + p] = -1;
      S.kept_mass[(int64_t)b * P + p] = 0.f;
    }
    tie_run += ties;
    cold_run += colds;
    __syncthreads();
  }

  const int64_t room = S.n_seqs * S.max_pages - end;  // the cold lists' unused tail, shared by the CTAs
  for (int64_t i = end + room * b / S.n_seqs + tid, z = end + room * (b + 1) / S.n_seqs; i < z; i += nt) {
    S.cold_blocks[i] = -1;
    S.cold_index[i] = -1;
  }
  if (tid == 0) {
    if (b == 0) S.cold_starts[0] = 0;
    S.cold_starts[b + 1] = (int32_t)(base + me.count);
    S.kept_lens[b] = (int32_t)(me.kv_len - me.count * S.page_tokens);
    S.status[b] = S.kv_lens[b] == me.kv_len ? ZTCP_SEQ_OK : ZTCP_SEQ_BAD_LENGTH;
  }
}

}  // namespace

void launch_select(const ztcp_cold_selection& S, cudaStream_t s) {
  select_kernel<<<(unsigned)S.n_seqs, S.max_pages <= 256 ? 256 : (S.max_pages <= 512 ? 512 : 1024), 0, s>>>(S);
}

}  // namespace ztcp
