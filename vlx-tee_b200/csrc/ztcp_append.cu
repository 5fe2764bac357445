// ztcp_append.cu -- norm, rotation and append of new tokens to the paged pool (ztcp_append_tokens).
//
// Mathematics.  Per query and key vector x: y = x * w / sqrt(mean(x^2) + eps) over the normed columns, then the
// leading rope_dim columns turn by the token's angles: (a, b) -> (a cos - b sin, b cos + a sin).  fp32 throughout,
// rounded once.
//
// A pass that is bound by memory: every vector is read once and written once, 16 bytes per lane.  A CTA takes one
// token (several CTAs share one where there are few) and a group of lanes one vector at a time: 8, 16 or 32 lanes,
// each with CH chunks of 8 columns, CH * lanes covering head_dim.  A pair's two columns lie in one chunk
// (interleaved) or in chunks rope_dim / 16 lanes apart, which trade values by shuffles; the token's cosines and
// sines stay in registers over its heads.
#include "ztcp_kvcache.cuh"
#include "../../include/ztcp_kvcache.h"

namespace ztcp {

namespace {

constexpr int kThreads = 256;

template <bool BF16>
__device__ __forceinline__ void unpack8(const uint4& v, float x[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2<BF16>(w[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

template <bool BF16, int GROUP, int CH>
__global__ void __launch_bounds__(kThreads) append_kernel(const __grid_constant__ ztcp_append A, int32_t* status) {
  constexpr int kGroups = kThreads / GROUP;
  const int tok = blockIdx.x;
  const int lane = threadIdx.x % GROUP, grp = threadIdx.x / GROUP + blockIdx.y * kGroups, step = kGroups * gridDim.y;
  const int D = (int)A.geom.head_dim, R = (int)A.geom.rope_dim, T = (int)A.geom.num_tokens;
  const int nk = (int)A.geom.num_heads, nq = A.q ? (int)A.num_q_heads : 0, nv = A.v ? nk : 0;

  const int32_t pos = R > 0 ? __ldg(A.positions + tok) : 0;
  const int64_t slot = __ldg(A.slots + tok);
  const bool bad_pos = R > 0 && (pos < 0 || pos >= A.max_pos);
  const bool bad_slot = slot < -1 || slot >= A.pool_pages * T;
  if (threadIdx.x == 0 && blockIdx.y == 0) status[tok] = bad_pos || bad_slot ? ZTCP_SEQ_BAD_BLOCK : ZTCP_SEQ_OK;
  if (bad_pos) return;
  const bool keep = slot >= 0 && !bad_slot;

  // The lane's chunk of rotated columns is its first one: rope_dim <= 8 * GROUP.
  const bool turns = lane * 8 < R;
  const int half = R / 16;  // lanes to a pair's other half
  float cs[8], sn[8];
  if (turns) {
    const float* const row = A.rope_table + (int64_t)pos * R;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int a = A.interleaved ? lane * 4 + i / 2 : (lane < half ? lane * 8 + i : (lane - half) * 8 + i);
      cs[i] = __ldg(row + a);
      sn[i] = __ldg(row + R / 2 + a);
    }
  }

  const int total = nq + (keep ? nk + nv : 0);
  for (int i = grp; i < total; i += step) {  // a group's lanes stay together
    const int kind = i < nq ? 0 : (i < nq + nk ? 1 : 2);
    const int h = kind == 0 ? i : (kind == 1 ? i - nq : i - nq - nk);
    const uint16_t* src;
    uint16_t* dst;
    if (kind == 0) {
      src = (const uint16_t*)A.q + tok * A.q_token_stride + h * A.q_head_stride;
      dst = (uint16_t*)A.q_out + ((int64_t)tok * nq + h) * D;
    } else if (kind == 1) {
      src = (const uint16_t*)A.k + tok * A.k_token_stride + h * A.k_head_stride;
      dst = (uint16_t*)A.k_pool + (slot * nk + h) * D;
    } else {
      src = (const uint16_t*)A.v + tok * A.v_token_stride + h * A.v_head_stride;
      dst = (uint16_t*)A.v_pool + (slot * nk + h) * D;
    }
    uint4 raw[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c)
      if ((lane + c * GROUP) * 8 < D) raw[c] = *reinterpret_cast<const uint4*>(src + (lane + c * GROUP) * 8);
    if (kind == 2) {
#pragma unroll
      for (int c = 0; c < CH; ++c)
        if ((lane + c * GROUP) * 8 < D) *reinterpret_cast<uint4*>(dst + (lane + c * GROUP) * 8) = raw[c];
      continue;
    }
    const unsigned mask = GROUP == 32 ? 0xffffffffu : ((1u << GROUP) - 1) << (threadIdx.x % 32 / GROUP * GROUP);
    float x[CH][8];
    float ss = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = (lane + c * GROUP) * 8;
      if (col < D) unpack8<BF16>(raw[c], x[c]);
      if (col >= A.norm_from && col < D)
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(x[c][e], x[c][e], ss);
    }
    const float* const w = kind == 0 ? A.q_weight : A.k_weight;
    if (w) {
#pragma unroll
      for (int d = GROUP / 2; d > 0; d >>= 1) ss += __shfl_xor_sync(mask, ss, d);
      const float r = 1.f / sqrtf(ss / (float)(D - A.norm_from) + A.eps);
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int col = (lane + c * GROUP) * 8;
        if (col >= A.norm_from && col < D)
#pragma unroll
          for (int e = 0; e < 8; ++e) x[c][e] = x[c][e] * r * __ldg(w + col - A.norm_from + e);
      }
    }
    if (R > 0) {
      if (A.interleaved) {
        if (turns)
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const float a = x[0][e], b = x[0][e + 1];
            x[0][e] = a * cs[e] - b * sn[e];
            x[0][e + 1] = b * cs[e] + a * sn[e];
          }
      } else {
        const int other = lane < half ? lane + half : (lane < 2 * half ? lane - half : lane);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float y = __shfl_sync(mask, x[0][e], other, GROUP);
          if (turns) x[0][e] = lane < half ? x[0][e] * cs[e] - y * sn[e] : x[0][e] * cs[e] + y * sn[e];
        }
      }
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = (lane + c * GROUP) * 8;
      if (col < D)
        *reinterpret_cast<uint4*>(dst + col) =
            make_uint4(pack2<BF16>(x[c][0], x[c][1]), pack2<BF16>(x[c][2], x[c][3]), pack2<BF16>(x[c][4], x[c][5]), pack2<BF16>(x[c][6], x[c][7]));
    }
  }
}

template <int GROUP, int CH>
void launch_group(const ztcp_append& A, int32_t* status, int sms, cudaStream_t s) {
  const int64_t vectors = (A.q ? A.num_q_heads : 0) + (A.v ? 2 : 1) * A.geom.num_heads;
  const int64_t most = (vectors + kThreads / GROUP - 1) / (kThreads / GROUP);
  // few tokens: several CTAs share one, so that its vectors are in flight on more SMs
  int64_t y = A.n_tokens >= 2 * sms ? 1 : (2 * sms + A.n_tokens - 1) / A.n_tokens;
  if (y > most) y = most;
  const dim3 grid((unsigned)A.n_tokens, (unsigned)y);
  if (A.dtype == ZTCP_DTYPE_BF16) append_kernel<true, GROUP, CH><<<grid, kThreads, 0, s>>>(A, status);
  else append_kernel<false, GROUP, CH><<<grid, kThreads, 0, s>>>(A, status);
}

}  // namespace

void launch_append(const ztcp_append& A, int32_t* status, cudaStream_t s) {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return;
  const int64_t D = A.geom.head_dim;
  if (D <= 64) launch_group<8, 1>(A, status, sms, s);
  else if (D <= 128) launch_group<16, 1>(A, status, sms, s);
  else if (D <= 256) launch_group<32, 1>(A, status, sms, s);
  else if (D <= 768) launch_group<32, 3>(A, status, sms, s);
  else launch_group<32, 4>(A, status, sms, s);
}

}  // namespace ztcp
