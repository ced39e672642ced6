// Attention over whole prompts: packed sequences, grouped heads, causal.
#include "serve.hpp"

namespace ohip {

// A block has 128 query rows of one head, 32 a wave, and walks the keys they
// see in tiles of 64 that all its waves share through LDS.  S^T = K Q^T, so a
// lane holds one query (its column) and the softmax's running maximum and sum
// need one exchange between a lane and the one 32 further; O^T = V^T P^T takes
// P as it lies in the registers: k index 8 h + j (h = lane / 32) stands for
// key 4 h + j of a block of 8, then of the next.
constexpr int kPrefillQ = 128, kPrefillK = 64;

// Which sequence a block's tile belongs to.  Sequence i has the tile slots
// from cu[i] / BQ + i on (at least as many as it has tiles), so that the grid
// needs only the totals; a slot past its sequence's end has nothing to do.
// One wave searches; offsets that are not ascending cannot lead outside
// [0, total].
__device__ __forceinline__ int slot_sequence(const int32_t* cu, int seqs, int64_t total, int tile, int bq) {
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int i0 = 0; i0 < seqs; i0 += 64) {
    const int i = i0 + lane;
    const int64_t c = i < seqs ? min(max((int64_t)cu[i], (int64_t)0), total) : 0;
    n += __popcll(__ballot(i < seqs && c / bq + i <= tile));
  }
  return n - 1;
}

template <class T, int D>
__global__ void __launch_bounds__(256)
attn_prefill_kernel(const AttnPrefillArgs p) {
  constexpr int BQ = kPrefillQ, BK = kPrefillK, KS = D / 16, OT = D / 32, RS = D + 8;
  __shared__ __align__(16) T ks[BK][RS], vs[BK][RS];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 31, h2 = lane >> 5;
  // heads of one key head next to each other in time, key heads eight apart: an XCD's L2 holds its own
  const int kvh = blockIdx.x % p.kv, head = kvh * p.g + blockIdx.x / p.kv;
  const int tile = (int)gridDim.y - 1 - (int)blockIdx.y;   // late tiles of a sequence see the most keys
  const int seq = slot_sequence(p.cu_q, p.seqs, p.q_tokens, tile, BQ);
  if (seq < 0) return;
  const int64_t q0 = min(max((int64_t)p.cu_q[seq], (int64_t)0), p.q_tokens);
  const int64_t q1 = min(max((int64_t)p.cu_q[seq + 1], q0), p.q_tokens);
  const int64_t k0 = min(max((int64_t)p.cu_k[seq], (int64_t)0), p.k_tokens);
  const int64_t k1 = min(max((int64_t)p.cu_k[seq + 1], k0), p.k_tokens);
  const int nq = (int)(q1 - q0), nk = (int)(k1 - k0);
  const int64_t first = (int64_t)(tile - (q0 / BQ + seq)) * BQ;
  if (first < 0 || first >= nq) return;
  const int qt = (int)first;
  const int qi = qt + wave * 32 + r;           // this lane's query
  const int shift = nk - nq;                   // query i stands at key place i + shift
  const int qrows = min(BQ, nq - qt);
  int kend = nk, kbeg = 0;
  if (p.causal) kend = min(nk, max(0, qt + qrows + shift));
  if (p.window > 0) kbeg = max(0, qt + shift - p.window + 1) / BK * BK;

  u32x4 qf[KS];
  {
    const T* src = static_cast<const T*>(p.q) + (q0 + min(qi, nq - 1)) * p.ldq + (int64_t)head * p.dim;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int ch = 16 * s + 8 * h2;
      qf[s] = u32x4{0, 0, 0, 0};
      if (ch < p.dim) __builtin_memcpy(&qf[s], __builtin_assume_aligned(src + ch, 16), 16);
    }
  }
  f32x16 o[OT];
#pragma unroll
  for (int t = 0; t < OT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[t][i] = 0.0f;
  float mx = -__builtin_inff(), l = 0.0f;
  const T* kb = static_cast<const T*>(p.k) + k0 * p.ldk + (int64_t)kvh * p.dim;
  const T* vb = static_cast<const T*>(p.v) + k0 * p.ldv + (int64_t)kvh * p.dim;

  for (int kt = kbeg; kt < kend; kt += BK) {
    __syncthreads();
    for (int i = threadIdx.x; i < BK * (D / 8); i += 256) {
      const int row = i / (D / 8), ch = i % (D / 8) * 8;
      u32x4 kv = u32x4{0, 0, 0, 0}, vv = u32x4{0, 0, 0, 0};   // rows of no key: finite
      if (kt + row < nk && ch < p.dim) {
        __builtin_memcpy(&kv, __builtin_assume_aligned(kb + (int64_t)(kt + row) * p.ldk + ch, 16), 16);
        __builtin_memcpy(&vv, __builtin_assume_aligned(vb + (int64_t)(kt + row) * p.ldv + ch, 16), 16);
      }
      *reinterpret_cast<u32x4*>(&ks[row][ch]) = kv;
      *reinterpret_cast<u32x4*>(&vs[row][ch]) = vv;
    }
    __syncthreads();
    f32x16 s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[t][i] = 0.0f;
#pragma unroll
      for (int k = 0; k < KS; ++k)
        s[t] = mma32<T>(*reinterpret_cast<const u32x4*>(&ks[32 * t + r][16 * k + 8 * h2]), qf[k], s[t]);
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int key = kt + 32 * t + 8 * (i / 4) + 4 * h2 + i % 4;
        const bool sees = key < nk && (!p.causal || key <= qi + shift) && (p.window <= 0 || key > qi + shift - p.window);
        if (!sees) s[t][i] = -__builtin_inff();
      }
    float m = s[0][0];
#pragma unroll
    for (int i = 0; i < 32; ++i) m = __builtin_fmaxf(m, s[i / 16][i % 16]);
    m = __builtin_fmaxf(m, __shfl_xor(m, 32, 64));
    const float now = __builtin_fmaxf(mx, m);
    const float base = now == -__builtin_inff() ? 0.0f : now;
    const float keep = __builtin_amdgcn_exp2f((mx - base) * p.c);
    mx = now;
    l *= keep;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[t][i] = __builtin_amdgcn_exp2f((s[t][i] - base) * p.c);
        l += s[t][i];
      }
#pragma unroll
    for (int t = 0; t < OT; ++t) o[t] *= keep;
#pragma unroll
    for (int k = 0; k < 4; ++k) {   // 16 keys
      u32x4 pf;
#pragma unroll
      for (int j = 0; j < 4; ++j) pf[j] = pack2<T>(s[k / 2][8 * (k % 2) + 2 * j], s[k / 2][8 * (k % 2) + 2 * j + 1]);
#pragma unroll
      for (int t = 0; t < OT; ++t) {
        T e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = vs[16 * k + 8 * (j / 4) + 4 * h2 + j % 4][32 * t + r];
        o[t] = mma32<T>(__builtin_bit_cast(u32x4, e), pf, o[t]);
      }
    }
  }
  l += __shfl_xor(l, 32, 64);
  if (qi >= nq) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;   // a row that sees no key: zeros
  T* dst = static_cast<T*>(p.out) + (q0 + qi) * p.ldo + (int64_t)head * p.dim;
#pragma unroll
  for (int t = 0; t < OT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int ch = 32 * t + 8 * (i / 4) + 4 * h2 + i % 4;
      if (ch < p.dim) dst[ch] = (T)(o[t][i] * inv);
    }
}

template <class T> static hipError_t prefill_t(const AttnPrefillArgs& p, hipStream_t st) {
  const dim3 grid((unsigned)(p.kv * p.g), (unsigned)(p.q_tokens / kPrefillQ + p.seqs)), block(256);
  if (p.dim <= 64) hipLaunchKernelGGL((attn_prefill_kernel<T, 64>), grid, block, 0, st, p);
  else if (p.dim <= 96) hipLaunchKernelGGL((attn_prefill_kernel<T, 96>), grid, block, 0, st, p);
  else if (p.dim <= 128) hipLaunchKernelGGL((attn_prefill_kernel<T, 128>), grid, block, 0, st, p);
  else return hipErrorInvalidValue;
  return hipGetLastError();
}
hipError_t run_attn_prefill(int dtype, const AttnPrefillArgs& p, hipStream_t st) {
  return dtype == DT_F16 ? prefill_t<_Float16>(p, st) : dtype == DT_BF16 ? prefill_t<__bf16>(p, st) : hipErrorInvalidValue;
}

}  // namespace ohip
