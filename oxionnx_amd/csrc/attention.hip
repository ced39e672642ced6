// Attention over whole prompts: packed sequences, grouped heads, causal.
#include "serve.hpp"

namespace ohip {

// A block has BQ = 32 * NW * QB query rows of one head, QB blocks of 32 a wave,
// and walks the keys they see in tiles of 64 that all its waves share through
// LDS.  S^T = K Q^T, so a lane holds one query (its column) and the softmax's
// running maximum and sum need one exchange between a lane and the one 32
// further; O^T = V^T P^T takes P as it lies in the registers: k index 8 h + j
// (h = lane / 32) stands for key 4 h + j of a block of 8, then of the next,
// and V's fragments come from LDS through the transposing read.
//
// LDS: two buffers of a K and a V tile.  Each thread loads its part of tile
// t + 1 into registers before the products of tile t and stores it to LDS
// after them, so one barrier a tile is enough.  (Loads that write LDS directly
// save the registers, but the compiler waits for all of them before any
// transposing read.)  Rows past the sequence's end and channels past the head
// read as zeros (the buffer's range check).
constexpr int kPrefillK = 64;

// Slot of 16-byte chunk c of a staged row r: rows of 16 (8) chunks, XOR with a
// permutation of r's low bits that puts 16 consecutive rows of one chunk (the
// K fragments) and four rows of four chunks (a transposing read) in different
// bank groups.
template <int CH> __device__ __forceinline__ int row_swizzle(int r) {
  if constexpr (CH == 16) return ((r & 3) << 2) | ((r >> 2) & 3);
  else return ((r & 2) << 1) | ((r >> 2) & 3);
}

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

typedef short s16x4 __attribute__((ext_vector_type(4)));

template <class T, int D, int NW, int QB>
__global__ void __launch_bounds__(64 * NW, QB == 1 ? 2 : 1)
attn_prefill_kernel(const AttnPrefillArgs p) {
  constexpr int BQ = 32 * NW * QB, BK = kPrefillK, KS = D / 16, OT = D / 32;
  constexpr int CH = D > 64 ? 16 : 8, RB = CH * 16;     // chunks and bytes of a staged row
  constexpr int NL = BK * CH / (64 * NW);               // loads a thread of a tile
  constexpr int kTile = BK * RB;
  static_assert(NL >= 1 && (64 / CH) * NW % 16 == 0, "a thread's loads share their swizzle");
  __shared__ __align__(16) char lds[2][2][kTile];       // [buffer][K, V]
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
  const int shift = nk - nq;                   // query i stands at key place i + shift
  const int qrows = min(BQ, nq - qt);
  int kend = nk, kbeg = 0;
  if (p.causal) kend = min(nk, max(0, qt + qrows + shift));
  if (p.window > 0) kbeg = max(0, qt + shift - p.window + 1) / BK * BK;
  // this wave's queries qw .. qw + 32 QB - 1; its lanes' are qw + 32 b + r
  const int qw = qt + wave * 32 * QB;
  const int wend = p.causal ? min(nk, min(qw + 32 * QB, nq) + shift) : nk;   // keys that any of them sees
  const bool idle = qw >= nq;

  u32x4 qf[QB][KS];
#pragma unroll
  for (int b = 0; b < QB; ++b) {
    const T* src = static_cast<const T*>(p.q) + (q0 + min(qw + 32 * b + r, nq - 1)) * p.ldq + (int64_t)head * p.dim;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int ch = 16 * s + 8 * h2;
      qf[b][s] = u32x4{0, 0, 0, 0};
      if (ch < p.dim) __builtin_memcpy(&qf[b][s], __builtin_assume_aligned(src + ch, 16), 16);
    }
  }
  f32x16 o[QB][OT];
  float mx[QB], l[QB];
#pragma unroll
  for (int b = 0; b < QB; ++b) {
    mx[b] = -__builtin_inff();
    l[b] = 0.0f;
#pragma unroll
    for (int t = 0; t < OT; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[b][t][i] = 0.0f;
  }
  const char* kb = static_cast<const char*>(p.k) + (k0 * p.ldk + (int64_t)kvh * p.dim) * 2;
  const char* vb = static_cast<const char*>(p.v) + (k0 * p.ldv + (int64_t)kvh * p.dim) * 2;
  // this thread's loads: row (i * NW + wave) * (64 / CH) + lane / CH, slot lane % CH
  const int lrow = wave * (64 / CH) + lane / CH;
  const int chunk = (lane % CH) ^ row_swizzle<CH>(lrow);
  const bool inside = chunk * 8 < p.dim;
  const int kvoff = inside ? (int)(lrow * p.ldk * 2) + chunk * 16 : (int)0x80000000u;
  const int vvoff = inside ? (int)(lrow * p.ldv * 2) + chunk * 16 : (int)0x80000000u;
  const int kstep = (int)(NW * (64 / CH) * p.ldk * 2), vstep = (int)(NW * (64 / CH) * p.ldv * 2);
  u32x4 kin[NL], vin[NL];
  auto fetch = [&](int kt) __attribute__((always_inline)) {
    const int rows = min(nk - kt, BK);   // > 0: rows of the sequence from kt on
    const auto kr = rows_resource(kb + (int64_t)kt * p.ldk * 2, (int)((rows - 1) * p.ldk + p.dim) * 2);
    const auto vr = rows_resource(vb + (int64_t)kt * p.ldv * 2, (int)((rows - 1) * p.ldv + p.dim) * 2);
#pragma unroll
    for (int i = 0; i < NL; ++i) kin[i] = __builtin_amdgcn_raw_buffer_load_b128(kr, kvoff + i * kstep, 0, 0);
#pragma unroll
    for (int i = 0; i < NL; ++i) vin[i] = __builtin_amdgcn_raw_buffer_load_b128(vr, vvoff + i * vstep, 0, 0);
  };
  char* const mine = lds[0][0] + threadIdx.x * 16;
  auto put = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NL; ++i) *reinterpret_cast<u32x4*>(mine + buf * 2 * kTile + i * NW * 1024) = kin[i];
#pragma unroll
    for (int i = 0; i < NL; ++i) *reinterpret_cast<u32x4*>(mine + (buf * 2 + 1) * kTile + i * NW * 1024) = vin[i];
  };
  // fragment addresses: K row r chunk 2 s + h2; V keys 4 h2 + (lane % 16) / 4 on, channels 16 ((lane / 16) % 2) + 4 (lane % 4)
  const int ksw = row_swizzle<CH>(r);
  const int vrow = 4 * h2 + (lane & 15) / 4, vch = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), vby = 8 * (lane & 1);

  auto tile_pass = [&](int kt, int buf) __attribute__((always_inline)) {
    const char* ks = lds[buf][0];
    const char* vs = lds[buf][1];
    f32x16 s[QB][2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int b = 0; b < QB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[b][t][i] = 0.0f;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const u32x4 f = *reinterpret_cast<const u32x4*>(ks + (32 * t + r) * RB + (((2 * k + h2) ^ ksw) * 16));
#pragma unroll
        for (int b = 0; b < QB; ++b) s[b][t] = mma32<T>(f, qf[b][k], s[b][t]);
      }
    }
    u32x4 pf[QB][4];
#pragma unroll
    for (int b = 0; b < QB; ++b) {
      const int qi = qw + 32 * b;   // the block's first query
      if (kt + BK > nk || (p.causal && kt + BK - 1 > qi + shift) || (p.window > 0 && kt <= qi + 31 + shift - p.window)) {
        const int last = p.causal ? min(nk - 1, qi + r + shift) : nk - 1;
        const int low = p.window > 0 ? qi + r + shift - p.window : -1;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int key = kt + 32 * t + 8 * (i / 4) + 4 * h2 + i % 4;
            if (key > last || key <= low) s[b][t][i] = -__builtin_inff();
          }
      }
      float m = s[b][0][0];
#pragma unroll
      for (int i = 1; i < 32; ++i) m = __builtin_fmaxf(m, s[b][i / 16][i % 16]);
      m = max_halves(m);
      if (__any(m > mx[b])) {
        const float now = __builtin_fmaxf(mx[b], m);
        const float keep = now == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f((mx[b] - now) * p.c);
        mx[b] = now;
        l[b] *= keep;
#pragma unroll
        for (int t = 0; t < OT; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[b][t][i] *= keep;
      }
      const float base = mx[b] == -__builtin_inff() ? 0.0f : mx[b] * p.c;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[b][t][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][t][i], p.c, -base));
          l[b] += s[b][t][i];
        }
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          pf[b][k][j] = pack2<T>(s[b][k / 2][8 * (k % 2) + 2 * j], s[b][k / 2][8 * (k % 2) + 2 * j + 1]);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)   // 16 keys
#pragma unroll
      for (int t = 0; t < OT; ++t) {
        u32x4 f;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int row = 16 * k + 8 * j + vrow;
          const char* at = vs + row * RB + (((4 * t + vch) ^ row_swizzle<CH>(row)) * 16) + vby;
          const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(at));
          const u32x2 w = __builtin_bit_cast(u32x2, v);
          f[2 * j] = w.x;
          f[2 * j + 1] = w.y;
        }
#pragma unroll
        for (int b = 0; b < QB; ++b) o[b][t] = mma32<T>(f, pf[b][k], o[b][t]);
      }
  };

  if (kbeg < kend) {
    fetch(kbeg);
    put(0);
  }
  int buf = 0;
  for (int kt = kbeg; kt < kend; kt += BK, buf ^= 1) {
    const bool more = kt + BK < kend;
    lds_barrier();
    if (more) fetch(kt + BK);
    if (!idle && kt < wend) tile_pass(kt, buf);
    if (more) put(buf ^ 1);   // last read in the pass before this one
  }
#pragma unroll
  for (int b = 0; b < QB; ++b) {
    const int qi = qw + 32 * b + r;
    const float sum = sum_halves(l[b]);
    if (qi >= nq) continue;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;   // a row that sees no key: zeros
    T* dst = static_cast<T*>(p.out) + (q0 + qi) * p.ldo + (int64_t)head * p.dim;
#pragma unroll
    for (int t = 0; t < OT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int ch = 32 * t + 8 * i + 4 * h2;
        const u32x2 w = {pack2<T>(o[b][t][4 * i] * inv, o[b][t][4 * i + 1] * inv),
                         pack2<T>(o[b][t][4 * i + 2] * inv, o[b][t][4 * i + 3] * inv)};
        if (ch < p.dim) *reinterpret_cast<u32x2*>(dst + ch) = w;
      }
  }
}

template <class T, int D, int NW, int QB> static hipError_t prefill_l(const AttnPrefillArgs& p, hipStream_t st) {
  constexpr int BQ = 32 * NW * QB;
  hipLaunchKernelGGL((attn_prefill_kernel<T, D, NW, QB>), dim3((unsigned)(p.kv * p.g), (unsigned)(p.q_tokens / BQ + p.seqs)),
                     dim3(64 * NW), 0, st, p);
  return hipGetLastError();
}
template <class T, int D> static hipError_t prefill_d(const AttnPrefillArgs& p, hipStream_t st) {
  return prefill_l<T, D, 8, 1>(p, st);
}
template <class T> static hipError_t prefill_t(const AttnPrefillArgs& p, hipStream_t st) {
  if (p.dim <= 64) return prefill_d<T, 64>(p, st);
  if (p.dim <= 96) return prefill_d<T, 96>(p, st);
  if (p.dim <= 128) return prefill_d<T, 128>(p, st);
  return hipErrorInvalidValue;
}
hipError_t run_attn_prefill(int dtype, const AttnPrefillArgs& p, hipStream_t st) {
  return dtype == DT_F16 ? prefill_t<_Float16>(p, st) : dtype == DT_BF16 ? prefill_t<__bf16>(p, st) : hipErrorInvalidValue;
}

}  // namespace ohip
