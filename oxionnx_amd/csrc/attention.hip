// Attention over whole prompts: packed sequences, grouped heads, causal.
#include "serve.hpp"

namespace ohip {

// A block has 128 query rows of one head, 32 a wave, and walks the keys they
// see in tiles of 64 that its four waves share through LDS.  S^T = K Q^T,
// so a lane holds one query (its column) and the softmax's running maximum and
// sum need one exchange between a lane and the one 32 further; O^T = V^T P^T
// takes P as it lies in the registers: k index 8 h + j (h = lane / 32) stands
// for key 4 h + j of a block of 8, then of the next, and V's fragments come
// from LDS through the transposing read.  P is rounded to T for that: two
// parts of it, as over the cache, would be half as many products again, and
// the matrix unit is the bound; against 64 bits the outputs are off by 1.25 to
// 1.4 times what f32 weights leave (rounding the output itself included).
//
// Bound: the matrix products, with about as many cycles of vector instructions
// (two thirds of them the exponentials and their arguments), so each stage
// interleaves the softmax of one half tile with the products of its
// neighbours.  Tiles are loaded straight into LDS a pass ahead; a CU has room
// for two blocks, each of which works through the other's barriers, its first
// tiles and its last rows.  32 heads, 8 of keys, of 128 channels: 8192 tokens
// 527 us (1043 TFLOP/s, 76 % of a large matrix product's rate), seven prompts
// of 8191 tokens 138, the last 1000 of 4000 within 2048 51.  In another run,
// these at 535, 141 and 51: eight waves that share a tile and load three
// passes ahead, one block a CU, 546, 153 and 71; four of them 728, 222 and
// 60; blocks in the order of their keys, most first, through all sequences
// 536, 141, and 0.2 us more for a short prompt.
constexpr int kPrefillK = 64, kPrefillQ = 128;

// Slot of 16-byte chunk c of a staged row r: rows of 16 (8) chunks, XOR with a
// permutation of r's low bits that puts 16 consecutive rows of one chunk (the
// K fragments) and four rows of four chunks (a transposing read) in different
// bank groups.
template <int CH> __device__ __forceinline__ int row_swizzle(int r) {
  if constexpr (CH == 16) return ((r & 3) << 2) | ((r >> 2) & 3);
  else return ((r & 2) << 1) | ((r >> 2) & 3);
}

// Which sequence a block's tile belongs to.  Sequence i has the tile slots
// from cu[i] / 128 + i on (at least as many as it has tiles), so that the grid
// needs only the totals; a slot past its sequence's end has nothing to do.
// One wave searches; offsets that are not ascending cannot lead outside
// [0, total].
__device__ __forceinline__ int slot_sequence(const int32_t* cu, int seqs, int64_t total, int tile) {
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int i0 = 0; i0 < seqs; i0 += 64) {
    const int i = i0 + lane;
    const int64_t c = i < seqs ? min(max((int64_t)cu[i], (int64_t)0), total) : 0;
    n += __popcll(__ballot(i < seqs && c / kPrefillQ + i <= tile));
  }
  return __builtin_amdgcn_readfirstlane(n - 1);
}

typedef short s16x4 __attribute__((ext_vector_type(4)));

template <class T, int D>
__global__ void __launch_bounds__(256, 2)
attn_prefill_kernel(const AttnPrefillArgs p) {
  constexpr int NW = 4, BQ = kPrefillQ, BK = kPrefillK, KS = D / 16, OT = D / 32;
  constexpr int CH = D > 64 ? 16 : 8, RB = CH * 16;     // chunks and bytes of a staged row
  constexpr int NL = BK * CH / (64 * NW);               // loads a thread of a tile
  constexpr int kTile = BK * RB;
  static_assert(NL >= 1 && (64 / CH) * NW % 16 == 0, "a thread's loads share their swizzle");
  // K and V tiles, each a variable of its own: the compiler then knows which
  // loads a fragment read may depend on, and waits for no later ones
  __shared__ __align__(256) char lk0[kTile], lk1[kTile], lv0[kTile], lv1[kTile];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 31, h2 = lane >> 5;
  // heads of one key head next to each other in time, key heads eight apart: an XCD's L2 holds its own
  const int kvh = blockIdx.x % p.kv, head = kvh * p.g + blockIdx.x / p.kv;
  const int tile = (int)gridDim.y - 1 - (int)blockIdx.y;   // late tiles of a sequence see the most keys
  const int seq = slot_sequence(p.cu_q, p.seqs, p.q_tokens, tile);
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
  const int tiles = kend > kbeg ? (kend - kbeg + BK - 1) / BK : 0;
  const int qw = __builtin_amdgcn_readfirstlane(qt + wave * 32);   // this wave's first query; its lanes' are qw + r
  // half tiles that this wave's queries see
  const int wend = min(kend, p.causal ? min(qw + 32, nq) + shift : nk);
  const int halves = qw < nq && wend > kbeg ? (wend - kbeg + 31) / 32 : 0;

  u32x4 qf[KS];
  {
    const T* src = static_cast<const T*>(p.q) + (q0 + min(qw + r, nq - 1)) * p.ldq + (int64_t)head * p.dim;
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
  float base = -__builtin_inff(), l = 0.0f;   // the maximum that weights are taken against, times c; their sum

  const char* kb = static_cast<const char*>(p.k) + (k0 * p.ldk + (int64_t)kvh * p.dim) * 2;
  const char* vb = static_cast<const char*>(p.v) + (k0 * p.ldv + (int64_t)kvh * p.dim) * 2;
  // this thread's loads: row (i * NW + wave) * (64 / CH) + lane / CH, slot lane % CH
  const int lrow = wave * (64 / CH) + lane / CH;
  const int chunk = (lane % CH) ^ row_swizzle<CH>(lrow);
  const bool inside = chunk * 8 < p.dim;
  const int kvoff = inside ? (int)(lrow * p.ldk * 2) + chunk * 16 : (int)0x80000000u;
  const int vvoff = inside ? (int)(lrow * p.ldv * 2) + chunk * 16 : (int)0x80000000u;
  const int kstep = (int)(NW * (64 / CH) * p.ldk * 2), vstep = (int)(NW * (64 / CH) * p.ldv * 2);
  // tile t into `to`; a tile past the end reads as zeros (every pass issues
  // the same number of loads, which its waits count)
  auto load = [&](const char* at, int64_t ld, int t, int voff, int step, char* to) __attribute__((always_inline)) {
    const int kt = kbeg + t * BK, rows = max(0, min(nk - kt, BK));
    const auto rs = rows_resource(at + (int64_t)min(kt, nk) * ld * 2, max(0, (int)((rows - 1) * ld + p.dim) * 2));
#pragma unroll
    for (int i = 0; i < NL; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)(to + (i * NW + wave) * 1024), 16,
                                               voff + i * step, 0, 0, 0);
  };
  // Fragment addresses within a tile: rows are aligned to their swizzle, so a
  // chunk is an XOR.  K: row r, chunk 2 s + h2.  V: keys 8 j + 4 h2 +
  // (lane % 16) / 4 on, channels 16 ((lane / 16) % 2) + 4 (lane % 4) of the 32
  // from 32 t on.
  int ka[KS], va[2][OT];
#pragma unroll
  for (int k = 0; k < KS; ++k) ka[k] = (r * RB + ((h2 ^ row_swizzle<CH>(r)) * 16)) ^ (32 * k);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int row = 8 * j + 4 * h2 + (lane & 15) / 4;
    const int at = row * RB + (((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ row_swizzle<CH>(row)) * 16) + 8 * (lane & 1);
#pragma unroll
    for (int t = 0; t < OT; ++t) va[j][t] = at ^ (64 * t);
  }

  // The three steps of a half tile of 32 keys.  Each stage of the pipeline
  // runs one half's softmax between the next one's scores and the previous
  // one's values, so that the matrix unit has independent work under the
  // softmax's vector instructions (in one wave: the waves of a SIMD pass the
  // barriers together and would all be at the same step).
  auto key_frag = [&](const char* at, int k) __attribute__((always_inline)) -> u32x4 {
    return *reinterpret_cast<const u32x4*>(at + ka[k]);
  };
  auto value_frag = [&](const char* at, int k, int t) __attribute__((always_inline)) -> u32x4 {   // 16 keys from 16 k on
    u32x4 f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s16x4*)(at + va[j][t] + 16 * k * RB));
      const u32x2 w = __builtin_bit_cast(u32x2, v);
      f[2 * j] = w.x;
      f[2 * j + 1] = w.y;
    }
    return f;
  };
  auto scores = [&](const char* at, f32x16& s) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
    for (int k = 0; k < KS; ++k) s = mma32<T>(key_frag(at, k), qf[k], s);
  };
  auto values = [&](const char* at, const u32x4 (&pf)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2 * OT; ++i) o[i % OT] = mma32<T>(value_frag(at, i / OT, i % OT), pf[i / OT], o[i % OT]);
  };
  // weights of half j from its scores, against a maximum that is taken anew
  // only when a score exceeds it by more than 8 powers of two; returns what
  // the sums so far have to be multiplied with
  auto mask = [&](int j, f32x16& s) __attribute__((always_inline)) {
    const int kj = kbeg + 32 * j;
    if (kj + 32 > nk || (p.causal && kj + 31 > qw + shift) || (p.window > 0 && kj <= qw + 31 + shift - p.window)) {
      const int last = (p.causal ? min(nk - 1, qw + r + shift) : nk - 1) - kj - 4 * h2;
      const int low = (p.window > 0 ? qw + r + shift - p.window : -1) - kj - 4 * h2;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int key = 8 * (i / 4) + i % 4;
        if (key > last || key <= low) s[i] = -__builtin_inff();
      }
    }
  };
  // the sums so far wait for a factor
  int grown = 0;
  float keep = 1.0f;
  auto softmax = [&](f32x16& s, u32x4 (&pf)[2]) __attribute__((always_inline)) {
    float m = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) m = __builtin_fmaxf(m, s[i]);
    m = max_halves(m) * p.c;
    const bool grow = __any(m - base > 8.0f);
    const float now = grow ? __builtin_fmaxf(base, m) : base;
    const float off = now == -__builtin_inff() ? 0.0f : now;
    keep = __builtin_amdgcn_exp2f(base - off);   // 0 the first time
    base = now;
    l *= grow ? keep : 1.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], p.c, -off));
      l += s[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) pf[i / 4][i % 4] = pack2<T>(s[2 * i], s[2 * i + 1]);
    grown = __builtin_amdgcn_readfirstlane((int)grow);
    asm("" : "+s"(grown));   // not known to be `grow`: the branch on it stays in the next stage
  };
  auto rescale = [&]() __attribute__((always_inline)) {
    if (grown)
#pragma unroll
      for (int i = 0; i < 16 * OT; ++i) o[i / 16][i % 16] *= keep;
  };

  f32x16 s[2];
  u32x4 pf[2];
  // stage of half j: scores of half j + 1 from LDS at kn, softmax of half j,
  // values of half j - 1 at vn
  auto stage = [&](int j, const char* kn, const char* vn, f32x16& cur, f32x16& next) __attribute__((always_inline)) {
    u32x4 w[2];
    rescale();
    mask(j, cur);
    u32x4 vf[2 * OT], kf[KS];
#pragma unroll
    for (int i = 0; i < 2 * OT; ++i) {
      vf[i] = value_frag(vn, i / OT, i % OT);
      kf[i] = key_frag(kn, i);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) next[i] = 0.0f;
    static_assert(KS == 2 * OT, "one of each in turn: the scores' products wait for each other");
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      o[i % OT] = mma32<T>(vf[i], pf[i / OT], o[i % OT]);
      next = mma32<T>(kf[i], qf[i], next);
    }
    softmax(cur, w);
    // In the wave's order: the fragments' loads and the maximum between the
    // first products, then the exponentials (3 % faster
    // than the compiler's order, 6 % than all loads in front: 8192 tokens).
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);     // LDS reads
      __builtin_amdgcn_sched_group_barrier(0x402, 5, 0);     // vector instructions
      __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);       // a matrix product
    }
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x402, 7, 0);
    }
    // here, not sunk past the next stage's branches
    asm volatile("" : "+v"(w[0]), "+v"(w[1]), "+v"(l));
    pf[0] = w[0];
    pf[1] = w[1];
  };
  constexpr int kHalf = 32 * RB;
  // Pass t: scores of tile t + 1, values of tile t.  All waves go through the
  // block's passes; a wave computes while its queries see keys.  K tile i is
  // in variable i % 2 and so is V tile i: pass t may overwrite K tile t and V
  // tile t - 1, the last ones that pass t - 1 read, with tiles t + 2 and t + 1,
  // which arrive during it.
  auto kvar = [&](auto i) __attribute__((always_inline)) -> char* {
    if constexpr (decltype(i)::value % 2 == 0) return lk0; else return lk1;
  };
  auto vvar = [&](auto i) __attribute__((always_inline)) -> char* {
    if constexpr (decltype(i)::value % 2 == 0) return lv0; else return lv1;
  };
  int t = 0;
  auto begin = [&](auto at) __attribute__((always_inline)) {   // at: t % 2
    constexpr int m = decltype(at)::value;
    loads_barrier<0>();
    load(kb, p.ldk, t + 2, kvoff, kstep, kvar(std::integral_constant<int, m>()));
    load(vb, p.ldv, t + 1, vvoff, vstep, vvar(std::integral_constant<int, m + 1>()));
  };
  auto pass = [&](auto at) __attribute__((always_inline)) {
    constexpr int m = decltype(at)::value;
    const char* kn = kvar(std::integral_constant<int, m + 1>());
    const char* vn = vvar(std::integral_constant<int, m>());
    begin(at);
    stage(2 * t + 1, kn, vn, s[1], s[0]);
    stage(2 * t + 2, kn + kHalf, vn + kHalf, s[0], s[1]);
    ++t;
  };
  auto last = [&](auto at) __attribute__((always_inline)) {   // the last one or two halves' values
    const char* vn = vvar(at);
    begin(at);
    rescale();
    values(vn, pf);
    if (2 * t + 1 < halves) {
      mask(2 * t + 1, s[1]);
      softmax(s[1], pf);
      rescale();
      values(vn + kHalf, pf);
    }
    ++t;
  };
  using C0 = std::integral_constant<int, 0>;
  using C1 = std::integral_constant<int, 1>;
  if (tiles) {
    load(kb, p.ldk, 0, kvoff, kstep, lk0);
    load(vb, p.ldv, 0, vvoff, vstep, lv0);
    load(kb, p.ldk, 1, kvoff, kstep, lk1);
    loads_barrier<2 * NL>();   // K tile 0
    if (halves > 0) {
      scores(lk0, s[0]);
      mask(0, s[0]);
      scores(lk0 + kHalf, s[1]);
      softmax(s[0], pf);
    }
  }
  while (2 * t + 4 < halves) {
    pass(C0());
    pass(C1());
  }
  if (2 * t + 2 < halves) pass(C0());
  if (halves > 0) {
    if (t % 2 == 0) last(C0()); else last(C1());
  }
  while (t < tiles) {
    if (t % 2 == 0) begin(C0()); else begin(C1());
    ++t;
  }
  loads_barrier<0>();   // those of tiles past the end write LDS too

  const int qi = qw + r;
  const float sum = sum_halves(l);
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;   // a row that sees no key: zeros
  T* dst = static_cast<T*>(p.out) + (q0 + min(qi, nq - 1)) * p.ldo + (int64_t)head * p.dim + 4 * h2;
  auto store = [&](const f32x16& x, int t) __attribute__((always_inline)) {
    if (qi >= nq) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const u32x2 w = {pack2<T>(x[4 * i] * inv, x[4 * i + 1] * inv), pack2<T>(x[4 * i + 2] * inv, x[4 * i + 3] * inv)};
      if (32 * t + 8 * i + 4 * h2 < p.dim) *reinterpret_cast<u32x2*>(dst + 32 * t + 8 * i) = w;
    }
  };
  float finite = 0.0f;
#pragma unroll
  for (int i = 0; i < 16 * OT; ++i) finite = __builtin_fmaf(o[i / 16][i % 16], 0.0f, finite);
  if (!__any(qi < nq && finite != 0.0f)) {
#pragma unroll
    for (int t = 0; t < OT; ++t) store(o[t], t);
    return;
  }
  // A weight of 0 times a value that is not finite is NaN: such a value of a
  // key that a query does not see has reached its sums, if the half tile holds
  // keys that it sees.  Such a wave takes its sums again, from memory and 32
  // channels at a time: of the finite values, and (with ones for weights) of
  // the infinities of either sign that each query sees; a NaN counts as both.
  constexpr uint32_t kExp = std::is_same<T, _Float16>::value ? 0x7c00u : 0x7f80u;
  constexpr uint32_t kOne = std::is_same<T, _Float16>::value ? 0x3c00u : 0x3f80u;
  const float off = base == -__builtin_inff() ? 0.0f : base;
#pragma unroll 1
  for (int t = 0; t < OT; ++t) {
    f32x16 x, plus, minus;
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = plus[i] = minus[i] = 0.0f;
#pragma unroll 1
    for (int j = 0; j < halves; ++j) {
      const int kj = kbeg + 32 * j;
      f32x16 a;
#pragma unroll
      for (int i = 0; i < 16; ++i) a[i] = 0.0f;
      const char* krow = kb + (int64_t)min(kj + r, nk - 1) * p.ldk * 2;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const int ch = 16 * k + 8 * h2;
        u32x4 f = {0, 0, 0, 0};
        if (ch < p.dim) __builtin_memcpy(&f, __builtin_assume_aligned(krow + ch * 2, 16), 16);
        a = mma32<T>(f, qf[k], a);
      }
      mask(j, a);
      const int ch = 32 * t + r;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        u32x4 w, sees, v, vp, vm;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float s0 = a[8 * k + 2 * e], s1 = a[8 * k + 2 * e + 1];
          sees[e] = (s0 == -__builtin_inff() ? 0u : kOne) | (s1 == -__builtin_inff() ? 0u : kOne << 16);
          w[e] = pack2<T>(__builtin_amdgcn_exp2f(__builtin_fmaf(s0, p.c, -off)), __builtin_amdgcn_exp2f(__builtin_fmaf(s1, p.c, -off)));
          v[e] = vp[e] = vm[e] = 0;
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const int key = min(kj + 16 * k + 8 * (e / 2) + 4 * h2 + 2 * (e % 2) + b, nk - 1);
            const uint32_t y = ch < p.dim ? *reinterpret_cast<const uint16_t*>(vb + ((int64_t)key * p.ldv + ch) * 2) : 0u;
            const bool big = (y & kExp) == kExp, nan = (y & 0x7fffu) > kExp;
            v[e] |= (big ? 0u : y) << (16 * b);
            vp[e] |= (nan || y == kExp ? kOne : 0u) << (16 * b);
            vm[e] |= (nan || y == (kExp | 0x8000u) ? kOne : 0u) << (16 * b);
          }
        }
        x = mma32<T>(v, w, x);
        plus = mma32<T>(vp, sees, plus);
        minus = mma32<T>(vm, sees, minus);
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      x[i] += plus[i] > 0.0f ? __builtin_inff() : 0.0f;
      x[i] -= minus[i] > 0.0f ? __builtin_inff() : 0.0f;
    }
    store(x, t);
  }
}

template <class T, int D> static hipError_t prefill_d(const AttnPrefillArgs& p, hipStream_t st) {
  hipLaunchKernelGGL((attn_prefill_kernel<T, D>), dim3((unsigned)(p.kv * p.g), (unsigned)(p.q_tokens / kPrefillQ + p.seqs)),
                     dim3(256), 0, st, p);
  return hipGetLastError();
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
