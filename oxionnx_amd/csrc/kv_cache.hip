// The paged cache of keys and values in 4 bits: appending with the position
// rotation, and attention of one query token a sequence over it.
#include "serve.hpp"

namespace ohip {

// ------------------------------------------------------------------ append
// Eight channels a thread, D / 8 lanes a head; a block has 256 * 8 / D tokens
// and walks a run of their rows (query heads, key heads, value heads), so the
// angles are loaded once and a tile of 16 tokens' value codes is written by
// one block.  Rotation, group extremes and codes in f32:
//   (o1, o2) = (x1 c - x2 s, x2 c + x1 s)          products rounded one by one
//   scale = f16((max - min) / 15), low = f16(min)  (kept finite)
//   code = clamp(rint((x - low) / scale), 0, 15)   (a group without extent: 0)
// Bound: memory (8191 tokens, 32 + 2 x 8 heads of 128: 46 us, 4.7 TB/s; with a
// thread a row and its angles read for each head 139).
__device__ __forceinline__ float finite_f16(float v) {
  return v != v ? v : __builtin_fminf(__builtin_fmaxf(v, -65504.0f), 65504.0f);
}

// the value of lane l ^ 1, l ^ 2, of the mirrored lane of its 8, of its 16
template <int CTRL> __device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true);
}
template <int CTRL> __device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, dpp<CTRL>(__builtin_bit_cast(uint32_t, v)));
}
constexpr int kXor1 = 0xb1, kXor2 = 0x4e, kXor3 = 0x1b, kMirror8 = 0x141, kMirror16 = 0x140, kRotate8 = 0x128;

// One step of a transposition of nibbles between lanes: those of index bit S
// against bit S of the lane's index i.
template <int S> __device__ __forceinline__ uint32_t swap_nibbles(uint32_t w, uint32_t x, int i) {
  constexpr uint32_t m = S == 1 ? 0x0f0f0f0fu : S == 2 ? 0x00ff00ffu : 0x0000ffffu;
  return i & S ? (w & ~m) | ((x & ~m) >> (4 * S)) : (w & m) | ((x & m) << (4 * S));
}

template <class T, int D>
__global__ void __launch_bounds__(256)
kv_append_kernel(const KvAppendArgs p) {
  constexpr int LPH = D / 8, TPB = 256 / LPH;   // lanes a head, tokens a block
  const int c = threadIdx.x % LPH;
  const int64_t token = (int64_t)blockIdx.x * TPB + threadIdx.x / LPH;
  const bool live = token < p.tokens;   // whole heads: a head's lanes agree
  const int64_t tk = live ? token : p.tokens - 1;
  const int rows = p.q_heads + 2 * p.kv, per = (rows + gridDim.y - 1) / gridDim.y;
  const int row0 = blockIdx.y * per, row1 = min(rows, row0 + per);
  const T* const q = static_cast<const T*>(p.q) + tk * p.ldq + 8 * c;
  const T* const k = static_cast<const T*>(p.k) + tk * p.ldk + 8 * c;
  const T* const v = static_cast<const T*>(p.v) + tk * p.ldv + 8 * c;
  auto fetch = [&](int row) __attribute__((always_inline)) -> u32x4 {   // row: uniform
    const T* src = row < p.q_heads ? q + (int64_t)row * D
                 : row < p.q_heads + p.kv ? k + (int64_t)(row - p.q_heads) * D : v + (int64_t)(row - p.q_heads - p.kv) * D;
    u32x4 raw;
    __builtin_memcpy(&raw, __builtin_assume_aligned(src, 16), 16);
    return raw;
  };
  if (row0 >= row1) return;
  u32x4 next = fetch(row0);

  // this lane's angles: its channel pairs' (four), or its eight channels'
  float cs[8], sn[8];
  const int half = p.rot / 16;   // lanes that half of the rotated channels takes
  const bool turned = p.cos && row0 < p.q_heads + p.kv && (p.interleaved ? 8 * c < p.rot : c < 2 * half);
  const bool low = c < half;
  if (turned) {
    int64_t pos = p.positions[tk];
    pos = pos < 0 ? 0 : pos >= p.max_position ? p.max_position - 1 : pos;
    const int64_t at = pos * (p.rot / 2) + (p.interleaved ? 4 * c : 8 * (low ? c : c - half));
    const int n = p.interleaved ? 4 : 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      cs[e] = e < n ? p.cos[at + e] : 0.0f;
      sn[e] = e < n ? p.sin[at + e] : 0.0f;
    }
  }
  const int mate = (threadIdx.x & 63) + (low ? half : -half);   // of a turned lane

  // where the token's codes and parameters go
  const int64_t slot = p.slots[tk], page = slot / p.page;
  const bool kept = live && slot >= 0 && slot < p.pages * p.page;   // else a padding token
  const int off = (int)(slot - page * p.page);
  const int gl = p.group / 8;   // lanes a group: 4, 8 or 16

  for (int row = row0; row < row1; ++row) {
    const u32x4 raw = next;
    if (row + 1 < row1) next = fetch(row + 1);
    const int kind = row < p.q_heads ? 0 : row < p.q_heads + p.kv ? 1 : 2;   // q, k, v
    const int h = row - (kind == 0 ? 0 : kind == 1 ? p.q_heads : p.q_heads + p.kv);
    T in[8];
    __builtin_memcpy(in, &raw, 16);
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (float)in[e];
    if (p.cos && kind != 2) {
      if (p.interleaved) {
        if (turned) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float a = x[2 * j], b = x[2 * j + 1];
            x[2 * j] = a * cs[j] - b * sn[j];
            x[2 * j + 1] = b * cs[j] + a * sn[j];
          }
        }
      } else {
        u32x4 theirs;   // the mate's eight channels as they came
#pragma unroll
        for (int i = 0; i < 4; ++i) theirs[i] = (uint32_t)__shfl((int)raw[i], mate, 64);
        T other[8];
        __builtin_memcpy(other, &theirs, 16);
        if (turned) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float own = x[e] * cs[e], cross = (float)other[e] * sn[e];
            x[e] = low ? own - cross : own + cross;
          }
        }
      }
    }
    if (kind != 0) {
      // the group's extremes; a NaN makes the whole group NaN
      float lo = x[0], hi = x[0];
      bool bad = x[0] != x[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) {
        lo = __builtin_fminf(lo, x[e]);
        hi = __builtin_fmaxf(hi, x[e]);
        bad |= x[e] != x[e];
      }
      lo = __builtin_fminf(lo, dpp<kXor1>(lo));
      hi = __builtin_fmaxf(hi, dpp<kXor1>(hi));
      lo = __builtin_fminf(lo, dpp<kXor2>(lo));
      hi = __builtin_fmaxf(hi, dpp<kXor2>(hi));
      if (gl >= 8) {
        lo = __builtin_fminf(lo, dpp<kMirror8>(lo));
        hi = __builtin_fmaxf(hi, dpp<kMirror8>(hi));
      }
      if (gl >= 16) {
        lo = __builtin_fminf(lo, dpp<kMirror16>(lo));
        hi = __builtin_fmaxf(hi, dpp<kMirror16>(hi));
      }
      const uint64_t any = __ballot(bad);
      // (finite, so that a group of nothing but one infinity has no extent)
      lo = __builtin_fminf(__builtin_fmaxf(lo, -__FLT_MAX__), __FLT_MAX__);
      hi = __builtin_fminf(__builtin_fmaxf(hi, -__FLT_MAX__), __FLT_MAX__);
      if (any && ((any >> (threadIdx.x & 63 & ~(gl - 1))) & ((1u << gl) - 1))) lo = hi = __builtin_nanf("");
      const _Float16 s16 = (_Float16)finite_f16((hi - lo) * (1.0f / 15.0f)), l16 = (_Float16)finite_f16(lo);
      const float sc = (float)s16, lw = (float)l16;
      uint32_t word = 0;   // nibble e: channel 8 c + e
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float t = sc > 0.0f ? __builtin_rintf((x[e] - lw) / sc) : 0.0f;
        const uint32_t code = t >= 15.0f ? 15u : t > 0.0f ? (uint32_t)t : 0u;
        word |= code << (4 * e);
        if (p.held) x[e] = (float)code * sc + lw;
      }
      const int64_t at = (page * p.kv + h) * p.page + off;   // the token's row of the head
      if (kept && c % gl == 0)
        static_cast<uint32_t*>(kind == 1 ? p.cache_kp : p.cache_vp)[at * (D / p.group) + c / gl] =
            (uint32_t)__builtin_bit_cast(uint16_t, s16) | (uint32_t)__builtin_bit_cast(uint16_t, l16) << 16;
      if (kind == 1) {   // word of channels 32 s + 8 q ..: [q][s]
        if (kept) static_cast<uint32_t*>(p.cache_kc)[at * (D / 8) + (c & 3) * (D / 32) + (c >> 2)] = word;
      } else {
        // A value column o holds the channels o + 16 i, which lane 2 i + o / 8
        // has as its nibble o % 8: a transposition among the lanes of one
        // parity, after which lane 2 i + h has column(s) 8 h + i (and 8 h + i + 4).
        const int i = c >> 1;
        word = swap_nibbles<1>(word, dpp<kXor2>(word), i);
        word = swap_nibbles<2>(word, dpp<kXor3>(dpp<kMirror8>(word)), i);   // lane ^ 4
        if constexpr (D == 128) word = swap_nibbles<4>(word, dpp<kRotate8>(word), i);
        if (kept) {
          char* to = static_cast<char*>(p.cache_vc) + (at - (off & 15)) * (D / 2) + ((8 * (c & 1) + i) * 16 + (off & 15)) * (D / 32);
          if constexpr (D == 128) {
            *reinterpret_cast<uint32_t*>(to) = word;
          } else {
            *reinterpret_cast<uint16_t*>(to) = (uint16_t)word;
            *reinterpret_cast<uint16_t*>(to + 4 * 16 * (D / 32)) = (uint16_t)(word >> 16);
          }
        }
      }
    }
    T* out = static_cast<T*>(kind == 0 ? p.q_out : kind == 1 ? p.k_out : p.v_out);
    if (out && live) {
      const int64_t ldo = kind == 0 ? p.ldqo : kind == 1 ? p.ldko : p.ldvo;
      T e8[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) e8[e] = (T)x[e];
      __builtin_memcpy(__builtin_assume_aligned(out + tk * ldo + h * D + 8 * c, 16), e8, 16);
    }
  }
}

template <class T> static hipError_t append_t(int dim, const KvAppendArgs& p, hipStream_t st) {
  const int64_t per_block = 256 * 8 / dim, tiles = (p.tokens + per_block - 1) / per_block;
  // rows a block: all of a token's where there are enough tokens for 1024 blocks
  const int rows = p.q_heads + 2 * p.kv;
  const int64_t runs = std::min<int64_t>(rows, std::max<int64_t>(1, (1024 + tiles - 1) / tiles));
  const dim3 grid((unsigned)tiles, (unsigned)runs), block(256);
  if (dim == 128) hipLaunchKernelGGL((kv_append_kernel<T, 128>), grid, block, 0, st, p);
  else if (dim == 64) hipLaunchKernelGGL((kv_append_kernel<T, 64>), grid, block, 0, st, p);
  else return hipErrorInvalidValue;
  return hipGetLastError();
}
hipError_t run_kv_append(int dtype, int dim, const KvAppendArgs& p, hipStream_t st) {
  return dtype == DT_F16 ? append_t<_Float16>(dim, p, st) : dtype == DT_BF16 ? append_t<__bf16>(dim, p, st) : hipErrorInvalidValue;
}

// ------------------------------------------------------------------ decode
// One query token a sequence.  With K = s c + m by group, the scores are
// sum_g s_tg (q_g . c_tg) + m_tg sum(q_g): the matrix instruction multiplies
// the codes themselves (exact in 16 bits) and the scale meets the f32 sums.
// The values alike: weights w_tg = p_t s_tg multiply the codes, taken from
// the middle of their range, c - 8, and sum_t p_t (m_tg + 8 s_tg) is added at
// the end: over a long context both are sums of either sign that stay as
// small as the output is.  The bias of the codes' bits goes step by step for
// the same reason: the step's products start from -136 times its weights.
// The weights are split in two bf16 parts (16 bits together, f32's range: no
// scale of the values can make them underflow).
//
// A block has the up to 16 query heads of one key head and a piece of the
// sequence, or several of both; its waves take steps of 32 tokens, the next
// step's codes in flight under the present one's sums (the batch below: three
// steps 56 us, two 54.6) and page entries 32 steps ahead.  The last step loads
// once more what it has: a load that only some steps issue would make all of
// them wait for it (60 us).  A step's scales and minima are loaded once, a word
// or more a lane, and spread to the lanes that need them through LDS.
// S^T = K Q^T, lane l = 16 q + h: head h, tokens 4 q + r of two tiles of 16,
// which is how O^T = V^T P^T wants its right operand when the values' tokens
// are counted 4 q + j of the first tile, then of the second.
//
// Up to eight heads leave half of the sixteen columns free: then (P = 2) a
// column is a head of one of the two tiles, so that a lane has the softmax of
// four tokens instead of eight; the columns of the other tile get no weight,
// and each column keeps a maximum and sums of its own until the end.
//
// Sequences of unequal lengths: a launch of two blocks a CU (the registers'
// limit) cuts all steps of all sequences and key heads, laid end to end, into
// equal pieces, wherever those end; the lengths are on the device, so each
// block finds its own.  (A batch of 64 with 512 to 4096 tokens: 7 % less time
// than ranges of one length for all, whose last blocks are those of the long
// sequences.)  Pieces of a sequence leave their maxima, sums and weighted values in
// `part`; a second launch adds them in order.  (Counting the blocks and letting
// the last one add saves the launch, but its fences write back and invalidate
// an XCD's cache once a block: 355 us for that batch where the launch made it
// 76.)
//
// Bound: the latency of a step with two waves a SIMD, for which the registers
// allow no third (that batch: 54.6 us, 7 of them the second launch; its loads
// alone 38; two sequences of 131071 and 73728 tokens 57.8, 6, 47).  Codes
// copied into LDS, 64 bytes a cache lookup instead of 16: 62 us.
constexpr int kDecodeWaves = 4;

// A sequence's tokens [lo, len) and their steps of 32 tokens.
struct Span { int len, lo, begin, steps; };
__device__ __forceinline__ Span span_of(const AttnDecodeArgs& p, int b) {
  Span s;
  s.len = (int)max((int64_t)0, min((int64_t)p.lens[b], (int64_t)p.width * p.tpp * 16));
  s.lo = p.window > 0 ? max(0, s.len - p.window) : 0;
  s.begin = s.lo / 32;
  s.steps = (s.len + 31) / 32 - s.begin;
  return s;
}

// The launch's positions: of every sequence, for each of its `groups` (head
// block, key head), kPieceCost that stand for what a piece costs however short
// it is, then its steps.  Block i has positions [i * per, (i + 1) * per).
constexpr int kPieceCost = 8, kLeastPiece = 32;
struct Layout { int64_t total, per, start; };   // start: of sequence b (if b < batch)
// One wave (all lanes) adds up the sequences; `pos` >= 0: b becomes the sequence that holds it.
__device__ __forceinline__ Layout layout_of(const AttnDecodeArgs& p, int groups, int64_t pos, int& b) {
  const int lane = threadIdx.x & 63;
  Layout s{0, 0, 0};
  const int want = b;
  for (int b0 = 0; b0 < p.batch; b0 += 64) {
    const int64_t v = b0 + lane < p.batch ? (int64_t)groups * (span_of(p, b0 + lane).steps + kPieceCost) : 0;
    int64_t sum = v;   // inclusive
#pragma unroll
    for (int i = 1; i < 64; i *= 2) {
      const int64_t other = __shfl_up(sum, i, 64);
      if (lane >= i) sum += other;
    }
    if (pos >= 0) {
      const uint64_t after = __ballot(v > 0 && s.total + sum > pos);   // sequences that end behind pos
      if (after && s.total <= pos) {
        const int at = __ffsll((unsigned long long)after) - 1;
        b = b0 + at;
        s.start = s.total + __shfl(sum - v, at, 64);
      }
    } else if (want >= b0 && want < b0 + 64) {
      s.start = s.total + __shfl(sum - v, want - b0, 64);
    }
    s.total += __shfl(sum, 63, 64);
  }
  s.per = max((s.total + p.blocks - 1) / p.blocks, (int64_t)kLeastPiece);
  return s;
}

template <int D, int NG> struct DecodeShared {
  float red[kDecodeWaves][16][D + 4];
  float red_m[kDecodeWaves][16], red_l[kDecodeWaves][16];
  // of a wave's step, [token][group]: the keys' pairs, the values' scales and middles (of code 8)
  __align__(16) uint32_t spread_k[kDecodeWaves][32 * NG];
  __align__(16) float spread_v[kDecodeWaves][2][32 * NG];
};

// Steps [x, y) of sequence b for group c; part: where they go if they are not all of it (null: the output).
template <class T, int D, int NG, int P>
__device__ __forceinline__ void decode_piece(const AttnDecodeArgs& p, DecodeShared<D, NG>& sh, int b, int c, const Span& span,
                                             int x, int y, float* part) {
  constexpr int NW = kDecodeWaves;
  constexpr int KW = D / 32;   // steps of 32 channels
  constexpr int CI = D / 16;   // channels of a value column
  constexpr int SG = KW / NG;  // steps a group
  constexpr int HC = 16 / P;   // heads of the columns
  constexpr int VS = 2 / P;    // tiles of a lane's columns
  auto& red = sh.red;
  auto& red_m = sh.red_m;
  auto& red_l = sh.red_l;
  auto& spread_k = sh.spread_k;
  auto& spread_v = sh.spread_v;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int kvh = c % p.kv, hb = c / p.kv;
  const int nh = min(HC, p.g - hb * HC);   // query heads of this block
  const int head0 = kvh * p.g + hb * HC;
  const int hr = r % HC, half = r / HC;    // this lane's head, and tile if P = 2
  const int len = span.len, lo = span.lo, first = span.begin + x, steps = y - x;
  const int mine = steps > wave ? (steps - wave + NW - 1) / NW : 0;   // this wave's: first + wave + NW i
  const int32_t* table = p.table + (int64_t)b * p.width;
  const int last_tile = len > 0 ? (len - 1) / 16 : 0;

  // page and place within it of the wave's tiles: lane 2 i + t holds tile t of step i0 + i
  auto entries = [&](int i0, int& id, int& place) __attribute__((always_inline)) {
    const int i = i0 + (lane >> 1);
    const int tile = min(2 * (first + wave + NW * i) + (lane & 1), last_tile);
    const int e = tile / p.tpp;
    place = tile - e * p.tpp;
    id = i < mine ? table[e] : 0;
  };
  int id0, place0, id1, place1;   // of this 32 steps and of the next
  entries(0, id0, place0);
  entries(32, id1, place1);

  // the queries' fragments, channels in the codes' order; sums of channels and of bias * channel
  u32x4 qf[KW];
  float qs[NG], qb[NG];
  {
    const T* src = static_cast<const T*>(p.q) + (int64_t)b * p.ldq + (int64_t)(head0 + min(hr, nh - 1)) * D;
#pragma unroll
    for (int g = 0; g < NG; ++g) qs[g] = qb[g] = 0.0f;
#pragma unroll
    for (int s = 0; s < KW; ++s) {
      T e[8], f[8];
      __builtin_memcpy(e, __builtin_assume_aligned(src + 32 * s + 8 * q, 16), 16);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        f[i] = hr < nh ? e[kCodeOrder[i]] : (T)0.0f;
        qs[s / SG] += (float)f[i];
        qb[s / SG] += code_bias<T>(i) * (float)f[i];
      }
      __builtin_memcpy(&qf[s], f, 16);
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      qs[g] += __shfl_xor(qs[g], 16, 64);
      qs[g] += __shfl_xor(qs[g], 32, 64);
      qb[g] += __shfl_xor(qb[g], 16, 64);
      qb[g] += __shfl_xor(qb[g], 32, 64);
    }
  }

  f32x4 o[CI];
#pragma unroll
  for (int i = 0; i < CI; ++i) o[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float om[NG];
#pragma unroll
  for (int g = 0; g < NG; ++g) om[g] = 0.0f;
  float mx = -__builtin_inff(), l = 0.0f;
  const uint32_t nibbles = code_mask();
  const u32x4 middle = u32x4{0xc308c308u, 0xc308c308u, 0xc308c308u, 0xc308c308u};   // -136

  struct Step {
    u32x4 kw[2], vw[2];
    uint32_t pw[NG];   // lane: token lane % 32, of keys (lanes under 32) or values
    int known;         // bit t: tile t's page exists
  };
  const char* const params = static_cast<const char*>(lane < 32 ? p.cache_kp : p.cache_vp) + (lane & 15) * (4 * NG);
  const int koff = r * (D / 2) + q * (D / 8), voff = (r * 16 + 4 * q) * (D / 32);
  auto load = [&](Step& f, int i) __attribute__((always_inline)) {   // i < mine
    if (i > 0 && i % 32 == 0) {
      id0 = id1;
      place0 = place1;
      entries(i + 32, id1, place1);
    }
    f.known = 0;
    int64_t row[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      int page = __builtin_amdgcn_readlane(id0, 2 * (i % 32) + t);
      const int place = __builtin_amdgcn_readlane(place0, 2 * (i % 32) + t);
      if (page >= 0 && page < p.pages) f.known |= 1 << t;
      else page = 0;   // (its tokens are masked)
      row[t] = (((int64_t)page * p.kv + kvh) * p.tpp + place) * 16;
      const char* kc = static_cast<const char*>(p.cache_kc) + row[t] * (D / 2) + koff;
      const char* vc = static_cast<const char*>(p.cache_vc) + row[t] * (D / 2) + voff;
      __builtin_memcpy(&f.kw[t], __builtin_assume_aligned(kc, D / 8), D / 8);
      __builtin_memcpy(&f.vw[t], __builtin_assume_aligned(vc, D / 8), D / 8);
    }
    __builtin_memcpy(f.pw, __builtin_assume_aligned(params + ((lane & 16) ? row[1] : row[0]) * (4 * NG), 4 * NG), 4 * NG);
  };
  auto sum = [&](Step& f, int i) __attribute__((always_inline)) {
    const int st = first + wave + NW * i;
    // (a wave's LDS accesses are in order)
    if (lane < 32) {
      __builtin_memcpy(__builtin_assume_aligned(&spread_k[wave][lane * NG], 4 * NG), f.pw, 4 * NG);
    } else {
      float sc[NG], mid[NG];
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        sc[g] = f16_lo(f.pw[g]);
        mid[g] = __builtin_fmaf(8.0f, sc[g], f16_hi(f.pw[g]));
      }
      __builtin_memcpy(__builtin_assume_aligned(&spread_v[wave][0][(lane & 31) * NG], 4 * NG), sc, 4 * NG);
      __builtin_memcpy(__builtin_assume_aligned(&spread_v[wave][1][(lane & 31) * NG], 4 * NG), mid, 4 * NG);
    }
    const int tile0 = P == 2 ? half : 0;   // of the lane's first values
    uint32_t kp[VS][4 * NG];
    float vs[VS][4 * NG], vm[VS][4 * NG];
#pragma unroll
    for (int u = 0; u < VS; ++u) {
      const int at = (16 * (tile0 + u) + 4 * q) * NG;
      __builtin_memcpy(kp[u], __builtin_assume_aligned(&spread_k[wave][at], 16), 16 * NG);
      __builtin_memcpy(vs[u], __builtin_assume_aligned(&spread_v[wave][0][at], 16), 16 * NG);
      __builtin_memcpy(vm[u], __builtin_assume_aligned(&spread_v[wave][1][at], 16), 16 * NG);
    }
    float s[VS][4];
#pragma unroll
    for (int u = 0; u < VS; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[u][j] = 0.0f;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      f32x4 raw[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        raw[t] = f32x4{-qb[g], -qb[g], -qb[g], -qb[g]};
#pragma unroll
        for (int k = 0; k < SG; ++k) raw[t] = mma16<T>(code_frag<T>(f.kw[t][g * SG + k], nibbles), qf[g * SG + k], raw[t]);
      }
#pragma unroll
      for (int u = 0; u < VS; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float v = P == 2 ? (half ? raw[1][j] : raw[0][j]) : raw[u][j];
          const uint32_t w = kp[u][j * NG + g];
          s[u][j] = __builtin_fmaf(f16_lo(w), v, s[u][j]);
          s[u][j] = __builtin_fmaf(f16_hi(w), qs[g], s[u][j]);
        }
    }
    // tokens outside [lo, len), and of page entries that name no page
    if (st * 32 < lo || st * 32 + 32 > len || f.known != 3) {
#pragma unroll
      for (int u = 0; u < VS; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int token = st * 32 + 16 * (tile0 + u) + 4 * q + j;
          if (!(f.known >> (tile0 + u) & 1) || token < lo || token >= len) {
            s[u][j] = -__builtin_inff();
#pragma unroll
            for (int g = 0; g < NG; ++g) vs[u][j * NG + g] = vm[u][j * NG + g] = 0.0f;   // whatever is there: 0 * it is 0
          }
        }
    }
    float m = s[0][0];
#pragma unroll
    for (int j = 1; j < 4 * VS; ++j) m = __builtin_fmaxf(m, s[j / 4][j % 4]);
    m = max_quarters(m);
    const float now = __builtin_fmaxf(mx, m);
    const float base = now == -__builtin_inff() ? 0.0f : now * p.c;
    const float keep = __builtin_amdgcn_exp2f(__builtin_fmaf(mx, p.c, -base));
    mx = now;
    float pt[VS][4];
    l *= keep;
#pragma unroll
    for (int u = 0; u < VS; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        pt[u][j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][j], p.c, -base));
        l += pt[u][j];
      }
    u32x4 hi[NG], lw[NG];
    f32x4 start[NG];
    const uint32_t front = half ? 0u : ~0u;   // P = 2: whose words are the first tile's
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      om[g] *= keep;
#pragma unroll
      for (int u = 0; u < VS; ++u) {
#pragma unroll
        for (int j = 0; j < 4; ++j) om[g] = __builtin_fmaf(pt[u][j], vm[u][j * NG + g], om[g]);
#pragma unroll
        for (int j = 0; j < 2; ++j) {   // a weight's upper half, and the rest of it rounded
          const float w0 = pt[u][2 * j] * vs[u][2 * j * NG + g], w1 = pt[u][2 * j + 1] * vs[u][(2 * j + 1) * NG + g];
          const uint32_t u0 = __builtin_bit_cast(uint32_t, w0), u1 = __builtin_bit_cast(uint32_t, w1);
          const uint32_t h = __builtin_amdgcn_perm(u1, u0, 0x07060302u);
          const float r0 = w0 - __builtin_bit_cast(float, u0 & 0xffff0000u), r1 = w1 - __builtin_bit_cast(float, u1 & 0xffff0000u);
          const uint32_t w = pack2<__bf16>(r0, r1);
          if constexpr (P == 2) {
            hi[g][j] = h & front;
            hi[g][2 + j] = h & ~front;
            lw[g][j] = w & front;
            lw[g][2 + j] = w & ~front;
          } else {
            hi[g][2 * u + j] = h;
            lw[g][2 * u + j] = w;
          }
        }
      }
      start[g] = mma16<__bf16>(middle, lw[g], f32x4{0.0f, 0.0f, 0.0f, 0.0f});
      start[g] = mma16<__bf16>(middle, hi[g], start[g]);
    }
#pragma unroll
    for (int i = 0; i < CI; ++i) {
      u32x4 vf;
#pragma unroll
      for (int j = 0; j < 4; ++j) {   // tokens 2 j, 2 j + 1 of the eight
        uint32_t w;
        if constexpr (D == 128)
          w = __builtin_amdgcn_perm(f.vw[j / 2][2 * j % 4 + 1], f.vw[j / 2][2 * j % 4], i < 4 ? 0x05040100u : 0x07060302u);
        else
          w = f.vw[j / 2][j % 2];
        vf[j] = ((w >> (4 * (i % 4))) & nibbles) | 0x43004300u;
      }
      const int g = i * NG / CI;
      const f32x4 add = mma16<__bf16>(vf, hi[g], mma16<__bf16>(vf, lw[g], start[g]));
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = __builtin_fmaf(o[i][j], keep, add[j]);
    }
  };
  Step ring[2];
  if (mine > 0) load(ring[0], 0);
  for (int i = 0; i < mine; i += 2) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (i + k >= mine) break;
      load(ring[1 - k], min(i + k + 1, mine - 1));
      sum(ring[k], i + k);
    }
  }
  // channel 4 q + j + 16 i of head r; the lanes of a head hold a part each of l and om
  l = sum_quarters(l);
#pragma unroll
  for (int g = 0; g < NG; ++g) om[g] = sum_quarters(om[g]);
#pragma unroll
  for (int i = 0; i < CI; ++i) {
    const int g = i * NG / CI;
#pragma unroll
    for (int j = 0; j < 4; ++j) red[wave][r][16 * i + 4 * q + j] = o[i][j] + om[g];
  }
  if (q == 0) {
    red_m[wave][r] = mx;
    red_l[wave][r] = l;
  }
  __syncthreads();
  T* out = static_cast<T*>(p.out) + (int64_t)b * p.ldo + (int64_t)head0 * D;
  for (int idx = threadIdx.x; idx < nh * D; idx += 64 * NW) {
    const int h = idx / D, ch = idx % D;
    float m = red_m[0][h];
#pragma unroll
    for (int w = 1; w < NW * P; ++w) m = __builtin_fmaxf(m, red_m[w / P][h + HC * (w % P)]);
    const float base = m == -__builtin_inff() ? 0.0f : m * p.c;
    float total_l = 0.0f, acc = 0.0f;
#pragma unroll
    for (int w = 0; w < NW * P; ++w) {
      const int col = h + HC * (w % P);
      const float f = __builtin_amdgcn_exp2f(__builtin_fmaf(red_m[w / P][col], p.c, -base));
      total_l += f * red_l[w / P][col];
      acc += f * red[w / P][col][ch];
    }
    if (!part) {
      out[h * D + ch] = (T)(total_l == 0.0f ? 0.0f : acc / total_l);   // no token: zeros
    } else {
      float* to = part + h * (D + 2);   // value, maximum, sum
      to[ch] = acc;
      if (ch == 0) {
        to[D] = m;
        to[D + 1] = total_l;
      }
    }
  }
  __syncthreads();   // the next piece's waves write `red`
}

template <class T, int D, int NG, int P>
__global__ void __launch_bounds__(64 * kDecodeWaves, NG == 4 && P == 1 ? 1 : 2)
attn_decode_kernel(const AttnDecodeArgs p) {
  __shared__ DecodeShared<D, NG> sh;
  const int groups = p.kv * ((p.g + 15) / 16);
  int64_t pos, end, start = 0;
  int b;
  if (p.blocks == 0) {   // a block for each sequence and group
    b = blockIdx.x / groups;
    pos = blockIdx.x % groups;
    end = pos + 1;
  } else {
    b = 0;
    const Layout s = layout_of(p, groups, -1, b);
    pos = blockIdx.x * s.per;
    end = min(s.total, pos + s.per);
  }
  while (pos < end) {
    int c = (int)pos, x = 0, y;
    Span span;
    if (p.blocks == 0) {
      span = span_of(p, b);
      y = span.steps;
      pos = end;
    } else {
      start = layout_of(p, groups, pos, b).start;
      b = __builtin_amdgcn_readfirstlane(b);
      span = span_of(p, b);
      const int64_t v = span.steps + kPieceCost;
      c = (int)((pos - start) / v);
      const int64_t at = start + c * v;
      x = (int)max((int64_t)0, pos - at - kPieceCost);
      y = (int)min((int64_t)span.steps, end - at - kPieceCost);
      const bool empty = span.steps == 0 && pos == at;   // zeros, from the block with its first position
      pos = at + v;
      if (y <= x && !empty) continue;
      y = max(y, 0);
    }
    // (the same in all lanes, which the compiler cannot see behind the shuffles)
    c = __builtin_amdgcn_readfirstlane(c);
    x = __builtin_amdgcn_readfirstlane(x);
    y = __builtin_amdgcn_readfirstlane(y);
    const bool whole = x == 0 && y == span.steps;
    // a block has at most one piece that began before it and one that goes on behind it
    float* part = whole ? nullptr : p.part + ((int64_t)blockIdx.x * 2 + (x > 0 ? 0 : 1)) * (16 * (D + 2));
    decode_piece<T, D, NG, P>(p, sh, b, c, span, x, y, part);
  }
}

// A block adds the pieces of one head; the factors of all pieces first, then
// 256 / D threads a channel, each a run of pieces, whose sums are added in order.
template <class T, int D>
__global__ void __launch_bounds__(256)
attn_decode_merge_kernel(const AttnDecodeArgs p) {
  constexpr int PARTS = 256 / D;
  __shared__ float factor[kDecodeBlocks], wave_m[4], wave_l[4], sums[PARTS][D];
  const int head = blockIdx.x, kvh = head / p.g, hb = (head - kvh * p.g) / 16, h = (head - kvh * p.g) % 16;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int b = blockIdx.y;
  const Layout s = layout_of(p, p.kv * ((p.g + 15) / 16), -1, b);
  const Span span = span_of(p, b);
  const int64_t at = s.start + (hb * p.kv + kvh) * (int64_t)(span.steps + kPieceCost) + kPieceCost;   // its first step
  const int64_t block0 = at / s.per, n64 = (at + span.steps - 1) / s.per - block0 + 1;
  if (span.steps == 0 || n64 == 1) return;   // written already
  const int n = (int)n64;
  const float* part0 = p.part + h * (D + 2);
  // piece k: of block0 + k, which it began in (k = 0) or before
  auto piece = [&](int k) __attribute__((always_inline)) -> const float* {
    return part0 + ((block0 + k) * 2 + (k == 0 ? 1 : 0)) * (16 * (D + 2));
  };
  float m = -__builtin_inff();
  for (int k = threadIdx.x; k < n; k += 256) {
    const float v = piece(k)[D];
    factor[k] = v;
    m = __builtin_fmaxf(m, v);
  }
  for (int i = 1; i < 64; i *= 2) m = __builtin_fmaxf(m, __shfl_xor(m, i, 64));
  if (lane == 0) wave_m[wave] = m;
  __syncthreads();
  m = __builtin_fmaxf(__builtin_fmaxf(wave_m[0], wave_m[1]), __builtin_fmaxf(wave_m[2], wave_m[3]));
  const float base = m == -__builtin_inff() ? 0.0f : m * p.c;
  float l = 0.0f;
  for (int k = threadIdx.x; k < n; k += 256) {
    const float f = __builtin_amdgcn_exp2f(__builtin_fmaf(factor[k], p.c, -base));
    factor[k] = f;
    l += f * piece(k)[D + 1];
  }
  for (int i = 1; i < 64; i *= 2) l += __shfl_xor(l, i, 64);
  if (lane == 0) wave_l[wave] = l;
  __syncthreads();
  l = (wave_l[0] + wave_l[1]) + (wave_l[2] + wave_l[3]);
  const int ch = threadIdx.x % D, run = threadIdx.x / D, per = (n + PARTS - 1) / PARTS;
  float acc = 0.0f;
#pragma unroll 8
  for (int k = run * per; k < min(n, (run + 1) * per); ++k) acc += factor[k] * piece(k)[ch];
  sums[run][ch] = acc;
  __syncthreads();
  if (threadIdx.x >= D) return;
#pragma unroll
  for (int i = 1; i < PARTS; ++i) acc += sums[i][ch];
  static_cast<T*>(p.out)[(int64_t)b * p.ldo + (int64_t)head * D + ch] = (T)(l == 0.0f ? 0.0f : acc / l);
}

// Blocks of equal pieces (0: a block for each sequence and key head, and no
// second launch): not where no sequence is longer than a piece has to be, nor
// where there are so many sequences that their blocks even out by themselves.
int decode_blocks(int64_t batch, int kv, int g, int64_t longest) {
  return longest <= 32 * kLeastPiece || batch * kv * ((g + 15) / 16) >= 8 * kDecodeBlocks ? 0 : kDecodeBlocks;
}

template <class T, int D, int NG> static void decode_g(const AttnDecodeArgs& p, const dim3& grid, hipStream_t st) {
  if (p.g <= 8) hipLaunchKernelGGL((attn_decode_kernel<T, D, NG, 2>), grid, dim3(64 * kDecodeWaves), 0, st, p);
  else hipLaunchKernelGGL((attn_decode_kernel<T, D, NG, 1>), grid, dim3(64 * kDecodeWaves), 0, st, p);
}
template <class T, int D> static hipError_t decode_d(int group, const AttnDecodeArgs& p, hipStream_t st) {
  const dim3 grid(p.blocks ? (unsigned)p.blocks : (unsigned)(p.batch * p.kv * ((p.g + 15) / 16)));
  switch (D / group) {
    case 1: decode_g<T, D, 1>(p, grid, st); break;
    case 2: decode_g<T, D, 2>(p, grid, st); break;
    case 4:
      if constexpr (D == 128) { decode_g<T, D, 4>(p, grid, st); break; }
      [[fallthrough]];
    default: return hipErrorInvalidValue;
  }
  if (p.blocks)
    hipLaunchKernelGGL((attn_decode_merge_kernel<T, D>), dim3((unsigned)(p.kv * p.g), (unsigned)p.batch), dim3(256), 0, st, p);
  return hipGetLastError();
}
hipError_t run_attn_decode(int dtype, int dim, int group, const AttnDecodeArgs& p, hipStream_t st) {
  if (dim != 64 && dim != 128) return hipErrorInvalidValue;
  if (dtype == DT_F16) return dim == 64 ? decode_d<_Float16, 64>(group, p, st) : decode_d<_Float16, 128>(group, p, st);
  if (dtype == DT_BF16) return dim == 64 ? decode_d<__bf16, 64>(group, p, st) : decode_d<__bf16, 128>(group, p, st);
  return hipErrorInvalidValue;
}

}  // namespace ohip
