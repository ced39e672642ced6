// Products with 4-bit weights: Y[m][n] = act(sum_k A[m][k] s[n][k / G] (c[n][k] - z[n][k / G]) + bias[n]),
// codes c in 0..15, scales s in the activations' type, zero points z in 0..15.
#include "launch.hpp"
#include "serve.hpp"

namespace ohip {

// ------------------------------------------------------------------ packing
// The packed form: tiles of 16 rows (n) by 128 k, each one kilobyte: lane
// l = 16 q + r of the product's wave finds the codes of row r in its 16 bytes,
// word s holding k = 32 s + 8 q + e, channel kCodeOrder[i] in nibble order so
// that code_frag gives e = 0..7 ascending.  Scales and zero points follow the
// rows: [n / 16][k / G][16].
__global__ void __launch_bounds__(256)
q4_pack_kernel(const uint8_t* __restrict__ src, uint32_t* __restrict__ dst, int N, int K, int group, int blocks, int kt,
               int64_t words) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= words) return;
  const int s = (int)(i & 3), lane = (int)(i >> 2) & 63;
  const int64_t tile = i >> 8;
  const int n = (int)(tile / kt) * 16 + (lane & 15);
  const int k = (int)(tile % kt) * 128 + 32 * s + 8 * (lane >> 4);
  uint32_t w = 0;
  if (n < N) {
    const uint8_t* row = src + (int64_t)n * blocks * (group / 2);   // a row's blocks lie one after another
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t c = k + e < K ? (row[(k + e) / 2] >> (4 * (e & 1))) & 15u : 0u;
      // element e of the fragment is nibble (e even: e / 2, odd: 4 + e / 2)
      w |= c << (4 * ((e >> 1) + 4 * (e & 1)));
    }
  }
  dst[i] = w;
}

template <class S, class D>
__global__ void __launch_bounds__(256)
q4_pack_rows_kernel(const S* __restrict__ src, D* __restrict__ dst, int N, int blocks, int64_t count) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= count) return;
  const int r = (int)(i & 15);
  const int64_t t = i >> 4;
  const int n = (int)(t / blocks) * 16 + r, b = (int)(t % blocks);
  if constexpr (std::is_same<S, uint8_t>::value) {   // zero points: two blocks a byte
    dst[i] = n < N ? (src[(int64_t)n * ((blocks + 1) / 2) + b / 2] >> (4 * (b & 1))) & 15 : 0;
  } else {
    dst[i] = n < N ? src[(int64_t)n * blocks + b] : D(0);
  }
}

hipError_t run_q4_pack(const uint8_t* src, void* dst, int N, int K, int group, hipStream_t st) {
  const int kt = (K + 127) / 128, blocks = (K + group - 1) / group;
  const int64_t words = (int64_t)((N + 15) / 16) * kt * 256;
  hipLaunchKernelGGL(q4_pack_kernel, dim3((unsigned)((words + 255) / 256)), dim3(256), 0, st, src,
                     static_cast<uint32_t*>(dst), N, K, group, blocks, kt, words);
  return hipGetLastError();
}
hipError_t run_q4_pack_rows(int elem_bytes, const void* src, void* dst, int N, int blocks, hipStream_t st) {
  const int64_t count = (int64_t)((N + 15) / 16) * blocks * 16;
  const dim3 grid((unsigned)((count + 255) / 256)), block(256);
  if (elem_bytes == 4)
    hipLaunchKernelGGL((q4_pack_rows_kernel<uint32_t, uint32_t>), grid, block, 0, st, static_cast<const uint32_t*>(src),
                       static_cast<uint32_t*>(dst), N, blocks, count);
  else if (elem_bytes == 2)
    hipLaunchKernelGGL((q4_pack_rows_kernel<uint16_t, uint16_t>), grid, block, 0, st, static_cast<const uint16_t*>(src),
                       static_cast<uint16_t*>(dst), N, blocks, count);
  else
    hipLaunchKernelGGL((q4_pack_rows_kernel<uint8_t, uint8_t>), grid, block, 0, st, static_cast<const uint8_t*>(src),
                       static_cast<uint8_t*>(dst), N, blocks, count);
  return hipGetLastError();
}

// ------------------------------------------------------------------ few rows
// Eight activations of a lane: a fragment of 16-bit elements, or f32.
template <class T> struct Act { u32x4 v; };
template <> struct Act<float> { float v[8]; };

// The sixteen-column product of one word of codes with activations, exact
// codes: f16 takes the bias off each code (exact); bf16 adds a second product
// with -(bias + z) (q4_kernel takes sums again where that leaves f32); f32
// runs the f32 instruction, element e of every lane a k of its own.
template <class T> struct Q4Mma;
template <> struct Q4Mma<_Float16> {
  u32x4 off;   // (1024 + z) twice, (64 + z) twice
  uint32_t mask = code_mask();
  __device__ __forceinline__ void zero(int z) {
    const _Float16 a = (_Float16)(1024 + z), b = (_Float16)(64 + z);
    const f16x8 v = {a, a, b, b, a, a, b, b};
    off = __builtin_bit_cast(u32x4, v);
  }
  __device__ __forceinline__ u32x4 frag(uint32_t w) const {
    return __builtin_bit_cast(u32x4, __builtin_bit_cast(f16x8, code_frag<_Float16>(w, mask)) - __builtin_bit_cast(f16x8, off));
  }
  __device__ __forceinline__ f32x4 mma(u32x4 f, const Act<_Float16>& a, f32x4 c) const { return mma16<_Float16>(f, a.v, c); }
};
template <> struct Q4Mma<__bf16> {
  u32x4 off;
  uint32_t mask = code_mask();
  __device__ __forceinline__ void zero(int z) {
    const uint32_t b = __builtin_bit_cast(uint32_t, (float)-(128 + z)) >> 16;
    off = u32x4{b * 0x10001u, b * 0x10001u, b * 0x10001u, b * 0x10001u};
  }
  __device__ __forceinline__ u32x4 frag(uint32_t w) const { return code_frag<__bf16>(w, mask); }
  __device__ __forceinline__ f32x4 mma(u32x4 f, const Act<__bf16>& a, f32x4 c) const {
    return mma16<__bf16>(f, a.v, mma16<__bf16>(off, a.v, c));
  }
};
template <> struct Q4Mma<float> {
  int z;
  struct Frag { float v[8]; };
  __device__ __forceinline__ void zero(int zp) { z = zp; }
  __device__ __forceinline__ Frag frag(uint32_t w) const {
    Frag f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f.v[e] = (float)((int)((w >> (4 * ((e >> 1) + 4 * (e & 1)))) & 15u) - z);
    return f;
  }
  __device__ __forceinline__ f32x4 mma(const Frag& f, const Act<float>& a, f32x4 c) const {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(f.v[e], a.v[e], c, 0, 0, 0);
    return c;
  }
};

// Slots of 128 k of activations that a wave has in LDS: four waves a block
// leave room for four blocks a CU (16 x 4096 x 11008 bf16 9.3 us, two blocks
// with twice the slots 11.0), eight are alone on theirs.
template <class T, int TM, int NW> constexpr int q4_slots() {
  constexpr int n = ((NW == 4 ? 32 : 128) << 10) / (NW * 16 * TM * 128 * (int)sizeof(T));
  return n >= 4 ? 4 : n;
}

// A block takes 16 rows of the weight; its NW waves split K and meet in LDS in
// wave order.  GS: steps of 32 k a group holds (four for any larger).
// Bound: streaming the weight once, and the lookups of the activations in the
// CU's cache: a fragment's neighbouring lanes are of different rows, so a load
// of it is 64 lookups of 16 bytes.  STAGE copies them into LDS instead, 64
// bytes a lookup, and reads the fragments there (16 x 11008 x 4096 bf16 14.5 ->
// 9.7 us, 64 rows 46 -> 21.5).  A ring of tiles of 128 k of codes and of
// activations is loaded ahead.  As compiled most tiles wait for all loads in
// flight all the same, the newest among them: the zero points' branch and the
// conditional prefetch join paths of different counts, and scales are unpacked
// next to their load.  So a deeper ring gains nothing.  (The waits for LDS
// count the loads behind them, which therefore go through plain pointers:
// loads of __restrict__ ones the compiler may move across the waits.)
template <class T, int TM, int GS, int NW, bool STAGE>
__global__ void __launch_bounds__(64 * NW, NW / 4)
q4_kernel(const Q4Args args, const FloatEpi<T> epi) {
  const T* const a = static_cast<const T*>(args.a);
  const u32x4* const codes = static_cast<const u32x4*>(args.codes);
  const T* const scales = static_cast<const T*>(args.scales);
  const uint8_t* const zp = args.zp;
  const int64_t lda = args.lda;
  const int M = args.M, N = args.N, K = args.K, group = args.group;
  __shared__ f32x4 red[NW][TM][64];
  constexpr int GN = 4 / GS;   // groups of a tile
  // (what the registers hold: a tile of activations is 16 TM registers of f16, 32 of f32)
  constexpr int kRing = TM * sizeof(T) <= 4 ? 4 : 2, kActs = TM * sizeof(T) <= 4 ? 2 : 1;
  // staged: slots of 16 TM rows, chunk c of row r in place c ^ r % 16
  constexpr int kChunks = 8 * sizeof(T), kSlot = 16 * TM * kChunks * 16, kSlots = q4_slots<T, TM, NW>();
  constexpr int kStage = 16 * TM * kChunks / 64;   // loads of a tile's activations
  static_assert(!STAGE || (kSlots >= 1 && kRing % kSlots == 0 && (kSlots - 1) * kStage + kSlots * (1 + GN) < 64), "");
  __shared__ __align__(256) char st0[STAGE ? NW * kSlot : 16], st1[STAGE && kSlots > 1 ? NW * kSlot : 16];
  __shared__ __align__(256) char st2[STAGE && kSlots > 2 ? NW * kSlot : 16], st3[STAGE && kSlots > 2 ? NW * kSlot : 16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int shift = GS == 1 ? 5 : GS == 2 ? 6 : group == 256 ? 8 : 7;   // log2(group)
  const int KT = (K + 127) / 128, blocks = (K + (1 << shift) - 1) >> shift;
  const int per = (KT + NW - 1) / NW;
  const int t0 = wave * per, mine = max(0, min(per, KT - t0));
  const u32x4* wt = codes + ((int64_t)blockIdx.x * KT + t0) * 64 + lane;
  const T* sc = scales + (int64_t)blockIdx.x * blocks * 16 + 4 * q;
  const uint8_t* zr = zp ? zp + (int64_t)blockIdx.x * blocks * 16 + r : nullptr;
  const T* ar[TM];   // (columns past M are not stored)
#pragma unroll
  for (int t = 0; t < TM; ++t) ar[t] = a + (int64_t)min(t * 16 + r, M - 1) * lda + 8 * q;
  f32x4 acc[TM];
#pragma unroll
  for (int t = 0; t < TM; ++t) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  struct Tile {
    u32x4 w;
    T s[GN][4];
    uint8_t z[GN];
  };
  struct Acts { Act<T> x[4][TM]; };
  auto load = [&](Tile& f, int i) __attribute__((always_inline)) {   // i < mine
    f.w = wt[(int64_t)i * 64];
#pragma unroll
    for (int g = 0; g < GN; ++g) {
      const int b = min(((t0 + i) * 128 + 32 * GS * g) >> shift, blocks - 1);
      __builtin_memcpy(f.s[g], __builtin_assume_aligned(sc + (int64_t)b * 16, 4 * sizeof(T)), 4 * sizeof(T));
      f.z[g] = zr ? zr[(int64_t)b * 16] : 8;
    }
  };
  auto load_acts = [&](Acts& f, int i) __attribute__((always_inline)) {
    const int kt = t0 + i;
    if (kt * 128 + 128 <= K) {
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int t = 0; t < TM; ++t) __builtin_memcpy(&f.x[s][t], ar[t] + (kt * 128 + 32 * s), sizeof(f.x[s][t]));
    } else {   // the rows' end
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int t = 0; t < TM; ++t) {
          const int k = kt * 128 + 32 * s;
          T e[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) e[j] = k + 8 * q + j < K ? ar[t][k + j] : T(0);
          __builtin_memcpy(&f.x[s][t], e, sizeof(f.x[s][t]));
        }
    }
  };
  auto slot = [&](int i) __attribute__((always_inline)) -> char* {
    const int v = i % kSlots;
    return (v == 0 ? st0 : v == 1 ? st1 : v == 2 ? st2 : st3) + wave * kSlot;
  };
  const auto rs = rows_resource(reinterpret_cast<const char*>(a), (int)(((M - 1) * lda + K) * sizeof(T)));
  const int srow = lane / kChunks, splace = lane % kChunks;
  auto stage = [&](int k, int i) __attribute__((always_inline)) {   // tile i into slot k
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // what was read there has arrived
    char* to = slot(k);
    const int k0 = (t0 + i) * 128;
#pragma unroll
    for (int j = 0; j < kStage; ++j) {
      constexpr int kRows = 64 / kChunks;
      const int row = j * kRows + srow, at = k0 + (splace ^ (row & 15)) * (int)(16 / sizeof(T));
      const int off = at < K && row < M ? (int)((row * lda + at) * sizeof(T)) : (int)0x80000000u;   // else zeros
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)(to + j * 1024), 16, off, 0, 0, 0);
    }
    asm volatile("" ::: "memory");   // the tile's other loads come after these
  };
  // The activations of the present tile are in LDS: after their loads the
  // wave has issued at least kSlots - 1 tiles' more, and kSlots times a tile's
  // codes and scales, unless these are the last tiles.
  auto arrived = [&](bool more) __attribute__((always_inline)) {
    if (more) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((kSlots - 1) * kStage + kSlots * (1 + GN)) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  };
  auto staged = [&](int k, int s, int t) __attribute__((always_inline)) {
    const char* row = slot(k) + (16 * t + r) * (kChunks * 16);
    Act<T> x;
    constexpr int kPer = sizeof(T) / 2;   // chunks of eight elements
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      __builtin_memcpy(reinterpret_cast<char*>(&x) + 16 * j,
                       __builtin_assume_aligned(row + (((kPer * (4 * s + q) + j) ^ r) * 16), 16), 16);
    return x;
  };
  auto sum = [&](const Tile& f, auto act) __attribute__((always_inline)) {
#pragma unroll
    for (int g = 0; g < GN; ++g) {
      Q4Mma<T> mul;
      mul.zero(f.z[g]);
      f32x4 raw[TM];
#pragma unroll
      for (int t = 0; t < TM; ++t) raw[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < GS; ++s) {
        const auto c = mul.frag(f.w[g * GS + s]);
#pragma unroll
        for (int t = 0; t < TM; ++t) raw[t] = mul.mma(c, act(g * GS + s, t), raw[t]);
      }
#pragma unroll
      for (int t = 0; t < TM; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][i] = __builtin_fmaf(to_f32(f.s[g][i]), raw[t][i], acc[t][i]);
    }
  };
  Tile ring[kRing];
  Acts acts[kActs];
  if (STAGE) {
#pragma unroll
    for (int i = 0; i < kSlots - 1; ++i)
      if (i < mine) stage(i, i);
  } else if (kActs > 1 && mine > 0) {
    load_acts(acts[0], 0);
  }
#pragma unroll
  for (int i = 0; i < kRing - 1; ++i)
    if (i < mine) load(ring[i], i);
  for (int i = 0; i < mine; i += kRing) {
#pragma unroll
    for (int k = 0; k < kRing; ++k) {
      if (i + k >= mine) break;
      // (the activations first: loads arrive in order, and these are waited for next)
      if (STAGE) {
        if (i + k + kSlots - 1 < mine) stage(k + kSlots - 1, i + k + kSlots - 1);
      } else if (i + k + kActs - 1 < mine) {
        load_acts(acts[(k + kActs - 1) % kActs], i + k + kActs - 1);
      }
      if (i + k + kRing - 1 < mine) load(ring[(k + kRing - 1) % kRing], i + k + kRing - 1);
      if constexpr (STAGE) arrived(i + k + kRing - 1 < mine);
      if constexpr (STAGE) sum(ring[k], [&](int s, int t) __attribute__((always_inline)) { return staged(k, s, t); });
      else sum(ring[k], [&](int s, int t) __attribute__((always_inline)) { return acts[k % kActs].x[s][t]; });
    }
  }
#pragma unroll
  for (int t = 0; t < TM; ++t) red[wave][t][lane] = acc[t];
  __syncthreads();
  if (wave >= TM) return;
  f32x4 v = red[0][wave][lane];
#pragma unroll
  for (int k = 1; k < NW; ++k) v += red[k][wave][lane];
  // The lane and the arguments anew: kept through the loop they cost it
  // registers (64 rows x 11008 x 4096 bf16 23.8 us for 21.2).
  uint64_t kernarg = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
  asm("" : "+s"(kernarg));
  const auto& again = *reinterpret_cast<const __attribute__((address_space(4))) Q4Args*>(kernarg);   // (the first one)
  const int M1 = TM > 2 ? again.M : M, N1 = TM > 2 ? again.N : N;   // (of few rows that load would be the last wait)
  const int l1 = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
  const int r1 = l1 & 15, q1 = l1 >> 4, i = blockIdx.x * 16 + 4 * q1, j = wave * 16 + r1;
  if constexpr (std::is_same<T, __bf16>::value) {
    // An infinity, or a number whose product with the codes' bias is beyond
    // f32, has left inf - inf: the wave takes its sums again, of all k, with
    // c - z itself (exact in bf16 too, but a conversion each).  One wave and no
    // care for speed: a call with such a row takes 60 to 190 us.
    const f32x4 test = v * 0.0f;
    if (__any(j < M1 && i < N1 && test[0] + test[1] + test[2] + test[3] != 0.0f)) {
      const int K = again.K, kt = (K + 127) / 128, blocks = (K + again.group - 1) / again.group;
      const T* x0 = static_cast<const T*>(again.a) + (int64_t)min(j, M1 - 1) * again.lda + 8 * q1;
      const uint32_t* words = static_cast<const uint32_t*>(again.codes) + ((int64_t)blockIdx.x * kt * 64 + l1) * 4;
      const T* s0 = static_cast<const T*>(again.scales) + (int64_t)blockIdx.x * blocks * 16 + 4 * q1;
      const uint8_t* z0 = again.zp ? again.zp + (int64_t)blockIdx.x * blocks * 16 + r1 : nullptr;
      v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
      for (int k = 0; k < K; k += 32) {
        const int b = k / again.group * 16, z = z0 ? z0[b] : 8;
        const uint32_t w = words[(int64_t)(k >> 7) * 256 + ((k >> 5) & 3)];
        T c[8], x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          c[e] = (T)(float)((int)((w >> (4 * ((e >> 1) + 4 * (e & 1)))) & 15u) - z);
          x[e] = k + 8 * q1 + e < K ? x0[k + e] : T(0);
        }
        u32x4 cf, xf;
        __builtin_memcpy(&cf, c, 16);
        __builtin_memcpy(&xf, x, 16);
        const f32x4 raw = mma16<T>(cf, xf, f32x4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(to_f32(s0[b + e]), raw[e], v[e]);
      }
    }
  }
  if (j >= M1 || i >= N1) return;
  typename FloatEpi<T>::PreI pi;
  typename FloatEpi<T>::PreJ pj;
  epi.load_i(pi, i);
  epi.load_j(pj, j);
  uint32_t bits[4];
  epi.finish(pi, pj, i, j, v, bits);
  const OutAddr out = epi.addr();
  store_group(out, epi.out_bytes(), out.row(i), i, j, bits);
}

template <class T, int TM, int NW, bool STAGE>
static hipError_t q4_w(const Q4Args& g, const FloatEpi<T>& epi, hipStream_t st) {
  const dim3 grid((unsigned)((g.N + 15) / 16)), block(64 * NW);
  if (g.group == 32)
    hipLaunchKernelGGL((q4_kernel<T, TM, 1, NW, STAGE>), grid, block, 0, st, g, epi);
  else if (g.group == 64)
    hipLaunchKernelGGL((q4_kernel<T, TM, 2, NW, STAGE>), grid, block, 0, st, g, epi);
  else
    hipLaunchKernelGGL((q4_kernel<T, TM, 4, NW, STAGE>), grid, block, 0, st, g, epi);
  return hipGetLastError();
}
template <class T, int TM, int NW> static hipError_t q4_s(const Q4Args& g, const FloatEpi<T>& epi, hipStream_t st) {
  if constexpr (q4_slots<T, TM, NW>() > 0) {
    const int64_t bytes = ((g.M - 1) * g.lda + g.K) * (int64_t)sizeof(T);
    // Whole aligned chunks, which 32 bits address; of fewer rows most of a
    // slot is filled for nothing (4096 x 11008 in groups of 128, bf16: 1 row
    // 7.3 us, staged 7.8; 4 rows 8.5 and 7.8; f32: 4 rows 23.5 and 23.1, 8 rows
    // 25.0 and 23.2).
    if (g.M > (sizeof(T) == 4 ? 4 : 2) && g.K * sizeof(T) % 16 == 0 && g.lda * sizeof(T) % 16 == 0 && reinterpret_cast<uintptr_t>(g.a) % 16 == 0 && bytes < INT_MAX)
      return q4_w<T, TM, NW, true>(g, epi, st);
  }
  return q4_w<T, TM, NW, false>(g, epi, st);
}
// Four waves a block where there are two blocks a CU or more (4096 x 11008
// bf16, 688 blocks: 1 row 7.3 us with either, 16 rows 8.0, eight waves 11.2, 32
// rows 11.1 and 15.4), else eight (16 x 11008 x 4096, 256 blocks: 9.7, four
// 14.8).
template <class T, int TM> static hipError_t q4_t(const Q4Args& g, const FloatEpi<T>& epi, hipStream_t st) {
  if constexpr (TM * sizeof(T) <= 4)
    if (g.N >= 512 * 16) return q4_s<T, TM, 4>(g, epi, st);
  return q4_s<T, TM, 8>(g, epi, st);
}

template <class T> static hipError_t q4_m(const Q4Args& g, const FloatOut& o, hipStream_t st) {
  const FloatEpi<T> epi = make_float_epi<T>(o);
  if (g.M <= 16) return q4_t<T, 1>(g, epi, st);
  if (g.M <= 32) return q4_t<T, 2>(g, epi, st);
  if (g.M <= kMaxQ4M) return q4_t<T, 4>(g, epi, st);
  return hipErrorInvalidValue;
}

hipError_t run_gemm_q4(int dtype, const Q4Args& g, const FloatOut& o, hipStream_t st) {
  switch (dtype) {
    case DT_F32: return q4_m<float>(g, o, st);
    case DT_F16: return q4_m<_Float16>(g, o, st);
    case DT_BF16: return q4_m<__bf16>(g, o, st);
    default: return hipErrorInvalidValue;
  }
}

// ------------------------------------------------------------------ many rows
// The weight as K-contiguous rows of T (ldw elements, zeros past K) for the
// MFMA engine: s * (c - z) in f32, rounded once.
// Four lanes write 64 bytes of a row (4096 x 22016 f16 88 us, 2.6 TB/s; in the
// codes' order, a row a lane, 95): a tenth of the product that follows for a
// few thousand rows.
template <class T>
__global__ void __launch_bounds__(256)
q4_unpack_kernel(const u32x4* __restrict__ codes, const T* __restrict__ scales, const uint8_t* __restrict__ zp,
                 T* __restrict__ dst, int N, int K, int64_t ldw, int group, int kt, int64_t tiles) {
  const int64_t tile = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (tile >= tiles) return;
  const int lane = threadIdx.x & 63, r = lane >> 2, q = lane & 3;   // four lanes write a row's 32 k
  const int64_t n16 = tile / kt;
  const int k0 = (int)(tile % kt) * 128, blocks = (K + group - 1) / group;
  const int64_t n = n16 * 16 + r;
  if (n >= N) return;
  const u32x4 w = codes[tile * 64 + 16 * q + r];
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const int k = k0 + 32 * s + 8 * q;
    if (k >= ldw) continue;
    const int64_t b = (n16 * blocks + min((k0 + 32 * s) / group, blocks - 1)) * 16 + r;
    const float sv = to_f32(scales[b]);
    const int z = zp ? zp[b] : 8;
    T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = (int)((w[s] >> (4 * ((i >> 1) + 4 * (i & 1)))) & 15u) - z;
      e[i] = k + i < K ? from_f32<T>(sv * (float)c) : from_f32<T>(0.0f);
    }
    T* to = dst + n * ldw + k;
    if (k + 8 <= ldw) {
      __builtin_memcpy(__builtin_assume_aligned(to, 16), e, sizeof(e));
    } else {   // rows of a whole number of 16-byte chunks: f32 may end in half of the eight
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (k + i < ldw) to[i] = e[i];
    }
  }
}

hipError_t run_q4_unpack(int dtype, const Q4Args& g, void* dst, int64_t ldw, hipStream_t st) {
  const int kt = (g.K + 127) / 128;
  const int64_t tiles = (int64_t)((g.N + 15) / 16) * kt;
  const dim3 grid((unsigned)((tiles + 3) / 4)), block(256);
  const u32x4* codes = static_cast<const u32x4*>(g.codes);
  switch (dtype) {
    case DT_F32:
      hipLaunchKernelGGL((q4_unpack_kernel<float>), grid, block, 0, st, codes, static_cast<const float*>(g.scales), g.zp,
                         static_cast<float*>(dst), g.N, g.K, ldw, g.group, kt, tiles);
      break;
    case DT_F16:
      hipLaunchKernelGGL((q4_unpack_kernel<_Float16>), grid, block, 0, st, codes, static_cast<const _Float16*>(g.scales),
                         g.zp, static_cast<_Float16*>(dst), g.N, g.K, ldw, g.group, kt, tiles);
      break;
    case DT_BF16:
      hipLaunchKernelGGL((q4_unpack_kernel<__bf16>), grid, block, 0, st, codes, static_cast<const __bf16*>(g.scales),
                         g.zp, static_cast<__bf16*>(dst), g.N, g.K, ldw, g.group, kt, tiles);
      break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace ohip
