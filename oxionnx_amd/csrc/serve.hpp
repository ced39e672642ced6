// The serving kernels (4-bit products, the 4-bit cache of keys and values,
// attention): their launchers, and the types and device helpers they share.
#pragma once
#include <type_traits>

#include "internal.hpp"

namespace ohip {

// ------------------------------------------------------------------ launchers
// A product with a packed 4-bit weight (q4.hip holds the packed form).
struct Q4Args {
  const void* a;          // [M][lda] activations
  int64_t lda;            // elements
  const void* codes;
  const void* scales;     // of the activations' type
  const uint8_t* zp;      // null: 8
  int M, N, K, group;
};
constexpr int kMaxQ4M = 64;   // rows of the few-row kernel
hipError_t run_q4_pack(const uint8_t* src, void* dst, int N, int K, int group, hipStream_t st);
// scales (4 or 2 bytes) and zero points (elem_bytes 1, two a source byte)
hipError_t run_q4_pack_rows(int elem_bytes, const void* src, void* dst, int N, int blocks, hipStream_t st);
hipError_t run_gemm_q4(int dtype, const Q4Args& g, const FloatOut& o, hipStream_t st);
hipError_t run_q4_unpack(int dtype, const Q4Args& g, void* dst, int64_t ldw, hipStream_t st);

// Rows of ld* elements, heads of 64 or 128 channels next to each other, 16-byte aligned.
struct KvAppendArgs {
  const void *q, *k, *v;       // q may be null with q_heads 0
  void *q_out, *k_out, *v_out; // any may be null
  int64_t ldq, ldk, ldv, ldqo, ldko, ldvo;
  int64_t tokens;
  int q_heads, kv, group, rot, interleaved, held;
  const int32_t* positions;
  const float *cos, *sin;      // [max_position][rot / 2]; null: no rotation
  int64_t max_position;
  const int32_t* slots;
  void *cache_kc, *cache_vc, *cache_kp, *cache_vp;
  int64_t pages;
  int page;
};
hipError_t run_kv_append(int dtype, int dim, const KvAppendArgs& p, hipStream_t st);

struct AttnDecodeArgs {
  const void* q;
  void* out;
  int64_t ldq, ldo;
  const int32_t *table, *lens;
  const void *cache_kc, *cache_vc, *cache_kp, *cache_vp;
  int64_t pages;
  int width, tpp;              // table entries a sequence; tiles of 16 tokens a page
  int batch, kv, g, window;
  float c;                     // softmax scale times log2(e)
  int blocks;                  // of equal pieces; 0: one for each sequence, key head and 16 query heads
  float* part;                 // blocks > 0: blocks * 2 * 16 * (dim + 2)
};
// The blocks for sequences of up to `longest` tokens.
constexpr int kDecodeBlocks = 512;
int decode_blocks(int64_t batch, int kv, int g, int64_t longest);
hipError_t run_attn_decode(int dtype, int dim, int group, const AttnDecodeArgs& p, hipStream_t st);

struct AttnPrefillArgs {
  const void *q, *k, *v;
  void* out;
  int64_t ldq, ldk, ldv, ldo;
  const int32_t *cu_q, *cu_k;  // seqs + 1 offsets
  int64_t q_tokens, k_tokens;
  int seqs, kv, g, dim, causal, window;
  float c;
};
hipError_t run_attn_prefill(int dtype, const AttnPrefillArgs& p, hipStream_t st);

// ------------------------------------------------------------------ device helpers
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// a 16x16 (K = 32) and a 32x32 (K = 16) product of 16-bit fragments: lane l
// holds row (column) l % 16 (l % 32), of K its eight elements 8 * (l / 16)
// (8 * (l / 32)) on; the result holds column l % 16 (l % 32), rows
// 4 * (l / 16) + r (8 * (r / 4) + 4 * (l / 32) + r % 4)
template <class T> __device__ __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (std::is_same<T, _Float16>::value)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <class T> __device__ __forceinline__ f32x16 mma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (std::is_same<T, _Float16>::value)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// two f32 rounded to nearest even as one word of T
template <class T> __device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef T t2 __attribute__((ext_vector_type(2)));
  t2 v = {static_cast<T>(a), static_cast<T>(b)};
  return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ float f16_lo(uint32_t w) { return (float)__builtin_bit_cast(f16x2, w)[0]; }
__device__ __forceinline__ float f16_hi(uint32_t w) { return (float)__builtin_bit_cast(f16x2, w)[1]; }

// Eight codes of a word as a fragment of T, each plus a bias that is exact in
// T, elements in the order of channels 0, 4, 1, 5, 2, 6, 3, 7: a code in the
// low mantissa bits of a power of two.  f16 biases 1024, 1024, 64, 64, twice
// (a code four bits up in the mantissa of 64 is that code); bf16 128.
// `mask`: 0x000f000f in a vector register (code_mask), so that mask and bias
// are one instruction, whose other constant is the one scalar it may read.
__device__ __forceinline__ uint32_t code_mask() {
  uint32_t m = 0x000f000fu;
  asm("" : "+v"(m));
  return m;
}
template <class T> __device__ __forceinline__ u32x4 code_frag(uint32_t w, uint32_t mask) {
  if constexpr (std::is_same<T, _Float16>::value) {
    const uint32_t h = w >> 8, high = mask << 4;
    return u32x4{(w & mask) | 0x64006400u, (w & high) | 0x54005400u, (h & mask) | 0x64006400u, (h & high) | 0x54005400u};
  } else {
    return u32x4{(w & mask) | 0x43004300u, ((w >> 4) & mask) | 0x43004300u, ((w >> 8) & mask) | 0x43004300u,
                 ((w >> 12) & mask) | 0x43004300u};
  }
}
__device__ constexpr int kCodeOrder[8] = {0, 4, 1, 5, 2, 6, 3, 7};
template <class T> __device__ __forceinline__ constexpr float code_bias(int element) {
  return std::is_same<T, _Float16>::value ? ((element & 2) ? 64.0f : 1024.0f) : 128.0f;
}

// the larger of a value and the other half wave's
__device__ __forceinline__ float max_halves(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
  const uint32_t a = r[0], b = r[1];
  return __builtin_fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}
__device__ __forceinline__ float sum_halves(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
  const uint32_t a = r[0], b = r[1];
  return __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
}

// the largest of, and the sum over, the four lanes l % 16 + 16 i
__device__ __forceinline__ float max_quarters(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
  const uint32_t a = r[0], b = r[1];
  return max_halves(__builtin_fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)));
}
__device__ __forceinline__ float sum_quarters(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
  const uint32_t a = r[0], b = r[1];
  return sum_halves(__builtin_bit_cast(float, a) + __builtin_bit_cast(float, b));
}

// Waits for all but the wave's last N loads and for its LDS reads, then the
// block's barrier: the loads that write LDS are there for every wave, and what
// the waves have read may be overwritten.  (A fence would wait for all loads.)
template <int N> __device__ __forceinline__ void loads_barrier() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4));   // vmcnt(N) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// A buffer resource of `bytes` from a wave-uniform address: loads beyond read as zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_resource(const char* at, int bytes) {
  const uint64_t a = (uint64_t)at;
  const uint64_t u = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a) |
                     (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32)) << 32;
  return __builtin_amdgcn_make_buffer_rsrc((void*)u, (short)0, __builtin_amdgcn_readfirstlane(bytes), 0x00020000);
}

}  // namespace ohip
