// Layout of the 4-bit key/value cache shared by its kernels.
//
// A pool is [layers][pages][page]; a page holds, per kv head, page_tokens / 16 granules of 16
// tokens. A granule of head dimension D is 18 D + 32 bytes:
//
//   K codes     [16][D/2]   two e2m1 codes a byte, the even channel in the low half
//   K scales    [16][D/16]  e4m3, one for 16 channels
//   K exponents [16]        one power of two a token's row, biased by 127; 255 = row not finite
//   V codes     [16][D/2]
//   V scales    [D/16][16]  transposed: the two tokens of a matrix operand's pair are neighbours
//   V exponents [16]
//
// value = code * scale * 2^(exponent - 127). A code has 2 significant bits and a scale 4, so
// code * scale is exact in fp16 (at most 6 * 448, a multiple of 2^-10) and in bf16; the row's
// power of two carries the range of the values.
#pragma once

#include "common.cuh"

namespace d3b_kv4 {

constexpr int kGrain = 16;
constexpr int kExpMin = -64;  // exponent of rows whose values are all below 2688 * 2^-64

// codes of the device error word
constexpr int kSiteBadSlot = 2101;    // a slot behind the pool's last
constexpr int kSiteBadPage = 2102;    // a page number behind the pool's last (or negative where one is read)
constexpr int kSiteBadLength = 2103;  // a length below 0 or above the table's tokens
constexpr int kSiteBadMove = 2104;    // page lists not ascending, or a destination among the sources

__host__ __device__ constexpr int granule_bytes(int dim) { return 18 * dim + 32; }
__host__ __device__ constexpr int off_k_scale(int dim) { return 8 * dim; }
__host__ __device__ constexpr int off_k_exp(int dim) { return 9 * dim; }
__host__ __device__ constexpr int off_v(int dim) { return 9 * dim + 16; }

inline bool supported(int kv_heads, int head_dim, int page_tokens) {
  return kv_heads > 0 && kv_heads <= 65535 && (head_dim == 64 || head_dim == 128 || head_dim == 256) &&
         page_tokens >= 16 && page_tokens <= 256 && (page_tokens & (page_tokens - 1)) == 0;
}

// D3B_OK, or why the cache and layer cannot be used.
inline int check_cache(const d3b_kv4_cache* c, int64_t layer) {
  if (!c || c->layers < 0 || c->pages < 0 || layer < 0 || layer >= c->layers) return D3B_EINVAL;
  if (!supported(c->kv_heads, c->head_dim, c->page_tokens)) return D3B_EUNSUPPORTED;
  if (c->pages > 0x7FFFFFFF) return D3B_EINVAL;
  if (c->pages > 0 && !c->pool) return D3B_EINVAL;
  if (reinterpret_cast<uintptr_t>(c->pool) % 16) return D3B_EALIGN;
  return D3B_OK;
}

inline int64_t page_bytes(const d3b_kv4_cache* c) {
  return (int64_t)c->kv_heads * (c->page_tokens / kGrain) * granule_bytes(c->head_dim);
}

inline uint8_t* layer_base(const d3b_kv4_cache* c, int64_t layer) {
  return static_cast<uint8_t*>(c->pool) + layer * c->pages * page_bytes(c);
}

inline int log2_of(int n) {
  int s = 0;
  while ((1 << s) < n) ++s;
  return s;
}

// 2^(byte - 127), NaN for 255
__device__ __forceinline__ float row_power(uint32_t byte) {
  // byte 0 would be the subnormal 2^-127; rows never carry it (exponents start at kExpMin)
  return byte == 255u ? __int_as_float(0x7FC00000) : __uint_as_float(byte << 23);
}

// four pairs of fp16 values (low half = low code) of a word of eight e2m1 codes
__device__ __forceinline__ void decode8(uint32_t w, uint32_t (&o)[4]) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3])
      : "r"(w));
}

// two e4m3 scales (low byte = low half)
__device__ __forceinline__ uint32_t decode_scales(uint32_t two) {
  uint32_t r;
  asm("{\n\t.reg .b16 s;\n\tcvt.u16.u32 s, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, s;\n\t}" : "=r"(r) : "r"(two));
  return r;
}

__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

}  // namespace d3b_kv4
