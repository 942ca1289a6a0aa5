// The 4-bit cache's writes, reads and page moves (layout: kv4.cuh).
//
// append: a row of D values is D/8 lanes x 8 values (one 16-byte load each), a lane takes a token's K
// and its V. The row's power of two comes from the exponent bits of its largest magnitude, a group's
// scale from the two lanes that hold its 16 channels; all of it is exact but the two roundings to e4m3
// and e2m1 that the format is.
// read: a lane turns one 4-byte word of codes into eight 16-bit values (one 16-byte store).
// move: pages are contiguous, so a move is a copy; a second set of CTAs rewrites the tables in
// the same launch.
//
// Measured (B200, launched back to back): append 16384 tokens x 4 heads x 128 12.5 us (43 MB: 3.4 TB/s; it is
// the instructions of the quantisation that bound it, issue slots three quarters busy), x 256 22.7 us; read of
// the same 10.4 and 18.6 us (4.1 and 4.6 TB/s; widening the codes keeps the ALU 71 % busy, waits for loads follow); 700 pages of 16 layers, 64 tokens x 4 heads x 128, moved in
// 131 us (6.4 TB/s read and written, as a plain copy).
#include "kv4.cuh"

namespace {

using namespace d3b_kv4;

constexpr int kThreads = 256;

template <bool BF>
__device__ __forceinline__ float widen(uint32_t half_word) {
  if constexpr (BF) return __uint_as_float(half_word << 16);
  const uint16_t h = (uint16_t)half_word;
  return __half2float(*reinterpret_cast<const __half*>(&h));
}

__device__ __forceinline__ uint32_t to_e4m3(float x) {  // to nearest even; x in [0, 448]
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(x));
  return r & 0xFFu;
}

// eight values to e2m1, to nearest even and saturating at 6, value i in nibble i
__device__ __forceinline__ uint32_t to_e2m1x8(const float (&x)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7]));
  return r;
}

// Quotients x / s are formed as x * (1 / s), and must round to codes as themselves would. x has at most 11
// significant bits and s 4, so a quotient that is not a border of two codes is 2^-12 of itself away from one,
// far more than the product is off by. One that is a border is b = 1, 3, 5 or 7 (times a power of two) and
// x = b * s; for every s the reciprocal's nearest float lies above 1 / s, by so little that the product with
// b * s, rounded towards zero, is b (all 32 cases tried). Scales: x = 6 b with b of 5 bits, and
// 6 b * float(1 / 6) rounds to b (all tried).

// One row's codes of a lane's eight values, its group's scale and the row's exponent byte.
struct Coded {
  uint32_t codes, scale, exponent;
};

template <int D, bool BF>
__device__ __forceinline__ Coded quantise(const uint4 raw) {
  constexpr int kLanes = D / 8;
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  // largest magnitude as bits: ordered like the values, and a NaN or infinity is the largest
  const uint32_t top2 = __vmaxu2(__vmaxu2(w[0] & 0x7FFF7FFFu, w[1] & 0x7FFF7FFFu),
                                 __vmaxu2(w[2] & 0x7FFF7FFFu, w[3] & 0x7FFF7FFFu));
  uint32_t group = max(top2 & 0xFFFFu, top2 >> 16);
  group = max(group, __shfl_xor_sync(0xffffffffu, group, 1));
  uint32_t most = group;
#pragma unroll
  for (int o = 2; o < kLanes; o <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
  const bool bad = most >= (BF ? 0x7F80u : 0x7C00u);
  // least e with most <= 2688 * 2^e: 2688 = 1.3125 * 2^11; at least kExpMin (rows of zeros and subnormals too)
  const uint32_t bits = __float_as_uint(widen<BF>(most));
  const int e = max((int)(bits >> 23) - 127 - 11 + ((bits & 0x7FFFFFu) > 0x280000u ? 1 : 0), kExpMin);
  const float down = __uint_as_float((uint32_t)(127 - e) << 23);  // e in [-64, 117]
  Coded c;
  c.scale = bad ? 0u : to_e4m3(__fmul_rn(widen<BF>(group) * down, 1.0f / 6.0f));
  c.exponent = bad ? 255u : (uint32_t)(e + 127);
  const float scale = __half2float(__ushort_as_half((unsigned short)(decode_scales(c.scale) & 0xFFFFu)));
  const float by = scale > 0.f ? __frcp_rn(scale) * down : 0.f;
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __fmul_rz(widen<BF>(w[i] & 0xFFFFu), by);
    x[2 * i + 1] = __fmul_rz(widen<BF>(w[i] >> 16), by);
  }
  c.codes = bad ? 0u : to_e2m1x8(x);  // a NaN times zero is not zero
  return c;
}

// grid: (groups of tokens, kv head); D/8 lanes take a token's K row and its V row
template <int D, bool BF>
__global__ void __launch_bounds__(kThreads) append_kernel(uint8_t* __restrict__ pool, int64_t page_bytes, int64_t pages,
                                                          int page_shift, const uint16_t* __restrict__ k, int64_t sk_t,
                                                          int64_t sk_h, const uint16_t* __restrict__ v, int64_t sv_t,
                                                          int64_t sv_h, const int64_t* __restrict__ slots, int64_t n,
                                                          int* err) {
  constexpr int kLanes = D / 8;
  const int sub = threadIdx.x % kLanes;
  const int head = blockIdx.y;
  int64_t tok = (int64_t)blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes;
  bool live = tok < n;  // every lane stays for the shuffles
  tok = live ? tok : 0;
  const uint4 k_raw = __ldg(reinterpret_cast<const uint4*>(k + tok * sk_t + head * sk_h) + sub);
  const uint4 v_raw = __ldg(reinterpret_cast<const uint4*>(v + tok * sv_t + head * sv_h) + sub);
  const int64_t slot = __ldg(slots + tok);
  const int64_t page = slot >> page_shift;
  live = live && slot >= 0;
  if (live && page >= pages) {
    if (sub == 0) d3b::record_input_error(err, kSiteBadSlot);
    live = false;
  }
  const Coded ck = quantise<D, BF>(k_raw), cv = quantise<D, BF>(v_raw);
  if (!live) return;
  const int in_page = (int)slot & ((1 << page_shift) - 1);
  const int t = in_page & 15, group = sub >> 1;
  uint8_t* g = pool + page * page_bytes + ((head << (page_shift - 4)) + (in_page >> 4)) * (int64_t)granule_bytes(D);
  uint8_t* codes = g + t * (D / 2) + 4 * sub;
  *reinterpret_cast<uint32_t*>(codes) = ck.codes;
  *reinterpret_cast<uint32_t*>(codes + off_v(D)) = cv.codes;
  if (!(sub & 1)) {
    g[off_k_scale(D) + t * (D / 16) + group] = (uint8_t)ck.scale;
    g[off_v(D) + off_k_scale(D) + group * 16 + t] = (uint8_t)cv.scale;
  }
  if (sub == 0) {
    g[off_k_exp(D) + t] = (uint8_t)ck.exponent;
    g[off_v(D) + off_k_exp(D) + t] = (uint8_t)cv.exponent;
  }
}

// eight values of one word of codes; `power` finite or NaN, `most` the magnitude that may not be passed
template <bool BF>
__device__ __forceinline__ uint4 widen_codes(uint32_t codes, uint32_t scale2, float power, bool clamp) {
  uint32_t h[4], r[4];
  decode8(codes, h);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t p = hmul2(h[i], scale2);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p));
    float a = f.x * power, b = f.y * power;
    if (clamp) {
      constexpr float m = BF ? 3.3895313892515355e38f : 65504.f;  // the type's largest
      a = a > m ? m : (a < -m ? -m : a);                          // a NaN stays
      b = b > m ? m : (b < -m ? -m : b);
    }
    if constexpr (BF) {
      const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
      r[i] = *reinterpret_cast<const uint32_t*>(&v);
    } else {
      const __half2 v = __floats2half2_rn(a, b);
      r[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}

// one lane: 8 channels of four tokens of K or V (a quarter of a granule)
template <int D, bool BF>
__global__ void __launch_bounds__(kThreads) read_kernel(const uint8_t* __restrict__ pool, int64_t page_bytes,
                                                        int64_t pages, int page_shift,
                                                        const int32_t* __restrict__ table, int64_t tokens,
                                                        uint16_t* __restrict__ k, uint16_t* __restrict__ v, int* err) {
  constexpr int kLanes = D / 8;
  const int sub = threadIdx.x % kLanes;
  const int head = blockIdx.y;
  const bool is_v = blockIdx.z;
  const int64_t tok = 4 * ((int64_t)blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes);
  if (tok >= tokens) return;
  const int64_t page = __ldg(table + (tok >> page_shift));
  uint4 o[4] = {};
  if (page < 0 || page >= pages) {
    if (sub == 0) d3b::record_input_error(err, kSiteBadPage);
  } else {
    const int in_page = (int)tok & ((1 << page_shift) - 1);
    const int t = in_page & 15, group = sub >> 1;
    const uint8_t* g = pool + page * page_bytes + ((head << (page_shift - 4)) + (in_page >> 4)) * (int64_t)granule_bytes(D) +
                       (is_v ? off_v(D) : 0);
    const uint32_t* codes = reinterpret_cast<const uint32_t*>(g + t * (D / 2)) + sub;
    uint32_t c[4], scales = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = __ldg(codes + i * (D / 8));
    if (is_v) {
      scales = __ldg(reinterpret_cast<const uint32_t*>(g + off_k_scale(D) + group * 16 + t));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) scales |= (uint32_t)__ldg(g + off_k_scale(D) + (t + i) * (D / 16) + group) << (8 * i);
    }
    const uint32_t exps = __ldg(reinterpret_cast<const uint32_t*>(g + off_k_exp(D) + t));
    // only a row whose 2688 * 2^e passes the type's largest value can
    const bool clamp = __vmaxu4(exps, BF ? 0xF3F3F3F3u : 0x83838383u) != (BF ? 0xF3F3F3F3u : 0x83838383u);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      o[i] = widen_codes<BF>(c[i], decode_scales(((scales >> (8 * i)) & 0xFFu) * 0x101u),
                             row_power((exps >> (8 * i)) & 0xFFu), clamp);
  }
  uint4* out = reinterpret_cast<uint4*>((is_v ? v : k) + (head * tokens + tok) * D) + sub;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (tok + i < tokens) out[i * (D / 8)] = o[i];
}

constexpr int kMoveVec = 4;  // 16-byte loads in flight per thread
constexpr int kMoveChunk = kThreads * kMoveVec;  // 16-byte units per CTA

// position of `id` in ascending src[0, n), or -1
__device__ __forceinline__ int64_t find(const int32_t* __restrict__ src, int64_t n, int id) {
  int64_t lo = 0, hi = n;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (__ldg(src + mid) < id) lo = mid + 1; else hi = mid;
  }
  return lo < n && __ldg(src + lo) == id ? lo : -1;
}

__global__ void __launch_bounds__(kThreads) move_kernel(uint8_t* __restrict__ pool, int64_t layers, int64_t pages,
                                                        int64_t page_bytes, const int32_t* __restrict__ src,
                                                        const int32_t* __restrict__ dst, int64_t n, int chunks,
                                                        int64_t copy_ctas, int32_t* __restrict__ tables,
                                                        int64_t entries, int* err) {
  const int64_t cta = blockIdx.x;
  if (cta >= copy_ctas) {  // tables
    const int64_t step = ((int64_t)gridDim.x - copy_ctas) * kThreads;
    for (int64_t i = (cta - copy_ctas) * kThreads + threadIdx.x; i < entries; i += step) {
      const int64_t at = tables[i] < 0 ? -1 : find(src, n, tables[i]);
      if (at >= 0) {
        const int to = __ldg(dst + at);
        if (to >= 0 && to < pages) tables[i] = to;
      }
    }
    for (int64_t i = (cta - copy_ctas) * kThreads + threadIdx.x; i < n; i += step) {
      const bool order = i + 1 < n && __ldg(src + i) >= __ldg(src + i + 1);
      if (order || find(src, n, __ldg(dst + i)) >= 0) d3b::record_input_error(err, kSiteBadMove);
    }
    return;
  }
  const int chunk = (int)(cta % chunks);
  const int64_t pl = cta / chunks;
  const int64_t i = pl % n, layer = pl / n;
  const int64_t from = __ldg(src + i), to = __ldg(dst + i);
  if (from < 0 || from >= pages || to < 0 || to >= pages) {
    if (threadIdx.x == 0) d3b::record_input_error(err, kSiteBadPage);
    return;
  }
  const uint4* s = reinterpret_cast<const uint4*>(pool + (layer * pages + from) * page_bytes);
  uint4* d = reinterpret_cast<uint4*>(pool + (layer * pages + to) * page_bytes);
  const int64_t units = page_bytes / 16, base = (int64_t)chunk * kMoveChunk + threadIdx.x;
  uint4 x[kMoveVec];
#pragma unroll
  for (int j = 0; j < kMoveVec; ++j)
    if (base + j * kThreads < units) x[j] = s[base + j * kThreads];
#pragma unroll
  for (int j = 0; j < kMoveVec; ++j)
    if (base + j * kThreads < units) d[base + j * kThreads] = x[j];
}

template <int D>
int launch_append(const d3b_kv4_cache* c, int64_t layer, const void* k, const int64_t* ks, const void* v,
                  const int64_t* vs, const int64_t* slots, int64_t n, bool bf, int* err, cudaStream_t s) {
  const int64_t per = kThreads / (D / 8), ctas = (n + per - 1) / per;
  if (ctas > 0x7FFFFFFF) return D3B_EINVAL;
  const dim3 grid((unsigned)ctas, (unsigned)c->kv_heads);
  auto* kp = static_cast<const uint16_t*>(k);
  auto* vp = static_cast<const uint16_t*>(v);
  const int shift = log2_of(c->page_tokens);
  if (bf)
    append_kernel<D, true><<<grid, kThreads, 0, s>>>(layer_base(c, layer), page_bytes(c), c->pages, shift, kp, ks[0], ks[1], vp,
                                                 vs[0], vs[1], slots, n, err);
  else
    append_kernel<D, false><<<grid, kThreads, 0, s>>>(layer_base(c, layer), page_bytes(c), c->pages, shift, kp, ks[0], ks[1], vp,
                                                 vs[0], vs[1], slots, n, err);
  return d3b_host::check_launch();
}

template <int D>
int launch_read(const d3b_kv4_cache* c, int64_t layer, const int32_t* table, int64_t tokens, void* k, void* v, bool bf,
                int* err, cudaStream_t s) {
  const int64_t per = 4 * (kThreads / (D / 8)), ctas = (tokens + per - 1) / per;
  if (ctas > 0x7FFFFFFF) return D3B_EINVAL;
  const dim3 grid((unsigned)ctas, (unsigned)c->kv_heads, 2);
  auto* kp = static_cast<uint16_t*>(k);
  auto* vp = static_cast<uint16_t*>(v);
  const int shift = log2_of(c->page_tokens);
  if (bf)
    read_kernel<D, true><<<grid, kThreads, 0, s>>>(layer_base(c, layer), page_bytes(c), c->pages, shift, table, tokens, kp, vp,
                                                err);
  else
    read_kernel<D, false><<<grid, kThreads, 0, s>>>(layer_base(c, layer), page_bytes(c), c->pages, shift, table, tokens, kp, vp,
                                                err);
  return d3b_host::check_launch();
}

}  // namespace

extern "C" {

int64_t d3b_kv4_page_bytes(int kv_heads, int head_dim, int page_tokens) {
  if (!supported(kv_heads, head_dim, page_tokens)) return 0;
  return (int64_t)kv_heads * (page_tokens / kGrain) * granule_bytes(head_dim);
}

int d3b_kv4_append(const d3b_kv4_cache* cache, int64_t layer, const void* k, const int64_t* k_strides, const void* v,
                   const int64_t* v_strides, const int64_t* slots, int64_t n, int dtype, d3b_stream_t stream) {
  if (int rc = check_cache(cache, layer)) return rc;
  if (n < 0) return D3B_EINVAL;
  if (dtype != D3B_F16 && dtype != D3B_BF16) return D3B_EUNSUPPORTED;
  if (n == 0) return D3B_OK;
  if (!k || !v || !k_strides || !v_strides || !slots) return D3B_EINVAL;
  if (reinterpret_cast<uintptr_t>(k) % 16 || reinterpret_cast<uintptr_t>(v) % 16) return D3B_EALIGN;
  if (reinterpret_cast<uintptr_t>(slots) % 8) return D3B_EALIGN;
  for (int i = 0; i < 2; ++i)
    if (k_strides[i] % 8 || v_strides[i] % 8) return D3B_EALIGN;
  int* err = d3b_host::device_error_word();
  if (!err) return D3B_ECUDA;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool bf = dtype == D3B_BF16;
  switch (cache->head_dim) {
    case 64: return launch_append<64>(cache, layer, k, k_strides, v, v_strides, slots, n, bf, err, s);
    case 128: return launch_append<128>(cache, layer, k, k_strides, v, v_strides, slots, n, bf, err, s);
    default: return launch_append<256>(cache, layer, k, k_strides, v, v_strides, slots, n, bf, err, s);
  }
}

int d3b_kv4_read(const d3b_kv4_cache* cache, int64_t layer, const int32_t* table, int64_t n_pages, int64_t tokens,
                 void* k, void* v, int dtype, d3b_stream_t stream) {
  if (int rc = check_cache(cache, layer)) return rc;
  if (tokens < 0 || n_pages < 0) return D3B_EINVAL;
  if (dtype != D3B_F16 && dtype != D3B_BF16) return D3B_EUNSUPPORTED;
  if (tokens == 0) return D3B_OK;
  if (!table || !k || !v || n_pages > 0x7FFFFFFF || n_pages * cache->page_tokens < tokens) return D3B_EINVAL;
  if (reinterpret_cast<uintptr_t>(k) % 16 || reinterpret_cast<uintptr_t>(v) % 16) return D3B_EALIGN;
  if (reinterpret_cast<uintptr_t>(table) % 4) return D3B_EALIGN;
  int* err = d3b_host::device_error_word();
  if (!err) return D3B_ECUDA;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool bf = dtype == D3B_BF16;
  switch (cache->head_dim) {
    case 64: return launch_read<64>(cache, layer, table, tokens, k, v, bf, err, s);
    case 128: return launch_read<128>(cache, layer, table, tokens, k, v, bf, err, s);
    default: return launch_read<256>(cache, layer, table, tokens, k, v, bf, err, s);
  }
}

int d3b_kv4_move_pages(const d3b_kv4_cache* cache, const int32_t* src, const int32_t* dst, int64_t n, int32_t* tables,
                       int64_t entries, d3b_stream_t stream) {
  if (cache && cache->layers == 0) return n == 0 ? D3B_OK : D3B_EINVAL;
  if (int rc = check_cache(cache, 0)) return rc;
  if (n < 0 || entries < 0 || (entries > 0 && !tables)) return D3B_EINVAL;
  if (n == 0) return D3B_OK;
  if (!src || !dst || n > cache->pages) return D3B_EINVAL;
  if (reinterpret_cast<uintptr_t>(src) % 4 || reinterpret_cast<uintptr_t>(dst) % 4 ||
      reinterpret_cast<uintptr_t>(tables) % 4)
    return D3B_EALIGN;
  const int64_t pb = page_bytes(cache), units = pb / 16;
  const int64_t chunks = (units + kMoveChunk - 1) / kMoveChunk, copy = n * cache->layers * chunks;
  int64_t extra = entries == 0 ? 0 : ((entries > n ? entries : n) + kThreads - 1) / kThreads;
  if (extra > 1024) extra = 1024;
  if (copy + extra > 0x7FFFFFFF) return D3B_EINVAL;
  int* err = d3b_host::device_error_word();
  if (!err) return D3B_ECUDA;
  move_kernel<<<(unsigned)(copy + extra), kThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      static_cast<uint8_t*>(cache->pool), cache->layers, cache->pages, pb, src, dst, n, (int)chunks, copy, tables,
      entries, err);
  return d3b_host::check_launch();
}

}  // extern "C"
