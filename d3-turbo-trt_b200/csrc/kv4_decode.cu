// Attention of a sequence's newest tokens over its 4-bit cache (layout: kv4.cuh).
//
// A kv head's queries (its group's heads x L tokens) are rows; a CTA takes up to 8 * NT of them
// against a share of the sequence's keys. Products are m16n8k16 on fp16 with fp32 sums, turned so
// that keys (then channels) are the 16 and query rows the 8:
//
//   S^T [16 keys x 8 rows]  = K [16 keys x D] . Q^T         A = decoded K codes
//   O^T [D x 8 rows]       += V^T [D x 16 keys] . W^T       A = decoded V codes
//
// Every thread decodes its own operand from the bytes it needs (a K row's quarter is 16 bytes at
// D = 128), so nothing is widened in shared memory. code * scale is exact in fp16 and queries are
// brought under a power of two a row, so S has no rounding but its fp32 sums. A V row's power of
// two cannot be applied after the sum over keys; it goes into the weight's exponent instead:
//
//   s_j in base 2, t_j = s_j + e_j, m = max t:
//   O = sum_j 2^(t_j - m) (code * scale)_j,  l = sum_j 2^(s_j - m),  out = O / l
//
// Weights 2^(t - m) stay at most 1 and keep fp16's 11 bits whatever the rows' powers are. The terms
// of l are fp32 numbers up to 2^64 (e >= -64); with V values beyond 2^100 the least of them fall
// below fp32's range, keys whose weight is under 2^-9 of the largest at the very end of bf16.
// The weights change from accumulator to operand layout by movmatrix.
//
// Each warp walks its own 32-key pairs of granules through its own cp.async ring, without barriers;
// the warps' and then the key shares' partial results are merged in a fixed order.
//
// Bound: the cache's bytes; 18 D + 32 of them per 16 tokens and kv head.
#include "kv4.cuh"

namespace {

using namespace d3b_kv4;

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;

struct DecodeArgs {
  const uint8_t* pool;
  int64_t page_bytes, pages, head_bytes;
  int page_shift;
  const uint16_t* q;
  int64_t sq_b, sq_h, sq_l;
  uint16_t* out;
  int64_t so_b, so_h, so_l;
  const int32_t* table;
  int64_t table_stride, width;
  const int32_t* lengths;
  int kv_heads, group, L, causal, splits, row_tiles;
  float scale_log2;
  float* part_o;   // [units][splits][8 NT][D]
  float* part_st;  // [units][splits][8 NT][2]: m, l
  int* err;
};

template <int D, int NT>
struct Shape {
  static constexpr int kStage = (granule_bytes(D) + 127) / 128 * 128;  // V rows start on 128-byte lines
  static constexpr int kRows = 8 * NT;
  static constexpr int kResident = NT == 1 ? (D == 64 ? 5 : D == 128 ? 4 : 3) : 2;  // CTAs an SM by registers
  static constexpr int kRing = kWarps * 2 * 2 * kStage;  // two pairs of granules a warp
  static constexpr int kMerge = kWarps * kRows * (D + 2) * 4;
  static constexpr int kQ = kRows * D * 2;
  static constexpr int kSmem = (kRing > kMerge ? kRing : kMerge) + kQ + kRows * 4;
  // where a granule's parts sit in a ring stage
  static constexpr int kKc = 0, kVc = 8 * D, kKs = 16 * D, kVs = 17 * D, kKe = 18 * D, kVe = 18 * D + 16;
};

// 16-byte unit of a V code line (128 bytes): spread so that the four row pairs of a load's lanes hit all banks
template <int D>
__device__ __forceinline__ int v_swizzle(int byte) {
  const int line = byte >> 7;
  const int x = D == 64 ? (line & 1) : D == 128 ? (line & 3) : ((line >> 1) & 3);
  return byte ^ (x << 5);
}

__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float max_over_rows(float x) {  // over the 8 lanes that share lane % 4; a NaN gives way
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
  return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
}

__device__ __forceinline__ float finite_or_zero(float m) { return m == -INFINITY ? 0.f : m; }

template <int W>
__device__ __forceinline__ void lds_words(uint32_t addr, uint32_t* w) {
  if constexpr (W == 1)
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0]) : "r"(addr));
  else if constexpr (W == 2)
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
  else
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
}
__device__ __forceinline__ uint32_t lds_u8(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t lds_u16(uint32_t addr) {
  uint32_t v;
  asm volatile("{\n\t.reg .b16 h;\n\tld.shared.b16 h, [%1];\n\tcvt.u32.u16 %0, h;\n\t}" : "=r"(v) : "r"(addr));
  return v;
}

// the low half of every byte from a, the high half from b
__device__ __forceinline__ uint32_t low_nibbles(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xCA;" : "=r"(r) : "r"(0x0F0F0F0Fu), "r"(a), "r"(b));
  return r;
}

template <bool BF>
__device__ __forceinline__ float2 widen2(uint32_t w) {
  if constexpr (BF) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

template <bool BF>
__device__ __forceinline__ uint16_t narrow(float x) {
  if constexpr (BF) {
    const __nv_bfloat16 r = __float2bfloat16_rn(x);
    return *reinterpret_cast<const uint16_t*>(&r);
  } else {
    const __half r = __float2half_rn(x);
    return *reinterpret_cast<const uint16_t*>(&r);
  }
}

template <int N>
struct Int {
  static constexpr int value = N;
};

// byte - 127 as a float, NaN for 255
__device__ __forceinline__ float exponent(uint32_t byte) {
  return byte == 255u ? __int_as_float(0x7FC00000) : __uint_as_float(0x4B000000u | byte) - 8388735.f;
}

// a partial result (O, (m, l)) brought to the reference `base` and added
__device__ __forceinline__ void add_part(float4& acc, float& sum, const float4 o, const float2 st, float base) {
  const float f = ex2(st.x - base);
  sum = fmaf(st.y, f, sum);
  acc.x = fmaf(o.x, f, acc.x);
  acc.y = fmaf(o.y, f, acc.y);
  acc.z = fmaf(o.z, f, acc.z);
  acc.w = fmaf(o.w, f, acc.w);
}

// four channels of a finished row; zeros where there was no key
template <bool BF>
__device__ __forceinline__ void store_row(const DecodeArgs& a, int b, int kvh, int row, int d, const float4 acc, float sum) {
  const float f = sum == 0.f ? 0.f : 1.f / sum;
  const int l = row / a.group, h = kvh * a.group + row % a.group;
  const uint32_t lo = narrow<BF>(acc.x * f) | ((uint32_t)narrow<BF>(acc.y * f) << 16);
  const uint32_t hi = narrow<BF>(acc.z * f) | ((uint32_t)narrow<BF>(acc.w * f) << 16);
  *reinterpret_cast<uint2*>(a.out + b * a.so_b + h * a.so_h + l * a.so_l + d) = make_uint2(lo, hi);
}

// Queries to shared memory in operand order, as fp16 under a power of two a row:
// [nt][word][lane] x 16 bytes, lane = 4 * row + quarter; row_scale = scale * log2(e) * 2^power.
template <int D, int NT, bool BF>
__device__ __forceinline__ void load_queries(const DecodeArgs& a, int b, int kvh, int row0, int rows, uint4* qs,
                                             float* row_scale) {
  constexpr int kLanes = D / 8;  // a lane takes 8 channels
  constexpr int kWords = D / 32;
  for (int i = threadIdx.x; i < 8 * NT * kLanes; i += kThreads) {
    const int row = i / kLanes, sub = i % kLanes;
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (row0 + row < rows) {
      const int l = (row0 + row) / a.group, g = (row0 + row) % a.group;
      raw = __ldg(reinterpret_cast<const uint4*>(a.q + b * a.sq_b + (int64_t)(kvh * a.group + g) * a.sq_h + l * a.sq_l) + sub);
    }
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    float2 f[4];
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[j] = widen2<BF>(w[j]);
      top = fmaxf(top, fmaxf(fabsf(f[j].x), fabsf(f[j].y)));
    }
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    // largest magnitude to [2^14, 2^15), as far as a factor of 2^126 goes; rows that are not finite stay
    int up = 0;
    if (top < INFINITY) up = min(126, 14 - ((int)(__float_as_uint(top) >> 23) - 127));
    const float by = __uint_as_float((uint32_t)(127 + up) << 23);  // up in [-113, 126]
    uint32_t h[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __half2 v = __floats2half2_rn(f[j].x * by, f[j].y * by);
      h[j] = *reinterpret_cast<const uint32_t*>(&v);
    }
    // channels 8 sub ...: which word of which quarter they are (see the K loads)
    const int half = D == 256 ? sub / 16 : 0, in = D == 256 ? sub % 16 : sub;
    const int per = D == 256 ? 4 : kWords;
    const int quarter = in / per, word = half * 4 + in % per;
    qs[((row / 8) * kWords + word) * 32 + (row % 8) * 4 + quarter] = make_uint4(h[0], h[1], h[2], h[3]);
    if (sub == 0) row_scale[row] = a.scale_log2 * __uint_as_float((uint32_t)(127 - up) << 23);
  }
}

template <int D, int NT, bool BF>
__global__ void __launch_bounds__(kThreads, Shape<D, NT>::kResident) decode_kernel(const __grid_constant__ DecodeArgs a) {
  using P = Shape<D, NT>;
  constexpr int kKWords = D / 32, kVWords = D / 64, kTiles = D / 16;
  extern __shared__ __align__(128) uint8_t smem[];
  uint4* qs = reinterpret_cast<uint4*>(smem + (P::kRing > P::kMerge ? P::kRing : P::kMerge));
  float* row_scale = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(qs) + P::kQ);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, r = lane / 4, c = lane % 4;

  int unit = blockIdx.x / a.splits;
  const int split = blockIdx.x % a.splits;
  const int64_t part = blockIdx.x;
  const int tile = unit % a.row_tiles;
  unit /= a.row_tiles;
  const int kvh = unit % a.kv_heads, b = unit / a.kv_heads;
  const int rows = a.group * a.L, row0 = tile * P::kRows;

  const int64_t most = a.width << a.page_shift;
  int64_t len = __ldg(a.lengths + b);
  if (len < 0 || len > most) {
    if (threadIdx.x == 0) d3b::record_device_error(a.err, kSiteBadLength);
    len = len < 0 ? 0 : most;
  }
  const int grains = (int)((len + 15) / 16);
  const int share = ((grains + a.splits - 1) / a.splits + 1) & ~1;  // even: a pair starts at an even granule
  const int g_first = (int)min((int64_t)split * share, (int64_t)grains), g_end = min(g_first + share, grains);
  const int my_first = g_first + 2 * warp;  // the warp's pairs: my_first, my_first + 2 kWarps, ...
  const int pairs = my_first < g_end ? (g_end - my_first + 2 * kWarps - 1) / (2 * kWarps) : 0;

  const uint32_t ring = d3b::smem_u32(smem) + warp * (2 * 2 * P::kStage);
  const int32_t* table = a.table + b * a.table_stride;
  const int grain_shift = a.page_shift - 4, in_page = (1 << grain_shift) - 1;
  // a lane copies units lane, lane + 32, ... of 16 bytes of a granule; where each goes in a stage
  constexpr int kUnits = granule_bytes(D) / 16, kCopies = (kUnits + 31) / 32;
  uint32_t place[kCopies];
#pragma unroll
  for (int i = 0; i < kCopies; ++i) {
    constexpr int kHalf = off_v(D) / 16, kCodes = 8 * D / 16, kScales = D / 16;
    const int u = 32 * i + lane;
    const bool is_v = u >= kHalf;
    const int x = is_v ? u - kHalf : u;  // unit within K's or V's part
    int to;
    if (x < kCodes) to = is_v ? P::kVc + v_swizzle<D>(16 * x) : P::kKc + 16 * x;
    else if (x < kCodes + kScales) to = (is_v ? P::kVs : P::kKs) + 16 * (x - kCodes);
    else to = is_v ? P::kVe : P::kKe;
    place[i] = ring + to;
    asm volatile("" : "+r"(place[i]));  // kept, not worked out again at every copy
  }
  const uint8_t* head_pool = a.pool + kvh * a.head_bytes + 16 * lane;
  int ids[2];  // page numbers of the pair that is loaded next
  auto look = [&](int pair) {
    const int g = my_first + pair * 2 * kWarps;
    ids[0] = __ldg(table + (g >> grain_shift));
    // pairs start at even granules: both lie in one page unless a page is one granule
    ids[1] = grain_shift || g + 1 >= g_end ? ids[0] : __ldg(table + g + 1);
  };
  // copies a pair to ring slot SLOT; 0, or one bit for each granule whose page is not in the pool
  auto load = [&](int pair, auto slot) -> uint32_t {
    constexpr int kSlot = decltype(slot)::value;
    const int g = my_first + pair * 2 * kWarps;
    uint32_t bad = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if ((uint32_t)ids[i] < (uint32_t)a.pages) {
        const uint8_t* src = head_pool + ids[i] * a.page_bytes + ((g + i) & in_page) * granule_bytes(D);
        if (i == 0 || g + 1 < g_end) {
#pragma unroll
          for (int x = 0; x < kCopies; ++x)
            if (32 * x + 31 < kUnits || 32 * x + lane < kUnits)
              cp16(place[x] + (2 * kSlot + i) * P::kStage, src + 512 * x);
        }
      } else {
        bad |= 1u << i;
        if (lane == 0) d3b::record_device_error(a.err, kSiteBadPage);
      }
    }
    return bad;
  };
  uint32_t bad_now = 0, bad_next = 0;
  if (pairs > 0) {
    look(0);
    bad_now = load(0, Int<0>{});
  }
  cp_commit();
  if (pairs > 1) look(1);

  load_queries<D, NT, BF>(a, b, kvh, row0, rows, qs, row_scale);
  __syncthreads();

  float o[NT][kTiles][4];
  float m[NT][2], l[NT][2], qf[NT][2];
  int limit[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[n][t][j] = 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int row = n * 8 + 2 * c + j;
      m[n][j] = -INFINITY;
      l[n][j] = 0.f;
      qf[n][j] = row_scale[row];
      limit[n][j] = a.causal ? (int)len - (a.L - 1 - (row0 + row) / a.group) : (int)len;
    }
  }
  constexpr bool kHold = NT * D <= 256;  // queries stay in registers
  uint4 qr[kHold ? NT : 1][kHold ? kKWords : 1];
  if constexpr (kHold) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int w = 0; w < kKWords; ++w) qr[n][w] = qs[(n * kKWords + w) * 32 + lane];
  }
  const int first_limit = a.causal ? (int)len - (a.L - 1) : (int)len;
  const uint32_t k_at = ring + P::kKc + r * (D / 2) + c * (D == 256 ? 16 : D / 8);
  const uint32_t ks_at = ring + P::kKs + r * (D / 16) + (D == 64 ? c : 2 * c);
  const uint32_t e_at = ring + P::kKe + r;
  const uint32_t vs_at = ring + P::kVs + (D == 64 ? r / 2 : D == 128 ? r : 2 * r) * 16 + 2 * c;
  uint32_t v_at[4];  // V rows 2c, 2c + 1, 2c + 8, 2c + 9
#pragma unroll
  for (int x = 0; x < 4; ++x)
    v_at[x] = ring + P::kVc + v_swizzle<D>((2 * c + (x & 1) + 8 * (x >> 1)) * (D / 2) + r * (D / 16));

  auto step = [&](int pair, auto slot) {
    constexpr int kAt = 2 * decltype(slot)::value * P::kStage;
    __syncwarp();  // every lane is done with the slot that is loaded next
    if (pair + 1 < pairs) {
      bad_next = load(pair + 1, Int<1 - decltype(slot)::value>{});
      if (pair + 2 < pairs) look(pair + 2);
    }
    cp_commit();
    cp_wait<1>();
    __syncwarp();

    const int key0 = 16 * (my_first + pair * 2 * kWarps);
    const bool edge = key0 + 32 > first_limit || bad_now;  // some key is masked for some row
    float s[2][NT][4], t[2][NT][4];
    int live[2] = {16, 16};  // tokens of the granule that are keys at all
    if (edge) {
#pragma unroll
      for (int i = 0; i < 2; ++i) live[i] = (bad_now >> i) & 1 ? 0 : min(16, (int)len - key0 - 16 * i);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int at = kAt + i * P::kStage;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][n][j] = 0.f;
      uint32_t k0[kKWords], k1[kKWords], s0[kKWords / 2], s1[kKWords / 2];  // keys r and r + 8; a scale per two words
      lds_words<D == 256 ? 4 : kKWords>(k_at + at, k0);
      lds_words<D == 256 ? 4 : kKWords>(k_at + at + 4 * D, k1);
      if constexpr (D == 256) {
        lds_words<4>(k_at + at + 64, k0 + 4);
        lds_words<4>(k_at + at + 4 * D + 64, k1 + 4);
      }
      if constexpr (D == 64) {
        s0[0] = decode_scales(lds_u8(ks_at + at) * 0x101u);
        s1[0] = decode_scales(lds_u8(ks_at + at + D / 2) * 0x101u);
      } else {
#pragma unroll
        for (int w = 0; w < kKWords / 4; ++w) {
          const uint32_t x0 = decode_scales(lds_u16(ks_at + at + 8 * w));
          const uint32_t x1 = decode_scales(lds_u16(ks_at + at + D / 2 + 8 * w));
          s0[2 * w] = __byte_perm(x0, 0, 0x1010);
          s0[2 * w + 1] = __byte_perm(x0, 0, 0x3232);
          s1[2 * w] = __byte_perm(x1, 0, 0x1010);
          s1[2 * w + 1] = __byte_perm(x1, 0, 0x3232);
        }
      }
#pragma unroll
      for (int w = 0; w < kKWords; ++w) {
        uint32_t d0[4], d1[4];
        decode8(k0[w], d0);
        decode8(k1[w], d1);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          d0[j] = hmul2(d0[j], s0[w / 2]);
          d1[j] = hmul2(d1[j], s1[w / 2]);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          uint4 qv;
          if constexpr (kHold) qv = qr[n][w];
          else qv = qs[(n * kKWords + w) * 32 + lane];
          mma16816(s[i][n], d0[0], d1[0], d0[1], d1[1], qv.x, qv.y);
          mma16816(s[i][n], d0[2], d1[2], d0[3], d1[3], qv.z, qv.w);
        }
      }
      // a marked row (255) has codes of zero: its score is 0 * infinity here
      const float kf0 = __uint_as_float(lds_u8(e_at + at) << 23), kf1 = __uint_as_float(lds_u8(e_at + at + 8) << 23);
      const float ev0 = exponent(lds_u8(e_at + at + P::kVe - P::kKe)), ev1 = exponent(lds_u8(e_at + at + P::kVe - P::kKe + 8));
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s[i][n][j] *= (j < 2 ? kf0 : kf1) * qf[n][j & 1];
          t[i][n][j] = s[i][n][j] + (j < 2 ? ev0 : ev1);
        }
        if (edge) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int key = r + (j < 2 ? 0 : 8);
            if (key >= live[i] || key0 + 16 * i + key >= limit[n][j & 1]) s[i][n][j] = t[i][n][j] = -INFINITY;
          }
        }
      }
    }

    uint32_t wf[2][NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float keep[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float top = max_over_rows(fmaxf(fmaxf(t[0][n][j], t[0][n][j + 2]), fmaxf(t[1][n][j], t[1][n][j + 2])));
        const float new_m = fmaxf(m[n][j], top), base = finite_or_zero(new_m);
        keep[j] = ex2(m[n][j] - base);
        m[n][j] = new_m;
        l[n][j] *= keep[j];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          l[n][j] += ex2(s[i][n][j] - base) + ex2(s[i][n][j + 2] - base);
          t[i][n][j] = ex2(t[i][n][j] - base);
          t[i][n][j + 2] = ex2(t[i][n][j + 2] - base);
        }
      }
      if (__any_sync(0xffffffffu, keep[0] != 1.f || keep[1] != 1.f)) {
#pragma unroll
        for (int x = 0; x < kTiles; ++x)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[n][x][j] *= keep[j & 1];
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const __half2 h = __floats2half2_rn(t[i][n][2 * j], t[i][n][2 * j + 1]);
          wf[i][n][j] = transpose8x8(*reinterpret_cast<const uint32_t*>(&h));
        }
    }

#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int at = kAt + i * P::kStage;
      uint32_t v[4][kVWords];
#pragma unroll
      for (int x = 0; x < 4; ++x) lds_words<kVWords>(v_at[x] + at, v[x]);
      uint32_t sc01 = 0, sc89 = 0;
#pragma unroll
      for (int w = 0; w < kVWords; ++w) {
        if (w == 0 || (D == 256 && w == 2)) {
          uint32_t b01 = lds_u16(vs_at + at + 8 * w), b89 = lds_u16(vs_at + at + 8 * w + 8);
          if (edge) {  // a granule's last rows may never have been written: their scales can be NaN
            b01 &= (2 * c < live[i] ? 0xFFu : 0u) | (2 * c + 1 < live[i] ? 0xFF00u : 0u);
            b89 &= (2 * c + 8 < live[i] ? 0xFFu : 0u) | (2 * c + 9 < live[i] ? 0xFF00u : 0u);
          }
          sc01 = decode_scales(b01);
          sc89 = decode_scales(b89);
        }
        uint32_t x0[4], x1[4], y0[4], y1[4];
        decode8(low_nibbles(v[0][w], v[1][w] << 4), x0);
        decode8(low_nibbles(v[0][w] >> 4, v[1][w]), x1);
        decode8(low_nibbles(v[2][w], v[3][w] << 4), y0);
        decode8(low_nibbles(v[2][w] >> 4, v[3][w]), y1);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint32_t a0 = hmul2(x0[x], sc01), a1 = hmul2(x1[x], sc01), a2 = hmul2(y0[x], sc89), a3 = hmul2(y1[x], sc89);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16816(o[n][4 * w + x], a0, a1, a2, a3, wf[i][n][0], wf[i][n][1]);
        }
      }
    }
    bad_now = bad_next;
  };
  for (int pair = 0; pair < pairs; pair += 2) {
    step(pair, Int<0>{});
    if (pair + 1 < pairs) step(pair + 1, Int<1>{});
  }
  cp_wait<0>();

  // merge the warps: O and (m, l) through shared memory, where the rings were
  __syncthreads();
  float* mo = reinterpret_cast<float*>(smem);   // [warp][row][D]
  float* ms = mo + kWarps * P::kRows * D;       // [warp][row][2]
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float sum = l[n][j];
      sum += __shfl_xor_sync(0xffffffffu, sum, 4);
      sum += __shfl_xor_sync(0xffffffffu, sum, 8);
      sum += __shfl_xor_sync(0xffffffffu, sum, 16);
      const int row = warp * P::kRows + n * 8 + 2 * c + j;
      if (r == 0) *reinterpret_cast<float2*>(ms + row * 2) = make_float2(m[n][j], sum);
      float* dst = mo + row * D + r * (D / 8);
#pragma unroll
      for (int x = 0; x < kTiles; x += 2)
        *reinterpret_cast<float4*>(dst + 2 * x) = make_float4(o[n][x][j], o[n][x][j + 2], o[n][x + 1][j], o[n][x + 1][j + 2]);
    }
  __syncthreads();
  for (int i = threadIdx.x; i < P::kRows * (D / 4); i += kThreads) {
    const int row = i / (D / 4), d = 4 * (i % (D / 4));
    if (row0 + row >= rows) continue;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, ms[(w * P::kRows + row) * 2]);
    const float base = finite_or_zero(top);
    float sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float2 st = *reinterpret_cast<const float2*>(ms + (w * P::kRows + row) * 2);
      add_part(acc, sum, *reinterpret_cast<const float4*>(mo + (w * P::kRows + row) * D + d), st, base);
    }
    if (a.splits == 1) {
      store_row<BF>(a, b, kvh, row0 + row, d, acc, sum);
    } else {
      *reinterpret_cast<float4*>(a.part_o + (part * P::kRows + row) * D + d) = acc;
      if (d == 0) *reinterpret_cast<float2*>(a.part_st + (part * P::kRows + row) * 2) = make_float2(top, sum);
    }
  }
}

// one CTA a row: the key shares' partial results in order
template <int D, bool BF>
__global__ void __launch_bounds__(D / 4) merge_kernel(const __grid_constant__ DecodeArgs a, int tile_rows) {
  const int rows = a.group * a.L;
  const int row = blockIdx.x % rows;
  const int64_t bk = blockIdx.x / rows;
  const int kvh = (int)(bk % a.kv_heads);
  const int64_t b = bk / a.kv_heads;
  const int64_t unit = bk * a.row_tiles + row / tile_rows;
  const int64_t first = unit * a.splits * tile_rows + row % tile_rows;
  float top = -INFINITY;
  for (int s = 0; s < a.splits; ++s) top = fmaxf(top, a.part_st[(first + (int64_t)s * tile_rows) * 2]);
  const float base = finite_or_zero(top);
  float sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  const int d = 4 * threadIdx.x;
#pragma unroll 4
  for (int s = 0; s < a.splits; ++s) {
    const int64_t at = first + (int64_t)s * tile_rows;
    const float2 st = *reinterpret_cast<const float2*>(a.part_st + at * 2);
    add_part(acc, sum, *reinterpret_cast<const float4*>(a.part_o + at * D + d), st, base);
  }
  store_row<BF>(a, (int)b, kvh, row, d, acc, sum);
}

struct Plan {
  int nt, row_tiles, splits;
  int64_t units;
};

bool make_plan(const d3b_kv4_cache* c, int B, int H, int L, int64_t width, Plan* p) {
  const int64_t rows = (int64_t)(H / c->kv_heads) * L;
  p->nt = rows <= 8 ? 1 : rows <= 16 || c->head_dim == 256 ? 2 : 4;
  const int64_t tiles = (rows + 8 * p->nt - 1) / (8 * p->nt);
  p->units = (int64_t)B * c->kv_heads * tiles;
  if (tiles > 0x7FFFFFFF || p->units > 0x7FFFFFFF) return false;
  p->row_tiles = (int)tiles;
  const int64_t grains = width * (c->page_tokens / kGrain);
  const int64_t want = 8ll * d3b_host::num_sms(d3b_host::current_device());
  int64_t splits = (want + p->units - 1) / p->units;
  const int64_t most = (grains + 2 * kWarps - 1) / (2 * kWarps);
  splits = splits > most ? most : splits;
  splits = splits > 128 ? 128 : splits;
  p->splits = splits < 1 ? 1 : (int)splits;
  return p->units * p->splits <= 0x7FFFFFFF;
}

size_t plan_bytes(const Plan& p, int D) {
  return p.splits == 1 ? 0 : (size_t)p.units * p.splits * 8 * p.nt * (D + 2) * 4;
}

template <int D, int NT, bool BF>
int launch(const DecodeArgs& a, const Plan& p, int B, cudaStream_t s) {
  constexpr int smem = Shape<D, NT>::kSmem;
  static bool ready[64];  // by device; setting it twice is harmless
  const int dev = d3b_host::current_device();
  if (smem > 48 * 1024 && (dev < 0 || dev >= 64 || !ready[dev])) {
    if (cudaFuncSetAttribute(decode_kernel<D, NT, BF>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
      return D3B_ECUDA;
    if (dev >= 0 && dev < 64) ready[dev] = true;
  }
  decode_kernel<D, NT, BF><<<(unsigned)(p.units * p.splits), kThreads, smem, s>>>(a);
  if (int rc = d3b_host::check_launch()) return rc;
  if (p.splits > 1) {
    const int64_t rows = (int64_t)B * a.kv_heads * a.group * a.L;
    if (rows > 0x7FFFFFFF) return D3B_EINVAL;
    merge_kernel<D, BF><<<(unsigned)rows, D / 4, 0, s>>>(a, 8 * NT);
    return d3b_host::check_launch();
  }
  return D3B_OK;
}

template <int D, bool BF>
int dispatch(const DecodeArgs& a, const Plan& p, int B, cudaStream_t s) {
  if (p.nt == 1) return launch<D, 1, BF>(a, p, B, s);
  if constexpr (D != 256)
    if (p.nt == 4) return launch<D, 4, BF>(a, p, B, s);
  return launch<D, 2, BF>(a, p, B, s);
}

int check_shape(const d3b_kv4_cache* c, int B, int H, int L, int64_t width) {
  if (!c || B < 0 || H <= 0 || L < 0 || width < 0) return D3B_EINVAL;
  if (!supported(c->kv_heads, c->head_dim, c->page_tokens)) return D3B_EUNSUPPORTED;
  if (H % c->kv_heads) return D3B_EINVAL;
  if ((int64_t)(H / c->kv_heads) * L > 0x7FFFFFFF || width * c->page_tokens > 0x7FFFFF00) return D3B_EINVAL;
  return D3B_OK;
}

}  // namespace

extern "C" {

size_t d3b_kv4_decode_workspace_size(const d3b_kv4_cache* cache, int B, int H, int L, int64_t width) {
  Plan p;
  if (check_shape(cache, B, H, L, width) != D3B_OK || B == 0 || L == 0 || !make_plan(cache, B, H, L, width, &p)) return 0;
  return plan_bytes(p, cache->head_dim);
}

int d3b_kv4_decode(const d3b_kv4_cache* cache, int64_t layer, const void* q, const int64_t* q_strides,
                   const int32_t* table, int64_t table_stride, int64_t width, const int32_t* lengths, int B, int H,
                   int L, int causal, int dtype, float scale, void* out, const int64_t* out_strides, void* workspace,
                   size_t workspace_bytes, d3b_stream_t stream) {
  if (int rc = check_cache(cache, layer)) return rc;
  if (int rc = check_shape(cache, B, H, L, width)) return rc;
  if (dtype != D3B_F16 && dtype != D3B_BF16) return D3B_EUNSUPPORTED;
  if (!(scale > 0.f) || !(scale < INFINITY)) return D3B_EINVAL;
  if (B == 0 || L == 0) return D3B_OK;
  if (!q || !q_strides || !lengths || !out || !out_strides || (width > 0 && !table)) return D3B_EINVAL;
  if (table_stride < 0 || (B > 1 && table_stride < width && table_stride != 0)) return D3B_EINVAL;
  if (reinterpret_cast<uintptr_t>(q) % 16 || reinterpret_cast<uintptr_t>(out) % 16) return D3B_EALIGN;
  if (reinterpret_cast<uintptr_t>(table) % 4 || reinterpret_cast<uintptr_t>(lengths) % 4) return D3B_EALIGN;
  for (int i = 0; i < 3; ++i)
    if (q_strides[i] % 8 || out_strides[i] % 8) return D3B_EALIGN;
  Plan p;
  if (!make_plan(cache, B, H, L, width, &p)) return D3B_EINVAL;
  const size_t need = plan_bytes(p, cache->head_dim);
  if (need > 0 && (!workspace || workspace_bytes < need)) return D3B_ENOSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) % 16) return D3B_EALIGN;
  DecodeArgs a;
  a.pool = layer_base(cache, layer);
  a.page_bytes = page_bytes(cache);
  a.pages = cache->pages;
  a.head_bytes = (int64_t)(cache->page_tokens / kGrain) * granule_bytes(cache->head_dim);
  a.page_shift = log2_of(cache->page_tokens);
  a.q = static_cast<const uint16_t*>(q);
  a.sq_b = q_strides[0], a.sq_h = q_strides[1], a.sq_l = q_strides[2];
  a.out = static_cast<uint16_t*>(out);
  a.so_b = out_strides[0], a.so_h = out_strides[1], a.so_l = out_strides[2];
  a.table = table;
  a.table_stride = table_stride;
  a.width = width;
  a.lengths = lengths;
  a.kv_heads = cache->kv_heads;
  a.group = H / cache->kv_heads;
  a.L = L;
  a.causal = causal != 0;
  a.splits = p.splits;
  a.row_tiles = p.row_tiles;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.part_o = static_cast<float*>(workspace);
  a.part_st = a.part_o + (size_t)p.units * p.splits * 8 * p.nt * cache->head_dim;
  a.err = d3b_host::device_error_word();
  if (!a.err) return D3B_ECUDA;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool bf = dtype == D3B_BF16;
  switch (cache->head_dim) {
    case 64: return bf ? dispatch<64, true>(a, p, B, s) : dispatch<64, false>(a, p, B, s);
    case 128: return bf ? dispatch<128, true>(a, p, B, s) : dispatch<128, false>(a, p, B, s);
    default: return bf ? dispatch<256, true>(a, p, B, s) : dispatch<256, false>(a, p, B, s);
  }
}

}  // extern "C"
