// What the attention kernels over the 4-bit cache share: operand primitives, the queries' layout in
// shared memory, how the work is dealt out, and the merge of partial results. Layout: kv4.cuh.
//
// A kv head's queries (its group's heads x L tokens) are rows. Products are m16n8k16 on fp16 with
// fp32 sums, turned so that keys (then channels) are the 16 and query rows the 8:
//
//   S^T [16 keys x 8 rows]  = K [16 keys x D] . Q^T         A = decoded K codes
//   O^T [D x 8 rows]       += V^T [D x 16 keys] . W^T       A = decoded V codes
//
// Every thread decodes its own operand from the bytes it needs (a K row's quarter is 16 bytes at
// D = 128), so nothing is widened in shared memory. code * scale is exact in fp16 and queries are
// brought under a power of two a row, so S has no rounding but its fp32 sums. With s_j in base 2:
//
//   w_j = 2^(s_j - m),  l = sum_j w_j,  O = sum_j w_j (code * scale * 2^(e_j - E))_j,  out = O 2^E / l
//
// e_j, a V row's power, goes into its scale: code * scale * 2^d is exact in fp16 for d from -14 to 4
// (a multiple of 2^-24, at most 43008). E is one power for all of a unit's rows that a warp (thin) or a CTA
// (wide) sees: kFirst, for rows whose largest value is 2^-10 to 2^7, or, where none of the first rows that are not
// zeros is such a one, kAbove over their largest. A step with powers outside E - 14 .. E + 4 is banded: its V rows go
// through the products once for every band of 19 powers that has rows, each with weights under their own
// maxima, and the fp32 sums go to O under the band's power. So a row keeps its weight whatever the others'
// magnitudes are; what it costs is another pass over the step's codes a band, with sums of its own (64 sequences of
// 16000 tokens, 8 rows x 128, with every 37th V row 2^30 times the others: 446 us instead of 130). Rows at the
// least power (all values under 2^-52; rows of zeros) count as zeros where E is more than 14 above it, as it is
// at first.
//
// m follows the maximum only when it has to: weights lie under 2^kHead where m has moved and may grow to
// 2^kRoom (fp16 holds 2^15) before it moves again; until then nothing is reduced over keys, rescaled or,
// where warps share rows, exchanged. A weight keeps fp16's 11 bits down to 2^-22 of the largest; below, it
// is off by 2^-33 of the largest at most.
// The weights change from accumulator to operand layout by movmatrix.
//
// Work is dealt out evenly whatever the lengths are: all units (sequence, kv head, tile of rows)
// are cut into pieces of keys, laid end to end, and every CTA takes the same number of pieces. A
// unit that lies in one CTA is finished there; the others leave partial results, at most two a
// CTA, which a second kernel adds in order. A CTA that goes from one unit to the next starts its loads anew,
// which takes as long as two or three tiles; with few sequences every unit begins with a CTA where that makes
// no share much longer, else a unit counts as some pieces more than it has.
#pragma once

#include "kv4.cuh"

namespace d3b_kv4 {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr float kHead = 8.f, kRoom = 15.f;
constexpr float kNone = -3e38f;  // m before any key: finite, so that a score of -infinity has no weight then either
// Powers of V rows are kept as their bytes (biased by 127).
constexpr int kLeastPower = kExpMin + 127;  // of rows of zeros
constexpr int kFirst = 119, kAbove = 3;
constexpr int kFar = 64;           // a row that far over E moves it all the same: O stays in fp32's range
constexpr int kMostPower = 40 + 127;  // E's largest, and the power of the partial results
constexpr int kDown = 14, kBand = 19;  // a band: from E - kDown + kBand * k, kBand powers
constexpr int kSiteOwnLength = 2010;  // a question block's length outside [0, L]

struct AttnArgs {
  const uint8_t* pool;
  int64_t page_bytes, head_bytes;
  int pages, page_shift;
  const uint16_t* q;
  int64_t sq_b, sq_h, sq_l;
  uint16_t* out;
  int64_t so_b, so_h, so_l;
  const int32_t* table;
  int64_t table_stride;    // 0: one table for all sequences
  const int32_t* lengths;  // cached tokens of each sequence; NULL: `most` for all
  int most;                // cached tokens a table can hold
  // a block's own keys in 16 bits, or NULL: k, v [B, kv_heads, L, D]
  const uint16_t *k_own, *v_own;
  int64_t sk_b, sk_h, sk_l, sv_b, sv_h, sv_l;
  const int32_t* own_lengths;
  int B, kv_heads, group, L, causal, row_tiles;
  float scale_log2;
  float* part_o;   // [CTAs][2][rows][D]
  float* part_st;  // [CTAs][2][rows][2]: m, l
  int2* ranges;    // [units]: the first and the last CTA that hold a part of the unit
  int* err;
};

int launch_thin(const AttnArgs& a, int D, int nt, bool bf, int ctas, cudaStream_t s);
int launch_wide(const AttnArgs& a, int D, int nt, bool bf, int ctas, cudaStream_t s);
int resident_thin(int D, int nt);  // CTAs an SM holds
int resident_wide(int D, int nt);

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

__device__ __forceinline__ void mma16816_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
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

// a word of four rows' bytes in shared memory, of which the first `keep` stay and the others become `byte`
__device__ __forceinline__ void keep_rows(uint32_t addr, int keep, int byte) {
  const uint32_t mask = keep <= 0 ? 0u : keep >= 4 ? 0xFFFFFFFFu : (1u << (8 * keep)) - 1u;
  uint32_t w[1];
  lds_words<1>(addr, w);
  asm volatile("st.shared.b32 [%0], %1;" ::"r"(addr), "r"((w[0] & mask) | ((uint32_t)byte * 0x01010101u & ~mask)) : "memory");
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

// two bytes of w to halves
__device__ __forceinline__ uint32_t two_bytes(uint32_t w) { return __byte_perm(w, 0, 0x4140); }

// two powers (halves) relative to E - kDown: those of E's band are 0 .. kBand - 1. A negative one borrows from the
// high half and is itself out of range.
__device__ __forceinline__ uint32_t relative(uint32_t two, int E) { return two + (uint32_t)((kDown - E) * 0x10001); }
__device__ __forceinline__ uint32_t max_halves(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ bool in_band(uint32_t rel) {
  constexpr uint32_t kTop = (uint32_t)(kBand - 1) * 0x10001u;
  return max_halves(rel, kTop) == kTop;
}
// fp16 factors 2^(e - E) of two powers of E's band
__device__ __forceinline__ uint32_t band_factors(uint32_t rel) { return (rel << 10) + (uint32_t)(15 - kDown) * 0x04000400u; }
// the factors of two powers in band k; 0 for a row of another one
__device__ __forceinline__ uint32_t band_factors(uint32_t two, int E, int k) {
  const int base = kDown - E - kBand * k;
  const int lo = (int)(two & 0xFFFFu) + base, hi = (int)(two >> 16) + base;
  return (lo >= 0 && lo < kBand ? (uint32_t)(lo + 15 - kDown) << 10 : 0u) |
         (hi >= 0 && hi < kBand ? (uint32_t)(hi + 15 - kDown) << 26 : 0u);
}
__device__ __forceinline__ int band_of(int e, int E) { return (e - E + kDown + kBand * 16) / kBand - 16; }

// What a step's rows span, marked rows and those at the least power apart: the largest power (0: no row), the
// smallest (255), and whether there is one in E's band.
struct Span {
  int most, least, near;
  // two rows' powers, of which the first `live` are of keys
  __device__ __forceinline__ void add(uint32_t two, int live, int E) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int e = (two >> (16 * h)) & 0xFF;
      if (h >= live || e == 255 || e == kLeastPower) continue;
      most = max(most, e);
      least = min(least, e);
      near |= (uint32_t)(e - E + kDown) < (uint32_t)kBand;
    }
  }
  __device__ __forceinline__ void over_warp() {
    most = (int)__reduce_max_sync(0xffffffffu, (uint32_t)most);
    least = (int)__reduce_min_sync(0xffffffffu, (uint32_t)least);
    near = (int)__reduce_or_sync(0xffffffffu, (uint32_t)near);
  }
};

// E after a step; first: no row but those of zeros came before
__device__ __forceinline__ int next_power(int E, const Span& s, bool first) {
  return s.most > 0 && ((first && !s.near) || s.most > E + kFar) ? min(s.most + kAbove, kMostPower) : E;
}

// the power of two that brings a row's largest finite magnitude to [2^14, 2^15), as far as 2^126 goes
__device__ __forceinline__ int row_up(float top) { return min(126, 14 - ((int)(__float_as_uint(top) >> 23) - 127)); }
__device__ __forceinline__ float power_of(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }  // e in [-126, 127]

// a partial result (O, (m, l)) brought to the reference `base` and added
__device__ __forceinline__ void add_part(float4& acc, float& sum, const float4 o, const float2 st, float base) {
  const float f = ex2(st.x - base);
  sum = fmaf(st.y, f, sum);
  acc.x = fmaf(o.x, f, acc.x);
  acc.y = fmaf(o.y, f, acc.y);
  acc.z = fmaf(o.z, f, acc.z);
  acc.w = fmaf(o.w, f, acc.w);
}

// four channels of a finished row, sums under 2^(kMostPower - 127); zeros where there was no key or the token is behind its block's length
template <bool BF>
__device__ __forceinline__ void store_row(const AttnArgs& a, int b, int kvh, int row, int tokens, int d, const float4 acc,
                                          float sum) {
  const int l = row / a.group, h = kvh * a.group + row % a.group;
  uint32_t lo = 0, hi = 0;
  if (sum != 0.f && l < tokens) {
    const float f = __uint_as_float((uint32_t)kMostPower << 23) / sum;
    lo = narrow<BF>(acc.x * f) | ((uint32_t)narrow<BF>(acc.y * f) << 16);
    hi = narrow<BF>(acc.z * f) | ((uint32_t)narrow<BF>(acc.w * f) << 16);
  }
  *reinterpret_cast<uint2*>(a.out + b * a.so_b + h * a.so_h + l * a.so_l + d) = make_uint2(lo, hi);
}

// a sequence's lengths, and its units' pieces
struct Sequence {
  int len, own, tokens;  // cached keys, own keys, tokens of the block that are real
  int cached, pieces;    // pieces of cached keys; of all keys, at least one
  int live;              // row tiles with real tokens; each other tile is one piece that writes zeros
  int step, dead;        // places of a live tile, of all other tiles: their pieces, filled up to `round` or with `start`
  int per_head, total;   // places of a kv head and of the sequence

  __device__ __forceinline__ void lay(const AttnArgs& a, int round, int start) {
    step = pieces + start;
    dead = a.row_tiles - live;
    if (round > 1) {
      step = (int)((uint32_t)(pieces + round - 1) / (uint32_t)round) * round;
      if (dead) dead = (int)((uint32_t)(dead + round - 1) / (uint32_t)round) * round;
    }
    per_head = live * step + dead;
    total = a.kv_heads * per_head;
  }
};

template <int KEYS, int ROWS, int START>
__device__ __forceinline__ Sequence sequence(const AttnArgs& a, int b, bool report) {
  Sequence s;
  s.len = a.most;
  if (a.lengths) {
    s.len = __ldg(a.lengths + b);
    if (s.len < 0 || s.len > a.most) {
      if (report) d3b::record_input_error(a.err, kSiteBadLength);
      s.len = s.len < 0 ? 0 : a.most;
    }
  }
  s.own = 0;
  s.tokens = a.L;
  if (a.own_lengths) {
    s.own = __ldg(a.own_lengths + b);
    if (s.own < 0 || s.own > a.L) {
      if (report) d3b::record_input_error(a.err, kSiteOwnLength);
      s.own = s.own < 0 ? 0 : a.L;
    }
    s.tokens = s.own;
  }
  s.cached = (s.len + KEYS - 1) / KEYS;
  s.pieces = max(1, s.cached + (s.own + KEYS - 1) / KEYS);
  s.live = (s.tokens * a.group + ROWS - 1) / ROWS;
  s.lay(a, 1, START);
  return s;
}

// where a CTA's pieces begin
struct Deal {
  int first, last;  // its places
  int share, round;  // round: 1, or the share where every unit begins with a CTA
  int start;         // else: places a unit has behind its pieces, for the time that starting it takes
  int b, offset;  // the sequence of the first, and how far into it
};

// Sums the sequences' pieces and finds the CTA's share; all threads, `box` in shared memory. STEP: what a share
// grows by so that units can begin with a CTA, twice at most.
template <int KEYS, int ROWS, int STEP, int START>
__device__ __forceinline__ Deal deal(const AttnArgs& a, int at_least, int* box) {
  const int t = threadIdx.x, warp = t / 32, lane = t % 32;
  if (a.B <= 32) {  // a lane a sequence, every warp for itself: no barrier
    Sequence s = {};
    if (lane < a.B) s = sequence<KEYS, ROWS, 0>(a, lane, t < 32 && blockIdx.x == 0);
    Deal d;
    const int places = (int)__reduce_add_sync(0xffffffffu, (uint32_t)s.total);
    d.share = max(at_least, (places + (int)gridDim.x - 1) / (int)gridDim.x);
    d.round = 1;
    d.start = 0;
    // one place each needs nothing; with no more units than CTAs, filled up they have at most twice the places: below 2^31 here
    if (d.share > 1 && places < (1 << 28) && (int64_t)a.B * a.kv_heads * a.row_tiles <= (int64_t)gridDim.x) {
#pragma unroll 1
      for (int i = 0; i < 3 && d.round == 1; ++i) {
        const int share = (d.share + STEP - 1) / STEP * STEP + i * STEP;
        if (lane < a.B) s.lay(a, share, 0);
        if ((int)__reduce_add_sync(0xffffffffu, (uint32_t)s.total / (uint32_t)share) <= (int)gridDim.x) d.round = share;
      }
    }
    if (d.round > 1) {
      d.share = d.round;
    } else if (d.share > 1) {
      d.start = START;
      if (lane < a.B) s.lay(a, 1, START);
      const int more = (int)__reduce_add_sync(0xffffffffu, (uint32_t)s.total);
      d.share = max(at_least, (more + (int)gridDim.x - 1) / (int)gridDim.x);
    }
    const int mine = s.total;
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const int total = __shfl_sync(0xffffffffu, upto, 31);
    d.first = (int)min((int64_t)blockIdx.x * d.share, (int64_t)total);
    d.last = min(d.first + d.share, total);
    d.b = min(__popc(__ballot_sync(0xffffffffu, upto <= d.first)), 31);
    d.offset = d.first - __shfl_sync(0xffffffffu, upto - mine, d.b);
    return d;
  }
  const int per = (a.B + kThreads - 1) / kThreads;
  const int b0 = min(t * per, a.B), b1 = min(b0 + per, a.B);
  int mine = 0;
  for (int b = b0; b < b1; ++b) mine += sequence<KEYS, ROWS, START>(a, b, blockIdx.x == 0).total;
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += x;
  }
  if (lane == 31) box[warp] = upto;
  __syncthreads();
  int before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    before += w < warp ? box[w] : 0;
    total += box[w];
  }
  before += upto - mine;
  Deal d;
  d.share = max(at_least, (total + (int)gridDim.x - 1) / (int)gridDim.x);
  d.round = 1;
  d.start = START;
  d.first = (int)min((int64_t)blockIdx.x * d.share, (int64_t)total);
  d.last = min(d.first + d.share, total);  // shares are far below 2^31 when first is not the total
  if (d.first >= before && d.first < before + mine) {
    int b = b0, at = before;
    for (;; ++b) {
      const int n = sequence<KEYS, ROWS, START>(a, b, false).total;
      if (d.first < at + n) break;
      at += n;
    }
    box[kWarps] = b;
    box[kWarps + 1] = d.first - at;
  }
  __syncthreads();
  d.b = box[kWarps];
  d.offset = box[kWarps + 1];
  return d;
}

// A CTA whose first place lies behind a unit's pieces begins with the next unit. (Only the first can: a unit that
// was worked on is left with all its places.)
template <int KEYS, int ROWS>
__device__ __forceinline__ void past_filling(const AttnArgs& a, Deal& d) {
  if (!d.start || d.first >= d.last) return;
  Sequence s = sequence<KEYS, ROWS, 0>(a, d.b, false);
  s.lay(a, 1, d.start);
  const int in_head = d.offset % s.per_head, place = in_head % s.step;
  if (in_head >= s.live * s.step || place < s.pieces) return;
  const int skip = min(s.step - place, d.last - d.first);
  d.first += skip;
  d.offset += skip;
  if (d.offset == s.total) {
    d.offset = 0;
    ++d.b;
  }
}

// the largest of a row's lanes; x is not negative
template <int LANES>
__device__ __forceinline__ float max_of_lanes(float x) {
  if constexpr (LANES == 32) {
    return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(x)));  // ordered as bits
  } else {
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
    return x;
  }
}

// Queries to shared memory in operand order, as fp16, each row under its own power of two:
// [nt][word][lane] x 16 bytes, lane = 4 * row + quarter. factors[row]: scale * log2(e) * 2^power, what a product is
// multiplied by. The row's largest finite magnitude goes to 2^14 or above; what is 2^-29 of it or less loses bits,
// scores by 2^-40 of the row's largest term. All threads; a barrier has to follow.
template <int D, int NT, bool BF>
__device__ __forceinline__ void load_queries(const AttnArgs& a, int b, int kvh, int row0, int rows, uint4* qs,
                                             float* factors) {
  constexpr int kLanes = D / 8;  // a lane takes 8 channels
  constexpr int kWords = D / 32;
  constexpr int kItems = (8 * NT * kLanes + kThreads - 1) / kThreads;
  uint4 raw[kItems];
#pragma unroll
  for (int x = 0; x < kItems; ++x) {
    const int i = x * kThreads + threadIdx.x, row = i / kLanes, sub = i % kLanes;
    raw[x] = make_uint4(0, 0, 0, 0);
    if (row < 8 * NT && row0 + row < rows) {
      const int l = (row0 + row) / a.group, g = (row0 + row) % a.group;
      raw[x] = __ldg(reinterpret_cast<const uint4*>(a.q + b * a.sq_b + (int64_t)(kvh * a.group + g) * a.sq_h + l * a.sq_l) + sub);
    }
  }
#pragma unroll
  for (int x = 0; x < kItems; ++x) {
    const int i = x * kThreads + threadIdx.x, row = i / kLanes, sub = i % kLanes;
    const uint32_t w[4] = {raw[x].x, raw[x].y, raw[x].z, raw[x].w};
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = widen2<BF>(w[j]);
      top = fabsf(f.x) < INFINITY ? fmaxf(top, fabsf(f.x)) : top;
      top = fabsf(f.y) < INFINITY ? fmaxf(top, fabsf(f.y)) : top;
    }
    const int up = row_up(max_of_lanes<kLanes>(top));
    if (row >= 8 * NT) continue;  // whole warps, or lanes of rows that do not exist
    if (sub == 0) factors[row] = a.scale_log2 * power_of(-up);
    const float by = power_of(up);
    uint32_t h[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = widen2<BF>(w[j]);
      const __half2 v = __floats2half2_rn(f.x * by, f.y * by);
      h[j] = *reinterpret_cast<const uint32_t*>(&v);
    }
    // channels 8 sub ...: which word of which quarter they are (see the K loads)
    const int half = D == 256 ? sub / 16 : 0, in = D == 256 ? sub % 16 : sub;
    const int per = D == 256 ? 4 : kWords;
    const int quarter = in / per, word = half * 4 + in % per;
    qs[((row / 8) * kWords + word) * 32 + (row % 8) * 4 + quarter] = make_uint4(h[0], h[1], h[2], h[3]);
  }
}

// lets `kernel` have `bytes` of dynamic shared memory, once a device (`ready` by device; twice is harmless)
template <typename K>
inline int allow_smem(K kernel, int bytes, bool (&ready)[64]) {
  const int dev = d3b_host::current_device();
  if (bytes <= 48 * 1024 || (dev >= 0 && dev < 64 && ready[dev])) return D3B_OK;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return D3B_ECUDA;
  if (dev >= 0 && dev < 64) ready[dev] = true;
  return D3B_OK;
}

}  // namespace d3b_kv4
