// Attention over the 4-bit cache for up to 32 query rows at a time: several new tokens a sequence, wide
// groups, and question blocks with their own keys beside the cached state.
//
// A CTA's four warps share tiles of 64 keys. Each takes the scores of 16 of them against all rows,
// so every K code is decoded once for 32 rows; the weights go through shared memory in operand
// layout, and each warp then adds a quarter of the channels over all 64 keys, so every V code is
// decoded once too and O is 1/4 of the rows' channels in a warp's registers. Two barriers a tile:
// maxima, weights.
//
// A block's own keys are tiles of the same kind whose operands come from the 16-bit rows: K brought under a
// power of two a row, so that bf16 values fit fp16 without rounding, V as it is.
//
// Bound: products. 32 rows x 64 keys are 2 D m16n8k16, 8 clocks each on one of four tensor pipes; at D = 256 they
// take 1.3 times as long as the cache's bytes, and the chain conversion, product with the scale, matrix
// instruction leaves the pipes idle half the time with two warps a scheduler. Measured (B200): three sequences of
// 98765 tokens, 5 x 6 rows, 4 heads x 256: 155 us with the merge (235 TFLOP/s, 2.2 TB/s of codes); one block of
// 11 tokens x 8 heads over 4096 tokens of 4 x 128 16 us. Tried and slower: 8 warps a CTA (162 us), 3 CTAs an SM (157
// us: spills); no faster: 128 keys a tile with two granules a warp (137 against 136 us then).
#include "kv4_attn.cuh"

namespace d3b_kv4 {
namespace {

constexpr int kKeys = 64;

template <int D, int NT>
struct Wide {
  static constexpr int kHalf = off_v(D);                    // bytes of a granule's K or V part
  static constexpr int kStage = (kHalf + 127) / 128 * 128;  // V rows start on 128-byte lines
  static constexpr int kRows = 8 * NT;
  static constexpr int kResident = 2;
  // pieces that starting a unit costs: 200 ragged sequences up to 800, 30 rows x 256, with 0, 2, 4, 6 and 8 of them
  // 151, 120, 107, 100 and 101 us
  static constexpr int kStart = 6;
  static constexpr int kRing = 2 * 2 * 4 * kStage;  // two tiles' K, then two tiles' V, of four granules
  static constexpr int kQ = kRows * D * 2;
  static constexpr int kW = 4 * NT * 32 * 8;    // weights: [granule][nt][lane] x 8 bytes
  static constexpr int kMax = kWarps * kRows * 4;
  static constexpr int kFactors = kKeys * 2;  // of the V rows: [granule][pair of rows] x 4 bytes
  static constexpr int kSmem = kRing + kQ + kW + kMax + kFactors;
  static constexpr int kScales = off_k_scale(D), kExps = off_k_exp(D);  // within a stage, after the codes
};

__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// What a unit's end needs to know, kept in shared memory while its tiles use the registers.
struct Unit {
  int b, kvh, tile, tokens, own, cached, pieces, piece0, piece1, taken, pos, offset, total;
};

template <int D, int NT, bool BF>
__global__ void __launch_bounds__(kThreads, Wide<D, NT>::kResident) wide_kernel(const __grid_constant__ AttnArgs a) {
  using P = Wide<D, NT>;
  constexpr int kKWords = D / 32, kTiles = D / 64;  // a lane's K words; a warp's 16-channel tiles
  constexpr int kRun = D / 32;                      // channels of V a lane has
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int box[kWarps + 2];
  __shared__ float factors[P::kRows];  // of the query rows' products
  __shared__ Span spans[kWarps];
  __shared__ Unit kept;
  uint4* qs = reinterpret_cast<uint4*>(smem + P::kRing);
  uint2* ws = reinterpret_cast<uint2*>(smem + P::kRing + P::kQ);
  float* maxima = reinterpret_cast<float*>(smem + P::kRing + P::kQ + P::kW);  // [warp][row]
  uint32_t* vfs = reinterpret_cast<uint32_t*>(maxima + kWarps * P::kRows);  // [granule][pair of V rows]: their factors
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, r = lane / 4, c = lane % 4;
  const int rows = a.group * a.L;
  Deal mine = deal<kKeys, P::kRows, 1, P::kStart>(a, 1, box);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the merge may take its place; it waits for our end
  const uint32_t k_ring = d3b::smem_u32(smem), v_ring = k_ring + 2 * 4 * P::kStage;
  const int grain_shift = a.page_shift - 4, in_page = (1 << grain_shift) - 1;
  // a lane copies units lane, lane + 32, ... of 16 bytes of its warp's granule's K or V; where V's go
  constexpr int kUnits = P::kHalf / 16, kCopies = (kUnits + 31) / 32;
  const uint32_t k_to = k_ring + warp * P::kStage + 16 * lane;
  uint32_t v_to[kCopies];
#pragma unroll
  for (int i = 0; i < kCopies; ++i) {
    const int at = 16 * (32 * i + lane);
    v_to[i] = v_ring + warp * P::kStage + (at < 8 * D ? v_swizzle<D>(at) : at);
    asm volatile("" : "+r"(v_to[i]));  // kept, not worked out again at every copy
  }
  const uint32_t k_at = k_ring + warp * P::kStage + r * (D / 2) + c * (D == 256 ? 16 : D / 8);
  const uint32_t ks_at = k_ring + warp * P::kStage + P::kScales + r * (D / 16) + (D == 64 ? c : 2 * c);
  const uint32_t ke_at = k_ring + warp * P::kStage + P::kExps + r, ve_at = v_ring + P::kExps;
  // V: channels warp * D/4 + r * D/32 ...; rows 2c, 2c + 1, 2c + 8, 2c + 9 of every granule
  uint32_t v_at[4];
#pragma unroll
  for (int x = 0; x < 4; ++x)
    v_at[x] = v_ring + v_swizzle<D>((2 * c + (x & 1) + 8 * (x >> 1)) * (D / 2) + warp * (D / 8) + r * (D / 64));
  const uint32_t vs_at = v_ring + P::kScales + ((warp * (D / 4) + r * kRun) / 16) * 16 + 2 * c;

  past_filling<kKeys, P::kRows>(a, mine);
  int pos = mine.first, b = mine.b, offset = mine.offset;
  while (pos < mine.last) {
    Sequence seq = sequence<kKeys, P::kRows, 0>(a, b, false);
    seq.lay(a, mine.round, mine.start);
    const int kvh = offset / seq.per_head;
    const int in_head = offset - kvh * seq.per_head;
    // live tiles have seq.step places each, the others one, the last of them also what fills up
    const int none = in_head - seq.live * seq.step;
    const bool dead = none >= 0;
    const int tile = dead ? seq.live + none : in_head / seq.step;
    const int pieces = dead ? 1 : seq.pieces, piece0 = dead ? 0 : in_head - tile * seq.step;
    const int left = !dead ? seq.step - piece0 : tile + 1 < a.row_tiles ? 1 : seq.dead - none;
    const int taken = min(left, mine.last - pos), piece1 = min(pieces, piece0 + taken);
    const int row0 = tile * P::kRows, len = seq.len, grains = (len + 15) / 16;
    const int last_cached = dead ? piece0 : min(piece1, seq.cached);
    const uint8_t* head_pool = a.pool + kvh * a.head_bytes + 16 * lane;
    const int32_t* table = a.table + b * a.table_stride;
    // page of the warp's granule of a tile; -1 where there is no such granule
    auto look = [&](int p) {
      const int g = 4 * p + warp;
      return p < last_cached && g < grains ? __ldg(table + (g >> grain_shift)) : -1;
    };
    auto in_pool = [&](int id) { return (uint32_t)id < (uint32_t)a.pages; };
    auto source = [&](int p, int id) {
      return head_pool + id * a.page_bytes + ((4 * p + warp) & in_page) * granule_bytes(D);
    };
    // copy the warp's granule of tile p to ring half HALF: K (how many of its tokens are keys), V
    auto load_k = [&](int p, int id, uint32_t half) -> int {
      if (!in_pool(id)) {
        if (lane == 0 && p < last_cached && 4 * p + warp < grains) d3b::record_input_error(a.err, kSiteBadPage);
        return 0;
      }
      const uint8_t* src = source(p, id);
#pragma unroll
      for (int x = 0; x < kCopies; ++x)
        if (32 * x + 31 < kUnits || 32 * x + lane < kUnits) cp16(k_to + half + 512 * x, src + 512 * x);
      return min(16, len - 16 * (4 * p + warp));
    };
    auto load_v = [&](int p, int id, uint32_t half) {
      if (!in_pool(id)) return;
      const uint8_t* src = source(p, id) + off_v(D);
#pragma unroll
      for (int x = 0; x < kCopies; ++x)
        if (32 * x + 31 < kUnits || 32 * x + lane < kUnits) cp16(v_to[x] + half, src + 512 * x);
    };
    constexpr uint32_t kHalfRing = 4 * P::kStage;
    // tokens of the warp's granule that are keys: of this tile, the next and the one after; pages of the latter two
    int live_now = 0, live_next = 0, live_after = 0, id_v = look(piece0), id_k = look(piece0 + 1);
    live_now = load_k(piece0, id_v, 0);
    cp_commit();
    load_v(piece0, id_v, 0);
    live_next = load_k(piece0 + 1, id_k, kHalfRing);
    cp_commit();
    id_v = id_k;
    id_k = look(piece0 + 2);

    if (threadIdx.x == 0)  // a dead tile has no own keys either
      kept = {b, kvh, tile, seq.tokens, seq.own, dead ? 1 : seq.cached, pieces, piece0, piece1, taken, pos, offset, seq.total};
    load_queries<D, NT, BF>(a, b, kvh, row0, rows, qs, factors);
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
        m[n][j] = kNone;
        l[n][j] = 0.f;
        qf[n][j] = factors[row];
        limit[n][j] = a.causal ? len - (a.L - 1 - (row0 + row) / a.group) : len;
      }
    }
    const int first_limit = a.causal ? len - (a.L - 1) : len;

    int E = kFirst, zero_tiles = 0;  // the sums' power, the same in every warp; tiles from the first on without a row that counts
    float s[NT][4], kq[2];  // products of keys r and r + 8 of the warp's granule, and the K rows' powers
    float x[NT][4];         // the weights' exponents
    // masked(n, j): key r + 8 * (j >> 1) is none for row n * 8 + 2 * c + (j & 1)
    auto exponents = [&](bool edge, auto masked) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) x[n][j] = fmaf(s[n][j], kq[j >> 1] * qf[n][j & 1], -m[n][j & 1]);
      if (edge) {  // apart from the sums above, so that it is a branch and not selects in every tile
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (masked(n, j)) x[n][j] = -INFINITY;
      }
      float most = -INFINITY;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) most = fmaxf(most, x[n][j]);
      return most;
    };
    // the warp's maxima for `settle`, behind a barrier
    auto offer = [&](bool edge, auto masked) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float top = -INFINITY;
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (!edge || !masked(n, j + 2 * h)) top = fmaxf(top, fmaf(s[n][j + 2 * h], kq[h] * qf[n][j], -kHead));
          top = max_over_rows(top);
          if (r == 0) maxima[warp * P::kRows + n * 8 + 2 * c + j] = top;
        }
    };
    // m moved to the warps' maxima
    auto settle = [&] {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float2 top = make_float2(m[n][0], m[n][1]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float2 z = *reinterpret_cast<const float2*>(maxima + w * P::kRows + n * 8 + 2 * c);
          top.x = fmaxf(top.x, z.x);
          top.y = fmaxf(top.y, z.y);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float now = j ? top.y : top.x, keep = ex2(m[n][j] - now);
          m[n][j] = now;
          l[n][j] *= keep;
#pragma unroll
          for (int z = 0; z < kTiles; ++z) {
            o[n][z][j] *= keep;
            o[n][z][j + 2] *= keep;
          }
        }
      }
    };
    auto rescale = [&](float by) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int z = 0; z < kTiles; ++z)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[n][z][j] *= by;
    };

    auto scores = [&](uint32_t half) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[n][j] = 0.f;
      uint32_t k0[kKWords], k1[kKWords], s0[kKWords / 2], s1[kKWords / 2];
      lds_words<D == 256 ? 4 : kKWords>(k_at + half, k0);
      lds_words<D == 256 ? 4 : kKWords>(k_at + half + 4 * D, k1);
      if constexpr (D == 256) {
        lds_words<4>(k_at + half + 64, k0 + 4);
        lds_words<4>(k_at + half + 4 * D + 64, k1 + 4);
      }
      if constexpr (D == 64) {
        s0[0] = decode_scales(lds_u8(ks_at + half) * 0x101u);
        s1[0] = decode_scales(lds_u8(ks_at + half + D / 2) * 0x101u);
      } else {
#pragma unroll
        for (int w = 0; w < kKWords / 4; ++w) {
          const uint32_t x0 = decode_scales(lds_u16(ks_at + half + 8 * w));
          const uint32_t x1 = decode_scales(lds_u16(ks_at + half + D / 2 + 8 * w));
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
        uint4 qv[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) qv[n] = qs[(n * kKWords + w) * 32 + lane];
        // products into the same sums stand apart
#pragma unroll
        for (int n = 0; n < NT; ++n) mma16816(s[n], d0[0], d1[0], d0[1], d1[1], qv[n].x, qv[n].y);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma16816(s[n], d0[2], d1[2], d0[3], d1[3], qv[n].z, qv[n].w);
      }
      // a marked row (255) has codes of zero: its score is 0 * infinity here
      kq[0] = __uint_as_float(lds_u8(ke_at + half) << 23);
      kq[1] = __uint_as_float(lds_u8(ke_at + half + 8) << 23);
    };
    if (piece0 < last_cached) {
      cp_wait<1>();
      __syncwarp();
      scores(0);
    }
    for (int p = piece0; p < last_cached; ++p) {
      const uint32_t half = ((p - piece0) & 1) * kHalfRing;
      cp_wait<0>();  // V of this tile and K of the next
      __syncwarp();
      const int key0 = 64 * p + 16 * warp;
      const uint32_t mine = ve_at + warp * P::kStage + half;  // the powers of the warp's own V rows
      if (live_now < 16) {
        // rows that were never written may have scales that are not numbers: their weights are zero,
        // their values have to be finite; their powers are set to E
        for (int i = lane; i < D / 4 + 4; i += 32)
          keep_rows(v_ring + warp * P::kStage + half + P::kScales + 4 * i, live_now - 4 * (i & 3), i < D / 4 ? 0 : E);
        __syncwarp();
      }
      auto masked = [&](int n, int j) {
        const int key = r + 8 * (j >> 1);
        return key >= live_now || key0 + key >= limit[n][j & 1];
      };
      const bool edge = live_now < 16 || key0 + 16 > first_limit;
      // rows 2 (lane % 8) and the one behind it
      const uint32_t rel = relative(two_bytes(lds_u16(mine + 2 * (lane & 7))), E);
      const bool odd = !in_band(rel);
      // Behind this barrier every warp's copies have landed and its work on the other half is done. Before any key m
      // makes every finite score pass kRoom.
      const bool move = __syncthreads_or(exponents(edge, masked) > kRoom || odd);
      if (lane < 8) vfs[8 * warp + lane] = band_factors(rel);
      load_v(p + 1, id_v, kHalfRing - half);
      live_after = load_k(p + 2, id_k, half);
      cp_commit();
      id_v = id_k;
      id_k = look(p + 3);
      // V's rows of granule i under factors of its pairs as operands: use(16-channel tile, a0 .. a3)
      auto values = [&](int i, uint32_t f01, uint32_t f89, auto use) {
        const uint32_t at = half + i * P::kStage;
        const uint32_t sc01 = hmul2(decode_scales(lds_u16(vs_at + at)), f01);
        const uint32_t sc89 = hmul2(decode_scales(lds_u16(vs_at + at + 8)), f89);
        auto add = [&](int t, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
          use(t, hmul2(a0, sc01), hmul2(a1, sc01), hmul2(a2, sc89), hmul2(a3, sc89));
        };
        if constexpr (D == 256) {  // 8 channels a lane: one word of each row
          uint32_t v[4], x0[4], x1[4], y0[4], y1[4];
#pragma unroll
          for (int z = 0; z < 4; ++z) lds_words<1>(v_at[z] + at, v + z);
          decode8(low_nibbles(v[0], v[1] << 4), x0);
          decode8(low_nibbles(v[0] >> 4, v[1]), x1);
          decode8(low_nibbles(v[2], v[3] << 4), y0);
          decode8(low_nibbles(v[2] >> 4, v[3]), y1);
#pragma unroll
          for (int z = 0; z < 4; ++z) add(z, x0[z], x1[z], y0[z], y1[z]);
        } else if constexpr (D == 128) {  // 4 channels: two bytes of each row, two rows a word
          const uint32_t u = lds_u16(v_at[0] + at) | (lds_u16(v_at[2] + at) << 16);
          const uint32_t w = lds_u16(v_at[1] + at) | (lds_u16(v_at[3] + at) << 16);
          uint32_t x0[4], x1[4];
          decode8(low_nibbles(u, w << 4), x0);
          decode8(low_nibbles(u >> 4, w), x1);
          add(0, x0[0], x1[0], x0[2], x1[2]);
          add(1, x0[1], x1[1], x0[3], x1[3]);
        } else {  // 2 channels: one byte of each row
          const uint32_t u = lds_u8(v_at[0] + at) | (lds_u8(v_at[2] + at) << 8);
          const uint32_t w = lds_u8(v_at[1] + at) | (lds_u8(v_at[3] + at) << 8);
          uint32_t x0[4];
          decode8((low_nibbles(u, w << 4) & 0xFFFFu) | (low_nibbles(u >> 4, w) << 16), x0);
          add(0, x0[0], x0[2], x0[1], x0[3]);
        }
      };
      if (move) {
        Span span = {0, 255, 0};
        span.add(two_bytes(lds_u16(mine + 2 * (lane & 7))), live_now - 2 * (lane & 7), E);
        span.over_warp();
        if (lane == 0) spans[warp] = span;
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (lds_u8(mine + r + 8 * h) == 255u) kq[h] = __int_as_float(0x7FC00000);
        offer(edge, masked);
        __syncthreads();
        settle();
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          span.most = max(span.most, spans[w].most);
          span.least = min(span.least, spans[w].least);
          span.near |= spans[w].near;
        }
        const int to = next_power(E, span, zero_tiles == p - piece0);
        zero_tiles += span.most == 0;
        if (to != E) rescale(power_of(E - to));
        E = to;
        const int band0 = min(band_of(span.least, E), 0);
        const int band1 = max(band_of(span.most, E), 0);
        if (lane < 8) vfs[8 * warp + lane] = band_factors(two_bytes(lds_u16(mine + 2 * lane)), E, 0);
        exponents(edge, masked);
        if (band0 != band1) {  // the common products below are those of band 0
#pragma unroll 1
          for (int k = band0; k <= band1; ++k) {
            // weights of the granule's rows in the band under their own largest one, and what brings their sums to O
            bool in[2];
#pragma unroll
            for (int h = 0; h < 2; ++h)
              in[h] = k != 0 && r + 8 * h < live_now && band_of((int)lds_u8(mine + r + 8 * h), E) == k;
            if (!__syncthreads_or(in[0] || in[1])) continue;  // and the weights and factors are free
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              float under[2];
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                float top = -INFINITY;
#pragma unroll
                for (int h = 0; h < 2; ++h)
                  if (in[h]) top = fmaxf(top, x[n][j + 2 * h]);
                under[j] = finite_or_zero(max_over_rows(top));
                if (r == 0) maxima[warp * P::kRows + n * 8 + 2 * c + j] = ex2(under[j] + (float)(kBand * k));
              }
              uint32_t w[2];
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                float w0 = 0.f, w1 = 0.f;
                if (in[h]) {
                  float &x0 = x[n][2 * h], &x1 = x[n][2 * h + 1];
                  l[n][0] += ex2(x0);
                  l[n][1] += ex2(x1);
                  w0 = ex2(x0 - under[0]);
                  w1 = ex2(x1 - under[1]);
                  x0 = x1 = -INFINITY;  // done
                }
                w[h] = transpose8x8(pack_half2(w0, w1));
              }
              ws[(warp * NT + n) * 32 + lane] = make_uint2(w[0], w[1]);
            }
            if (lane < 8) vfs[8 * warp + lane] = band_factors(two_bytes(lds_u16(mine + 2 * lane)), E, k);
            __syncthreads();
#pragma unroll 1
            for (int i = 0; i < 4; ++i)
              values(i, vfs[8 * i + c], vfs[8 * i + 4 + c], [&](int t, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                  const uint2 w = ws[(i * NT + n) * 32 + lane];
                  const float2 to = *reinterpret_cast<const float2*>(maxima + i * P::kRows + n * 8 + 2 * c);
                  float part[4] = {0.f, 0.f, 0.f, 0.f};
                  mma16816(part, a0, a1, a2, a3, w.x, w.y);
#pragma unroll
                  for (int j = 0; j < 4; ++j) o[n][t][j] = fmaf(part[j], j & 1 ? to.y : to.x, o[n][t][j]);
                }
              });
          }
          __syncthreads();  // the weights and factors are free
          if (lane < 8) vfs[8 * warp + lane] = band_factors(two_bytes(lds_u16(mine + 2 * lane)), E, 0);
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = ex2(x[n][j]);
        l[n][0] += w[0] + w[2];
        l[n][1] += w[1] + w[3];
        ws[(warp * NT + n) * 32 + lane] =
            make_uint2(transpose8x8(pack_half2(w[0], w[1])), transpose8x8(pack_half2(w[2], w[3])));
      }
      __syncthreads();
      // the next tile's scores beside this one's values: they have nothing to do with each other, and behind
      // the last tile the former are of whatever lies there and not used
      scores(kHalfRing - half);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint2 wf[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) wf[n] = ws[(i * NT + n) * 32 + lane];
        values(i, vfs[8 * i + c], vfs[8 * i + 4 + c], [&](int t, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16816(o[n][t], a0, a1, a2, a3, wf[n].x, wf[n].y);
        });
      }
      live_now = live_next;
      live_next = live_after;
    }
    cp_wait<0>();

    const volatile Unit& u = kept;  // read where it is needed, not held

    // The block's own keys. V's rows are operands as they are, in the inputs' type, so O goes under the power of the
    // partial results and takes each product's fp32 sums times 2^(127 - kMostPower). In bf16 a weight is the sum of two
    // bf16 numbers, both above zero (an infinity times either is one), under 2^-kSmall so that no product of
    // finite numbers leaves fp32; rows of V below 2^-90 count as zeros.
    constexpr int kSmall = BF ? 20 : 0;
    uint2* ws_low = reinterpret_cast<uint2*>(smem);  // the smaller numbers, where the ring was
    for (int p = max(u.piece0, u.cached); p < u.piece1 && a.k_own; ++p) {
      const int own = u.own, cached = u.cached;
      const int key0 = 64 * (p - cached) + 16 * warp;  // the warp's 16 keys
      if (64 * (p - cached) >= own) break;         // a unit without any key has one empty piece
      const uint16_t* k_base = a.k_own + u.b * a.sk_b + u.kvh * a.sk_h;
      const uint16_t* v_base = a.v_own + u.b * a.sv_b + u.kvh * a.sv_h;
      if (E != kMostPower) {
        rescale(power_of(E - kMostPower));
        E = kMostPower;
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[n][j] = 0.f;
      int up_k[2] = {0, 0};  // of keys r and r + 8
      auto channel = [&](int w) { return D == 256 ? 128 * (w / 4) + 32 * c + 8 * (w % 4) : c * (D / 4) + 8 * w; };
      auto fetch = [&](int i, int w) {
        const int key = key0 + r + 8 * i;
        return key < own ? __ldg(reinterpret_cast<const uint4*>(k_base + key * a.sk_l + channel(w))) : make_uint4(0, 0, 0, 0);
      };
      if constexpr (BF) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float top = 0.f;
#pragma unroll
          for (int w = 0; w < kKWords; ++w) {
            const uint4 k4 = fetch(i, w);
            const uint32_t kw[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 f = widen2<BF>(kw[j]);
              top = fabsf(f.x) < INFINITY ? fmaxf(top, fabsf(f.x)) : top;  // the largest finite one, as for queries
              top = fabsf(f.y) < INFINITY ? fmaxf(top, fabsf(f.y)) : top;
            }
          }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          up_k[i] = row_up(fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2)));
        }
      }
#pragma unroll
      for (int w = 0; w < kKWords; ++w) {
        uint32_t d[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint4 k4 = fetch(i, w);
          const uint32_t kw[4] = {k4.x, k4.y, k4.z, k4.w};
          const float by = power_of(up_k[i]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if constexpr (BF) {
              const float2 f = widen2<BF>(kw[j]);
              d[i][j] = pack_half2(f.x * by, f.y * by);
            } else {
              d[i][j] = kw[j];
            }
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint4 qv = qs[(n * kKWords + w) * 32 + lane];
          mma16816(s[n], d[0][0], d[1][0], d[0][1], d[1][1], qv.x, qv.y);
          mma16816(s[n], d[0][2], d[1][2], d[0][3], d[1][3], qv.z, qv.w);
        }
      }
      kq[0] = power_of(-up_k[0]);
      kq[1] = power_of(-up_k[1]);
      auto masked = [&](int, int j) { return key0 + r + 8 * (j >> 1) >= own; };
      if (__syncthreads_or(exponents(true, masked) > kRoom)) {
        offer(true, masked);
        __syncthreads();
        settle();
        exponents(true, masked);
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = ex2(x[n][j]);
        l[n][0] += w[0] + w[2];
        l[n][1] += w[1] + w[3];
        if constexpr (BF) {
          uint32_t high[4], low[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float small = w[j] * power_of(-kSmall);
            high[j] = __float_as_uint(small * 0.99609375f) >> 16;
            low[j] = narrow<true>(small - __uint_as_float(high[j] << 16));
          }
          const int at = (warp * NT + n) * 32 + lane;
          ws[at] = make_uint2(transpose8x8(high[0] | high[1] << 16), transpose8x8(high[2] | high[3] << 16));
          ws_low[at] = make_uint2(transpose8x8(low[0] | low[1] << 16), transpose8x8(low[2] | low[3] << 16));
        } else {
          ws[(warp * NT + n) * 32 + lane] =
              make_uint2(transpose8x8(pack_half2(w[0], w[1])), transpose8x8(pack_half2(w[2], w[3])));
        }
      }
      __syncthreads();
#pragma unroll 1
      for (int i = 0; i < 4; ++i) {
        uint32_t h[4][kRun / 2];  // channels of keys 2c, 2c + 1, 2c + 8, 2c + 9
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const int key = 64 * (p - cached) + 16 * i + 2 * c + (y & 1) + 8 * (y >> 1);
          const uint32_t* src = reinterpret_cast<const uint32_t*>(v_base + key * a.sv_l + warp * (D / 4) + r * kRun);
#pragma unroll
          for (int j = 0; j < kRun / 2; ++j) h[y][j] = key < own ? __ldg(src + j) : 0u;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint2 w = ws[(i * NT + n) * 32 + lane];
          const uint2 w_low = BF ? ws_low[(i * NT + n) * 32 + lane] : w;
#pragma unroll
          for (int t = 0; t < kTiles; ++t) {
            const uint32_t a0 = __byte_perm(h[0][t], h[1][t], 0x5410), a1 = __byte_perm(h[0][t], h[1][t], 0x7632);
            const uint32_t a2 = __byte_perm(h[2][t], h[3][t], 0x5410), a3 = __byte_perm(h[2][t], h[3][t], 0x7632);
            float part[4] = {0.f, 0.f, 0.f, 0.f};
            if constexpr (BF) {
              mma16816_bf16(part, a0, a1, a2, a3, w.x, w.y);
              mma16816_bf16(part, a0, a1, a2, a3, w_low.x, w_low.y);
            } else {
              mma16816(part, a0, a1, a2, a3, w.x, w.y);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) o[n][t][j] = fmaf(part[j], power_of(kSmall + 127 - kMostPower), o[n][t][j]);
          }
        }
      }
      __syncthreads();  // the weights are free again
    }

    // the rows' sums over the warps; O goes out from where it is
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float sum = l[n][j];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        l[n][j] = sum;
      }
    __syncthreads();  // the last maxima have been read
    if (r == 0) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) maxima[warp * P::kRows + n * 8 + 2 * c + j] = l[n][j];
    }
    __syncthreads();
    const int first_piece = u.piece0, first_row = u.tile * P::kRows;
    const bool whole = first_piece == 0 && u.piece1 == u.pieces;
    const int64_t part = 2 * (int64_t)blockIdx.x + (first_piece == 0);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int row = n * 8 + 2 * c + j;
        if (first_row + row >= rows) continue;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) sum += maxima[w * P::kRows + row];
        const int d = warp * (D / 4) + r * kRun;
        if (whole) {
          const int li = (first_row + row) / a.group, h = u.kvh * a.group + (first_row + row) % a.group;
          const bool real = sum != 0.f && li < u.tokens;
          const float f = real ? power_of(E - 127) / sum : 0.f;
          uint32_t* dst = reinterpret_cast<uint32_t*>(a.out + u.b * a.so_b + h * a.so_h + li * a.so_l + d);
#pragma unroll
          for (int x = 0; x < kTiles; ++x)
            dst[x] = real ? narrow<BF>(o[n][x][j] * f) | ((uint32_t)narrow<BF>(o[n][x][j + 2] * f) << 16) : 0u;
        } else {
          float2* dst = reinterpret_cast<float2*>(a.part_o + (part * P::kRows + row) * D + d);
#pragma unroll
          for (int x = 0; x < kTiles; ++x)
            dst[x] = make_float2(o[n][x][j] * power_of(E - kMostPower), o[n][x][j + 2] * power_of(E - kMostPower));
          if (warp == 0 && r == 0)
            *reinterpret_cast<float2*>(a.part_st + (part * P::kRows + row) * 2) = make_float2(m[n][j], sum);
        }
      }
    if (first_piece == 0 && threadIdx.x == 0)
      a.ranges[((int64_t)u.b * a.kv_heads + u.kvh) * a.row_tiles + u.tile] =
          make_int2(u.pos / mine.share, (u.pos + u.pieces - 1) / mine.share);
    pos = u.pos + u.taken;
    offset = u.offset + u.taken;
    b = u.b;
    if (offset == u.total) {
      offset = 0;
      ++b;
    }
    __syncthreads();  // ring, queries, sums and the unit's data are free again
  }
}

template <int D, int NT, bool BF>
int launch(const AttnArgs& a, int ctas, cudaStream_t s) {
  constexpr int smem = Wide<D, NT>::kSmem;
  static bool ready[64];
  if (int rc = allow_smem(wide_kernel<D, NT, BF>, smem, ready)) return rc;
  wide_kernel<D, NT, BF><<<(unsigned)ctas, kThreads, smem, s>>>(a);
  return d3b_host::check_launch();
}

template <int D>
int pick(const AttnArgs& a, int nt, bool bf, int ctas, cudaStream_t s) {
  if (nt == 2) return bf ? launch<D, 2, true>(a, ctas, s) : launch<D, 2, false>(a, ctas, s);
  return bf ? launch<D, 4, true>(a, ctas, s) : launch<D, 4, false>(a, ctas, s);
}

}  // namespace

int launch_wide(const AttnArgs& a, int D, int nt, bool bf, int ctas, cudaStream_t s) {
  return D == 64 ? pick<64>(a, nt, bf, ctas, s) : D == 128 ? pick<128>(a, nt, bf, ctas, s) : pick<256>(a, nt, bf, ctas, s);
}

int resident_wide(int, int) { return Wide<128, 4>::kResident; }

}  // namespace d3b_kv4
