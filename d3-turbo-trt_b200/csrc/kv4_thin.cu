// Attention over the 4-bit cache for few query rows a kv head (up to 16): decoding.
//
// A warp takes GP granules (32 keys, 16 at D = 256) a step by itself, from its own cp.async ring of
// two steps and without barriers, and keeps all of O for its rows; a unit's warps are merged at the
// end of the CTA's share. One m16n8k16 serves 8 rows, so a group of up to 8 heads costs one product.
//
// Bound: the cache's bytes, 18 D + 32 for 16 tokens and kv head, with the ALU close behind: a code
// pair costs a conversion (64 lanes a clock and SM) and a product with its scale. Measured (B200, 4 kv heads,
// up to 8 rows): 64 sequences of 16000 tokens D = 128 129 us (4.7 TB/s, 0.71 of a plain copy's rate), D = 256
// 225 us (5.3 TB/s, 0.81); D = 64, 2 heads, 48 us (3.1 TB/s: the instructions for a key do not halve with D). At 64
// ragged sequences up to 16384 the loads alone took 91 us, loads and arithmetic together take 104. One token of
// one sequence of 1000 8.3 us at D = 128.
#include "kv4_attn.cuh"

namespace d3b_kv4 {
namespace {

constexpr int kLeast = kWarps;  // pieces a CTA takes at least: one a warp
// Steps in a warp's ring. Three are 1 to 8 % slower: what they hold is not needed with 12 warps an SM and more.
constexpr int kDepth = 2;

template <int D, int NT>
struct Thin {
  static constexpr int GP = D == 256 ? 1 : 2;                          // granules a step
  static constexpr int kKeys = 16 * GP;                                // keys of a piece
  // pieces that starting a unit costs: 64 ragged sequences up to 4000 with 0, 8, 12, 16 and 24 of them 54, 31, 30,
  // 31 and 32 us at D = 128; 68, 58, 52, 47 and 47 at D = 256
  static constexpr int kStart = D == 256 ? 20 : 12;
  static constexpr int kStage = (granule_bytes(D) + 127) / 128 * 128;  // V rows start on 128-byte lines
  static constexpr int kRows = 8 * NT;
  // CTAs an SM. 8 rows x 64 with 4 of them, 64 x 16000 keys, 49 us, with 5 (registers spilled) and 3 51; 16 x 64 with 3
  // 64 us, with 2 70; 16 x 128 with 3 175 against 181, but one sequence of 16000 19 against 17 us. (Measured before V's
  // powers went into the scales; at these choices 48, 64 and 178 us now.)
  static constexpr int kResident = NT == 1 ? (D == 64 ? 4 : 3) : (D == 64 ? 3 : 2);
  static constexpr int kWarpRing = kDepth * GP * kStage;
  static constexpr int kRing = kWarps * kWarpRing;
  static constexpr int kMerge = kWarps * kRows * (D + 2) * 4;
  static constexpr int kQ = kRows * D * 2;
  static constexpr int kSmem = (kRing > kMerge ? kRing : kMerge) + kQ;
  // where a granule's parts sit in a ring stage
  static constexpr int kKc = 0, kVc = 8 * D, kKs = 16 * D, kVs = 17 * D, kKe = 18 * D, kVe = 18 * D + 16;
};

template <int D, int NT, bool BF>
__global__ void __launch_bounds__(kThreads, Thin<D, NT>::kResident) thin_kernel(const __grid_constant__ AttnArgs a) {
  using P = Thin<D, NT>;
  constexpr int kKWords = D / 32, kVWords = D / 64, kTiles = D / 16;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int box[kWarps + 2];
  __shared__ float factors[P::kRows];  // of the query rows' products
  __shared__ int zero_steps[kWarps];   // steps from a warp's first on without a V row that counts
  uint4* qs = reinterpret_cast<uint4*>(smem + (P::kRing > P::kMerge ? P::kRing : P::kMerge));
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, r = lane / 4, c = lane % 4;
  const int rows = a.group * a.L;
  Deal mine = deal<P::kKeys, P::kRows, kWarps, P::kStart>(a, kLeast, box);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the merge may take its place; it waits for our end
  const uint32_t ring = d3b::smem_u32(smem) + warp * P::kWarpRing;
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

  past_filling<P::kKeys, P::kRows>(a, mine);
  int pos = mine.first, b = mine.b, offset = mine.offset;
  while (pos < mine.last) {
    Sequence seq = sequence<P::kKeys, P::kRows, 0>(a, b, false);
    seq.lay(a, mine.round, mine.start);
    const int kvh = offset / seq.per_head, tile = (offset - kvh * seq.per_head) / seq.step;  // every tile is live
    const int piece0 = offset - kvh * seq.per_head - tile * seq.step, taken = min(seq.step - piece0, mine.last - pos);
    const int piece1 = min(seq.pieces, piece0 + taken);
    const int row0 = tile * P::kRows, len = seq.len, grains = (len + 15) / 16;
    // the warp's steps: granules my_first + step * kStride ...
    constexpr int kStride = P::GP * kWarps;
    const int my_first = P::GP * (piece0 + warp), g_end = min(P::GP * piece1, grains);
    const int steps = my_first < g_end ? (g_end - my_first + kStride - 1) / kStride : 0;
    const uint8_t* head_pool = a.pool + kvh * a.head_bytes + 16 * lane;
    const int32_t* table = a.table + b * a.table_stride;
    int ids[P::GP];  // page numbers of the step that is loaded next
    // two granules of a step start at an even one: they lie in one page unless a page is one granule
    auto look = [&](int step) {
      const int g = my_first + step * kStride;
      if (step >= steps) return;
      ids[0] = __ldg(table + (g >> grain_shift));
      if constexpr (P::GP == 2) ids[1] = grain_shift || g + 1 >= g_end ? ids[0] : __ldg(table + g + 1);
    };
    // copies a step to ring slot SLOT; a bit for each granule whose page is not in the pool
    auto load = [&](int step, auto slot) -> uint32_t {
      constexpr int kAt = decltype(slot)::value * P::GP * P::kStage;
      if (step >= steps) return 0;
      const int g = my_first + step * kStride;
      uint32_t bad = 0;
#pragma unroll
      for (int i = 0; i < P::GP; ++i) bad |= (uint32_t)ids[i] < (uint32_t)a.pages ? 0u : 1u << i;
      const uint8_t* src = head_pool + ids[0] * a.page_bytes + (g & in_page) * granule_bytes(D);
      if (!bad && (P::GP == 1 || grain_shift)) {  // behind a sequence's last granule: the page's next, not used
#pragma unroll
        for (int i = 0; i < P::GP; ++i)
#pragma unroll
          for (int x = 0; x < kCopies; ++x)
            if (32 * x + 31 < kUnits || 32 * x + lane < kUnits)
              cp16(place[x] + kAt + i * P::kStage, src + i * granule_bytes(D) + 512 * x);
        return 0;
      }
#pragma unroll 1
      for (int i = 0; i < P::GP; ++i) {
        if ((bad >> i) & 1) {
          if (lane == 0) d3b::record_input_error(a.err, kSiteBadPage);
          continue;
        }
        src = head_pool + (i ? ids[P::GP - 1] : ids[0]) * a.page_bytes + ((g + i) & in_page) * granule_bytes(D);
#pragma unroll
        for (int x = 0; x < kCopies; ++x)
          if (32 * x + 31 < kUnits || 32 * x + lane < kUnits) cp16(place[x] + kAt + i * P::kStage, src + 512 * x);
      }
      return bad;
    };
    uint32_t bad_now = 0, bad_next = 0;
    look(0);
    bad_now = load(0, Int<0>{});
    cp_commit();
    look(1);

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
    constexpr bool kHold = NT * D <= 128;  // queries stay in registers
    uint4 qr[kHold ? NT : 1][kHold ? kKWords : 1];
    if constexpr (kHold) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int w = 0; w < kKWords; ++w) qr[n][w] = qs[(n * kKWords + w) * 32 + lane];
    }
    const int first_limit = a.causal ? len - (a.L - 1) : len;
    int E = kFirst;  // the sums' power
    if (lane == 0) zero_steps[warp] = 0;
    __syncwarp();
    const uint32_t k_at = ring + P::kKc + r * (D / 2) + c * (D == 256 ? 16 : D / 8);
    const uint32_t ks_at = ring + P::kKs + r * (D / 16) + (D == 64 ? c : 2 * c);
    const uint32_t e_at = ring + P::kKe + r, ve_at = ring + P::kVe + 2 * c;
    const uint32_t vs_at = ring + P::kVs + (D == 64 ? r / 2 : D == 128 ? r : 2 * r) * 16 + 2 * c;
    uint32_t v_at[4];  // V rows 2c, 2c + 1, 2c + 8, 2c + 9
#pragma unroll
    for (int x = 0; x < 4; ++x)
      v_at[x] = ring + P::kVc + v_swizzle<D>((2 * c + (x & 1) + 8 * (x >> 1)) * (D / 2) + r * (D / 16));

    auto step = [&](int now, auto slot) {
      constexpr int kSlot = decltype(slot)::value, kAt = kSlot * P::GP * P::kStage;
      __syncwarp();  // every lane is done with the slot that is loaded next
      bad_next = load(now + 1, Int<1 - kSlot>{});
      cp_commit();
      look(now + 2);
      cp_wait<kDepth - 1>();
      __syncwarp();

      const int key0 = 16 * (my_first + now * kStride);
      const bool edge = key0 + P::kKeys > first_limit || bad_now;  // some key is masked for some row
      float s[P::GP][NT][4], kq[P::GP][2];  // of keys r and r + 8: products, K's power
      int live[P::GP];  // tokens of the granule that are keys at all
#pragma unroll
      for (int i = 0; i < P::GP; ++i)
        live[i] = edge ? ((bad_now >> i) & 1 ? 0 : min(16, len - key0 - 16 * i)) : 16;
      if (edge) {
        // V rows that are no keys may never have been written: their scales, which can be NaN, become zero and
        // their powers E
#pragma unroll
        for (int i = 0; i < P::GP; ++i)
          for (int at = lane; at < D / 4 + 4 && live[i] < 16; at += 32)
            keep_rows(ring + kAt + i * P::kStage + (at < D / 4 ? P::kVs + 4 * at : P::kVe + 4 * (at - D / 4)),
                      live[i] - 4 * (at & 3), at < D / 4 ? 0 : E);
        __syncwarp();
      }
#pragma unroll
      for (int i = 0; i < P::GP; ++i) {
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
        kq[i][0] = __uint_as_float(lds_u8(e_at + at) << 23);
        kq[i][1] = __uint_as_float(lds_u8(e_at + at + 8) << 23);
      }

      // powers of V rows 2c, 2c + 1 and 2c + 8, 2c + 9
      auto powers = [&](int i, int h) { return two_bytes(lds_u16(ve_at + kAt + i * P::kStage + 8 * h)); };
      uint32_t vf[P::GP][2], worst = 0;  // their factors
#pragma unroll
      for (int i = 0; i < P::GP; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t rel = relative(powers(i, h), E);
          worst = max_halves(worst, rel);
          vf[i][h] = band_factors(rel);
        }
      const bool odd = !in_band(worst);

      // exponents of the weights, masked keys at -infinity
      float x[P::GP][NT][4];
      auto exponents = [&] {
#pragma unroll
        for (int i = 0; i < P::GP; ++i)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              x[i][n][j] = fmaf(s[i][n][j], kq[i][j >> 1] * qf[n][j & 1], -m[n][j & 1]);
            }
        if (edge) {  // apart from the sums above, so that it is a branch and not selects in every step
#pragma unroll
          for (int i = 0; i < P::GP; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const int key = r + 8 * (j >> 1);
                if (key >= live[i] || key0 + 16 * i + key >= limit[n][j & 1]) x[i][n][j] = -INFINITY;
              }
        }
        float most = -INFINITY;
#pragma unroll
        for (int i = 0; i < P::GP; ++i)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) most = fmaxf(most, x[i][n][j]);
        return most;
      };
      // V's rows under factors `f` as operands: use(granule, 16-channel tile, a0 .. a3)
      auto values = [&](const uint32_t (&f)[P::GP][2], auto use) {
#pragma unroll
        for (int i = 0; i < P::GP; ++i) {
          const int at = kAt + i * P::kStage;
          uint32_t v[4][kVWords];
#pragma unroll
          for (int x = 0; x < 4; ++x) lds_words<kVWords>(v_at[x] + at, v[x]);
          uint32_t sc01 = 0, sc89 = 0;
#pragma unroll
          for (int w = 0; w < kVWords; ++w) {
            if (w == 0 || (D == 256 && w == 2)) {
              sc01 = hmul2(decode_scales(lds_u16(vs_at + at + 8 * w)), f[i][0]);
              sc89 = hmul2(decode_scales(lds_u16(vs_at + at + 8 * w + 8)), f[i][1]);
            }
            uint32_t x0[4], x1[4], y0[4], y1[4];
            decode8(low_nibbles(v[0][w], v[1][w] << 4), x0);
            decode8(low_nibbles(v[0][w] >> 4, v[1][w]), x1);
            decode8(low_nibbles(v[2][w], v[3][w] << 4), y0);
            decode8(low_nibbles(v[2][w] >> 4, v[3][w]), y1);
#pragma unroll
            for (int x = 0; x < 4; ++x)
              use(i, 4 * w + x, hmul2(x0[x], sc01), hmul2(x1[x], sc01), hmul2(y0[x], sc89), hmul2(y1[x], sc89));
          }
        }
      };
      uint32_t wf[P::GP][NT][2];
      // before any key m makes every finite score pass kRoom
      if (__any_sync(0xffffffffu, exponents() > kRoom || odd)) {
        int band0 = 0, band1 = 0;  // the step's bands; the common products below are those of band 0
        if (__any_sync(0xffffffffu, odd)) {
          Span span = {0, 255, 0};
#pragma unroll
          for (int i = 0; i < P::GP; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (lds_u8(e_at + kAt + i * P::kStage + P::kVe - P::kKe + 8 * h) == 255u) kq[i][h] = __int_as_float(0x7FC00000);
              span.add(powers(i, h), live[i] - 2 * c - 8 * h, E);
            }
          span.over_warp();
          const int zeros = zero_steps[warp], to = next_power(E, span, zeros == now);
          __syncwarp();
          if (lane == 0 && span.most == 0) zero_steps[warp] = zeros + 1;
          __syncwarp();
          if (to != E) {
            const float by = power_of(E - to);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int z = 0; z < kTiles; ++z)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[n][z][j] *= by;
          }
          // what is no key has the old E: a row of zeros
#pragma unroll
          for (int i = 0; i < P::GP; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) vf[i][h] = band_factors(powers(i, h), to, 0);
          E = to;
          band0 = min(band_of(span.least, E), 0);
          band1 = max(band_of(span.most, E), 0);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float old = m[n][j];
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < P::GP; ++i)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int key = r + 8 * h;
                const bool in = !edge || (key < live[i] && key0 + 16 * i + key < limit[n][j]);
                if (in) top = fmaxf(top, fmaf(s[i][n][j + 2 * h], kq[i][h] * qf[n][j], -kHead));
              }
            const float now = fmaxf(old, max_over_rows(top));
            const float keep = ex2(old - now);
            m[n][j] = now;
            l[n][j] *= keep;
#pragma unroll
            for (int z = 0; z < kTiles; ++z) {
              o[n][z][j] *= keep;
              o[n][z][j + 2] *= keep;
            }
          }
        exponents();
        if (band0 != band1) {
#pragma unroll 1
          for (int k = band0; k <= band1; ++k) {
            uint32_t any = 0;
#pragma unroll
            for (int i = 0; i < P::GP; ++i)
#pragma unroll
              for (int h = 0; h < 2; ++h) any |= vf[i][h] = band_factors(powers(i, h), E, k);
            if (k == 0 || !__any_sync(0xffffffffu, any)) continue;
            // the weights of the band's rows under their own largest one, and what brings a sum of theirs to O
            bool mine[P::GP][2];
#pragma unroll
            for (int i = 0; i < P::GP; ++i)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int e = (int)lds_u8(e_at + kAt + i * P::kStage + P::kVe - P::kKe + 8 * h);
                mine[i][h] = r + 8 * h < live[i] && band_of(e, E) == k;
              }
            float to[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              float under[2];
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                float top = -INFINITY;
#pragma unroll
                for (int i = 0; i < P::GP; ++i)
#pragma unroll
                  for (int h = 0; h < 2; ++h)
                    if (mine[i][h]) top = fmaxf(top, x[i][n][j + 2 * h]);
                under[j] = finite_or_zero(max_over_rows(top));
                to[n][j] = ex2(under[j] + (float)(kBand * k));
              }
#pragma unroll
              for (int i = 0; i < P::GP; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  float w0 = 0.f, w1 = 0.f;
                  if (mine[i][h]) {
                    float &x0 = x[i][n][2 * h], &x1 = x[i][n][2 * h + 1];
                    l[n][0] += ex2(x0);
                    l[n][1] += ex2(x1);
                    w0 = ex2(x0 - under[0]);
                    w1 = ex2(x1 - under[1]);
                    x0 = x1 = -INFINITY;  // done
                  }
                  const __half2 w = __floats2half2_rn(w0, w1);
                  wf[i][n][h] = transpose8x8(*reinterpret_cast<const uint32_t*>(&w));
                }
            }
            values(vf, [&](int i, int tile, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                float part[4] = {0.f, 0.f, 0.f, 0.f};
                mma16816(part, a0, a1, a2, a3, wf[i][n][0], wf[i][n][1]);
#pragma unroll
                for (int j = 0; j < 4; ++j) o[n][tile][j] = fmaf(part[j], to[n][j & 1], o[n][tile][j]);
              }
            });
          }
#pragma unroll
          for (int i = 0; i < P::GP; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) vf[i][h] = band_factors(powers(i, h), E, 0);
        }
      }
#pragma unroll
      for (int i = 0; i < P::GP; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j] = ex2(x[i][n][j]);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            l[n][j] += w[j] + w[j + 2];
            const __half2 h = __floats2half2_rn(w[2 * j], w[2 * j + 1]);
            wf[i][n][j] = transpose8x8(*reinterpret_cast<const uint32_t*>(&h));
          }
        }
      values(vf, [&](int i, int tile, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
#pragma unroll
        for (int n = 0; n < NT; ++n) mma16816(o[n][tile], a0, a1, a2, a3, wf[i][n][0], wf[i][n][1]);
      });
      bad_now = bad_next;
    };
    for (int now = 0; now < steps; now += kDepth) {
      step(now, Int<0>{});
      if (now + 1 < steps) step(now + 1, Int<1>{});
    }
    cp_wait<0>();

    // merge the warps: O and (m, l) through shared memory, where the rings were
    __syncthreads();
    float* mo = reinterpret_cast<float*>(smem);   // [warp][row][D]
    float* ms = mo + kWarps * P::kRows * D;       // [warp][row][2]
    const float to_part = power_of(E - kMostPower);
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
          *reinterpret_cast<float4*>(dst + 2 * x) =
              make_float4(o[n][x][j] * to_part, o[n][x][j + 2] * to_part, o[n][x + 1][j] * to_part,
                          o[n][x + 1][j + 2] * to_part);
      }
    __syncthreads();
    const bool whole = piece0 == 0 && piece1 == seq.pieces;
    const int64_t part = 2 * (int64_t)blockIdx.x + (piece0 == 0);
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
      if (whole) {
        store_row<BF>(a, b, kvh, row0 + row, seq.tokens, d, acc, sum);
      } else {
        *reinterpret_cast<float4*>(a.part_o + (part * P::kRows + row) * D + d) = acc;
        if (d == 0) *reinterpret_cast<float2*>(a.part_st + (part * P::kRows + row) * 2) = make_float2(top, sum);
      }
    }
    if (piece0 == 0 && threadIdx.x == 0)
      a.ranges[((int64_t)b * a.kv_heads + kvh) * a.row_tiles + tile] =
          make_int2(pos / mine.share, (pos + seq.pieces - 1) / mine.share);
    __syncthreads();  // the rings and the queries are free again
    pos += taken;
    offset += taken;
    if (offset == seq.total) {
      offset = 0;
      ++b;
    }
  }
}

template <int D, int NT, bool BF>
int launch(const AttnArgs& a, int ctas, cudaStream_t s) {
  constexpr int smem = Thin<D, NT>::kSmem;
  static bool ready[64];
  if (int rc = allow_smem(thin_kernel<D, NT, BF>, smem, ready)) return rc;
  thin_kernel<D, NT, BF><<<(unsigned)ctas, kThreads, smem, s>>>(a);
  return d3b_host::check_launch();
}

template <int D>
int pick(const AttnArgs& a, int nt, bool bf, int ctas, cudaStream_t s) {
  if (nt == 1) return bf ? launch<D, 1, true>(a, ctas, s) : launch<D, 1, false>(a, ctas, s);
  if constexpr (D < 256) return bf ? launch<D, 2, true>(a, ctas, s) : launch<D, 2, false>(a, ctas, s);
  return D3B_EUNSUPPORTED;
}

}  // namespace

int launch_thin(const AttnArgs& a, int D, int nt, bool bf, int ctas, cudaStream_t s) {
  return D == 64 ? pick<64>(a, nt, bf, ctas, s) : D == 128 ? pick<128>(a, nt, bf, ctas, s) : pick<256>(a, nt, bf, ctas, s);
}

int resident_thin(int D, int nt) {
  if (nt == 2) return D == 64 ? Thin<64, 2>::kResident : Thin<128, 2>::kResident;
  return D == 64 ? Thin<64, 1>::kResident : D == 128 ? Thin<128, 1>::kResident : Thin<256, 1>::kResident;
}

}  // namespace d3b_kv4
