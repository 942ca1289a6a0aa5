// Per-head RMSNorm of queries and keys and a rotary embedding whose frequencies take their
// positions from several axes, in one pass and one launch:
//
//   y = x * rsqrt(sum(x^2) / D + eps) * (1 + w)
//   angle_i = position[axis_i] * inv_freq_i                                    (i < half)
//   out_i = y_i cos - y_{i+half} sin,  out_{i+half} = y_{i+half} cos + y_i sin, the rest y
//
// All of it in fp32 and rounded once. The angle is formed and brought into one turn in fp64:
// position * inv_freq in fp32 is off by half a unit of the product's last place, 0.004 rad at
// position 100 000, and a turn is what sincospi takes.
//
// A warp takes one token and a run of its heads. Cosines and sines of the channels that a lane
// turns, and its channels' weights, stay in registers over the run; the next heads' rows are
// loaded before the present ones are worked on. A head of D values is D/8 lanes x 8 values (one
// 16-byte load and store each): the sum of squares is a shuffle reduction, a rotary partner is
// half/8 lanes away. How many heads a warp takes is the host's choice: few tokens are spread over
// as many warps as there are heads, many tokens share the table's cost.
//
// Bound: bytes, each value read and written once, with instructions close behind (about 90 for
// the 256 values a warp holds, where memory leaves room for 170). Measured (B200): 255 x 47 tokens of 32 + 4
// heads x 128 49 us (4.5 TB/s, 0.69 of a plain copy's rate, issue slots 62 % busy); one token 6 us.
#include "common.cuh"

namespace {

constexpr int kMaxAxes = 8;
constexpr int kMaxHalf = 128;

struct Axes {
  uint8_t of[kMaxHalf];
};

template <bool BF>
__device__ __forceinline__ float2 widen2(uint32_t w) {
  if constexpr (BF) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

template <bool BF>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (BF) {
    const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&r);
  } else {
    const __half2 r = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&r);
  }
}

constexpr int kWarps = 4;

template <int D, bool BF>
__global__ void __launch_bounds__(32 * kWarps) qk_norm_mrope_kernel(
    const uint16_t* __restrict__ q, int64_t sq_r, int64_t sq_t, int64_t sq_h, int q_heads,
    const uint16_t* __restrict__ k, int64_t sk_r, int64_t sk_t, int64_t sk_h, int k_heads,
    const uint16_t* __restrict__ wq, const uint16_t* __restrict__ wk, const int64_t* __restrict__ pos, int64_t sp_a,
    int64_t sp_r, int64_t sp_t, const float* __restrict__ inv_freq, const __grid_constant__ Axes axis, int half,
    uint16_t* __restrict__ q_out, uint16_t* __restrict__ k_out, int T, int64_t tokens, int runs, int run, float eps) {
  constexpr int kLanes = D / 8, kHeads = 32 / kLanes;  // heads a warp holds at once
  __shared__ __align__(16) float2 table[kWarps][D / 2];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, sub = lane % kLanes;
  const int64_t item = (int64_t)blockIdx.x * kWarps + warp;
  const int64_t rt = item / runs;
  if (rt >= tokens) return;
  const int first = (int)(item - rt * runs) * run;
  const int64_t r = rt / T, t = rt - r * T;
  // passes: kHeads heads of q each, then of k
  const int q_passes = (q_heads + kHeads - 1) / kHeads, passes = q_passes + (k_heads + kHeads - 1) / kHeads;
  const int last = min(first + run, passes);
  const uint16_t* q_row = q + r * sq_r + t * sq_t;
  const uint16_t* k_row = k + r * sk_r + t * sk_t;
  const int shift = half / 8;  // lanes to the rotary partner
  const bool low = sub < shift, turned = sub < 2 * shift;
  const int partner = lane - sub + (turned ? (low ? sub + shift : sub - shift) : sub);
  float cs[8], sn[8];
  bool ready = false;
  auto make_table = [&] {
    for (int i = lane; i < half; i += 32) {
      const double turns =
          (double)__ldg(pos + axis.of[i] * sp_a + r * sp_r + t * sp_t) * (double)__ldg(inv_freq + i) *
          0.15915494309189533577;  // 1 / (2 pi)
      float s, c;
      sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
      table[warp][i] = make_float2(c, s);
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 x = turned ? table[warp][8 * (low ? sub : sub - shift) + i] : make_float2(1.f, 0.f);
      cs[i] = x.x;
      sn[i] = low ? -x.y : x.y;
    }
    ready = true;
  };
  // passes p0 .. p1 of one tensor's heads
  auto turn = [&](const uint16_t* row, int64_t s_h, uint16_t* out, int heads, const uint16_t* weight, int p0, int p1) {
    if (p0 >= p1) return;
    const int h0 = p0 * kHeads + lane / kLanes;
    int left = (heads - h0 + kHeads - 1) / kHeads;  // this lane's heads from p0 on
    left = min(left, p1 - p0);
    const uint4* src = reinterpret_cast<const uint4*>(row + h0 * s_h) + sub;
    uint4* dst = reinterpret_cast<uint4*>(out + (int64_t)h0 * D) + sub;
    const int64_t step = kHeads * s_h / 8;
    auto fetch = [&](int i) { return i < left ? __ldg(src + i * step) : make_uint4(0, 0, 0, 0); };
    uint4 next = fetch(0), after = fetch(1);
    if (!ready) make_table();  // while the first rows are on their way
    float w1[8];
    const uint4 wraw = __ldg(reinterpret_cast<const uint4*>(weight) + sub);
    const uint32_t wr[4] = {wraw.x, wraw.y, wraw.z, wraw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = widen2<BF>(wr[i]);
      w1[2 * i] = 1.f + f.x;
      w1[2 * i + 1] = 1.f + f.y;
    }
    for (int i = 0; i < p1 - p0; ++i) {
      const uint4 raw = next;
      next = after;
      after = fetch(i + 2);
      const uint32_t xr[4] = {raw.x, raw.y, raw.z, raw.w};
      float y[8], ss = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = widen2<BF>(xr[j]);
        y[2 * j] = f.x;
        y[2 * j + 1] = f.y;
        ss = fmaf(f.x, f.x, ss);
        ss = fmaf(f.y, f.y, ss);
      }
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float rs = rsqrtf(ss * (1.0f / D) + eps);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] *= rs * w1[j];
      if (shift > 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float z = __shfl_sync(0xffffffffu, y[j], partner);
          y[j] = fmaf(y[j], cs[j], z * sn[j]);
        }
      }
      if (i < left)
        dst[i * (kHeads * D / 8)] = make_uint4(pack2<BF>(y[0], y[1]), pack2<BF>(y[2], y[3]), pack2<BF>(y[4], y[5]),
                                               pack2<BF>(y[6], y[7]));
    }
  };
  turn(q_row, sq_h, q_out + rt * q_heads * D, q_heads, wq, min(first, q_passes), min(last, q_passes));
  turn(k_row, sk_h, k_out + rt * k_heads * D, k_heads, wk, max(first - q_passes, 0), last - q_passes);
}

}  // namespace

extern "C" int d3b_qk_norm_mrope(const void* q, const int64_t* q_strides, int q_heads, const void* k,
                                 const int64_t* k_strides, int k_heads, const void* q_weight, const void* k_weight,
                                 const int64_t* positions, const int64_t* pos_strides, const float* inv_freq,
                                 const uint8_t* axis, int axes, int half, void* q_out, void* k_out, int rows, int T,
                                 int head_dim, int dtype, float eps, d3b_stream_t stream) {
  if (rows < 0 || T < 0 || q_heads < 0 || k_heads < 0 || half < 0) return D3B_EINVAL;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return D3B_EUNSUPPORTED;
  if (dtype != D3B_F16 && dtype != D3B_BF16) return D3B_EUNSUPPORTED;
  if (half % 8 || 2 * half > head_dim || q_heads > 65535 || k_heads > 65535) return D3B_EUNSUPPORTED;
  if (half > 0 && (axes < 1 || axes > kMaxAxes)) return D3B_EUNSUPPORTED;
  const int64_t tokens = (int64_t)rows * T;
  if (tokens == 0 || q_heads + k_heads == 0) return D3B_OK;
  if (tokens > 0x7FFFFFFF) return D3B_EINVAL;
  if (half > 0 && (!positions || !pos_strides || !inv_freq || !axis)) return D3B_EINVAL;
  if (q_heads && (!q || !q_strides || !q_weight || !q_out)) return D3B_EINVAL;
  if (k_heads && (!k || !k_strides || !k_weight || !k_out)) return D3B_EINVAL;
  const void* wide[6] = {q, k, q_weight, k_weight, q_out, k_out};
  for (int i = 0; i < 6; ++i)
    if ((i % 2 ? k_heads : q_heads) && reinterpret_cast<uintptr_t>(wide[i]) % 16) return D3B_EALIGN;
  for (int i = 0; i < 3; ++i)
    if ((q_heads && q_strides[i] % 8) || (k_heads && k_strides[i] % 8)) return D3B_EALIGN;
  if (reinterpret_cast<uintptr_t>(positions) % 8 || reinterpret_cast<uintptr_t>(inv_freq) % 4) return D3B_EALIGN;
  Axes ax = {};
  for (int i = 0; i < half; ++i) {
    if (axis[i] >= axes) return D3B_EINVAL;
    ax.of[i] = axis[i];
  }
  const int64_t zero[3] = {0, 0, 0};
  const int64_t *qs = q_heads ? q_strides : zero, *ks = k_heads ? k_strides : zero, *ps = half ? pos_strides : zero;
  // heads at once, passes over a token's heads, and how many of them a warp takes: enough warps for
  // 32 an SM before a warp takes a second pass
  const int at_once = 256 / head_dim;
  const int passes = (q_heads + at_once - 1) / at_once + (k_heads + at_once - 1) / at_once;
  const int64_t warps = 32ll * d3b_host::num_sms(d3b_host::current_device());
  int64_t run = tokens * passes / warps;
  run = run < 1 ? 1 : run > passes ? passes : run;
  const int64_t runs = (passes + run - 1) / run;
  const int64_t ctas = (tokens * runs + kWarps - 1) / kWarps;
  if (ctas > 0x7FFFFFFF) return D3B_EINVAL;
  auto* qp = static_cast<const uint16_t*>(q);
  auto* kp = static_cast<const uint16_t*>(k);
  auto* wq = static_cast<const uint16_t*>(q_weight);
  auto* wk = static_cast<const uint16_t*>(k_weight);
  auto* qo = static_cast<uint16_t*>(q_out);
  auto* ko = static_cast<uint16_t*>(k_out);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool bf = dtype == D3B_BF16;
  auto launch = [&](auto kernel) {
    kernel<<<(unsigned)ctas, 32 * kWarps, 0, s>>>(qp, qs[0], qs[1], qs[2], q_heads, kp, ks[0], ks[1], ks[2], k_heads, wq,
                                                wk, positions, ps[0], ps[1], ps[2], inv_freq, ax, half, qo, ko, T, tokens, (int)runs,
                                                  (int)run, eps);
    return d3b_host::check_launch();
  };
  switch (head_dim) {
    case 64: return bf ? launch(qk_norm_mrope_kernel<64, true>) : launch(qk_norm_mrope_kernel<64, false>);
    case 128: return bf ? launch(qk_norm_mrope_kernel<128, true>) : launch(qk_norm_mrope_kernel<128, false>);
    default: return bf ? launch(qk_norm_mrope_kernel<256, true>) : launch(qk_norm_mrope_kernel<256, false>);
  }
}
