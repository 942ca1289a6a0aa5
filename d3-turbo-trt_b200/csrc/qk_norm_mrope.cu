// Per-head RMSNorm of queries and keys and a rotary embedding whose frequencies take their
// positions from several axes, in one pass and one launch:
//
//   y = x * rsqrt(sum(x^2) / D + eps) * (1 + w)
//   angle_i = position[axis_i] * inv_freq_i                                    (i < half)
//   out_i = y_i cos - y_{i+half} sin,  out_{i+half} = y_{i+half} cos + y_i sin, the rest y
//
// All of it in fp32 and rounded once. The angle is formed and brought into one turn in fp64:
// position * inv_freq in fp32 is off by half a unit of the product's last place, 0.004 rad at
// position 100 000, and a turn is what sincospi takes. That is `half` products a token, shared by
// all its heads: one CTA holds one token's heads, its first threads make the table in shared
// memory while the others' rows are on their way.
//
// Bound: each value is read and written once, so bytes. A head of D values is D/8 lanes x 8
// values (one 16-byte load and store each); the sum of squares is a shuffle reduction and a
// rotary partner is half/8 lanes away.
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

template <int D, bool BF>
__global__ void __launch_bounds__(1024) qk_norm_mrope_kernel(
    const uint16_t* __restrict__ q, int64_t sq_r, int64_t sq_t, int64_t sq_h, int q_heads,
    const uint16_t* __restrict__ k, int64_t sk_r, int64_t sk_t, int64_t sk_h, int k_heads,
    const uint16_t* __restrict__ wq, const uint16_t* __restrict__ wk, const int64_t* __restrict__ pos, int64_t sp_a,
    int64_t sp_r, int64_t sp_t, const float* __restrict__ inv_freq, const __grid_constant__ Axes axis, int half,
    uint16_t* __restrict__ q_out, uint16_t* __restrict__ k_out, int T, float eps) {
  constexpr int kLanes = D / 8;
  __shared__ __align__(16) float cos_t[kMaxHalf], sin_t[kMaxHalf];
  const int64_t rt = blockIdx.x;
  const int64_t r = rt / T;
  const int t = (int)(rt % T);
  const int sub = threadIdx.x % kLanes;
  const int heads = q_heads + k_heads;
  const int per_pass = blockDim.x / kLanes;
  const int shift = half / 8;  // lanes to the rotary partner
  for (int first = 0; first < heads; first += per_pass) {
    const int h = first + threadIdx.x / kLanes;
    const bool live = h < heads;
    const bool is_k = live && h >= q_heads;
    uint4 raw = make_uint4(0, 0, 0, 0), wraw = raw;
    if (live) {
      const uint16_t* src = is_k ? k + r * sk_r + t * sk_t + (h - q_heads) * sk_h : q + r * sq_r + t * sq_t + h * sq_h;
      raw = __ldg(reinterpret_cast<const uint4*>(src) + sub);
      wraw = __ldg(reinterpret_cast<const uint4*>(is_k ? wk : wq) + sub);
    }
    if (first == 0) {
      for (int i = threadIdx.x; i < half; i += blockDim.x) {
        const double turns = (double)pos[axis.of[i] * sp_a + r * sp_r + t * sp_t] * (double)inv_freq[i] *
                             0.15915494309189533577;  // 1 / (2 pi)
        const float x = (float)(2.0 * (turns - rint(turns)));
        sincospif(x, &sin_t[i], &cos_t[i]);
      }
      __syncthreads();
    }
    const uint32_t xr[4] = {raw.x, raw.y, raw.z, raw.w}, wr[4] = {wraw.x, wraw.y, wraw.z, wraw.w};
    float y[8];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = widen2<BF>(xr[i]);
      y[2 * i] = f.x;
      y[2 * i + 1] = f.y;
      ss = fmaf(f.x, f.x, ss);
      ss = fmaf(f.y, f.y, ss);
    }
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float rs = rsqrtf(ss * (1.0f / D) + eps);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = widen2<BF>(wr[i]);
      y[2 * i] *= rs * (1.f + f.x);
      y[2 * i + 1] *= rs * (1.f + f.y);
    }
    const bool low = sub < shift, turned = sub < 2 * shift;
    const int partner = turned ? (low ? sub + shift : sub - shift) : sub;
    const int lane = (threadIdx.x & 31 & ~(kLanes - 1)) + partner;
    uint32_t o[4];
    float z[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) z[i] = __shfl_sync(0xffffffffu, y[i], lane);
    if (turned) {
      const int at = 8 * (low ? sub : sub - shift);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float s = low ? -sin_t[at + i] : sin_t[at + i];
        y[i] = fmaf(y[i], cos_t[at + i], z[i] * s);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = pack2<BF>(y[2 * i], y[2 * i + 1]);
    if (live) {
      uint16_t* dst = is_k ? k_out + (rt * k_heads + (h - q_heads)) * D : q_out + (rt * q_heads + h) * D;
      reinterpret_cast<uint4*>(dst)[sub] = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
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
  int threads = (q_heads + k_heads) * (head_dim / 8);
  threads = threads > 1024 ? 1024 : (threads + 31) / 32 * 32;
  auto* qp = static_cast<const uint16_t*>(q);
  auto* kp = static_cast<const uint16_t*>(k);
  auto* wq = static_cast<const uint16_t*>(q_weight);
  auto* wk = static_cast<const uint16_t*>(k_weight);
  auto* qo = static_cast<uint16_t*>(q_out);
  auto* ko = static_cast<uint16_t*>(k_out);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool bf = dtype == D3B_BF16;
  auto launch = [&](auto kernel) {
    kernel<<<(unsigned)tokens, threads, 0, s>>>(qp, qs[0], qs[1], qs[2], q_heads, kp, ks[0], ks[1], ks[2], k_heads, wq,
                                                wk, positions, ps[0], ps[1], ps[2], inv_freq, ax, half, qo, ko, T, eps);
    return d3b_host::check_launch();
  };
  switch (head_dim) {
    case 64: return bf ? launch(qk_norm_mrope_kernel<64, true>) : launch(qk_norm_mrope_kernel<64, false>);
    case 128: return bf ? launch(qk_norm_mrope_kernel<128, true>) : launch(qk_norm_mrope_kernel<128, false>);
    default: return bf ? launch(qk_norm_mrope_kernel<256, true>) : launch(qk_norm_mrope_kernel<256, false>);
  }
}
