// Entry points of the attention over the 4-bit cache, the choice of its kernels, and the merge of
// units that more than one CTA worked on.
#include "kv4_attn.cuh"

namespace {

using namespace d3b_kv4;

// One CTA a query row: the parts of its unit, added in a fixed order by groups of D/4 threads, every
// kGroups-th part a group, then the groups in turn. Bound: latency. Behind the attention kernel stand one
// load of the unit's range, one of its parts and their factors side by side, and one barrier: with up to 32
// parts every warp works out all factors by itself. THREADS is 64 where a unit has few parts (64 sequences
// of 16384 tokens: 2048 rows of 4 parts) and 256 where it has many. Launched before the attention kernel has
// finished; it waits for it here.
template <int D, int THREADS, bool BF>
__global__ void __launch_bounds__(THREADS) merge_kernel(const __grid_constant__ AttnArgs a, int tile_rows) {
  constexpr int kGroups = THREADS / (D / 4);
  constexpr int kAhead = 32 / kGroups < 8 ? 32 / kGroups : 8;  // parts a thread loads at once
  __shared__ float4 part[kGroups][D / 4];
  __shared__ float factor[THREADS], tops[THREADS / 32], sums[THREADS / 32];
  const int rows = a.group * a.L;
  const int row = blockIdx.x % rows, bk = blockIdx.x / rows;
  const int kvh = bk % a.kv_heads, b = bk / a.kv_heads;
  const int t = threadIdx.x, d4 = t % (D / 4), group = t / (D / 4);
  int tokens = a.L;
  if (a.own_lengths) tokens = min(max(__ldg(a.own_lengths + b), 0), a.L);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int2 range = a.ranges[(int64_t)bk * a.row_tiles + row / tile_rows];
  if (range.x == range.y) return;  // finished where it was computed
  // the unit's first CTA began it (slot 1), the others went on with it (slot 0)
  auto at = [&](int cta) { return (2 * (int64_t)cta + (cta == range.x)) * tile_rows + row % tile_rows; };
  auto load_st = [&](int cta) { return *reinterpret_cast<const float2*>(a.part_st + at(cta) * 2); };
  auto load_o = [&](int cta) { return *reinterpret_cast<const float4*>(a.part_o + at(cta) * D + 4 * d4); };
  float sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](const float4& x, float f) {
    acc.x = fmaf(x.x, f, acc.x);
    acc.y = fmaf(x.y, f, acc.y);
    acc.z = fmaf(x.z, f, acc.z);
    acc.w = fmaf(x.w, f, acc.w);
  };
  const int count = range.y + 1 - range.x, lane = t % 32;
  if (count <= 32) {
    const float2 st = lane < count ? load_st(range.x + lane) : make_float2(-INFINITY, 0.f);
    float4 x[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      x[i] = group + i * kGroups < count ? load_o(range.x + group + i * kGroups) : make_float4(0.f, 0.f, 0.f, 0.f);
    float top = st.x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float f = lane < count ? ex2(st.x - finite_or_zero(top)) : 0.f;
    sum = st.y * f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) add(x[i], __shfl_sync(0xffffffffu, f, (group + i * kGroups) & 31));
    for (int i = kAhead; i * kGroups < count; ++i) {  // the same number of times in every lane
      const int p = group + i * kGroups;
      const float g = __shfl_sync(0xffffffffu, f, p & 31);
      if (p < count) add(load_o(range.x + p), g);
    }
  } else {
    float top = -INFINITY;
    for (int c = range.x + t; c <= range.y; c += THREADS) top = fmaxf(top, a.part_st[at(c) * 2]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) tops[t / 32] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) top = fmaxf(top, tops[w]);
    const float base = finite_or_zero(top);
    for (int c0 = range.x; c0 <= range.y; c0 += THREADS) {
      const int n = min(THREADS, range.y + 1 - c0);
      __syncthreads();
      if (t < n) {
        const float2 st = load_st(c0 + t);
        const float f = ex2(st.x - base);
        factor[t] = f;
        sum = fmaf(st.y, f, sum);
      }
      __syncthreads();
#pragma unroll 8
      for (int i = group; i < n; i += kGroups) add(load_o(c0 + i), factor[i]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) sums[t / 32] = sum;
  }
  if constexpr (kGroups > 1) part[group][d4] = acc;
  if (kGroups > 1 || count > 32) __syncthreads();
  if (group) return;
  if (count > 32) {
    sum = 0.f;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) sum += sums[w];
  }
#pragma unroll
  for (int g = 1; g < kGroups; ++g) {
    const float4 x = part[g][d4];
    acc.x += x.x;
    acc.y += x.y;
    acc.z += x.z;
    acc.w += x.w;
  }
  store_row<BF>(a, b, kvh, row, tokens, 4 * d4, acc, sum);
}

struct Plan {
  bool wide;
  int nt, row_tiles, ctas;
  int64_t units;
};

// Up to 8 rows a kv head (16 where O for 16 rows still fits a warp's registers) go to the thin kernel,
// whose warps work alone; more rows to the wide one, which decodes each code once for up to 32 rows.
// 64 sequences of 16000 tokens, 4 heads: 8 rows x 256 225 us thin and 354 wide, 8 x 128 129 and 240, 16 x 128 178
// and 242; below 16 sequences of 4000 the two are within 2 us of each other.
bool make_plan(const d3b_kv4_cache* c, int B, int H, int L, int64_t keys, bool own, Plan* p) {
  const int D = c->head_dim;
  const int64_t rows = (int64_t)(H / c->kv_heads) * L;
  p->wide = own || rows > (D == 256 ? 8 : 16);
  p->nt = rows <= 8 && !p->wide ? 1 : rows <= 16 ? 2 : 4;
  const int64_t tiles = (rows + 8 * p->nt - 1) / (8 * p->nt);
  p->units = (int64_t)B * c->kv_heads * tiles;
  const int64_t piece = p->wide ? 64 : D == 256 ? 16 : 32, least = p->wide ? 1 : 4;
  // own keys add at most L / 64 pieces, which `keys` holds
  const int64_t most = p->units * (keys / piece + 3);
  if (p->units > (1 << 28) || most + 20 * p->units > (1 << 30)) return false;  // a unit counts as up to 20 pieces more
  p->row_tiles = (int)tiles;
  int64_t ctas = (int64_t)d3b_host::num_sms(d3b_host::current_device()) *
                 (p->wide ? resident_wide(D, p->nt) : resident_thin(D, p->nt));
  if (ctas > (most + least - 1) / least) ctas = (most + least - 1) / least;
  p->ctas = (int)ctas;
  return true;
}

size_t plan_bytes(const Plan& p, int D) {
  return (size_t)p.ctas * 2 * 8 * p.nt * (D + 2) * 4 + (size_t)p.units * 8;
}

template <int D, int THREADS>
int launch_merge(const AttnArgs& a, int nt, bool bf, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((int64_t)a.B * a.kv_heads * a.group * a.L));
  cfg.blockDim = dim3(THREADS);
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = bf ? cudaLaunchKernelEx(&cfg, merge_kernel<D, THREADS, true>, a, 8 * nt)
                           : cudaLaunchKernelEx(&cfg, merge_kernel<D, THREADS, false>, a, 8 * nt);
  return e == cudaSuccess ? d3b_host::check_launch() : D3B_ECUDA;
}

template <int D>
int launch_merge(const AttnArgs& a, const Plan& p, bool bf, cudaStream_t s) {
  return p.ctas <= 6 * p.units ? launch_merge<D, 64>(a, p.nt, bf, s) : launch_merge<D, 256>(a, p.nt, bf, s);
}

int run(AttnArgs& a, const d3b_kv4_cache* c, const Plan& p, bool bf, void* workspace, cudaStream_t s) {
  const int D = c->head_dim;
  a.err = d3b_host::device_error_word();
  if (!a.err) return D3B_ECUDA;
  a.row_tiles = p.row_tiles;
  a.part_o = static_cast<float*>(workspace);
  a.part_st = a.part_o + (size_t)p.ctas * 2 * 8 * p.nt * D;
  a.ranges = reinterpret_cast<int2*>(a.part_st + (size_t)p.ctas * 2 * 8 * p.nt * 2);
  if (int rc = p.wide ? launch_wide(a, D, p.nt, bf, p.ctas, s) : launch_thin(a, D, p.nt, bf, p.ctas, s)) return rc;
  if (p.ctas == 1) return D3B_OK;  // nothing to merge
  return D == 64 ? launch_merge<64>(a, p, bf, s) : D == 128 ? launch_merge<128>(a, p, bf, s)
                                                                   : launch_merge<256>(a, p, bf, s);
}

int check_shape(const d3b_kv4_cache* c, int B, int H, int L, int64_t width) {
  if (!c || B < 0 || H <= 0 || L < 0 || width < 0) return D3B_EINVAL;
  if (!supported(c->kv_heads, c->head_dim, c->page_tokens)) return D3B_EUNSUPPORTED;
  if (H % c->kv_heads) return D3B_EINVAL;
  if ((int64_t)(H / c->kv_heads) * L > (1 << 28) || (int64_t)B * H * L > 0x7FFFFFFF) return D3B_EINVAL;
  if (width > (1 << 30) / c->page_tokens) return D3B_EINVAL;
  return D3B_OK;
}

// what both entry points check; D3B_OK with a->q == nullptr: nothing to do
int prepare(const d3b_kv4_cache* cache, int64_t layer, const void* q, const int64_t* q_strides, const int32_t* table,
            int64_t table_stride, int64_t width, int B, int H, int L, int dtype, float scale, void* out,
            const int64_t* out_strides, AttnArgs* a) {
  if (int rc = check_cache(cache, layer)) return rc;
  if (int rc = check_shape(cache, B, H, L, width)) return rc;
  if (dtype != D3B_F16 && dtype != D3B_BF16) return D3B_EUNSUPPORTED;
  if (!(scale > 0.f) || !(scale < INFINITY)) return D3B_EINVAL;
  *a = {};
  if (B == 0 || L == 0) return D3B_OK;
  if (!q || !q_strides || !out || !out_strides || (width > 0 && !table)) return D3B_EINVAL;
  if (reinterpret_cast<uintptr_t>(q) % 16 || reinterpret_cast<uintptr_t>(out) % 16) return D3B_EALIGN;
  if (reinterpret_cast<uintptr_t>(table) % 4) return D3B_EALIGN;
  for (int i = 0; i < 3; ++i)
    if (q_strides[i] % 8 || out_strides[i] % 8) return D3B_EALIGN;
  a->pool = layer_base(cache, layer);
  a->page_bytes = page_bytes(cache);
  a->pages = (int)cache->pages;
  a->head_bytes = (int64_t)(cache->page_tokens / kGrain) * granule_bytes(cache->head_dim);
  a->page_shift = log2_of(cache->page_tokens);
  a->q = static_cast<const uint16_t*>(q);
  a->sq_b = q_strides[0], a->sq_h = q_strides[1], a->sq_l = q_strides[2];
  a->out = static_cast<uint16_t*>(out);
  a->so_b = out_strides[0], a->so_h = out_strides[1], a->so_l = out_strides[2];
  a->table = table;
  a->table_stride = table_stride;
  a->most = (int)(width * cache->page_tokens);
  a->B = B;
  a->kv_heads = cache->kv_heads;
  a->group = H / cache->kv_heads;
  a->L = L;
  a->scale_log2 = scale * 1.4426950408889634f;
  return D3B_OK;
}

int check_workspace(const void* workspace, size_t have, size_t need) {
  if (!workspace || have < need) return D3B_ENOSPACE;
  return reinterpret_cast<uintptr_t>(workspace) % 16 ? D3B_EALIGN : D3B_OK;
}

}  // namespace

extern "C" {

size_t d3b_kv4_decode_workspace_size(const d3b_kv4_cache* cache, int B, int H, int L, int64_t width) {
  Plan p;
  if (check_shape(cache, B, H, L, width) != D3B_OK || B == 0 || L == 0) return 0;
  if (!make_plan(cache, B, H, L, width * cache->page_tokens, false, &p)) return 0;
  return plan_bytes(p, cache->head_dim);
}

int d3b_kv4_decode(const d3b_kv4_cache* cache, int64_t layer, const void* q, const int64_t* q_strides,
                   const int32_t* table, int64_t table_stride, int64_t width, const int32_t* lengths, int B, int H,
                   int L, int causal, int dtype, float scale, void* out, const int64_t* out_strides, void* workspace,
                   size_t workspace_bytes, d3b_stream_t stream) {
  AttnArgs a;
  if (int rc = prepare(cache, layer, q, q_strides, table, table_stride, width, B, H, L, dtype, scale, out, out_strides, &a))
    return rc;
  if (!a.q) return D3B_OK;
  if (!lengths || table_stride < 0 || (B > 1 && table_stride < width && table_stride != 0)) return D3B_EINVAL;
  if (reinterpret_cast<uintptr_t>(lengths) % 4) return D3B_EALIGN;
  a.lengths = lengths;
  a.causal = causal != 0;
  Plan p;
  if (!make_plan(cache, B, H, L, a.most, false, &p)) return D3B_EINVAL;
  if (int rc = check_workspace(workspace, workspace_bytes, plan_bytes(p, cache->head_dim))) return rc;
  return run(a, cache, p, dtype == D3B_BF16, workspace, reinterpret_cast<cudaStream_t>(stream));
}

size_t d3b_kv4_question_workspace_size(const d3b_kv4_cache* cache, int B, int H, int L, int64_t state_len) {
  Plan p;
  if (state_len < 0 || state_len > (1 << 30) || check_shape(cache, B, H, L, 0) != D3B_OK || B == 0 || L == 0) return 0;
  if (!make_plan(cache, B, H, L, state_len + L, true, &p)) return 0;
  return plan_bytes(p, cache->head_dim);
}

int d3b_kv4_question(const d3b_kv4_cache* cache, int64_t layer, const void* q, const int64_t* q_strides,
                     const int32_t* table, int64_t width, int64_t state_len, const void* k_q, const int64_t* k_strides,
                     const void* v_q, const int64_t* v_strides, const int32_t* lengths, int B, int H, int L, int dtype,
                     float scale, void* out, const int64_t* out_strides, void* workspace, size_t workspace_bytes,
                     d3b_stream_t stream) {
  AttnArgs a;
  if (int rc = prepare(cache, layer, q, q_strides, table, 0, width, B, H, L, dtype, scale, out, out_strides, &a)) return rc;
  if (!a.q) return D3B_OK;
  if (state_len < 0 || state_len > a.most) return D3B_EINVAL;
  if (!k_q || !v_q || !k_strides || !v_strides || !lengths) return D3B_EINVAL;
  if (reinterpret_cast<uintptr_t>(k_q) % 16 || reinterpret_cast<uintptr_t>(v_q) % 16) return D3B_EALIGN;
  if (reinterpret_cast<uintptr_t>(lengths) % 4) return D3B_EALIGN;
  for (int i = 0; i < 3; ++i)
    if (k_strides[i] % 8 || v_strides[i] % 8) return D3B_EALIGN;
  a.most = (int)state_len;
  a.k_own = static_cast<const uint16_t*>(k_q);
  a.v_own = static_cast<const uint16_t*>(v_q);
  a.sk_b = k_strides[0], a.sk_h = k_strides[1], a.sk_l = k_strides[2];
  a.sv_b = v_strides[0], a.sv_h = v_strides[1], a.sv_l = v_strides[2];
  a.own_lengths = lengths;
  Plan p;
  if (!make_plan(cache, B, H, L, state_len + L, true, &p)) return D3B_EINVAL;
  if (int rc = check_workspace(workspace, workspace_bytes, plan_bytes(p, cache->head_dim))) return rc;
  return run(a, cache, p, dtype == D3B_BF16, workspace, reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
