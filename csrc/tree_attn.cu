// Attention of a tree of drafted tokens over a paged cache (T = 1: plain decoding).
//
// For node t of a sequence with n cached rows and ancestor set A(t) (t included):
//   s_j = scale q_t.k_j over j in [0, n) of the cache and j in A(t) of the nodes' own k,
//   out_t = sum_j softmax(s)_j v_j  (times sigmoid(gate)),   lse_t = log sum_j e^{s_j}.
//
// First form: one CTA per (node, query head, sequence), one pass over the keys with a
// running maximum and sum per warp, the warps' parts joined in shared memory.
#include <cuda_fp8.h>

#include "decode.h"
#include "sm100.cuh"

namespace ns {

using bf16 = __nv_bfloat16;

namespace tattn {

constexpr int EXP_BIAS = 127, EXP_MIN = -117, EXP_MAX = 118;

struct Args {
  const bf16 *q, *k, *v, *gate;
  int64_t q_bs, q_ts, q_hs, k_bs, k_ts, k_hs, v_bs, v_ts, v_hs, g_bs, g_ts, g_hs;
  const void *kp, *vp;
  const uint8_t *ke, *ve;
  const int *table, *lens, *parents, *counts;
  int64_t p_bs, pages, max_pages;
  int b, T, Hq, Hk, D, page;
  float scale_log2;
  bf16* out;   // [b, T, Hq, D]
  float* lse;  // [b, Hq, T]
  int* err;
};

__device__ __forceinline__ float bf(bf16 x) { return __bfloat162float(x); }

__device__ __forceinline__ float row_value(const void* p, const uint8_t* ex, int64_t row, int D, int d) {
  if (!ex) return bf(reinterpret_cast<const bf16*>(p)[row * D + d]);
  const __half_raw h = __nv_cvt_fp8_to_halfraw(reinterpret_cast<const uint8_t*>(p)[row * D + d], __NV_E4M3);
  const int e = min(max((int)ex[row] - EXP_BIAS, EXP_MIN), EXP_MAX);
  return __half2float(__half(h)) * __uint_as_float((uint32_t)(e + 127) << 23);
}

constexpr int NW = 4, E = 8;  // warps per CTA; channels per lane (head_dim <= 256)

__global__ void __launch_bounds__(NW * 32) tree_attn_kernel(Args a) {
  __shared__ float part[NW][256 + 2];
  const int t = blockIdx.x, h = blockIdx.y, s = blockIdx.z;
  const int hk = h / (a.Hq / a.Hk);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int cnt = a.counts ? a.counts[s] : a.T;
  int64_t len = a.lens[s];
  if (cnt < 0 || cnt > a.T || len < 0 || len > a.max_pages * a.page) {
    if (threadIdx.x == 0) atomicExch(a.err, ERR_INDEX);
    cnt = min(max(cnt, 0), a.T);
    len = min(max(len, (int64_t)0), a.max_pages * a.page);
  }
  bf16* out = a.out + (((int64_t)s * a.T + t) * a.Hq + h) * a.D;
  float* lse = a.lse + ((int64_t)s * a.Hq + h) * a.T + t;
  if (t >= cnt) {
    for (int d = threadIdx.x; d < a.D; d += NW * 32) out[d] = __float2bfloat16(0.f);
    if (threadIdx.x == 0) *lse = -INFINITY;
    return;
  }
  // ancestors of node t as a bit set
  unsigned long long anc = 0;
  for (int n = t; n >= 0;) {
    anc |= 1ull << n;
    int p = a.parents[s * a.p_bs + n];
    if (p < -1 || p >= n) {
      if (threadIdx.x == 0) atomicExch(a.err, ERR_INDEX);
      p = -1;
    }
    n = p;
  }
  float q[E], o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int d = lane + 32 * e;
    q[e] = d < a.D ? bf(a.q[s * a.q_bs + t * a.q_ts + h * a.q_hs + d]) * a.scale_log2 : 0.f;
    o[e] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int64_t j = warp; j < len + a.T; j += NW) {
    float kv[E], vv[E];
    if (j < len) {
      const int64_t pg = a.table[s * a.max_pages + j / a.page];
      if (pg < 0 || pg >= a.pages) {
        if (lane == 0) atomicExch(a.err, ERR_INDEX);
        continue;
      }
      const int64_t row = (pg * a.Hk + hk) * a.page + j % a.page;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int d = lane + 32 * e;
        kv[e] = d < a.D ? row_value(a.kp, a.ke, row, a.D, d) : 0.f;
        vv[e] = d < a.D ? row_value(a.vp, a.ve, row, a.D, d) : 0.f;
      }
    } else {
      const int n = (int)(j - len);
      if (!((anc >> n) & 1)) continue;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int d = lane + 32 * e;
        kv[e] = d < a.D ? bf(a.k[s * a.k_bs + n * a.k_ts + hk * a.k_hs + d]) : 0.f;
        vv[e] = d < a.D ? bf(a.v[s * a.v_bs + n * a.v_ts + hk * a.v_hs + d]) : 0.f;
      }
    }
    float x = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) x = fmaf(q[e], kv[e], x);
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) x += __shfl_xor_sync(0xffffffff, x, i);
    const float mn = fmaxf(m, x);
    const float al = mn == -INFINITY ? 1.f : exp2f(m - mn), p = mn == -INFINITY ? 0.f : exp2f(x - mn);
    m = mn;
    l = l * al + p;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * al + p * vv[e];
  }
#pragma unroll
  for (int e = 0; e < E; ++e) part[warp][lane + 32 * e] = o[e];
  if (lane == 0) part[warp][256] = m, part[warp][257] = l;
  __syncthreads();
  float mt = -INFINITY, lt = 0.f, w[NW];
  for (int i = 0; i < NW; ++i) mt = fmaxf(mt, part[i][256]);
  for (int i = 0; i < NW; ++i) {
    w[i] = mt == -INFINITY ? 0.f : exp2f(part[i][256] - mt);
    lt += w[i] * part[i][257];
  }
  for (int d = threadIdx.x; d < a.D; d += NW * 32) {
    float x = 0.f;
    for (int i = 0; i < NW; ++i) x += w[i] * part[i][d];
    x = x / lt;
    if (a.gate) x = x / (1.f + expf(-bf(a.gate[s * a.g_bs + t * a.g_ts + h * a.g_hs + d])));
    out[d] = __float2bfloat16(x);
  }
  if (threadIdx.x == 0) *lse = (mt + log2f(lt)) * 0.6931471805599453f;
}

}  // namespace tattn

std::vector<at::Tensor> tree_attention(at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor k_pool, at::Tensor v_pool,
                                       OptTensor k_exp, OptTensor v_exp, at::Tensor table, at::Tensor lens,
                                       at::Tensor parents, OptTensor counts, OptTensor gate,
                                       c10::optional<double> scale) {
  const CacheView c = check_cache(k_pool, v_pool, k_exp, v_exp);
  const at::Device dev = k_pool.device();
  const at::cuda::CUDAGuard guard(dev);
  NS_VALUE(q.dim() == 4 && q.scalar_type() == at::kBFloat16 && q.device() == dev,
           "tree_attention: q must be bfloat16 [b, T, Hq, D] on the cache's device");
  const int64_t b = q.size(0), T = q.size(1), Hq = q.size(2), D = q.size(3);
  for (const at::Tensor* x : {&k, &v})
    NS_VALUE(x->dim() == 4 && x->scalar_type() == at::kBFloat16 && x->device() == dev && x->size(0) == b &&
                 x->size(1) == T && x->size(2) == c.heads && x->size(3) == c.d,
             "tree_attention: k and v must be bfloat16 [b, T, Hk, D] like the cache");
  NS_VALUE(D == c.d, "tree_attention: q and the cache differ in head_dim");
  NS_VALUE(Hq >= 1 && Hq % c.heads == 0, "tree_attention: query heads must be a multiple of key heads");
  NS_VALUE(T >= 1 && T <= MAX_NODES, "a tree has 1 to 64 nodes");
  NS_VALUE(!gate.has_value() || (gate->sizes() == q.sizes() && gate->scalar_type() == at::kBFloat16 &&
                                 gate->device() == dev),
           "tree_attention: gate must be bfloat16 with q's shape");
  NS_VALUE(!scale.has_value() || *scale > 0, "tree_attention: scale must be positive");
  NS_VALUE(b < 65536 && Hq < 65536, "tree_attention: too many sequences or heads");
  NS_VALUE(table.device() == dev && table.scalar_type() == at::kInt && table.dim() == 2 && table.size(0) == b &&
               table.is_contiguous(),
           "table must be contiguous int32 [b, max_pages]");
  tattn::Args a{};
  a.lens = check_index(lens, b, dev, "lens");
  a.counts = check_index(counts, b, dev, "counts");
  a.parents = check_parents(parents, b, T, dev, a.p_bs);
  at::Tensor out = at::empty({b, T, Hq, D}, q.options());
  at::Tensor lse = at::empty({b, Hq, T}, q.options().dtype(at::kFloat));
  if (b == 0) return {out, lse};
  q = aligned_rows(q);
  k = aligned_rows(k);
  v = aligned_rows(v);
  a.q = reinterpret_cast<const bf16*>(q.data_ptr());
  a.q_bs = q.stride(0), a.q_ts = q.stride(1), a.q_hs = q.stride(2);
  a.k = reinterpret_cast<const bf16*>(k.data_ptr());
  a.k_bs = k.stride(0), a.k_ts = k.stride(1), a.k_hs = k.stride(2);
  a.v = reinterpret_cast<const bf16*>(v.data_ptr());
  a.v_bs = v.stride(0), a.v_ts = v.stride(1), a.v_hs = v.stride(2);
  at::Tensor g;
  if (gate.has_value()) {
    g = aligned_rows(*gate);
    a.gate = reinterpret_cast<const bf16*>(g.data_ptr());
    a.g_bs = g.stride(0), a.g_ts = g.stride(1), a.g_hs = g.stride(2);
  }
  a.kp = c.k, a.vp = c.v, a.ke = c.ke, a.ve = c.ve;
  a.table = table.data_ptr<int>();
  a.pages = c.pages, a.max_pages = table.size(1);
  a.b = (int)b, a.T = (int)T, a.Hq = (int)Hq, a.Hk = c.heads, a.D = (int)D, a.page = c.page;
  a.scale_log2 = (float)(scale.value_or(1.0 / std::sqrt((double)D)) * 1.4426950408889634);
  a.out = reinterpret_cast<bf16*>(out.data_ptr());
  a.lse = lse.data_ptr<float>();
  a.err = device_error_flag();
  tattn::tree_attn_kernel<<<dim3((unsigned)T, (unsigned)Hq, (unsigned)b), tattn::NW * 32, 0, stream()>>>(a);
  NS_CUDA(cudaGetLastError());
  return {out, lse};
}

}  // namespace ns
