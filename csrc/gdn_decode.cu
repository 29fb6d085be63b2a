// The gated delta rule from a carried state: tokens that move it on, a tree of drafted
// tokens that leaves it alone, and the state after the accepted path of such a tree.
//
// With k^ = k / sqrt(|k|^2 + 1e-6), q^ = d^-1/2 q / sqrt(|q|^2 + 1e-6), node t continuing
// from the state S_p of its parent p (the carried state S for p = -1):
//   u_t = beta_t (v_t - e^{g_t} S_p^T k^_t),   S_t = e^{g_t} S_p + k^_t u_t^T,   o_t = S_t^T q^_t.
// Written out over a tree no state per node is needed. Let w_t be the product of e^{g} on
// the way from the root to t, and D[t, a] the product of e^{g} after a on the way to t
// (1 for a = t, 0 when a is not an ancestor); both follow row by row from the parent's row,
//   D[t, :] = e^{g_t} D[p, :],  D[t, t] = 1,   w_t = e^{g_t} w_p.
// Then with S read once
//   u_t = beta_t (v_t - w_t S^T k^_t - sum_{a < t} D[t, a] (k^_t.k^_a) u_a)
//   o_t = w_t S^T q^_t + sum_{a <= t} D[t, a] (q^_t.k^_a) u_a.
// Products of decays (rather than e^{G_t - G_a} of summed logs) keep their relative
// precision when fast and slow decays meet, and g = -inf (a reset) needs no care.
//
// First form: one CTA per (value head, sequence), thread = value channel with its column
// of the state in registers; everything in fp32.
#include "decode.h"
#include "sm100.cuh"

namespace ns {

using bf16 = __nv_bfloat16;

namespace gdnd {

__device__ __forceinline__ float bf(bf16 x) { return __bfloat162float(x); }

struct Args {
  const bf16 *q, *k, *v, *beta;
  int64_t q_bs, q_ts, q_hs, k_bs, k_ts, k_hs, v_bs, v_ts, v_hs, b_bs, b_ts;
  const float* g;
  int64_t g_bs, g_ts;
  const float *state, *u_in;
  float* out_state;
  int64_t s_rs, o_rs, n;
  const int *rows, *counts, *parents, *path;
  int64_t p_bs;
  int T, m, nv, groups;
  bf16* out;
  float* u;
  int* err;
};

__device__ __forceinline__ float block_sum(float x, float* buf) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffff, x, o);
  const int nw = (blockDim.x + 31) / 32;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = x;
  __syncthreads();
  float s = 0.f;
  for (int i = 0; i < nw; ++i) s += buf[i];
  return s;
}

// row of the state pool of sequence s, or -1 (idle or out of range)
__device__ __forceinline__ int64_t state_row(const Args& a, int s) {
  const int64_t r = a.rows ? a.rows[s] : s;
  if (r < -1 || r >= a.n) {
    if (threadIdx.x == 0) atomicExch(a.err, ERR_INDEX);
    return -1;
  }
  return r;
}

__device__ __forceinline__ int node_count(const Args& a, int s) {
  int c = a.counts ? a.counts[s] : a.T;
  if (c < 0 || c > a.T) {
    if (threadIdx.x == 0) atomicExch(a.err, ERR_INDEX);
    c = min(max(c, 0), a.T);
  }
  return c;
}

// Threads: max(D, 32); threads at or beyond D take part in reductions only.
template <int D>
__global__ void __launch_bounds__(D < 32 ? 32 : D) gdn_advance_kernel(Args a) {
  __shared__ float ks[D], qs[D], buf[8];
  const int h = blockIdx.x, s = blockIdx.y, c = threadIdx.x, hk = h / a.groups;
  const bool on = c < D;
  const int64_t row = state_row(a, s);
  const int cnt = row < 0 ? 0 : node_count(a, s);
  float S[D];
  const float* st = a.state + (row < 0 ? 0 : row) * a.s_rs + (int64_t)h * D * D;
#pragma unroll
  for (int i = 0; i < D; ++i) S[i] = on && row >= 0 ? st[i * D + c] : 0.f;
  for (int t = 0; t < cnt; ++t) {
    const float kv = on ? bf(a.k[s * a.k_bs + t * a.k_ts + hk * a.k_hs + c]) : 0.f;
    const float qv = on ? bf(a.q[s * a.q_bs + t * a.q_ts + hk * a.q_hs + c]) : 0.f;
    const float ik = rsqrtf(block_sum(kv * kv, buf) + 1e-6f);
    const float iq = rsqrtf(block_sum(qv * qv, buf) + 1e-6f) * rsqrtf((float)D);
    if (on) ks[c] = kv * ik, qs[c] = qv * iq;
    __syncthreads();
    const float eg = expf(a.g[s * a.g_bs + t * a.g_ts + h]);
    const float be = bf(a.beta[s * a.b_bs + t * a.b_ts + h]);
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < D; ++i) {
      S[i] *= eg;
      x = fmaf(S[i], ks[i], x);
    }
    const float u = on ? be * (bf(a.v[s * a.v_bs + t * a.v_ts + h * a.v_hs + c]) - x) : 0.f;
    float o = 0.f;
#pragma unroll
    for (int i = 0; i < D; ++i) {
      S[i] = fmaf(ks[i], u, S[i]);
      o = fmaf(S[i], qs[i], o);
    }
    if (on) a.out[(((int64_t)s * a.T + t) * a.nv + h) * D + c] = __float2bfloat16(o);
  }
  for (int t = cnt; t < a.T; ++t)
    if (on) a.out[(((int64_t)s * a.T + t) * a.nv + h) * D + c] = __float2bfloat16(0.f);
  if (row < 0 || !on) return;
  float* so = a.out_state + row * a.o_rs + (int64_t)h * D * D;
#pragma unroll
  for (int i = 0; i < D; ++i) so[i * D + c] = S[i];
}

template <int D>
__global__ void __launch_bounds__(D < 32 ? 32 : D) gdn_verify_kernel(Args a) {
  extern __shared__ float sm[];
  float* ks = sm;                // [T][D] normalised keys
  float* qs = ks + a.T * D;      // [T][D]
  float* us = qs + a.T * D;      // [T][D]
  float* dec = us + a.T * D;     // [T][T] decays between nodes
  float* kk = dec + a.T * a.T;   // [T] products of the current node with every earlier key
  float* qk = kk + a.T;          // [T]
  float* w = qk + a.T;           // [T] decays from the carried state
  __shared__ float buf[8];
  const int h = blockIdx.x, s = blockIdx.y, c = threadIdx.x, hk = h / a.groups;
  const bool on = c < D;
  const int64_t row = state_row(a, s);
  const int cnt = row < 0 ? 0 : node_count(a, s);
  float S[D];
  const float* st = a.state + (row < 0 ? 0 : row) * a.s_rs + (int64_t)h * D * D;
#pragma unroll
  for (int i = 0; i < D; ++i) S[i] = on && row >= 0 ? st[i * D + c] : 0.f;
  for (int t = 0; t < cnt; ++t) {
    const float kv = on ? bf(a.k[s * a.k_bs + t * a.k_ts + hk * a.k_hs + c]) : 0.f;
    const float qv = on ? bf(a.q[s * a.q_bs + t * a.q_ts + hk * a.q_hs + c]) : 0.f;
    const float ik = rsqrtf(block_sum(kv * kv, buf) + 1e-6f);
    const float iq = rsqrtf(block_sum(qv * qv, buf) + 1e-6f) * rsqrtf((float)D);
    if (on) ks[t * D + c] = kv * ik, qs[t * D + c] = qv * iq;
    int p = a.parents[s * a.p_bs + t];
    if (p < -1 || p >= t) {
      if (c == 0) atomicExch(a.err, ERR_INDEX);
      p = -1;
    }
    const float eg = expf(a.g[s * a.g_bs + t * a.g_ts + h]);
    const float be = bf(a.beta[s * a.b_bs + t * a.b_ts + h]);
    for (int j = c; j <= t; j += blockDim.x)  // row p holds columns up to p
      dec[t * a.T + j] = j == t ? 1.f : j > p ? 0.f : eg * dec[p * a.T + j];
    if (c == 0) w[t] = p < 0 ? eg : eg * w[p];
    __syncthreads();
    for (int j = c; j <= t; j += blockDim.x) {
      float x = 0.f, y = 0.f;
      for (int i = 0; i < D; ++i) {
        x = fmaf(ks[t * D + i], ks[j * D + i], x);
        y = fmaf(qs[t * D + i], ks[j * D + i], y);
      }
      kk[j] = x * dec[t * a.T + j];
      qk[j] = y * dec[t * a.T + j];
    }
    __syncthreads();
    float x = 0.f, y = 0.f;
#pragma unroll
    for (int i = 0; i < D; ++i) {
      x = fmaf(S[i], ks[t * D + i], x);
      y = fmaf(S[i], qs[t * D + i], y);
    }
    x *= w[t], y *= w[t];
    if (on) {
      for (int j = 0; j < t; ++j) {
        x = fmaf(kk[j], us[j * D + c], x);
        y = fmaf(qk[j], us[j * D + c], y);
      }
      const float u = be * (bf(a.v[s * a.v_bs + t * a.v_ts + h * a.v_hs + c]) - x);
      us[t * D + c] = u;
      const int64_t at = (((int64_t)s * a.T + t) * a.nv + h) * D + c;
      a.u[at] = u;
      a.out[at] = __float2bfloat16(fmaf(qk[t], u, y));
    }
  }
  for (int t = cnt; t < a.T; ++t)
    if (on) {
      const int64_t at = (((int64_t)s * a.T + t) * a.nv + h) * D + c;
      a.u[at] = 0.f;
      a.out[at] = __float2bfloat16(0.f);
    }
}

template <int D>
__global__ void __launch_bounds__(D < 32 ? 32 : D) gdn_accept_kernel(Args a) {
  __shared__ float ks[D], buf[8];
  const int h = blockIdx.x, s = blockIdx.y, c = threadIdx.x, hk = h / a.groups;
  const bool on = c < D;
  const int64_t row = state_row(a, s);
  if (row < 0) return;
  float S[D];
  const float* st = a.state + row * a.s_rs + (int64_t)h * D * D;
#pragma unroll
  for (int i = 0; i < D; ++i) S[i] = on ? st[i * D + c] : 0.f;
  for (int j = 0; j < a.m; ++j) {
    const int t = a.path[(int64_t)s * a.m + j];
    if (t < 0 || t >= a.T) {
      if (t != -1 && c == 0) atomicExch(a.err, ERR_INDEX);
      continue;
    }
    const float kv = on ? bf(a.k[s * a.k_bs + t * a.k_ts + hk * a.k_hs + c]) : 0.f;
    const float ik = rsqrtf(block_sum(kv * kv, buf) + 1e-6f);
    if (on) ks[c] = kv * ik;
    __syncthreads();
    const float eg = expf(a.g[s * a.g_bs + t * a.g_ts + h]);
    const float u = on ? a.u_in[(((int64_t)s * a.T + t) * a.nv + h) * D + c] : 0.f;
#pragma unroll
    for (int i = 0; i < D; ++i) S[i] = fmaf(ks[i], u, S[i] * eg);
    __syncthreads();
  }
  if (!on) return;
  float* so = a.out_state + row * a.o_rs + (int64_t)h * D * D;
#pragma unroll
  for (int i = 0; i < D; ++i) so[i * D + c] = S[i];
}

}  // namespace gdnd

namespace {

struct Delta {
  gdnd::Args a{};
  int64_t b, T, nk, nv, D;
  at::Device dev{at::kCUDA};
  std::vector<at::Tensor> keep;  // aligned copies that outlive the launch call
};

const bf16* bf_ptr(const at::Tensor& t) { return reinterpret_cast<const bf16*>(t.data_ptr()); }

void bind_state(Delta& d, const at::Tensor& state, const OptTensor& rows, const at::Tensor* out) {
  auto ok = [&](const at::Tensor& s) {
    return s.dim() == 4 && s.size(1) == d.nv && s.size(2) == d.D && s.size(3) == d.D && s.scalar_type() == at::kFloat &&
           s.device() == d.dev && (s.size(0) == 0 || s[0].is_contiguous()) && s.stride(0) % 4 == 0 &&
           reinterpret_cast<uintptr_t>(s.data_ptr()) % 16 == 0;
  };
  NS_VALUE(ok(state), "gated delta rule: state must be fp32 [n, nv, D, D], dense and aligned within a row");
  NS_VALUE(rows.has_value() || state.size(0) == d.b, "gated delta rule: one state per sequence, or rows");
  d.a.state = state.data_ptr<float>();
  d.a.s_rs = state.stride(0);
  d.a.n = state.size(0);
  d.a.rows = check_index(rows, d.b, d.dev, "rows");
  if (out) {
    NS_VALUE(ok(*out) && out->size(0) == state.size(0), "gated delta rule: out_state must be like state");
    d.a.out_state = out->data_ptr<float>();
    d.a.o_rs = out->stride(0);
  }
}

Delta bind_nodes(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& g,
                 const at::Tensor& beta, int64_t groups, const OptTensor& counts) {
  Delta d;
  d.dev = q.device();
  NS_VALUE(q.dim() == 4 && v.dim() == 4 && groups >= 1, "gated delta rule: q, k, v must be [b, T, heads, D]");
  d.b = q.size(0), d.T = q.size(1), d.nk = q.size(2), d.D = q.size(3), d.nv = d.nk * groups;
  for (const at::Tensor* x : {&q, &k, &v, &beta})
    NS_VALUE(x->scalar_type() == at::kBFloat16 && x->device() == d.dev,
             "gated delta rule: q, k, v and beta must be bfloat16 on one device");
  NS_VALUE(k.sizes() == q.sizes() && v.sizes() == at::IntArrayRef({d.b, d.T, d.nv, d.D}),
           "gated delta rule: k must have q's shape, v groups * nk heads");
  NS_VALUE(g.scalar_type() == at::kFloat && g.device() == d.dev && g.sizes() == at::IntArrayRef({d.b, d.T, d.nv}) &&
               beta.sizes() == g.sizes(),
           "gated delta rule: g (fp32) and beta must be [b, T, nv]");
  NS_VALUE(d.D == 16 || d.D == 32 || d.D == 64 || d.D == 128, "gated delta rule: head_dim must be 16, 32, 64 or 128");
  NS_VALUE(d.T >= 1, "gated delta rule: no tokens");
  NS_VALUE(d.b < 65536 && d.nv < 65536, "gated delta rule: too many sequences or heads");
  d.keep = {aligned_rows(q), aligned_rows(k), aligned_rows(v), g.stride(2) == 1 ? g : g.contiguous(),
            beta.stride(2) == 1 ? beta : beta.contiguous()};
  gdnd::Args& a = d.a;
  a.q = bf_ptr(d.keep[0]);
  a.q_bs = d.keep[0].stride(0), a.q_ts = d.keep[0].stride(1), a.q_hs = d.keep[0].stride(2);
  a.k = bf_ptr(d.keep[1]);
  a.k_bs = d.keep[1].stride(0), a.k_ts = d.keep[1].stride(1), a.k_hs = d.keep[1].stride(2);
  a.v = bf_ptr(d.keep[2]);
  a.v_bs = d.keep[2].stride(0), a.v_ts = d.keep[2].stride(1), a.v_hs = d.keep[2].stride(2);
  a.g = d.keep[3].data_ptr<float>();
  a.g_bs = d.keep[3].stride(0), a.g_ts = d.keep[3].stride(1);
  a.beta = bf_ptr(d.keep[4]);
  a.b_bs = d.keep[4].stride(0), a.b_ts = d.keep[4].stride(1);
  a.counts = check_index(counts, d.b, d.dev, "counts");
  a.T = (int)d.T, a.nv = (int)d.nv, a.groups = (int)groups;
  a.err = device_error_flag();
  return d;
}

}  // namespace

#define NS_GDN_CASES(D_, X) \
  switch (D_) {             \
    case 16: X(16) break;   \
    case 32: X(32) break;   \
    case 64: X(64) break;   \
    default: X(128) break;  \
  }

at::Tensor gdn_advance(at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor g, at::Tensor beta, at::Tensor state,
                       int64_t groups, OptTensor counts, OptTensor rows, at::Tensor out_state) {
  const at::cuda::CUDAGuard guard(q.device());
  Delta d = bind_nodes(q, k, v, g, beta, groups, counts);
  bind_state(d, state, rows, &out_state);
  at::Tensor out = at::empty({d.b, d.T, d.nv, d.D}, v.options());
  if (out.numel() == 0) return out;
  d.a.out = reinterpret_cast<bf16*>(out.data_ptr());
  const dim3 grid((unsigned)d.nv, (unsigned)d.b);
#define NS_X(DD) gdnd::gdn_advance_kernel<DD><<<grid, DD < 32 ? 32 : DD, 0, stream()>>>(d.a);
  NS_GDN_CASES(d.D, NS_X)
#undef NS_X
  NS_CUDA(cudaGetLastError());
  return out;
}

std::vector<at::Tensor> gdn_verify(at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor g, at::Tensor beta,
                                   at::Tensor state, at::Tensor parents, int64_t groups, OptTensor counts,
                                   OptTensor rows) {
  const at::cuda::CUDAGuard guard(q.device());
  Delta d = bind_nodes(q, k, v, g, beta, groups, counts);
  NS_VALUE(d.T <= MAX_NODES, "a tree has 1 to 64 nodes");
  bind_state(d, state, rows, nullptr);
  d.a.parents = check_parents(parents, d.b, d.T, d.dev, d.a.p_bs);
  at::Tensor out = at::empty({d.b, d.T, d.nv, d.D}, v.options());
  at::Tensor u = at::empty({d.b, d.T, d.nv, d.D}, g.options());
  if (out.numel() == 0) return {out, u};
  d.a.out = reinterpret_cast<bf16*>(out.data_ptr());
  d.a.u = u.data_ptr<float>();
  const dim3 grid((unsigned)d.nv, (unsigned)d.b);
  const int smem = (int)((3 * d.T * d.D + d.T * d.T + 3 * d.T) * 4);
#define NS_X(DD)                                                                                       \
  {                                                                                                    \
    static std::atomic<unsigned long long> attr{0};                                                    \
    once_per_device(attr, [&] {                                                                        \
      NS_CUDA(cudaFuncSetAttribute(gdnd::gdn_verify_kernel<DD>, cudaFuncAttributeMaxDynamicSharedMemorySize, \
                                   (3 * MAX_NODES * DD + MAX_NODES * MAX_NODES + 3 * MAX_NODES) * 4)); \
    });                                                                                                \
    gdnd::gdn_verify_kernel<DD><<<grid, DD < 32 ? 32 : DD, smem, stream()>>>(d.a);                     \
  }
  NS_GDN_CASES(d.D, NS_X)
#undef NS_X
  NS_CUDA(cudaGetLastError());
  return {out, u};
}

void gdn_accept(at::Tensor k, at::Tensor g, at::Tensor u, at::Tensor path, at::Tensor state, int64_t groups,
                OptTensor rows, at::Tensor out_state) {
  const at::cuda::CUDAGuard guard(k.device());
  Delta d;
  d.dev = k.device();
  NS_VALUE(k.dim() == 4 && k.scalar_type() == at::kBFloat16 && groups >= 1,
           "gated_delta_accept: k must be bfloat16 [b, T, nk, D]");
  d.b = k.size(0), d.T = k.size(1), d.nk = k.size(2), d.D = k.size(3), d.nv = d.nk * groups;
  NS_VALUE(d.D == 16 || d.D == 32 || d.D == 64 || d.D == 128, "gated delta rule: head_dim must be 16, 32, 64 or 128");
  NS_VALUE(u.device() == d.dev && u.scalar_type() == at::kFloat &&
               u.sizes() == at::IntArrayRef({d.b, d.T, d.nv, d.D}),
           "gated_delta_accept: u must be fp32 [b, T, nv, D]");
  NS_VALUE(g.device() == d.dev && g.scalar_type() == at::kFloat && g.sizes() == at::IntArrayRef({d.b, d.T, d.nv}),
           "gated_delta_accept: g must be fp32 [b, T, nv]");
  NS_VALUE(path.device() == d.dev && path.scalar_type() == at::kInt && path.dim() == 2 && path.size(0) == d.b &&
               path.is_contiguous(),
           "gated_delta_accept: path must be contiguous int32 [b, m]");
  NS_VALUE(d.b < 65536 && d.nv < 65536, "gated delta rule: too many sequences or heads");
  bind_state(d, state, rows, &out_state);
  if (d.b * d.nv == 0) return;
  d.keep = {aligned_rows(k), g.stride(2) == 1 ? g : g.contiguous(), u.contiguous()};
  d.a.k = bf_ptr(d.keep[0]);
  d.a.k_bs = d.keep[0].stride(0), d.a.k_ts = d.keep[0].stride(1), d.a.k_hs = d.keep[0].stride(2);
  d.a.g = d.keep[1].data_ptr<float>();
  d.a.g_bs = d.keep[1].stride(0), d.a.g_ts = d.keep[1].stride(1);
  d.a.u_in = d.keep[2].data_ptr<float>();
  d.a.path = path.data_ptr<int>();
  d.a.T = (int)d.T, d.a.m = (int)path.size(1), d.a.nv = (int)d.nv, d.a.groups = (int)groups;
  d.a.err = device_error_flag();
  const dim3 grid((unsigned)d.nv, (unsigned)d.b);
#define NS_X(DD) gdnd::gdn_accept_kernel<DD><<<grid, DD < 32 ? 32 : DD, 0, stream()>>>(d.a);
  NS_GDN_CASES(d.D, NS_X)
#undef NS_X
  NS_CUDA(cudaGetLastError());
}

}  // namespace ns
