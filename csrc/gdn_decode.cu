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
// Bound: the states' bytes (4 D^2 per head and sequence, each read once, and written once where
// it moves on); for wide trees and prompts the T x T algebra and the products with S.
//
// A CTA takes 64 value channels (columns of S are independent) of one head, a warp 16 of
// them, as S^T in the accumulator layout of mma.sync m16n8k16 (fp32, 64 registers), which is
// also the layout of its A operand: S^T K^T and S^T Q^T take S as the sum of three bf16
// matrices (24 bits) against the raw bf16 keys, exact up to fp32 accumulation; the norms are
// factored out. Moving S on adds U^T K, with U split the same way, into the same registers.
// (mma.sync and not tcgen05: the fp32 state has to be split in registers anyway, and at the
// sizes of a decoding step the loads of S dominate.) The unit triangular system in u is
// solved by blocks of 16 nodes in fp32.
//
// Measured (48 heads of 128): one token of 64 sequences 75 us and short paths 76 us (5.4 TB/s,
// 84 % of the copy rate), the states' bytes. Trees: 16 sequences x 16 nodes 44 us, 32 x 61 nodes
// 224 us (0.95 TB/s); 333 tokens of 2 sequences 132 us, six chunks in a row. A CTA's phases wait
// for one another (loads, S K, M, solve, A u) with few warps an SM to hide it: 12 up to 32 nodes (3
// CTAs by registers), 8 beyond (2 by shared memory; kept to the 168 registers of three, 243 and 156 us).
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

// ------------------------------------------------------------------ tensor-core pieces
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldsm_x4_trans(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(sm100::smem_u32(p)));
}

// x = hi + mid + lo in bf16, for a pair of values; the parts packed
__device__ __forceinline__ void split3(float x, float y, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  const float2 hf = __bfloat1622float2(h);
  const float rx = x - hf.x, ry = y - hf.y;
  const __nv_bfloat162 m = __floats2bfloat162_rn(rx, ry);
  const float2 mf = __bfloat1622float2(m);
  const __nv_bfloat162 l = __floats2bfloat162_rn(rx - mf.x, ry - mf.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  mid = *reinterpret_cast<const uint32_t*>(&m);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

// One warp's 16 value channels of S^T: register [j][..] holds key channels 8j + 2q, + 1 of
// value channels 2g (first two) and 2g + 1 (last two), lane = 4g + q.
template <int D>
struct State {
  float s[D / 8][4];
  __device__ __forceinline__ void load(const float* p, int g, int q) {
#pragma unroll
    for (int j = 0; j < D / 8; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float2 x = *reinterpret_cast<const float2*>(p + (int64_t)(8 * j + 2 * q + i) * D + 2 * g);
        s[j][i] = x.x;
        s[j][2 + i] = x.y;
      }
  }
  __device__ __forceinline__ void store(float* p, int g, int q) const {
#pragma unroll
    for (int j = 0; j < D / 8; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        *reinterpret_cast<float2*>(p + (int64_t)(8 * j + 2 * q + i) * D + 2 * g) = make_float2(s[j][i], s[j][2 + i]);
  }
  __device__ __forceinline__ void scale(float f) {
#pragma unroll
    for (int j = 0; j < D / 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[j][i] *= f;
  }
  // S^T += W^T K over 16 rows: w(row, value pair) in fp32, K rows bf16 in shared memory
  template <int US, int KS>
  __device__ __forceinline__ void add(const float* u, const float* coef, const bf16* k, int lane) {
    const int g = lane >> 2, q = lane & 3;
    uint32_t a[3][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = 8 * h + 2 * q;
      const float2 x = *reinterpret_cast<const float2*>(u + r * US + 2 * g);
      const float2 y = *reinterpret_cast<const float2*>(u + (r + 1) * US + 2 * g);
      const float c0 = coef[r], c1 = coef[r + 1];
      split3(x.x * c0, y.x * c1, a[0][2 * h], a[1][2 * h], a[2][2 * h]);
      split3(x.y * c0, y.y * c1, a[0][2 * h + 1], a[1][2 * h + 1], a[2][2 * h + 1]);
    }
#pragma unroll
    for (int j = 0; j < D / 8; j += 2) {
      uint32_t b[4];  // rows 0-7 and 8-15 of key channels 8j.., then of 8j + 8..
      ldsm_x4_trans(b, k + ((lane & 7) + (lane & 8)) * KS + 8 * j + (lane >> 4) * 8);
#pragma unroll
      for (int x = 0; x < 3; ++x) {
        mma16816(s[j], a[x], b[0], b[1]);
        mma16816(s[j + 1], a[x], b[2], b[3]);
      }
    }
  }
};

// Rows [0, rows) of D channels into shared memory, asynchronously; zeros at and beyond `live`
// (`live` >= 1).
template <int D, int ST>
__device__ __forceinline__ void copy_rows(const bf16* src, int64_t ts, int live, int rows, bf16* dst) {
  constexpr int L = D / 8;  // 16-byte chunks of one row
  for (int i = threadIdx.x; i < rows * L; i += blockDim.x) {
    const int r = i / L, c = i % L;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(sm100::smem_u32(dst + r * ST + c * 8)),
                 "l"(src + min(r, live - 1) * ts + c * 8), "r"(r < live ? 16 : 0)
                 : "memory");
  }
}

__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// 1 / sqrt(|row|^2 + 1e-6) of rows in shared memory, D / 8 lanes a row.
template <int D, int ST>
__device__ __forceinline__ void row_norms(const bf16* rows, int n, float* inv) {
  constexpr int L = D / 8;
  for (int i = threadIdx.x; i < (n * L + 31) / 32 * 32; i += blockDim.x) {
    const int r = i / L, c = i % L;
    uint4 w = make_uint4(0, 0, 0, 0);
    if (r < n) w = *reinterpret_cast<const uint4*>(rows + r * ST + c * 8);
    const uint32_t in[4] = {w.x, w.y, w.z, w.w};
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = __uint_as_float(in[e] << 16), y = __uint_as_float(in[e] & 0xffff0000u);
      ss = fmaf(x, x, fmaf(y, y, ss));
    }
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffff, ss, o);
    if (r < n && c == 0) inv[r] = rsqrtf(ss + 1e-6f);
  }
}

// x = hi + lo in bf16 (16 bits), for a pair of values
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  const float2 hf = __bfloat1622float2(h);
  const __nv_bfloat162 l = __floats2bfloat162_rn(x - hf.x, y - hf.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

// ------------------------------------------------------------------ nodes (a tree, or tokens in chunks)
template <int D, int NT>
struct Nodes {
  static constexpr int COLS = D < 64 ? D : 64;         // value channels of a CTA
  static constexpr int THREADS = COLS * 2;             // a warp per 16
  static constexpr int TP = NT < 2 ? 16 : 8 * NT;      // nodes held (zero padded)
  static constexpr int KST = D + 8;                    // row strides: 4 banks apart
  static constexpr int US = COLS + 4;
  static constexpr int MS = TP + 4;
  static constexpr int AS = TP + 8;                    // words of a row of node pairs (8 banks apart)
  static constexpr int ROWS = TP * KST * 2;            // bytes of K or Q
  static constexpr int SMEM = 2 * ROWS + TP * US * 4 + TP * MS * 4 + TP * AS * 4 + 8 * TP * 4;
  // CTAs an SM that registers are kept for (three leave each of 128 threads 168, two 255): no more than an SM's
  // 228 KB of shared memory holds, each with the 1 KB that the system takes
  static constexpr int CTAS = 3 * (SMEM + 1024) <= 228 * 1024 ? 3 : 2;
  static_assert(CTAS * (SMEM + 1024) <= 228 * 1024, "shared memory");
};

// TREE: T <= 8 NT nodes with parents; the state is only read. Otherwise tokens in chunks of
// 8 NT whose state moves on.
template <int D, int NT, bool TREE>
__global__ void __launch_bounds__(Nodes<D, NT>::THREADS, Nodes<D, NT>::CTAS) gdn_nodes_kernel(Args a) {
  using C = Nodes<D, NT>;
  constexpr int TP = C::TP, TN = 8 * NT, KST = C::KST, US = C::US, MS = C::MS, AS = C::AS, COLS = C::COLS, SL = D / COLS;
  extern __shared__ __align__(16) uint8_t sm[];
  bf16* ks = reinterpret_cast<bf16*>(sm);               // [TP][KST]
  bf16* qs = ks + TP * KST;                             // [TP][KST]
  float* us = reinterpret_cast<float*>(qs + TP * KST);  // [TP][US] right-hand sides, then u
  float* mt = us + TP * US;                             // [a][t] decays D[t, a], then M
  uint32_t* at = reinterpret_cast<uint32_t*>(mt + TP * MS);  // [2][a / 2][t] A: bf16 pairs, high and low parts
  float* ik = reinterpret_cast<float*>(at + TP * C::AS);  // [TP] 1 / |k|
  float* iq = ik + TP;                                  // [TP] D^-1/2 / |q|
  float* eg = iq + TP;                                  // [TP] e^g
  float* be = eg + TP;                                  // [TP] beta
  float* wt = be + TP;                                  // [TP] decay from the carried state
  float* cf = wt + TP;                                  // [TP] what u adds to the state
  int* par = reinterpret_cast<int*>(cf + TP);           // [TP]
  const int h = blockIdx.x / SL, cs = blockIdx.x % SL * COLS, s = blockIdx.y, hk = h / a.groups;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
  const int64_t row = state_row(a, s);
  const int cnt = row < 0 ? 0 : node_count(a, s);
  const int col0 = cs + 16 * warp;  // this warp's value channels
  State<D> S;
  if (row >= 0)
    S.load(a.state + row * a.s_rs + (int64_t)h * D * D + col0, g, q);
  else
    S.scale(0.f);
  const int64_t ob = ((int64_t)s * a.T * a.nv + h) * D + cs;  // outputs: node t at ob + t nv D
  const int64_t ots = (int64_t)a.nv * D;

  for (int t0 = 0; t0 < cnt; t0 += TN) {
    const int n = min(cnt - t0, TN);
    const bf16* kp = a.k + s * a.k_bs + t0 * a.k_ts + hk * a.k_hs;
    const bf16* qp = a.q + s * a.q_bs + t0 * a.q_ts + hk * a.q_hs;
    const bf16* vp = a.v + s * a.v_bs + t0 * a.v_ts + h * a.v_hs + col0 + 2 * g;
    // everything from global memory is asked for before anything is waited for
    if (t0 > 0) __syncthreads();  // the previous chunk's readers
    copy_rows<D, KST>(kp, a.k_ts, n, TP, ks);
    copy_rows<D, KST>(qp, a.q_ts, n, TP, qs);
    uint32_t v[NT][2];  // v of this thread's accumulators
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int t = 8 * j + 2 * q + i;
        v[j][i] = t < n ? *reinterpret_cast<const uint32_t*>(vp + t * a.v_ts) : 0u;
      }
    for (int t = tid; t < TP; t += C::THREADS) {
      const bool in = t < n;
      const float gv = in ? a.g[s * a.g_bs + (t0 + t) * a.g_ts + h] : 0.f;
      const float bv = in ? bf(a.beta[s * a.b_bs + (t0 + t) * a.b_ts + h]) : 0.f;
      if constexpr (TREE) {
        int p = in ? a.parents[s * a.p_bs + t] : -1;
        if (p < -1 || p >= t) {
          atomicExch(a.err, ERR_INDEX);
          p = -1;
        }
        par[t] = p;
      }
      eg[t] = expf(gv);
      be[t] = bv;
    }
    for (int i = tid; i < TP * MS / 4; i += C::THREADS) reinterpret_cast<float4*>(mt)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if constexpr (TN < TP)  // rows of u that no node fills
      for (int i = tid; i < (TP - TN) * US; i += C::THREADS) us[TN * US + i] = 0.f;
    copies_done();
    __syncthreads();
    row_norms<D, KST>(ks, TP, ik);
    row_norms<D, KST>(qs, TP, iq);
    // decays: a tree's rows walk up to the root, a chain's columns run down
    if constexpr (TREE) {
      for (int t = tid; t < TP; t += C::THREADS) {
        float d = 1.f;
        for (int i = t; i >= 0; i = par[i]) {
          mt[i * MS + t] = d;
          d *= eg[i];
        }
        wt[t] = d;
      }
    } else {
      for (int i = tid; i <= TP; i += C::THREADS) {  // thread TP: from the carried state
        float d = 1.f;
#pragma unroll 8
        for (int t = 0; t < TP; ++t) {
          if (i == TP) {
            d *= eg[t];
            wt[t] = d;
          } else if (t >= i) {
            if (t > i) d *= eg[t];
            mt[i * MS + t] = d;
          }
        }
      }
    }
    // (S^T K^T), (S^T Q^T): value channels x nodes
    float ka[NT][4], qa[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) ka[j][i] = qa[j][i] = 0.f;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      uint32_t f[3][4];
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y)
          split3(S.s[2 * kk + x][2 * y], S.s[2 * kk + x][2 * y + 1], f[0][2 * x + y], f[1][2 * x + y], f[2][2 * x + y]);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const bf16* kr = ks + (8 * j + g) * KST + 16 * kk + 2 * q;
        const bf16* qr = qs + (8 * j + g) * KST + 16 * kk + 2 * q;
        const uint32_t k0 = *reinterpret_cast<const uint32_t*>(kr), k1 = *reinterpret_cast<const uint32_t*>(kr + 8);
        const uint32_t q0 = *reinterpret_cast<const uint32_t*>(qr), q1 = *reinterpret_cast<const uint32_t*>(qr + 8);
#pragma unroll
        for (int x = 2; x >= 0; --x) {
          mma16816(ka[j], f[x], k0, k1);
          mma16816(qa[j], f[x], q0, q1);
        }
      }
    }
    __syncthreads();  // decays are complete
    if constexpr (!TREE)  // (a CTA of narrow heads has fewer threads than nodes)
      for (int t = tid; t < TP; t += C::THREADS) cf[t] = ik[t] * mt[t * MS + TP - 1];
    // right-hand sides beta (v - w S^T k^)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int t = 8 * j + 2 * q + i;
        const float w = wt[t] * ik[t], b = be[t];
        *reinterpret_cast<float2*>(us + t * US + 16 * warp + 2 * g) =
            make_float2(b * (__uint_as_float(v[j][i] << 16) - w * ka[j][i]),
                        b * (__uint_as_float(v[j][i] & 0xffff0000u) - w * ka[j][2 + i]));
      }
    if (!TREE) __syncthreads();  // cf before mt changes
    // K K^T and Q K^T on the lower triangle, with their decays: M and A, transposed
    const float rd = rsqrtf((float)D);
    for (int x = warp; x < TP / 16 * (TP / 16 + 1); x += C::THREADS / 32) {  // tiles of 16 x 8
      int mi = 0;
      while ((mi + 1) * (mi + 2) <= x) ++mi;
      const int nj = x - mi * (mi + 1);
      float kk4[4] = {}, qk4[4] = {};
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const bf16* ar = ks + (16 * mi + g) * KST + 16 * kk + 2 * q;
        const bf16* aq = qs + (16 * mi + g) * KST + 16 * kk + 2 * q;
        const bf16* br = ks + (8 * nj + g) * KST + 16 * kk + 2 * q;
        auto u32 = [](const bf16* p) { return *reinterpret_cast<const uint32_t*>(p); };
        const uint32_t b0 = u32(br), b1 = u32(br + 8);
        const uint32_t fa[4] = {u32(ar), u32(ar + 8 * KST), u32(ar + 8), u32(ar + 8 * KST + 8)};
        const uint32_t fq[4] = {u32(aq), u32(aq + 8 * KST), u32(aq + 8), u32(aq + 8 * KST + 8)};
        mma16816(kk4, fa, b0, b1);
        mma16816(qk4, fq, b0, b1);
      }
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        const int t = 16 * mi + g + (i >> 1) * 8, c = 8 * nj + 2 * q;
        const float d0 = mt[c * MS + t] * ik[c], d1 = mt[(c + 1) * MS + t] * ik[c + 1];
        const float sq = iq[t] * rd, sk = ik[t] * be[t];
        split2(d0 * sq * qk4[i], d1 * sq * qk4[i + 1], at[(c >> 1) * AS + t], at[(TP / 2 + (c >> 1)) * AS + t]);
        mt[c * MS + t] = c < t ? d0 * sk * kk4[i] : 0.f;
        mt[(c + 1) * MS + t] = c + 1 < t ? d1 * sk * kk4[i + 1] : 0.f;
      }
    }
    __syncthreads();
    // (I + M) u = right-hand side, by blocks of 16 nodes; thread = (value channel, half of the rows)
    const int c = tid % COLS, half = tid / COLS;
    constexpr int R = TN < 16 ? TN / 2 : 8;  // rows of one thread
    for (int r0 = 0; r0 < TN; r0 += 2 * R) {
      if (r0 > 0) {
        float x[R];
        const int r = r0 + half * R;
#pragma unroll
        for (int i = 0; i < R; ++i) x[i] = us[(r + i) * US + c];
#pragma unroll 4
        for (int m = 0; m < r0; ++m) {
          const float u = us[m * US + c];
#pragma unroll
          for (int i = 0; i < R; i += 4) {
            const float4 f = *reinterpret_cast<const float4*>(mt + m * MS + r + i);
            x[i] -= f.x * u, x[i + 1] -= f.y * u, x[i + 2] -= f.z * u, x[i + 3] -= f.w * u;
          }
        }
#pragma unroll
        for (int i = 0; i < R; ++i) us[(r + i) * US + c] = x[i];
        __syncthreads();
      }
      if (half == 0) {
        float x[2 * R];
#pragma unroll
        for (int i = 0; i < 2 * R; ++i) x[i] = us[(r0 + i) * US + c];
#pragma unroll
        for (int m = 0; m + 1 < 2 * R; ++m)
#pragma unroll
          for (int i = (m + 1) & ~3; i < 2 * R; i += 4) {
            const float4 f = *reinterpret_cast<const float4*>(mt + (r0 + m) * MS + r0 + i);
            if (i > m) x[i] -= f.x * x[m];
            if (i + 1 > m) x[i + 1] -= f.y * x[m];
            if (i + 2 > m) x[i + 2] -= f.z * x[m];
            x[i + 3] -= f.w * x[m];
          }
#pragma unroll
        for (int i = 0; i < 2 * R; ++i) us[(r0 + i) * US + c] = x[i];
      }
      __syncthreads();
    }
    // o = w S^T q^ + A u, in the accumulators of S^T Q^T. Two parts (16 bits) of u and of A are
    // plenty for an output of bf16.
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float w = wt[8 * j + 2 * q + i] * iq[8 * j + 2 * q + i] * rd;
        qa[j][i] *= w;
        qa[j][2 + i] *= w;
      }
#pragma unroll
    for (int b = 0; b < TP / 16; ++b) {  // 16 nodes a
      uint32_t f[2][4];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float* up = us + (16 * b + 8 * x + 2 * q) * US + 16 * warp + 2 * g;
        const float2 u0 = *reinterpret_cast<const float2*>(up), u1 = *reinterpret_cast<const float2*>(up + US);
        split2(u0.x, u1.x, f[0][2 * x], f[1][2 * x]);
        split2(u0.y, u1.y, f[0][2 * x + 1], f[1][2 * x + 1]);
      }
#pragma unroll
      for (int j = 2 * b; j < NT; ++j) {  // nodes t at or after them
        const uint32_t* hp = at + (8 * b + q) * AS + 8 * j + g;
        const uint32_t* lp = hp + TP / 2 * AS;
        const uint32_t h0 = hp[0], h1 = hp[4 * AS];
        mma16816(qa[j], f[1], h0, h1);
        mma16816(qa[j], f[0], lp[0], lp[4 * AS]);
        mma16816(qa[j], f[0], h0, h1);
      }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int t = 8 * j + 2 * q + i;
        if (t < n)
          *reinterpret_cast<__nv_bfloat162*>(a.out + ob + (t0 + t) * ots + 16 * warp + 2 * g) =
              __floats2bfloat162_rn(qa[j][i], qa[j][2 + i]);
      }
    if constexpr (TREE)
      for (int i = tid; i < n * COLS / 4; i += C::THREADS) {
        const int t = i / (COLS / 4), x = i % (COLS / 4) * 4;
        *reinterpret_cast<float4*>(a.u + ob + t * ots + x) = *reinterpret_cast<const float4*>(us + t * US + x);
      }
    if constexpr (!TREE) {
      S.scale(wt[TP - 1]);
#pragma unroll 1
      for (int r = 0; r < n; r += 16)
        S.template add<US, KST>(us + r * US + 16 * warp, cf + r, ks + r * KST, lane);
    }
  }
  for (int i = cnt * COLS + tid; i < a.T * COLS; i += C::THREADS) {  // padding
    const int64_t o = ob + (i / COLS) * ots + i % COLS;
    a.out[o] = __float2bfloat16(0.f);
    if constexpr (TREE) a.u[o] = 0.f;
  }
  if (!TREE && row >= 0) S.store(a.out_state + row * a.o_rs + (int64_t)h * D * D + col0, g, q);
}

// ------------------------------------------------------------------ accepted path
// S' = gamma S + sum over the path of (decay after the node) k^ u^T.
template <int D>
__global__ void __launch_bounds__(Nodes<D, 2>::THREADS) gdn_accept_kernel(Args a) {
  using C = Nodes<D, 2>;
  constexpr int KST = C::KST, US = C::US, COLS = C::COLS, SL = D / COLS;
  __shared__ __align__(16) bf16 ks[16 * KST];
  __shared__ __align__(16) float us[16 * US];
  __shared__ float ik[16], cf[MAX_NODES];
  __shared__ int node[MAX_NODES], count;
  __shared__ float gamma;
  const int h = blockIdx.x / SL, cs = blockIdx.x % SL * COLS, s = blockIdx.y, hk = h / a.groups;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
  const int64_t row = state_row(a, s);
  if (row < 0) return;
  State<D> S;
  S.load(a.state + row * a.s_rs + (int64_t)h * D * D + cs + 16 * warp, g, q);
  if (warp == 0) {
    // nodes of the path in order, then the decay after each, from the last one back
    int m = 0;
    for (int j0 = 0; j0 < a.m; j0 += 32) {
      int t = j0 + lane < a.m ? a.path[(int64_t)s * a.m + j0 + lane] : -1;
      if (t < -1 || t >= a.T) {
        atomicExch(a.err, ERR_INDEX);
        t = -1;
      }
      const uint32_t on = __ballot_sync(0xffffffff, t >= 0);
      if (t >= 0) {
        const int at = m + __popc(on & ((1u << lane) - 1));
        node[at] = t;
        cf[at] = expf(a.g[s * a.g_bs + t * a.g_ts + h]);
      }
      m += __popc(on);
    }
    __syncwarp();
    if (lane == 0) {
      float d = 1.f;
      for (int j = m - 1; j >= 0; --j) {
        const float e = cf[j];
        cf[j] = d;
        d *= e;
      }
      gamma = d;
      count = m;
    }
  }
  __syncthreads();
  const int m = count;
  S.scale(gamma);
  for (int r0 = 0; r0 < m; r0 += 16) {
    if (r0 > 0) __syncthreads();
    constexpr int L = D / 8, LU = COLS / 4;
    for (int i = tid; i < 16 * L; i += C::THREADS) {  // key rows and their norms (L lanes a row)
      const int r = i / L, c = i % L;
      uint4 w = make_uint4(0, 0, 0, 0);
      if (r0 + r < m)
        w = *reinterpret_cast<const uint4*>(a.k + s * a.k_bs + node[r0 + r] * a.k_ts + hk * a.k_hs + c * 8);
      const uint32_t in[4] = {w.x, w.y, w.z, w.w};
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = __uint_as_float(in[e] << 16), y = __uint_as_float(in[e] & 0xffff0000u);
        ss = fmaf(x, x, fmaf(y, y, ss));
      }
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffff, ss, o);
      *reinterpret_cast<uint4*>(ks + r * KST + c * 8) = w;
      if (c == 0) ik[r] = rsqrtf(ss + 1e-6f);
    }
    __syncthreads();
    for (int i = tid; i < 16 * LU; i += C::THREADS) {
      const int r = i / LU, c = i % LU;
      float4 w = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r0 + r < m) {
        w = *reinterpret_cast<const float4*>(a.u_in + (((int64_t)s * a.T + node[r0 + r]) * a.nv + h) * D + cs + c * 4);
        const float f = ik[r];
        w = make_float4(w.x * f, w.y * f, w.z * f, w.w * f);
      }
      *reinterpret_cast<float4*>(us + r * US + c * 4) = w;
    }
    for (int r = m + tid; r < ((m + 15) & ~15); r += C::THREADS) cf[r] = 0.f;
    __syncthreads();
    S.template add<US, KST>(us + 16 * warp, cf + r0, ks, lane);
  }
  S.store(a.out_state + row * a.o_rs + (int64_t)h * D * D + cs + 16 * warp, g, q);
}

// ------------------------------------------------------------------ one token; short paths
// Plain loads and FMAs where a state's elements meet few nodes: a warp takes 32 value
// channels of a head on its own (lanes of a row group hold 4 channels each, a group D / GR key
// channels), so nothing but its own loads is waited for and 12 warps keep 190 KB an SM under way.
template <int D>
struct Slice {
  static constexpr int CW = D < 32 ? D : 32;   // value channels of a warp
  static constexpr int LR = CW / 4;            // lanes of one row
  static constexpr int GR = 32 / LR;           // row groups
  static constexpr int N = D / GR;             // key channels of a lane: [group N, group N + N)
  static constexpr int WARPS = 2;              // of a CTA
};

// D bf16 channels into fp32 shared memory by one warp; returns 1 / sqrt(|x|^2 + 1e-6).
template <int D>
__device__ __forceinline__ float warp_row(const bf16* x, float* dst, int lane) {
  float ss = 0.f;
#pragma unroll
  for (int i = lane * 2; i < D; i += 64) {
    const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(x + i));
    *reinterpret_cast<float2*>(dst + i) = f;
    ss = fmaf(f.x, f.x, fmaf(f.y, f.y, ss));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffff, ss, o);
  return rsqrtf(ss + 1e-6f);
}

template <int D>
__global__ void __launch_bounds__(Slice<D>::WARPS * 32) gdn_step_kernel(Args a, int slices) {
  using C = Slice<D>;
  constexpr int N = C::N;
  __shared__ __align__(16) float kq[C::WARPS][2][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int x = blockIdx.x * C::WARPS + warp;  // (head, slice)
  if (x >= slices) return;
  const int h = x / (D / C::CW), s = blockIdx.y, hk = h / a.groups;
  const int col = x % (D / C::CW) * C::CW + lane % C::LR * 4, k0 = lane / C::LR * N;
  const int64_t row = a.rows ? a.rows[s] : s;
  const bool valid = row >= 0 && row < a.n;
  if (!valid && row != -1 && lane == 0) atomicExch(a.err, ERR_INDEX);
  const int64_t at = (int64_t)h * D * D + (int64_t)k0 * D + col;
  float4 S[N];
  if (valid) {
    const float* st = a.state + row * a.s_rs + at;
#pragma unroll
    for (int i = 0; i < N; ++i) S[i] = *reinterpret_cast<const float4*>(st + i * D);
  }
  const int cnt = a.counts ? a.counts[s] : 1;
  if ((cnt < 0 || cnt > 1) && lane == 0) atomicExch(a.err, ERR_INDEX);
  const bool live = valid && cnt > 0;
  float o[4] = {};
  if (live) {
    const uint2 vr = *reinterpret_cast<const uint2*>(a.v + s * a.v_bs + h * a.v_hs + col);
    const float eg = expf(a.g[s * a.g_bs + h]), be = bf(a.beta[s * a.b_bs + h]);
    const float ik = warp_row<D>(a.k + s * a.k_bs + hk * a.k_hs, kq[warp][0], lane);
    const float iq = warp_row<D>(a.q + s * a.q_bs + hk * a.q_hs, kq[warp][1], lane) * rsqrtf((float)D);
    __syncwarp();
    const float* ks = kq[warp][0] + k0;
    const float* qs = kq[warp][1] + k0;
    float xk[4] = {}, xq[4] = {}, dot = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float k = ks[i], q = qs[i];
      xk[0] = fmaf(k, S[i].x, xk[0]), xk[1] = fmaf(k, S[i].y, xk[1]);
      xk[2] = fmaf(k, S[i].z, xk[2]), xk[3] = fmaf(k, S[i].w, xk[3]);
      xq[0] = fmaf(q, S[i].x, xq[0]), xq[1] = fmaf(q, S[i].y, xq[1]);
      xq[2] = fmaf(q, S[i].z, xq[2]), xq[3] = fmaf(q, S[i].w, xq[3]);
      dot = fmaf(k, q, dot);
    }
#pragma unroll
    for (int w = C::LR; w < 32; w <<= 1) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        xk[c] += __shfl_xor_sync(0xffffffff, xk[c], w);
        xq[c] += __shfl_xor_sync(0xffffffff, xq[c], w);
      }
      dot += __shfl_xor_sync(0xffffffff, dot, w);
    }
    const float v[4] = {__uint_as_float(vr.x << 16), __uint_as_float(vr.x & 0xffff0000u), __uint_as_float(vr.y << 16),
                        __uint_as_float(vr.y & 0xffff0000u)};
    float u[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      u[c] = be * (v[c] - eg * ik * xk[c]);
      o[c] = iq * fmaf(eg, xq[c], dot * ik * u[c]);
      u[c] *= ik;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float k = ks[i];
      S[i].x = fmaf(k, u[0], eg * S[i].x), S[i].y = fmaf(k, u[1], eg * S[i].y);
      S[i].z = fmaf(k, u[2], eg * S[i].z), S[i].w = fmaf(k, u[3], eg * S[i].w);
    }
  }
  if (lane < C::LR) {
    __nv_bfloat162 w[2] = {__floats2bfloat162_rn(o[0], o[1]), __floats2bfloat162_rn(o[2], o[3])};
    *reinterpret_cast<uint2*>(a.out + ((int64_t)s * a.nv + h) * D + col) = *reinterpret_cast<const uint2*>(w);
  }
  if (valid) {
    float* so = a.out_state + row * a.o_rs + at;
#pragma unroll
    for (int i = 0; i < N; ++i) *reinterpret_cast<float4*>(so + i * D) = S[i];
  }
}

// Up to here (of a batch's longest path) nodes one by one, beyond in blocks of 16 on tensor cores.
// Measured, 64 sequences (us, one by one and in blocks): paths of 1 to m nodes 70 and 91 at m =
// 4, 86 and 96 at 12, 96 and 98 at 16; all of m nodes 79 and 92 at 4, 99 and 95 at 8, 139 and 107 at 16.
constexpr int SHORT_PATH = 16;

template <int D>
__global__ void __launch_bounds__(Slice<D>::WARPS * 32) gdn_accept_short_kernel(Args a, int slices) {
  using C = Slice<D>;
  constexpr int N = C::N;
  __shared__ __align__(16) float kr[C::WARPS][2][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int x = blockIdx.x * C::WARPS + warp;
  if (x >= slices) return;
  const int h = x / (D / C::CW), s = blockIdx.y, hk = h / a.groups;
  const int col = x % (D / C::CW) * C::CW + lane % C::LR * 4, k0 = lane / C::LR * N;
  const int64_t row = a.rows ? a.rows[s] : s;
  if (row < 0 || row >= a.n) {
    if (row != -1 && lane == 0) atomicExch(a.err, ERR_INDEX);
    return;
  }
  const int64_t at = (int64_t)h * D * D + (int64_t)k0 * D + col;
  const float* st = a.state + row * a.s_rs + at;
  float4 S[N];
#pragma unroll
  for (int i = 0; i < N; ++i) S[i] = *reinterpret_cast<const float4*>(st + i * D);
  // lane j: node j of the path, its decay, and the product of the later ones
  int node = lane < a.m ? a.path[(int64_t)s * a.m + lane] : -1;
  if (node < -1 || node >= a.T) {
    atomicExch(a.err, ERR_INDEX);
    node = -1;
  }
  float after = node >= 0 ? expf(a.g[s * a.g_bs + node * a.g_ts + h]) : 1.f;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const float y = __shfl_down_sync(0xffffffff, after, o);
    if (lane + o < 32) after *= y;
  }
  const float gamma = __shfl_sync(0xffffffff, after, 0);
  after = __shfl_down_sync(0xffffffff, after, 1);  // (lane 31 is beyond a short path)
#pragma unroll
  for (int i = 0; i < N; ++i) S[i].x *= gamma, S[i].y *= gamma, S[i].z *= gamma, S[i].w *= gamma;
  uint32_t left = __ballot_sync(0xffffffff, node >= 0);
  for (int b = 0; left; b ^= 1, left &= left - 1) {
    const int j = __ffs(left) - 1, t = __shfl_sync(0xffffffff, node, j);
    const float f = __shfl_sync(0xffffffff, after, j);
    const float4 ur = *reinterpret_cast<const float4*>(a.u_in + (((int64_t)s * a.T + t) * a.nv + h) * D + col);
    const float w = warp_row<D>(a.k + s * a.k_bs + t * a.k_ts + hk * a.k_hs, kr[warp][b], lane) * f;
    __syncwarp();
    const float* ks = kr[warp][b] + k0;
    const float4 u = make_float4(ur.x * w, ur.y * w, ur.z * w, ur.w * w);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float k = ks[i];
      S[i].x = fmaf(k, u.x, S[i].x), S[i].y = fmaf(k, u.y, S[i].y);
      S[i].z = fmaf(k, u.z, S[i].z), S[i].w = fmaf(k, u.w, S[i].w);
    }
  }
  float* so = a.out_state + row * a.o_rs + at;
#pragma unroll
  for (int i = 0; i < N; ++i) *reinterpret_cast<float4*>(so + i * D) = S[i];
}

template <int D, int NT, bool TREE>
void launch_nodes(const Args& a, int64_t b) {
  using C = Nodes<D, NT>;
  static std::atomic<unsigned long long> attr{0};
  once_per_device(attr, [&] {
    NS_CUDA(cudaFuncSetAttribute(gdn_nodes_kernel<D, NT, TREE>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
  });
  gdn_nodes_kernel<D, NT, TREE><<<dim3((unsigned)(a.nv * (D / C::COLS)), (unsigned)b), C::THREADS, C::SMEM, stream()>>>(a);
}

// the fewest nodes per pass that hold T (chunks of 64 beyond)
template <int D>
dim3 slice_grid(int nv, int64_t b) {
  return dim3((unsigned)((nv * (D / Slice<D>::CW) + Slice<D>::WARPS - 1) / Slice<D>::WARPS), (unsigned)b);
}

template <int D, bool TREE>
void launch_for(const Args& a, int64_t b) {
  if (!TREE && a.T == 1)
    gdn_step_kernel<D><<<slice_grid<D>(a.nv, b), Slice<D>::WARPS * 32, 0, stream()>>>(a, a.nv * (D / Slice<D>::CW));
  else if (a.T <= 8)
    launch_nodes<D, 1, TREE>(a, b);
  else if (a.T <= 16)
    launch_nodes<D, 2, TREE>(a, b);
  else if (a.T <= 32)
    launch_nodes<D, 4, TREE>(a, b);
  else
    launch_nodes<D, 8, TREE>(a, b);
}

template <int D>
void launch_accept(const Args& a, int64_t b) {
  if (a.m <= SHORT_PATH)
    gdn_accept_short_kernel<D><<<slice_grid<D>(a.nv, b), Slice<D>::WARPS * 32, 0, stream()>>>(a, a.nv * (D / Slice<D>::CW));
  else
    gdn_accept_kernel<D><<<dim3((unsigned)(a.nv * (D / Nodes<D, 2>::COLS)), (unsigned)b), Nodes<D, 2>::THREADS, 0,
                           stream()>>>(a);
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

// No row of x (`row` fp32 each) shares memory with a row of y: their extents are apart, or rows of
// one stride interleave.
bool rows_apart(const at::Tensor& x, const at::Tensor& y, int64_t row) {
  const int64_t n = x.size(0), sx = x.stride(0), sy = y.stride(0), off = y.data_ptr<float>() - x.data_ptr<float>();
  if (n == 0 || off >= (n - 1) * sx + row || -off >= (n - 1) * sy + row) return true;
  if (n == 1 || sx != sy || sx < 2 * row) return false;
  const int64_t in = (off % sx + sx) % sx;
  return in >= row && in + row <= sx;
}

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
    // one CTA's rows must not be another's: out's own, and those of state unless it is state itself
    const int64_t row = d.nv * d.D * d.D, n = state.size(0);
    NS_VALUE(n <= 1 || out->stride(0) >= row, "gated delta rule: rows of out_state overlap");
    const bool same = out->data_ptr() == state.data_ptr() && (n <= 1 || out->stride(0) == state.stride(0));
    NS_VALUE(same || rows_apart(state, *out, row), "gated delta rule: out_state must be state or lie apart from it");
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
#define NS_X(DD) gdnd::launch_for<DD, false>(d.a, d.b);
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
#define NS_X(DD) gdnd::launch_for<DD, true>(d.a, d.b);
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
  NS_VALUE(d.T <= MAX_NODES && path.size(1) <= MAX_NODES, "gated_delta_accept: at most 64 nodes, and path entries");
  NS_VALUE(d.b < 65536 && d.nv < 65536, "gated delta rule: too many sequences or heads");
  bind_state(d, state, rows, &out_state);
  if (d.b * d.nv == 0) return;
  d.keep = {aligned_rows(k), g.stride(2) == 1 ? g : g.contiguous(), aligned_dense(u)};
  d.a.k = bf_ptr(d.keep[0]);
  d.a.k_bs = d.keep[0].stride(0), d.a.k_ts = d.keep[0].stride(1), d.a.k_hs = d.keep[0].stride(2);
  d.a.g = d.keep[1].data_ptr<float>();
  d.a.g_bs = d.keep[1].stride(0), d.a.g_ts = d.keep[1].stride(1);
  d.a.u_in = d.keep[2].data_ptr<float>();
  d.a.path = path.data_ptr<int>();
  d.a.T = (int)d.T, d.a.m = (int)path.size(1), d.a.nv = (int)d.nv, d.a.groups = (int)groups;
  d.a.err = device_error_flag();
#define NS_X(DD) gdnd::launch_accept<DD>(d.a, d.b);
  NS_GDN_CASES(d.D, NS_X)
#undef NS_X
  NS_CUDA(cudaGetLastError());
}

}  // namespace ns
