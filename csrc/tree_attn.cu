// Attention of a tree of drafted tokens over a paged cache (T = 1: plain decoding).
//
// For node t of a sequence with n cached rows and ancestor set A(t) (t included):
//   s_j = scale q_t.k_j over j in [0, n) of the cache and j in A(t) of the nodes' own k,
//   out_t = sum_j softmax(s)_j v_j  (times sigmoid(gate)),   lse_t = log sum_j e^{s_j}.
//
// The bytes of the cache bound it: each K/V byte serves the G = Hq / Hk heads of a group
// and all T nodes, so up to G T = 250 rows or so the tensor cores wait for HBM. So K/V is
// read once for 128 stacked rows (GT heads x TPM tokens) and one pass keeps the running
// maximum and sum:
//   S_j = Q K_j^T      M=128, N=64, K=D -> TMEM (two 64-column buffers)
//   O  += P_j V_j      M=128, N=D, K=64 -> TMEM, P_j read from TMEM
// over tiles of 64 keys: the tiles of the cached prefix, then one tile of the nodes' own
// keys whose mask is the row's ancestor set.
//
// Work is split over the long axis without knowing the lengths on the host: the tiles of
// all segments (sequence, key head, row tile) are numbered through, and CTA i of N (one per
// SM) takes tiles [U i / N, U (i+1) / N), so ragged batches and single long sequences load
// every SM alike. A segment that one CTA holds whole is finished there; parts of a segment
// leave unnormalised O with its reference maximum and sum in a workspace (two parts per CTA
// at most), and tree_join_kernel adds them up in the order of the CTAs.
//
// e4m3 pages: raw codes arrive by TMA, two converter warps turn them into f16 operand tiles
// (exact), and the rows' power-of-two scales stay outside the products: K's multiplies the
// score, V's the probability, relative to the largest V scale seen so far (when that
// grows by more than 2^4, O is rescaled like for a growing maximum). q rows are
// scaled by a power of two each so that f16 holds all of bf16's digits; the nodes' own
// rows are scaled the same way. Probabilities are f16 (11 bits) there. Against bf16 V they
// must be bf16, whose 8 bits would cost as much as the output's own rounding, so P is the
// sum of two bf16 matrices (16 bits) and P V two products: the tensor cores have the time.
//
// Rows of V beyond a sequence's end (stale pages, NaN) are zeroed in shared memory, since
// 0 * NaN would reach O; masked scores are replaced, not added to. Every mbarrier wait is
// bounded; a timeout sets the device error word and the kernel unwinds.
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "decode.h"
#include "sm100.cuh"

namespace ns {

using bf16 = __nv_bfloat16;

namespace tattn {

constexpr int EXP_BIAS = 127, EXP_MIN = -117, EXP_MAX = 118;
constexpr int BM = 128, BN = 64;
constexpr float RESCALE_LOG2 = 8.f;   // the reference maximum may lag by this much
constexpr int V_RESCALE = 4;          // and the reference V exponent by this much
constexpr float F16_OFFSET = 3.f;     // f16 probabilities are at most 2^(3 + 8 + 4)
constexpr int FAC = 4;                // scale buffers of the e4m3 form, see below
constexpr int CONV_WARPS = 4;

struct Args {
  const bf16 *q, *k, *v, *gate;
  int64_t q_bs, q_ts, q_hs, k_bs, k_ts, k_hs, v_bs, v_ts, v_hs, g_bs, g_ts, g_hs;
  const uint8_t *ke, *ve;
  const int *table, *lens, *parents, *counts;
  int64_t p_bs, pages, max_pages;
  int b, T, Hq, Hk, D, page;
  int G, GT, HB, TPM, M;  // heads of a group, per row tile, head blocks; tokens per row tile, token blocks
  float scale_log2;
  bf16* out;    // [b, T, Hq, D]
  float* lse;   // [b, Hq, T]
  float* part;  // [N][2][GT * TPM][D] unnormalised O
  float2* ml;   // [N][2][GT * TPM] reference maximum (log2) and sum
  int4* info;   // [segments] first CTA, last CTA, workspace slot of the first
  int* err;
};

__device__ __forceinline__ float bf(bf16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126..127

// Bounded wait: gives up after two seconds (a lost arrival), sets the error word.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, int* err) {
  if (sm100::mbar_try_wait(bar, parity)) return true;
  uint64_t t0, t1;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
  for (uint32_t i = 1; i < (1u << 26); ++i) {
    if (sm100::mbar_try_wait(bar, parity)) return true;
    if ((i & 63) == 0) {
      asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t1));
      if (t1 - t0 > 2000000000ull) break;
    }
  }
  atomicExch(err, 1);
  return false;
}

// ------------------------------------------------------------------ work split
struct Seq {
  int len, cnt;
};

__device__ __forceinline__ Seq sequence(const Args& a, int s, bool flag) {
  int len = a.lens[s], cnt = a.counts ? a.counts[s] : a.T;
  const int64_t most = a.max_pages * a.page;
  if (cnt < 0 || cnt > a.T || len < 0 || len > most) {
    if (flag) atomicExch(a.err, ERR_INDEX);
    cnt = min(max(cnt, 0), a.T);
    len = (int)min((int64_t)max(len, 0), most);
  }
  return {len, cnt};
}

// tiles of a row tile whose first token is live: the prefix and the nodes; one (of zeros) otherwise
__device__ __forceinline__ int64_t seq_units(const Args& a, Seq q) {
  const int live = (q.cnt + a.TPM - 1) / a.TPM;
  return (int64_t)a.Hk * a.HB * (live * ((q.len + BN - 1) / BN + 1) + (a.M - live));
}

// A contiguous run of tiles of one segment.
struct Piece {
  int s, hk, hb, m;       // sequence, key head, head block, token block
  Seq q;
  int nt;                 // prefix tiles of the segment (0 when no token is live)
  int t0, t1;             // tiles [t0, t1) of [0, nt]; tile nt is the nodes' own
  bool whole;
};

struct Walk {
  int s, seg, tile;       // next sequence, segment within it, tile within that
  int64_t unit, end;      // its global number; end of this CTA's run
  Seq q;
  __device__ __forceinline__ bool next(const Args& a, Piece& p) {
    if (unit >= end) return false;
    const int segs = a.Hk * a.HB * a.M;
    if (seg == segs) {
      seg = 0;
      q = sequence(a, ++s, false);
    }
    p.s = s;
    p.q = q;
    p.m = seg % a.M;
    p.hb = (seg / a.M) % a.HB;
    p.hk = seg / (a.M * a.HB);
    p.nt = p.m * a.TPM < q.cnt ? (q.len + BN - 1) / BN : 0;
    p.t0 = tile;
    p.t1 = (int)min((int64_t)p.nt + 1, tile + (end - unit));
    p.whole = p.t0 == 0 && p.t1 == p.nt + 1;
    unit += p.t1 - p.t0;
    tile = p.t1;
    if (tile == p.nt + 1) tile = 0, ++seg;
    return true;
  }
};

// First position and end of CTA blockIdx.x (warp-wide); total tiles in U, working CTAs in N
// (each has a tile at least).
__device__ __forceinline__ Walk plan(const Args& a, int lane, int64_t& U, int& N) {
  int64_t sum = 0;
  for (int s = lane; s < a.b; s += 32) sum += seq_units(a, sequence(a, s, blockIdx.x == 0));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffff, sum, o);
  U = sum;
  Walk w;
  N = (int)min((int64_t)gridDim.x, U);
  w.unit = U * min((int)blockIdx.x, N) / N;
  w.end = U * min((int)blockIdx.x + 1, N) / N;
  int64_t before = 0;
  w.s = a.b, w.seg = w.tile = 0, w.q = {0, 0};
  for (int s0 = 0; s0 < a.b; s0 += 32) {
    const int s = s0 + lane;
    const Seq q = s < a.b ? sequence(a, s, false) : Seq{0, 0};
    const int64_t n = s < a.b ? seq_units(a, q) : 0;
    int64_t inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffff, inc, o);
      if (lane >= o) inc += x;
    }
    const uint32_t hit = __ballot_sync(0xffffffff, before + inc > w.unit);
    if (hit) {
      const int l = __ffs(hit) - 1;
      int64_t rem = w.unit - before - __shfl_sync(0xffffffff, inc - n, l);
      w.s = s0 + l;
      w.q.len = __shfl_sync(0xffffffff, q.len, l);
      w.q.cnt = __shfl_sync(0xffffffff, q.cnt, l);
      const int live = (w.q.cnt + a.TPM - 1) / a.TPM;
      const int64_t tiles = (w.q.len + BN - 1) / BN + 1;
      const int64_t group = live * tiles + (a.M - live);  // one (key head, head block)
      w.seg = (int)(rem / group) * a.M;
      rem %= group;
      if (rem < live * tiles) {
        w.seg += (int)(rem / tiles);
        w.tile = (int)(rem % tiles);
      } else {
        w.seg += live + (int)(rem - live * tiles);
      }
      break;
    }
    before += __shfl_sync(0xffffffff, inc, 31);
  }
  return w;
}

// ------------------------------------------------------------------ shared memory
template <int DT, bool E4M3>
struct Cfg {
  static constexpr int DA = DT / 64;               // 128-byte swizzle atoms along D
  static constexpr int Q_BYTES = BM * DT * 2;
  static constexpr int SLOT = BN * DT * 2;         // one operand tile (K or V)
  static constexpr int NS = E4M3 ? 3 : (DT == 256 ? 4 : 8);
  static constexpr int RAW = BN * DT;              // one tile of codes
  static constexpr int NR = E4M3 ? (DT == 256 ? 3 : 8) : 0;
  static constexpr int FACS = E4M3 ? FAC * 2 * BN * 4 + FAC * 16 : 0;
  static constexpr int EXPS = NR * 2 * BN;
  static constexpr int SMEM = Q_BYTES + NS * SLOT + NR * RAW + FACS + EXPS + 512 + 1024;
  static constexpr int PP = E4M3 ? 1 : 2;          // matrices whose sum is P
  static constexpr int S_COL = DT, P_COL = DT + 2 * BN, P_COLS = PP * (BN / 2);
  static constexpr int TMEM_COLS = P_COL + 2 * P_COLS <= 256 ? 256 : 512;
  static constexpr int THREADS = 192 + (E4M3 ? CONV_WARPS * 32 : 0);
  // Scale buffer of tile n is reused by tile n + FAC, whose K enters ring slot
  // 2 (n + FAC) - 1; that slot is free once item 2 (n + FAC) - 1 - NS, at or after V of
  // tile n (item 2n + 2), was consumed, i.e. after tile n's probabilities were formed.
  static_assert(!E4M3 || 2 * FAC - 1 - NS >= 2, "scale buffers");
};

// Ring items of a piece of n tiles, in the order of the MMAs: K0, (K1, V0), (K2, V1), .., V(n-1).
// f(tile, is_v) returns false to stop.
template <class F>
__device__ __forceinline__ bool ring_order(int t0, int t1, F&& f) {
  if (!f(t0, false)) return false;
  for (int t = t0; t < t1; ++t) {
    if (t + 1 < t1 && !f(t + 1, false)) return false;
    if (!f(t, true)) return false;
  }
  return true;
}

// exponent that brings a row with largest magnitude bits `top` into [2^8, 2^9)
__device__ __forceinline__ int f16_exponent(uint32_t top) {
  return top == 0 ? EXP_MIN : max(min(max((int)(top >> 23), 1) - 127 - 8, EXP_MAX), EXP_MIN);
}

__device__ __forceinline__ uint32_t finite_top(uint32_t w) {  // of two packed bf16
  const uint32_t lo = (w << 16) & 0x7fffffffu, hi = w & 0x7fff0000u;
  return max(lo < 0x7f800000u ? lo : 0u, hi < 0x7f800000u ? hi : 0u);
}

__device__ __forceinline__ uint32_t scale_to_f16(uint32_t w, float s) {  // two packed bf16
  const __half2 h = __floats2half2_rn(__uint_as_float(w << 16) * s, __uint_as_float(w & 0xffff0000u) * s);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// offset of 16-byte chunk c (8 elements) of row r in a K-major 128-byte-swizzled tile of `rows` rows
__device__ __forceinline__ uint32_t tile_offset(int rows, int r, int c) {
  return (uint32_t)((c >> 3) * rows * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

template <int DT, bool E4M3>
__global__ void __launch_bounds__(Cfg<DT, E4M3>::THREADS, 1)
    tree_attn_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                     const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap tkp,
                     const __grid_constant__ CUtensorMap tvp, Args a) {
  using C = Cfg<DT, E4M3>;
  constexpr int DA = C::DA, NS = C::NS, NR = C::NR;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sQ = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sKV = sQ + C::Q_BYTES;
  uint8_t* sRaw = sKV + NS * C::SLOT;
  float* kfac = reinterpret_cast<float*>(sRaw + NR * C::RAW);    // [FAC][BN] 2^e of K rows
  float* vfac = kfac + (E4M3 ? FAC * BN : 0);                    // [FAC][BN] 2^(e - emax) of V rows
  int* vmax = reinterpret_cast<int*>(vfac + (E4M3 ? FAC * BN : 0));  // [FAC][4] emax of each tile
  uint8_t* sExp = reinterpret_cast<uint8_t*>(sRaw + NR * C::RAW + C::FACS);  // [NR][2][BN]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sExp + C::EXPS);
  uint64_t* full = bars;             // [NS] operand tile ready
  uint64_t* empty = full + NS;       // [NS]
  uint64_t* raw_full = empty + NS;   // [NR] codes landed
  uint64_t* raw_empty = raw_full + NR;
  uint64_t* fac_full = raw_empty + NR;  // [FAC] (e4m3)
  uint64_t* s_full = fac_full + (E4M3 ? FAC : 0);
  uint64_t* s_free = s_full + 2;
  uint64_t* p_full = s_free + 2;
  uint64_t* p_free = p_full + 2;
  uint64_t* q_full = p_free + 2;
  uint64_t* q_empty = q_full + 1;
  uint64_t* o_done = q_empty + 1;  // one completion per PV (rescales wait for the previous one)
  uint64_t* o_last = o_done + 1;   // one per piece, after its last PV
  uint64_t* o_free = o_last + 1;   // one per piece, O has been read
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_free + 1);
  static_assert(2 * NS + 2 * NR + FAC + 13 + 1 <= 64, "barrier area");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int64_t U;
  int N;
  Walk walk = plan(a, lane, U, N);  // every warp on its own: no shared state
  if (walk.unit >= walk.end) return;

  if (warp == 0 && lane == 0) {
    for (int i = 0; i < NS; ++i) {
      sm100::mbar_init(&full[i], E4M3 ? CONV_WARPS : 1);
      sm100::mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < NR; ++i) {
      sm100::mbar_init(&raw_full[i], 1);
      sm100::mbar_init(&raw_empty[i], CONV_WARPS);
    }
    for (int i = 0; i < (E4M3 ? FAC : 0); ++i) sm100::mbar_init(&fac_full[i], CONV_WARPS);
    for (int i = 0; i < 2; ++i) {
      sm100::mbar_init(&s_full[i], 1);
      sm100::mbar_init(&s_free[i], 4);
      sm100::mbar_init(&p_full[i], 4);
      sm100::mbar_init(&p_free[i], 1);
    }
    sm100::mbar_init(q_full, E4M3 ? 4 : 1);
    sm100::mbar_init(q_empty, 1);
    sm100::mbar_init(o_done, 1);
    sm100::mbar_init(o_last, 1);
    sm100::mbar_init(o_free, 4);
    sm100::fence_barrier_init();
    sm100::tma_prefetch_desc(&tkp);
    sm100::tma_prefetch_desc(&tvp);
  }
  if (warp == 1) {
    sm100::tmem_alloc(tmem_slot, C::TMEM_COLS);
    sm100::tmem_relinquish();
  }
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int br = min(a.page, BN);  // rows of one page that one copy brings

  // pool row of key `key` of a sequence (a page out of range is replaced by page 0)
  auto pool_row = [&](const Piece& p, int key) -> int {
    int pg = __ldg(a.table + p.s * a.max_pages + key / a.page);
    if (pg < 0 || pg >= a.pages) {
      atomicExch(a.err, ERR_INDEX);
      pg = 0;
    }
    return (pg * a.Hk + p.hk) * a.page + key % a.page;
  };

  Piece p;
  if (warp == 0) {
    // ---------------------------------------------------------- TMA producer
    if (lane == 0) {
      int it = 0, pc = 0;
      bool ok = true;
      while (ok && walk.next(a, p)) {
        if constexpr (!E4M3) {
          if (pc > 0 && !(ok = wait(q_empty, (pc - 1) & 1, a.err))) break;
          sm100::mbar_expect_tx(q_full, DA * a.GT * a.TPM * 128);
#pragma unroll
          for (int j = 0; j < DA; ++j)
            sm100::tma_load_4d(sQ + j * (BM * 128), &tq, q_full, 64 * j, p.hk * a.G + p.hb * a.GT, p.m * a.TPM, p.s);
          ++pc;
        }
        ok = ring_order(p.t0, p.t1, [&](int t, bool is_v) -> bool {
          constexpr int R = E4M3 ? NR : NS;
          const int st = it % R, use = it / R;
          uint64_t* fb = E4M3 ? &raw_full[st] : &full[st];
          if (t == p.nt) {  // the nodes' own rows (the e4m3 form reads them in the converters)
            if constexpr (!E4M3) {
              if (use > 0 && !wait(&empty[st], (use - 1) & 1, a.err)) return false;
              uint8_t* d = sKV + st * C::SLOT;
              sm100::mbar_expect_tx(fb, DA * a.T * 128);
#pragma unroll
              for (int j = 0; j < DA; ++j)
                sm100::tma_load_4d(d + j * (BN * 128), is_v ? &tv : &tk, fb, 64 * j, p.hk, 0, p.s);
              ++it;
            }
            return true;
          }
          if (use > 0 && !wait(E4M3 ? &raw_empty[st] : &empty[st], (use - 1) & 1, a.err)) return false;
          const int k0 = t * BN, n = min(BN, p.q.len - k0), runs = (n + br - 1) / br;
          if constexpr (E4M3) {
            uint8_t* d = sRaw + st * C::RAW;
            sm100::mbar_expect_tx(fb, runs * br * (DA * 64 + (is_v ? 0 : 2)));
            for (int r = 0; r < runs; ++r) {
              const int row = pool_row(p, k0 + r * br);
#pragma unroll
              for (int j = 0; j < DA; ++j)
                sm100::tma_load_2d(d + j * (BN * 64) + r * br * 64, is_v ? &tvp : &tkp, fb, 64 * j, row);
              if (!is_v) {
                sm100::bulk_load(sExp + (st * 2) * BN + r * br, a.ke + row, br, fb);
                sm100::bulk_load(sExp + (st * 2 + 1) * BN + r * br, a.ve + row, br, fb);
              }
            }
          } else {
            uint8_t* d = sKV + st * C::SLOT;
            sm100::mbar_expect_tx(fb, runs * br * DA * 128);
            for (int r = 0; r < runs; ++r) {
              const int row = pool_row(p, k0 + r * br);
#pragma unroll
              for (int j = 0; j < DA; ++j)
                sm100::tma_load_2d(d + j * (BN * 128) + r * br * 128, is_v ? &tvp : &tkp, fb, 64 * j, row);
            }
          }
          ++it;
          return true;
        });
      }
      // drain: every issued copy has landed before the CTA may exit
      constexpr int R = E4M3 ? NR : NS;
      if (!E4M3 && pc > 0) wait(q_full, (pc - 1) & 1, a.err);
      for (int i = max(0, it - R); i < it; ++i)
        wait(E4M3 ? &raw_full[i % R] : &full[i % R], (i / R) & 1, a.err);
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------- MMA issuer
    constexpr uint32_t idesc_s = E4M3 ? sm100::idesc_f16(BM, BN, false, false) : sm100::idesc_bf16(BM, BN, false, false);
    constexpr uint32_t idesc_o = E4M3 ? sm100::idesc_f16(BM, DT, false, true) : sm100::idesc_bf16(BM, DT, false, true);
    const uint32_t q_base = sm100::smem_u32(sQ);
    int it = 0, n = 0, ns = 0, pc = 0;  // ring item, PV tile, S tile, piece
    bool ok = true;
    while (ok && walk.next(a, p)) {
      ok = wait(q_full, pc & 1, a.err);
      ok = ok && ring_order(p.t0, p.t1, [&](int t, bool is_v) -> bool {
        const int st = it % NS;
        if (!wait(&full[st], (it / NS) & 1, a.err)) return false;
        uint8_t* tile = sKV + st * C::SLOT;
        const uint32_t base = sm100::smem_u32(tile);
        if (!is_v) {
          const int sb = ns & 1;
          if (ns >= 2 && !wait(&s_free[sb], ((ns >> 1) - 1) & 1, a.err)) return false;
          sm100::tc_fence_after();
          if (lane == 0) {
#pragma unroll
            for (int kk = 0; kk < DT / 16; ++kk) {
              const uint64_t ad = sm100::smem_desc_sw128(q_base + (kk >> 2) * (BM * 128) + (kk & 3) * 32, 0, 1024);
              const uint64_t bd = sm100::smem_desc_sw128(base + (kk >> 2) * (BN * 128) + (kk & 3) * 32, 0, 1024);
              sm100::mma_bf16(tmem + C::S_COL + sb * BN, ad, bd, idesc_s, kk > 0 ? 1u : 0u);
            }
            sm100::mma_commit(&s_full[sb]);
            sm100::mma_commit(&empty[st]);
            if (t == p.t1 - 1) sm100::mma_commit(q_empty);
          }
          __syncwarp();
          ++ns;
        } else {
          if constexpr (!E4M3) {  // rows of V beyond the end: stale or another sequence's
            const int live = t == p.nt ? p.q.cnt : min(BN, p.q.len - t * BN);
            if (live < BN) {
              for (int i = lane; i < (BN - live) * 8 * DA; i += 32) {
                const int r = live + i / (8 * DA), c = i % (8 * DA);
                *reinterpret_cast<uint4*>(tile + tile_offset(BN, r, c)) = make_uint4(0, 0, 0, 0);
              }
              sm100::fence_proxy_async_smem();
              __syncwarp();
            }
          }
          const int pb = n & 1;
          if (!wait(&p_full[pb], (n >> 1) & 1, a.err)) return false;
          if (t == p.t0 && pc > 0 && !wait(o_free, (pc - 1) & 1, a.err)) return false;
          sm100::tc_fence_after();
          if (lane == 0) {
#pragma unroll
            for (int kk = 0; kk < C::PP * (BN / 16); ++kk) {
              const uint64_t bd = sm100::smem_desc_sw128(base + (kk % (BN / 16)) * 2048, BN * 128, 1024);
              sm100::mma_f16_ts(tmem, tmem + C::P_COL + pb * C::P_COLS + kk * 8, bd, idesc_o,
                                (t > p.t0 || kk > 0) ? 1u : 0u);
            }
            sm100::mma_commit(o_done);
            if (t == p.t1 - 1) sm100::mma_commit(o_last);
            sm100::mma_commit(&p_free[pb]);
            sm100::mma_commit(&empty[st]);
          }
          __syncwarp();
          ++n;
        }
        ++it;
        return true;
      });
      ++pc;
    }
  } else if (warp < 6) {
    // ---------------------------------------------------------- softmax warps, one row per thread
    const int qw = warp & 3;  // TMEM lane quarter of this warp
    const int row = qw * 32 + lane;
    const uint32_t lane_off = (uint32_t)(qw * 32) << 16;
    const int rows = a.GT * a.TPM;
    const bool warp_on = qw * 32 < rows;
    int n = 0, pc = 0;
    bool ok = true;
    while (ok && walk.next(a, p)) {
      const int tok = p.m * a.TPM + row / a.GT, g = p.hb * a.GT + row % a.GT;
      const bool in = row < rows && g < a.G && tok < a.T;
      const bool live = in && tok < p.q.cnt;
      const int hq = p.hk * a.G + g;
      float rs = a.scale_log2;  // multiplies the products of this row
      if constexpr (E4M3) {
        // q row -> f16 with a power-of-two scale, into the operand tile (the previous piece's
        // products are complete: this thread has seen all of its scores)
        if (live) {
          const bf16* q = a.q + p.s * a.q_bs + tok * a.q_ts + hq * a.q_hs;
          uint32_t top = 0;
          for (int c = 0; c < a.D / 8; ++c) {
            const uint4 w = *reinterpret_cast<const uint4*>(q + c * 8);
            top = max(max(max(top, finite_top(w.x)), max(finite_top(w.y), finite_top(w.z))), finite_top(w.w));
          }
          const int e = f16_exponent(top);
          const float s = pow2(-e);
          rs *= pow2(e);
          for (int c = 0; c < DT / 8; ++c) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (c * 8 < a.D) {
              w = *reinterpret_cast<const uint4*>(q + c * 8);
              w = make_uint4(scale_to_f16(w.x, s), scale_to_f16(w.y, s), scale_to_f16(w.z, s), scale_to_f16(w.w, s));
            }
            *reinterpret_cast<uint4*>(sQ + tile_offset(BM, row, c)) = w;
          }
        }
        sm100::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive(q_full);
      }
      // ancestors of this row's node
      uint64_t anc = 0;
      if (live && p.t1 == p.nt + 1) {
        for (int i = tok; i >= 0;) {
          anc |= 1ull << i;
          int up = a.parents[p.s * a.p_bs + i];
          if (up < -1 || up >= i) {
            atomicExch(a.err, ERR_INDEX);
            up = -1;
          }
          i = up;
        }
      }
      float m = -INFINITY, l = 0.f;  // reference maximum (log2) and sum
      int ev = 0;                    // reference exponent of V (e4m3)
      for (int t = p.t0; t < p.t1; ++t, ++n) {
        const int sb = n & 1;
        const uint64_t mask = !live ? 0ull
                              : t == p.nt ? anc
                              : p.q.len - t * BN >= BN ? ~0ull
                                                       : (1ull << (p.q.len - t * BN)) - 1;
        ok = __all_sync(0xffffffff, wait(&s_full[sb], (n >> 1) & 1, a.err));
        if (E4M3 && ok) ok = __all_sync(0xffffffff, wait(&fac_full[n % FAC], (n / FAC) & 1, a.err));
        if (!ok) break;
        sm100::tc_fence_after();
        const float* kf = kfac + (n % FAC) * BN;
        const float* vf = vfac + (n % FAC) * BN;
        float x[BN];
        if (warp_on) {
          float tmp[32];
#pragma unroll
          for (int hlf = 0; hlf < 2; ++hlf) {
            sm100::tmem_ld32(tmem + lane_off + C::S_COL + sb * BN + hlf * 32, tmp);
#pragma unroll
            for (int c = 0; c < 32; ++c) x[hlf * 32 + c] = tmp[c];
          }
        }
        sm100::tc_fence_before();
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive(&s_free[sb]);
        float alpha = 1.f, alpha_o = 1.f;
        bool grow = false;
        uint32_t pk[BN / 2];
        if (warp_on) {
          float mt = -INFINITY;
#pragma unroll
          for (int c = 0; c < BN; ++c) x[c] = E4M3 ? x[c] * (rs * kf[c]) : x[c] * rs;
          if (mask != ~0ull) {
#pragma unroll
            for (int c = 0; c < BN; ++c)
              if (!((mask >> c) & 1)) x[c] = -INFINITY;
          }
#pragma unroll
          for (int c = 0; c < BN; ++c) mt = fmaxf(mt, x[c]);
          const float top = E4M3 ? mt - F16_OFFSET : mt;
          if (top > m + RESCALE_LOG2) {
            alpha = alpha_o = sm100::exp2_approx(m - top);  // 0 on the first tile
            m = top;
            grow = true;
          }
          const float ref = m == -INFINITY ? 0.f : m;
          float vs = 1.f;
          if constexpr (E4M3) {
            const int e = vmax[(n % FAC) * 4];
            if (t == p.t0) ev = e;
            if (e > ev + V_RESCALE) {
              alpha_o *= pow2(max(ev - e, -126));
              ev = e;
              grow = true;
            }
            vs = pow2(max(e - ev, -126));
          }
          float ps = 0.f;
#pragma unroll
          for (int c = 0; c < BN; c += 2) {
            const float p0 = sm100::exp2_approx(x[c] - ref), p1 = sm100::exp2_approx(x[c + 1] - ref);
            ps += p0 + p1;
            x[c] = p0, x[c + 1] = p1;
            if constexpr (E4M3) {
              const __half2 h2 = __floats2half2_rn(p0 * (vs * vf[c]), p1 * (vs * vf[c + 1]));
              pk[c / 2] = *reinterpret_cast<const uint32_t*>(&h2);
            } else {
              const __nv_bfloat162 h2 = __floats2bfloat162_rn(p0, p1);
              pk[c / 2] = *reinterpret_cast<const uint32_t*>(&h2);
            }
          }
          l = l * alpha + ps;
        }
        // the P buffer is free once PV of tile n - 2 completed
        if (n >= 2) {
          ok = __all_sync(0xffffffff, wait(&p_free[sb], ((n >> 1) - 1) & 1, a.err));
          if (!ok) break;
        }
        // rescale O rows once the previous PV completed (warp-wide, rare after the first tiles)
        if (__any_sync(0xffffffff, grow && t > p.t0)) {
          ok = __all_sync(0xffffffff, wait(o_done, (n - 1) & 1, a.err));
          if (!ok) break;
          sm100::tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < DT; c += 32) {
            float o[32];
            sm100::tmem_ld32(tmem + lane_off + c, o);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] *= alpha_o;
            sm100::tmem_st32(tmem + lane_off + c, o);
          }
        }
        if (warp_on) {
          float f[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(pk[i]);
          sm100::tmem_st32(tmem + lane_off + C::P_COL + sb * C::P_COLS, f);
          if constexpr (!E4M3) {  // what the first rounding left
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const __nv_bfloat162 h2 = __floats2bfloat162_rn(x[2 * i] - __uint_as_float(pk[i] << 16),
                                                              x[2 * i + 1] - __uint_as_float(pk[i] & 0xffff0000u));
              f[i] = __uint_as_float(*reinterpret_cast<const uint32_t*>(&h2));
            }
            sm100::tmem_st32(tmem + lane_off + C::P_COL + sb * C::P_COLS + BN / 2, f);
          }
        }
        sm100::tc_fence_before();
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive(&p_full[sb]);
      }
      if (!ok) break;
      ok = __all_sync(0xffffffff, wait(o_last, pc & 1, a.err));
      if (!ok) break;
      sm100::tc_fence_after();
      if (warp_on) {
        // O -> the output (a whole segment) or the workspace
        const float vs = E4M3 ? pow2(ev) : 1.f;
        const float inv = l > 0.f ? vs / l : (l == 0.f ? 0.f : l);
        // the piece a CTA begins in the middle of its run starts a segment and ends the run
        const int slot = p.t0 == 0 && walk.end - (p.t1 - p.t0) != U * blockIdx.x / N ? 1 : 0;
        const int64_t at = ((int64_t)blockIdx.x * 2 + slot) * rows + row;
        bf16* o = a.out + (((int64_t)p.s * a.T + tok) * a.Hq + hq) * a.D;
        const bf16* gt = a.gate ? a.gate + p.s * a.g_bs + tok * a.g_ts + hq * a.g_hs : nullptr;
#pragma unroll 1
        for (int c = 0; c < DT; c += 32) {
          float v[32];
          sm100::tmem_ld32(tmem + lane_off + c, v);
          if (!in) continue;
          if (p.whole) {
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
              if (c + i < a.D) {
                uint32_t w[4], gw[4] = {0, 0, 0, 0};
                if (gt && live) *reinterpret_cast<uint4*>(gw) = *reinterpret_cast<const uint4*>(gt + c + i);
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                  float o0 = v[i + j] * inv, o1 = v[i + j + 1] * inv;
                  if (gt) {
                    o0 /= 1.f + __expf(-__uint_as_float(gw[j / 2] << 16));
                    o1 /= 1.f + __expf(-__uint_as_float(gw[j / 2] & 0xffff0000u));
                  }
                  const __nv_bfloat162 h2 = __floats2bfloat162_rn(live ? o0 : 0.f, live ? o1 : 0.f);
                  w[j / 2] = *reinterpret_cast<const uint32_t*>(&h2);
                }
                *reinterpret_cast<uint4*>(o + c + i) = *reinterpret_cast<uint4*>(w);
              }
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              if (c + i < a.D)
                *reinterpret_cast<float4*>(a.part + at * a.D + c + i) =
                    live ? make_float4(v[i] * vs, v[i + 1] * vs, v[i + 2] * vs, v[i + 3] * vs)
                         : make_float4(0.f, 0.f, 0.f, 0.f);
          }
        }
        if (in) {
          if (p.whole)
            a.lse[((int64_t)p.s * a.Hq + hq) * a.T + tok] =
                live ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
          else
            a.ml[at] = make_float2(m, l);
        }
        if (row == 0 && p.t0 == 0) {  // where the segment's parts are
          const int64_t first = walk.unit - (p.t1 - p.t0), last = first + p.nt;
          const int c1 = (int)(((last + 1) * N - 1) / U);
          a.info[(((int64_t)p.s * a.Hk + p.hk) * a.HB + p.hb) * a.M + p.m] = make_int4(blockIdx.x, c1, slot, 0);
        }
      }
      sm100::tc_fence_before();
      __syncwarp();
      if (lane == 0) sm100::mbar_arrive(o_free);
      ++pc;
    }
  } else if constexpr (E4M3) {
    // ---------------------------------------------------------- converters: codes -> f16 operand tiles
    const int cw = warp - 6;
    const int r8 = lane >> 2, q4 = lane & 3;  // row of 8, 16 codes of 64
    int it = 0, ri = 0, n = 0;
    bool ok = true;
    while (ok && walk.next(a, p)) {
      ok = ring_order(p.t0, p.t1, [&](int t, bool is_v) -> bool {
        const int st = it % NS, use = it / NS;
        const bool own = t == p.nt;
        const int live = own ? p.q.cnt : min(BN, p.q.len - t * BN);
        const int rst = ri % max(NR, 1);
        if (!own && !wait(&raw_full[rst], (ri / max(NR, 1)) & 1, a.err)) return false;
        if (use > 0 && !wait(&empty[st], (use - 1) & 1, a.err)) return false;
        uint8_t* tile = sKV + st * C::SLOT;
        const int fb = n % FAC;
        if (own) {
          // one row per warp pass: exponent from its largest magnitude, then scaled to f16
          const bf16* src = is_v ? a.v + p.s * a.v_bs + p.hk * a.v_hs : a.k + p.s * a.k_bs + p.hk * a.k_hs;
          const int64_t ts = is_v ? a.v_ts : a.k_ts;
          auto row_exp = [&](const bf16* x, uint4& w) {
            w = make_uint4(0, 0, 0, 0);
            if (lane * 8 < a.D) w = *reinterpret_cast<const uint4*>(x + lane * 8);
            uint32_t top = max(max(finite_top(w.x), finite_top(w.y)), max(finite_top(w.z), finite_top(w.w)));
            return f16_exponent(__reduce_max_sync(0xffffffff, top));
          };
          for (int r = cw; r < BN; r += CONV_WARPS) {
            uint4 w = make_uint4(0, 0, 0, 0);
            int e = EXP_MIN;
            if (r < live) {
              e = row_exp(src + r * ts, w);
              const float s = pow2(-e);
              w = make_uint4(scale_to_f16(w.x, s), scale_to_f16(w.y, s), scale_to_f16(w.z, s), scale_to_f16(w.w, s));
            }
            if (lane < DT / 8) *reinterpret_cast<uint4*>(tile + tile_offset(BN, r, lane)) = w;
            if (!is_v && lane == 0) kfac[fb * BN + r] = pow2(e);
          }
          if (!is_v) {  // V's scales: every warp finds the largest, then writes its own rows
            int top = EXP_MIN, mine = EXP_MIN;
            uint4 w;
            for (int r = 0; r < live; ++r) {
              const int e = row_exp(a.v + p.s * a.v_bs + p.hk * a.v_hs + r * a.v_ts, w);
              top = max(top, e);
              if (r % CONV_WARPS == cw && r / CONV_WARPS == lane) mine = e;
            }
            const int r = lane * CONV_WARPS + cw;
            if (r < BN) vfac[fb * BN + r] = r < live ? pow2(max(mine - top, -126)) : 0.f;
            if (cw == 0 && lane == 0) vmax[fb * 4] = top;
          }
        } else {
          const uint8_t* raw = sRaw + rst * C::RAW;
          for (int i = cw; i < DA * (BN / 8); i += CONV_WARPS) {
            const int j = i / (BN / 8), r = (i % (BN / 8)) * 8 + r8;
            uint4 w = make_uint4(0, 0, 0, 0);
            if (r < live) w = *reinterpret_cast<const uint4*>(raw + j * (BN * 64) + r * 64 + q4 * 16);
            const uint32_t in[4] = {w.x, w.y, w.z, w.w};
            uint32_t h[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) {
              const __half2_raw hr =
                  __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)((in[x / 2] >> (16 * (x & 1))) & 0xffff), __NV_E4M3);
              h[x] = (uint32_t)hr.x | ((uint32_t)hr.y << 16);
            }
            const int c = j * 8 + q4 * 2;
            *reinterpret_cast<uint4*>(tile + tile_offset(BN, r, c)) = make_uint4(h[0], h[1], h[2], h[3]);
            *reinterpret_cast<uint4*>(tile + tile_offset(BN, r, c + 1)) = make_uint4(h[4], h[5], h[6], h[7]);
          }
          if (!is_v && cw == 0) {  // this tile's scales, two rows per lane
            const uint8_t* ex = sExp + rst * 2 * BN;
            int e[2], top = EXP_MIN;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int r = lane + 32 * i;
              kfac[fb * BN + r] = r < live ? pow2(min(max((int)ex[r] - EXP_BIAS, EXP_MIN), EXP_MAX)) : 0.f;
              e[i] = min(max((int)ex[BN + r] - EXP_BIAS, EXP_MIN), EXP_MAX);
              if (r < live) top = max(top, e[i]);
            }
            top = __reduce_max_sync(0xffffffff, top);
#pragma unroll
            for (int i = 0; i < 2; ++i)
              vfac[fb * BN + lane + 32 * i] = lane + 32 * i < live ? pow2(max(e[i] - top, -126)) : 0.f;
            if (lane == 0) vmax[fb * 4] = top;
          }
        }
        sm100::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          sm100::mbar_arrive(&full[st]);
          if (!own) sm100::mbar_arrive(&raw_empty[rst]);
          if (!is_v) sm100::mbar_arrive(&fac_full[fb]);
        }
        if (!own) ++ri;
        if (!is_v) ++n;
        ++it;
        return true;
      });
    }
  }
  sm100::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    sm100::tc_fence_after();
    sm100::tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

// ------------------------------------------------------------------ joining parts
// One warp per (sequence, token, query head): rows of segments that lie in one CTA are done;
// the others add their parts in the order of the CTAs.
__global__ void __launch_bounds__(256) tree_join_kernel(Args a) {
  const int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (i >= (int64_t)a.b * a.T * a.Hq) return;
  const int hq = (int)(i % a.Hq), tok = (int)((i / a.Hq) % a.T), s = (int)(i / ((int64_t)a.Hq * a.T));
  const int hk = hq / a.G, g = hq % a.G, hb = g / a.GT, m = tok / a.TPM;
  const int4 inf = a.info[(((int64_t)s * a.Hk + hk) * a.HB + hb) * a.M + m];
  if (inf.x == inf.y) return;
  const int rows = a.GT * a.TPM, row = (tok - m * a.TPM) * a.GT + g - hb * a.GT;
  float top = -INFINITY;
  for (int c = inf.x; c <= inf.y; ++c)
    top = fmaxf(top, a.ml[((int64_t)c * 2 + (c == inf.x ? inf.z : 0)) * rows + row].x);
  float l = 0.f, o[8] = {};
  const bool on = lane * 8 < a.D;
  for (int c = inf.x; c <= inf.y; ++c) {
    const int64_t at = ((int64_t)c * 2 + (c == inf.x ? inf.z : 0)) * rows + row;
    const float2 ml = a.ml[at];
    const float w = ml.x == -INFINITY ? 0.f : sm100::exp2_approx(ml.x - top);
    l += w * ml.y;
    if (on) {
      const float4 u = *reinterpret_cast<const float4*>(a.part + at * a.D + lane * 8);
      const float4 v = *reinterpret_cast<const float4*>(a.part + at * a.D + lane * 8 + 4);
      o[0] += w * u.x, o[1] += w * u.y, o[2] += w * u.z, o[3] += w * u.w;
      o[4] += w * v.x, o[5] += w * v.y, o[6] += w * v.z, o[7] += w * v.w;
    }
  }
  const bool live = tok < sequence(a, s, false).cnt;
  const float inv = live ? 1.f / l : 0.f;
  if (on) {
    uint32_t gw[4] = {0, 0, 0, 0}, w[4];
    if (a.gate && live)
      *reinterpret_cast<uint4*>(gw) =
          *reinterpret_cast<const uint4*>(a.gate + s * a.g_bs + tok * a.g_ts + hq * a.g_hs + lane * 8);
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      float o0 = live ? o[j] * inv : 0.f, o1 = live ? o[j + 1] * inv : 0.f;
      if (a.gate) {
        o0 /= 1.f + __expf(-__uint_as_float(gw[j / 2] << 16));
        o1 /= 1.f + __expf(-__uint_as_float(gw[j / 2] & 0xffff0000u));
      }
      const __nv_bfloat162 h2 = __floats2bfloat162_rn(o0, o1);
      w[j / 2] = *reinterpret_cast<const uint32_t*>(&h2);
    }
    *reinterpret_cast<uint4*>(a.out + i * a.D + lane * 8) = *reinterpret_cast<uint4*>(w);
  }
  if (lane == 0)
    a.lse[((int64_t)s * a.Hq + hq) * a.T + tok] = live ? (top + log2f(l)) * 0.6931471805599453f : -INFINITY;
}

// ------------------------------------------------------------------ host
// Tensor map over [b][T][heads][D] bf16 rows, box 64 x heads x tokens x 1, 128-byte swizzle.
CUtensorMap node_map(const at::Tensor& x, int heads, int tokens) {
  CUtensorMap map;
  cuuint64_t dims[4], strides[3];
  for (int i = 0; i < 4; ++i) dims[i] = (cuuint64_t)x.size(3 - i);
  for (int i = 0; i < 3; ++i)  // the stride of a dimension of one is never used
    strides[i] = x.size(2 - i) == 1 ? 16 : (cuuint64_t)x.stride(2 - i) * 2;
  cuuint32_t box[4] = {64, (cuuint32_t)heads, (cuuint32_t)tokens, 1}, estr[4] = {1, 1, 1, 1};
  CUresult r = encode_fn()(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, x.data_ptr(), dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  NS_CHECK(r == CUDA_SUCCESS, "tree_attention: cuTensorMapEncodeTiled failed");
  return map;
}

// Tensor map over the pages as [rows][D]: 64 channels x `rows` box; codes unswizzled.
CUtensorMap pool_map(const void* base, const CacheView& c, int rows) {
  const int64_t n = c.pages * c.heads * c.page;
  if (!c.e4m3) return make_tmap_bf16(base, n, c.d, c.d, rows, 64);
  CUtensorMap map;
  cuuint64_t dims[2] = {(cuuint64_t)c.d, (cuuint64_t)n}, strides[1] = {(cuuint64_t)c.d};
  cuuint32_t box[2] = {64, (cuuint32_t)rows}, estr[2] = {1, 1};
  CUresult r = encode_fn()(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  NS_CHECK(r == CUDA_SUCCESS, "tree_attention: cuTensorMapEncodeTiled failed");
  return map;
}

template <int DT, bool E4M3>
void launch(const Args& a, int grid, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
            const CUtensorMap& tkp, const CUtensorMap& tvp) {
  using C = Cfg<DT, E4M3>;
  static_assert(C::SMEM <= 232448, "shared memory");
  static std::atomic<unsigned long long> attr{0};
  once_per_device(attr, [&] {
    NS_CUDA(cudaFuncSetAttribute(tree_attn_kernel<DT, E4M3>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
  });
  tree_attn_kernel<DT, E4M3><<<grid, C::THREADS, C::SMEM, stream()>>>(tq, tk, tv, tkp, tvp, a);
  NS_CUDA(cudaGetLastError());
}

// A node operand as TMA can read it: aligned rows, no broadcast dimension.
at::Tensor node_rows(const at::Tensor& t) {
  for (int i = 0; i + 1 < t.dim(); ++i)
    if (t.size(i) > 1 && t.stride(i) == 0) return t.contiguous();
  return aligned_rows(t);
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
  NS_VALUE(c.pages >= 1, "tree_attention: the cache has no pages");
  NS_VALUE(!gate.has_value() || (gate->sizes() == q.sizes() && gate->scalar_type() == at::kBFloat16 &&
                                 gate->device() == dev),
           "tree_attention: gate must be bfloat16 with q's shape");
  NS_VALUE(!scale.has_value() || *scale > 0, "tree_attention: scale must be positive");
  NS_VALUE(b < (1 << 20) && Hq < (1 << 16), "tree_attention: too many sequences or heads");
  NS_VALUE(table.device() == dev && table.scalar_type() == at::kInt && table.dim() == 2 && table.size(0) == b &&
               table.is_contiguous(),
           "table must be contiguous int32 [b, max_pages]");
  NS_VALUE(table.size(1) * c.page < (int64_t(1) << 31), "tree_attention: sequences of more than 2^31 rows");
  tattn::Args a{};
  a.lens = check_index(lens, b, dev, "lens");
  a.counts = check_index(counts, b, dev, "counts");
  a.parents = check_parents(parents, b, T, dev, a.p_bs);
  at::Tensor out = at::empty({b, T, Hq, D}, q.options());
  at::Tensor lse = at::empty({b, Hq, T}, q.options().dtype(at::kFloat));
  if (b == 0) return {out, lse};
  q = tattn::node_rows(q);
  k = tattn::node_rows(k);
  v = tattn::node_rows(v);
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
  a.ke = c.ke, a.ve = c.ve;
  a.table = table.data_ptr<int>();
  a.pages = c.pages, a.max_pages = table.size(1);
  a.b = (int)b, a.T = (int)T, a.Hq = (int)Hq, a.Hk = c.heads, a.D = (int)D, a.page = c.page;
  a.G = (int)Hq / c.heads;
  a.HB = (a.G + tattn::BM - 1) / tattn::BM;
  a.GT = (a.G + a.HB - 1) / a.HB;
  a.TPM = std::min((int)T, tattn::BM / a.GT);
  a.M = ((int)T + a.TPM - 1) / a.TPM;
  a.scale_log2 = (float)(scale.value_or(1.0 / std::sqrt((double)D)) * 1.4426950408889634);
  a.out = reinterpret_cast<bf16*>(out.data_ptr());
  a.lse = lse.data_ptr<float>();
  a.err = device_error_flag();
  const int grid = num_sms();
  // workspace: parts [grid][2][rows][D], their (maximum, sum), and the segments' whereabouts
  const int64_t rows = (int64_t)a.GT * a.TPM, segs = b * a.Hk * a.HB * a.M;
  const int64_t n_part = 2 * grid * rows * D, n_ml = 2 * 2 * grid * rows;
  at::Tensor ws = at::empty({n_part + ((n_ml + 3) & ~int64_t(3)) + 4 * segs}, lse.options());
  a.part = ws.data_ptr<float>();
  a.ml = reinterpret_cast<float2*>(a.part + n_part);
  a.info = reinterpret_cast<int4*>(a.part + n_part + ((n_ml + 3) & ~int64_t(3)));
  const int br = std::min(c.page, tattn::BN);
  const CUtensorMap tq = tattn::node_map(q, a.GT, a.TPM), tk = tattn::node_map(k, 1, (int)T),
                    tv = tattn::node_map(v, 1, (int)T), tkp = tattn::pool_map(c.k, c, br),
                    tvp = tattn::pool_map(c.v, c, br);
#define NS_X(DT)                                                   \
  {                                                                \
    if (c.e4m3)                                                    \
      tattn::launch<DT, true>(a, grid, tq, tk, tv, tkp, tvp);      \
    else                                                           \
      tattn::launch<DT, false>(a, grid, tq, tk, tv, tkp, tvp);     \
  }
  if (D <= 64) NS_X(64) else if (D <= 128) NS_X(128) else NS_X(256)
#undef NS_X
  const int64_t nrows = b * T * Hq;
  tattn::tree_join_kernel<<<(unsigned)((nrows + 7) / 8), 256, 0, stream()>>>(a);
  NS_CUDA(cudaGetLastError());
  return {out, lse};
}

}  // namespace ns
