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
//   S_j = Q K_j^T      M=128, N=128, K=D -> TMEM (two 128-column buffers)
//   O  += P_j V_j      M=128, N=D, K=128 -> TMEM, P_j over its own S_j in TMEM
// over tiles of 128 keys: the tiles of the cached prefix, then one tile of the nodes' own
// keys whose mask is the row's ancestor set. S_{j+1} is issued before P_j V_j, so the tensor
// cores work while the softmax warps (two threads per row) form P.
//
// Work is split over the long axis without knowing the lengths on the host: the tiles of
// all segments (sequence, key head, row tile) are numbered through, and CTA i of N (one per
// SM) takes units [U i / N, U (i+1) / N) (every segment counts a few more for its beginning
// and end), so ragged batches and single long sequences load
// every SM alike. A segment that one CTA holds whole is finished there; parts of a segment
// leave their output with its reference maximum and sum in a workspace (two parts per CTA
// at most), and tree_join_kernel adds them up in the order of the CTAs.
//
// bf16 pages: P must be bf16 like V, whose 8 bits would cost as much as the output's own
// rounding, so P is the sum of two bf16 matrices (16 bits) and P V two products.
//
// e4m3 pages: the codes of K go to the tensor cores as they are (kind::f8f6f4). q, scaled by
// a power of two per row, is the sum of an e4m3 and an e5m2 matrix: rounding q's 8
// significant bits to 4 leaves at most 8 units of the last of them, which the 3 of e5m2 hold
// exactly (elements below 2^-14 of the row's largest are held to 2^-22 of it). V's codes are
// multiplied in 8 bits too: P as f16 (11 bits) is the sum of four e5m2 matrices, each the high
// bytes of what the ones before left. The rows' scales stay outside the products: K's
// multiplies the score, V's, 2^e_j, the probability: P_j = 2^(s_j + e_j - r) with r a running
// maximum of s_j + e_j (log2) over the keys that the row sees, apart from that of s_j which
// the sum is relative to. So a V row of any scale counts by what it adds to the output: terms below
// 2^-28 of the row's largest 2^(s_j + e_j) are dropped (2^-28 of it at most per key, half a
// rounding of the output at 2^18 such keys), the others keep 11 bits. The nodes' own
// K and V are split like q. So no operand is converted on its way to the tensor cores.
//
// Measured (32 sequences of 14000 keys, 4 key heads of 256, pages of 64): bf16 378 us at one
// node (4.86 TB/s) and 413 at 21 (561 TFLOP/s of products, 4.51 TB/s); e4m3 587 and 597 us
// (1.6 TB/s). bf16 waits for K tiles at 75 % of the copy rate. e4m3 is bound by neither its products
// nor its softmax: a quarter of the products with P takes 2 % less, half of the softmax 7 %, so
// mostly by the steps of a tile waiting for one another. (Counting V's scale with the score
// is 8 % of it: 548 and 552 us with V relative to the largest scale seen, which lost rows.)
//
// Rows of V beyond a sequence's end (stale pages, NaN) are zeroed in shared memory, since
// 0 * NaN would reach O; masked scores are replaced, not added to. Every mbarrier wait is
// bounded; a timeout sets the device error word and the kernel unwinds.
#include <cfloat>

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "decode.h"
#include "sm100.cuh"

namespace ns {

using bf16 = __nv_bfloat16;

namespace tattn {

constexpr int EXP_BIAS = 127, EXP_MIN = -117, EXP_MAX = 118;
constexpr int BM = 128, BN = 128;
constexpr float LAG = 8.f;      // the reference maximum of the scores may lag by this much (log2)
constexpr float LAG8 = 3.f;     // e4m3: that of score and V scale together by this, so P is at most
constexpr float OFFSET8 = 12.f; // 2^(OFFSET8 + LAG8) = 2^15, the top of e5m2, whose smallest step, 2^-16, is 2^-28
                                // of the largest P when the reference has just been set
constexpr int SLOT = 16384;           // bytes of one ring slot
constexpr int SOFT_WARPS = 8, CONV_WARPS = 2;

struct Args {
  const bf16 *q, *k, *v, *gate;
  int64_t q_bs, q_ts, q_hs, k_bs, k_ts, k_hs, v_bs, v_ts, v_hs, g_bs, g_ts, g_hs;
  const uint8_t *ke, *ve;
  const int *table, *lens, *parents, *counts;
  int64_t p_bs, pages, max_pages;
  int b, T, Hq, Hk, D, page, page_log2;
  int seg;                // what beginning and ending a segment costs, in tiles
  int G, GT, HB, TPM, M;  // heads of a group, per row tile, head blocks; tokens per row tile, token blocks
  float scale_log2;
  bf16* out;    // [b, T, Hq, D]
  float* lse;   // [b, Hq, T]
  float* part;  // [N][2][GT * TPM][D] the parts' outputs
  float2* ml;   // [N][2][GT * TPM] reference maximum (log2) and sum
  int2* info;   // [segments] first CTA, last CTA
  int* err;
};

__device__ __forceinline__ float bf(bf16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126..127

// Bounded wait: gives up after two seconds (a lost arrival), sets the error word. One lane
// waits for its warp (32 lanes polling one barrier queue up on it); a wait that ran out makes
// its later waits and products void (`ok`), and every role still walks to its end, so
// no other wait of the CTA is left without a partner for longer than its own limit.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, int* err) {
  uint64_t t0 = 0;
  for (uint32_t i = 1; i < (1u << 28); ++i) {
    if (sm100::mbar_try_wait(bar, parity)) return true;
    if ((i & 255) == 0) {
      uint64_t now;
      asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
      if (t0 == 0) t0 = now;
      if (now - t0 > 2000000000ull) break;
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

// Units of work: a row tile whose first token is live has the prefix's tiles and the nodes',
// others one tile of zeros; every segment starts with `seg` units that stand for its beginning
// and end (q, first loads, output).
__device__ __forceinline__ int64_t group_units(const Args& a, Seq q, int live) {
  return (int64_t)live * ((q.len + BN - 1) / BN + 1 + a.seg) + (int64_t)(a.M - live) * (1 + a.seg);
}
__device__ __forceinline__ int64_t seq_units(const Args& a, Seq q) {
  return (int64_t)a.Hk * a.HB * group_units(a, q, (q.cnt + a.TPM - 1) / a.TPM);
}

// A contiguous run of tiles of one segment.
struct Piece {
  int s, hk, hb, m;       // sequence, key head, head block, token block
  Seq q;
  int nt;                 // prefix tiles of the segment (0 when no token is live)
  int t0, t1;             // tiles [t0, t1) of [0, nt]; tile nt is the nodes' own
  bool whole;
  __device__ __forceinline__ int keys(int t) const { return t < nt ? min(BN, q.len - t * BN) : own; }
  int own;                // keys of the nodes' tile
  int64_t last;           // the segment's last unit
};

struct Walk {
  int s, seg, off;        // next sequence, segment within it, unit within that
  int64_t unit, end;      // its global number; end of this CTA's run
  Seq q;
  // the next tiles of one segment; false at the end of the run
  __device__ __forceinline__ bool next(const Args& a, Piece& p) {
    const int segs = a.Hk * a.HB * a.M;
    while (unit < end) {
      if (seg == segs) {
        seg = 0;
        q = sequence(a, ++s, false);
      }
      p.s = s;
      p.q = q;
      p.m = seg % a.M;
      p.hb = (seg / a.M) % a.HB;
      p.hk = seg / (a.M * a.HB);
      p.own = p.m * a.TPM < q.cnt ? q.cnt : 0;
      p.nt = p.own > 0 ? (q.len + BN - 1) / BN : 0;
      const int units = p.nt + 1 + a.seg;
      p.last = unit - off + units - 1;
      const int to = (int)min((int64_t)units, off + (end - unit));
      p.t0 = max(off - a.seg, 0);
      p.t1 = max(to - a.seg, 0);
      p.whole = p.t0 == 0 && p.t1 == p.nt + 1;
      unit += to - off;
      off = to;
      if (off == units) off = 0, ++seg;
      if (p.t1 > p.t0) return true;
    }
    return false;
  }
};

// First position and end of CTA blockIdx.x (warp-wide); total units in U, CTAs that have any in N. A
// run may lie wholly within a segment's first `seg` units: such a CTA has no tile and leaves no part.
__device__ __forceinline__ Walk plan(const Args& a, int lane, int64_t& U, int& N) {
  int64_t sum = 0, n = 0;
  Seq q{0, 0};
  for (int s = lane; s < a.b; s += 32) {
    q = sequence(a, s, blockIdx.x == 0);
    n = seq_units(a, q);
    sum += n;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffff, sum, o);
  U = sum;
  N = (int)min((int64_t)gridDim.x, U);
  Walk w;
  w.unit = U * min((int)blockIdx.x, N) / N;
  w.end = U * min((int)blockIdx.x + 1, N) / N;
  int64_t before = 0;
  w.s = a.b, w.seg = w.off = 0, w.q = {0, 0};
  for (int s0 = 0; s0 < a.b; s0 += 32) {
    const int s = s0 + lane;
    if (a.b > 32) {  // (otherwise each lane still has its sequence)
      q = s < a.b ? sequence(a, s, false) : Seq{0, 0};
      n = s < a.b ? seq_units(a, q) : 0;
    }
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
      const int64_t units = (w.q.len + BN - 1) / BN + 1 + a.seg;
      const int64_t group = group_units(a, w.q, live);  // one (key head, head block)
      w.seg = (int)(rem / group) * a.M;
      rem %= group;
      if (rem < live * units) {
        w.seg += (int)(rem / units);
        w.off = (int)(rem % units);
      } else {
        rem -= live * units;
        w.seg += live + (int)(rem / (1 + a.seg));
        w.off = (int)(rem % (1 + a.seg));
      }
      break;
    }
    before += __shfl_sync(0xffffffff, inc, 31);
  }
  return w;
}

// ------------------------------------------------------------------ shared memory
// A ring of 16 KB slots with its position and phase.
struct Ring {
  int st = 0, ph = 0;
  __device__ __forceinline__ void step(int size) {
    if (++st == size) st = 0, ph ^= 1;
  }
};

template <int DT, bool E4M3>
struct Cfg {
  static constexpr int DA = E4M3 ? DT / 128 : DT / 64;  // 128-byte swizzle atoms along D: ring slots of a K or V tile
  static constexpr int AC = E4M3 ? 128 : 64;       // channels of one
  static constexpr int VK = BN / DA;               // keys in one slot of V
  static constexpr int KQ = E4M3 ? 32 : 16;        // keys of one product with P
  static constexpr int PP = E4M3 ? 4 : 2;          // matrices whose sum is P
  static constexpr int Q_BYTES = BM * DT * 2;      // bf16, or the two 8-bit matrices
  static constexpr int NK = DT == 256 ? 9 : 11;    // ring slots, K and V in the order of the products
  // maxima, sums, q's maxima and those with V's scale exchanged by a row's threads
  static constexpr int XCH = 4 * 2 * 2 * BM * 4;
  // e4m3 scales of FAC tiles: exponent bytes, K's factors and V's exponents
  static constexpr int FAC = 4;
  static constexpr int FACS = E4M3 ? FAC * (2 * BN + 2 * BN * 2) + MAX_NODES * 4 : 0;
  static constexpr int SMEM = Q_BYTES + NK * SLOT + FACS + XCH + 128 + 512 + 1024;
  static constexpr int S_COL = DT;
  static constexpr int TMEM_COLS = 512;            // DT + 2 BN, a power of two
  static constexpr int THREADS = 32 * (2 + SOFT_WARPS + (E4M3 ? CONV_WARPS : 0));
  static_assert(SMEM <= 232448, "shared memory");
};

// Tiles of a piece in the order of the products: S0, (S1, PV0), (S2, PV1), .., PV(n-1).
template <class F>
__device__ __forceinline__ void product_order(int t0, int t1, F&& f) {
  f(t0, false);
  for (int t = t0; t < t1; ++t) {
    if (t + 1 < t1) f(t + 1, false);
    f(t, true);
  }
}

// exponent that brings a row whose largest magnitude has the bits `top` into [2^at, 2^(at+1))
__device__ __forceinline__ int row_exponent(uint32_t top, int at) {
  return max(min((int)(top >> 23) - 127 - at, EXP_MAX), EXP_MIN);
}

// largest magnitude (its bits) of 8 bf16; infinities and NaN do not count, or are above all others
template <bool FINITE>
__device__ __forceinline__ uint32_t largest(uint4 w) {
  const uint32_t in[4] = {w.x, w.y, w.z, w.w};
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = (in[i] << 16) & 0x7fffffffu, hi = in[i] & 0x7fff0000u;
    top = max(top, max(!FINITE || lo < 0x7f800000u ? lo : 0u, !FINITE || hi < 0x7f800000u ? hi : 0u));
  }
  return top;
}

// 8 bf16 times s as the sum of e4m3 and e5m2
__device__ __forceinline__ void split_fp8(uint4 w, float s, uint2& hi, uint2& lo) {
  const uint32_t x[4] = {w.x, w.y, w.z, w.w};
  uint32_t h[2] = {0, 0}, l[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = __uint_as_float(x[i] << 16) * s, b = __uint_as_float(x[i] & 0xffff0000u) * s;
    const __nv_fp8x2_storage_t c = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(c, __NV_E4M3)));
    const __nv_fp8x2_storage_t r = __nv_cvt_float2_to_fp8x2(make_float2(a - f.x, b - f.y), __NV_SATFINITE, __NV_E5M2);
    h[i / 2] |= (uint32_t)c << (16 * (i & 1));
    l[i / 2] |= (uint32_t)r << (16 * (i & 1));
  }
  hi = make_uint2(h[0], h[1]);
  lo = make_uint2(l[0], l[1]);
}

__device__ __forceinline__ uint4 lds4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}

// what e5m2 leaves of two f16
__device__ __forceinline__ uint32_t high_bytes_off(uint32_t w) {
  const uint32_t top = w & 0xff00ff00u;
  const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&w), *reinterpret_cast<const __half2*>(&top));
  return *reinterpret_cast<const uint32_t*>(&d);
}

// byte offset of 16-byte chunk c of row r in a K-major 128-byte-swizzled tile of `rows` rows
__device__ __forceinline__ uint32_t tile_offset(int rows, int r, int c) {
  return (uint32_t)((c >> 3) * rows * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

template <int DT, bool E4M3>
__global__ void __launch_bounds__(Cfg<DT, E4M3>::THREADS, 1)
    tree_attn_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                     const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap tkp,
                     const __grid_constant__ CUtensorMap tvp, Args a) {
  using C = Cfg<DT, E4M3>;
  constexpr int DA = C::DA, VK = C::VK, NK = C::NK, FAC = C::FAC;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sQ = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sKV = sQ + C::Q_BYTES;                                        // [NK]
  bf16* kfac = reinterpret_cast<bf16*>(sKV + NK * SLOT);                 // [FAC][BN] 2^e of K rows
  bf16* vlog = kfac + (E4M3 ? FAC * BN : 0);                             // [FAC][BN] e of V rows
  int* vexp = reinterpret_cast<int*>(vlog + (E4M3 ? FAC * BN : 0));      // [MAX_NODES] exponents of the nodes' V
  uint8_t* sExp = reinterpret_cast<uint8_t*>(vexp + (E4M3 ? MAX_NODES : 0));  // [FAC][2][BN] exponent bytes
  float* xmax = reinterpret_cast<float*>(sExp + (E4M3 ? FAC * 2 * BN : 0));   // [2][2][BM]
  float* xsum = xmax + 2 * 2 * BM;                                            // [2][2][BM]
  float* xq = xsum + 2 * 2 * BM;                                              // [2][2][BM]
  float* xtop = xq + 2 * 2 * BM;                                              // [2][2][BM]
  int* page_rows = reinterpret_cast<int*>(xtop + 2 * 2 * BM);               // [4][8] of the producer
  uint64_t* bars = reinterpret_cast<uint64_t*>(page_rows + 32);
  uint64_t* full = bars;             // [NK]
  uint64_t* empty = full + NK;       // [NK]
  uint64_t* e_full = empty + NK;     // [FAC] exponent bytes landed (e4m3)
  uint64_t* f_full = e_full + FAC;   // [FAC] factors ready
  uint64_t* f_free = f_full + FAC;   // [FAC] factors read
  uint64_t* s_full = f_free + FAC;   // [2]
  uint64_t* p_full = s_full + 2;     // [2]
  uint64_t* q_full = p_full + 2;
  uint64_t* q_empty = q_full + 1;
  uint64_t* o_done = q_empty + 1;  // one completion per PV (rescales wait for the previous one)
  uint64_t* o_last = o_done + 1;   // one per piece, after its last PV
  uint64_t* o_free = o_last + 1;   // one per piece, O has been read
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_free + 1);
  static_assert(2 * NK + 3 * FAC + 9 + 1 <= 64, "barrier area");

  // the join may be set up now; it waits for this kernel's end
  asm volatile("griddepcontrol.launch_dependents;");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int64_t U;
  int N;
  Walk walk = plan(a, lane, U, N);  // every warp on its own: no shared state
  if (walk.unit >= walk.end) return;

  if (warp == 0 && lane == 0) {
    for (int i = 0; i < NK; ++i) sm100::mbar_init(&full[i], 1), sm100::mbar_init(&empty[i], 1);
    for (int i = 0; i < FAC; ++i) {
      sm100::mbar_init(&e_full[i], 1);
      sm100::mbar_init(&f_full[i], 1);
      sm100::mbar_init(&f_free[i], SOFT_WARPS);
    }
    for (int i = 0; i < 2; ++i) sm100::mbar_init(&s_full[i], 1), sm100::mbar_init(&p_full[i], SOFT_WARPS);
    sm100::mbar_init(q_full, E4M3 ? SOFT_WARPS : 1);
    sm100::mbar_init(q_empty, 1);
    sm100::mbar_init(o_done, 1);
    sm100::mbar_init(o_last, 1);
    sm100::mbar_init(o_free, SOFT_WARPS);
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

  Piece p;
  if (warp == 0) {
    // ---------------------------------------------------------- TMA producer
    // The whole warp waits; one elected lane issues (ptxas then keeps the operands uniform).
    const int kb = min(a.page, BN), vb = min(a.page, VK);  // rows that one copy brings
    Ring r;
    int n = 0, pc = 0;
    bool ok = true;
    // pool rows of 16 keys each (lane l: keys 16 l ..) of tile t, kept in shared memory for the
    // issuing lane: a page out of range is replaced by page 0
    auto look_up = [&](int t) {
      const int key = t * BN + lane * 16;
      if (lane < 8 && t < p.nt && key < p.q.len) {
        int pg = __ldg(a.table + p.s * a.max_pages + (key >> a.page_log2));
        if (pg < 0 || pg >= a.pages) {
          atomicExch(a.err, ERR_INDEX);
          pg = 0;
        }
        page_rows[(t & 3) * 8 + lane] = ((pg * a.Hk + p.hk) << a.page_log2) + (key & (a.page - 1));
      }
      __syncwarp();
    };
    while (walk.next(a, p)) {
      look_up(p.t0);
      if constexpr (!E4M3) {
        if (pc > 0) ok = ok && wait(q_empty, (pc - 1) & 1, a.err);
        if (sm100::elect_one() && ok) {
          sm100::mbar_expect_tx(q_full, DA * a.GT * a.TPM * 128);
#pragma unroll
          for (int j = 0; j < DA; ++j)
            sm100::tma_load_4d(sQ + j * (BM * 128), &tq, q_full, 64 * j, p.hk * a.G + p.hb * a.GT, p.m * a.TPM, p.s);
        }
        __syncwarp();
        ++pc;
      }
      product_order(p.t0, p.t1, [&](int t, bool pv) {
        const int keys = p.keys(t);
        const bool own = t == p.nt;
        const int* rows = page_rows + (t & 3) * 8;
        if (E4M3 && own) {  // the converters fill these
          for (int j = 0; j < (pv && keys == 0 ? 0 : DA); ++j) r.step(NK);
          n += !pv;
        } else if (!pv) {
          const int runs = (keys + kb - 1) / kb;
          if (t + 1 < p.t1) look_up(t + 1);
#pragma unroll 1
          for (int j = 0; j < DA; ++j) {
            ok = ok && wait(&empty[r.st], r.ph ^ 1, a.err);
            if (sm100::elect_one() && ok) {
              uint64_t* fb = &full[r.st];
              uint8_t* d = sKV + r.st * SLOT;
              if (own) {
                sm100::mbar_expect_tx(fb, a.T * 128);
                sm100::tma_load_4d(d, &tk, fb, 64 * j, p.hk, 0, p.s);
              } else {
                sm100::mbar_expect_tx(fb, runs * kb * 128);
                for (int x = 0; x < runs; ++x)
                  sm100::tma_load_2d(d + x * kb * 128, &tkp, fb, C::AC * j, rows[x * kb / 16]);
              }
            }
            __syncwarp();
            r.step(NK);
          }
          if constexpr (E4M3) {
            uint64_t* eb = &e_full[n % FAC];
            if (n >= FAC) ok = ok && wait(&f_free[n % FAC], (n / FAC - 1) & 1, a.err);
            if (sm100::elect_one() && ok) {
              sm100::mbar_expect_tx(eb, runs * kb * 2);
              for (int x = 0; x < runs; ++x) {
                sm100::bulk_load(sExp + (n % FAC) * 2 * BN + x * kb, a.ke + rows[x * kb / 16], kb, eb);
                sm100::bulk_load(sExp + ((n % FAC) * 2 + 1) * BN + x * kb, a.ve + rows[x * kb / 16], kb, eb);
              }
            }
            __syncwarp();
            ++n;
          }
        } else {
#pragma unroll 1
          for (int i = 0; i * VK < keys; ++i) {
            ok = ok && wait(&empty[r.st], r.ph ^ 1, a.err);
            if (sm100::elect_one() && ok) {
              uint64_t* fb = &full[r.st];
              uint8_t* d = sKV + r.st * SLOT;
              if (own) {
                sm100::mbar_expect_tx(fb, DA * min(a.T, VK) * 128);
#pragma unroll
                for (int j = 0; j < DA; ++j)
                  sm100::tma_load_4d(d + j * (VK * 128), &tv, fb, 64 * j, p.hk, i * VK, p.s);
              } else {
                const int runs = (min(VK, keys - i * VK) + vb - 1) / vb;
                sm100::mbar_expect_tx(fb, DA * runs * vb * 128);
                for (int u = 0; u < runs; ++u) {
                  const int row = rows[(i * VK + u * vb) / 16];
#pragma unroll
                  for (int j = 0; j < DA; ++j)
                    sm100::tma_load_2d(d + j * (VK * 128) + u * vb * 128, &tvp, fb, C::AC * j, row);
                }
              }
            }
            __syncwarp();
            r.step(NK);
          }
        }
      });
    }
    // drain: every issued copy has landed before the CTA may exit
    if (!E4M3 && pc > 0) wait(q_full, (pc - 1) & 1, a.err);
    for (int i = 0; i < NK; ++i) {  // slots that were never armed count as empty
      wait(&empty[r.st], r.ph ^ 1, a.err);
      r.step(NK);
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------- MMA issuer
    // The tensor cores wait for this warp's own instructions first, so the loops hold little but
    // waits (the whole warp) and products (one elected lane: ptxas then keeps the operands
    // uniform, without a loop over lanes around each); descriptors are a constant plus offsets
    // in 16-byte units.
    constexpr uint32_t E5M2_A = 1u << 7, E5M2_B = 1u << 10;  // kind::f8f6f4: e4m3 otherwise
    constexpr uint32_t idesc_o =
        E4M3 ? sm100::idesc_e4m3(BM, DT, false, true) | E5M2_A : sm100::idesc_bf16(BM, DT, false, true);
    const uint64_t dq = sm100::smem_desc_sw128(sm100::smem_u32(sQ), 0, 1024);
    const uint64_t dk = sm100::smem_desc_sw128(sm100::smem_u32(sKV), 0, 1024);
    const uint64_t dv = sm100::smem_desc_sw128(sm100::smem_u32(sKV), VK * 128, 1024);
    Ring r;
    int n = 0, ns = 0, pc = 0;  // PV tile, S tile, piece
    bool ok = true;
    while (walk.next(a, p)) {
      ok = ok && wait(q_full, pc & 1, a.err);
      product_order(p.t0, p.t1, [&](int t, bool pv) {
        const int keys = p.keys(t);
        const bool own = t == p.nt;
        // the slots of the second matrix of the nodes' rows (e4m3 form)
        const uint64_t lo_off = DT == 256 ? (uint64_t)((r.st + 1) % NK * (SLOT / 16)) : r.st * (SLOT / 16) + MAX_NODES * 8;
        if (!pv) {
          const uint32_t cols = max(16, (keys + 15) & ~15);
          const uint32_t idesc = (E4M3 ? sm100::idesc_e4m3(BM, 0, false, false) : sm100::idesc_bf16(BM, 0, false, false)) +
                                 ((cols >> 3) << 17);
          const uint32_t d = tmem + C::S_COL + (ns & 1) * BN;
          // the buffer's last reader, and every product before it, is done
          if (n > 0) ok = ok && wait(o_done, (n - 1) & 1, a.err);
          if (E4M3 && own) {  // (Q hi + Q lo) (K hi + K lo), K matrices of 64 rows
            const Ring k0 = r;
            for (int j = 0; j < DA; ++j) {
              ok = ok && wait(&full[r.st], r.ph, a.err);
              r.step(NK);
            }
            sm100::tc_fence_after();
            if (sm100::elect_one() && ok) {
              const uint64_t hi = dk + k0.st * (SLOT / 16), lo = dk + lo_off;
#pragma unroll 1
              for (int x = 0; x < 4; ++x) {
#pragma unroll
                for (int kk = 0; kk < DT / 32; ++kk)
                  sm100::mma_f8(d, dq + (x & 1) * (BM * DT / 16) + (kk >> 2) * (BM * 8) + (kk & 3) * 2,
                                (x >> 1 ? lo : hi) + (kk >> 2) * (MAX_NODES * 8) + (kk & 3) * 2,
                                idesc | (x & 1) * E5M2_A | (x >> 1) * E5M2_B, x + kk > 0 ? 1u : 0u);
              }
              sm100::mma_commit(&empty[k0.st]);
              if (DA == 2) sm100::mma_commit(&empty[(k0.st + 1) % NK]);
              sm100::mma_commit(&s_full[ns & 1]);
            }
          } else {
#pragma unroll
            for (int j = 0; j < DA; ++j) {
              ok = ok && wait(&full[r.st], r.ph, a.err);
              sm100::tc_fence_after();
              if (sm100::elect_one() && ok) {
                const uint64_t kd = dk + r.st * (SLOT / 16);
                if constexpr (E4M3) {
#pragma unroll
                  for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)
                      sm100::mma_f8(d, dq + (x * (BM * DT / 16) + j * (BM * 8) + kk * 2), kd + kk * 2,
                                    idesc | x * E5M2_A, j + x + kk > 0 ? 1u : 0u);
                } else {
#pragma unroll
                  for (int kk = 0; kk < 4; ++kk)
                    sm100::mma_bf16(d, dq + (j * (BM * 8) + kk * 2), kd + kk * 2, idesc, j + kk > 0 ? 1u : 0u);
                }
                sm100::mma_commit(&empty[r.st]);
                if (j == DA - 1) sm100::mma_commit(&s_full[ns & 1]);
              }
              r.step(NK);
            }
          }
          if (!E4M3 && t == p.t1 - 1 && sm100::elect_one() && ok) sm100::mma_commit(q_empty);
          ++ns;
        } else {
          const int pb = n & 1;
          const uint32_t ps = tmem + C::S_COL + pb * BN;
          ok = ok && wait(&p_full[pb], (n >> 1) & 1, a.err);
          if (t == p.t0 && pc > 0) ok = ok && wait(o_free, (pc - 1) & 1, a.err);
          // P of KQ keys: 8 columns of each of its matrices, 32 keys in the columns of their scores
          auto product = [&](int kq, uint64_t bd, uint32_t idesc, bool first) {
            constexpr int H = 32 / C::KQ;  // products of 32 keys
#pragma unroll
            for (int x = 0; x < C::PP; ++x) {
              const uint32_t ad = ps + kq / H * 32 + x * (H * 8) + kq % H * 8;
              const uint32_t acc = (first && x == 0) ? 0u : 1u;
              if constexpr (E4M3)
                sm100::mma_f8_ts(tmem, ad, bd, idesc, acc);
              else
                sm100::mma_f16_ts(tmem, ad, bd, idesc, acc);
            }
          };
          constexpr int KS = VK / C::KQ;  // products of one slot
          if (E4M3 && own) {
            if (keys > 0) {
              const Ring v0 = r;
              for (int j = 0; j < DA; ++j) {
                ok = ok && wait(&full[r.st], r.ph, a.err);
                r.step(NK);
              }
              sm100::tc_fence_after();
              if (sm100::elect_one() && ok) {
#pragma unroll 1
                for (int kk = 0; kk * C::KQ < keys; ++kk) {
                  product(kk, dv + v0.st * (SLOT / 16) + kk * (C::KQ * 8), idesc_o, t == p.t0 && kk == 0);
                  product(kk, dv + lo_off + kk * (C::KQ * 8), idesc_o | E5M2_B, false);
                }
                sm100::mma_commit(&empty[v0.st]);
                if (DA == 2) sm100::mma_commit(&empty[(v0.st + 1) % NK]);
              }
            }
            if (sm100::elect_one() && ok) sm100::mma_commit(o_done);
          } else if (keys == BN) {
#pragma unroll
            for (int i = 0; i < DA; ++i) {
              ok = ok && wait(&full[r.st], r.ph, a.err);
              sm100::tc_fence_after();
              if (sm100::elect_one() && ok) {
#pragma unroll
                for (int kk = 0; kk < KS; ++kk)
                  product(i * KS + kk, dv + r.st * (SLOT / 16) + kk * (C::KQ * 8), idesc_o, t == p.t0 && i + kk == 0);
                sm100::mma_commit(&empty[r.st]);
                if (i == DA - 1) sm100::mma_commit(o_done);
              }
              r.step(NK);
            }
          } else {
#pragma unroll 1
            for (int i = 0; i * VK < keys; ++i) {
              const int live = min(VK, keys - i * VK), dead = -live & (C::KQ - 1);
              ok = ok && wait(&full[r.st], r.ph, a.err);
              if (dead) {  // rows beyond the end, up to the next product's edge
                for (int x = lane; x < dead * 8 * DA; x += 32)
                  *reinterpret_cast<uint4*>(sKV + r.st * SLOT + tile_offset(VK, live + x / (8 * DA), x % (8 * DA))) =
                      make_uint4(0, 0, 0, 0);
                sm100::fence_proxy_async_smem();
                __syncwarp();
              }
              sm100::tc_fence_after();
              if (sm100::elect_one() && ok) {
#pragma unroll 1
                for (int kk = 0; kk * C::KQ < live; ++kk)
                  product(i * KS + kk, dv + r.st * (SLOT / 16) + kk * (C::KQ * 8), idesc_o, t == p.t0 && i + kk == 0);
                sm100::mma_commit(&empty[r.st]);
              }
              r.step(NK);
            }
            if (sm100::elect_one() && ok) sm100::mma_commit(o_done);
          }
          if (t == p.t1 - 1 && sm100::elect_one() && ok) sm100::mma_commit(o_last);
          ++n;
        }
      });
      ++pc;
    }
  } else if (warp < 2 + SOFT_WARPS) {
    // ---------------------------------------------------------- softmax warps
    // Two threads per row, each with 64 of a tile's 128 scores and half of O's columns. They
    // exchange their maxima through shared memory.
    const int qw = warp & 3, half = (warp - 2) >> 2;  // TMEM lane quarter, column half
    const int row = qw * 32 + lane;
    const uint32_t lane_off = (uint32_t)(qw * 32) << 16;
    const int rows = a.GT * a.TPM;
    const bool warp_on = qw * 32 < rows;
    int n = 0, pc = 0;
    bool ok = true;
    auto wait_all = [&](uint64_t* bar, uint32_t parity) {
      if (lane == 0) ok = ok && wait(bar, parity, a.err);
      __syncwarp();
    };
    auto exchange = [&](float* buf, float v) -> float {  // the partner's value
      buf[half * BM + row] = v;
      sm100::named_sync(1 + qw, 64);
      return buf[(half ^ 1) * BM + row];
    };
    while (walk.next(a, p)) {
      const int tok = p.m * a.TPM + row / a.GT, g = p.hb * a.GT + row % a.GT;
      const bool in = row < rows && g < a.G && tok < a.T;
      const bool live = in && tok < p.q.cnt;
      const int hq = p.hk * a.G + g;
      // multiplies the products of this row; never 0, which masked scores of -inf would turn into NaN
      float rs = fmaxf(a.scale_log2, FLT_MIN);
      if constexpr (E4M3) {
        // q row -> e4m3 and e5m2 rows with a power-of-two scale (the previous piece's products are
        // complete: this thread has seen all of its scores); this thread's half
        if (warp_on) {
          constexpr int QC = DT / 16;  // 16-byte chunks of a half, 8 at a time (registers)
          const bf16* q = a.q + p.s * a.q_bs + tok * a.q_ts + hq * a.q_hs + half * (DT / 2);
          auto load = [&](int c0, uint4 (&w)[8]) {
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              w[c] = make_uint4(0, 0, 0, 0);
              if (live && half * (DT / 2) + (c0 + c) * 8 < a.D) w[c] = *reinterpret_cast<const uint4*>(q + (c0 + c) * 8);
            }
          };
          uint32_t top = 0;
          uint4 w[8];
#pragma unroll 1
          for (int c0 = 0; c0 < QC; c0 += 8) {
            load(c0, w);
#pragma unroll
            for (int c = 0; c < 8; ++c) top = max(top, largest<false>(w[c]));
          }
          top = max(top, __float_as_uint(exchange(xq + (pc & 1) * 2 * BM, __uint_as_float(top))));
          const int e = row_exponent(top, 7);
          // a row that is not finite has no finite score (e4m3 would saturate)
          rs = top < 0x7f800000u ? fmaxf(rs * pow2(e), FLT_MIN) : NAN;
          const float sc = pow2(-e);
#pragma unroll 1
          for (int c0 = 0; c0 < QC; c0 += 8) {
            if (QC > 8) load(c0, w);
#pragma unroll
            for (int c = 0; c < 8; c += 2) {
              uint2 hi[2], lo[2];
              split_fp8(w[c], sc, hi[0], lo[0]);
              split_fp8(w[c + 1], sc, hi[1], lo[1]);
              const uint32_t at = tile_offset(BM, row, half * (DT / 32) + (c0 + c) / 2);
              *reinterpret_cast<uint4*>(sQ + at) = make_uint4(hi[0].x, hi[0].y, hi[1].x, hi[1].y);
              *reinterpret_cast<uint4*>(sQ + BM * DT + at) = make_uint4(lo[0].x, lo[0].y, lo[1].x, lo[1].y);
            }
          }
        }
        sm100::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive(q_full);
      }
      // ancestors of this row's node (all in the first half's columns)
      uint64_t anc = 0;
      if (live && half == 0 && p.t1 == p.nt + 1) {
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
      float m = -INFINITY, l = 0.f;  // reference maximum (log2) and this half's sum
      float mp = -INFINITY;          // e4m3: that of score and V exponent, which P is relative to
      for (int t = p.t0; t < p.t1; ++t, ++n) {
        const int sb = n & 1, left = p.keys(t) - half * 64;
        const uint64_t mask = t == p.nt ? anc : left >= 64 ? ~0ull : left <= 0 ? 0ull : (1ull << left) - 1;
        wait_all(&s_full[sb], (n >> 1) & 1);
        if constexpr (E4M3) wait_all(&f_full[n % FAC], (n / FAC) & 1);
        sm100::tc_fence_after();
        float alpha_o = 1.f;
        bool grow = false;
        const uint32_t scol = tmem + lane_off + C::S_COL + sb * BN + half * 64;
        const uint32_t kf = sm100::smem_u32(kfac + (n % FAC) * BN + half * 64);
        const uint32_t vl = sm100::smem_u32(vlog + (n % FAC) * BN + half * 64);
        // 32 scores: read, K's scale (e4m3), mask
        auto scores = [&](int c0, float (&x)[32]) {
          sm100::tmem_ld32(scol + c0, x);
          if constexpr (E4M3) {
            uint4 f[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) f[c] = lds4(kf + (c0 + c * 8) * 2);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const uint32_t w[4] = {f[c].x, f[c].y, f[c].z, f[c].w};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                x[c * 8 + 2 * i] *= __uint_as_float(w[i] << 16);
                x[c * 8 + 2 * i + 1] *= __uint_as_float(w[i] & 0xffff0000u);
              }
            }
          }
          const uint32_t mk = (uint32_t)(mask >> c0);
          if (mk != 0xffffffffu) {
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (!(mk & (1u << c))) x[c] = -INFINITY;
          }
        };
        // V's exponents of 8 keys
        auto exponents = [&](int c, float (&f)[8]) {
          const uint4 v4 = lds4(vl + c * 2);
          const uint32_t w[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
          }
        };
        // maximum first, then P, each a loop over 32 scores. One pass over all 64 with a second one
        // when the maximum grew was slower: its code is fetched faster than the instruction cache
        // gives it (e4m3, 32 x 14000 keys, 21 nodes, before V's scale counted with the score: 760
        // us, these loops 552).
        if (warp_on) {
          float mt = -INFINITY, mpt = -INFINITY;
#pragma unroll 1
          for (int c0 = 0; c0 < 64; c0 += 32) {
            float x[32];
            scores(c0, x);
            float mx[2] = {x[0], x[1]};
#pragma unroll
            for (int c = 2; c < 32; ++c) mx[c & 1] = fmaxf(mx[c & 1], x[c]);
            mt = fmaxf(mt, fmaxf(mx[0], mx[1]));
            if constexpr (E4M3) {
              float px[2] = {-INFINITY, -INFINITY};
#pragma unroll
              for (int c = 0; c < 32; c += 8) {
                float ve[8];
                exponents(c0 + c, ve);
#pragma unroll
                for (int i = 0; i < 8; ++i) px[i & 1] = fmaxf(px[i & 1], fmaf(x[c + i], rs, ve[i]));
              }
              mpt = fmaxf(mpt, fmaxf(px[0], px[1]));
            }
          }
          if constexpr (E4M3) xtop[(sb * 2 + half) * BM + row] = mpt;  // exchanged with the next
          mt = fmaxf(mt, exchange(xmax + sb * 2 * BM, mt));
          const float top = mt * rs;
          if (live && top > m + LAG) {
            const float f = sm100::exp2_approx(m - top);  // 0 on the first tile
            l *= f;
            m = top;
            if constexpr (!E4M3) {
              alpha_o = f;
              grow = true;
            }
          }
          if constexpr (E4M3) {
            mpt = fmaxf(mpt, xtop[(sb * 2 + (half ^ 1)) * BM + row]);
            if (live && mpt > mp + LAG8) {
              alpha_o = sm100::exp2_approx(mp - mpt);
              mp = mpt;
              grow = true;
            }
          }
        }
        // rescale O rows once the previous PV completed (warp-wide, rare after the first tiles)
        if (__any_sync(0xffffffff, warp_on && grow && t > p.t0)) {
          wait_all(o_done, (n - 1) & 1);
          sm100::tc_fence_after();
#pragma unroll 1
          for (int c = half * (DT / 2); c < (half + 1) * (DT / 2); c += 32) {
            float o[32];
            sm100::tmem_ld32(tmem + lane_off + c, o);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] *= alpha_o;
            sm100::tmem_st32(tmem + lane_off + c, o);
          }
        }
        if (warp_on) {
          const float ref = m == -INFINITY ? 0.f : m;
          const float ref_p = (mp == -INFINITY ? 0.f : mp) - OFFSET8;
          float sum[2] = {0.f, 0.f};
#pragma unroll 1
          for (int c0 = 0; c0 < 64; c0 += 32) {
            float x[32];
            uint32_t pk[32];
            scores(c0, x);
            float ve[8];
#pragma unroll
            for (int c = 0; c < 32; c += 4) {
              if (E4M3 && c % 8 == 0) exponents(c0 + c, ve);
              float pr[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) pr[i] = sm100::exp2_approx(fmaf(x[c + i], rs, -ref));
              sum[0] += pr[0] + pr[1];
              sum[1] += pr[2] + pr[3];
              if constexpr (E4M3) {
#pragma unroll
                for (int i = 0; i < 4; ++i)  // with V's scale: on its own range, whatever that of the sum is
                  pr[i] = sm100::exp2_approx(fmaf(x[c + i], rs, ve[c % 8 + i]) - ref_p);
                const __half2 h0 = __floats2half2_rn(pr[0], pr[1]), h1 = __floats2half2_rn(pr[2], pr[3]);
                uint32_t w0 = *reinterpret_cast<const uint32_t*>(&h0), w1 = *reinterpret_cast<const uint32_t*>(&h1);
#pragma unroll
                for (int y = 0; y < 4; ++y) {  // the high byte of an f16 is an e5m2
                  pk[y * 8 + c / 4] = __byte_perm(w0, w1, 0x7531);
                  if (y < 3) {
                    w0 = high_bytes_off(w0);
                    w1 = high_bytes_off(w1);
                  }
                }
              } else {
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                  const __nv_bfloat162 h2 = __floats2bfloat162_rn(pr[i], pr[i + 1]);
                  const uint32_t w = *reinterpret_cast<const uint32_t*>(&h2);
                  const __nv_bfloat162 l2 = __floats2bfloat162_rn(pr[i] - __uint_as_float(w << 16),
                                                                  pr[i + 1] - __uint_as_float(w & 0xffff0000u));
                  pk[(c + i) / 2] = w;
                  pk[16 + (c + i) / 2] = *reinterpret_cast<const uint32_t*>(&l2);
                }
              }
            }
            sm100::tmem_st32_async(scol + c0, pk);  // over the scores just read
          }
          l += sum[0] + sum[1];
          sm100::tmem_st_wait();
        }
        sm100::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          sm100::mbar_arrive(&p_full[sb]);
          if constexpr (E4M3) sm100::mbar_arrive(&f_free[n % FAC]);
        }
      }
      // the gate, read 32 channels ahead: the first while the last products run
      const bool gated = a.gate && live && p.whole;
      uint4 gw[4];
      auto read_gate = [&](int c) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (gated && c + i * 8 < a.D)
            gw[i] = *reinterpret_cast<const uint4*>(a.gate + p.s * a.g_bs + tok * a.g_ts + hq * a.g_hs + c + i * 8);
      };
      read_gate(half * (DT / 2));
      wait_all(o_last, pc & 1);
      sm100::tc_fence_after();
      if (warp_on) {
        l += exchange(xsum + (pc & 1) * 2 * BM, l);
        // O -> the output (a whole segment) or the workspace
        // e4m3: O is relative to mp and OFFSET8, l to m. Two factors, since their product may leave the
        // range of fp32 where the result does not.
        const float inv = (l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l)) * (E4M3 ? pow2(-(int)OFFSET8) : 1.f);
        const float vs = !E4M3 ? 1.f : mp == -INFINITY ? 0.f : sm100::exp2_approx(mp - m);
        // a CTA has one part that begins a segment (slot 1) and one that goes on with one (0) at most
        const int slot = p.t0 == 0;
        const int64_t at = ((int64_t)blockIdx.x * 2 + slot) * rows + row;
        bf16* o = a.out + (((int64_t)p.s * a.T + tok) * a.Hq + hq) * a.D;
#pragma unroll 1
        for (int c = half * (DT / 2); c < (half + 1) * (DT / 2); c += 32) {
          float v[32];
          sm100::tmem_ld32(tmem + lane_off + c, v);
          if (!in) continue;
          if (p.whole) {
            uint4 gc[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) gc[i] = gw[i];
            if (c + 32 < (half + 1) * (DT / 2)) read_gate(c + 32);
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
              if (c + i < a.D) {
                uint32_t w[4];
                const uint32_t gg[4] = {gc[i / 8].x, gc[i / 8].y, gc[i / 8].z, gc[i / 8].w};
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                  float o0 = v[i + j] * inv * vs, o1 = v[i + j + 1] * inv * vs;
                  if (gated) {
                    o0 *= __fdividef(1.f, 1.f + __expf(-__uint_as_float(gg[j / 2] << 16)));
                    o1 *= __fdividef(1.f, 1.f + __expf(-__uint_as_float(gg[j / 2] & 0xffff0000u)));
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
                    live ? make_float4(v[i] * inv * vs, v[i + 1] * inv * vs, v[i + 2] * inv * vs, v[i + 3] * inv * vs)
                         : make_float4(0.f, 0.f, 0.f, 0.f);
          }
        }
        if (in && half == 0) {
          if (p.whole)
            a.lse[((int64_t)p.s * a.Hq + hq) * a.T + tok] =
                live ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
          else
            a.ml[at] = live ? make_float2(m, l) : make_float2(-INFINITY, 0.f);
        }
        if (row == 0 && half == 0 && p.t0 == 0) {  // where the segment's parts are
          const int c1 = p.whole ? (int)blockIdx.x : (int)(((p.last + 1) * N - 1) / U);
          a.info[(((int64_t)p.s * a.Hk + p.hk) * a.HB + p.hb) * a.M + p.m] = make_int2(blockIdx.x, c1);
        }
      }
      sm100::tc_fence_before();
      __syncwarp();
      if (lane == 0) sm100::mbar_arrive(o_free);
      ++pc;
    }
  } else if constexpr (E4M3) {
    // ---------------------------------------------------------- scales, and the nodes' own rows
    // Per tile: the scales' factors in the place of S. Of the nodes' tile also K (in the place of S)
    // and V (of PV) as two 8-bit matrices of 64 rows each, one row per warp pass, four under way.
    const int cw = warp - 2 - SOFT_WARPS;
    Ring r;
    int n = 0;
    bool ok = true;
    auto wait_all = [&](uint64_t* bar, uint32_t parity) {
      if (lane == 0) ok = ok && wait(bar, parity, a.err);
      __syncwarp();
    };
    while (walk.next(a, p)) {
      product_order(p.t0, p.t1, [&](int t, bool pv) {
        const int keys = p.keys(t), fb = n % FAC;
        const bool own = t == p.nt;
        if (!own) {
          for (int i = 0; i * VK < (pv ? keys : BN); ++i) r.step(NK);
          if (pv) return;
          if (cw == n % CONV_WARPS) {
            if (n >= FAC) wait_all(&f_free[fb], (n / FAC - 1) & 1);
            wait_all(&e_full[fb], (n / FAC) & 1);
            const uint8_t* ex = sExp + fb * 2 * BN;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int x = lane + 32 * i;
              kfac[fb * BN + x] = __float2bfloat16(x < keys ? pow2(min(max((int)ex[x] - EXP_BIAS, EXP_MIN), EXP_MAX)) : 0.f);
              vlog[fb * BN + x] = __float2bfloat16((float)min(max((int)ex[BN + x] - EXP_BIAS, EXP_MIN), EXP_MAX));
            }
            __syncwarp();
            if (lane == 0) sm100::mbar_arrive(&f_full[fb]);
          }
          ++n;
          return;
        }
        if (pv && keys == 0) return;
        const Ring r0 = r;
        for (int j = 0; j < DA; ++j) {
          wait_all(&empty[r.st], r.ph ^ 1);
          r.step(NK);
        }
        if (!pv && n >= FAC) wait_all(&f_free[fb], (n / FAC - 1) & 1);
        uint8_t* hi_at = sKV + r0.st * SLOT;
        uint8_t* lo_at = DT == 256 ? sKV + (r0.st + 1) % NK * SLOT : hi_at + MAX_NODES * 128;
        const bf16* ks = a.k + p.s * a.k_bs + p.hk * a.k_hs + lane * 8;
        const bf16* vs = a.v + p.s * a.v_bs + p.hk * a.v_hs + lane * 8;
        const int rows = (keys + 31) & ~31;  // up to the edge of the last product with P
#pragma unroll 1
        for (int x0 = cw; x0 < rows; x0 += 4 * CONV_WARPS) {
          uint4 k4[4], v4[4];
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const int x = x0 + y * CONV_WARPS;
            k4[y] = v4[y] = make_uint4(0, 0, 0, 0);
            if (x < keys && lane * 8 < a.D) {
              if (!pv) k4[y] = *reinterpret_cast<const uint4*>(ks + x * a.k_ts);
              v4[y] = *reinterpret_cast<const uint4*>(vs + x * a.v_ts);
            }
          }
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const int x = x0 + y * CONV_WARPS;
            int e;
            if (!pv) {  // exponents that bring the rows into [2^7, 2^8)
              e = x < keys ? row_exponent(__reduce_max_sync(0xffffffff, largest<true>(k4[y])), 7) : EXP_MIN;
              const int ve = row_exponent(__reduce_max_sync(0xffffffff, largest<true>(v4[y])), 7);
              if (lane == 0) {
                kfac[fb * BN + x] = __float2bfloat16(x < keys ? pow2(e) : 0.f);
                vexp[x] = x < keys ? ve : EXP_MIN;
              }
            } else {
              e = vexp[x];
            }
            uint2 hi, lo;
            split_fp8(pv ? v4[y] : k4[y], pow2(-e), hi, lo);
            if (lane < DT / 8) {
              const uint32_t at = tile_offset(MAX_NODES, x, lane >> 1) + (lane & 1) * 8;
              *reinterpret_cast<uint2*>(hi_at + at) = hi;
              *reinterpret_cast<uint2*>(lo_at + at) = lo;
            }
          }
        }
        sm100::fence_proxy_async_smem();
        sm100::named_sync(5, CONV_WARPS * 32);
        if (cw == 0) {
          if (lane < DA) sm100::mbar_arrive(&full[(r0.st + lane) % NK]);
          if (!pv) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int x = lane + 32 * i;
              vlog[fb * BN + x] = __float2bfloat16(x < keys ? (float)vexp[x] : 0.f);
              if (i >= 2) kfac[fb * BN + x] = __float2bfloat16(0.f);
            }
            __syncwarp();
            if (lane == 0) {
              sm100::mbar_arrive(&e_full[fb]);  // keeps its phase in step with the tiles
              sm100::mbar_arrive(&f_full[fb]);
            }
          }
        }
        if (!pv) ++n;
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
  asm volatile("griddepcontrol.wait;" ::: "memory");  // launched while the tiles are still at work
  const int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (i >= (int64_t)a.b * a.T * a.Hq) return;
  const int hq = (int)(i % a.Hq), tok = (int)((i / a.Hq) % a.T), s = (int)(i / ((int64_t)a.Hq * a.T));
  const int hk = hq / a.G, g = hq % a.G, hb = g / a.GT, m = tok / a.TPM;
  const int2 inf = a.info[(((int64_t)s * a.Hk + hk) * a.HB + hb) * a.M + m];
  if (inf.x == inf.y) return;
  const int rows = a.GT * a.TPM, row = (tok - m * a.TPM) * a.GT + g - hb * a.GT, parts = inf.y - inf.x + 1;
  const bool on = lane * 8 < a.D;
  const int64_t oi = i * a.D + lane * 8;
  uint4 gw = make_uint4(0, 0, 0, 0);
  if (a.gate && on)
    gw = *reinterpret_cast<const uint4*>(a.gate + s * a.g_bs + tok * a.g_ts + hq * a.g_hs + lane * 8);
  auto at = [&](int c) -> int64_t { return ((int64_t)(inf.x + c) * 2 + (c == 0)) * rows + row; };
  float top = -INFINITY, l = 0.f, o[8] = {};
  for (int c = lane; c < parts; c += 32) top = fmaxf(top, a.ml[at(c)].x);
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffff, top, x));
  for (int c0 = 0; c0 < parts; c0 += 32) {
    float w = 0.f;  // lane c: weight of part c0 + c
    if (c0 + lane < parts) {
      const float2 ml = a.ml[at(c0 + lane)];
      w = ml.x == -INFINITY ? ml.y : sm100::exp2_approx(ml.x - top) * ml.y;  // (0, or NaN of a row that is)
      l += w;
    }
    const int n = min(32, parts - c0);
#pragma unroll 4
    for (int c = 0; c < n; ++c) {
      const float wc = __shfl_sync(0xffffffff, w, c);
      if (on) {
        const float4* p = reinterpret_cast<const float4*>(a.part + at(c0 + c) * a.D + lane * 8);
        const float4 u = p[0], v = p[1];
        o[0] = fmaf(wc, u.x, o[0]), o[1] = fmaf(wc, u.y, o[1]), o[2] = fmaf(wc, u.z, o[2]), o[3] = fmaf(wc, u.w, o[3]);
        o[4] = fmaf(wc, v.x, o[4]), o[5] = fmaf(wc, v.y, o[5]), o[6] = fmaf(wc, v.z, o[6]), o[7] = fmaf(wc, v.w, o[7]);
      }
    }
  }
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) l += __shfl_xor_sync(0xffffffff, l, x);
  const bool live = tok < sequence(a, s, false).cnt;
  const float inv = l == 0.f ? 0.f : 1.f / l;  // 0: every score was -inf
  if (on) {
    const uint32_t gg[4] = {gw.x, gw.y, gw.z, gw.w};
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      float o0 = o[j] * inv, o1 = o[j + 1] * inv;
      if (a.gate) {
        o0 *= __fdividef(1.f, 1.f + __expf(-__uint_as_float(gg[j / 2] << 16)));
        o1 *= __fdividef(1.f, 1.f + __expf(-__uint_as_float(gg[j / 2] & 0xffff0000u)));
      }
      const __nv_bfloat162 h2 = __floats2bfloat162_rn(live ? o0 : 0.f, live ? o1 : 0.f);
      w[j / 2] = *reinterpret_cast<const uint32_t*>(&h2);
    }
    *reinterpret_cast<uint4*>(a.out + oi) = *reinterpret_cast<uint4*>(w);
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

// Tensor map over the pages as [rows][D], box `cols` x `rows`.
CUtensorMap pool_map(const void* base, const CacheView& c, int cols, int rows) {
  const int64_t n = c.pages * c.heads * c.page;
  if (!c.e4m3) return make_tmap_bf16(base, n, c.d, c.d, rows, cols);
  CUtensorMap map;
  cuuint64_t dims[2] = {(cuuint64_t)c.d, (cuuint64_t)n}, strides[1] = {(cuuint64_t)c.d};
  cuuint32_t box[2] = {(cuuint32_t)cols, (cuuint32_t)rows}, estr[2] = {1, 1};
  CUresult r = encode_fn()(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  NS_CHECK(r == CUDA_SUCCESS, "tree_attention: cuTensorMapEncodeTiled failed");
  return map;
}

template <int DT, bool E4M3>
void launch(const Args& a, int grid, const CacheView& c, const at::Tensor& q, const at::Tensor& k,
            const at::Tensor& v) {
  using C = Cfg<DT, E4M3>;
  static std::atomic<unsigned long long> attr{0};
  once_per_device(attr, [&] {
    NS_CUDA(cudaFuncSetAttribute(tree_attn_kernel<DT, E4M3>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
  });
  const CUtensorMap tq = node_map(q, a.GT, a.TPM), tk = node_map(k, 1, a.T), tv = node_map(v, 1, std::min(a.T, C::VK)),
                    tkp = pool_map(c.k, c, C::AC, std::min(c.page, BN)), tvp = pool_map(c.v, c, C::AC, std::min(c.page, C::VK));
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
  NS_VALUE(Hq >= 1 && c.heads >= 1 && Hq % c.heads == 0, "tree_attention: query heads must be a multiple of key heads");
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
  // positions are 32-bit, those of the last tile's end included
  NS_VALUE(table.size(1) * c.page <= (int64_t(1) << 31) - 2 * tattn::BN, "tree_attention: sequences of 2^31 rows");
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
  a.page_log2 = c.page == 16 ? 4 : c.page == 32 ? 5 : c.page == 64 ? 6 : 7;
  // measured at 2 and 4 (us): e4m3, one node of 64 ragged sequences, 522 and 487, bf16 short
  // trees 66 and 71 (71 at 1 too); an e4m3 segment also splits the nodes' rows
  a.seg = c.e4m3 ? 4 : 2;
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
  at::Tensor ws = at::empty({n_part + ((n_ml + 3) & ~int64_t(3)) + 2 * segs}, lse.options());
  a.part = ws.data_ptr<float>();
  a.ml = reinterpret_cast<float2*>(a.part + n_part);
  a.info = reinterpret_cast<int2*>(a.part + n_part + ((n_ml + 3) & ~int64_t(3)));
  // the narrowest tile that holds D; e4m3 operands are at least 128 wide (one swizzle atom)
  if (c.e4m3)
    D <= 128 ? tattn::launch<128, true>(a, grid, c, q, k, v) : tattn::launch<256, true>(a, grid, c, q, k, v);
  else if (D <= 64)
    tattn::launch<64, false>(a, grid, c, q, k, v);
  else
    D <= 128 ? tattn::launch<128, false>(a, grid, c, q, k, v) : tattn::launch<256, false>(a, grid, c, q, k, v);
  const int64_t nrows = b * T * Hq;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((nrows + 7) / 8));
  cfg.blockDim = dim3(256);
  cfg.stream = stream();
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  NS_CUDA(cudaLaunchKernelEx(&cfg, tattn::tree_join_kernel, a));
  return {out, lse};
}

}  // namespace ns
