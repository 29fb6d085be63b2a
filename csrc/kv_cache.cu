// Paged K/V cache: rows quantised as they are written, and read back.
//
// A row x[D] of one (token, head) is kept as bf16, or as e4m3 codes with one power-of-two
// scale: with a the largest finite |x|, e is the smallest integer for which
// a <= 448 * 2^e, clamped to [-117, 118] (-117 for a row of zeros, so that
// it never sets the scale of others), and
//   code = e4m3(x * 2^-e)  (nearest even, saturating, NaN kept),   byte = e + 127,
//   read  = code * 2^e.
// Multiplying by a power of two is exact both ways and bf16 holds every code * 2^e, so the
// only rounding is e4m3's own. e follows from the bits of a: a = 1.m * 2^E needs e = E - 8
// when 1.m <= 1.75 (448 = 1.75 * 2^8) and E - 7 otherwise.
//
// Both kernels move each byte once: 16 channels per thread (16 bytes of codes, 32 of bf16), index
// arithmetic in 32 bits with shifts, several rows' loads under way. Writing 12288 rows x 8 heads x
// 128 as e4m3 and reading 33147 back: 99 us, 2.8 TB/s (one 8-channel thread per element group
// with 64-bit divisions: 338 us). Less than half the copy rate: neighbouring threads take the heads
// of one position, whose rows lie in different runs of the pages (a head's rows of one page adjoin),
// and the arguments are indexed by block, so each thread holds a copy in local memory.
#include <cuda_fp8.h>

#include "decode.h"
#include "sm100.cuh"

namespace ns {

using bf16 = __nv_bfloat16;

namespace kvc {

constexpr int EXP_BIAS = 127, EXP_MIN = -117, EXP_MAX = 118;

// exponent byte of a row whose largest finite magnitude has the fp32 bits `a`
__device__ __forceinline__ int row_exponent(uint32_t a) {
  const int E = (int)(a >> 23) - 127;  // zero and subnormals are far below EXP_MIN
  const int e = E - 8 + ((a & 0x7fffff) > 0x600000 ? 1 : 0);
  return min(max(e, EXP_MIN), EXP_MAX);
}

__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

struct WriteArgs {
  const bf16* x[2];
  int64_t x_ts[2], x_hs[2];  // element strides of token and head
  void* pool[2];
  uint8_t* exps[2];
  const int64_t* slots;
  int64_t slots_end;
  int n, heads, page_log2, d;
  int* err;
};

// 16 channels per thread, G (a power of two) neighbouring lanes per (token, head) row of K
// (blockIdx.y = 0) or V (1); two rows per thread, so that two rows' loads are under way.
template <bool E4M3, int G>
__global__ void __launch_bounds__(256) cache_write_kernel(WriteArgs a) {
  const int which = blockIdx.y, c = threadIdx.x % G * 16;
  const unsigned r0 = blockIdx.x * (512 / G) + threadIdx.x / G, rows = (unsigned)a.n * a.heads;
  uint4 w[2][2];
  int64_t dst[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const unsigned r = r0 + i * (256 / G);
    dst[i] = -1;
    w[i][0] = w[i][1] = make_uint4(0, 0, 0, 0);
    if (r < rows) {
      const unsigned tok = r / a.heads, h = r % a.heads;
      const int64_t slot = a.slots[tok];
      if (slot >= 0 && slot < a.slots_end)
        dst[i] = ((((slot >> a.page_log2) * a.heads + h) << a.page_log2) + (slot & ((1 << a.page_log2) - 1)));
      else if (slot != -1 && c == 0)
        atomicExch(a.err, ERR_INDEX);
      if (dst[i] >= 0 && c < a.d) {
        const uint4* x = reinterpret_cast<const uint4*>(a.x[which] + tok * a.x_ts[which] + h * a.x_hs[which] + c);
        w[i][0] = x[0];
        w[i][1] = x[1];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (!E4M3) {
      if (dst[i] >= 0 && c < a.d) {
        uint4* o = reinterpret_cast<uint4*>(reinterpret_cast<bf16*>(a.pool[which]) + dst[i] * a.d + c);
        o[0] = w[i][0];
        o[1] = w[i][1];
      }
    } else {
      const uint32_t in[8] = {w[i][0].x, w[i][0].y, w[i][0].z, w[i][0].w, w[i][1].x, w[i][1].y, w[i][1].z, w[i][1].w};
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {  // infinities and NaN do not count
        const uint32_t lo = (in[j] << 16) & 0x7fffffffu, hi = in[j] & 0x7fff0000u;
        top = max(top, max(lo < 0x7f800000u ? lo : 0u, hi < 0x7f800000u ? hi : 0u));
      }
#pragma unroll
      for (int o = G / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffff, top, o));
      const int e = row_exponent(top);
      const float s = pow2(-e);
      uint32_t code[4];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const __nv_fp8x2_storage_t p = __nv_cvt_float2_to_fp8x2(
            make_float2(__uint_as_float(in[j] << 16) * s, __uint_as_float(in[j] & 0xffff0000u) * s), __NV_SATFINITE,
            __NV_E4M3);
        code[j / 2] = j & 1 ? code[j / 2] | (uint32_t)p << 16 : (uint32_t)p;
      }
      if (dst[i] >= 0) {
        if (c < a.d)
          *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(a.pool[which]) + dst[i] * a.d + c) =
              make_uint4(code[0], code[1], code[2], code[3]);
        if (c == 0) a.exps[which][dst[i]] = (uint8_t)(e + EXP_BIAS);
      }
    }
  }
}

struct ReadArgs {
  const void* pool[2];
  const uint8_t* exps[2];
  bf16* out[2];
  const int *table, *lens, *starts;
  int length, pages, max_pages, heads, page_log2, d, per;
  int* err;
};

constexpr int READ_POS = 32;  // positions of one CTA

// CTA: 32 positions of one sequence, K or V (blockIdx.z). Thread: 16 channels of one head at
// every `per`-th position; neighbouring threads write neighbouring bytes.
template <bool E4M3>
__global__ void __launch_bounds__(256) cache_read_kernel(ReadArgs a) {
  const int s = blockIdx.y, which = blockIdx.z, cols = a.d / 16, hc = a.heads * cols;
  const int p0 = blockIdx.x * READ_POS;
  const int64_t first = a.starts ? a.starts[s] : 0;
  int64_t len = a.lens[s];
  const int64_t most = (int64_t)a.max_pages << a.page_log2;
  if (len < 0 || len > most || first < 0) {
    if (threadIdx.x == 0) atomicExch(a.err, ERR_INDEX);
    len = first < 0 ? 0 : min(max(len, (int64_t)0), most);
  }
  const int* table = a.table + (int64_t)s * a.max_pages;
  for (int x0 = threadIdx.x; x0 < hc * a.per; x0 += 256) {
    const int x = x0 % hc, h = x / cols, c = x % cols * 16;
    bf16* out = a.out[which] + ((int64_t)s * a.length * a.heads + h) * a.d + c;
#pragma unroll 4
    for (int i = x0 / hc; i < READ_POS; i += a.per) {
      if (p0 + i >= a.length) break;
      const int64_t pos = first + p0 + i;
      uint4 w[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
      if (pos < len) {
        const int pg = table[pos >> a.page_log2];
        if (pg < 0 || pg >= a.pages) {
          atomicExch(a.err, ERR_INDEX);
        } else {
          const int64_t src = (((int64_t)pg * a.heads + h) << a.page_log2) + (pos & ((1 << a.page_log2) - 1));
          if constexpr (!E4M3) {
            const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<const bf16*>(a.pool[which]) + src * a.d + c);
            w[0] = p[0];
            w[1] = p[1];
          } else {
            const uint4 code =
                *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(a.pool[which]) + src * a.d + c);
            const float sc = pow2(min(max((int)a.exps[which][src] - EXP_BIAS, EXP_MIN), EXP_MAX));
            const uint32_t in[4] = {code.x, code.y, code.z, code.w};
            uint32_t o[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const uint32_t pair = (in[j / 2] >> (16 * (j & 1))) & 0xffff;
              const float2 f =
                  __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)pair, __NV_E4M3)));
              const __nv_bfloat162 v = __floats2bfloat162_rn(f.x * sc, f.y * sc);
              o[j] = *reinterpret_cast<const uint32_t*>(&v);
            }
            w[0] = make_uint4(o[0], o[1], o[2], o[3]);
            w[1] = make_uint4(o[4], o[5], o[6], o[7]);
          }
        }
      }
      uint4* o = reinterpret_cast<uint4*>(out + (int64_t)(p0 + i) * a.heads * a.d);
      o[0] = w[0];
      o[1] = w[1];
    }
  }
}

inline int log2_of(int page) { return page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : 7; }

}  // namespace kvc

void cache_write(at::Tensor k_pool, at::Tensor v_pool, OptTensor k_exp, OptTensor v_exp, at::Tensor k, at::Tensor v,
                 at::Tensor slots) {
  const CacheView c = check_cache(k_pool, v_pool, k_exp, v_exp);
  const at::cuda::CUDAGuard guard(k_pool.device());
  for (const at::Tensor* x : {&k, &v})
    NS_VALUE(x->device() == k_pool.device() && x->scalar_type() == at::kBFloat16 && x->dim() == 3 &&
                 x->size(0) == k.size(0) && x->size(1) == c.heads && x->size(2) == c.d,
             "cache_write: k and v must be bfloat16 [n, heads, D] on the cache's device");
  NS_VALUE(slots.device() == k_pool.device() && slots.scalar_type() == at::kLong && slots.dim() == 1 &&
               slots.size(0) == k.size(0) && slots.is_contiguous(),
           "cache_write: slots must be int64 [n]");
  const int64_t rows = k.size(0) * c.heads;
  if (rows == 0) return;
  k = aligned_rows(k);
  v = aligned_rows(v);
  kvc::WriteArgs a{};
  const at::Tensor* xs[2] = {&k, &v};
  for (int i = 0; i < 2; ++i) {
    a.x[i] = reinterpret_cast<const bf16*>(xs[i]->data_ptr());
    a.x_ts[i] = xs[i]->stride(0);
    a.x_hs[i] = xs[i]->stride(1);
  }
  a.pool[0] = k_pool.data_ptr();
  a.pool[1] = v_pool.data_ptr();
  a.exps[0] = const_cast<uint8_t*>(c.ke);
  a.exps[1] = const_cast<uint8_t*>(c.ve);
  NS_VALUE(rows < (int64_t(1) << 31), "cache_write: too many rows");
  a.slots = slots.data_ptr<int64_t>();
  a.slots_end = c.pages * c.page;
  a.n = (int)k.size(0);
  a.heads = c.heads;
  a.page_log2 = kvc::log2_of(c.page);
  a.d = c.d;
  a.err = device_error_flag();
#define NS_X(G)                                                                      \
  {                                                                                  \
    const dim3 grid((unsigned)((rows + 512 / G - 1) / (512 / G)), 2);                \
    if (c.e4m3)                                                                      \
      kvc::cache_write_kernel<true, G><<<grid, 256, 0, stream()>>>(a);               \
    else                                                                             \
      kvc::cache_write_kernel<false, G><<<grid, 256, 0, stream()>>>(a);              \
  }
  if (c.d <= 64) NS_X(4) else if (c.d <= 128) NS_X(8) else NS_X(16)
#undef NS_X
  NS_CUDA(cudaGetLastError());
}

std::vector<at::Tensor> cache_read(at::Tensor k_pool, at::Tensor v_pool, OptTensor k_exp, OptTensor v_exp,
                                   at::Tensor table, at::Tensor lens, OptTensor starts, int64_t length) {
  const CacheView c = check_cache(k_pool, v_pool, k_exp, v_exp);
  const at::Device dev = k_pool.device();
  const at::cuda::CUDAGuard guard(dev);
  NS_VALUE(lens.dim() == 1 && length >= 0, "cache_read: lens must be [b] and length not negative");
  const int64_t b = lens.size(0);
  kvc::ReadArgs a{};
  a.lens = check_index(lens, b, dev, "lens");
  a.starts = check_index(starts, b, dev, "starts");
  NS_VALUE(table.device() == dev && table.scalar_type() == at::kInt && table.dim() == 2 && table.size(0) == b &&
               table.is_contiguous(),
           "table must be contiguous int32 [b, max_pages]");
  a.table = table.data_ptr<int>();
  auto opt = k_pool.options().dtype(at::kBFloat16);
  at::Tensor ko = at::empty({b, length, c.heads, c.d}, opt), vo = at::empty({b, length, c.heads, c.d}, opt);
  if (b * length * c.heads == 0) return {ko, vo};
  NS_VALUE(b < 65536 && length < (int64_t(1) << 31) && table.size(1) < (int64_t(1) << 31),
           "cache_read: too many sequences or positions");
  a.pool[0] = c.k;
  a.pool[1] = c.v;
  a.exps[0] = c.ke;
  a.exps[1] = c.ve;
  a.out[0] = reinterpret_cast<bf16*>(ko.data_ptr());
  a.out[1] = reinterpret_cast<bf16*>(vo.data_ptr());
  a.length = (int)length;
  a.pages = (int)c.pages;
  a.max_pages = (int)table.size(1);
  a.heads = c.heads;
  a.page_log2 = kvc::log2_of(c.page);
  a.d = c.d;
  a.per = std::max(1, std::min(kvc::READ_POS, 256 / (c.heads * (c.d / 16))));
  a.err = device_error_flag();
  const dim3 grid((unsigned)((length + kvc::READ_POS - 1) / kvc::READ_POS), (unsigned)b, 2);
  if (c.e4m3)
    kvc::cache_read_kernel<true><<<grid, 256, 0, stream()>>>(a);
  else
    kvc::cache_read_kernel<false><<<grid, 256, 0, stream()>>>(a);
  NS_CUDA(cudaGetLastError());
  return {ko, vo};
}

}  // namespace ns
