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
// Both kernels move each byte once and are bound by HBM.
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
  int64_t n, pages;
  int heads, page, d;
  int* err;
};

// One warp per (token, head) row of K (blockIdx.y = 0) or V (1); lane l holds channels
// [8l, 8l + 8).
template <bool E4M3>
__global__ void __launch_bounds__(256) cache_write_kernel(WriteArgs a) {
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, which = blockIdx.y;
  if (row >= a.n * a.heads) return;
  const int64_t tok = row / a.heads;
  const int h = (int)(row % a.heads);
  const int64_t slot = a.slots[tok];
  if (slot < 0 || slot >= a.pages * a.page) {
    if (slot != -1 && lane == 0) atomicExch(a.err, ERR_INDEX);
    return;
  }
  const int64_t dst = ((slot / a.page) * a.heads + h) * a.page + slot % a.page;
  const bool on = lane * 8 < a.d;
  uint4 raw = make_uint4(0, 0, 0, 0);
  if (on) raw = *reinterpret_cast<const uint4*>(a.x[which] + tok * a.x_ts[which] + h * a.x_hs[which] + lane * 8);
  if constexpr (!E4M3) {
    if (on) *reinterpret_cast<uint4*>(reinterpret_cast<bf16*>(a.pool[which]) + dst * a.d + lane * 8) = raw;
  } else {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    float x[8];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t b = (i & 1) ? (w[i / 2] & 0xffff0000u) : (w[i / 2] << 16);
      x[i] = __uint_as_float(b);
      const uint32_t m = b & 0x7fffffffu;
      top = max(top, m < 0x7f800000u ? m : 0u);  // infinities and NaN do not count
    }
    top = __reduce_max_sync(0xffffffff, top);
    const int e = row_exponent(top);
    const float s = pow2(-e);
    uint32_t code[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const __nv_fp8x2_storage_t c =
          __nv_cvt_float2_to_fp8x2(make_float2(x[i] * s, x[i + 1] * s), __NV_SATFINITE, __NV_E4M3);
      code[i / 4] |= (uint32_t)c << (8 * (i & 3));
    }
    if (on)
      *reinterpret_cast<uint2*>(reinterpret_cast<uint8_t*>(a.pool[which]) + dst * a.d + lane * 8) =
          make_uint2(code[0], code[1]);
    if (lane == 0) a.exps[which][dst] = (uint8_t)(e + EXP_BIAS);
  }
}

struct ReadArgs {
  const void* pool[2];
  const uint8_t* exps[2];
  bf16* out[2];
  const int *table, *lens, *starts;
  int64_t b, length, pages, max_pages;
  int heads, page, d;
  int* err;
};

// One thread per 8 channels of (sequence, position, head) of K (blockIdx.y = 0) or V (1).
template <bool E4M3>
__global__ void __launch_bounds__(256) cache_read_kernel(ReadArgs a) {
  const int cols = a.d / 8;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int which = blockIdx.y;
  if (i >= a.b * a.length * a.heads * cols) return;
  const int c = (int)(i % cols);
  const int64_t r = i / cols;
  const int h = (int)(r % a.heads);
  const int64_t bt = r / a.heads;
  const int64_t s = bt / a.length;
  const int64_t pos = bt % a.length + (a.starts ? a.starts[s] : 0);
  uint4 out = make_uint4(0, 0, 0, 0);
  const int64_t len = min((int64_t)a.lens[s], a.max_pages * a.page);
  if (c == 0 && h == 0 && (a.lens[s] != len || len < 0 || pos < 0)) atomicExch(a.err, ERR_INDEX);
  if (pos >= 0 && pos < len) {
    const int64_t pg = a.table[s * a.max_pages + pos / a.page];
    if (pg < 0 || pg >= a.pages) {
      if (c == 0) atomicExch(a.err, ERR_INDEX);
    } else {
      const int64_t src = (pg * a.heads + h) * a.page + pos % a.page;
      if constexpr (!E4M3) {
        out = *reinterpret_cast<const uint4*>(reinterpret_cast<const bf16*>(a.pool[which]) + src * a.d + c * 8);
      } else {
        const uint2 code =
            *reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(a.pool[which]) + src * a.d + c * 8);
        const float sc = pow2(min(max((int)a.exps[which][src] - EXP_BIAS, EXP_MIN), EXP_MAX));
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t pair = ((j < 2 ? code.x : code.y) >> (16 * (j & 1))) & 0xffff;
          const __half2_raw hr = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)pair, __NV_E4M3);
          const float2 f = __half22float2(__half2(hr));
          const __nv_bfloat162 o = __floats2bfloat162_rn(f.x * sc, f.y * sc);
          w[j] = *reinterpret_cast<const uint32_t*>(&o);
        }
        out = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
  *reinterpret_cast<uint4*>(a.out[which] + i * 8) = out;
}

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
  a.slots = slots.data_ptr<int64_t>();
  a.n = k.size(0);
  a.pages = c.pages;
  a.heads = c.heads;
  a.page = c.page;
  a.d = c.d;
  a.err = device_error_flag();
  NS_VALUE((rows + 7) / 8 < (int64_t(1) << 31), "cache_write: too many rows");
  const dim3 grid((unsigned)((rows + 7) / 8), 2);
  if (c.e4m3)
    kvc::cache_write_kernel<true><<<grid, 256, 0, stream()>>>(a);
  else
    kvc::cache_write_kernel<false><<<grid, 256, 0, stream()>>>(a);
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
  const int64_t n = b * length * c.heads * (c.d / 8);
  if (n == 0) return {ko, vo};
  a.pool[0] = c.k;
  a.pool[1] = c.v;
  a.exps[0] = c.ke;
  a.exps[1] = c.ve;
  a.out[0] = reinterpret_cast<bf16*>(ko.data_ptr());
  a.out[1] = reinterpret_cast<bf16*>(vo.data_ptr());
  a.b = b;
  a.length = length;
  a.pages = c.pages;
  a.max_pages = table.size(1);
  a.heads = c.heads;
  a.page = c.page;
  a.d = c.d;
  a.err = device_error_flag();
  NS_VALUE((n + 255) / 256 < (int64_t(1) << 31), "cache_read: too many rows");
  const dim3 grid((unsigned)((n + 255) / 256), 2);
  if (c.e4m3)
    kvc::cache_read_kernel<true><<<grid, 256, 0, stream()>>>(a);
  else
    kvc::cache_read_kernel<false><<<grid, 256, 0, stream()>>>(a);
  NS_CUDA(cudaGetLastError());
  return {ko, vo};
}

}  // namespace ns
