// Argument checks shared by the decoding ops (kv_cache.cu, tree_attn.cu, gdn_decode.cu).
#pragma once

#include "common.h"

// Bad arguments of the decoding ops are ValueErrors, as on the CPU path.
#define NS_VALUE(cond, ...) TORCH_CHECK_VALUE(cond, "nanospec_b200: ", __VA_ARGS__)

namespace ns {

using OptTensor = c10::optional<at::Tensor>;

// Device error word code of an index value out of range (the access was skipped).
constexpr int ERR_INDEX = 4;
constexpr int MAX_NODES = 64;  // nodes of one tree

// The pages of one layer's cache, checked.
struct CacheView {
  int64_t pages;
  int heads, page, d;
  bool e4m3;
  const void *k, *v;
  const uint8_t *ke, *ve;
};

inline CacheView check_cache(const at::Tensor& k, const at::Tensor& v, const OptTensor& ke, const OptTensor& ve) {
  NS_VALUE(k.is_cuda() && v.is_cuda() && k.device() == v.device(), "cache: pages must be on one CUDA device");
  NS_VALUE(k.dim() == 4 && k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type(),
           "cache: k and v pages differ");
  NS_VALUE(k.is_contiguous() && v.is_contiguous(), "cache: pages must be contiguous");
  const int64_t page = k.size(2), d = k.size(3);
  NS_VALUE(page == 16 || page == 32 || page == 64 || page == 128, "cache: page_size must be 16, 32, 64 or 128");
  NS_VALUE(d % 16 == 0 && d >= 16 && d <= 256, "cache: head_dim must be a multiple of 16 up to 256");
  NS_VALUE(k.size(0) * k.size(1) * page < (int64_t(1) << 31), "cache: more than 2^31 rows");
  NS_VALUE(reinterpret_cast<uintptr_t>(k.data_ptr()) % 16 == 0 && reinterpret_cast<uintptr_t>(v.data_ptr()) % 16 == 0,
           "cache: pages must be 16-byte aligned");
  CacheView c{k.size(0), (int)k.size(1), (int)page, (int)d, k.scalar_type() == at::kFloat8_e4m3fn,
              k.data_ptr(), v.data_ptr(), nullptr, nullptr};
  if (c.e4m3) {
    for (const OptTensor* e : {&ke, &ve}) {
      NS_VALUE(e->has_value() && (*e)->scalar_type() == at::kByte && (*e)->device() == k.device() &&
                   (*e)->sizes() == k.sizes().slice(0, 3) && (*e)->is_contiguous() &&
                   reinterpret_cast<uintptr_t>((*e)->data_ptr()) % 16 == 0,
               "cache: e4m3 pages need aligned uint8 exponents [pages, heads, page_size]");
    }
    c.ke = ke->data_ptr<uint8_t>();
    c.ve = ve->data_ptr<uint8_t>();
  } else {
    NS_VALUE(k.scalar_type() == at::kBFloat16, "cache: pages must be bfloat16 or float8_e4m3fn");
    NS_VALUE(!ke.has_value() && !ve.has_value(), "cache: only e4m3 pages have exponents");
  }
  return c;
}

// An int32 index tensor [n] on `dev`.
inline const int* check_index(const at::Tensor& t, int64_t n, const at::Device& dev, const char* name) {
  NS_VALUE(t.device() == dev && t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n && t.is_contiguous(),
           name, " must be a contiguous int32 tensor with one entry per sequence on the same device");
  return t.data_ptr<int>();
}

inline const int* check_index(const OptTensor& t, int64_t n, const at::Device& dev, const char* name) {
  return t.has_value() ? check_index(*t, n, dev, name) : nullptr;
}

// parents [T] (shared, stride 0) or [b, T] int32: pointer and row stride.
inline const int* check_parents(const at::Tensor& p, int64_t b, int64_t t, const at::Device& dev, int64_t& stride) {
  const bool one = p.dim() == 1 && p.size(0) == t;
  const bool many = p.dim() == 2 && p.size(0) == b && p.size(1) == t;
  NS_VALUE(p.device() == dev && p.scalar_type() == at::kInt && (one || many) && (t <= 1 || p.stride(-1) == 1),
           "parents must be int32 [T] or [b, T]");
  stride = one ? 0 : p.stride(0);
  return p.data_ptr<int>();
}

// Whether 16-byte accesses may start at t's first element.
inline bool aligned16(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// t, dense and 16-byte aligned: anything else is copied (`contiguous` alone keeps a dense view
// that begins at an odd offset of its storage).
inline at::Tensor aligned_dense(const at::Tensor& t) {
  return t.is_contiguous() && aligned16(t) ? t : t.clone(at::MemoryFormat::Contiguous);
}

// A bf16 operand [.., heads, D] on `dev` as the kernels read it: D contiguous, every row
// 16-byte aligned; anything else is copied.
inline at::Tensor aligned_rows(const at::Tensor& t) {
  bool ok = (t.size(-1) <= 1 || t.stride(-1) == 1) && aligned16(t);
  for (int i = 0; i + 1 < t.dim(); ++i) ok = ok && (t.size(i) <= 1 || t.stride(i) % 8 == 0);
  return ok ? t : aligned_dense(t);
}

}  // namespace ns
