// What the decode-step calls share: the cache as the kernels see it, places of positions in it, rounded
// division, the workspace, and the checks of arguments.
#pragma once
#include <cstdarg>
#include <cstdint>

#include "ctx.cuh"

namespace grape {

// n / d by one high product (d >= 1; Granlund and Montgomery's division by invariant integers): with l = ceil(log2 d) and
// m = floor(2^32 (2^l - d) / d) + 1 the quotient is (hi(m n) + n) >> l.
struct FastDiv {
  uint32_t d, m, l;
  static FastDiv of(uint32_t d) {
    uint32_t l = 0;
    while ((uint64_t(1) << l) < d) l++;
    return {d, (uint32_t)(((uint64_t(1) << 32) * ((uint64_t(1) << l) - d)) / d + 1), l};
  }
  __host__ __device__ uint32_t div(uint32_t n) const {
    return (uint32_t)(((((uint64_t)m * n) >> 32) + n) >> l);
  }
};

struct KvView {
  char *k, *v, *bounds;
  int64_t page_stride, head_stride, slot_stride;  // bytes
  uint32_t n_pages, page_size, kv_heads, head_dim;
  FastDiv by_page;
  const int32_t* table;
  uint32_t width, batch;
  uint32_t* status;
};

__device__ __forceinline__ void kv_flag(const KvView& c, uint32_t bit) { atomicOr(c.status, bit); }

// Page number of place `at` (a page's index in its sequence) of sequence b, or -1 outside the cache.
__device__ __forceinline__ int32_t kv_page(const KvView& c, uint32_t b, uint32_t at) {
  if (at >= c.width) return -1;
  const int32_t p = __ldg(c.table + (uint64_t)b * c.width + at);
  return (uint32_t)p < c.n_pages ? p : -1;
}

// Tokens of sequence b that the table can hold; a length outside [0, that] sets the status bit.
__device__ __forceinline__ uint32_t kv_length(const KvView& c, const int32_t* d_len, uint32_t b, uint64_t most, bool report) {
  const int64_t n = __ldg(d_len + b);
  const uint64_t cap = min((uint64_t)c.width * c.page_size, most);
  if (n >= 0 && (uint64_t)n <= cap) return (uint32_t)n;
  if (report) kv_flag(c, STATUS_KV_PLACE);
  return n < 0 ? 0u : (uint32_t)cap;
}

// Rounded division by 2^s; the sums wrap like unsigned ones, so no input has undefined results.
__device__ __forceinline__ int64_t rdiv(int64_t x, uint32_t s) {
  return (int64_t)((uint64_t)x + ((uint64_t(1) << s) >> 1)) >> s;
}

__device__ __forceinline__ int32_t saturate(int64_t x, int64_t low, int64_t high, bool& out_of_range) {
  if (x < low) { out_of_range = true; return (int32_t)low; }
  if (x > high) { out_of_range = true; return (int32_t)high; }
  return (int32_t)x;
}

// Asynchronous copies into a lane's own queue in shared memory.
template <int BYTES>
__device__ __forceinline__ void copy_async(void* to, const void* from) {
  if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// ---- host side ---------------------------------------------------------------------------------
int kv_refuse(grape_ctx* ctx, int code, const char* format, ...);
int kv_check_cache(grape_ctx* ctx, const grape_kv_cache* c, const int32_t* d_table, uint32_t width, uint32_t batch,
                   bool keys, bool values, bool bounds);
int kv_check_rows(grape_ctx* ctx, const char* what, const int32_t* d, uint64_t stride, uint64_t row);
KvView kv_view(grape_ctx* ctx, const grape_kv_cache* c, const int32_t* d_table, uint32_t width, uint32_t batch);
// `bytes` of the context's decode-step workspace; the same address for every call that fits the block.
int kv_workspace(grape_ctx* ctx, size_t bytes, void** out);

// Raises a kernel's limit of dynamic shared memory to `most`, once: the call would cost as much as a launch.
template <class K>
inline int kv_allow_shared(grape_ctx* ctx, K* kernel, size_t most) {
  const void* k = reinterpret_cast<const void*>(kernel);
  for (const void* have : ctx->kv_allowed)
    if (have == k) return GRAPE_OK;
  GRAPE_CUDA_TRY(ctx, cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
  ctx->kv_allowed.push_back(k);
  return GRAPE_OK;
}

inline bool misaligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

}  // namespace grape
