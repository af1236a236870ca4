// Shared declarations of the shared-prefix decode (general path and entry point in
// prefix_decode.cu, the tensor-core path in prefix_decode_sm100.cu).
#pragma once

#include "common.cuh"

namespace sa {

struct PrefixParams {
  int64_t B, H, Hkv, G, D, page, num_pages;
  int64_t Lp, L;  // widths of the prefix page list and of the block tables
  int64_t plen;   // prefix tokens where plen_dev is null
  const int32_t* plen_dev;
  int64_t TD, r, local_blocks;
  int sink;
  const void* q;
  int64_t qs[3];
  const void* kc;
  int64_t ks[4];
  const void* vc;
  int64_t vs[4];
  const int32_t* ppages;
  const int32_t* bt;
  int64_t bts[2];
  const int32_t* ctx;
  const void* router;
  int router_dtype;
  int64_t rs[3];
  const void* qrouter;
  int qrouter_dtype;
  int64_t qrs[3];
  void* out;
  int64_t os[3];
  float* lse;  // (B, H) natural log, or null
  unsigned* status;
};

// Tokens of the prefix and of request b's own pages, within the widths of their page lists.
__device__ __forceinline__ int64_t prefix_tokens(const PrefixParams& p) {
  const int64_t n = p.plen_dev ? (int64_t)*p.plen_dev : p.plen;
  return max((int64_t)0, min(n, p.Lp * p.page));
}
__device__ __forceinline__ int64_t own_tokens(const PrefixParams& p, int64_t b) {
  return max((int64_t)0, min((int64_t)p.ctx[b], p.L * p.page));
}

// Whether head h of request b attends logical page l (of n), held in physical page phys: kLevels levels
// in flight.  (The join, which needs it only for rows that are computed again, takes 1: more code there
// costs every call 2 us.)
template <int kLevels>
__device__ __forceinline__ bool page_attended(const PrefixParams& p, int64_t b, int64_t h, int64_t l, int64_t n,
                                              int64_t phys) {
  if ((p.sink && l == 0) || l >= n - p.local_blocks) return true;
#pragma unroll 1
  for (int64_t i0 = 0; i0 < p.r; i0 += kLevels) {  // those past r repeat the last
    bool same = true;
#pragma unroll
    for (int k = 0; k < kLevels; ++k) {
      const int64_t i = min(i0 + k, p.r - 1);
      same &= load_any_i64(p.router, p.router_dtype, phys * p.rs[0] + h * p.rs[1] + i * p.rs[2]) ==
              load_any_i64(p.qrouter, p.qrouter_dtype, b * p.qrs[0] + h * p.qrs[1] + i * p.qrs[2]);
    }
    if (!same) return false;
  }
  return true;
}

// Tensor-core path: bf16/fp16, D % 8 == 0 and <= 128, page % 8 == 0, <= 128 query heads per KV
// head and <= 256 in all (prefix_fast_shape), 16-byte aligned rows, and page lists whose tiles
// can be counted in 32 bits (prefix_fast_eligible).
bool prefix_fast_shape(int dtype, int64_t B, int64_t H, int64_t Hkv, int64_t D, int64_t page);
bool prefix_fast_eligible(const PrefixParams& p, int dtype);
int64_t prefix_fast_workspace_bytes(int64_t B, int64_t H, int64_t Hkv, int64_t D, int64_t page, int64_t Lp, int64_t L);
int launch_prefix_fast(const PrefixParams& p, int dtype, void* workspace, cudaStream_t stream);

}  // namespace sa
