// Ragged write into the paged K/V cache: token t's K and V rows go to the cache row that a slot
// map names (slot = page * page_size + row; -1: none), and each page that receives tokens takes the
// routing vector of the last of them.
//
// The many-token form of paged.cu's append: prompts of any lengths and decode tokens of one step
// in one call.  Pure byte movement, every K/V byte read once and written once.
#include <algorithm>
#include <string>

#include "common.cuh"

namespace sa {
namespace {

constexpr int kWriteThreads = 256;

struct WriteParams {
  const char* kn;
  const char* vn;
  int64_t kns[2], vns[2];  // token, head strides in bytes
  const int64_t* slots;
  char* kc;
  char* vc;
  int64_t ks[3], vs[3];  // page, head, row strides in bytes
  const void* routes;    // (T, H, TD) or null
  int routes_dtype;
  int64_t rts[3];
  void* router;  // (P, H, TD)
  int router_dtype;
  int64_t rrs[3];
  int64_t T, Hkv, row_bytes, page, num_pages, H, TD;
  unsigned* status;
};

// One CTA per token; V is the unit of the copies (16, 8, 4 or 2 bytes: the widest that every
// address and stride allows).
template <typename V>
__global__ void __launch_bounds__(kWriteThreads) paged_write_kernel(const WriteParams p) {
  const int64_t t = blockIdx.x;
  const int64_t slot = p.slots[t];
  if (slot < 0) return;
  const int64_t page = slot / p.page, row = slot - page * p.page;
  if (page >= p.num_pages) {
    if (threadIdx.x == 0) raise_status(p.status, kStatusBadIndex);
    return;
  }
  const int per_head = (int)(p.row_bytes / sizeof(V)), units = per_head * (int)p.Hkv;
  for (int u = threadIdx.x; u < 2 * units; u += kWriteThreads) {
    const bool is_v = u >= units;
    const int uu = is_v ? u - units : u, h = uu / per_head, c = uu - h * per_head;
    const int64_t* ns = is_v ? p.vns : p.kns;
    const int64_t* cs = is_v ? p.vs : p.ks;
    const V* src = reinterpret_cast<const V*>((is_v ? p.vn : p.kn) + t * ns[0] + h * ns[1]) + c;
    V* dst = reinterpret_cast<V*>((is_v ? p.vc : p.kc) + page * cs[0] + h * cs[1] + row * cs[2]) + c;
    *dst = *src;
  }
  // the page's routing vector: from the last of its rows, i.e. where the next row with a slot is in
  // another page (rows without one are passed over, a block of them at a time)
  if (!p.routes) return;
  for (int64_t n0 = t + 1; n0 < p.T; n0 += kWriteThreads) {
    const int64_t n = n0 + threadIdx.x;
    const int64_t next = n < p.T ? p.slots[n] : -1;
    const bool found = next >= 0;
    __shared__ int64_t s_first;  // index of the first row with a slot in this block of rows
    if (threadIdx.x == 0) s_first = INT64_MAX;
    __syncthreads();
    if (found) atomicMin(reinterpret_cast<long long*>(&s_first), (long long)n);
    __syncthreads();
    const int64_t first = s_first;
    __syncthreads();  // s_first is set anew for the next block
    if (first == INT64_MAX) continue;
    if (p.slots[first] / p.page == page) return;
    break;
  }
  for (int64_t i = threadIdx.x; i < p.H * p.TD; i += kWriteThreads) {
    const int64_t h = i / p.TD, l = i - h * p.TD;
    const int64_t v = load_any_i64(p.routes, p.routes_dtype, t * p.rts[0] + h * p.rts[1] + l * p.rts[2]);
    const int64_t o = page * p.rrs[0] + h * p.rrs[1] + l * p.rrs[2];
    if (p.router_dtype == SA_I64)
      static_cast<int64_t*>(p.router)[o] = v;
    else
      static_cast<int32_t*>(p.router)[o] = (int32_t)v;
  }
}

}  // namespace
}  // namespace sa

extern "C" {

int sa_paged_kv_write(int dtype, int64_t T, int64_t Hkv, int64_t D, int64_t page_size, int64_t num_pages,
                      const void* k_new, const int64_t* k_new_strides, const void* v_new,
                      const int64_t* v_new_strides, const int64_t* slot_mapping, void* k_cache,
                      const int64_t* k_strides, void* v_cache, const int64_t* v_strides, const void* routes,
                      int routes_dtype, const int64_t* routes_strides, int64_t H, int64_t TD, void* router,
                      int router_dtype, const int64_t* router_strides, void* stream) {
  using namespace sa;
  if (T < 0 || Hkv <= 0 || D <= 0 || page_size <= 0 || num_pages < 0)
    return fail(SA_EINVAL, "paged write: bad sizes");
  if (dtype != SA_F32 && dtype != SA_F16 && dtype != SA_BF16)
    return fail(SA_EUNSUPPORTED, "paged write: dtype must be fp32, fp16 or bf16");
  if (T == 0) return SA_OK;
  if (!k_new || !v_new || !slot_mapping || !k_new_strides || !v_new_strides || !k_strides || !v_strides ||
      (num_pages && (!k_cache || !v_cache)))
    return fail(SA_EINVAL, "paged write: null pointer argument");
  if (k_new_strides[2] != 1 || v_new_strides[2] != 1 || k_strides[3] != 1 || v_strides[3] != 1)
    return fail(SA_EUNSUPPORTED, "paged write: head_dim must be contiguous");
  if (routes) {
    if (!router || !routes_strides || !router_strides || H <= 0 || TD <= 0)
      return fail(SA_EINVAL, "paged write: routes need the router table, strides, H and TD");
    if ((routes_dtype != SA_I32 && routes_dtype != SA_I64) || (router_dtype != SA_I32 && router_dtype != SA_I64))
      return fail(SA_EUNSUPPORTED, "paged write: routes must be int32 or int64");
  }
  if (T > INT32_MAX || Hkv * D > (1 << 24)) return fail(SA_EUNSUPPORTED, "paged write: sizes too large");
  if (int rc = check_stream_device(stream, "paged write")) return rc;
  const int64_t esz = dtype == SA_F32 ? 4 : 2;
  WriteParams p{};
  p.kn = static_cast<const char*>(k_new);
  p.vn = static_cast<const char*>(v_new);
  p.kc = static_cast<char*>(k_cache);
  p.vc = static_cast<char*>(v_cache);
  uint64_t bits = (uint64_t)(D * esz) | reinterpret_cast<uintptr_t>(k_new) | reinterpret_cast<uintptr_t>(v_new) |
                  reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache);
  for (int i = 0; i < 2; ++i) {
    p.kns[i] = k_new_strides[i] * esz;
    p.vns[i] = v_new_strides[i] * esz;
    bits |= (uint64_t)p.kns[i] | (uint64_t)p.vns[i];
  }
  for (int i = 0; i < 3; ++i) {
    p.ks[i] = k_strides[i] * esz;
    p.vs[i] = v_strides[i] * esz;
    bits |= (uint64_t)p.ks[i] | (uint64_t)p.vs[i];
    p.rts[i] = routes ? routes_strides[i] : 0;
    p.rrs[i] = routes ? router_strides[i] : 0;
  }
  p.slots = slot_mapping;
  p.routes = routes;
  p.routes_dtype = routes_dtype;
  p.router = router;
  p.router_dtype = router_dtype;
  p.T = T;
  p.Hkv = Hkv;
  p.row_bytes = D * esz;
  p.page = page_size;
  p.num_pages = num_pages;
  p.H = H;
  p.TD = TD;
  p.status = device_status_ptr();
  if (!p.status) return fail(SA_ELAUNCH, std::string("paged write: ") + sa_last_error());
  const unsigned grid = (unsigned)T;
  cudaStream_t s = (cudaStream_t)stream;
  if (bits % 16 == 0)
    paged_write_kernel<uint4><<<grid, kWriteThreads, 0, s>>>(p);
  else if (bits % 8 == 0)
    paged_write_kernel<uint2><<<grid, kWriteThreads, 0, s>>>(p);
  else if (bits % 4 == 0)
    paged_write_kernel<uint32_t><<<grid, kWriteThreads, 0, s>>>(p);
  else
    paged_write_kernel<uint16_t><<<grid, kWriteThreads, 0, s>>>(p);
  return check_launch("paged_write_kernel");
}

}  // extern "C"
