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

// A CTA copies kTok consecutive tokens; V is the unit of the copies (16, 8, 4 or 2 bytes: the
// widest that every address and stride allows).  A thread keeps its place within the row (K or V,
// head, unit) and takes that unit of all the CTA's tokens: the loads, which need no slot, are all in
// flight while the slots arrive and are divided into page and row, once per token.
//
// Bound by HBM: 2 T Hkv D elements in and as many out.  32768 tokens of 8 heads of 128 bf16 (268 MB
// of traffic): one token per CTA 95 us, 8 tokens 48 us (5.6 TB/s; a plain copy runs at 6.5).  Below
// about 8 tokens per SM the CTAs would not cover the GPU, and one token per CTA ends sooner.
template <typename V, int kTok>
__global__ void __launch_bounds__(kWriteThreads) paged_write_kernel(const WriteParams p) {
  __shared__ int64_t s_page[kTok], s_row[kTok];  // page -1: no slot
  const int64_t t0 = (int64_t)blockIdx.x * kTok;
  const int tid = threadIdx.x;
  const int per_head = (int)(p.row_bytes / sizeof(V)), units = per_head * (int)p.Hkv;
  int u = tid;
  V x[kTok];
  bool is_v = false;
  int h = 0, c = 0;
  auto load = [&]() {  // unit u of every token
    is_v = u >= units;
    const int uu = is_v ? u - units : u;
    h = uu / per_head;
    c = uu - h * per_head;
    const int64_t* ns = is_v ? p.vns : p.kns;
    const char* src = (is_v ? p.vn : p.kn) + t0 * ns[0] + h * ns[1] + (int64_t)c * (int)sizeof(V);
#pragma unroll
    for (int j = 0; j < kTok; ++j)
      if (t0 + j < p.T) x[j] = *reinterpret_cast<const V*>(src + j * ns[0]);
  };
  if (u < 2 * units) load();
  if (tid < kTok) {
    const int64_t slot = t0 + tid < p.T ? p.slots[t0 + tid] : -1;
    int64_t page = slot < 0 ? -1 : slot / p.page;
    s_row[tid] = slot - page * p.page;
    if (page >= p.num_pages) {
      raise_status(p.status, kStatusBadIndex);
      page = -1;
    }
    s_page[tid] = page;
  }
  __syncthreads();
  while (u < 2 * units) {
    const int64_t* cs = is_v ? p.vs : p.ks;
    char* dst = (is_v ? p.vc : p.kc) + h * cs[1] + (int64_t)c * (int)sizeof(V);
#pragma unroll
    for (int j = 0; j < kTok; ++j)
      if (s_page[j] >= 0) *reinterpret_cast<V*>(dst + s_page[j] * cs[0] + s_row[j] * cs[2]) = x[j];
    u += kWriteThreads;
    if (u < 2 * units) load();
  }
  if (!p.routes) return;
  // Routing vectors, one warp per token: a page takes that of the last of its rows, i.e. of a row whose
  // next row with a slot is in another page (rows without one are passed over, 32 at a time).
  const int lane = tid & 31;
  constexpr bool kAll = kTok == 1;  // the CTA's warps share its only token
  for (int j = kAll ? 0 : tid >> 5; j < kTok; j += kAll ? 1 : kWriteThreads / 32) {
    const int64_t t = t0 + j, page = s_page[j];
    if (page < 0) continue;
    bool last = true;
    for (int64_t n0 = t + 1; n0 < p.T; n0 += 32) {
      const int64_t next = n0 + lane < p.T ? p.slots[n0 + lane] : -1;
      const unsigned has = __ballot_sync(0xffffffffu, next >= 0);
      if (!has) continue;
      const int64_t first = __shfl_sync(0xffffffffu, next, __ffs(has) - 1);
      last = first < page * p.page || first >= (page + 1) * p.page;
      break;
    }
    if (!last) continue;
    const int n = (int)(p.H * p.TD), TD = (int)p.TD;
    for (int i = kAll ? tid : lane; i < n; i += kAll ? kWriteThreads : 32) {
      const int hh = i / TD, l = i - hh * TD;
      const int64_t v = load_any_i64(p.routes, p.routes_dtype, t * p.rts[0] + hh * p.rts[1] + l * p.rts[2]);
      const int64_t o = page * p.rrs[0] + hh * p.rrs[1] + l * p.rrs[2];
      if (p.router_dtype == SA_I64)
        static_cast<int64_t*>(p.router)[o] = v;
      else
        static_cast<int32_t*>(p.router)[o] = (int32_t)v;
    }
  }
}

// Tokens per CTA: kWide where that still gives every SM a CTA, else 1.
constexpr int kWide = 8;

template <typename V>
void launch_write(const WriteParams& p, cudaStream_t s) {
  if (p.T >= (int64_t)kWide * device_sm_count())
    paged_write_kernel<V, kWide><<<(unsigned)((p.T + kWide - 1) / kWide), kWriteThreads, 0, s>>>(p);
  else
    paged_write_kernel<V, 1><<<(unsigned)p.T, kWriteThreads, 0, s>>>(p);
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
  if (T > INT32_MAX || Hkv * D > (1 << 24) || (routes && H * TD > (1 << 24)))
    return fail(SA_EUNSUPPORTED, "paged write: sizes too large");
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
  cudaStream_t s = (cudaStream_t)stream;
  if (bits % 16 == 0)
    launch_write<uint4>(p, s);
  else if (bits % 8 == 0)
    launch_write<uint2>(p, s);
  else if (bits % 4 == 0)
    launch_write<uint32_t>(p, s);
  else
    launch_write<uint16_t>(p, s);
  return check_launch("paged_write_kernel");
}

}  // extern "C"
