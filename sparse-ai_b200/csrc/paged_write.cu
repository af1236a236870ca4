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
constexpr int kMaxGroups = 16;

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
  int groups;  // token groups side by side in a CTA
  unsigned* status;
};

// A CTA copies groups * kTok consecutive tokens; V is the unit of the copies (16, 8, 4 or 2 bytes: the
// widest that every address and stride allows).  A token takes 2 Hkv row_bytes / sizeof(V) threads
// (at most all of them, in turns); where that is a half or less of the CTA, `groups` of them work
// side by side on neighbouring tokens.  A thread keeps its place within the row (K or V, head, unit)
// and takes that unit of its kTok tokens: the loads, which need no slot, are all in flight while
// the slots arrive and are divided into page and row, once per token.
//
// Bound by HBM: 2 T Hkv D elements in and as many out.  32768 tokens of 8 heads of 128 bf16 (268 MB
// of traffic): one token per CTA 95 us, 8 tokens 46 us (5.9 TB/s; a plain copy runs at 6.5).  Below
// about 8 tokens per SM the CTAs would not cover the GPU, and one token per CTA ends sooner.
// 32768 tokens of 2 heads of 64 bf16 (32 threads a token): one group 14.3 us, 8 groups 10.0.
template <typename V, int kTok>
__global__ void __launch_bounds__(kWriteThreads) paged_write_kernel(const WriteParams p) {
  __shared__ int64_t s_page[kTok * kMaxGroups], s_row[kTok * kMaxGroups];  // page -1: no slot
  const int groups = p.groups, tokens = kTok * groups;
  const int64_t t0 = (int64_t)blockIdx.x * tokens;
  const int tid = threadIdx.x;
  const int per_head = (int)(p.row_bytes / sizeof(V)), units = per_head * (int)p.Hkv;
  int u = tid, g = 0;
  if (groups > 1) {
    g = tid / (2 * units);
    u = g < groups ? tid - g * 2 * units : 2 * units;
  }
  V x[kTok];
  bool is_v = false;
  int h = 0, c = 0;
  auto load = [&]() {  // unit u of tokens g, g + groups, ...
    is_v = u >= units;
    const int uu = is_v ? u - units : u;
    h = uu / per_head;
    c = uu - h * per_head;
    const int64_t* ns = is_v ? p.vns : p.kns;
    const char* src = (is_v ? p.vn : p.kn) + (t0 + g) * ns[0] + h * ns[1] + (int64_t)c * (int)sizeof(V);
    const int64_t step = groups * ns[0];
#pragma unroll
    for (int j = 0; j < kTok; ++j)
      if (t0 + g + j * groups < p.T) x[j] = *reinterpret_cast<const V*>(src + j * step);
  };
  if (u < 2 * units) load();
  if (tid < tokens) {
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
    for (int j = 0; j < kTok; ++j) {
      const int i = g + j * groups;
      if (s_page[i] >= 0) *reinterpret_cast<V*>(dst + s_page[i] * cs[0] + s_row[i] * cs[2]) = x[j];
    }
    u += kWriteThreads;
    if (u < 2 * units) load();
  }
  if (!p.routes) return;
  // Routing vectors, one warp per token: a page takes that of the last of its rows, i.e. of a row whose
  // next row with a slot is in another page.  Rows without one are passed over: 32 at first, then 512
  // at a time (a batch padded to a fixed size ends in thousands of them).  So are those whose slot lies
  // past the cache: taken for another page's, they would leave a page with two last rows, and two
  // warps writing its vector.
  const int lane = tid & 31;
  const uint64_t slots_end = (uint64_t)(p.num_pages * p.page);
  const bool all = tokens == 1;  // the CTA's warps share its only token
  for (int j = all ? 0 : tid >> 5; j < tokens; j += all ? 1 : kWriteThreads / 32) {
    const int64_t t = t0 + j, page = s_page[j];
    if (page < 0) continue;
    int64_t n0 = t + 1, first = -1;  // the next slot
    int64_t next = n0 + lane < p.T ? p.slots[n0 + lane] : -1;
    unsigned has = __ballot_sync(0xffffffffu, (uint64_t)next < slots_end);
    if (has) first = __shfl_sync(0xffffffffu, next, __ffs(has) - 1);
#pragma unroll 1
    for (n0 += 32; !has && n0 < p.T; n0 += 32 * 16) {
      unsigned found = 0;  // bit k: row n0 + 32 k + lane has a slot
#pragma unroll
      for (int k = 0; k < 16; ++k)
        found |= n0 + 32 * k + lane < p.T && (uint64_t)p.slots[n0 + 32 * k + lane] < slots_end ? 1u << k : 0u;
      const unsigned any = __reduce_or_sync(0xffffffffu, found);
      if (!any) continue;
      const int k = __ffs(any) - 1;
      has = __ballot_sync(0xffffffffu, (found >> k) & 1u);
      first = p.slots[n0 + 32 * k + __ffs(has) - 1];
    }
    const bool last = !has || first < page * p.page || first >= (page + 1) * p.page;
    if (!last) continue;
    const int n = (int)(p.H * p.TD), TD = (int)p.TD;
    for (int i = all ? tid : lane; i < n; i += all ? kWriteThreads : 32) {
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

// Tokens per thread: kWide where that still gives every SM a CTA, else 1.
constexpr int kWide = 8;

template <typename V>
void launch_write(WriteParams p, cudaStream_t s) {
  const int64_t threads = 2 * p.Hkv * (p.row_bytes / (int64_t)sizeof(V)), sms = device_sm_count();
  // as many groups as fit, but not so many that there are fewer than two CTAs per SM (3001 tokens of
  // 120 threads: one group 3.2 us, two 3.6)
  p.groups = (int)std::max<int64_t>(1, std::min<int64_t>({kMaxGroups, kWriteThreads / threads, p.T / (2 * kWide * sms)}));
  const bool wide = p.T >= kWide * sms;
  const int64_t tokens = p.groups * (wide ? kWide : 1);
  const unsigned grid = (unsigned)((p.T + tokens - 1) / tokens);
  if (wide)
    paged_write_kernel<V, kWide><<<grid, kWriteThreads, 0, s>>>(p);
  else
    paged_write_kernel<V, 1><<<grid, kWriteThreads, 0, s>>>(p);
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
