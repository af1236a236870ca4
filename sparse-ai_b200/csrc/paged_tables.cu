// Block tables and slot map of a ragged step, built on the device from request lengths, and the
// return of finished requests' pages.
//
// Request b holds ctx_b tokens in ceil(ctx_b / page) pages and gets new_b more.  With
// need_b = ceil((ctx_b + new_b) / page) - ceil(ctx_b / page) pages to add and `incl` the inclusive
// sum of need over the requests in order, request b is admitted while incl_b <= num_free; its
// j-th new page is entry num_free - 1 - (incl_b - need_b + j) of the stack of free pages.  New
// token i of the request sits at position ctx_b + i, in row position % page of its page.
//
// Integer work on a few KB per request and 16 bytes per token: what it costs is the launch, the
// two dependent sums over the requests and one page lookup per token.  So there is one launch:
// every CTA repeats the sums over all requests in its own shared memory (B / 256 rounds of two
// block scans) instead of waiting for a first kernel's, and then fills its share of the token rows.
// 64 requests with a token each: 5.9 us; 256 requests with 120001 tokens (2.0 MB written): 5.8 us, all of
// it latency (launch, lengths, sums, search, page, store).
#include <algorithm>
#include <string>

#include "common.cuh"

namespace sa {
namespace {

constexpr int kTabThreads = 256;
constexpr int kTabWarps = kTabThreads / 32;
constexpr int kTabRows = 4;            // token rows per thread and step (16-byte stores)
constexpr int64_t kMaxRequests = 16384;  // 8 bytes of shared memory each

// Inclusive sum of v over the CTA's threads; *total gets the sum over all of them.
__device__ __forceinline__ int64_t cta_incl_sum(int64_t v, int64_t* s_warp, int64_t* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  if (lane == 31) s_warp[warp] = v;
  __syncthreads();
  int64_t base = 0, tot = 0;
#pragma unroll
  for (int w = 0; w < kTabWarps; ++w) {
    const int64_t t = s_warp[w];
    base += w < warp ? t : 0;
    tot += t;
  }
  __syncthreads();  // s_warp may be rewritten by the next call
  *total = tot;
  return base + v;
}

struct TablesParams {
  int64_t B, L, page, rows, free_cap, pos_base;
  const int32_t* ctx;
  const int32_t* nlen;
  int32_t* bt;
  int64_t bts[2];
  const int32_t* free_pages;
  const int32_t* num_free;
  int64_t* slots;
  int32_t* rid;
  int32_t* pos;
  int32_t* cu;
  int32_t* ctx_out;
  int32_t* num_free_out;
  unsigned* status;
};

__global__ void __launch_bounds__(kTabThreads) build_tables_kernel(const TablesParams p) {
  extern __shared__ int32_t s_tab[];
  int32_t* s_cu = s_tab;                // [B + 1] first row of each request
  int32_t* s_first = s_tab + p.B + 1;   // [B] its first page in the order of taking, -1: refused
  __shared__ int64_t s_warp[kTabWarps];
  const int tid = threadIdx.x;
  int64_t nf = p.num_free[0];
  bool bad = nf < 0 || nf > p.free_cap;
  nf = max((int64_t)0, min(nf, p.free_cap));
  int64_t run_rows = 0, run_need = 0, used = 0;
  for (int64_t b0 = 0; b0 < p.B; b0 += kTabThreads) {
    const int64_t b = b0 + tid;
    const bool in = b < p.B;
    const int64_t c = in ? p.ctx[b] : 0, n = in ? p.nlen[b] : 0;
    int64_t tot;
    const int64_t end = run_rows + cta_incl_sum(max(n, (int64_t)0), s_warp, &tot);
    run_rows += tot;
    const int64_t old_pages = (max(c, (int64_t)0) + p.page - 1) / p.page;
    const int64_t all_pages = (max(c, (int64_t)0) + max(n, (int64_t)0) + p.page - 1) / p.page;
    // lengths and positions are 32-bit numbers
    const bool ok = in && c >= 0 && n >= 0 && all_pages <= p.L && end <= p.rows && c + n <= INT32_MAX &&
                    (n == 0 || p.pos_base + c + n - 1 <= INT32_MAX);
    const int64_t need = ok ? all_pages - old_pages : 0;
    const int64_t incl = run_need + cta_incl_sum(need, s_warp, &tot);
    run_need += tot;
    const bool fits = ok && (need == 0 || incl <= nf);
    if (in) {
      s_cu[b] = (int32_t)min(end - max(n, (int64_t)0), (int64_t)INT32_MAX);
      s_first[b] = fits ? (int32_t)(incl - need) : -1;
      if (blockIdx.x == 0) {
        p.cu[b] = s_cu[b];
        p.ctx_out[b] = (int32_t)(fits ? c + n : c);
      }
    }
    if (fits && need > 0) used = max(used, incl);
    bad |= in && !fits;
  }
  if (tid == 0) s_cu[p.B] = (int32_t)min(run_rows, (int64_t)INT32_MAX);
  if (blockIdx.x == 0) {
#pragma unroll
    for (int o = 16; o; o >>= 1) used = max(used, (int64_t)__shfl_xor_sync(0xffffffffu, used, o));
    if ((tid & 31) == 0) s_warp[tid >> 5] = used;
    if (bad) raise_status(p.status, kStatusBadIndex);
  }
  __syncthreads();
  if (blockIdx.x == 0 && tid == 0) {
    for (int w = 0; w < kTabWarps; ++w) used = max(used, s_warp[w]);
    p.cu[p.B] = s_cu[p.B];
    p.num_free_out[0] = (int32_t)(nf - used);
  }

  // token rows, kTabRows consecutive ones per thread
  const int64_t live = min((int64_t)s_cu[p.B], p.rows);
  for (int64_t t0 = ((int64_t)blockIdx.x * kTabThreads + tid) * kTabRows; t0 < p.rows;
       t0 += (int64_t)gridDim.x * kTabThreads * kTabRows) {
    int lo = 0;
    if (t0 < live) {  // last request whose first row is <= t0 (those after it with none are skipped)
      int hi = (int)p.B - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (s_cu[mid] <= t0) lo = mid;
        else hi = mid - 1;
      }
    }
    int64_t slot[kTabRows];
    int32_t rid[kTabRows], pos[kTabRows];
#pragma unroll
    for (int i = 0; i < kTabRows; ++i) {
      const int64_t t = t0 + i;
      slot[i] = -1;
      rid[i] = -1;
      pos[i] = 0;
      if (t >= live) continue;
      while (s_cu[lo + 1] <= t) ++lo;
      const int64_t c = p.ctx[lo], ps = max(c, (int64_t)0) + (t - s_cu[lo]);
      rid[i] = lo;
      pos[i] = (int32_t)min(p.pos_base + ps, (int64_t)INT32_MAX);  // past it: a refused request's rows
      const int first = s_first[lo];
      if (first < 0) continue;
      const int64_t lp = ps / p.page, off = ps - lp * p.page, old_pages = (c + p.page - 1) / p.page;
      int32_t* entry = p.bt + lo * p.bts[0] + lp * p.bts[1];
      int32_t phys;
      if (lp >= old_pages) {
        phys = p.free_pages[nf - 1 - (first + (lp - old_pages))];
        if (off == 0) *entry = phys;  // a new page always receives its first row in this step
      } else {
        phys = *entry;
      }
      if (phys >= 0)
        slot[i] = phys * p.page + off;
      else
        raise_status(p.status, kStatusBadIndex);
    }
    if (t0 + kTabRows <= p.rows) {
      *reinterpret_cast<longlong2*>(p.slots + t0) = make_longlong2(slot[0], slot[1]);
      *reinterpret_cast<longlong2*>(p.slots + t0 + 2) = make_longlong2(slot[2], slot[3]);
      *reinterpret_cast<int4*>(p.rid + t0) = make_int4(rid[0], rid[1], rid[2], rid[3]);
      *reinterpret_cast<int4*>(p.pos + t0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
    } else {
#pragma unroll
      for (int i = 0; i < kTabRows; ++i)
        if (t0 + i < p.rows) {
          p.slots[t0 + i] = slot[i];
          p.rid[t0 + i] = rid[i];
          p.pos[t0 + i] = pos[i];
        }
    }
  }
}

struct ReleaseParams {
  int64_t B, L, page, free_cap;
  const uint8_t* finished;
  const int32_t* ctx;
  const int32_t* bt;
  int64_t bts[2];
  int32_t* free_pages;
  const int32_t* num_free;
  int32_t* ctx_out;
  int32_t* num_free_out;
  unsigned* status;
};

// Finished request b pushes table[b][0 .. ceil(ctx_b / page)) on the stack, requests in order.
// Every CTA repeats the sum over the requests; requests go round the CTAs.
__global__ void __launch_bounds__(kTabThreads) release_kernel(const ReleaseParams p) {
  extern __shared__ int32_t s_tab[];
  int32_t* s_off = s_tab;  // [B] first stack entry of each request's pages, -1: nothing to push
  __shared__ int64_t s_warp[kTabWarps];
  const int tid = threadIdx.x;
  int64_t nf = p.num_free[0];
  bool bad = nf < 0 || nf > p.free_cap;
  nf = max((int64_t)0, min(nf, p.free_cap));
  int64_t run = 0, top = 0;
  for (int64_t b0 = 0; b0 < p.B; b0 += kTabThreads) {
    const int64_t b = b0 + tid;
    const bool in = b < p.B;
    const bool done = in && p.finished[b] != 0;
    const int64_t c = in ? p.ctx[b] : 0;
    const int64_t pages = (max(c, (int64_t)0) + p.page - 1) / p.page;
    const bool ok = done && c >= 0 && pages <= p.L;
    int64_t tot;
    const int64_t incl = run + cta_incl_sum(ok ? pages : 0, s_warp, &tot);
    run += tot;
    const bool fits = ok && (pages == 0 || nf + incl <= p.free_cap);
    if (in) {
      s_off[b] = fits && pages > 0 ? (int32_t)(nf + incl - pages) : -1;
      if (blockIdx.x == 0) p.ctx_out[b] = fits ? 0 : p.ctx[b];
    }
    if (fits && pages > 0) top = max(top, incl);
    bad |= done && !fits;
  }
  if (blockIdx.x == 0) {
#pragma unroll
    for (int o = 16; o; o >>= 1) top = max(top, (int64_t)__shfl_xor_sync(0xffffffffu, top, o));
    if ((tid & 31) == 0) s_warp[tid >> 5] = top;
    if (bad) raise_status(p.status, kStatusBadIndex);
  }
  __syncthreads();
  if (blockIdx.x == 0 && tid == 0) {
    for (int w = 0; w < kTabWarps; ++w) top = max(top, s_warp[w]);
    p.num_free_out[0] = (int32_t)(nf + top);
  }
  for (int64_t b = blockIdx.x; b < p.B; b += gridDim.x) {
    if (s_off[b] < 0) continue;
    const int64_t pages = (p.ctx[b] + p.page - 1) / p.page;
    for (int64_t j = tid; j < pages; j += kTabThreads) p.free_pages[s_off[b] + j] = p.bt[b * p.bts[0] + j * p.bts[1]];
  }
}

int check_sizes(int64_t B, int64_t L, int64_t page, int64_t cap, const char* what) {
  if (B < 0 || L < 0 || page <= 0 || cap < 0) return fail(SA_EINVAL, std::string(what) + ": bad sizes");
  if (B > kMaxRequests)
    return fail(SA_EUNSUPPORTED, std::string(what) + ": more than " + std::to_string(kMaxRequests) + " requests");
  if (cap > INT32_MAX || L > INT32_MAX) return fail(SA_EUNSUPPORTED, std::string(what) + ": more than 2^31 pages");
  return SA_OK;
}

}  // namespace
}  // namespace sa

extern "C" {

int sa_paged_build_tables(int64_t B, int64_t max_logical_pages, int64_t page_size, int64_t num_tokens,
                          const int32_t* context_lens, const int32_t* new_lens, int32_t* block_tables,
                          const int64_t* bt_strides, const int32_t* free_pages, int64_t free_capacity,
                          const int32_t* num_free, int64_t position_base, int64_t* slot_mapping,
                          int32_t* request_ids, int32_t* positions, int32_t* cu_new_lens,
                          int32_t* context_lens_out, int32_t* num_free_out, void* stream) {
  using namespace sa;
  const char* what = "paged tables";
  if (int rc = check_sizes(B, max_logical_pages, page_size, free_capacity, what)) return rc;
  if (num_tokens < 0 || position_base < 0 || position_base > INT32_MAX)
    return fail(SA_EINVAL, "paged tables: bad num_tokens or position_base");
  if (num_tokens > INT32_MAX) return fail(SA_EUNSUPPORTED, "paged tables: more than 2^31 tokens");
  if ((B && (!context_lens || !new_lens || !context_lens_out)) || (B && max_logical_pages && !block_tables) ||
      !bt_strides || (free_capacity && !free_pages) || !num_free || !cu_new_lens || !num_free_out ||
      (num_tokens && (!slot_mapping || !request_ids || !positions)))
    return fail(SA_EINVAL, "paged tables: null pointer argument");
  if ((B && context_lens_out == context_lens) || num_free_out == num_free)
    return fail(SA_EINVAL, "paged tables: the outputs may not alias the inputs");
  if (reinterpret_cast<uintptr_t>(slot_mapping) % 16 || reinterpret_cast<uintptr_t>(request_ids) % 16 ||
      reinterpret_cast<uintptr_t>(positions) % 16)
    return fail(SA_EUNSUPPORTED, "paged tables: the row outputs must be 16-byte aligned");
  if (int rc = check_stream_device(stream, what)) return rc;
  TablesParams p{};
  p.B = B;
  p.L = max_logical_pages;
  p.page = page_size;
  p.rows = num_tokens;
  p.free_cap = free_capacity;
  p.pos_base = position_base;
  p.ctx = context_lens;
  p.nlen = new_lens;
  p.bt = block_tables;
  p.bts[0] = bt_strides[0];
  p.bts[1] = bt_strides[1];
  p.free_pages = free_pages;
  p.num_free = num_free;
  p.slots = slot_mapping;
  p.rid = request_ids;
  p.pos = positions;
  p.cu = cu_new_lens;
  p.ctx_out = context_lens_out;
  p.num_free_out = num_free_out;
  p.status = device_status_ptr();
  if (!p.status) return fail(SA_ELAUNCH, std::string("paged tables: ") + sa_last_error());
  const size_t smem = (size_t)(2 * B + 1) * 4;
  if (smem > 48 * 1024)
    cudaFuncSetAttribute(build_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  const int64_t per = kTabThreads * kTabRows, want = (num_tokens + per - 1) / per;
  const int grid = (int)std::max<int64_t>(1, std::min<int64_t>(want, device_sm_count()));
  build_tables_kernel<<<grid, kTabThreads, smem, (cudaStream_t)stream>>>(p);
  return check_launch("build_tables_kernel");
}

int sa_paged_release(int64_t B, int64_t max_logical_pages, int64_t page_size, const uint8_t* finished,
                     const int32_t* context_lens, const int32_t* block_tables, const int64_t* bt_strides,
                     int32_t* free_pages, int64_t free_capacity, const int32_t* num_free,
                     int32_t* context_lens_out, int32_t* num_free_out, void* stream) {
  using namespace sa;
  const char* what = "paged release";
  if (int rc = check_sizes(B, max_logical_pages, page_size, free_capacity, what)) return rc;
  if ((B && (!finished || !context_lens || !context_lens_out)) || (B && max_logical_pages && !block_tables) ||
      !bt_strides || (free_capacity && !free_pages) || !num_free || !num_free_out)
    return fail(SA_EINVAL, "paged release: null pointer argument");
  if ((B && context_lens_out == context_lens) || num_free_out == num_free)
    return fail(SA_EINVAL, "paged release: the outputs may not alias the inputs");
  if (int rc = check_stream_device(stream, what)) return rc;
  ReleaseParams p{};
  p.B = B;
  p.L = max_logical_pages;
  p.page = page_size;
  p.free_cap = free_capacity;
  p.finished = finished;
  p.ctx = context_lens;
  p.bt = block_tables;
  p.bts[0] = bt_strides[0];
  p.bts[1] = bt_strides[1];
  p.free_pages = free_pages;
  p.num_free = num_free;
  p.ctx_out = context_lens_out;
  p.num_free_out = num_free_out;
  p.status = device_status_ptr();
  if (!p.status) return fail(SA_ELAUNCH, std::string("paged release: ") + sa_last_error());
  const size_t smem = (size_t)std::max<int64_t>(B, 1) * 4;
  if (smem > 48 * 1024)
    cudaFuncSetAttribute(release_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  const int grid = (int)std::max<int64_t>(1, std::min<int64_t>(B, device_sm_count()));
  release_kernel<<<grid, kTabThreads, smem, (cudaStream_t)stream>>>(p);
  return check_launch("release_kernel");
}

}  // extern "C"
