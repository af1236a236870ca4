// Routed paged decode of a batch whose requests share a prefix: one query token per request,
// the prefix's K/V read once per KV head for all requests instead of once per request.
//
// Request b attends the logical pages of the shared prefix followed by its own; head h attends
// logical page l when its routing vector router[phys, h, :r] equals q_router[b, h, :r], or l is
// page 0 and `sink`, or l is one of the last `local_blocks` pages (the rule of
// src/ultrametric/kernel_decode.py:79-89 in sparse-ai over the joined page list).  Softmax over a
// row's keys splits over any partition of them: with m = max s, l = sum exp(s - m) and
// acc = sum exp(s - m) v of each part, the parts join by weights exp(m_i - max m).  So the keys
// are cut into the prefix (rows of all requests against the same keys: one product per KV head)
// and each request's own pages, both cut further along the keys to fill the GPU, and a second
// kernel joins the parts.
//
// This file: the entry point and the general path (any head_dim up to 256, any page size,
// stride and element type; fp32 arithmetic on the CUDA cores).  A CTA takes up to kRows rows of one
// KV head and a range of 32-key tiles: K and V of a tile go to shared memory once and serve all
// its rows, as float4s: 16 products per 5 loads.  Batches that need it are small (a 32-bit cache, odd
// sizes), so it is bound by latency: the round trips to memory one after the other (page, routes, Q, K,
// V, parts), of which each has all its loads in flight.  5 requests, 12 heads of 80 fp32, 1000 + up to
// 100 tokens: 20.6 us (34.3 with loads in short loops and the join as an ordinary launch).  Large
// batches are bound by shared memory: 8 requests of 64 / 8 heads of 128 fp32 on 2000 tokens, 71 us.
#include <algorithm>
#include <string>

#include "prefix_decode.cuh"

namespace sa {
namespace {

constexpr int kPdThreads = 128;
constexpr int kRows = 16;   // rows (request, head of the group) per CTA
constexpr int kKeys = 32;   // keys per tile
constexpr int kTpr = kPdThreads / kRows;  // threads per row
constexpr int kMaxD = 256;
constexpr int kMaxSplits = 64;

struct PdSplit {
  int row_tiles, own_tiles;  // CTAs along the rows: prefix (B * G rows), own (G rows)
  int sp, so;                // splits of the prefix's and of each request's own keys
};

// Splits so that both kinds of work reach about four CTAs per SM, down to one key tile each over the
// lists' widths (the lengths are on the device): a tile takes a CTA about 5 us, all latency.
PdSplit pd_split(int64_t B, int64_t H, int64_t Hkv, int64_t page, int64_t Lp, int64_t L) {
  PdSplit s;
  const int64_t G = H / Hkv;
  s.row_tiles = (int)((B * G + kRows - 1) / kRows);
  s.own_tiles = (int)((G + kRows - 1) / kRows);
  auto splits = [](int64_t ctas, int64_t tokens) {
    const int64_t want = (4 * device_sm_count() + ctas - 1) / std::max<int64_t>(ctas, 1);
    const int64_t cap = (tokens + kKeys - 1) / kKeys;
    return (int)std::max<int64_t>(1, std::min<int64_t>({want, cap, kMaxSplits}));
  };
  s.sp = Lp > 0 ? splits(Hkv * s.row_tiles, Lp * page) : 0;
  s.so = L > 0 ? splits(B * Hkv * s.own_tiles, L * page) : 0;
  return s;
}

// Partials of row (b, h): [sp + so][D + 2] floats: m (log2 units), l, acc[D].
int64_t pd_bytes(int64_t B, int64_t H, int64_t D, const PdSplit& s) {
  return B * H * (int64_t)(s.sp + s.so) * (D + 2) * 4;
}

// NI: float4 output columns per thread, D <= 32 NI.  Registers are held to what five CTAs per SM leave (three
// above 128 columns, whose K and V take the shared memory): all of a small batch's CTAs run at once.
template <typename T, int NI>
__global__ void __launch_bounds__(kPdThreads, NI <= 4 ? 5 : 3) prefix_split_kernel(const PrefixParams p, const PdSplit s, float* part) {
  extern __shared__ float sm[];
  // rows of D floats, padded with zeros to whole float4s and by one more, so that the eight keys that
  // a row's threads read at a time lie in different banks
  const int D = (int)p.D, D4 = (D + 3) / 4, DP = 4 * D4 + 4;
  float* s_q = sm;                    // [kRows][DP]
  float* s_k = s_q + kRows * DP;      // [kKeys][DP]
  float* s_v = s_k + kKeys * DP;      // [kKeys][DP]
  float* s_p = s_v + kKeys * DP;      // [kRows][kKeys + 1]
  // page of each key of the tile (-1: none), its logical index, and the key's K and V rows
  __shared__ int s_phys[kKeys], s_lp[kKeys];
  __shared__ const T *s_krow[kKeys], *s_vrow[kKeys];
  const int tid = threadIdx.x;
  pdl_trigger();  // the join waits for the whole grid

  // ---- which rows and which keys
  const int64_t prefix_ctas = p.Hkv * s.row_tiles * s.sp;
  int64_t x = blockIdx.x;
  const bool own = x >= prefix_ctas;
  int64_t g, row0, nrows, b_own = 0, tokens, split, splits;
  const int64_t plen = prefix_tokens(p);
  const int64_t pre_pages = (plen + p.page - 1) / p.page;
  if (!own) {
    split = x % s.sp;
    x /= s.sp;
    row0 = (x % s.row_tiles) * kRows;
    g = x / s.row_tiles;
    nrows = min((int64_t)kRows, p.B * p.G - row0);
    tokens = plen;
    splits = s.sp;
  } else {
    x -= prefix_ctas;
    split = x % s.so;
    x /= s.so;
    const int64_t rt = x % s.own_tiles;
    x /= s.own_tiles;
    g = x % p.Hkv;
    b_own = x / p.Hkv;
    row0 = b_own * p.G + rt * kRows;
    nrows = min((int64_t)kRows, p.G - rt * kRows);
    tokens = own_tokens(p, b_own);
    splits = s.so;
  }
  const int64_t ntiles = (tokens + kKeys - 1) / kKeys, per = (ntiles + splits - 1) / splits;
  const int64_t t_lo = min(ntiles, split * per), t_hi = min(ntiles, t_lo + per);

  // ---- this thread's row
  const int row = tid / kTpr, li = tid % kTpr;
  const bool live = row < nrows;
  const int64_t b = live ? (row0 + row) / p.G : 0, h = live ? g * p.G + (row0 + row) % p.G : 0;
  const int64_t n_pages = pre_pages + (live ? (own_tokens(p, b) + p.page - 1) / p.page : 0);
  const float scale2 = rsqrtf((float)D) * kLog2e;
  {
    const int warp = tid >> 5, lane = tid & 31;
    constexpr int kPer = kRows / (kPdThreads / 32);
    const T* q[kPer];
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const int rg = (int)min(row0 + warp + u * (kPdThreads / 32), p.B * p.G - 1), bb = rg / (int)p.G;
      q[u] = static_cast<const T*>(p.q) + bb * p.qs[0] + (g * p.G + rg - bb * p.G) * p.qs[1];
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int d = lane + 32 * i;
      float x[kPer];
#pragma unroll
      for (int u = 0; u < kPer; ++u) x[u] = d < D ? to_f32<T>(q[u][d]) * scale2 : 0.f;
#pragma unroll
      for (int u = 0; u < kPer; ++u)
        if (d < 4 * D4) s_q[(warp + u * (kPdThreads / 32)) * DP + d] = x[u];
    }
  }
  float m = -INFINITY, l = 0.f;
  float4 acc[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);

  for (int64_t t = t_lo; t < t_hi; ++t) {
    __syncthreads();  // the last tile's shared arrays are read
    if (tid < kKeys) {
      const int tok = (int)(t * kKeys) + tid;
      int phys = -1, lp = 0;
      if (tok < tokens) {
        lp = tok / (int)p.page;
        phys = own ? p.bt[b_own * p.bts[0] + lp * p.bts[1]] : p.ppages[lp];
        if (phys < 0 || phys >= p.num_pages) {
          raise_status(p.status, kStatusBadIndex);
          phys = -1;
        }
        const int off = tok - lp * (int)p.page;
        s_krow[tid] = static_cast<const T*>(p.kc) + (int64_t)phys * p.ks[0] + g * p.ks[1] + off * p.ks[2];
        s_vrow[tid] = static_cast<const T*>(p.vc) + (int64_t)phys * p.vs[0] + g * p.vs[1] + off * p.vs[2];
      }
      s_phys[tid] = phys;
      s_lp[tid] = lp;
    }
    __syncthreads();
    // keys of this row in the tile: li, li + kTpr, ...
    bool see[kKeys / kTpr], any = false;
    int last_lp = -1;
    bool last_on = false;
#pragma unroll
    for (int u = 0; u < kKeys / kTpr; ++u) {
      const int phys = s_phys[li + u * kTpr], lp = s_lp[li + u * kTpr];
      see[u] = live && phys >= 0;
      if (see[u] && p.r > 0) {
        if (lp != last_lp) {
          last_lp = lp;
          last_on = page_attended<4>(p, b, h, (own ? pre_pages : 0) + lp, n_pages, phys);
        }
        see[u] = last_on;
      }
      any |= see[u];
    }
    if (!__syncthreads_or(any)) continue;
    // one warp per key, lanes along the row; all of a warp's loads in flight
    const int warp = tid >> 5, lane = tid & 31;
    constexpr int kPer = kKeys / (kPdThreads / 32), kRound = NI < 4 ? NI : 4;
#pragma unroll
    for (int i0 = 0; i0 < NI; i0 += kRound) {
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        float x[kRound][kPer];
#pragma unroll
        for (int u = 0; u < kPer; ++u) {
          const int kk = warp + u * (kPdThreads / 32);
          const bool have = s_phys[kk] >= 0;
          const T* src = kv ? s_vrow[kk] : s_krow[kk];
#pragma unroll
          for (int i = 0; i < kRound; ++i) {
            const int d = lane + 32 * (i0 + i);
            x[i][u] = have && d < D ? to_f32<T>(src[d]) : 0.f;
          }
        }
#pragma unroll
        for (int u = 0; u < kPer; ++u)
#pragma unroll
          for (int i = 0; i < kRound; ++i) {
            const int d = lane + 32 * (i0 + i);
            if (d < 4 * D4) (kv ? s_v : s_k)[(warp + u * (kPdThreads / 32)) * DP + d] = x[i][u];
          }
      }
    }
    __syncthreads();
    float sc[kKeys / kTpr];
#pragma unroll
    for (int u = 0; u < kKeys / kTpr; ++u) sc[u] = 0.f;
#pragma unroll 4
    for (int d = 0; d < D4; ++d) {
      const float4 q = *reinterpret_cast<const float4*>(s_q + row * DP + 4 * d);
#pragma unroll
      for (int u = 0; u < kKeys / kTpr; ++u) {
        const float4 k = *reinterpret_cast<const float4*>(s_k + (li + u * kTpr) * DP + 4 * d);
        sc[u] = fmaf(q.x, k.x, fmaf(q.y, k.y, fmaf(q.z, k.z, fmaf(q.w, k.w, sc[u]))));
      }
    }
    float mt = -INFINITY;
#pragma unroll
    for (int u = 0; u < kKeys / kTpr; ++u) {
      sc[u] = see[u] ? sc[u] : -INFINITY;  // by selection: a masked key's NaN does not spread
      mt = fmaxf(mt, sc[u]);
    }
#pragma unroll
    for (int o = kTpr / 2; o; o >>= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, o));
    const float m_new = fmaxf(m, mt), ref = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = exp2f(m - ref);
    float ps = 0.f;
#pragma unroll
    for (int u = 0; u < kKeys / kTpr; ++u) {
      const float e = see[u] ? exp2f(sc[u] - ref) : 0.f;
      ps += e;
      s_p[row * (kKeys + 1) + li + u * kTpr] = see[u] ? e : -1.f;  // -1: masked
    }
#pragma unroll
    for (int o = kTpr / 2; o; o >>= 1) ps += __shfl_xor_sync(0xffffffffu, ps, o);
    l = l * alpha + ps;
    m = m_new;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      acc[i].x *= alpha;
      acc[i].y *= alpha;
      acc[i].z *= alpha;
      acc[i].w *= alpha;
    }
    __syncwarp();  // a row's threads are one warp's
#pragma unroll 4
    for (int kk = 0; kk < kKeys; ++kk) {
      const float e = s_p[row * (kKeys + 1) + kk];
      const bool on = !(e < 0.f);  // masked: whatever V holds there does not count
#pragma unroll
      for (int i = 0; i < NI; ++i)
        if (li + i * kTpr < D4) {
          const float4 v = *reinterpret_cast<const float4*>(s_v + kk * DP + 4 * (li + i * kTpr));
          acc[i].x = on ? fmaf(e, v.x, acc[i].x) : acc[i].x;
          acc[i].y = on ? fmaf(e, v.y, acc[i].y) : acc[i].y;
          acc[i].z = on ? fmaf(e, v.z, acc[i].z) : acc[i].z;
          acc[i].w = on ? fmaf(e, v.w, acc[i].w) : acc[i].w;
        }
    }
  }
  if (!live) return;
  float* o = part + ((b * p.H + h) * (s.sp + s.so) + (own ? s.sp : 0) + split) * (D + 2);
  if (li == 0) {
    o[0] = m;
    o[1] = l;
  }
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int c = 4 * (li + i * kTpr);
    if (c < D) o[2 + c] = acc[i].x;
    if (c + 1 < D) o[3 + c] = acc[i].y;
    if (c + 2 < D) o[4 + c] = acc[i].z;
    if (c + 3 < D) o[5 + c] = acc[i].w;
  }
}

// Joins the parts of (b, h) = blockIdx.x.  Two dependent rounds of loads (the parts' m and l, then their
// accumulators): warps share the parts, lanes the columns, 16 loads in flight each.
constexpr int kJoinThreads = 256, kJoinWarps = kJoinThreads / 32;

template <typename T>
__global__ void __launch_bounds__(kJoinThreads) prefix_join_kernel(const PrefixParams p, const PdSplit s,
                                                                   const float* part) {
  const int64_t b = blockIdx.x / p.H, h = blockIdx.x % p.H;
  const int n = s.sp + s.so, D = (int)p.D, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const float* base = part + (int64_t)blockIdx.x * n * (D + 2);
  __shared__ float s_m[2 * kMaxSplits], s_l[2 * kMaxSplits], s_w[2 * kMaxSplits];
  __shared__ float s_a[kJoinWarps][128];
  pdl_wait();
  if (tid < 2 * kMaxSplits) {
    s_m[tid] = tid < n ? base[(int64_t)tid * (D + 2)] : -INFINITY;
    s_l[tid] = tid < n ? base[(int64_t)tid * (D + 2) + 1] : 0.f;
  }
  __syncthreads();
  float M = -INFINITY;
#pragma unroll
  for (int k = 0; k < 2 * kMaxSplits; k += 32) M = fmaxf(M, s_m[k + lane]);
#pragma unroll
  for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  const float ref = M == -INFINITY ? 0.f : M;
  float L = 0.f;
#pragma unroll
  for (int k = 0; k < 2 * kMaxSplits; k += 32) {
    const float w = exp2f(s_m[k + lane] - ref);
    if (warp == 0) s_w[k + lane] = w;
    L += s_l[k + lane] * w;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
  __syncthreads();
  const float inv = L == 0.f ? 0.f : 1.f / L;  // NaN stays NaN
  T* o = static_cast<T*>(p.out) + b * p.os[0] + h * p.os[1];
  for (int d0 = 0; d0 < D; d0 += 128) {
    float a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int i0 = warp; i0 < n; i0 += 4 * kJoinWarps) {
      float x[4][4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int i = i0 + u * kJoinWarps, d = d0 + 32 * k + lane;
          x[u][k] = i < n && d < D ? base[(int64_t)i * (D + 2) + 2 + d] : 0.f;
        }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + u * kJoinWarps;
        if (i < n && s_m[i] != -INFINITY)
#pragma unroll
          for (int k = 0; k < 4; ++k) a[k] = fmaf(x[u][k], s_w[i], a[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) s_a[warp][32 * k + lane] = a[k];
    __syncthreads();
    if (tid < 128 && d0 + tid < D) {
      float y = 0.f;
#pragma unroll
      for (int w = 0; w < kJoinWarps; ++w) y += s_a[w][tid];
      o[d0 + tid] = from_f32<T>(L == 0.f ? 0.f : y * inv);
    }
    __syncthreads();
  }
  if (p.lse && tid == 0) p.lse[blockIdx.x] = L == 0.f ? -INFINITY : M * kLn2 + logf(L);
}

static_assert(2 * kMaxSplits == 128, "whole warps of parts in the join");

template <typename T>
int launch_general(const PrefixParams& p, float* part, cudaStream_t stream) {
  const PdSplit s = pd_split(p.B, p.H, p.Hkv, p.page, p.Lp, p.L);
  const int64_t ctas = p.Hkv * s.row_tiles * s.sp + p.B * p.Hkv * s.own_tiles * s.so;
  if (ctas > INT32_MAX) return fail(SA_EUNSUPPORTED, "prefix decode: too many requests");
  if (ctas > 0) {
    const size_t smem = ((size_t)(kRows + 2 * kKeys) * ((p.D + 3) / 4 * 4 + 4) + kRows * (kKeys + 1)) * 4;
    auto kern = p.D <= 64    ? prefix_split_kernel<T, 2>
                : p.D <= 128 ? prefix_split_kernel<T, 4>
                             : prefix_split_kernel<T, 8>;
    if (smem > 48 * 1024) cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    kern<<<(unsigned)ctas, kPdThreads, smem, stream>>>(p, s, part);
    if (int rc = check_launch("prefix_split_kernel")) return rc;
  }
  return launch_dependent(prefix_join_kernel<T>, dim3((unsigned)(p.B * p.H)), dim3(kJoinThreads), 0, stream,
                          "prefix_join_kernel", p, s, (const float*)part);
}

}  // namespace
}  // namespace sa

extern "C" {

int64_t sa_ultrametric_prefix_decode_workspace_bytes(int dtype, int64_t B, int64_t H, int64_t Hkv, int64_t D,
                                                     int64_t page_size, int64_t max_prefix_pages,
                                                     int64_t max_logical_pages) {
  if (B <= 0 || H <= 0 || Hkv <= 0 || D <= 0 || page_size <= 0 || max_prefix_pages < 0 || max_logical_pages < 0 ||
      H % Hkv)
    return 0;
  // alignment decides the path at the call: the larger of the two serves either
  const int64_t general = sa::pd_bytes(B, H, D, sa::pd_split(B, H, Hkv, page_size, max_prefix_pages, max_logical_pages));
  if (!sa::prefix_fast_shape(dtype, B, H, Hkv, D, page_size)) return general;
  return std::max(general, sa::prefix_fast_workspace_bytes(B, H, Hkv, D, page_size, max_prefix_pages, max_logical_pages));
}

int sa_ultrametric_prefix_decode(int dtype, int64_t B, int64_t H, int64_t Hkv, int64_t D, int64_t page_size,
                                 int64_t num_pages, const void* q, const int64_t* q_strides, const void* k_cache,
                                 const int64_t* k_strides, const void* v_cache, const int64_t* v_strides,
                                 const int32_t* prefix_pages, int64_t max_prefix_pages, int64_t prefix_len,
                                 const int32_t* prefix_len_dev, const int32_t* block_tables,
                                 const int64_t* bt_strides, int64_t max_logical_pages, const int32_t* context_lens,
                                 const void* router, int router_dtype, const int64_t* router_strides,
                                 const void* q_router, int q_router_dtype, const int64_t* q_router_strides,
                                 int64_t TD, int64_t req_depth, int64_t local_blocks, int sink_block, void* out,
                                 const int64_t* out_strides, float* lse, void* workspace, int64_t workspace_bytes,
                                 void* stream) {
  using namespace sa;
  if (B < 0 || H <= 0 || Hkv <= 0 || D <= 0 || page_size <= 0 || num_pages < 0 || max_prefix_pages < 0 ||
      max_logical_pages < 0 || TD < 1)
    return fail(SA_EINVAL, "prefix decode: bad sizes");
  if (H % Hkv) return fail(SA_EINVAL, "prefix decode: num_heads must be a multiple of the cache heads");
  if (prefix_len < 0 || (!prefix_len_dev && prefix_len > max_prefix_pages * page_size))
    return fail(SA_EINVAL, "prefix decode: prefix_len does not fit the prefix pages");
  if (req_depth < 0 || req_depth > TD) return fail(SA_EINVAL, "prefix decode: req_depth must be in [0, TD]");
  if (local_blocks < 0) return fail(SA_EINVAL, "prefix decode: local_blocks must be >= 0");
  if (dtype != SA_F32 && dtype != SA_F16 && dtype != SA_BF16)
    return fail(SA_EUNSUPPORTED, "prefix decode: dtype must be fp32, fp16 or bf16");
  if (D > kMaxD) return fail(SA_EUNSUPPORTED, "prefix decode: head_dim above 256");
  if ((router_dtype != SA_I32 && router_dtype != SA_I64) || (q_router_dtype != SA_I32 && q_router_dtype != SA_I64))
    return fail(SA_EUNSUPPORTED, "prefix decode: routing vectors must be int32 or int64");
  if (B == 0) return SA_OK;
  if (!q || !q_strides || !k_strides || !v_strides || (num_pages && (!k_cache || !v_cache)) ||
      (max_prefix_pages && !prefix_pages) || (max_logical_pages && !block_tables) || !bt_strides || !context_lens ||
      !router_strides || !q_router_strides || (req_depth && ((num_pages && !router) || !q_router)) || !out || !out_strides)
    return fail(SA_EINVAL, "prefix decode: null pointer argument");
  if (q_strides[2] != 1 || k_strides[3] != 1 || v_strides[3] != 1 || out_strides[2] != 1)
    return fail(SA_EUNSUPPORTED, "prefix decode: head_dim must be the contiguous dimension");
  if (B * H > INT32_MAX || max_prefix_pages * page_size > INT32_MAX || max_logical_pages * page_size > INT32_MAX)
    return fail(SA_EUNSUPPORTED, "prefix decode: sizes too large");
  const int64_t need = sa_ultrametric_prefix_decode_workspace_bytes(dtype, B, H, Hkv, D, page_size, max_prefix_pages,
                                                                    max_logical_pages);
  if (workspace_bytes < need || (need && !workspace))
    return fail(SA_EWORKSPACE, "prefix decode: workspace too small (" + std::to_string(workspace_bytes) + " < " +
                                   std::to_string(need) + ")");
  if (reinterpret_cast<uintptr_t>(workspace) % 256)
    return fail(SA_EINVAL, "prefix decode: workspace must be 256-byte aligned");
  if (int rc = check_stream_device(stream, "prefix decode")) return rc;
  PrefixParams p{};
  p.B = B;
  p.H = H;
  p.Hkv = Hkv;
  p.G = H / Hkv;
  p.D = D;
  p.page = page_size;
  p.num_pages = num_pages;
  p.Lp = max_prefix_pages;
  p.L = max_logical_pages;
  p.plen = prefix_len;
  p.plen_dev = prefix_len_dev;
  p.TD = TD;
  p.r = req_depth;
  p.local_blocks = local_blocks;
  p.sink = sink_block;
  p.q = q;
  p.kc = k_cache;
  p.vc = v_cache;
  p.ppages = prefix_pages;
  p.bt = block_tables;
  p.ctx = context_lens;
  p.router = router;
  p.router_dtype = router_dtype;
  p.qrouter = q_router;
  p.qrouter_dtype = q_router_dtype;
  for (int i = 0; i < 4; ++i) {
    p.ks[i] = k_strides[i];
    p.vs[i] = v_strides[i];
  }
  for (int i = 0; i < 3; ++i) {
    p.qs[i] = q_strides[i];
    p.rs[i] = router_strides[i];
    p.qrs[i] = q_router_strides[i];
    p.os[i] = out_strides[i];
  }
  p.bts[0] = bt_strides[0];
  p.bts[1] = bt_strides[1];
  p.out = out;
  p.lse = lse;
  p.status = device_status_ptr();
  if (!p.status) return fail(SA_ELAUNCH, std::string("prefix decode: ") + sa_last_error());
  float* part = static_cast<float*>(workspace);
  cudaStream_t s = (cudaStream_t)stream;
  if (prefix_fast_eligible(p, dtype)) return launch_prefix_fast(p, dtype, workspace, s);
  switch (dtype) {
    case SA_F32: return launch_general<float>(p, part, s);
    case SA_F16: return launch_general<__half>(p, part, s);
    default: return launch_general<__nv_bfloat16>(p, part, s);
  }
}

}  // extern "C"
