// Shared-prefix decode on sm_100a: TMA page loads, tcgen05 products with TMEM accumulators.
// Semantics in prefix_decode.cu.
//
// Per KV head the query rows (request b, head g of the group) of `nb` = 128 / G requests fill one
// 128-row MMA tile.  Work is cut into key tiles of up to 128 keys (up to kMaxPpt pages), in
// three segments laid end to end:
//   pair    prefix tiles against two row tiles at once (2 nb requests): each K/V tile that is
//           loaded serves 256 rows;
//   single  prefix tiles against one row tile (the last one where their number is odd);
//   own     each request's own pages against its G rows.
// CTA i takes the weighted range [i W / n, (i + 1) W / n) of that line (computed on the device:
// lengths live there), so every SM gets the same work whatever the lengths, and a unit (KV head
// and rows) is cut only where a range ends.  Each (unit, CTA) piece leaves one partial state per
// row (max, sum, accumulator), which prefix_combine_kernel joins.
//
// Items of at most kThin = 16 rows (own items of groups up to 16, the prefix of a few requests)
// turn the products around: S^T = K Q^T and O^T = V^T P^T, keys (then columns of V) along the 128
// lanes and the rows along 16 columns.  A tile then costs the tensor pipe an eighth, and its softmax
// NR <= 16 exponentials per thread in place of 128 in G of 128 threads: own items of up to 768 tokens
// of 256 requests went from 127 to 90 us.  More rows than that stay in the 128-row form, where rows
// need no exchange between threads.
//
// Up to three kernels, chained by programmatic dependent launch: prefix_mask_kernel (with
// routing only) says which rows attend each page, prefix_sm100_kernel leaves partial states,
// prefix_combine_kernel joins them.  The second is persistent, one CTA per SM, 12 warps (register
// split as in attn_fwd_sm100.cu):
//   warp 11     scheduler: walks the CTA's range, reads page ids and row masks 32 pages per load,
//               drops pages that no row attends and pushes tile descriptors into a ring; then its
//               share of the join's plan (where each row's partial states are);
//   warps 8, 10 TMA producers, of Q (two buffers) and K, and of V, into one ring of kSlots tiles;
//   warp 9      MMA issuer, one thread.  Jobs (key tile x row tile) alternate between two lanes
//               g = 0, 1, each with S[g] (fp32, 128 columns) and O[g] in TMEM: for job i it issues
//               O[g] += P(i-2) V, then S[g] = Q K^T of job i, which may overwrite P(i-2) because
//               the tensor pipe takes one thread's products in order;
//   warps 0-7   two softmax warpgroups, one per lane; thread = row (thin: = key): masks by
//               selection, running maximum (O rescaled in TMEM only when it grows by more than
//               2^8; full prefix tiles keep the reference they find, 0 in a row's first tile,
//               while the sums of their exponentials stay within bounds), exp2, P to TMEM over
//               S's columns (A operand of the next product; thin: to shared memory, B operand),
//               partials to global memory.
// S, the sums and O are fp32; P is rounded to the cache's type, as the tensor product takes it,
// and the sums are over the unrounded P.
//
// What bounds it, at 32 query and 8 KV heads of 128 bf16, pages of 64 (times of the whole decode in a CUDA
// graph):
//   prefix (256 requests, 32768 tokens): 141 us, 970 TFLOP/s.  A pair tile takes 4 k cycles, in which
//     the tensor pipe works 2 k (46 % of the kernel) and the exponential unit 2 k (50 %): each lane's
//     product -> softmax -> product chain is serial, TMEM holds no third S beside two O of 128
//     columns, and two lanes cover each other only in part;
//   own (64 requests, 8192 tokens each): 320 us, 6.7 TB/s, DRAM 83 % busy: HBM;
//   both (256 requests, 32768 + up to 768): 195 us (222 to 232 called back to back for seconds, where
//     the board's power limit lowers the clock);
//   small batches: launches, a prologue of 2.8 us, one tile's latency and the join: 14 us.
#include <algorithm>
#include <string>
#include <type_traits>

#include "prefix_decode.cuh"

namespace sa {
namespace {

constexpr int kT = 128;          // rows of a row tile, keys of a key tile
constexpr int kThreads = 384;
constexpr int kProducerWarp = 8, kMmaWarp = 9, kVWarp = 10, kSchedWarp = 11;
constexpr int kLaunchRegs = 168, kCtrlRegs = 120, kSoftmaxRegs = 192;
static_assert(4 * 32 * kCtrlRegs + 8 * 32 * kSoftmaxRegs <= kThreads * kLaunchRegs,
              "register split exceeds the launch allocation");
constexpr int kGroupThreads = 128;
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kColS = 0, kColO = 256;  // S[g] at kColS + 128 g, O[g] at kColO + 128 g
constexpr int kThin = 16;                   // rows up to which an item's products are transposed
constexpr uint32_t kThinP = 8192;           // offset of a lane's P^T in the Q buffer of the same index
constexpr int kMaxPpt = 8;                  // pages per key tile
constexpr uint32_t kMaxSmem = 232448;
constexpr float kRescaleThreshold = 8.0f;   // log2 units
constexpr int kMaxHeadWords = 8;            // query heads <= 256 (mask kernel)

// Relative cost of one key tile in the split of the work over CTAs: a pair tile (about 4000 cycles),
// a tile of either other kind, and what an item costs besides its tiles (fill, drain and partial
// states; of a pair item twice that), spread over its tiles.  With routing, own and single tiles
// count by the share of their pages that some row attends.  Fitted by timing: 256 requests on a
// prefix of 32768 and up to 768 own tokens take 195 us with these, 226 with 16 / 11 / 14 (the traced
// cycles of a tile on an idle GPU: beside pair tiles, own tiles have more of HBM to themselves),
// 228 with 24 / 9 / 9, 202 with 18 / 9 / 12, 229 with 18 / 7 / 6, 213 with 18 / 12 / 6.  Against these five, in
// the same order, at other sizes: head_dim 64, the same lengths 172 (202, 186, 179, 186, 188); prefix
// 8192 and 500 to 2000 own 238 (266, 247, 238, 244, 259), at head_dim 64 187 (238, 184, 187, 180, 232); 200
// requests of 16 / 4 heads on 6000 and up to 150 39 (46, 42, 42, 40, 40); 128 requests of 16 / 16 heads of 96
// on 5000 and up to 600 91 (98, 96, 104, 94, 87).  The worst found: 96 requests of 64 / 8 heads on 20000
// and up to 900, 114 (111, 136, 104, 131, 107).
constexpr int kCostPair = 18, kCostOne = 9, kCostItem = 6;

enum { F_FIRST = 1, F_LAST = 2, F_EMPTY = 4, F_END = 8, F_PAIR = 16, F_OWN = 32, F_THIN = 64 };

struct TileDesc {
  int flags;
  int n;     // pages
  int vr;    // valid keys: rows [0, vr) of the tile
  int kvh;
  int b0;    // first request of the row tile(s), or the request of an own item
  int slot;  // partial slot of the item
  int t0;    // first row within the page (pages longer than a tile)
  int pad;
  int phys[kMaxPpt];
  uint32_t mask[kMaxPpt][8];  // rows that attend the page: 4 words per row tile
};
static_assert(sizeof(TileDesc) == 32 + 32 + 256, "TileDesc");

template <int DT>
struct Layout {
  static constexpr uint32_t kTile = kT * DT * 2;  // one K, V or Q tile
  static constexpr int kSlots = DT == 128 ? 5 : 10;
  static constexpr int kDescs = DT == 128 ? 4 : 7;
  static constexpr uint32_t kQ = 0;
  static constexpr uint32_t kRing = kQ + 2 * kTile;
  static constexpr uint32_t kDesc = kRing + kSlots * kTile;
  static constexpr uint32_t kBars = kDesc + kDescs * sizeof(TileDesc);
  // barriers
  static constexpr int bFull = 0, bEmpty = bFull + kSlots, bQFull = bEmpty + kSlots, bQEmpty = bQFull + 2,
                       bSFull = bQEmpty + 2, bPFull = bSFull + 2, bODone = bPFull + 2, bOFree = bODone + 2,
                       bDFull = bOFree + 2, bDEmpty = bDFull + kDescs, bDrain = bDEmpty + kDescs, bNum = bDrain + 1;
  static constexpr uint32_t kMisc = kBars + bNum * 8;  // tmem slot, scan scratch, maxima of thin items
  static constexpr uint32_t kBytes = kMisc + 192 + 2 * 4 * kThin * 4;
  static constexpr uint32_t kAlloc = kBytes + 1024 <= kMaxSmem ? kBytes + 1024 : kMaxSmem;
  static_assert(kBytes <= kMaxSmem, "prefix decode: shared-memory layout too large");
};

// Sizes of the split, the same on host and device.  32-bit throughout the kernels: the launcher
// sends anything larger to the general path.
struct Split {
  int units[2];   // pair, single: KV heads x groups of row tiles
  int nb;         // requests per row tile
  int row_tiles;  // ceil(B / nb)
  int ppt;        // pages per key tile
  int sub;        // tiles per page (pages longer than a key tile), else 1
  int span;       // keys per `sub` tiles: ppt pages, or one long page
  int bn;         // TMA box rows
  int grid;
  int B, G, Hkv, page, Lp, L, D;
};

// The partial states of one (request, KV head): n states from `first`, `stride` apart.
struct Pieces {
  int first_p, n_p, stride_p, r0;  // prefix: r0 = the request's first row in the row tile
  int first_o, n_o, pad[2];        // own, one apart
};
static_assert(sizeof(Pieces) == 32, "Pieces");

struct Ws {
  Pieces* plan;       // [B][Hkv] where a request's partial states are
  uint32_t* mask_p;   // [Hkv][row_tiles][Lp][4]
  uint32_t* mask_o;   // [B][Hkv][L][WO]
  float2* ml_p;       // [prefix slots][2][128]
  float4* acc_p;      // [prefix slots][2][D / 4][128]
  float2* ml_o;       // [own slots][2][G]
  float4* acc_o;      // [own slots][2][D / 4][G]
  int* cnt_o;         // [B][chunks of own pages] selected (page, KV head) pairs
  int* cnt_p;         // [Hkv][chunks of prefix pages] pages attended by the last row tile's first 32 rows
  int WO;
};

struct Args {
  CUtensorMap tm_q, tm_q1, tm_k, tm_v;
  Split s;
  Ws w;
  const int32_t* ppages;
  const int32_t* bt;
  int64_t bts0, bts1;
  const int32_t* ctx;
  const int32_t* plen_dev;
  int plen, num_pages;
  float scale2;
  int masked;  // row masks are in w (req_depth > 0)
  unsigned* status;
};

inline Split make_split(int64_t B, int64_t G, int64_t Hkv, int64_t page, int64_t Lp, int64_t L, int64_t D) {
  Split s;
  s.nb = (int)std::min<int64_t>(B, kT / G);
  s.row_tiles = (int)((B + s.nb - 1) / s.nb);
  s.units[0] = (int)(Hkv * (s.row_tiles / 2));
  s.units[1] = (int)(Hkv * (s.row_tiles & 1));
  s.bn = (int)std::min<int64_t>(page, kT);
  s.sub = (int)((page + kT - 1) / kT);
  s.ppt = (int)std::max<int64_t>(1, std::min<int64_t>(kMaxPpt, kT / page));
  s.span = (int)page * s.ppt;
  s.grid = device_sm_count();
  s.B = (int)B;
  s.G = (int)G;
  s.Hkv = (int)Hkv;
  s.page = (int)page;
  s.Lp = (int)Lp;
  s.L = (int)L;
  s.D = (int)D;
  return s;
}

// Chunks of kMaskPages pages (the mask kernel's tasks).
constexpr int kMaskPages = 16;
__host__ __device__ inline int prefix_chunks(const Split& s) { return (s.Lp + kMaskPages - 1) / kMaskPages; }
__host__ __device__ inline int own_chunks(const Split& s) { return (s.L + kMaskPages - 1) / kMaskPages; }

inline size_t al256(size_t x) { return (x + 255) & ~(size_t)255; }

size_t carve(void* base, const Split& s, Ws* w) {
  const int64_t B = s.B, Hkv = s.Hkv, G = s.G, D = s.D, Lp = s.Lp, L = s.L;
  char* c = static_cast<char*>(base);
  size_t o = 0;
  auto take = [&](size_t bytes) {
    char* r = c ? c + o : nullptr;
    o += al256(bytes);
    return r;
  };
  Ws t;
  t.WO = G <= 32 ? 1 : 4;
  const size_t sp = (size_t)s.units[0] + s.units[1] + s.grid, so = (size_t)(B * Hkv + s.grid);
  t.plan = reinterpret_cast<Pieces*>(take((size_t)B * Hkv * sizeof(Pieces)));
  t.mask_p = reinterpret_cast<uint32_t*>(take((size_t)Hkv * s.row_tiles * Lp * 16));
  t.mask_o = reinterpret_cast<uint32_t*>(take((size_t)B * Hkv * L * t.WO * 4));
  t.cnt_o = reinterpret_cast<int*>(take((size_t)B * own_chunks(s) * 4));
  t.cnt_p = reinterpret_cast<int*>(take((size_t)Hkv * prefix_chunks(s) * 4));
  t.ml_p = reinterpret_cast<float2*>(take(sp * 2 * kT * 8));
  t.acc_p = reinterpret_cast<float4*>(take(sp * 2 * kT * D * 4));
  t.ml_o = reinterpret_cast<float2*>(take(so * 2 * G * 8));
  t.acc_o = reinterpret_cast<float4*>(take(so * 2 * G * D * 4));
  if (w) *w = t;
  return o;
}

// ---------------------------------------------------------------------------------------
// the line of work
// ---------------------------------------------------------------------------------------
struct Line {
  int tiles_p;      // key tiles of the prefix
  int wt[3];        // weight of a tile of each segment
  int64_t len[3];   // weighted lengths of the segments
  int64_t W;
  int n;            // CTAs that get a range
};

// Valid tokens of a length within a list of `width` pages.
__device__ __forceinline__ int tokens_in(int n, int width, int page) { return max(0, min(n, width * page)); }
__device__ __forceinline__ int pre_tokens(const Split& s, const int32_t* dev, int plen) {
  return tokens_in(dev ? *dev : plen, s.Lp, s.page);
}
// Key tiles of n tokens.
__device__ __forceinline__ int tiles_of(const Split& s, int n) {
  return (int)(((unsigned)n + (unsigned)s.span - 1u) / (unsigned)s.span) * s.sub;
}

// own_pages: selected (page, KV head) pairs of the own part; seen: selected (page, KV head) pairs
// of the single segment's first 32 rows.  Negative: all.
__device__ __forceinline__ Line make_line(const Split& s, int prefix_tokens, int own_total, int own_pages, int seen) {
  Line l;
  l.tiles_p = tiles_of(s, prefix_tokens);
  const int tiles1 = max(1, l.tiles_p);
  l.wt[0] = kCostPair + 2 * kCostItem / tiles1;
  l.wt[1] = kCostOne + kCostItem / tiles1;
  l.wt[2] = kCostOne;
  const int pages = (prefix_tokens + s.page - 1) / s.page;
  if (seen >= 0 && s.units[1] > 0 && pages > 0) {
    // pages that none of the row tile's 32-row words attends, taken as independent
    const int words = ((s.B - (s.row_tiles - 1) * s.nb) * s.G + 31) / 32;
    const float none = 1.f - (float)seen / ((float)s.Hkv * (float)pages);
    float all = none;
#pragma unroll 1
    for (int w = 1; w < words; ++w) all *= none;
    l.wt[1] = max(1, (int)(kCostOne * (1.f - all) + 0.5f) + kCostItem / tiles1);
  }
  if (own_total > 0) {
    const float tiles = (float)own_total * (float)s.Hkv;
    const float full = own_pages < 0 ? tiles : (float)own_pages / (float)s.ppt * (float)s.sub;
    const float items = (float)min(s.B, own_total) * (float)s.Hkv;
    l.wt[2] = max(1, (int)((kCostOne * min(full, tiles) + kCostItem * items) / tiles + 0.5f));
  }
  l.len[0] = (int64_t)s.units[0] * l.tiles_p * l.wt[0];
  l.len[1] = (int64_t)s.units[1] * l.tiles_p * l.wt[1];
  l.len[2] = (int64_t)own_total * s.Hkv * l.wt[2];
  l.W = l.len[0] + l.len[1] + l.len[2];
  // every range spans at least one tile of the heaviest kind, so that a CTA whose range lies inside
  // a unit holds a piece of it
  l.n = (int)max((int64_t)1, min((int64_t)s.grid, l.W / max(l.wt[0], max(l.wt[1], l.wt[2]))));
  return l;
}

__device__ __forceinline__ int64_t range_start(const Line& l, int i) { return i * l.W / l.n; }
// The CTA whose range holds position x.
__device__ __forceinline__ int range_of(const Line& l, int64_t x) { return (int)(((x + 1) * l.n - 1) / l.W); }

__device__ __forceinline__ uint32_t pack2(float lo, float hi, bool bf16) {
  uint32_t r;
  if (bf16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// ---------------------------------------------------------------------------------------
// row masks (req_depth > 0): which rows attend each page
// ---------------------------------------------------------------------------------------
// Warp task: 16 pages against 32 rows (prefix: rows of one mask word; own: 32 heads at a time of one
// request).  Lane = row: its r levels against the 16 pages' vectors, 16 loads in flight per
// level; a ballot per page is the page's mask word.  Integer compares of a few MB that sit in L2.
constexpr int kMaskWarps = 4;

struct MaskArgs {
  Split s;
  Ws w;
  const int32_t* ppages;
  const int32_t* bt;
  int64_t bts0, bts1;
  const int32_t* ctx;
  const int32_t* plen_dev;
  const void* router;
  int64_t rs[3];
  const void* qrouter;
  int64_t qrs[3];
  int plen, num_pages, q64, r, local, sink, H;
  int prefix_tasks, tasks;
};

template <typename RT>
__global__ void __launch_bounds__(kMaskWarps * 32) prefix_mask_kernel(const __grid_constant__ MaskArgs a) {
  __shared__ uint32_t s_bits[kMaskWarps][kMaskPages][kMaxHeadWords];
  pdl_trigger();
  const Split& s = a.s;
  const Ws& w = a.w;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const RT* router = static_cast<const RT*>(a.router);
  const int pre_pages = (pre_tokens(s, a.plen_dev, a.plen) + s.page - 1) / s.page;
  // bits u < pages: whether page u's vector equals the row's on the first r levels.  All pages of a level
  // in flight, r round trips (4 pages x 4 levels at a time take 4 at least: the whole decode at depth 1,
  // 9001 tokens of 32 per page, 26.2 us against 24.5; at depth 4 they are level, 86 to 88).
  auto match = [&](int phys, int pages, int b, int h) -> uint32_t {
    uint32_t on = (1u << pages) - 1u;
    const RT* rh = router + h * a.rs[1];
    const int64_t qo = b * a.qrs[0] + h * a.qrs[1];
#pragma unroll 1
    for (int lv = 0; lv < a.r; ++lv) {
      const int64_t q = load_any_i64(a.qrouter, a.q64 ? SA_I64 : SA_I32, qo + lv * a.qrs[2]);
      RT v[kMaskPages];
#pragma unroll
      for (int u = 0; u < kMaskPages; ++u)
        v[u] = __ldg(rh + (int64_t)__shfl_sync(0xffffffffu, phys, u) * a.rs[0] + lv * a.rs[2]);
#pragma unroll
      for (int u = 0; u < kMaskPages; ++u)
        if ((int64_t)v[u] != q) on &= ~(1u << u);
    }
    return on;
  };
  for (int task = (int)blockIdx.x * kMaskWarps + warp; task < a.tasks; task += (int)gridDim.x * kMaskWarps) {
    if (task < a.prefix_tasks) {
      const int chunks = prefix_chunks(s);
      int x = task / chunks;
      const int chunk = task - x * chunks, l0 = chunk * kMaskPages, word = x & 3;
      x >>= 2;
      const int g = x / s.row_tiles, rt = x - g * s.row_tiles;
      const bool counted = word == 0 && rt == s.row_tiles - 1 && (s.row_tiles & 1);
      uint32_t bits = 0;
      const int row = word * 32 + lane, rb = row / s.G, b = rt * s.nb + rb;
      const bool live = row < s.nb * s.G && b < s.B;
      int n = pre_pages;
      if (l0 < pre_pages && word * 32 < s.nb * s.G) {
        int phys = lane < kMaskPages && l0 + lane < pre_pages ? a.ppages[l0 + lane] : 0;
        if (phys < 0 || phys >= a.num_pages) phys = 0;  // dropped by the scheduler
        if (a.local > 0 && live) n += (tokens_in(a.ctx[b], s.L, s.page) + s.page - 1) / s.page;
        bits = match(phys, min(kMaskPages, pre_pages - l0), live ? b : 0, live ? g * s.G + row - rb * s.G : 0);
      }
      // forced pages: the sink, and the last `local` of the row's n pages
      uint32_t forced = a.sink && l0 == 0 ? 1u : 0u;
      const int first = n - a.local - l0;  // first forced page of this chunk
      if (a.local > 0 && first < kMaskPages) forced |= ~0u << max(0, first);
      bits = live ? bits | forced : 0u;
      int count = 0;
#pragma unroll 1
      for (int u = 0; u < kMaskPages; ++u) {
        const uint32_t m = __ballot_sync(0xffffffffu, (bits >> u) & 1u);
        if (l0 + u < pre_pages) {
          count += m != 0u;
          if (lane == 0) w.mask_p[(((int64_t)g * s.row_tiles + rt) * s.Lp + l0 + u) * 4 + word] = m;
        }
      }
      if (counted && lane == 0) w.cnt_p[g * chunks + chunk] = count;
    } else {
      const int t = task - a.prefix_tasks, chunks = own_chunks(s), b = t / chunks, l0 = (t - b * chunks) * kMaskPages;
      const int pages = (tokens_in(a.ctx[b], s.L, s.page) + s.page - 1) / s.page;
      if (l0 >= pages) {
        if (lane == 0) w.cnt_o[t] = 0;
        continue;
      }
      int phys = lane < kMaskPages && l0 + lane < pages ? a.bt[b * a.bts0 + (l0 + lane) * a.bts1] : 0;
      if (phys < 0 || phys >= a.num_pages) phys = 0;
      uint32_t forced = a.sink && pre_pages + l0 == 0 ? 1u : 0u;
      const int first = pages - a.local - l0;
      if (a.local > 0 && first < kMaskPages) forced |= ~0u << max(0, first);
      const int HW = (a.H + 31) / 32;
      for (int hw = 0; hw < HW; ++hw) {
        const int h = hw * 32 + lane;
        const bool live = h < a.H;
        uint32_t bits = match(phys, min(kMaskPages, pages - l0), b, live ? h : 0) | forced;
        if (!live) bits = 0;
#pragma unroll 1
        for (int u = 0; u < kMaskPages; ++u) {
          const uint32_t m = __ballot_sync(0xffffffffu, (bits >> u) & 1u);
          if (lane == 0) s_bits[warp][u][hw] = m;
        }
      }
      __syncwarp();
      // each KV head's G bits out of the H
      int count = 0;  // (page, KV head) pairs that some head attends
      const int per = s.Hkv * w.WO;
      for (int i = lane; i < kMaskPages * per; i += 32) {
        const int u = i / per, gw = i - u * per, g = gw / w.WO, wd = gw - g * w.WO;
        if (l0 + u >= pages) continue;
        const int first_h = g * s.G + wd * 32, cnt = min(32, s.G - wd * 32);
        uint32_t m = 0;
        if (cnt > 0) {
          const int q = first_h >> 5;
          uint64_t v = s_bits[warp][u][q];
          if (q + 1 < HW) v |= (uint64_t)s_bits[warp][u][q + 1] << 32;
          m = (uint32_t)(v >> (first_h & 31));
          if (cnt < 32) m &= (1u << cnt) - 1u;
        }
        w.mask_o[(((int64_t)b * s.Hkv + g) * s.L + l0 + u) * w.WO + wd] = m;
        count += m != 0u;
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) count += __shfl_xor_sync(0xffffffffu, count, o);
      if (lane == 0) w.cnt_o[t] = count;
      __syncwarp();
    }
  }
}

// ---------------------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------------------
// Warp maximum of a float, and a barrier of `threads` threads that returns how many brought pred.
__device__ __forceinline__ float redux_max(float x) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ int named_bar_count(uint32_t id, uint32_t threads, bool pred) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.popc.u32 %0, %2, %3, p;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)pred), "r"(id), "r"(threads)
      : "memory");
  return (int)r;
}

// 32 lanes x N consecutive 32-bit columns (N = 4, 8 or 16).
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

template <int N>
__device__ __forceinline__ void tmem_ldn(uint32_t taddr, float (&v)[N]) {
  if constexpr (N == 16) {
    tmem_ld16(taddr, v);
  } else if constexpr (N == 8) {
    uint32_t r[8];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]);
  } else {
    uint32_t r[4];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(taddr));
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(r[i]);
  }
}
template <int N>
__device__ __forceinline__ void tmem_stn(uint32_t taddr, const uint32_t (&v)[N]) {
  if constexpr (N == 16)
    tmem_st16(taddr, v);
  else if constexpr (N == 8)
    tmem_st8(taddr, v);
  else
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" ::"r"(taddr), "r"(v[0]), "r"(v[1]),
                 "r"(v[2]), "r"(v[3])
                 : "memory");
}

// Bounded waits as in common.cuh, counted in tries instead of timed: half the instructions at each
// of the kernel's dozen waits, which matters where every role's code competes for the
// instruction cache.  A try on a phase that stays incomplete suspends the thread for about 8 k
// cycles, so kMaxTries of them are about a second.  A warp whose wait gives up leaves its role, and the
// others run into their own limits; the MMA issuer ends after its products and, where it did not come
// to the last item (so that loads may be unused), after the loads in flight, with a limit too.
constexpr uint32_t kMaxTries = 1u << 18;

__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, unsigned* st) {
  for (uint32_t n = 0; !mbar_try_wait(bar, parity); ++n)
    if (n == kMaxTries) {
      raise_status(st, kStatusWaitTimeout);
      return false;
    }
  return true;
}
__device__ __forceinline__ bool wait_bar_warp(uint64_t* bar, uint32_t parity, unsigned* st) {
  return __all_sync(0xffffffffu, wait_bar(bar, parity, st));
}

// Loads in flight where the MMA issuer gave up: the ring's entries from the oldest that is not released
// (u), then the Q buffers.  Entries released out of turn (K of tiles before k_end / 2) have passed to
// the entry a ring's length on.  What was never issued runs into the limit.
template <uint32_t kSlots>
__device__ __noinline__ void settle(uint64_t* full, uint64_t* q_full, uint32_t u, uint32_t k_end, uint32_t nq) {
  uint32_t open = (1u << (kSlots + 2)) - 1u;
  const long long t0 = clock64();
  while (open && clock64() - t0 < (1ll << 31)) {
#pragma unroll 1
    for (uint32_t i = 0; i < kSlots + 2; ++i) {
      uint32_t e = u + i;
      if (!(e & 1) && e < k_end) e += kSlots;
      const uint32_t q = nq + i - kSlots;
      if (i < kSlots ? mbar_test(full + e % kSlots, (e / kSlots) & 1) : mbar_test(q_full + (q & 1), (q >> 1) & 1))
        open &= ~(1u << i);
    }
  }
}

template <int DT, bool BF16>
__global__ void __launch_bounds__(kThreads, 1) prefix_sm100_kernel(const __grid_constant__ Args a) {
  using L = Layout<DT>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  {
    const uint32_t base = smem_u32(smem_raw);
    uint32_t dyn;
    asm("mov.u32 %0, %%dynamic_smem_size;" : "=r"(dyn));
    if ((((base + 1023u) & ~1023u) - base) + L::kBytes > dyn) {  // uniform over the CTA
      if (threadIdx.x == 0) raise_status(a.status, kStatusSmemLayout);
      return;
    }
  }
  unsigned char* sm = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + L::kBars);
  TileDesc* descs = reinterpret_cast<TileDesc*>(sm + L::kDesc);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + L::kMisc);
  int* s_warp = reinterpret_cast<int*>(sm + L::kMisc + 16);       // [12] scan
  int* s_start = reinterpret_cast<int*>(sm + L::kMisc + 64);      // first own request, tiles before it
  int* s_cnt = reinterpret_cast<int*>(sm + L::kMisc + 80);        // [12][2] selected pages
  const Split& S = a.s;
  unsigned* st = a.status;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kSlots; ++i) {
      mbar_init(&bars[L::bFull + i], 1);
      mbar_init(&bars[L::bEmpty + i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars[L::bQFull + i], 1);
      mbar_init(&bars[L::bQEmpty + i], 1);
      mbar_init(&bars[L::bSFull + i], 1);
      mbar_init(&bars[L::bPFull + i], 4);  // the group's warps
      mbar_init(&bars[L::bODone + i], 1);
      mbar_init(&bars[L::bOFree + i], 4);
    }
    mbar_init(&bars[L::bDrain], 1);
    for (int i = 0; i < L::kDescs; ++i) {
      mbar_init(&bars[L::bDFull + i], 1);
      mbar_init(&bars[L::bDEmpty + i], 3 + 8);  // two producers, MMA warp, 8 softmax warps
    }
    fence_mbar_init();
    prefetch_tmap(&a.tm_k);
    prefetch_tmap(&a.tm_v);
    prefetch_tmap(&a.tm_q);
    prefetch_tmap(&a.tm_q1);
  }
  if (warp == kVWarp) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  // ---- own tiles over the requests: every CTA scans them (thread = consecutive requests)
  const int bper = (S.B + kThreads - 1) / kThreads;
  const int bfirst = min(S.B, (int)threadIdx.x * bper), bend = min(S.B, bfirst + bper);
  int mine = 0;
#pragma unroll 1
  for (int b = bfirst; b < bend; ++b) mine += tiles_of(S, tokens_in(a.ctx[b], S.L, S.page));
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) s_warp[warp] = incl;
  if (threadIdx.x == 0) s_start[0] = S.B;
  const int ptok = pre_tokens(S, a.plen_dev, a.plen);
  if (a.masked) {  // selected pages, for the tiles' weights
    pdl_wait();    // the row masks and their counts are complete from here on
    int2 sel = make_int2(0, 0);
    const int no = S.B * own_chunks(S), npc = S.units[1] > 0 ? S.Hkv * prefix_chunks(S) : 0;
#pragma unroll 4
    for (int i = threadIdx.x; i < no; i += kThreads) sel.x += __ldcg(a.w.cnt_o + i);
#pragma unroll 4
    for (int i = threadIdx.x; i < npc; i += kThreads) sel.y += __ldcg(a.w.cnt_p + i);
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      sel.x += __shfl_xor_sync(0xffffffffu, sel.x, o);
      sel.y += __shfl_xor_sync(0xffffffffu, sel.y, o);
    }
    if (lane == 0) {
      s_cnt[2 * warp] = sel.x;
      s_cnt[2 * warp + 1] = sel.y;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  int before = incl - mine, own_total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    const int t = s_warp[w];
    before += w < warp ? t : 0;
    own_total += t;
  }
  int own_pages = -1, seen = -1;
  if (a.masked) {
    own_pages = seen = 0;
#pragma unroll 1
    for (int w = 0; w < kThreads / 32; ++w) {
      own_pages += s_cnt[2 * w];
      seen += s_cnt[2 * w + 1];
    }
  }
  const Line line = make_line(S, ptok, own_total, own_pages, seen);
  const bool active = (int)blockIdx.x < line.n && line.W > 0;
  const int64_t x0 = active ? range_start(line, blockIdx.x) : 0, x1 = active ? range_start(line, blockIdx.x + 1) : 0;
  // the CTA's tiles [lo, hi) of a segment that starts at `base` and whose tiles weigh wt
  auto seg_lo = [&](int64_t base, int wt) { return (int)((max((int64_t)0, x0 - base) + wt - 1) / wt); };
  auto seg_hi = [&](int64_t base, int64_t len, int wt) {
    return (int)((max((int64_t)0, min(len, x1 - base)) + wt - 1) / wt);
  };
  const int64_t own_base = line.len[0] + line.len[1];
  // own tiles [k0, k1) of the CTA; the thread whose requests hold k0 publishes the first one
  const int k0 = seg_lo(own_base, line.wt[2]), k1 = seg_hi(own_base, line.len[2], line.wt[2]);
  {
    int c = before;
#pragma unroll 1
    for (int b = bfirst; b < bend; ++b) {
      const int t = tiles_of(S, tokens_in(a.ctx[b], S.L, S.page));
      if (k0 >= c * S.Hkv && k0 < (c + t) * S.Hkv) {
        s_start[0] = b;
        s_start[1] = c;
      }
      c += t;
    }
  }
  __syncthreads();
  pdl_trigger();
  const uint32_t tmem = *tmem_slot;

  if (warp >= kProducerWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kCtrlRegs));
    if (warp == kSchedWarp) {
      // ---------------------------------------------------------------- scheduler
      const int ppt = S.ppt, sub = S.sub, bn = S.bn;
      uint32_t d = 0;  // descriptors pushed
      bool ok = true;
      // position in the line: segment (pair, single, own), tiles [k, hi) of it, and in the own
      // segment the request b with c tiles (of one KV head) before it and t of its own
      int seg = -1, k = 0, hi = 0, b = 0, c = 0, t = 0, own_tok = 0;
      while (ok) {
        while (k >= hi && seg < 3) {  // the next segment with work
          ++seg;
          if (!active || seg > 2) {
            seg = 3;
          } else if (seg == 2) {
            k = k0;
            hi = k1;
            b = s_start[0];
            c = s_start[1];
            if (k < hi) {
              own_tok = tokens_in(a.ctx[b], S.L, S.page);
              t = tiles_of(S, own_tok);
            }
          } else {
            const int64_t base = seg ? line.len[0] : 0, len = seg ? line.len[1] : line.len[0];
            const int wt = seg ? line.wt[1] : line.wt[0];
            k = seg_lo(base, wt);
            hi = seg_hi(base, len, wt);
          }
        }
        // ---- the next item: tiles [ta, tb) of one unit
        int flags = F_END, kvh = 0, b0 = 0, slot = 0, ta = 0, tb = 0, tokens = 0, mwords = 4;
        const int32_t* ids = a.ppages;
        int64_t ids_stride = 1;
        const uint32_t *mask0 = nullptr, *mask1 = nullptr;
        if (seg < 2) {
          const int u = k / line.tiles_p, groups = seg == 0 ? S.row_tiles / 2 : 1;
          ta = k - u * line.tiles_p;
          tb = min(line.tiles_p, ta + hi - k);
          kvh = u / groups;
          const int rt = seg == 0 ? (u - kvh * groups) * 2 : S.row_tiles - 1;
          flags = seg == 0 ? F_PAIR : S.B * S.G <= kThin ? F_THIN : 0;
          b0 = rt * S.nb;
          slot = (seg ? S.units[0] : 0) + u + (int)blockIdx.x;
          tokens = ptok;
          mask0 = a.w.mask_p + ((int64_t)kvh * S.row_tiles + rt) * S.Lp * 4;
          if (seg == 0) mask1 = mask0 + (int64_t)S.Lp * 4;
        } else if (seg == 2) {
          while (k >= (c + t) * S.Hkv) {  // hi > k: there is such a request
            c += t;
            own_tok = tokens_in(a.ctx[++b], S.L, S.page);
            t = tiles_of(S, own_tok);
          }
          const int r = k - c * S.Hkv;
          kvh = r / t;
          ta = r - kvh * t;
          tb = min(t, ta + hi - k);
          flags = F_OWN | (S.G <= kThin ? F_THIN : 0);
          b0 = b;
          slot = b * S.Hkv + kvh + (int)blockIdx.x;
          tokens = own_tok;
          ids = a.bt + b * a.bts0;
          ids_stride = a.bts1;
          mwords = a.w.WO;
          mask0 = a.w.mask_o + ((int64_t)b * S.Hkv + kvh) * S.L * mwords;
        }
        k += tb - ta;
        // ---- its entries: pages, or 128-key parts of longer pages
        TileDesc* td;
        int cur = 0, vr = 0, t0cur = 0, more = 1;
        int eb = ta * ppt, e1 = tb * ppt;
        int first = F_FIRST, total = 0, done = 0, phys = 0, valid = 0, t0 = 0, rank = 0;
        bool live = false;
        uint4 m0, m1;
        while (more) {  // one descriptor per turn
          td = &descs[d % L::kDescs];
          if (!(ok = wait_bar_warp(&bars[L::bDEmpty + d % L::kDescs], ((d / L::kDescs) & 1) ^ 1, st))) break;
          cur = 0;
          while (true) {
            if (done == total) {  // the next 32 entries
              if (eb >= e1) break;
              const int e = eb + lane, l = sub == 1 ? e : e / sub;
              t0 = sub == 1 ? 0 : (e - l * sub) * kT;
              valid = e < e1 ? min(kT, min(S.page, tokens - l * S.page) - t0) : 0;
              phys = -1;
              m0 = m1 = make_uint4(~0u, ~0u, ~0u, ~0u);
              if (valid > 0) {
                phys = ids[l * ids_stride];
                if (a.masked) {
                  m1 = make_uint4(0u, 0u, 0u, 0u);
                  if (mwords == 1) {
                    m0 = make_uint4(__ldcg(mask0 + l), 0u, 0u, 0u);
                  } else {
                    m0 = __ldcg(reinterpret_cast<const uint4*>(mask0) + l);
                    if (mask1) m1 = __ldcg(reinterpret_cast<const uint4*>(mask1) + l);
                  }
                }
                if (phys < 0 || phys >= a.num_pages) {
                  raise_status(st, kStatusBadIndex);
                  valid = 0;
                }
              }
              live = valid > 0 && ((m0.x | m0.y | m0.z | m0.w) | (m1.x | m1.y | m1.z | m1.w)) != 0u;
              const unsigned bal = __ballot_sync(0xffffffffu, live);
              total = __popc(bal);
              rank = __popc(bal & ((1u << lane) - 1u));
              done = 0;
              eb += 32;
              continue;
            }
            if (cur == ppt) break;
            const int take = min(ppt - cur, total - done);
            if (live && rank >= done && rank < done + take) {
              const int j = cur + rank - done;
              td->phys[j] = phys;
              *reinterpret_cast<uint4*>(&td->mask[j][0]) = m0;
              *reinterpret_cast<uint4*>(&td->mask[j][4]) = m1;
            }
            cur += take;
            done += take;
            // the lane that holds the last page taken
            const int last = __ffs(__ballot_sync(0xffffffffu, live && rank == done - 1)) - 1;
            vr = (cur - 1) * bn + __shfl_sync(0xffffffffu, valid, last);
            t0cur = __shfl_sync(0xffffffffu, t0, last);
          }
          more = done < total;  // a page is left over for another tile
          if (lane == 0) {
            td->flags = flags | first | (more ? 0 : F_LAST) | (cur == 0 ? F_EMPTY : 0);
            td->n = cur;
            td->vr = vr;
            td->kvh = kvh;
            td->b0 = b0;
            td->slot = slot;
            td->t0 = t0cur;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars[L::bDFull + d % L::kDescs]);
          ++d;
          first = 0;
        }
        if (flags & F_END) break;
      }
      // ---- plan of the join, while the last tiles are under way
      // Where the partial states of the CTA's share of the requests are (lane = KV head): the CTAs
      // whose ranges hold the first and last tile of the prefix unit and of the own unit.
      const int per = (S.B + (int)gridDim.x - 1) / (int)gridDim.x;
      const int ba = min(S.B, (int)blockIdx.x * per), bz = min(S.B, ba + per);
      int cum = 0;
      if (ba < bz) {
#pragma unroll 4
        for (int b = lane; b < ba; b += 32) cum += tiles_of(S, tokens_in(a.ctx[b], S.L, S.page));
#pragma unroll
        for (int o = 16; o; o >>= 1) cum += __shfl_xor_sync(0xffffffffu, cum, o);
      }
#pragma unroll 1
      for (int b = ba; b < bz; ++b) {
        const int t = tiles_of(S, tokens_in(a.ctx[b], S.L, S.page));
        const int rt = b / S.nb, pairs = S.row_tiles / 2;
        const bool pr = rt < 2 * pairs;
#pragma unroll 1
        for (int g = lane; g < S.Hkv; g += 32) {
          Pieces q{0, 0, pr ? 2 : 1, (b - rt * S.nb) * S.G, 0, 0, {0, 0}};
          if (line.tiles_p > 0) {
            const int u = pr ? g * pairs + rt / 2 : S.units[0] + g, wt = pr ? line.wt[0] : line.wt[1];
            const int64_t x = pr ? (int64_t)u * line.tiles_p * wt : line.len[0] + (int64_t)g * line.tiles_p * wt;
            const int i0 = range_of(line, x);
            q.n_p = (range_of(line, x + (int64_t)(line.tiles_p - 1) * wt) - i0 + 1) * (pr ? 1 : 2);
            q.first_p = (u + i0) * 2 + (pr ? rt & 1 : 0);
          }
          if (t > 0) {
            const int64_t x = own_base + ((int64_t)cum * S.Hkv + g * t) * line.wt[2];
            const int i0 = range_of(line, x);
            q.n_o = (range_of(line, x + (int64_t)(t - 1) * line.wt[2]) - i0 + 1) * 2;
            q.first_o = (b * S.Hkv + g + i0) * 2;
          }
          a.w.plan[(int64_t)b * S.Hkv + g] = q;
        }
        cum += t;
      }
    } else if (warp == kProducerWarp || warp == kVWarp) {
      // ---------------------------------------------------------------- TMA producers
      // Warp kProducerWarp loads Q and K, warp kVWarp V: issuing a tile's loads takes a warp up to 800
      // cycles, and items of one tile (short own contexts) come every 2 k.
      const bool is_v = warp == kVWarp;
      const CUtensorMap* tm = is_v ? &a.tm_v : &a.tm_k;
      const int dc = (S.D + 63) / 64;  // 64-column chunks
      const int bn = S.bn;
      uint32_t d = 0, seq = is_v ? 1 : 0, nq = 0;
      bool ok = true;
      while (ok) {
        const uint32_t ds = d % L::kDescs;
        if (!wait_bar_warp(&bars[L::bDFull + ds], (d / L::kDescs) & 1, st)) break;
        const TileDesc& td = descs[ds];
        const int flags = td.flags;
        if (flags & F_END) break;
        if (!(flags & F_EMPTY)) {
          const int kvh = td.kvh, b0 = td.b0, n = td.n, t0 = td.t0;
          if (!is_v && (flags & F_FIRST)) {
            const int tiles = flags & F_PAIR ? 2 : 1;
            for (int i = 0; i < tiles && ok; ++i, ++nq) {
              const uint32_t qb = nq & 1;
              if (!(ok = wait_bar_warp(&bars[L::bQEmpty + qb], ((nq >> 1) & 1) ^ 1, st))) break;
              if (elect_one()) {
                unsigned char* dst = sm + L::kQ + qb * L::kTile;
                const uint32_t rows = (uint32_t)((flags & F_OWN) ? S.G : S.nb * S.G);
                mbar_arrive_expect_tx(&bars[L::bQFull + qb], rows * 128 * dc);
                for (int c = 0; c < dc; ++c)
                  tma_load_4d(dst + c * (kT * 128), (flags & F_OWN) ? &a.tm_q1 : &a.tm_q, &bars[L::bQFull + qb], c * 64,
                              0, kvh, b0 + i * S.nb);
              }
              __syncwarp();
            }
          }
          const uint32_t sl = seq % L::kSlots;
          if (!ok || !wait_bar_warp(&bars[L::bEmpty + sl], ((seq / L::kSlots) & 1) ^ 1, st)) break;
          if (elect_one()) {
            unsigned char* dst = sm + L::kRing + sl * L::kTile;
            mbar_arrive_expect_tx(&bars[L::bFull + sl], (uint32_t)(n * bn * 128 * dc));
#pragma unroll 1
            for (int j = 0; j < n; ++j, dst += bn * 128) {
              const int phys = td.phys[j];
              tma_load_4d(dst, tm, &bars[L::bFull + sl], 0, t0, kvh, phys);
              if (dc > 1) tma_load_4d(dst + kT * 128, tm, &bars[L::bFull + sl], 64, t0, kvh, phys);
            }
          }
          __syncwarp();
          seq += 2;
        }
        if (lane == 0) mbar_arrive(&bars[L::bDEmpty + ds]);
        ++d;
      }
    } else if (warp == kMmaWarp) {
      // ---------------------------------------------------------------- MMA issuer (one thread)
      if (elect_one()) {
      const int dk = (S.D + 15) / 16;  // K steps of Q K^T, and N / 16 of P V
      const uint32_t id_pv = idesc_f16(kT, dk * 16, BF16, false, true);
      // thin items: S^T = K Q^T and O^T = V^T P^T, the keys (the head_dim) along the 128 lanes and the
      // rows along 16 columns.  V^T spans 128 lanes in two 64-column chunks; where the tile has only
      // one, the second half (any in-bounds data) lands in lanes that nobody reads.
      constexpr uint32_t id_qk_t = idesc_f16(kT, kThin, BF16, false, false);
      constexpr uint32_t id_pv_t = idesc_f16(kT, kThin, BF16, true, false);
      constexpr uint32_t kVtLbo = DT == 128 ? kT * 128 : 1024;
      struct Job {
        uint32_t tile;  // key tile index: K in ring entry 2 tile, V in 2 tile + 1
        int vr;
        uint32_t bits;  // lane | J_*
      };
      enum : uint32_t { J_FIRST = 2, J_LAST = 4, J_REL = 8, J_THIN = 16 };
      Job j0{}, j1{};  // pending P V products, j0 the older
      int np = 0;
      uint32_t d = 0, tile = 0, job = 0, nq = 0, pc[2] = {0, 0}, of[2] = {0, 0};
      int in_item = 0;          // key tiles of the item so far
      int left = 0, rts = 0;    // row tiles of the current key tile still to multiply, of how many
      int flags = 0, vr = 0, stage = 0;
      bool flush = false, end = false;
      long long idle = clock64();
      // Polls what it may do next: a pending P V once its P is there (at the latest before the Q K^T
      // that reuses its lane), and meanwhile the next key tile's descriptor, Q and K, so that
      // the lane's next Q K^T follows its P V at once.
      while (true) {
        bool busy = false;
        // ---- the next key tile: descriptor, then Q of a new item, then K
        if (stage == 0 && !flush && mbar_test(&bars[L::bDFull + d % L::kDescs], (d / L::kDescs) & 1)) {
          const uint32_t ds = d % L::kDescs;
          flags = descs[ds].flags;
          vr = descs[ds].vr;
          // at the end, and where an item has nothing to multiply, finish what is pending: the softmax
          // groups wait for their last item's accumulators before they release more descriptors
          flush = flags & (F_END | F_EMPTY);
          if (!(flags & F_END)) mbar_arrive(&bars[L::bDEmpty + ds]);
          ++d;
          if (!flush) {
            rts = flags & F_PAIR ? 2 : 1;
            stage = flags & F_FIRST ? 1 : 2;
            if (flags & F_FIRST) in_item = 0;
          }
          busy = true;
        }
        if (stage == 1 && mbar_test(&bars[L::bQFull + (nq & 1)], (nq >> 1) & 1) &&
            (rts == 1 || mbar_test(&bars[L::bQFull + ((nq + 1) & 1)], ((nq + 1) >> 1) & 1)))
          stage = 2;
        if (stage == 2 && mbar_test(&bars[L::bFull + (2 * tile) % L::kSlots], ((2 * tile) / L::kSlots) & 1)) {
          stage = 3;
          left = rts;
          busy = true;
        }
        const uint32_t pg = j0.bits & 1u, pph = (pg ? pc[1] : pc[0]) & 1;
        // nothing else to do before the older pending P arrives: wait for it
        if (np == 2 && stage == 3 && !wait_bar(&bars[L::bPFull + pg], pph, st)) break;
        if (np > 0 && (np == 2 || stage != 3) && mbar_test(&bars[L::bPFull + pg], pph)) {
          // ---- O[g] += P V
          const uint32_t g = pg;
          const uint32_t seq = 2 * j0.tile + 1, sl = seq % L::kSlots;
          if (j0.bits & J_FIRST) {  // O[g] has been read by the last item's epilogue
            if (!wait_bar(&bars[L::bOFree + g], ((g ? of[1] : of[0]) & 1) ^ 1, st)) break;
            if (g) ++of[1]; else ++of[0];
          }
          if (!wait_bar(&bars[L::bFull + sl], (seq / L::kSlots) & 1, st)) break;
          const int n16 = (j0.vr + 15) & ~15;
          if (g) ++pc[1]; else ++pc[0];
          tc_fence_after();
          uint64_t vd = smem_desc(smem_u32(sm + L::kRing + sl * L::kTile), kT * 128, 1024);
          const uint32_t d_o = tmem + kColO + g * kT;
          uint32_t a_p = tmem + kColS + g * kT, acc = (j0.bits & J_FIRST) ? 0u : 1u;
          if (j0.bits & J_THIN) {
            vd = smem_desc(smem_u32(sm + L::kRing + sl * L::kTile), kVtLbo, 1024);
            uint64_t pd = smem_desc(smem_u32(sm + L::kQ + g * L::kTile + kThinP), 16, 1024);
#pragma unroll 1
            for (int kk = 0; kk < n16; kk += 16, acc = 1u, vd = desc_add(vd, 16 * 128)) {
              tc_mma_f16(d_o, vd, pd, id_pv_t, acc);
              pd = desc_add(pd, (kk & 48) == 48 ? kThin * 128 - 96 : 32);
            }
          } else {
#pragma unroll 1
            for (int kk = 0; kk < n16; kk += 16, a_p += 8, acc = 1u, vd = desc_add(vd, 16 * 128))
              tc_mma_f16_ts(d_o, a_p, vd, id_pv, acc);
          }
          if (j0.bits & J_REL) tc_commit(&bars[L::bEmpty + sl]);
          if (j0.bits & J_LAST) tc_commit(&bars[L::bODone + g]);
          j0 = j1;
          --np;
          busy = true;
        } else if (flush && np == 0) {
          if ((end = flags & F_END)) break;
          flush = false;
        }
        if (stage == 3 && np < 2) {
          // ---- S[g] = Q K^T
          const uint32_t g = job & 1, sl = (2 * tile) % L::kSlots, qb = (nq + rts - left) & 1;
          tc_fence_after();
          const bool thin = flags & F_THIN;
          const uint32_t id_qk = thin ? id_qk_t : idesc_f16(kT, (vr + 15) & ~15, BF16, false, false);
          uint64_t qd = smem_desc(smem_u32(sm + L::kQ + qb * L::kTile), 16, 1024);
          uint64_t kd = smem_desc(smem_u32(sm + L::kRing + sl * L::kTile), 16, 1024);
          const uint32_t d_s = tmem + kColS + g * kT;
#pragma unroll 1
          for (int kk = 0; kk < dk; ++kk) {
            tc_mma_f16(d_s, thin ? kd : qd, thin ? qd : kd, id_qk, kk > 0 ? 1u : 0u);
            const uint32_t step = (kk & 3) == 3 ? kT * 128 - 96 : 32;  // the next 16 columns
            qd = desc_add(qd, step);
            kd = desc_add(kd, step);
          }
          tc_commit(&bars[L::bSFull + g]);
          if (left == 1) tc_commit(&bars[L::bEmpty + sl]);
          if (flags & F_LAST) tc_commit(&bars[L::bQEmpty + qb]);
          // the lane's first product of the item: its first tile's, or, where the lanes take the tiles
          // in turn, its second tile's
          Job j;
          j.tile = tile;
          j.vr = vr;
          j.bits = g | ((in_item == 0 || (rts == 1 && in_item == 1)) ? J_FIRST : 0u) | ((flags & F_LAST) ? J_LAST : 0u) |
                   (left == 1 ? J_REL : 0u) | (thin ? J_THIN : 0u);
          if (rts == 1 && (flags & F_LAST) && in_item > 0) {
            // the other lane's last product of the item is the one before this: pending, or issued
            if (np > 0) j0.bits |= J_LAST;
            else tc_commit(&bars[L::bODone + (g ^ 1)]);
          }
          if (np == 0) j0 = j; else j1 = j;
          ++np;
          ++job;
          if (--left == 0) {
            stage = 0;
            ++tile;
            ++in_item;
            if (flags & F_LAST) nq += rts;
          }
          busy = true;
        }
        if (busy) {
          idle = clock64();
        } else if (clock64() - idle > (1ll << 31)) {
          raise_status(st, kStatusWaitTimeout);
          break;
        }
      }
      tc_commit(&bars[L::bDrain]);
      wait_bar(&bars[L::bDrain], 0, st);
      if (__builtin_expect(!end, 0)) {
        settle<L::kSlots>(&bars[L::bFull], &bars[L::bQFull], np > 0 ? 2 * j0.tile + 1 : 2 * tile, 2 * tile, nq);
      }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    // ------------------------------------------------------------------ softmax warpgroups
    const int grp = warp >> 2, quarter = warp & 3;
    const int rl = quarter * 32 + lane;  // row of the tile == TMEM lane
    const uint32_t lane_addr = tmem + ((uint32_t)(quarter * 32) << 16);
    const uint32_t col_s = kColS + grp * kT, col_o = kColO + grp * kT;
    const float sc2 = a.scale2;
    const int G = S.G;
    uint32_t d = 0, job = 0, tile = 0, sc = 0, od = 0;
    float m_used = -INFINITY, l_sum = 0.f;
    bool had = false;
    int sub = 0;        // which of the slot's two states this group writes
    bool row_ok = false;
    int slot = 0;
    const int my_page = rl / S.bn;  // page of this key within a tile
    float* s_max = reinterpret_cast<float*>(sm + L::kMisc + 192) + grp * 4 * kThin;  // [4 warps][kThin]
    // The group's warps meet at a named barrier, which has no limit of its own: a warp whose wait gave
    // up must not leave the others in it.  So a warp at the end of its role keeps meeting them until
    // all four are there, one thread of it counted; the others, 32 threads of a warp or none, run
    // into their own limits meanwhile.
    auto meet = [&](bool pred) -> bool { return named_bar_count(1 + grp, kGroupThreads, pred) >= 32; };
    // V rows past the valid keys meet P = 0 in the product's last K step: they must be finite, so they
    // are cleared (in a pair tile by both groups, with the same zeros).
    auto clear_tail = [&](int vr) -> bool {
      const uint32_t seq = 2 * (tile - 1) + 1, sl = seq % L::kSlots;
      if (!wait_bar_warp(&bars[L::bFull + sl], (seq / L::kSlots) & 1, st)) return false;
      unsigned char* vt = sm + L::kRing + sl * L::kTile;
      const int units = (16 - (vr & 15)) * (DT / 8);
#pragma unroll 1
      for (int i = rl; i < units; i += kGroupThreads) {
        const int rr = vr + i / (DT / 8), c = i % (DT / 8);
        *reinterpret_cast<uint4*>(vt + (c >> 3) * (kT * 128) + rr * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
      }
      fence_proxy_async_smem();
      return true;
    };

    // One thin item of nrow <= NR rows, from its first descriptor to its partial state.  Thread = key:
    // its NR scores are one row of S^T, its probabilities NR columns of P^T; all threads of the group
    // carry the rows' reference, each its own part of the rows' sums.
    auto thin_item = [&](auto nr_, int nrow) -> bool {
      constexpr int NR = decltype(nr_)::value;
      float ref[NR], sum[NR];
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        ref[r] = -INFINITY;
        sum[r] = 0.f;
      }
      bool had_t = false;
      int flags, slot;
      do {
        const uint32_t ds = d % L::kDescs;
        if (!wait_bar_warp(&bars[L::bDFull + ds], (d / L::kDescs) & 1, st)) return false;
        const TileDesc& td = descs[ds];
        const int vr = td.vr;
        flags = td.flags;
        slot = td.slot;
        const uint32_t on = a.masked ? td.mask[my_page & (kMaxPpt - 1)][0] : ~0u;
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[L::bDEmpty + ds]);
        ++d;
        if (flags & F_EMPTY) break;
        ++tile;
        if ((int)(job++ & 1) != grp) continue;
        const uint32_t gm = rl < vr ? on & ((1u << nrow) - 1u) : 0u;  // rows that attend this key
        if (!wait_bar_warp(&bars[L::bSFull + grp], sc & 1, st)) return false;
        ++sc;
        tc_fence_after();
        float x[NR];
        tmem_ldn<NR>(lane_addr + col_s, x);
        tmem_wait_ld();
        // Scores in log2 units, -inf by selection where a row does not attend this key; each row's
        // maximum over the warp's keys against the shared reference.
        bool up = false;  // the same in all of a warp's lanes
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          x[r] = (gm >> r) & 1u ? x[r] * sc2 : -INFINITY;
          const float wm = redux_max(x[r]);
          up |= wm > ref[r] + kRescaleThreshold || (ref[r] == -INFINITY && wm != -INFINITY);
          if (lane == 0) s_max[quarter * kThin + r] = wm;
        }
        if (meet(up)) {
          // some row's reference moves, to its maximum over the tile's keys; the sums and O^T (a row is a
          // column of it; S(i) being complete implies that the lane's last product is) follow
          float f[NR];
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            f[r] = 1.f;
            const float mt = fmaxf(fmaxf(s_max[r], s_max[kThin + r]), fmaxf(s_max[2 * kThin + r], s_max[3 * kThin + r]));
            if (mt > ref[r] + kRescaleThreshold || (ref[r] == -INFINITY && mt != -INFINITY)) {
              f[r] = ref[r] == -INFINITY ? 0.f : fast_exp2(ref[r] - mt);
              sum[r] *= f[r];
              ref[r] = mt;
            }
          }
          meet(false);  // s_max is read
          if (had_t) {
            float o[NR];
            uint32_t u[NR];
            tmem_ldn<NR>(lane_addr + col_o, o);
            tmem_wait_ld();
#pragma unroll
            for (int r = 0; r < NR; ++r) u[r] = f[r] == 0.f ? 0u : __float_as_uint(o[r] * f[r]);
            tmem_stn<NR>(lane_addr + col_o, u);
            tmem_wait_st();
          }
        }
        // P^T: a row's 128 keys as two 128-byte swizzled rows of 64, in the unused part of a Q buffer.  A
        // reference of -inf (no attended score yet, or none that is a number) is taken as 0: masked
        // keys still get exp2(-inf) = 0, and an attended NaN reaches the sum and the result.
        unsigned char* pt = sm + L::kQ + grp * L::kTile + kThinP + (rl >> 6) * (kThin * 128) + (rl & 7) * 2;
        const int unit = (rl & 63) >> 3;
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          const float e = fast_exp2(x[r] - (ref[r] == -INFINITY ? 0.f : ref[r]));
          sum[r] += e;
          *reinterpret_cast<uint16_t*>(pt + r * 128 + ((unit ^ (r & 7)) << 4)) = (uint16_t)pack2(e, 0.f, BF16);
        }
        fence_proxy_async_smem();
        if (__builtin_expect(vr & 15, 0) && !clear_tail(vr)) return false;
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[L::bPFull + grp]);
        had_t = true;
      } while (!(flags & F_LAST));
      // ---- the item's partial state: each row's sum over the keys; O^T's lane d is column d of every row
      const bool own = flags & F_OWN;
      const int rows = own ? G : kT;
      const int64_t state = (int64_t)slot * 2 + grp;
      float2* ml = (own ? a.w.ml_o : a.w.ml_p) + state * rows;
      float* acc = reinterpret_cast<float*>((own ? a.w.acc_o : a.w.acc_p) + state * (S.D / 4) * rows);
      if (!had_t) {
        if (rl < nrow) ml[rl] = make_float2(-INFINITY, 0.f);
        return true;
      }
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        float l = sum[r];
#pragma unroll
        for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        if (lane == 0) s_max[quarter * kThin + r] = l;
      }
      if (!wait_bar_warp(&bars[L::bODone + grp], od & 1, st)) return false;
      ++od;
      tc_fence_after();
      float o[NR];
      tmem_ldn<NR>(lane_addr + col_o, o);
      tmem_wait_ld();
      tc_fence_before();
      meet(false);  // s_max is complete, O^T is read
      if (lane == 0) mbar_arrive(&bars[L::bOFree + grp]);
      float m = -INFINITY;
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        if (r < nrow && rl < S.D) acc[((int64_t)(rl >> 2) * rows + r) * 4 + (rl & 3)] = o[r];
        if (r == rl) m = ref[r];
      }
      if (rl < nrow) ml[rl] = make_float2(m, s_max[rl] + s_max[kThin + rl] + s_max[2 * kThin + rl] + s_max[3 * kThin + rl]);
      meet(false);  // s_max is read: the next tile may write it
      return true;
    };

    while (true) {
      const uint32_t ds = d % L::kDescs;
      if (!wait_bar_warp(&bars[L::bDFull + ds], (d / L::kDescs) & 1, st)) break;
      const TileDesc& td = descs[ds];
      const int flags = td.flags, vr = td.vr, n = td.n;
      if (flags & F_FIRST) slot = td.slot;
      if (flags & F_END) break;
      if (flags & F_THIN) {  // a whole item; its first descriptor is not released yet
        const int nrow = flags & F_OWN ? G : S.B * G;
        const bool ok = nrow <= 4   ? thin_item(std::integral_constant<int, 4>{}, nrow)
                        : nrow <= 8 ? thin_item(std::integral_constant<int, 8>{}, nrow)
                                    : thin_item(std::integral_constant<int, 16>{}, nrow);
        if (!ok) break;
        continue;
      }
      const bool pair = flags & F_PAIR, own = flags & F_OWN, empty = flags & F_EMPTY;
      if (flags & F_FIRST) {
        sub = pair ? ((int)(job & 1) ^ grp) : grp;
        m_used = -INFINITY;
        l_sum = 0.f;
        had = false;
        row_ok = own ? rl < G : rl < S.nb * G && td.b0 + (pair ? sub * S.nb : 0) + rl / G < S.B;
      }
      const bool mine = !empty && (pair || (int)(job & 1) == grp);
      // keys in groups of 8 that this row attends (pages are multiples of 8 rows)
      uint32_t gm = row_ok ? 0xffffu : 0u;
      if (mine && a.masked) {
        const int wd = (pair ? sub * 4 : 0) + quarter, g8 = S.bn / 8;
        gm = 0;
        for (int j = 0; j < n; ++j)
          if ((td.mask[j][wd] >> lane) & 1u) gm |= (g8 >= 16 ? 0xffffu : (1u << g8) - 1u) << (j * g8);
        if (!row_ok) gm = 0;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[L::bDEmpty + ds]);
      ++d;
      if (!empty) {
        job += pair ? 2 : 1;
        ++tile;
      }
      if (mine) {
        if (!wait_bar_warp(&bars[L::bSFull + grp], sc & 1, st)) break;
        ++sc;
        tc_fence_after();
        uint64_t ls = 0;
        float la = 1.f;  // the sum's rescale
        if (__any_sync(0xffffffffu, row_ok)) {
          bool done = false;
          if (vr == kT && !own) {
            // Full prefix tile, one pass: the reference stays what it is (0 in the row's first tile), and nothing
            // needs the maximum as long as the exponentials' sum tells that none overflowed and, in a
            // first tile, that the row's largest is not lost in the type's small numbers: within
            // [1, 2^13] the largest of 128 is at least 2^-7, and fp16 holds 2^13.  Any row outside (or a
            // NaN) sends the warp through the two-pass form below; P is kept in registers till then, as
            // it overwrites S.  (Own items are short and wait for memory: there the two-pass form, whose
            // loops are a third of this code, measured faster, 127 against 141 us at 256 requests of
            // up to 768 tokens; over the prefix one pass takes 1.6 k cycles a tile, two take 2.7 k.)
            const float ref = m_used == -INFINITY ? 0.f : m_used;
            const uint64_t scale_x2 = f32x2(sc2, sc2);
            uint64_t rs[2] = {0, 0};
            uint32_t pk[kT / 2];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              float x[2][32];
              tmem_ld32(lane_addr + col_s + half * 64, x[0]);
              tmem_ld32(lane_addr + col_s + half * 64 + 32, x[1]);
              tmem_wait_ld();
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const float bk = (gm >> (half * 8 + k)) & 1u ? -ref : -INFINITY;
                const uint64_t bias_x2 = f32x2(bk, bk);
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                  float e0, e1;
                  const float* y = &x[k >> 2][(k & 3) * 8 + i];
                  f32x2_split(fma_f32x2(f32x2(y[0], y[1]), scale_x2, bias_x2), e0, e1);
                  const float p0 = fast_exp2(e0), p1 = fast_exp2(e1);
                  rs[(i >> 1) & 1] = add_f32x2(rs[(i >> 1) & 1], f32x2(p0, p1));
                  pk[half * 32 + k * 4 + i / 2] = pack2(p0, p1, BF16);
                }
              }
              // the first half's columns end here: loaded any earlier, the second half's would push
              // the warp past its registers
#pragma unroll
              for (int i = 0; i < 32; i += 8)
                asm volatile("" ::"r"(pk[half * 32 + i]), "r"(pk[half * 32 + i + 1]), "r"(pk[half * 32 + i + 2]),
                             "r"(pk[half * 32 + i + 3]), "r"(pk[half * 32 + i + 4]), "r"(pk[half * 32 + i + 5]),
                             "r"(pk[half * 32 + i + 6]), "r"(pk[half * 32 + i + 7]));
            }
            ls = add_f32x2(rs[0], rs[1]);
            float r0, r1;
            f32x2_split(ls, r0, r1);
            const float sum = r0 + r1;
            done = __all_sync(0xffffffffu, gm == 0u || (sum <= 8192.f && (m_used != -INFINITY || sum >= 1.f)));
            if (done) {
#pragma unroll
              for (int c = 0; c < kT / 32; ++c) tmem_st16(lane_addr + col_s + c * 16, pk + c * 16);
              if (gm != 0u) m_used = ref;
            }
          }
          if (__builtin_expect(!done, 0)) {
            const int nch = (vr + 31) >> 5;  // 32-key chunks with valid keys
            if (vr & 31) {
              // the last chunk's columns past the valid keys hold whatever was there: -inf in place
              float x[32];
              tmem_ld32(lane_addr + col_s + (nch - 1) * 32, x);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) x[i] = i < (vr & 31) ? x[i] : -INFINITY;
              tmem_st32(lane_addr + col_s + (nch - 1) * 32, x);
              tmem_wait_st();
            }
            // Row maximum, per group of 8 keys so that a masked group falls away by selection.
            float mraw = -INFINITY;
#pragma unroll 1
            for (int c = 0; c < nch; c += 2) {
              float x[64];
              tmem_ld32(lane_addr + col_s + c * 32, reinterpret_cast<float(&)[32]>(x[0]));
              if (c + 1 < nch) tmem_ld32(lane_addr + col_s + c * 32 + 32, reinterpret_cast<float(&)[32]>(x[32]));
              tmem_wait_ld();
              const int nk = c + 1 < nch ? 8 : 4;
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const float* y = x + 8 * k;
                const float mg = fmax3(fmax3(y[0], y[1], y[2]), fmax3(y[3], y[4], y[5]), fmaxf(y[6], y[7]));
                if (k < nk) mraw = fmaxf(mraw, (gm >> (c * 4 + k)) & 1u ? mg : -INFINITY);
              }
            }
            const float mt = mraw * sc2;
            float m_new = m_used;
            if (mt > -INFINITY && (m_used == -INFINITY || mt > m_used + kRescaleThreshold)) m_new = mt;
            const float m_ref = m_new == -INFINITY ? 0.f : m_new;
            const float alpha = m_used == -INFINITY ? 1.f : fast_exp2(m_used - m_ref);
            const bool rescale = m_new != m_used && m_used != -INFINITY;
            const uint64_t scale_x2 = f32x2(sc2, sc2);
            uint64_t rs0 = 0, rs1 = 0;
            // Exponentials and P, 32 keys at a time from a second read of S: a loop this short stays in
            // the instruction cache beside the MMA warp's code, which the 128 unrolled columns of a
            // single read evict.  A masked group's bias is -inf.
            auto chunk = [&](const float(&x)[32], int c) {
              uint32_t pk[16];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const float bk = (gm >> (c * 4 + k)) & 1u ? -m_ref : -INFINITY;
                const uint64_t bias_x2 = f32x2(bk, bk);
#pragma unroll
                for (int i = k * 8; i < k * 8 + 8; i += 2) {
                  float e0, e1;
                  f32x2_split(fma_f32x2(f32x2(x[i], x[i + 1]), scale_x2, bias_x2), e0, e1);
                  const float p0 = fast_exp2(e0), p1 = fast_exp2(e1);
                  if (i & 2) rs1 = add_f32x2(rs1, f32x2(p0, p1));
                  else rs0 = add_f32x2(rs0, f32x2(p0, p1));
                  pk[i / 2] = pack2(p0, p1, BF16);
                }
              }
              tmem_st16(lane_addr + col_s + c * 16, pk);
            };
#pragma unroll 1
            for (int c = 0; c < nch; ++c) {
              float x[32];
              tmem_ld32(lane_addr + col_s + c * 32, x);
              tmem_wait_ld();
              chunk(x, c);
            }
            // S(i) being complete implies that the lane's last P V is: O[g] may be rescaled here
            if (had && __any_sync(0xffffffffu, rescale)) {
              const float f = rescale ? alpha : 1.f;
#pragma unroll 1
              for (int c = 0; c < DT / 32; ++c) {
                float o[32];
                tmem_ld32(lane_addr + col_o + c * 32, o);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] *= f;
                tmem_st32(lane_addr + col_o + c * 32, o);
              }
            }
            ls = add_f32x2(rs0, rs1);
            la = m_used == -INFINITY ? 0.f : alpha;
            m_used = m_new;
          }
          tmem_wait_st();
        }
        if (__builtin_expect(vr & 15, 0)) {
          if (!clear_tail(vr)) break;
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[L::bPFull + grp]);
        float r0, r1;
        f32x2_split(ls, r0, r1);
        l_sum = fmaf(l_sum, la, r0 + r1);
        had = true;
      }
      if (!(flags & F_LAST)) continue;
      // ---------------------------------------------------------------- the item's partial state
      const int rows = own ? G : kT;
      const int64_t state = (int64_t)slot * 2 + sub;
      float2* ml = (own ? a.w.ml_o : a.w.ml_p) + state * rows;
      float4* acc = (own ? a.w.acc_o : a.w.acc_p) + state * (S.D / 4) * rows;
      if (row_ok) ml[rl] = make_float2(had ? m_used : -INFINITY, l_sum);
      if (had) {
        if (!wait_bar_warp(&bars[L::bODone + grp], od & 1, st)) break;
        ++od;
        tc_fence_after();
        if (__any_sync(0xffffffffu, row_ok)) {
          const bool put = row_ok && (m_used != -INFINITY || l_sum != 0.f);
          float4* dst = acc + rl;
#pragma unroll 1
          for (int c = 0; c * 32 < S.D; ++c, dst += 8 * rows) {
            float o[32];
            tmem_ld32(lane_addr + col_o + c * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (put && c * 32 + 4 * i < S.D) dst[i * rows] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[L::bOFree + grp]);
      }
    }
    while (named_bar_count(1 + grp, kGroupThreads, lane == 0) != 4) {
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kVWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// ---------------------------------------------------------------------------------------
// join of the partial states, one CTA per (request, KV head)
// ---------------------------------------------------------------------------------------
constexpr int kCombThreads = 256;  // at most

// Row (b, h) by itself, one warp: for rows whose joined state is not finite.  In the tensor-core
// product a page's V meets every row of the tile, with weight 0 where the row does not attend
// it; 0 * inf or 0 * NaN would leave a NaN in rows that have nothing to do with the page, so
// such rows are computed again over their attended keys alone (columns d0..d1 of the output: those
// of the calling CTA).  Costs tokens x ~100 cycles: only
// non-finite values get here.
template <typename T>
__device__ __noinline__ void exact_row(const PrefixParams& p, int64_t b, int64_t h, float scale2, int d0, int d1) {
  const int lane = threadIdx.x & 31;
  const int64_t g = h / p.G, ptok = prefix_tokens(p), otok = own_tokens(p, b);
  const int64_t pp = (ptok + p.page - 1) / p.page, n = pp + (otok + p.page - 1) / p.page;
  const T* q = static_cast<const T*>(p.q) + b * p.qs[0] + h * p.qs[1];
  float qv[4], acc[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) qv[i] = lane + 32 * i < p.D ? to_f32<T>(q[lane + 32 * i]) * scale2 : 0.f;
  for (int64_t pg = 0; pg < n; ++pg) {
    const int64_t phys = pg < pp ? p.ppages[pg] : p.bt[b * p.bts[0] + (pg - pp) * p.bts[1]];
    if (phys < 0 || phys >= p.num_pages || !page_attended<1>(p, b, h, pg, n, phys)) continue;
    const int64_t valid = min(p.page, pg < pp ? ptok - pg * p.page : otok - (pg - pp) * p.page);
    for (int64_t t = 0; t < valid; ++t) {
      const T* k = static_cast<const T*>(p.kc) + phys * p.ks[0] + g * p.ks[1] + t * p.ks[2];
      const T* v = static_cast<const T*>(p.vc) + phys * p.vs[0] + g * p.vs[1] + t * p.vs[2];
      float x = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (lane + 32 * i < p.D) x = fmaf(qv[i], to_f32<T>(k[lane + 32 * i]), x);
#pragma unroll
      for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
      const float mn = fmaxf(m, x), ref = mn == -INFINITY ? 0.f : mn;
      const float al = exp2f(m - ref), e = exp2f(x - ref);
      m = mn;
      l = l * al + e;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (lane + 32 * i < p.D) acc[i] = fmaf(e, to_f32<T>(v[lane + 32 * i]), acc[i] * al);
    }
  }
  T* o = static_cast<T*>(p.out) + b * p.os[0] + h * p.os[1];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 32 * i >= d0 && lane + 32 * i < d1) o[lane + 32 * i] = from_f32<T>(l == 0.f ? 0.f : acc[i] * (1.f / l));
  if (p.lse && lane == 0 && d0 == 0) p.lse[b * p.H + h] = l == 0.f ? -INFINITY : m * kLn2 + logf(l);
}

// CTA = (unit, some of its cells); a cell is one head's float4 of the output.  CG groups of threads
// share the states of the CTA's cells and are joined through shared memory.  A chain of three
// dependent round trips (plan, states, store): bound by latency, so all of a group's loads of a round
// are issued together and nothing is divided by more than CG here.
template <typename T>
__global__ void __launch_bounds__(kCombThreads) prefix_combine_kernel(const __grid_constant__ PrefixParams p,
                                                                      const Split s, const Ws w, float scale2,
                                                                      int cpb) {
  __shared__ float4 s_acc[kCombThreads];
  __shared__ float2 s_ml[kCombThreads];
  __shared__ unsigned s_bad[4];  // rows (of the group) to compute again
  const int G = s.G, D4 = s.D / 4, tid = threadIdx.x;
  const int b = blockIdx.x / s.Hkv, g = blockIdx.x - b * s.Hkv;
  const int CG = (int)blockDim.x / cpb;  // thread groups over the states
  const int cg = tid / cpb, ci = tid - cg * cpb;
  if (tid < 4) s_bad[tid] = 0;
  pdl_wait();
  const Pieces q = w.plan[blockIdx.x];
  const int total = q.n_p + q.n_o;
  const int cell0 = (int)blockIdx.y * cpb, cell = cell0 + ci, cells = G * D4;
  const bool live = cell < cells;
  const int c4 = live ? cell / G : 0, hh = live ? cell - c4 * G : 0;
  {
    float M = -INFINITY, Ls = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    // (m, l) and acc of state (ml, x) into (M, Ls) and acc
    auto fold = [&](const float2& ml, const float4& x) {
      if (ml.x == -INFINITY && ml.y == 0.f) return;  // nothing attended: its acc is not written
      const float mn = fmaxf(M, ml.x), ref = mn == -INFINITY ? 0.f : mn;
      const float so = fast_exp2(M - ref), sn = fast_exp2(ml.x - ref);
      acc.x = acc.x * so + x.x * sn;
      acc.y = acc.y * so + x.y * sn;
      acc.z = acc.z * so + x.z * sn;
      acc.w = acc.w * so + x.w * sn;
      Ls = Ls * so + ml.y * sn;
      M = mn;
    };
    constexpr int NU = 4;
#pragma unroll 1
    for (int k0 = cg; live && k0 < total; k0 += NU * CG) {
      float2 ml[NU];
      float4 x[NU];
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        const int k = k0 + u * CG;
        ml[u] = make_float2(-INFINITY, 0.f);
        if (k < total) {
          const bool pre = k < q.n_p;
          const int64_t state = pre ? q.first_p + k * q.stride_p : q.first_o + (k - q.n_p);
          const int rows = pre ? kT : G, row = pre ? q.r0 + hh : hh;
          ml[u] = __ldcg((pre ? w.ml_p : w.ml_o) + state * rows + row);
          x[u] = __ldcg((pre ? w.acc_p : w.acc_o) + (state * D4 + c4) * rows + row);
        }
      }
#pragma unroll
      for (int u = 0; u < NU; ++u) fold(ml[u], x[u]);
    }
    if (CG > 1) {
      s_acc[tid] = acc;
      s_ml[tid] = make_float2(M, Ls);
    }
    __syncthreads();
    if (cg == 0 && live) {
#pragma unroll 1
      for (int c = 1; c < CG; ++c) fold(s_ml[c * cpb + ci], s_acc[c * cpb + ci]);
      const float inv = Ls == 0.f ? 0.f : 1.f / Ls;
      // an infinite weight or a NaN anywhere makes this sum NaN or infinite
      if (!(fabsf(acc.x) + fabsf(acc.y) + fabsf(acc.z) + fabsf(acc.w) + fabsf(Ls) < INFINITY))
        atomicOr(&s_bad[hh >> 5], 1u << (hh & 31));
      T* o = static_cast<T*>(p.out) + b * p.os[0] + (int64_t)(g * G + hh) * p.os[1] + 4 * c4;
      o[0] = from_f32<T>(acc.x * inv);
      o[1] = from_f32<T>(acc.y * inv);
      o[2] = from_f32<T>(acc.z * inv);
      o[3] = from_f32<T>(acc.w * inv);
      if (p.lse && c4 == 0) p.lse[(int64_t)b * s.Hkv * G + g * G + hh] = Ls == 0.f ? -INFINITY : M * kLn2 + logf(Ls);
    }
  }
  __syncthreads();
  // (the CTA's cells of head r are the columns 4 c with cell0 <= c G + r < cell0 + cpb)
  for (int r = tid >> 5; r < G; r += (int)blockDim.x / 32)
    if ((s_bad[r >> 5] >> (r & 31)) & 1u)
      exact_row<T>(p, b, g * G + r, scale2, 4 * max(0, (cell0 - r + G - 1) / G),
                   4 * min(D4, max(0, (cell0 + cpb - r + G - 1) / G)));
}

template <int DT, bool BF16>
int launch_main(const Args& a, bool dependent, cudaStream_t stream) {
  auto kern = prefix_sm100_kernel<DT, BF16>;
  // setmaxnreg.inc waits until the registers it asks for are free: launch only when the
  // per-thread launch allocation is the one the split was sized against
  static const int regs = [] {
    cudaFuncAttributes fa{};
    if (cudaFuncGetAttributes(&fa, prefix_sm100_kernel<DT, BF16>) != cudaSuccess) return -1;
    return fa.numRegs;
  }();
  if (regs != kLaunchRegs)
    return fail(SA_ELAUNCH, "prefix decode: launch register count " + std::to_string(regs) +
                                " differs from the register split's " + std::to_string(kLaunchRegs));
  static bool opted[64] = {};  // per device; setting it again is harmless
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64 || !opted[dev]) {
    cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<DT>::kAlloc);
    if (dev >= 0 && dev < 64) opted[dev] = true;
  }
  if (dependent)
    return launch_dependent(kern, dim3(a.s.grid), dim3(kThreads), Layout<DT>::kAlloc, stream, "prefix_sm100_kernel", a);
  kern<<<a.s.grid, kThreads, Layout<DT>::kAlloc, stream>>>(a);
  return check_launch("prefix_sm100_kernel");
}

}  // namespace

bool prefix_fast_shape(int dtype, int64_t B, int64_t H, int64_t Hkv, int64_t D, int64_t page) {
  return (dtype == SA_BF16 || dtype == SA_F16) && D % 8 == 0 && D <= 128 && page % 8 == 0 && H / Hkv <= kT &&
         H <= 32 * kMaxHeadWords && B * Hkv <= (1 << 26) && page <= (1 << 20);
}

int64_t prefix_fast_workspace_bytes(int64_t B, int64_t H, int64_t Hkv, int64_t D, int64_t page, int64_t Lp, int64_t L) {
  return (int64_t)carve(nullptr, make_split(B, H / Hkv, Hkv, page, Lp, L, D), nullptr);
}

// Key tiles, weighted lengths of the line of work and tasks of the mask kernel are 32-bit numbers on the
// device.  The host knows the widths of the page lists, not the lengths: with every page in use, the
// tiles at their highest weights (make_line) have to stay below 2^31 and the tasks below 2^30 (a
// task index runs past the last by less than the grid).  Weighted tiles reach that at about
// 18 billion own tokens x KV heads over all requests: 256 requests of 8 heads, tables for 8.9
// million tokens each.
static bool counts_fit(const Split& s) {
  auto tiles = [&](int64_t pages) { return (double)((pages + s.ppt - 1) / s.ppt) * s.sub; };
  const double weight = tiles(s.Lp) * ((double)s.units[0] * (kCostPair + 2 * kCostItem) + (double)s.units[1] * (kCostOne + kCostItem)) +
                        tiles(s.L) * s.B * s.Hkv * (kCostOne + kCostItem);
  const double tasks = 4.0 * s.Hkv * s.row_tiles * prefix_chunks(s) + (double)s.B * own_chunks(s);
  return weight < 2147483648.0 && tasks < 1073741824.0;
}

bool prefix_fast_eligible(const PrefixParams& p, int dtype) {
  if (!prefix_fast_shape(dtype, p.B, p.H, p.Hkv, p.D, p.page)) return false;
  if (p.num_pages < 1 || p.num_pages > INT32_MAX) return false;
  if (!counts_fit(make_split(p.B, p.G, p.Hkv, p.page, p.Lp, p.L, p.D))) return false;
  if (reinterpret_cast<uintptr_t>(p.q) % 16 || reinterpret_cast<uintptr_t>(p.kc) % 16 ||
      reinterpret_cast<uintptr_t>(p.vc) % 16)
    return false;
  // tensor maps take strides of whole 16 bytes, and no broadcast dimensions
  const int64_t qn[2] = {p.B, p.H}, kn[3] = {p.num_pages, p.Hkv, p.page};
  auto loadable = [](int64_t stride, int64_t n) { return stride % 8 == 0 && (stride > 0 || n == 1); };
  for (int i = 0; i < 2; ++i)
    if (!loadable(p.qs[i], qn[i])) return false;
  for (int i = 0; i < 3; ++i)
    if (!loadable(p.ks[i], kn[i]) || !loadable(p.vs[i], kn[i])) return false;
  return true;
}

int launch_prefix_fast(const PrefixParams& p, int dtype, void* workspace, cudaStream_t stream) {
  Args a{};
  a.s = make_split(p.B, p.G, p.Hkv, p.page, p.Lp, p.L, p.D);
  carve(workspace, a.s, &a.w);
  a.ppages = p.ppages;
  a.bt = p.bt;
  a.bts0 = p.bts[0];
  a.bts1 = p.bts[1];
  a.ctx = p.ctx;
  a.plen_dev = p.plen_dev;
  a.plen = (int)p.plen;
  a.num_pages = (int)p.num_pages;
  a.status = p.status;
  a.scale2 = (1.0f / sqrtf((float)p.D)) * kLog2e;
  a.masked = p.r > 0;
  // query rows as (D, G, KV head, request): a box of nb requests is one row tile
  const int64_t qst[4] = {p.qs[0], p.G * p.qs[1], p.qs[1], 1};
  int rc = make_tmap_4d(&a.tm_q, p.q, dtype, p.B, p.Hkv, p.G, p.D, qst, 64, (uint32_t)p.G, (uint32_t)a.s.nb);
  if (!rc) rc = make_tmap_4d(&a.tm_q1, p.q, dtype, p.B, p.Hkv, p.G, p.D, qst, 64, (uint32_t)p.G);
  if (!rc) rc = make_tmap_4d(&a.tm_k, p.kc, dtype, p.num_pages, p.Hkv, p.page, p.D, p.ks, 64, (uint32_t)a.s.bn);
  if (!rc) rc = make_tmap_4d(&a.tm_v, p.vc, dtype, p.num_pages, p.Hkv, p.page, p.D, p.vs, 64, (uint32_t)a.s.bn);
  if (rc) return fail(SA_ELAUNCH, std::string("prefix decode tensor maps: ") + sa_last_error());
  if (a.masked) {
    MaskArgs ma{};
    ma.s = a.s;
    ma.w = a.w;
    ma.ppages = p.ppages;
    ma.bt = p.bt;
    ma.bts0 = p.bts[0];
    ma.bts1 = p.bts[1];
    ma.ctx = p.ctx;
    ma.plen_dev = p.plen_dev;
    ma.plen = (int)p.plen;
    ma.num_pages = (int)p.num_pages;
    ma.router = p.router;
    ma.qrouter = p.qrouter;
    for (int i = 0; i < 3; ++i) {
      ma.rs[i] = p.rs[i];
      ma.qrs[i] = p.qrs[i];
    }
    ma.q64 = p.qrouter_dtype == SA_I64;
    ma.r = (int)p.r;
    ma.local = (int)std::min<int64_t>(p.local_blocks, INT32_MAX / 2);
    ma.sink = p.sink;
    ma.H = (int)p.H;
    ma.prefix_tasks = (int)(p.Hkv * a.s.row_tiles * 4 * prefix_chunks(a.s));
    ma.tasks = ma.prefix_tasks + (int)(p.B * own_chunks(a.s));
    const int grid = std::max(1, std::min((ma.tasks + kMaskWarps - 1) / kMaskWarps, device_sm_count() * 8));
    if (p.router_dtype == SA_I64)
      prefix_mask_kernel<int64_t><<<grid, kMaskWarps * 32, 0, stream>>>(ma);
    else
      prefix_mask_kernel<int32_t><<<grid, kMaskWarps * 32, 0, stream>>>(ma);
    if ((rc = check_launch("prefix_mask_kernel"))) return rc;
  }
  const bool bf = dtype == SA_BF16;
  if (p.D <= 64)
    rc = bf ? launch_main<64, true>(a, a.masked, stream) : launch_main<64, false>(a, a.masked, stream);
  else
    rc = bf ? launch_main<128, true>(a, a.masked, stream) : launch_main<128, false>(a, a.masked, stream);
  if (rc) return rc;
  // Groups of threads per cell: enough to fill the GPU with threads, 16 at most; a batch with few
  // cells is one whose prefix is cut finely, with many states to join.
  const int64_t cells = p.G * p.D / 4, all = cells * p.B * p.Hkv, fill = (int64_t)device_sm_count() * 1024;
  int groups = 1;
  while (groups < 16 && all * groups * 2 <= fill) groups *= 2;
  const int cpb = (int)std::min<int64_t>(kCombThreads / groups, (cells + 31) / 32 * 32);
  const dim3 grid((unsigned)(p.B * p.Hkv), (unsigned)((cells + cpb - 1) / cpb)), block((unsigned)(cpb * groups));
  if (bf)
    return launch_dependent(prefix_combine_kernel<__nv_bfloat16>, grid, block, 0, stream, "prefix_combine_kernel", p, a.s,
                            a.w, a.scale2, cpb);
  return launch_dependent(prefix_combine_kernel<__half>, grid, block, 0, stream, "prefix_combine_kernel", p, a.s, a.w,
                          a.scale2, cpb);
}

}  // namespace sa
