// Attention over a bounded part of the paged cache, for sm_100a (B200): one new token per sequence, at position
// p = L - 1, sees the first `sinks` tokens and the last `window` tokens,
//   V(p) = { t <= p : t < sinks or t > p - window },   out = sum_V softmax(q.k * scale) v;
// and decode attention over the whole cache that also adds up, per cached token and KV head, the probability the token
// received from the query heads of its group. (The prompt-chunk form is an instance of the prefill kernel.)
//
// What bounds it: each visible K and V row is read once and used for 1 to 8 queries, far below the tensor cores' need,
// so the kernel is a stream over pages and everything is arranged for bytes in flight:
//  * The visible pages of all (sequence, KV head) items - sink pages, then window pages, as one list per item - are laid
//    end to end and cut into one equal share per CTA, one persistent CTA per SM; few items are cut into chunks with a CTA
//    each instead, and many small ones go to teams of warps whole. Eight warps walk a share page by page, each with its own ring of three 8 KiB stages (K tile and V tile
//    of a page in one TMA copy, 128-byte swizzled): 192 KB in flight per SM, more than latency x bandwidth asks for.
//    64 sequences with a window of 4096 and 16 sinks: 45.4 us, 5.7 TB/s. What is left around the stream is a chain of
//    ~6 us - lengths, table, first pages; fold, record, ticket, merge - which is all there is to a small call (300 tokens: 6.3 us).
//  * S^T = K.Q^T and O^T = V^T.P^T on mma.sync m16n8k16: 16 tokens of a page fill M, the group's queries fill N = 8.
//    The online softmax keeps FP32 maxima and sums; probabilities go to FP16 for P.V (off by half a step, at most 2^-11
//    relative like the output's own rounding, and by up to 2^-25 of a row's largest where that falls below FP16's normal range);
//    their sum is taken before that rounding. Against 64 bits the outputs are off by 2.6e-4 of their size, 2.1e-4 with P in 32 bits.
//  * An item cut by a share boundary leaves (o, m, l) records in the workspace; whoever of its contributors arrives last
//    folds them in CTA order, so the result does not depend on who that is. A contributor that finds all others already
//    there - usual at the end of a share, whose neighbour met the item first thing - reads them straight away.
#include <cuda.h>

#include <mutex>

#include "mma_ptx.cuh"
#include "tc_ptx.cuh"

namespace rl {
namespace wattn {

using namespace rl::mma;
using rl::tc::L2PolicyEvictFirst;
using rl::tc::MbarExpectTx;
using rl::tc::MbarInit;
using rl::tc::MbarWait;
using rl::tc::SmemAddr;

constexpr int kHeadDim = 128;
constexpr int kMaxGroup = 8;         // query heads per KV head: N of the products
constexpr int kMaxKvHeads = 8;       // element stride of the tensor copy that joins a page's K and V tile
constexpr int kMaxBlocks = 1 << 26;  // token positions stay inside 31 bits
constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kStages = 3;
constexpr int kPageBytes = kKvBlock * kHeadDim * 2;
constexpr int kStageBytes = 2 * kPageBytes;
constexpr int kMaxSeqsPerLaunch = 96;
static_assert(kWarps == kMaxGroup && kHeadDim == 4 * 32, "a fold gives each warp one query head and each lane four columns");
constexpr int kInlineOthers = 3;     // items over at most this many other CTAs are merged from registers
constexpr int kMergeBatch = 16;      // longer ones: records in flight per thread
constexpr int kMinPagesPerCta = kWarps;
constexpr int kMinChunk = 2 * kWarps;      // an item is not cut finer than this ...
constexpr int kWholeItem = 3 * kWarps;     // ... and not at all up to this: a ring holds three pages per warp, and handing over
                                           // costs 1 us (300 tokens take 1.1 us longer in two; 8000 tokens: 11.5 us in
                                           // chunks of 16 pages, 14.8 in chunks of 8, 11.6 in chunks of 32)
constexpr int kTeamPages = 32;            // pages of an item that one warp of a team may take: their tile indices sit one per lane
constexpr int kSegmentPages = 12;    // what a second item costs a CTA (fold and hand-over, 2-3 us), in pages
constexpr int kMaxCtas = 256;
constexpr int kNewestPageBit = 1 << 30;

// Shared memory, from a 1024-byte aligned base.
constexpr int kRingBytes = kWarps * kStages * kStageBytes;
constexpr int kOBufOff = kRingBytes;                                   // [warp][query][128], columns permuted
constexpr int kMlOff = kOBufOff + kWarps * kMaxGroup * kHeadDim * 4;   // m[query][warp], l[query][warp]
constexpr int kBarOff = kMlOff + 2 * kMaxGroup * kWarps * 4;
constexpr int kPrefixOff = kBarOff + kWarps * kStages * 8;
constexpr int kChunkOff = kPrefixOff + (kMaxSeqsPerLaunch + 4) * 4;
constexpr int kSkipOff = kChunkOff + (kMaxSeqsPerLaunch + 4) * 4;
constexpr int kSmemBytes = kSkipOff + kMaxSeqsPerLaunch * 4 + 1024;
static_assert(kSmemBytes <= 227 * 1024, "window attention shared memory exceeds the 227 KB per-CTA limit");

// Workspace: error flag and tickets, then two records per CTA, then (weights) the statistics and scores.
constexpr int kTicketOff = 16;                                        // in ints
constexpr size_t kMetaBytes = 2048;
static_assert((kTicketOff + kMaxCtas) * 4 <= kMetaBytes, "tickets outgrow their place");
constexpr int kRecordFloats = kMaxGroup * kHeadDim + 2 * kMaxGroup;   // o[8][128], m[8], l[8]
constexpr size_t kRecordBytes = static_cast<size_t>(kMaxCtas) * 2 * kRecordFloats * 4;

struct Params {
  half* out;
  int64_t out_stride;
  const half* q;
  int64_t q_stride;
  const int32_t* tables;
  const int32_t* seq_lens;
  int num_seqs;
  int max_blocks;
  int kv_heads;
  int group;
  float scale_log2e;
  int window;
  int sinks;
  int sink_pages;      // pages that hold the first `sinks` tokens
  int* meta;
  float* records;
  float2* stats;       // [sequence][query head]: maximum (log2 domain), 1 / sum
  float* scores;       // [sequence][KV head][page][query of the group][16], log2 domain
  float* weights;
  bool wide_out;       // out rows are 8-byte aligned
  bool run_ahead;      // the overlap option: lengths, tables and all but the newest pages may be read before the wait
  bool drop_first_copy;   // test hook: warp 0 of CTA 0 never requests its first page, so its wait must run out
  long long wait_cycles;  // limit of every mbarrier wait
};

// A page's K tile and V tile of one KV head, 8 KiB, in one copy into this CTA's shared memory (no multicast).
__device__ __forceinline__ void TmaLoadPage(uint32_t dst, const CUtensorMap* map, int tile, uint32_t bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint "
      "[%0], [%1, {%2, %2, %2, %3}], [%4], %5;" ::"r"(dst),
      "l"(map), "r"(0), "r"(tile), "r"(bar), "l"(policy)
      : "memory");
}
__device__ __forceinline__ int LoadAcquire(const int* p) {
  int v;
  asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}

// Flattened pages: sequence-major, then KV head, then the item's page list; the launcher keeps their number inside 31 bits.
// n pages in `parts` equal parts: the first n % parts have one more.
__device__ __forceinline__ int PartBegin(int part, int n, int parts) {
  const int each = n / parts;
  return part * each + min(part, n - each * parts);
}
__device__ __forceinline__ int PartOf(int page, int n, int parts) {   // the inverse; n >= parts
  const int each = n / parts, longer = n - each * parts, there = longer * (each + 1);
  return page < there ? page / (each + 1) : longer + (page - there) / each;
}
struct Cursor {
  int seq, head, entry, entries;   // entry of the item's page list, which has `entries`
};
__device__ __forceinline__ Cursor Locate(int t, const int* prefix, int num_seqs, int heads) {
  int lo = 0, hi = num_seqs - 1;
  while (lo < hi) {   // the first sequence whose pages end behind t
    const int mid = (lo + hi) >> 1;
    if (heads * prefix[mid + 1] <= t) lo = mid + 1; else hi = mid;
  }
  Cursor c;
  c.seq = lo;
  c.entries = prefix[lo + 1] - prefix[lo];
  const int rem = t - heads * prefix[lo];
  c.head = rem / c.entries;
  c.entry = rem - c.head * c.entries;
  return c;
}

// One page of an item: scores of its 16 tokens against the group's queries, online softmax, P.V. `st` is the stage that holds
// its K and V tile, t0 the position of its first token; w0 is the first token of the window.
struct PageOffsets {
  uint32_t k[4], v[4];   // ldmatrix offsets of this lane inside a stage; dims 64..127 of a tile sit kHiDims further
};
constexpr uint32_t kHiDims = 2048;
__device__ __forceinline__ PageOffsets MakePageOffsets(int lane) {
  // K rows as the A operand of S^T, V transposed as the A operand of O^T
  const int k_row = (lane & 7) + ((lane >> 3) & 1) * 8, k_sel = lane >> 4;
  const int v_row = (lane & 7) + (lane >> 4) * 8, v_sel = (lane >> 3) & 1;
  PageOffsets off;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    off.k[j] = k_row * 128 + (((2 * j + k_sel) ^ (k_row & 7)) << 4);
    off.v[j] = kPageBytes + v_row * 128 + (((2 * j + v_sel) ^ (v_row & 7)) << 4);
  }
  return off;
}
// Where a running maximum starts: finite, so that a visible score of -inf (a key that overflowed) has weight zero on a page that
// shows nothing else, and not the NaN of inf - inf.
constexpr float kLowest = -3.402823466e38f;
struct Running {
  float o[8][4];            // O^T: dims 16 i + g (+ 8) of queries 2 tig, 2 tig + 1
  float m0, m1, l0, l1;     // of the two queries; l is this lane's share of the sum
  __device__ __forceinline__ void Clear() {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    m0 = m1 = kLowest;
    l0 = l1 = 0.0f;
  }
};
template <bool kScores>
__device__ __forceinline__ void PageStep(const Params& p, uint32_t st, const PageOffsets& off, const uint32_t (&qb)[8][2], int t0,
                                         int len, int w0, float* scores, int lane, Running& r) {
  const int g = lane >> 2, tig = lane & 3;
  // token i of the page is visible if i < end and (i < sink or i >= win); all 16 are on a page in the middle
  const int end = len - t0, sink = p.sinks - t0, win = w0 - t0;
  const bool full = end >= kKvBlock && (sink >= kKvBlock || win <= 0);

  float s[4] = {0.0f, 0.0f, 0.0f, 0.0f}, s2[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t a[4], a2[4];
    Ldsm4(st + off.k[j], a);
    Ldsm4(st + off.k[j] + kHiDims, a2);
    Mma16816(s, a, qb[j][0], qb[j][1]);
    Mma16816(s2, a2, qb[j + 4][0], qb[j + 4][1]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) s[i] = (s[i] + s2[i]) * p.scale_log2e;
  if (kScores) {   // [query][token]: the eight lanes of a query fill whole sectors
    float* dst = scores + static_cast<int64_t>(t0) * p.group + 2 * tig * kKvBlock + g;
    if (2 * tig < p.group) {
      __stcg(dst, s[0]);
      __stcg(dst + 8, s[2]);
    }
    if (2 * tig + 1 < p.group) {
      __stcg(dst + kKvBlock, s[1]);
      __stcg(dst + kKvBlock + 8, s[3]);
    }
  }
  auto visible = [&](int i) { return i < end && (i < sink || i >= win); };
  if (!full) {
    if (!visible(g)) s[0] = s[1] = -INFINITY;
    if (!visible(g + 8)) s[2] = s[3] = -INFINITY;
  }
  float mx0 = fmaxf(s[0], s[2]), mx1 = fmaxf(s[1], s[3]);
  if (__any_sync(0xffffffffu, mx0 > r.m0 || mx1 > r.m1)) {
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) {
      mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, off));
      mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, off));
    }
    const float n0 = fmaxf(r.m0, mx0), n1 = fmaxf(r.m1, mx1);
    const float a0 = Exp2(r.m0 - n0), a1 = Exp2(r.m1 - n1);
    r.m0 = n0;
    r.m1 = n1;
    r.l0 *= a0;
    r.l1 *= a1;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      r.o[i][0] *= a0;
      r.o[i][1] *= a1;
      r.o[i][2] *= a0;
      r.o[i][3] *= a1;
    }
  }
  const float p0 = Exp2(s[0] - r.m0), p1 = Exp2(s[1] - r.m1);
  const float p2 = Exp2(s[2] - r.m0), p3 = Exp2(s[3] - r.m1);
  r.l0 += p0 + p2;
  r.l1 += p1 + p3;
  const uint32_t b0 = MovmT(PackHalf2(p0, p1)), b1 = MovmT(PackHalf2(p2, p3));
  if (full) {
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) {
      uint32_t a[4];
      Ldsm4T(st + off.v[mt & 3] + (mt >> 2) * kHiDims, a);
      Mma16816(r.o[mt], a, b0, b1);
    }
  } else {
    // V rows of invisible tokens may hold NaN, and 0 * NaN would poison the sums: cleared in registers.
    const uint32_t k01 = (visible(2 * tig) ? 0x0000FFFFu : 0u) | (visible(2 * tig + 1) ? 0xFFFF0000u : 0u);
    const uint32_t k23 = (visible(2 * tig + 8) ? 0x0000FFFFu : 0u) | (visible(2 * tig + 9) ? 0xFFFF0000u : 0u);
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) {
      uint32_t a[4];
      Ldsm4T(st + off.v[mt & 3] + (mt >> 2) * kHiDims, a);
      a[0] &= k01;
      a[1] &= k01;
      a[2] &= k23;
      a[3] &= k23;
      Mma16816(r.o[mt], a, b0, b1);
    }
  }
}
// The group's queries as the B operand of S^T: query g in column g, zeros past the group.
__device__ __forceinline__ void LoadQueries(const Params& p, int seq, int head, int lane, uint32_t (&qb)[8][2]) {
  const int g = lane >> 2, tig = lane & 3;
  const half* qrow = p.q + static_cast<int64_t>(seq) * p.q_stride + (static_cast<int64_t>(head) * p.group + g) * kHeadDim + 2 * tig;
#pragma unroll
  for (int kk = 0; kk < 8; ++kk) {
    qb[kk][0] = g < p.group ? __ldg(reinterpret_cast<const uint32_t*>(qrow + 16 * kk)) : 0u;
    qb[kk][1] = g < p.group ? __ldg(reinterpret_cast<const uint32_t*>(qrow + 16 * kk + 8)) : 0u;
  }
}
// A warp's running sums into its part of the fold's buffer: o[query][128] (columns permuted by the query pair: no bank is
// met twice), m and l of each query.
__device__ __forceinline__ void LeaveInBuffer(Running& r, float* obuf, float* mbuf, float* lbuf, int warp, int lane) {
  const int g = lane >> 2, tig = lane & 3;
#pragma unroll
  for (int off = 4; off < 32; off <<= 1) {
    r.l0 += __shfl_xor_sync(0xffffffffu, r.l0, off);
    r.l1 += __shfl_xor_sync(0xffffffffu, r.l1, off);
  }
  float* ob = obuf + (warp * kMaxGroup + 2 * tig) * kHeadDim;
#pragma unroll
  for (int mt = 0; mt < 8; ++mt) {
    const int c0 = (16 * mt + g) ^ (tig * 8), c1 = (16 * mt + g + 8) ^ (tig * 8);
    ob[c0] = r.o[mt][0];
    ob[kHeadDim + c0] = r.o[mt][1];
    ob[c1] = r.o[mt][2];
    ob[kHeadDim + c1] = r.o[mt][3];
  }
  if (g == 0) {
    mbuf[(2 * tig) * kWarps + warp] = r.m0;
    mbuf[(2 * tig + 1) * kWarps + warp] = r.m1;
    lbuf[(2 * tig) * kWarps + warp] = r.l0;
    lbuf[(2 * tig + 1) * kWarps + warp] = r.l1;
  }
}
// Columns 4 lane .. 4 lane + 3 of a finished row: divided by the sum, rounded once.
template <bool kScores>
__device__ __forceinline__ void WriteRow(const Params& p, int seq, int qh, int lane, const float4& a, float m, float l) {
  half* dst = p.out + static_cast<int64_t>(seq) * p.out_stride + static_cast<int64_t>(qh) * kHeadDim + 4 * lane;
  const half2 lo = __floats2half2_rn(a.x / l, a.y / l), hi = __floats2half2_rn(a.z / l, a.w / l);
  if (p.wide_out) {
    *reinterpret_cast<uint2*>(dst) = make_uint2(AsU32(lo), AsU32(hi));
  } else {
    dst[0] = __low2half(lo);
    dst[1] = __high2half(lo);
    dst[2] = __low2half(hi);
    dst[3] = __high2half(hi);
  }
  if (kScores && lane == 0) p.stats[static_cast<int64_t>(seq) * p.kv_heads * p.group + qh] = make_float2(m, 1.0f / l);
}

template <bool kScores>
__global__ void __launch_bounds__(kThreads, 1)
DecodeKernel(const Params p, const __grid_constant__ CUtensorMap tile_map) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  float* obuf = reinterpret_cast<float*>(smem + kOBufOff);
  float* mbuf = reinterpret_cast<float*>(smem + kMlOff);
  float* lbuf = mbuf + kMaxGroup * kWarps;
  int* prefix = reinterpret_cast<int*>(smem + kPrefixOff);
  int* chunk_prefix = reinterpret_cast<int*>(smem + kChunkOff);
  int* skip = reinterpret_cast<int*>(smem + kSkipOff);   // pages between a sequence's sinks and its window
  __shared__ int warp_total[kMaxSeqsPerLaunch / 32], warp_live[kMaxSeqsPerLaunch / 32], warp_most[kMaxSeqsPerLaunch / 32], warp_chunks[kMaxSeqsPerLaunch / 32];
  __shared__ bool merge_here, others_done;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int heads = p.kv_heads;
  if (!kScores) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid == kThreads - 1) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tile_map) : "memory");
    for (int b = 0; b < kStages * kWarps; ++b) MbarInit(SmemAddr(smem + kBarOff) + b * 8, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (!p.run_ahead) asm volatile("griddepcontrol.wait;" ::: "memory");
  // Page prefix over the sequences, one per thread; every CTA works out the same table.
  int my_pages = 0;
  auto scan_sequences = [&](int value, int* totals) {   // inclusive scan over the first kMaxSeqsPerLaunch threads
    int incl = value;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += v;
    }
    if (lane == 31 && tid < kMaxSeqsPerLaunch) totals[warp] = incl;
    __syncthreads();
    for (int w = 0; w < warp && w < kMaxSeqsPerLaunch / 32; ++w) incl += totals[w];
    return incl;
  };
  if (tid < p.num_seqs) {
    const int len = min(p.seq_lens[tid], p.max_blocks * kKvBlock);
    if (len > 0) {
      const int window_page = max(0, len - p.window) >> kKvBlockShift;
      const int gap = max(0, window_page - p.sink_pages);
      my_pages = ((len + kKvBlock - 1) >> kKvBlockShift) - gap;
      skip[tid] = gap;
    }
  }
  {
    const unsigned live = __ballot_sync(0xffffffffu, my_pages > 0);
    const int most = __reduce_max_sync(0xffffffffu, my_pages);
    if (lane == 0 && tid < kMaxSeqsPerLaunch) {
      warp_live[warp] = __popc(live);
      warp_most[warp] = most;
    }
    const int incl = scan_sequences(my_pages, warp_total);
    if (tid < kMaxSeqsPerLaunch) prefix[tid + 1] = incl;
    if (tid == 0) prefix[0] = chunk_prefix[0] = 0;
    __syncthreads();
  }
  const int total = heads * prefix[p.num_seqs];
  if (total == 0) {
    asm volatile("griddepcontrol.wait;" ::: "memory");   // this grid never completes ahead of the one before it
    return;
  }
  int items = 0, most_pages = 0;
  for (int w = 0; w < kMaxSeqsPerLaunch / 32; ++w) {
    items += heads * warp_live[w];
    most_pages = max(most_pages, warp_most[w]);
  }
  const int cta = blockIdx.x;
  // How the pages are cut: equal shares of the flattened list, whatever items they meet - or, where there are few items,
  // each item in equal chunks with a CTA each. The longest chunk is longer than a share (74 pages against 62 where 24 items
  // of 380 meet 148 CTAs), but no CTA meets a second item, whose fold and hand-over cost it as much as kSegmentPages pages.
  // (Both measured, shares and chunks: 7 sequences of 3-2500 tokens, 28 items, 21.3 and 10.8 us; 8 x 4096, 16 items, 21.2
  // and 14.4 us.)
  int longest = 0;
  bool chunked = false;
  if (items <= static_cast<int>(gridDim.x)) {
    const int spare = static_cast<int>(gridDim.x) - items;
    const int fit = spare > 0 ? (total - 1) / spare + 1 : most_pages;   // sum of ceil(pages / fit) <= total / fit + items <= the grid
    longest = max(min(fit, most_pages), kMinChunk);
    chunked = longest <= max(total / static_cast<int>(gridDim.x), kMinChunk) + kSegmentPages;
  }
  const uint32_t my_ring = SmemAddr(smem) + warp * (kStages * kStageBytes);
  const uint32_t my_bars = SmemAddr(smem + kBarOff) + warp * (kStages * 8);
  const uint64_t policy = L2PolicyEvictFirst();   // pages are read once per launch
  const PageOffsets off = MakePageOffsets(lane);
  bool failed = false;
  int fail_at = 0;
  auto request = [&](int k, int tile) {   // this warp's k-th page
    const int stage = k % kStages;
    if (lane == 0 && !(p.drop_first_copy && k == 0 && blockIdx.x == 0 && warp == 0)) {
      MbarExpectTx(my_bars + stage * 8, kStageBytes);
      TmaLoadPage(my_ring + stage * kStageBytes, &tile_map, tile & ~kNewestPageBit, my_bars + stage * 8, policy);
    }
  };

  // Many items, none of them long: a CTA takes one or several at a time, each with `team` of its warps from the first page to
  // the finished rows; no record is handed over, and no team waits for another. It must not load the CTAs too unevenly: the
  // fullest has `heaviest` pages, a share has total / grid and a fold per item that it meets.
  // (Both measured, teams and shares: 41 sequences x 8 KV heads of 7-85 tokens 6.8 and 24.4 us; 64 x 8 of 300-500 tokens 22.3
  // and 31.0; 80 x 2 with a window of 400 tokens 10.6 and 16.5; 64 x 2 of 1024-1280 tokens, a CTA each, 16.1 and 18.4.)
  const int rounds = (items + gridDim.x - 1) / gridDim.x, heaviest = rounds * most_pages;
  const int team = rounds <= 1 ? 8 : rounds <= 2 ? 4 : rounds <= 4 ? 2 : 1;
  if (!chunked && most_pages <= kTeamPages * team &&
      heaviest <= total / static_cast<int>(gridDim.x) + kSegmentPages * (2 + items / static_cast<int>(gridDim.x))) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (kScores) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // (see below)
    const int teams = kWarps / team, my_team = warp / team, member = warp - my_team * team;
    auto team_meets = [&]() {
      if (team == 1) __syncwarp(); else asm volatile("bar.sync %0, %1;" ::"r"(1 + my_team), "r"(32 * team) : "memory");
    };
    int used = 0, issued = 0;   // pages of this warp, through all its items
#pragma unroll 1
    for (int id = my_team * gridDim.x + cta; id < p.num_seqs * heads; id += teams * gridDim.x) {
      const int seq = id / heads, head = id - seq * heads, entries = prefix[seq + 1] - prefix[seq];
      if (entries == 0) continue;
      const int n = entries > member ? (entries - member + team - 1) / team : 0;   // this warp's: member, member + team, ...
      const int len = min(p.seq_lens[seq], p.max_blocks * kKvBlock), w0 = max(0, len - p.window), gap = skip[seq];
      auto page_of = [&](int i) {
        const int entry = member + team * i;
        return entry >= p.sink_pages ? entry + gap : entry;
      };
      int tile = 0;
      if (lane < n) tile = __ldg(p.tables + static_cast<int64_t>(seq) * p.max_blocks + page_of(lane)) * 2 * heads + head;
      const int base = used;
      auto request_up_to = [&](int end) {
        for (; issued < end && !failed; ++issued) request(issued, __shfl_sync(0xffffffffu, tile, issued - base));
      };
      request_up_to(base + min(n, kStages));
      uint32_t qb[8][2];
      LoadQueries(p, seq, head, lane, qb);
      float* scores = kScores ? p.scores + (static_cast<int64_t>(seq) * heads + head) * p.max_blocks * (kKvBlock * p.group) : nullptr;
      Running run;
      run.Clear();
#pragma unroll 1
      for (int i = 0; i < n && !failed; ++i) {
        const int stage = used % kStages;
        const bool arrived = MbarWait(my_bars + stage * 8, (used / kStages) & 1, p.wait_cycles);
        if (!__all_sync(0xffffffffu, arrived)) {
          failed = true;
          if (lane == 0) atomicExch(p.meta, 1);
          break;
        }
        PageStep<kScores>(p, my_ring + stage * kStageBytes, off, qb, page_of(i) * kKvBlock, len, w0, scores, lane, run);
        ++used;
        __syncwarp();   // every lane is done with the stage before it is refilled
        request_up_to(base + min(n, i + 1 + kStages));
      }
      LeaveInBuffer(run, obuf, mbuf, lbuf, warp, lane);
      team_meets();
      for (int q = member; q < p.group; q += team) {
        float mx = -INFINITY, den = 0.0f;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int w = warp - member; w < warp - member + team; ++w) mx = fmaxf(mx, mbuf[q * kWarps + w]);
        for (int w = warp - member; w < warp - member + team; ++w) {
          const float f = Exp2(mbuf[q * kWarps + w] - mx);   // 0 for a warp that had no page
          const float4 v = *reinterpret_cast<const float4*>(obuf + (w * kMaxGroup + q) * kHeadDim + ((4 * lane) ^ ((q >> 1) * 8)));
          acc.x = fmaf(f, v.x, acc.x);
          acc.y = fmaf(f, v.y, acc.y);
          acc.z = fmaf(f, v.z, acc.z);
          acc.w = fmaf(f, v.w, acc.w);
          den = fmaf(f, lbuf[q * kWarps + w], den);
        }
        WriteRow<kScores>(p, seq, head * p.group + q, lane, acc, mx, den);
      }
      team_meets();
    }
    if (failed) {   // copies in flight get one more bounded chance to land before the shared memory goes away
      for (int k = used; k < issued; ++k) MbarWait(my_bars + (k % kStages) * 8, (k / kStages) & 1, p.wait_cycles);
    }
    return;
  }

  int share_begin, share_end;
  int ctas, chunk_first = 0, chunk_last = 0;   // (chunked) the CTAs of this CTA's item
  if (chunked) {
    const int chunks = my_pages > kWholeItem ? (my_pages + longest - 1) / longest : my_pages > 0 ? 1 : 0;
    const int incl = scan_sequences(chunks, warp_chunks);
    if (tid < kMaxSeqsPerLaunch) chunk_prefix[tid + 1] = incl;
    __syncthreads();
    ctas = heads * chunk_prefix[p.num_seqs];   // <= total / longest + items <= gridDim.x
    const Cursor c = Locate(cta < ctas ? cta : 0, chunk_prefix, p.num_seqs, heads);   // entry = chunk, entries = chunks
    const int pages = prefix[c.seq + 1] - prefix[c.seq];
    const int item = heads * prefix[c.seq] + c.head * pages;
    share_begin = item + PartBegin(c.entry, pages, c.entries);
    share_end = item + PartBegin(c.entry + 1, pages, c.entries);
    chunk_first = cta - c.entry;
    chunk_last = chunk_first + c.entries - 1;
  } else {
    ctas = min(static_cast<int>(gridDim.x), max(1, total / kMinPagesPerCta));
    share_begin = PartBegin(cta, total, ctas);
    share_end = PartBegin(cta + 1, total, ctas);
  }
  if (cta >= ctas) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }

  // ---- this warp's pages: share-relative indices warp, warp + 8, ...
  const int share_len = share_end - share_begin;
  const int n_mine = share_len > warp ? (share_len - warp + kWarps - 1) / kWarps : 0;

  // Tile indices (4 KiB tiles of the pool; V lies `heads` tiles behind K) of 32 of this warp's pages at a time, one per
  // lane, read a batch ahead. A sequence's last page is marked: it holds the token that this step writes.
  auto fetch_tiles = [&](int batch) -> int {
    const int k = 32 * batch + lane;
    if (k >= n_mine) return 0;
    const Cursor c = Locate(share_begin + warp + kWarps * k, prefix, p.num_seqs, heads);
    const int page = c.entry >= p.sink_pages ? c.entry + skip[c.seq] : c.entry;
    const int block = __ldg(p.tables + static_cast<int64_t>(c.seq) * p.max_blocks + page);
    return (block * 2 * heads + c.head) | (c.entry == c.entries - 1 ? kNewestPageBit : 0);
  };
  int tiles_cur = fetch_tiles(0);
  int tiles_next = n_mine > 32 ? fetch_tiles(1) : 0;
  // Under the overlap option this grid may run ahead of the previous kernel's end: pages that an earlier step wrote
  // are requested at once, a sequence's newest page - and everything else - after the wait.
  const int first = n_mine < kStages ? n_mine : kStages;
#pragma unroll 1
  for (int i = 0; i < first; ++i) {
    const int tile = __shfl_sync(0xffffffffu, tiles_cur, i);
    if (!(tile & kNewestPageBit)) request(i, tile);
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // The kernel that adds the weights up reads the old ones ahead of its own wait: it may start only now that whatever
  // wrote them before this grid is done.
  if (kScores) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
#pragma unroll 1
  for (int i = 0; i < first; ++i) {
    const int tile = __shfl_sync(0xffffffffu, tiles_cur, i);
    if (tile & kNewestPageBit) request(i, tile);
  }
  int n_issue = first, n_use = 0;
  auto issue_one = [&]() {
    request(n_issue, __shfl_sync(0xffffffffu, tiles_cur, n_issue & 31));
    ++n_issue;
    if ((n_issue & 31) == 0) {
      tiles_cur = tiles_next;
      tiles_next = fetch_tiles((n_issue >> 5) + 1);
    }
  };
  // ---- one (sequence, KV head) segment of the share after the other
  int seg_begin = share_begin;
#pragma unroll 1
  while (seg_begin < share_end) {
    const Cursor sc = Locate(seg_begin, prefix, p.num_seqs, heads);
    const int item_begin = seg_begin - sc.entry, item_end = item_begin + sc.entries;
    const int seg_end = item_end < share_end ? item_end : share_end;
    const int len = min(p.seq_lens[sc.seq], p.max_blocks * kKvBlock);
    const int w0 = max(0, len - p.window);   // first token of the window
    const int gap = skip[sc.seq];
    const int seg_end_rel = seg_end - share_begin;
    const int entry0 = sc.entry - (seg_begin - share_begin);   // entry of the share's page `rel` is rel + entry0
    uint32_t qb[8][2];
    LoadQueries(p, sc.seq, sc.head, lane, qb);
    const bool whole = seg_begin == item_begin && seg_end == item_end;
    int c_first = cta, c_last = cta;
    if (chunked) {
      c_first = chunk_first;
      c_last = chunk_last;
    } else if (!whole) {
      if (item_begin < share_begin) c_first = PartOf(item_begin, total, ctas);
      if (item_end > share_end) c_last = PartOf(item_end - 1, total, ctas);
    }
    const int others = c_last - c_first;
    const bool may_read_inline = !whole && others <= kInlineOthers;
    int* ticket = p.meta + kTicketOff + c_first;
    float* seg_scores = kScores ? p.scores + (static_cast<int64_t>(sc.seq) * heads + sc.head) * p.max_blocks * (kKvBlock * p.group) : nullptr;
    int seen = -1;   // thread 0: how many of the others had published when it looked

    Running run;
    run.Clear();
#pragma unroll 1
    for (int rel = warp + kWarps * n_use; rel < seg_end_rel; rel += kWarps) {
      const int stage = n_use % kStages;
      const uint32_t st = my_ring + stage * kStageBytes;
      if (!failed) {   // (the whole warp goes on or none of it: a page's products and shuffles need all lanes)
        const bool arrived = MbarWait(my_bars + stage * 8, (n_use / kStages) & 1, p.wait_cycles);
        if (!__all_sync(0xffffffffu, arrived)) {
          failed = true;
          fail_at = n_use;
          if (lane == 0) atomicExch(p.meta, 1);
        }
      }
      if (may_read_inline && tid == 0 && seen < 0 && rel + 2 * kWarps >= seg_end_rel) seen = LoadAcquire(ticket);
      if (!failed) {
        const int entry = rel + entry0;
        const int page = entry >= p.sink_pages ? entry + gap : entry;
        PageStep<kScores>(p, st, off, qb, page * kKvBlock, len, w0, seg_scores, lane, run);
      }
      ++n_use;
      __syncwarp();   // every lane is done with the stage before it is refilled
      if (!failed && n_issue < n_mine) issue_one();
    }

    // ---- fold the warps' (o, m, l), then write the item or hand it on
    if (tid == 0) {
      if (may_read_inline && seen < 0) seen = LoadAcquire(ticket);   // warp 0 had fewer than two pages here
      others_done = may_read_inline && seen == others;
    }
    LeaveInBuffer(run, obuf, mbuf, lbuf, warp, lane);
    __syncthreads();
    // From here on warp h has query head h of the group, lane i its columns 4i .. 4i + 3.
    const bool has_head = warp < p.group;
    const int d = 4 * lane;
    // a contributor's record 0 is of an item that began before its share, record 1 of one that begins in it
    auto record = [&](int c) { return p.records + (static_cast<size_t>(c) * 2 + (c == c_first ? 1 : 0)) * kRecordFloats; };
    float om[kInlineOthers], ol[kInlineOthers];
    float4 oo[kInlineOthers];
    auto load_others = [&]() {   // the other contributors' records, in CTA order
#pragma unroll
      for (int j = 0; j < kInlineOthers; ++j) {
        if (j < others && has_head) {
          const float* r = record(c_first + j + (c_first + j >= cta ? 1 : 0));
          om[j] = __ldcg(r + kMaxGroup * kHeadDim + warp);
          ol[j] = __ldcg(r + kMaxGroup * kHeadDim + kMaxGroup + warp);
          oo[j] = __ldcg(reinterpret_cast<const float4*>(r + warp * kHeadDim + d));
        }
      }
    };
    const bool fast = !whole && others_done;
    if (fast) load_others();
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float mx = -INFINITY, den = 0.0f;
    auto add_part = [](float f, const float4& v, float l, float4& a, float& sum) {
      a.x = fmaf(f, v.x, a.x);
      a.y = fmaf(f, v.y, a.y);
      a.z = fmaf(f, v.z, a.z);
      a.w = fmaf(f, v.w, a.w);
      sum = fmaf(f, l, sum);
    };
    if (has_head) {
      float mw[kWarps];
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, mw[w] = mbuf[warp * kWarps + w]);
#pragma unroll
      for (int w = 0; w < kWarps; ++w)   // a factor of 0 for a warp that saw no page
        add_part(Exp2(mw[w] - mx), *reinterpret_cast<const float4*>(obuf + (w * kMaxGroup + warp) * kHeadDim + (d ^ ((warp >> 1) * 8))),
                 lbuf[warp * kWarps + w], acc, den);
    }
    auto write_item = [&](const float4& a, float m, float l) {
      if (has_head) WriteRow<kScores>(p, sc.seq, sc.head * p.group + warp, lane, a, m, l);
    };
    // Few contributors: from registers, in CTA order with one common maximum, whoever does it.
    auto merge_few = [&]() {
      float m = mx;
#pragma unroll
      for (int j = 0; j < kInlineOthers; ++j)
        if (j < others) m = fmaxf(m, om[j]);
      float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      float l = 0.0f;
#pragma unroll
      for (int j = 0; j <= kInlineOthers; ++j) {   // own record in its place among the others
        if (c_first + j == cta) add_part(Exp2(mx - m), acc, den, a, l);
        if (j < kInlineOthers && j < others) add_part(Exp2(om[j] - m), oo[j], ol[j], a, l);
      }
      write_item(a, m, l);
    };
    // Many: the factors of all records first (in the fold's buffer, which is free), then the records themselves,
    // kMergeBatch in flight - one L2 latency per batch on the path that the whole grid waits for.
    auto merge_many = [&]() {
      if (!has_head) return;
      float* factor = obuf + warp * kMaxCtas;
      float m = -INFINITY;
      for (int c = c_first + lane; c <= c_last; c += 32) {
        const float mc = __ldcg(record(c) + kMaxGroup * kHeadDim + warp);
        factor[c - c_first] = mc;
        m = fmaxf(m, mc);
      }
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
      float l = 0.0f;
      for (int c = c_first + lane; c <= c_last; c += 32) {
        const float f = Exp2(factor[c - c_first] - m);
        factor[c - c_first] = f;
        l = fmaf(f, __ldcg(record(c) + kMaxGroup * kHeadDim + kMaxGroup + warp), l);
      }
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
      __syncwarp();
      float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
      for (int c0 = c_first; c0 <= c_last; c0 += kMergeBatch) {
        float4 v[kMergeBatch];
#pragma unroll
        for (int j = 0; j < kMergeBatch; ++j)
          if (c0 + j <= c_last) v[j] = __ldcg(reinterpret_cast<const float4*>(record(c0 + j) + warp * kHeadDim + d));
        float unused = 0.0f;
#pragma unroll
        for (int j = 0; j < kMergeBatch; ++j)
          if (c0 + j <= c_last) add_part(factor[c0 + j - c_first], v[j], 0.0f, a, unused);
      }
      write_item(a, m, l);
    };
    if (whole) {
      write_item(acc, mx, den);
    } else if (fast) {
      merge_few();
      if (tid == 0) *ticket = 0;   // everyone had arrived: ready for the next launch
    } else {
      float* rec = p.records + (static_cast<size_t>(cta) * 2 + (item_begin < share_begin ? 0 : 1)) * kRecordFloats;
      if (has_head) {
        *reinterpret_cast<float4*>(rec + warp * kHeadDim + d) = acc;
        if (lane == 0) {
          rec[kMaxGroup * kHeadDim + warp] = mx;
          rec[kMaxGroup * kHeadDim + kMaxGroup + warp] = den;
        }
      }
      __syncthreads();
      if (tid == 0) {
        __threadfence();   // the CTA's record, ordered before its ticket
        merge_here = atomicAdd(ticket, 1) == others;
        if (merge_here) *ticket = 0;
      }
      __syncthreads();
      if (merge_here) {
        __threadfence();
        if (others <= kInlineOthers) {
          load_others();
          merge_few();
        } else {
          merge_many();
        }
      }
    }
    __syncthreads();   // obuf and the flags are free for the next segment
    seg_begin = seg_end;
  }
  if (failed) {   // copies in flight get one more bounded chance to land before the shared memory goes away
    for (int k = fail_at; k < n_issue; ++k) MbarWait(my_bars + (k % kStages) * 8, (k / kStages) & 1, p.wait_cycles);
  }
}

// Second kernel of the weights launcher: per cached token and KV head, the sum over the group of
// exp2(score - maximum) / sum, added to the token's weight. One thread per token, 16 neighbours to a page: scores of a
// query, and weights, are read and written in whole lines. What the kernel before it does not write - lengths, table,
// old weights - is read ahead of the wait for it.
constexpr int kAccumulateThreads = 256;
constexpr int kTokensPerThread = 2;   // in flight together: the kernel is a chain of loads, not a stream
constexpr int kAccumulateTokens = kAccumulateThreads * kTokensPerThread;
__global__ void __launch_bounds__(kAccumulateThreads) AccumulateKernel(const Params p, int parts) {
  const int part = blockIdx.x % parts, head = blockIdx.y;
  const int64_t seq = blockIdx.x / parts;
  const int len = min(p.seq_lens[seq], p.max_blocks * kKvBlock);
  const int32_t* table = p.tables + seq * p.max_blocks;
  const float2* st = p.stats + (seq * p.kv_heads + head) * p.group;
  const float* scores = p.scores + (seq * p.kv_heads + head) * p.max_blocks * (kKvBlock * p.group);
  bool waited = false;
  float2 ml[kMaxGroup];
#pragma unroll 1
  for (int64_t t0 = part * kAccumulateTokens; t0 < len; t0 += static_cast<int64_t>(parts) * kAccumulateTokens) {
    float* w[kTokensPerThread];
    float old[kTokensPerThread];
#pragma unroll
    for (int k = 0; k < kTokensPerThread; ++k) {
      const int64_t t = t0 + k * kAccumulateThreads + threadIdx.x;
      w[k] = t < len ? p.weights + (static_cast<int64_t>(table[t >> kKvBlockShift]) * p.kv_heads + head) * kKvBlock + (t & (kKvBlock - 1)) : nullptr;
    }
#pragma unroll
    for (int k = 0; k < kTokensPerThread; ++k)
      old[k] = w[k] && t0 + k * kAccumulateThreads + threadIdx.x != len - 1 ? *w[k] : 0.0f;
    if (!waited) {
      asm volatile("griddepcontrol.wait;" ::: "memory");
      waited = true;
#pragma unroll
      for (int q = 0; q < kMaxGroup; ++q) ml[q] = q < p.group ? __ldcg(st + q) : make_float2(0.0f, 0.0f);
    }
    float x[kTokensPerThread][kMaxGroup];
#pragma unroll
    for (int k = 0; k < kTokensPerThread; ++k) {
      const int64_t t = t0 + k * kAccumulateThreads + threadIdx.x;
      const float* s = scores + (t >> kKvBlockShift) * (kKvBlock * p.group) + (t & (kKvBlock - 1));
#pragma unroll
      for (int q = 0; q < kMaxGroup; ++q) x[k][q] = w[k] && q < p.group ? __ldcg(s + q * kKvBlock) : 0.0f;
    }
#pragma unroll
    for (int k = 0; k < kTokensPerThread; ++k) {
      float sum = 0.0f;
#pragma unroll
      for (int q = 0; q < kMaxGroup; ++q)
        if (q < p.group) sum = fmaf(Exp2(x[k][q] - ml[q].x), ml[q].y, sum);
      if (w[k]) *w[k] = old[k] + sum;
    }
  }
  if (!waited) asm volatile("griddepcontrol.wait;" ::: "memory");
}

// ----------------------------------------------------------- host side

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
constexpr int kMaxDevices = 64;
bool g_ready[kMaxDevices];
EncodeTiledFn g_encode = nullptr;
std::mutex g_mutex;

// First use on a device: driver entry point and shared-memory opt-in.
int EnsureReady(const char* fn) {
  bool& ready = g_ready[CurrentDeviceIndex()];
  std::lock_guard<std::mutex> lock(g_mutex);
  if (ready) return RL_OK;
  if (!g_encode) {
    void* entry = nullptr;
    cudaDriverEntryPointQueryResult qres;
    const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &entry, cudaEnableDefault, &qres);
    if (e != cudaSuccess || qres != cudaDriverEntryPointSuccess || !entry)
      return Fail(e != cudaSuccess ? static_cast<int>(e) : RL_E_WORKSPACE, "%s: cuTensorMapEncodeTiled is not available from this driver", fn);
    g_encode = reinterpret_cast<EncodeTiledFn>(entry);
  }
  if (CurrentDeviceFacts().max_smem_optin < kSmemBytes)
    return Fail(RL_E_WORKSPACE, "%s: device offers %d B of shared memory per block, %d needed", fn,
                CurrentDeviceFacts().max_smem_optin, kSmemBytes);
  cudaError_t e = cudaFuncSetAttribute(DecodeKernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(DecodeKernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
  if (e != cudaSuccess) return Fail(static_cast<int>(e), "%s: shared-memory opt-in: %s", fn, cudaGetErrorString(e));
  ready = true;
  return RL_OK;
}

// The pool slice as [tile][dim half][token][64 halves]; a box of kv_heads + 1 tiles at element stride kv_heads is the K
// tile and the V tile of a head. The view claims more tiles than a device holds; only tiles of real pages are requested.
int EncodeTileMap(const char* fn, const void* pool, int heads, CUtensorMap* map) {
  const cuuint64_t dims[4] = {64, static_cast<cuuint64_t>(kKvBlock), 2, 1ull << 26};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(kHeadDim) * 2, 128, static_cast<cuuint64_t>(kPageBytes)};
  const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(kKvBlock), 2, static_cast<cuuint32_t>(heads + 1)};
  const cuuint32_t estr[4] = {1, 1, 1, static_cast<cuuint32_t>(heads)};
  const CUresult r = g_encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(pool), dims, strides, box, estr,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return Fail(RL_E_BAD_SHAPE, "%s: tile map encode failed (CUresult %d)", fn, static_cast<int>(r));
  return RL_OK;
}

bool ShapeOk(int max_blocks, int q_heads, int kv_heads) {
  return max_blocks >= 1 && max_blocks <= kMaxBlocks && kv_heads >= 1 && kv_heads <= kMaxKvHeads && q_heads >= kv_heads &&
         q_heads % kv_heads == 0 && q_heads / kv_heads <= kMaxGroup;
}
size_t StatsBytes(int64_t num_seqs, int q_heads) { return (static_cast<size_t>(num_seqs) * q_heads * sizeof(float2) + 255) & ~static_cast<size_t>(255); }
size_t Workspace(int64_t num_seqs, int max_blocks, int q_heads, int kv_heads, bool weights) {
  size_t bytes = kMetaBytes + kRecordBytes;
  if (weights)
    bytes += StatsBytes(num_seqs, q_heads) + static_cast<size_t>(num_seqs) * q_heads * max_blocks * kKvBlock * sizeof(float);
  return bytes;
}

struct Call {
  const char* fn;
  void* out;
  int64_t out_row_stride;
  const void* q;
  int64_t q_row_stride;
  const void* pool;
  const int32_t* tables;
  const int32_t* seq_lens;
  int num_seqs, max_blocks, q_heads, kv_heads, head_dim;
  float scale;
  int window, sinks;
  float* weights;
  void* workspace;
  size_t workspace_bytes;
  cudaStream_t stream;
};

// Pages that a row can see at most.
int64_t LongestList(const Call& c) {
  const int64_t list = (static_cast<int64_t>(c.sinks) + kKvBlock - 1) / kKvBlock + (static_cast<int64_t>(c.window) + kKvBlock - 2) / kKvBlock + 1;
  return list < c.max_blocks ? list : c.max_blocks;
}

int Check(const Call& c, bool with_weights) {
  if (!c.out || !c.q || !c.pool || !c.tables || !c.seq_lens || !c.workspace || (with_weights && !c.weights))
    return Fail(RL_E_NULL_POINTER, "%s: null device pointer", c.fn);
  if (c.head_dim != kHeadDim) return Fail(RL_E_BAD_SHAPE, "%s: head_dim must be 128", c.fn);
  if (c.max_blocks > kMaxBlocks) return Fail(RL_E_TOO_LARGE, "%s: at most 2^26 blocks per sequence", c.fn);
  if (!ShapeOk(c.max_blocks, c.q_heads, c.kv_heads))
    return Fail(RL_E_BAD_SHAPE, "%s: 1 to 8 KV heads with 1 to 8 query heads each, max_blocks_per_seq >= 1", c.fn);
  const int64_t width = static_cast<int64_t>(c.q_heads) * c.head_dim;
  if (c.q_row_stride < width || c.out_row_stride < width) return Fail(RL_E_BAD_SHAPE, "%s: row stride smaller than the row", c.fn);
  if (!(c.scale > 0.0f) || !(c.scale * 1.4426950408889634f <= 3.402823466e38f))
    return Fail(RL_E_BAD_SHAPE, "%s: scale must be positive and finite", c.fn);
  if (c.window < 1 || c.sinks < 0) return Fail(RL_E_BAD_SHAPE, "%s: window >= 1 and sinks >= 0", c.fn);
  const int64_t rows = c.num_seqs < kMaxSeqsPerLaunch ? c.num_seqs : kMaxSeqsPerLaunch;
  if (LongestList(c) * rows * c.kv_heads > INT32_MAX - 65536)
    return Fail(RL_E_TOO_LARGE, "%s: more than 2^31 pages (times KV heads) in one launch", c.fn);
  if (!Aligned16(c.pool)) return Fail(RL_E_BAD_SHAPE, "%s: the pool slice must be 16-byte aligned", c.fn);
  if ((c.q_row_stride & 1) || (reinterpret_cast<uintptr_t>(c.q) & 3)) return Fail(RL_E_BAD_SHAPE, "%s: q rows must be 4-byte aligned", c.fn);
  if ((reinterpret_cast<uintptr_t>(c.out) & 1) || (reinterpret_cast<uintptr_t>(c.weights) & 3) || !Aligned16(c.workspace))
    return Fail(RL_E_BAD_SHAPE, "%s: out 2-byte, weights 4-byte, workspace 16-byte aligned", c.fn);
  const size_t need = Workspace(c.num_seqs, c.max_blocks, c.q_heads, c.kv_heads, with_weights);
  if (c.workspace_bytes < need) return Fail(RL_E_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", c.fn, c.workspace_bytes, need);
  return RL_OK;
}

template <bool kScores>
int Launch(const Call& c) {
  int rc = Check(c, kScores);
  if (rc != RL_OK) return rc;
  if ((rc = EnsureReady(c.fn)) != RL_OK) return rc;
  CUtensorMap tile_map;
  if ((rc = EncodeTileMap(c.fn, c.pool, c.kv_heads, &tile_map)) != RL_OK) return rc;
  Params p = {};
  p.q_stride = c.q_row_stride;
  p.out_stride = c.out_row_stride;
  p.max_blocks = c.max_blocks;
  p.kv_heads = c.kv_heads;
  p.group = c.q_heads / c.kv_heads;
  p.scale_log2e = c.scale * 1.4426950408889634f;
  // cut at the longest sequence: nothing changes, and sums of positions with them stay inside 32 bits
  const int longest = c.max_blocks * kKvBlock;
  p.window = c.window < longest ? c.window : longest;
  p.sinks = c.sinks < longest ? c.sinks : longest;
  p.sink_pages = (p.sinks + kKvBlock - 1) >> kKvBlockShift;
  char* ws = static_cast<char*>(c.workspace);
  p.meta = reinterpret_cast<int*>(ws);
  p.records = reinterpret_cast<float*>(ws + kMetaBytes);
  float2* stats = reinterpret_cast<float2*>(ws + kMetaBytes + kRecordBytes);
  float* scores = reinterpret_cast<float*>(ws + kMetaBytes + kRecordBytes + StatsBytes(c.num_seqs, c.q_heads));
  p.run_ahead = g_launch_overlap;
  p.drop_first_copy = g_drop_first_copy;
  p.wait_cycles = g_wait_cycles;
  p.wide_out = (reinterpret_cast<uintptr_t>(c.out) & 7) == 0 && (c.out_row_stride & 3) == 0;
  const int64_t pages = LongestList(c);   // no more CTAs than shares of kMinPagesPerCta pages can exist
  const int sms = CurrentDeviceFacts().sm_count < kMaxCtas ? CurrentDeviceFacts().sm_count : kMaxCtas;
  const int64_t row = static_cast<int64_t>(c.q_heads) * c.max_blocks * kKvBlock;
  for (int first = 0; first < c.num_seqs; first += kMaxSeqsPerLaunch) {
    const int n = c.num_seqs - first < kMaxSeqsPerLaunch ? c.num_seqs - first : kMaxSeqsPerLaunch;
    p.out = static_cast<half*>(c.out) + first * c.out_row_stride;
    p.q = static_cast<const half*>(c.q) + first * c.q_row_stride;
    p.tables = c.tables + static_cast<int64_t>(first) * c.max_blocks;
    p.seq_lens = c.seq_lens + first;
    p.num_seqs = n;
    p.stats = stats + static_cast<int64_t>(first) * c.q_heads;
    p.scores = scores + first * row;
    const int64_t shares = static_cast<int64_t>(n) * c.kv_heads * ((pages + kMinPagesPerCta - 1) / kMinPagesPerCta);
    const int grid = static_cast<int>(shares < 1 ? 1 : shares < sms ? shares : sms);
    const cudaError_t e = LaunchDependent(DecodeKernel<kScores>, dim3(grid), dim3(kThreads), kSmemBytes, 1, c.stream, p, tile_map);
    if (e != cudaSuccess) return Fail(static_cast<int>(e), "%s: %s", c.fn, cudaGetErrorString(e));
  }
  if (kScores) {
    p.tables = c.tables;
    p.seq_lens = c.seq_lens;
    p.stats = stats;
    p.scores = scores;
    p.weights = c.weights;
    // enough CTAs per item for its longest possible cache, but no more in all than fill the machine
    const int64_t most = (static_cast<int64_t>(c.max_blocks) * kKvBlock + kAccumulateTokens - 1) / kAccumulateTokens;
    const int64_t items = static_cast<int64_t>(c.num_seqs) * c.kv_heads;
    const int64_t fair = (8LL * sms + items - 1) / items;
    const int parts = static_cast<int>(most < fair ? most : fair);
    const cudaError_t e = LaunchDependent(AccumulateKernel, dim3(static_cast<unsigned>(c.num_seqs) * parts, c.kv_heads),
                                          dim3(kAccumulateThreads), 0, 1, c.stream, p, parts);
    if (e != cudaSuccess) return Fail(static_cast<int>(e), "%s (weights): %s", c.fn, cudaGetErrorString(e));
  }
  return LaunchStatus(c.fn);
}

}  // namespace wattn
int WindowAttentionInit() { return wattn::EnsureReady("window attention"); }
}  // namespace rl

extern "C" int rl_window_attention_workspace_bytes(int32_t num_seqs, int32_t max_blocks_per_seq, int32_t num_q_heads,
                                                   int32_t num_kv_heads, int32_t weights, size_t* bytes_out) {
  using namespace rl;
  using namespace rl::wattn;
  if (!bytes_out) return Fail(RL_E_NULL_POINTER, "window_attention_workspace_bytes: null pointer");
  *bytes_out = 0;
  if (num_seqs < 0 || !ShapeOk(max_blocks_per_seq, num_q_heads, num_kv_heads))
    return Fail(RL_E_BAD_SHAPE, "window_attention_workspace_bytes: not a shape the launchers take");
  *bytes_out = Workspace(num_seqs, max_blocks_per_seq, num_q_heads, num_kv_heads, weights != 0);
  return RL_OK;
}

extern "C" int rl_window_attention_health(void* workspace, int* flag_out) {
  using namespace rl;
  if (!workspace || !flag_out) return Fail(RL_E_NULL_POINTER, "rl_window_attention_health: null pointer");
  *flag_out = 0;
  cudaError_t e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = cudaMemcpy(flag_out, workspace, sizeof(int), cudaMemcpyDeviceToHost);
  if (e == cudaSuccess && *flag_out != 0) e = cudaMemset(workspace, 0, sizeof(int));
  if (e != cudaSuccess) return Fail(static_cast<int>(e), "rl_window_attention_health: %s", cudaGetErrorString(e));
  return RL_OK;
}

extern "C" int rl_launch_paged_window_attention_decode(void* out, int64_t out_row_stride, const void* q,
                                                       int64_t q_row_stride, const void* kv_pool_layer,
                                                       const int32_t* block_tables, const int32_t* seq_lens,
                                                       int32_t num_seqs, int32_t max_blocks_per_seq,
                                                       int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                                                       float scale, int32_t window, int32_t sinks, void* workspace,
                                                       size_t workspace_bytes, void* stream) {
  if (num_seqs <= 0) return RL_OK;
  return rl::wattn::Launch<false>({"paged_window_attention_decode", out, out_row_stride, q, q_row_stride, kv_pool_layer,
                                   block_tables, seq_lens, num_seqs, max_blocks_per_seq, num_q_heads, num_kv_heads, head_dim,
                                   scale, window, sinks, nullptr, workspace, workspace_bytes, static_cast<cudaStream_t>(stream)});
}

extern "C" int rl_launch_paged_attention_decode_weights(void* out, int64_t out_row_stride, const void* q,
                                                        int64_t q_row_stride, const void* kv_pool_layer,
                                                        const int32_t* block_tables, const int32_t* seq_lens,
                                                        int32_t num_seqs, int32_t max_blocks_per_seq,
                                                        int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                                                        float scale, float* weights, void* workspace,
                                                        size_t workspace_bytes, void* stream) {
  if (num_seqs <= 0) return RL_OK;
  return rl::wattn::Launch<true>({"paged_attention_decode_weights", out, out_row_stride, q, q_row_stride, kv_pool_layer,
                                  block_tables, seq_lens, num_seqs, max_blocks_per_seq, num_q_heads, num_kv_heads, head_dim,
                                  scale, INT32_MAX, 0, weights, workspace, workspace_bytes, static_cast<cudaStream_t>(stream)});
}
