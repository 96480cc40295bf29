// Attention over a bounded part of the paged cache, for sm_100a (B200): one new token per sequence, at position
// p = L - 1, sees the first `sinks` tokens and the last `window` tokens,
//   V(p) = { t <= p : t < sinks or t > p - window },   out = sum_V softmax(q.k * scale) v;
// and decode attention over the whole cache that also adds up, per cached token and KV head, the probability the token
// received from the query heads of its group. (The prompt-chunk form is an instance of the prefill kernel.)
//
// What bounds it: each visible K and V row is read once and used for 1 to 8 queries, far below the tensor cores' need,
// so the kernel is a stream over pages and everything is arranged for bytes in flight:
//  * The visible pages of all (sequence, KV head) items - sink pages, then window pages, as one list per item - are laid
//    end to end and cut into one equal share per CTA, one persistent CTA per SM (fewer when there are fewer than eight
//    pages for each: a page per warp is the finest useful cut). Eight warps walk a share page by page, each with its own
//    ring of three 8 KiB stages (K tile and V tile of a page in one TMA copy, 128-byte swizzled): 192 KB in flight
//    per SM, more than latency x bandwidth asks for.
//  * S^T = K.Q^T and O^T = V^T.P^T on mma.sync m16n8k16: 16 tokens of a page fill M, the group's queries fill N = 8.
//    The online softmax keeps FP32 maxima and sums; probabilities go to FP16 for P.V (relative 2^-12 on average, the
//    size of the output's own rounding), their sum is taken before that rounding.
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
constexpr int kMaxSeqsPerLaunch = 128;
constexpr int kHeadsPerThread = kMaxGroup / (kThreads / kHeadDim);  // 4: at a merge a thread owns one column of these
constexpr int kMergeBatch = 4;       // records in flight per thread while merging
constexpr int kMinPagesPerCta = kWarps;
constexpr int kMaxCtas = 256;
constexpr int kNewestPageBit = 1 << 30;

// Shared memory, from a 1024-byte aligned base.
constexpr int kRingBytes = kWarps * kStages * kStageBytes;
constexpr int kOBufOff = kRingBytes;                                   // [warp][query][128], columns permuted
constexpr int kMlOff = kOBufOff + kWarps * kMaxGroup * kHeadDim * 4;   // m[query][warp], l[query][warp]
constexpr int kBarOff = kMlOff + 2 * kMaxGroup * kWarps * 4;
constexpr int kPrefixOff = kBarOff + kWarps * kStages * 8;
constexpr int kSkipOff = kPrefixOff + (kMaxSeqsPerLaunch + 4) * 4;
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
  float* scores;       // [sequence][KV head][page][16][score_pitch], log2 domain
  int score_pitch;
  float* weights;
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

// Flattened pages: sequence-major, then KV head, then the item's page list.
__device__ __forceinline__ long long ShareBegin(long long c, long long total, int ctas) { return c * total / ctas; }
__device__ __forceinline__ int ShareOf(long long t, long long total, int ctas) {
  return static_cast<int>(((t + 1) * ctas - 1) / total);
}
struct Cursor {
  int seq, head, entry, entries;   // entry of the item's page list, which has `entries`
};
__device__ __forceinline__ Cursor Locate(long long t, const int* prefix, int num_seqs, int heads) {
  int lo = 0, hi = num_seqs - 1;
  while (lo < hi) {   // the first sequence whose pages end behind t
    const int mid = (lo + hi) >> 1;
    if (static_cast<long long>(heads) * prefix[mid + 1] <= t) lo = mid + 1; else hi = mid;
  }
  Cursor c;
  c.seq = lo;
  c.entries = prefix[lo + 1] - prefix[lo];
  const long long rem = t - static_cast<long long>(heads) * prefix[lo];
  c.head = static_cast<int>(rem / c.entries);
  c.entry = static_cast<int>(rem - static_cast<long long>(c.head) * c.entries);
  return c;
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
  int* skip = reinterpret_cast<int*>(smem + kSkipOff);   // pages between a sequence's sinks and its window
  __shared__ int warp_total[kMaxSeqsPerLaunch / 32];
  __shared__ bool merge_here, others_done;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, tig = lane & 3;
  const int heads = p.kv_heads;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid == kThreads - 1) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tile_map) : "memory");
    for (int b = 0; b < kStages * kWarps; ++b) MbarInit(SmemAddr(smem + kBarOff) + b * 8, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  {  // page prefix over the sequences, one per thread; every CTA works out the same table
    int n = 0, incl = 0;
    if (tid < kMaxSeqsPerLaunch) {
      const int len = tid < p.num_seqs ? min(p.seq_lens[tid], p.max_blocks * kKvBlock) : 0;
      if (len > 0) {
        const int pages = (len + kKvBlock - 1) >> kKvBlockShift;
        const int window_page = max(0, len - p.window) >> kKvBlockShift;
        const int gap = max(0, window_page - p.sink_pages);
        n = pages - gap;
        skip[tid] = gap;
      }
      incl = n;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl += v;
      }
      if (lane == 31) warp_total[warp] = incl;
    }
    __syncthreads();
    if (tid < kMaxSeqsPerLaunch) {
      for (int w = 0; w < warp; ++w) incl += warp_total[w];
      prefix[tid + 1] = incl;
      if (tid == 0) prefix[0] = 0;
    }
    __syncthreads();
  }
  const long long total = static_cast<long long>(heads) * prefix[p.num_seqs];
  const int ctas = static_cast<int>(min(static_cast<long long>(gridDim.x), max(1LL, total / kMinPagesPerCta)));
  const int cta = blockIdx.x;
  if (total == 0 || cta >= ctas) {
    asm volatile("griddepcontrol.wait;" ::: "memory");   // this grid never completes ahead of the one before it
    return;
  }
  const long long share_begin = ShareBegin(cta, total, ctas), share_end = ShareBegin(cta + 1, total, ctas);

  // ---- this warp's pages: share-relative indices warp, warp + 8, ...
  const int share_len = static_cast<int>(share_end - share_begin);
  const int n_mine = share_len > warp ? (share_len - warp + kWarps - 1) / kWarps : 0;
  const uint32_t my_ring = SmemAddr(smem) + warp * (kStages * kStageBytes);
  const uint32_t my_bars = SmemAddr(smem + kBarOff) + warp * (kStages * 8);
  const uint64_t policy = L2PolicyEvictFirst();   // pages are read once per launch
  bool failed = false;
  int fail_at = 0;

  // Tile indices (4 KiB tiles of the pool; V lies `heads` tiles behind K) of 32 of this warp's pages at a time, one per
  // lane, read a batch ahead. A sequence's last page is marked: it holds the token that this step writes.
  auto fetch_tiles = [&](int batch) -> int {
    const int k = 32 * batch + lane;
    if (k >= n_mine) return 0;
    const Cursor c = Locate(share_begin + warp + static_cast<long long>(kWarps) * k, prefix, p.num_seqs, heads);
    const int page = c.entry >= p.sink_pages ? c.entry + skip[c.seq] : c.entry;
    const int block = __ldg(p.tables + static_cast<int64_t>(c.seq) * p.max_blocks + page);
    return (block * 2 * heads + c.head) | (c.entry == c.entries - 1 ? kNewestPageBit : 0);
  };
  int tiles_cur = fetch_tiles(0);
  int tiles_next = n_mine > 32 ? fetch_tiles(1) : 0;
  auto request = [&](int stage, int tile) {
    if (lane == 0) {
      MbarExpectTx(my_bars + stage * 8, kStageBytes);
      TmaLoadPage(my_ring + stage * kStageBytes, &tile_map, tile & ~kNewestPageBit, my_bars + stage * 8, policy);
    }
  };
  // Under the overlap option this grid may run ahead of the previous kernel's end: pages that an earlier step wrote
  // are requested at once, a sequence's newest page - and everything else - after the wait.
  const int first = n_mine < kStages ? n_mine : kStages;
#pragma unroll 1
  for (int i = 0; i < first; ++i) {
    const int tile = __shfl_sync(0xffffffffu, tiles_cur, i);
    if (!(tile & kNewestPageBit)) request(i, tile);
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
#pragma unroll 1
  for (int i = 0; i < first; ++i) {
    const int tile = __shfl_sync(0xffffffffu, tiles_cur, i);
    if (tile & kNewestPageBit) request(i, tile);
  }
  int n_issue = first, n_use = 0;
  auto issue_one = [&]() {
    request(n_issue % kStages, __shfl_sync(0xffffffffu, tiles_cur, n_issue & 31));
    ++n_issue;
    if ((n_issue & 31) == 0) {
      tiles_cur = tiles_next;
      tiles_next = fetch_tiles((n_issue >> 5) + 1);
    }
  };
  // ldmatrix offsets inside a stage: K rows as the A operand of S^T, V transposed as the A operand of O^T; dims 64..127
  // of a tile sit one 2 KiB box further.
  uint32_t koff[4], voff[4];
  {
    const int k_row = (lane & 7) + ((lane >> 3) & 1) * 8, k_sel = lane >> 4;
    const int v_row = (lane & 7) + (lane >> 4) * 8, v_sel = (lane >> 3) & 1;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      koff[j] = k_row * 128 + (((2 * j + k_sel) ^ (k_row & 7)) << 4);
      voff[j] = kPageBytes + v_row * 128 + (((2 * j + v_sel) ^ (v_row & 7)) << 4);
    }
  }
  constexpr uint32_t kHiDims = 2048;

  // ---- one (sequence, KV head) segment of the share after the other
  long long seg_begin = share_begin;
#pragma unroll 1
  while (seg_begin < share_end) {
    const Cursor sc = Locate(seg_begin, prefix, p.num_seqs, heads);
    const long long item_begin = seg_begin - sc.entry, item_end = item_begin + sc.entries;
    const long long seg_end = item_end < share_end ? item_end : share_end;
    const int len = min(p.seq_lens[sc.seq], p.max_blocks * kKvBlock);
    const int w0 = max(0, len - p.window);   // first token of the window
    const int gap = skip[sc.seq];
    const int seg_end_rel = static_cast<int>(seg_end - share_begin);
    const int entry0 = sc.entry - static_cast<int>(seg_begin - share_begin);   // entry of the share's page `rel` is rel + entry0
    uint32_t qb[8][2];   // B operand of S^T: query g of the group in column g, zeros past the group
    {
      const half* qrow = p.q + static_cast<int64_t>(sc.seq) * p.q_stride +
                         (static_cast<int64_t>(sc.head) * p.group + g) * kHeadDim + 2 * tig;
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
        qb[kk][0] = g < p.group ? __ldg(reinterpret_cast<const uint32_t*>(qrow + 16 * kk)) : 0u;
        qb[kk][1] = g < p.group ? __ldg(reinterpret_cast<const uint32_t*>(qrow + 16 * kk + 8)) : 0u;
      }
    }
    const bool whole = seg_begin == item_begin && seg_end == item_end;
    int c_first = cta, c_last = cta;
    if (!whole) {
      if (item_begin < share_begin) c_first = ShareOf(item_begin, total, ctas);
      if (item_end > share_end) c_last = ShareOf(item_end - 1, total, ctas);
    }
    const int others = c_last - c_first;
    const bool may_read_inline = !whole && others < kMergeBatch;
    int* ticket = p.meta + kTicketOff + c_first;
    int seen = -1;   // thread 0: how many of the others had published when it looked

    float o[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;

#pragma unroll 1
    for (int rel = warp + kWarps * n_use; rel < seg_end_rel; rel += kWarps) {
      const int stage = n_use % kStages;
      const uint32_t st = my_ring + stage * kStageBytes;
      if (!failed && !MbarWait(my_bars + stage * 8, (n_use / kStages) & 1)) {
        failed = true;
        fail_at = n_use;
        if (lane == 0) atomicExch(p.meta, 1);
      }
      if (may_read_inline && tid == 0 && seen < 0 && rel + 2 * kWarps >= seg_end_rel) seen = LoadAcquire(ticket);
      if (!failed) {
        const int entry = rel + entry0;
        const int page = entry >= p.sink_pages ? entry + gap : entry;
        const int t0 = page * kKvBlock;
        // token i of the page is visible if i < end and (i < sink or i >= win); all 16 are on a page in the middle
        const int end = len - t0, sink = p.sinks - t0, win = w0 - t0;
        const bool full = end >= kKvBlock && (sink >= kKvBlock || win <= 0);

        float s[4] = {0.0f, 0.0f, 0.0f, 0.0f}, s2[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t a[4], a2[4];
          Ldsm4(st + koff[j], a);
          Ldsm4(st + koff[j] + kHiDims, a2);
          Mma16816(s, a, qb[j][0], qb[j][1]);
          Mma16816(s2, a2, qb[j + 4][0], qb[j + 4][1]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = (s[i] + s2[i]) * p.scale_log2e;
        if (kScores && 2 * tig < p.score_pitch) {
          float* row = p.scores + ((static_cast<int64_t>(sc.seq) * heads + sc.head) * p.max_blocks + page) * (kKvBlock * p.score_pitch) +
                       g * p.score_pitch + 2 * tig;
          *reinterpret_cast<float2*>(row) = make_float2(s[0], s[1]);
          *reinterpret_cast<float2*>(row + 8 * p.score_pitch) = make_float2(s[2], s[3]);
        }
        auto visible = [&](int i) { return i < end && (i < sink || i >= win); };
        if (!full) {
          if (!visible(g)) s[0] = s[1] = -INFINITY;
          if (!visible(g + 8)) s[2] = s[3] = -INFINITY;
        }
        float mx0 = fmaxf(s[0], s[2]), mx1 = fmaxf(s[1], s[3]);
        if (__any_sync(0xffffffffu, mx0 > m0 || mx1 > m1)) {
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) {
            mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, off));
            mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, off));
          }
          const float n0 = fmaxf(m0, mx0), n1 = fmaxf(m1, mx1);
          const float a0 = Exp2(m0 - n0), a1 = Exp2(m1 - n1);
          m0 = n0;
          m1 = n1;
          l0 *= a0;
          l1 *= a1;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            o[i][0] *= a0;
            o[i][1] *= a1;
            o[i][2] *= a0;
            o[i][3] *= a1;
          }
        }
        const float p0 = Exp2(s[0] - m0), p1 = Exp2(s[1] - m1);
        const float p2 = Exp2(s[2] - m0), p3 = Exp2(s[3] - m1);
        l0 += p0 + p2;
        l1 += p1 + p3;
        const uint32_t b0 = MovmT(PackHalf2(p0, p1)), b1 = MovmT(PackHalf2(p2, p3));
        if (full) {
#pragma unroll
          for (int mt = 0; mt < 8; ++mt) {
            uint32_t a[4];
            Ldsm4T(st + voff[mt & 3] + (mt >> 2) * kHiDims, a);
            Mma16816(o[mt], a, b0, b1);
          }
        } else {
          // V rows of invisible tokens may hold NaN, and 0 * NaN would poison the sums: cleared in registers.
          const uint32_t k01 = (visible(2 * tig) ? 0x0000FFFFu : 0u) | (visible(2 * tig + 1) ? 0xFFFF0000u : 0u);
          const uint32_t k23 = (visible(2 * tig + 8) ? 0x0000FFFFu : 0u) | (visible(2 * tig + 9) ? 0xFFFF0000u : 0u);
#pragma unroll
          for (int mt = 0; mt < 8; ++mt) {
            uint32_t a[4];
            Ldsm4T(st + voff[mt & 3] + (mt >> 2) * kHiDims, a);
            a[0] &= k01;
            a[1] &= k01;
            a[2] &= k23;
            a[3] &= k23;
            Mma16816(o[mt], a, b0, b1);
          }
        }
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
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, off);
      l1 += __shfl_xor_sync(0xffffffffu, l1, off);
    }
    {
      float* ob = obuf + (warp * kMaxGroup + 2 * tig) * kHeadDim;
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) {   // columns permuted by the query pair: no bank is met twice
        const int c0 = (16 * mt + g) ^ (tig * 8), c1 = (16 * mt + g + 8) ^ (tig * 8);
        ob[c0] = o[mt][0];
        ob[kHeadDim + c0] = o[mt][1];
        ob[c1] = o[mt][2];
        ob[kHeadDim + c1] = o[mt][3];
      }
      if (g == 0) {
        mbuf[(2 * tig) * kWarps + warp] = m0;
        mbuf[(2 * tig + 1) * kWarps + warp] = m1;
        lbuf[(2 * tig) * kWarps + warp] = l0;
        lbuf[(2 * tig + 1) * kWarps + warp] = l1;
      }
    }
    __syncthreads();
    const int d = tid & (kHeadDim - 1), q0 = (tid >> 7) * kHeadsPerThread;   // this thread: column d of queries q0 .. q0 + 3
    float rm[kMergeBatch][kHeadsPerThread], rl_[kMergeBatch][kHeadsPerThread], ro[kMergeBatch][kHeadsPerThread];
    auto load_records = [&](int c0) {
#pragma unroll
      for (int j = 0; j < kMergeBatch; ++j) {
        const int c = c0 + j;
        if (c <= c_last && c != cta) {
          // a contributor's record 0 is of an item that began before its share, record 1 of one that begins in it
          const float* r = p.records + (static_cast<size_t>(c) * 2 + (c == c_first ? 1 : 0)) * kRecordFloats;
#pragma unroll
          for (int qi = 0; qi < kHeadsPerThread; ++qi) {
            if (q0 + qi < p.group) {
              ro[j][qi] = __ldcg(r + (q0 + qi) * kHeadDim + d);
              rm[j][qi] = __ldcg(r + kMaxGroup * kHeadDim + q0 + qi);
              rl_[j][qi] = __ldcg(r + kMaxGroup * kHeadDim + kMaxGroup + q0 + qi);
            }
          }
        }
      }
    };
    const bool fast = !whole && others_done;
    if (fast) load_records(c_first);
    float acc[kHeadsPerThread], mx[kHeadsPerThread], den[kHeadsPerThread];
#pragma unroll
    for (int qi = 0; qi < kHeadsPerThread; ++qi) {
      const int q = q0 + qi;
      acc[qi] = den[qi] = 0.0f;
      mx[qi] = -INFINITY;
      if (q < p.group) {
        float mw[kWarps], lw[kWarps];
#pragma unroll
        for (int i = 0; i < kWarps / 4; ++i) {
          const float4 m4 = reinterpret_cast<const float4*>(mbuf + q * kWarps)[i];
          const float4 l4 = reinterpret_cast<const float4*>(lbuf + q * kWarps)[i];
          mw[4 * i] = m4.x, mw[4 * i + 1] = m4.y, mw[4 * i + 2] = m4.z, mw[4 * i + 3] = m4.w;
          lw[4 * i] = l4.x, lw[4 * i + 1] = l4.y, lw[4 * i + 2] = l4.z, lw[4 * i + 3] = l4.w;
        }
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mx[qi] = fmaxf(mx[qi], mw[w]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float f = Exp2(mw[w] - mx[qi]);   // 0 for a warp that saw no page
          acc[qi] = fmaf(f, obuf[(w * kMaxGroup + q) * kHeadDim + (d ^ ((q >> 1) * 8))], acc[qi]);
          den[qi] = fmaf(f, lw[w], den[qi]);
        }
      }
    }
    auto write_item = [&](const float (&a)[kHeadsPerThread], const float (&m)[kHeadsPerThread], const float (&l)[kHeadsPerThread]) {
#pragma unroll
      for (int qi = 0; qi < kHeadsPerThread; ++qi) {
        if (q0 + qi < p.group) {
          const int qh = sc.head * p.group + q0 + qi;
          p.out[static_cast<int64_t>(sc.seq) * p.out_stride + static_cast<int64_t>(qh) * kHeadDim + d] = __float2half_rn(a[qi] / l[qi]);
          if (kScores && d == 0) p.stats[static_cast<int64_t>(sc.seq) * heads * p.group + qh] = make_float2(m[qi], 1.0f / l[qi]);
        }
      }
    };
    // The item from every contributor's record, in CTA order (this CTA's own from its registers).
    auto merge = [&](bool first_loaded) {
      float a[kHeadsPerThread], m[kHeadsPerThread], l[kHeadsPerThread];
#pragma unroll
      for (int qi = 0; qi < kHeadsPerThread; ++qi) a[qi] = l[qi] = 0.0f, m[qi] = -INFINITY;
#pragma unroll 1
      for (int c0 = c_first; c0 <= c_last; c0 += kMergeBatch) {
        if (!first_loaded) load_records(c0);
        first_loaded = false;
#pragma unroll
        for (int j = 0; j < kMergeBatch; ++j) {
          if (c0 + j <= c_last) {
            const bool mine = c0 + j == cta;
#pragma unroll
            for (int qi = 0; qi < kHeadsPerThread; ++qi) {
              if (q0 + qi < p.group) {
                const float mc = mine ? mx[qi] : rm[j][qi], lc = mine ? den[qi] : rl_[j][qi], oc = mine ? acc[qi] : ro[j][qi];
                const float n = fmaxf(m[qi], mc), keep = Exp2(m[qi] - n), add = Exp2(mc - n);
                a[qi] = fmaf(add, oc, a[qi] * keep);
                l[qi] = fmaf(add, lc, l[qi] * keep);
                m[qi] = n;
              }
            }
          }
        }
      }
      write_item(a, m, l);
    };
    if (whole) {
      write_item(acc, mx, den);
    } else if (fast) {
      merge(true);
      if (tid == 0) *ticket = 0;   // everyone had arrived: ready for the next launch
    } else {
      float* rec = p.records + (static_cast<size_t>(cta) * 2 + (item_begin < share_begin ? 0 : 1)) * kRecordFloats;
#pragma unroll
      for (int qi = 0; qi < kHeadsPerThread; ++qi) {
        if (q0 + qi < p.group) {
          rec[(q0 + qi) * kHeadDim + d] = acc[qi];
          if (d == 0) {
            rec[kMaxGroup * kHeadDim + q0 + qi] = mx[qi];
            rec[kMaxGroup * kHeadDim + kMaxGroup + q0 + qi] = den[qi];
          }
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
        merge(false);
      }
    }
    __syncthreads();   // obuf and the flags are free for the next segment
    seg_begin = seg_end;
  }
  if (failed) {   // copies in flight get one more bounded chance to land before the shared memory goes away
    for (int k = fail_at; k < n_issue; ++k) MbarWait(my_bars + (k % kStages) * 8, (k / kStages) & 1);
  }
}

// Second kernel of the weights launcher: per cached token and KV head, the sum over the group of
// exp2(score - maximum) / sum, added to the token's weight. One thread per (head, page, slot) of a sequence; a token's
// scores of the group lie side by side, so a warp reads and writes whole lines.
__global__ void __launch_bounds__(256) AccumulateKernel(const Params p, int parts) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t seq = blockIdx.x / parts;
  const int part = blockIdx.x % parts;
  const int len = min(p.seq_lens[seq], p.max_blocks * kKvBlock);
  if (len <= 0) return;
  const int slots = ((len + kKvBlock - 1) >> kKvBlockShift) * kKvBlock;
  const int32_t* table = p.tables + seq * p.max_blocks;
  for (int64_t i = part * 256 + threadIdx.x; i < static_cast<int64_t>(slots) * p.kv_heads; i += static_cast<int64_t>(parts) * 256) {
    const int head = static_cast<int>(i / slots), t = static_cast<int>(i - static_cast<int64_t>(head) * slots);
    if (t >= len) continue;
    const float2* st = p.stats + (seq * p.kv_heads + head) * p.group;
    const float* s = p.scores + ((seq * p.kv_heads + head) * p.max_blocks * kKvBlock + t) * p.score_pitch;
    float sum = 0.0f;
    for (int q = 0; q < p.group; ++q) {
      const float2 ml = __ldcg(st + q);
      sum = fmaf(Exp2(__ldcg(s + q) - ml.x), ml.y, sum);
    }
    float* w = p.weights + (static_cast<int64_t>(table[t >> kKvBlockShift]) * p.kv_heads + head) * kKvBlock + (t & (kKvBlock - 1));
    *w = t == len - 1 ? sum : *w + sum;
  }
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
int ScorePitch(int group) { return (group + 1) & ~1; }
size_t StatsBytes(int64_t num_seqs, int q_heads) { return (static_cast<size_t>(num_seqs) * q_heads * sizeof(float2) + 255) & ~static_cast<size_t>(255); }
size_t Workspace(int64_t num_seqs, int max_blocks, int q_heads, int kv_heads, bool weights) {
  size_t bytes = kMetaBytes + kRecordBytes;
  if (weights)
    bytes += StatsBytes(num_seqs, q_heads) + static_cast<size_t>(num_seqs) * kv_heads * max_blocks * kKvBlock *
                                                 ScorePitch(q_heads / kv_heads) * sizeof(float);
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
  p.score_pitch = ScorePitch(p.group);
  // No more CTAs than shares of kMinPagesPerCta pages can exist: a row's list is at most this long.
  const int64_t list = p.sink_pages + ((p.window + kKvBlock - 2) >> kKvBlockShift) + 1;
  const int64_t pages = list < c.max_blocks ? list : c.max_blocks;
  if (pages * kMaxSeqsPerLaunch > INT32_MAX && pages * c.num_seqs > INT32_MAX)
    return Fail(RL_E_TOO_LARGE, "%s: more than 2^31 pages in one call", c.fn);
  const int sms = CurrentDeviceFacts().sm_count < kMaxCtas ? CurrentDeviceFacts().sm_count : kMaxCtas;
  const int64_t row = static_cast<int64_t>(c.kv_heads) * c.max_blocks * kKvBlock * p.score_pitch;
  for (int first = 0; first < c.num_seqs; first += kMaxSeqsPerLaunch) {
    const int n = c.num_seqs - first < kMaxSeqsPerLaunch ? c.num_seqs - first : kMaxSeqsPerLaunch;
    p.out = static_cast<half*>(c.out) + first * c.out_row_stride;
    p.q = static_cast<const half*>(c.q) + first * c.q_row_stride;
    p.tables = c.tables + static_cast<int64_t>(first) * c.max_blocks;
    p.seq_lens = c.seq_lens + first;
    p.num_seqs = n;
    p.stats = stats + static_cast<int64_t>(first) * c.q_heads;
    p.scores = scores + first * row;
    const int64_t shares = (n * c.kv_heads * pages) / kMinPagesPerCta;
    const int grid = static_cast<int>(shares < 1 ? 1 : shares < sms ? shares : sms);
    const cudaError_t e = LaunchOverlapped(DecodeKernel<kScores>, dim3(grid), dim3(kThreads), kSmemBytes, c.stream, p, tile_map);
    if (e != cudaSuccess) return Fail(static_cast<int>(e), "%s: %s", c.fn, cudaGetErrorString(e));
  }
  if (kScores) {
    p.tables = c.tables;
    p.seq_lens = c.seq_lens;
    p.stats = stats;
    p.scores = scores;
    p.weights = c.weights;
    // enough CTAs per sequence for its longest possible cache, but no more in all than fill the machine a few times
    const int64_t most = (static_cast<int64_t>(c.max_blocks) * kKvBlock * c.kv_heads + 255) / 256;
    const int64_t fair = (8LL * sms + c.num_seqs - 1) / c.num_seqs;
    const int parts = static_cast<int>(most < fair ? most : fair);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(c.num_seqs) * parts);
    cfg.blockDim = dim3(256);
    cfg.stream = c.stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;   // it begins with the wait for the kernel above
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, AccumulateKernel, p, parts);
    if (e != cudaSuccess) return Fail(static_cast<int>(e), "%s (weights): %s", c.fn, cudaGetErrorString(e));
  }
  return LaunchStatus(c.fn);
}

}  // namespace wattn
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
