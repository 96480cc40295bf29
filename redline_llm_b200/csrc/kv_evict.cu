// Eviction from the paged cache by accumulated attention weight, for sm_100a (B200). Per sequence and KV head: a
// cache of L tokens shrinks to L' = min(L, budget); the first `sinks` and the last `recent` tokens stay, and of the
// rest the budget - sinks - recent with the largest weight (equal weights: the lower position stays first; a NaN
// counts below every number). Kept tokens move, in cache order, to slots 0 .. L'-1 of the destination table's pages,
// K row, V row and weight together.
//
// Two kernels. What bounds them: the selection is a chain of short dependent passes (latency), the move is a copy of
// the kept rows (HBM).
//  * Select, one CTA or a cluster of them per (sequence, KV head): weights become integers that compare the same way and stay in shared
//    memory; a histogram over their range and its suffix sums name the bin of the last kept token, whose keys leave the
//    crowd - one per thread - and are divided further until the last few are ranked against one another; then an ordered
//    sweep writes the kept positions, each warp a stretch of the sequence, warp scans giving the ranks.
//  * Move, 32 rows per warp: a lane looks up one row's source and destination, then the warp copies the rows 16 bytes a
//    lane, eight rows in flight. In place a cluster of up to eight CTAs walks a (sequence, head) in cache order, every row of a round
//    read before any of it is written: a row never moves to a higher slot, so what a round overwrites was read in it or
//    before it.
#include <mutex>

#include "common.cuh"

namespace rl {
namespace evict {

struct Params {
  half* pool;
  float* weights;
  const int32_t* tables;
  const int32_t* dst_tables;
  const int32_t* seq_lens;
  int32_t* new_lens;
  int32_t* kept;
  int max_blocks;
  int dst_max_blocks;
  int kv_heads;
  int head_dim;
  int budget;
  int sinks;
  int recent;
  int cached_keys;   // keys that fit the select kernel's shared memory
};

// Weights as unsigned integers that compare the same way: 0 for a NaN, -0 like +0.
__device__ __forceinline__ uint32_t OrderKey(float w) {
  if (w != w) return 0u;
  const uint32_t b = __float_as_uint(w + 0.0f);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ int CachedTokens(const Params& p, int seq) {
  return max(0, min(p.seq_lens[seq], p.max_blocks * kKvBlock));
}

constexpr int kMaxSelectCluster = 8;
constexpr int kBinBits = 11, kBins = 1 << kBinBits;
constexpr int kMaxListed = 1024;   // candidates of a bin that are taken out of the crowd: one per thread
constexpr int kRanked = 64;        // of those, as many as are simply ranked against one another
constexpr int kLoadAhead = 8;      // quads of weights a thread has in flight
constexpr int kMaxCachedKeys = 45 * 1024;   // 180 KB
constexpr int kPairKeys = 22 * 1024;        // two CTAs' keys fit an SM beside 24 KB each of everything else

// What the CTAs of a cluster tell one another.
struct Shared {
  int bins[kBins];
  uint32_t list[kMaxListed];
  uint32_t lo, hi;       // range of this CTA's keys
  int listed;            // keys in its list
  int sure, equal;       // its tokens above the threshold (or kept in any case), and at it
};

__device__ __forceinline__ void ClusterBarrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A 32-bit word of the same variable in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t LoadPeer(const void* mine, int rank) {
  uint32_t addr = static_cast<uint32_t>(__cvta_generic_to_shared(mine)), v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ int2 LoadPeer2(const int* mine, int rank) {   // two words, 8-byte aligned
  uint32_t addr = static_cast<uint32_t>(__cvta_generic_to_shared(mine));
  int2 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.v2.s32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}

// Grid: (sequences * cluster, KV heads). CTA `rank` of an item's cluster has every quad of tokens of its slice. 1024 threads
// where a CTA has its SM to itself; 512, without clusters, where there are more items than SMs and two CTAs share one.
template <int kSelectThreads>
__global__ void __launch_bounds__(kSelectThreads, 1024 / kSelectThreads) SelectKernel(const Params p, int cluster) {
  constexpr int kSelectWarps = kSelectThreads / 32, kListed = kSelectThreads, kPerThread = kBins / kSelectThreads;
  static_assert(kListed <= kMaxListed && kPerThread % 2 == 0, "a thread per listed key, pairs of bins");
  static_assert(2 * (kPairKeys * 4 + sizeof(Shared) + (kListed + 4 + kBins + 4 * kSelectWarps + 8) * 4 + 1024) <= 228 * 1024 || kSelectThreads > 512,
                "two CTAs share an SM");
  extern __shared__ __align__(16) uint32_t keys[];
  __shared__ __align__(16) Shared sh;
  __shared__ __align__(16) uint32_t crowd[kListed + 4];
  __shared__ int local_bins[kBins];
  __shared__ int warp_sum[kSelectWarps], warp_equal[kSelectWarps];
  __shared__ uint32_t warp_lo[kSelectWarps], warp_hi[kSelectWarps], found_key;
  __shared__ int found_bin, found_above, found_count, crowded;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int seq = blockIdx.x / cluster, rank = blockIdx.x % cluster, head = blockIdx.y;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int len = CachedTokens(p, seq);
  const int n = min(len, p.budget);
  const int32_t* table = p.tables + static_cast<int64_t>(seq) * p.max_blocks;
  int32_t* kept = p.kept + (static_cast<int64_t>(seq) * p.kv_heads + head) * p.budget;
  for (int j = n + rank * kSelectThreads + tid; j < p.budget; j += cluster * kSelectThreads) kept[j] = -1;
  if (len <= p.budget) {   // (the same for the whole cluster)
    for (int j = rank * kSelectThreads + tid; j < n; j += cluster * kSelectThreads) kept[j] = j;
    return;
  }
  // Candidates are tokens [a, b). Tokens are handled in quads - four neighbours share a page; this CTA has quads
  // [q_first, q_last), keys[] holds theirs from q_first on.
  const int a = p.sinks, b = len - p.recent;
  const int all_quads = (len + 3) >> 2;
  const int slice = (all_quads + cluster - 1) / cluster;
  const int q_first = min(all_quads, rank * slice), q_last = min(all_quads, q_first + slice);
  const int quads = q_last - q_first;
  const bool cached = quads * 4 <= p.cached_keys;
  auto order = [](const float4& w) { return make_uint4(OrderKey(w.x), OrderKey(w.y), OrderKey(w.z), OrderKey(w.w)); };
  auto weights_of = [&](int q, int block) {
    return *reinterpret_cast<const float4*>(p.weights + (static_cast<int64_t>(block) * p.kv_heads + head) * kKvBlock + ((4 * q) & (kKvBlock - 1)));
  };
  auto quad = [&](int q) { return cached ? reinterpret_cast<const uint4*>(keys)[q - q_first] : order(weights_of(q, table[q >> 2])); };
  auto use_quad = [&](int q, const uint4& k, auto&& use) {
    const int t = 4 * q;
    if (t >= a && t + 3 < b) {
      use(k.x), use(k.y), use(k.z), use(k.w);
    } else {
      if (t >= a && t < b) use(k.x);
      if (t + 1 >= a && t + 1 < b) use(k.y);
      if (t + 2 >= a && t + 2 < b) use(k.z);
      if (t + 3 >= a && t + 3 < b) use(k.w);
    }
  };
  auto for_each = [&](auto&& use) {
#pragma unroll 4
    for (int q = q_first + tid; q < q_last; q += kSelectThreads) use_quad(q, quad(q), use);
  };
  auto clear_bins = [&](int* bins) {
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) bins[tid + i * kSelectThreads] = 0;
  };

  // thr: tokens with a larger key stay, and the first `ties` of those whose key equals it
  uint32_t thr = 0xFFFFFFFFu;   // no weight has this key
  int ties = 0;
  int need = p.budget - p.sinks - p.recent;
  if (need > 0) {
    // The keys' range first, while they are fetched: bins that divide the RANGE spread over the candidates, where bins
    // of leading bits would all be hit in the few octaves that attention weights lie in.
    uint32_t lo = 0xFFFFFFFFu, hi = 0;
    auto widen = [&](uint32_t k) {
      lo = min(lo, k);
      hi = max(hi, k);
    };
    clear_bins(sh.bins);
    if (tid == 0) sh.listed = crowded = 0;
#pragma unroll 1
    for (int q0 = q_first + tid; q0 < q_last; q0 += kLoadAhead * kSelectThreads) {
      int block[kLoadAhead];   // all table entries of a round in flight, then all weights
      float4 w[kLoadAhead];
#pragma unroll
      for (int j = 0; j < kLoadAhead; ++j) block[j] = table[min(q0 + j * kSelectThreads, q_last - 1) >> 2];
#pragma unroll
      for (int j = 0; j < kLoadAhead; ++j) w[j] = weights_of(min(q0 + j * kSelectThreads, q_last - 1), block[j]);
#pragma unroll
      for (int j = 0; j < kLoadAhead; ++j) {
        const int q = q0 + j * kSelectThreads;
        if (q < q_last) {
          const uint4 k = order(w[j]);
          if (cached) reinterpret_cast<uint4*>(keys)[q - q_first] = k;
          use_quad(q, k, widen);
        }
      }
    }
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    if (lane == 0) {
      warp_lo[warp] = lo;
      warp_hi[warp] = hi;
    }
    __syncthreads();
    lo = __reduce_min_sync(0xffffffffu, warp_lo[lane % kSelectWarps]);
    hi = __reduce_max_sync(0xffffffffu, warp_hi[lane % kSelectWarps]);
    if (cluster > 1) {
      if (tid == 0) {
        sh.lo = lo;
        sh.hi = hi;
      }
      ClusterBarrier();
      lo = __reduce_min_sync(0xffffffffu, lane < cluster ? LoadPeer(&sh.lo, lane) : 0xFFFFFFFFu);
      hi = __reduce_max_sync(0xffffffffu, lane < cluster ? LoadPeer(&sh.hi, lane) : 0u);
    }
    // Each round: the need-th largest key among those in [lo, hi] lies in one of up to 2048 bins of 2^shift keys. The
    // counts of all CTAs are summed by each of them, which then go on alike.
    uint32_t mine = 0;   // once the keys of one bin are listed: this thread's
    int count = 0;       // of keys listed
#pragma unroll 1
    while (true) {
      const int shift = max(0, 32 - __clz(hi - lo) - kBinBits);
      int bin[kPerThread];   // this thread's bins, from the top down: bin[i] is number top - i
      const int top = kBins - 1 - kPerThread * tid;
      if (count == 0) {
        for_each([&](uint32_t k) {
          if (k >= lo && k <= hi) atomicAdd(&sh.bins[(k - lo) >> shift], 1);
        });
        if (cluster > 1) {
          ClusterBarrier();
          static_assert(kMaxSelectCluster == 8, "unrolled below");
#pragma unroll
          for (int i = 0; i < kPerThread; i += 2) {
            int2 pair[kMaxSelectCluster];   // all requests under way before the first is used
#pragma unroll
            for (int r = 0; r < kMaxSelectCluster; ++r) pair[r] = r < cluster ? LoadPeer2(&sh.bins[top - i - 1], r) : make_int2(0, 0);
            bin[i] = bin[i + 1] = 0;
#pragma unroll
            for (int r = 0; r < kMaxSelectCluster; ++r) {
              bin[i] += pair[r].y;
              bin[i + 1] += pair[r].x;
            }
          }
        } else {
          __syncthreads();
#pragma unroll
          for (int i = 0; i < kPerThread; ++i) bin[i] = sh.bins[top - i];
        }
      } else {
        clear_bins(local_bins);
        __syncthreads();
        if (tid < count && mine >= lo && mine <= hi) atomicAdd(&local_bins[(mine - lo) >> shift], 1);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) bin[i] = local_bins[top - i];
      }
      int sum = 0;
#pragma unroll
      for (int i = 0; i < kPerThread; ++i) sum += bin[i];
      int incl = sum;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl += v;
      }
      if (lane == 31) warp_sum[warp] = incl;
      __syncthreads();
      int above = __reduce_add_sync(0xffffffffu, lane < warp && lane < kSelectWarps ? warp_sum[lane] : 0) + incl - sum;
#pragma unroll
      for (int i = 0; i < kPerThread; ++i) {
        if (above < need && above + bin[i] >= need) {   // one bin of one thread
          found_bin = top - i;
          found_above = above;
          found_count = bin[i];
        }
        above += bin[i];
      }
      __syncthreads();
      need -= found_above;
      lo += static_cast<uint32_t>(found_bin) << shift;
      const int found = found_count;
      if (found == need) {   // all of this bin stay: whatever is below it does not
        thr = lo - 1;        // (never below 0: some candidate is left out)
        break;
      }
      if (shift == 0) {
        thr = lo;
        ties = need;
        break;
      }
      hi = min(hi, lo + ((1u << shift) - 1u));
      if (count == 0 && found <= kListed) {
        // Few enough to leave the crowd: every CTA lists its own, then copies the lists of all, in CTA order.
        for_each([&](uint32_t k) {
          if (k >= lo && k <= hi) sh.list[atomicAdd(&sh.listed, 1)] = k;
        });
        if (cluster > 1) ClusterBarrier(); else __syncthreads();
        count = found;
        int from = tid, r = 0;
        if (cluster > 1) {
          for (; r < cluster; ++r) {
            const int theirs = static_cast<int>(LoadPeer(&sh.listed, r));
            if (from < theirs) break;
            from -= theirs;
          }
        }
        if (tid < count) mine = cluster > 1 ? LoadPeer(&sh.list[from], r) : sh.list[from];
      } else if (count == 0) {
        if (cluster > 1) ClusterBarrier(); else __syncthreads();   // every peer has read these counts
        clear_bins(sh.bins);
        __syncthreads();
        continue;
      }
      if (found <= kRanked) {   // rank the last few against one another
        const bool in = tid < count && mine >= lo && mine <= hi;
        if (in) crowd[atomicAdd(&crowded, 1)] = mine;
        __syncthreads();
        if (in) {
          int larger = 0, equal = 0;
          for (int i = 0; i < found; ++i) {
            larger += crowd[i] > mine;
            equal += crowd[i] == mine;
          }
          if (larger < need && larger + equal >= need) {   // every thread with this key says the same
            found_key = mine;
            found_above = larger;
          }
        }
        __syncthreads();
        thr = found_key;
        ties = need - found_above;
        break;
      }
    }
  }

  // ---- the kept positions in cache order: each CTA its slice, each warp a stretch of it, four tokens per lane
  __syncthreads();
  const int stretch = ((quads + kSelectThreads - 1) / kSelectThreads) * 32;
  const int q_begin = min(q_last, q_first + warp * stretch), q_end = min(q_last, q_begin + stretch);
  // of the four tokens from 4q on, one bit each: those that stay in any case, and those whose key equals the threshold
  auto classify = [&](int q, uint32_t& sure, uint32_t& equal) {
    sure = equal = 0;
    if (q >= q_end) return;
    const int t = 4 * q;
    const bool inside = t >= a && t + 3 < b;
    uint4 k = make_uint4(0, 0, 0, 0);
    if (t + 3 >= a && t < b) k = quad(q);
    sure = (k.x > thr ? 1u : 0u) | (k.y > thr ? 2u : 0u) | (k.z > thr ? 4u : 0u) | (k.w > thr ? 8u : 0u);
    equal = (k.x == thr ? 1u : 0u) | (k.y == thr ? 2u : 0u) | (k.z == thr ? 4u : 0u) | (k.w == thr ? 8u : 0u);
    if (ties == 0) equal = 0;
    if (!inside) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (t + e < a || t + e >= b) {   // not a candidate: stays if it is a token at all
          sure |= 1u << e;
          equal &= ~(1u << e);
        }
        if (t + e >= len) sure &= ~(1u << e);
      }
    }
  };
  int n_sure = 0, n_equal = 0;
#pragma unroll 4
  for (int q0 = q_begin; q0 < q_end; q0 += 32) {
    uint32_t sure, equal;
    classify(q0 + lane, sure, equal);
    n_sure += __popc(sure);
    n_equal += __popc(equal);
  }
  n_sure = __reduce_add_sync(0xffffffffu, n_sure);
  n_equal = __reduce_add_sync(0xffffffffu, n_equal);
  if (lane == 0) {
    warp_sum[warp] = n_sure;
    warp_equal[warp] = n_equal;
  }
  __syncthreads();
  int equal_before = __reduce_add_sync(0xffffffffu, lane < warp ? warp_equal[lane] : 0);
  int sure_before = __reduce_add_sync(0xffffffffu, lane < warp ? warp_sum[lane] : 0);
  if (cluster > 1) {
    if (tid == kSelectThreads - 1) {
      sh.sure = sure_before + warp_sum[warp];
      sh.equal = equal_before + warp_equal[warp];
    }
    ClusterBarrier();
    sure_before += __reduce_add_sync(0xffffffffu, lane < rank ? static_cast<int>(LoadPeer(&sh.sure, lane)) : 0);
    equal_before += __reduce_add_sync(0xffffffffu, lane < rank ? static_cast<int>(LoadPeer(&sh.equal, lane)) : 0);
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");   // (waited for at the end: a peer may still read)
  }
  int at = sure_before + min(equal_before, ties);
#pragma unroll 2
  for (int q0 = q_begin; q0 < q_end; q0 += 32) {
    uint32_t sure, equal;
    classify(q0 + lane, sure, equal);
    const uint32_t mine = __popc(sure) | __popc(equal) << 16;
    uint32_t incl = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += v;
    }
    const uint32_t sum = __shfl_sync(0xffffffffu, incl, 31), excl = incl - mine;
    const int stay = max(0, ties - equal_before);   // equals that still stay from here on
    int left = stay - static_cast<int>(excl >> 16);
    int j = at + static_cast<int>(excl & 0xFFFFu) + min(static_cast<int>(excl >> 16), stay);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool tie = (equal >> e) & 1u;
      if (((sure >> e) & 1u) || (tie && left > 0)) kept[j++] = 4 * (q0 + lane) + e;
      left -= tie;
    }
    at += static_cast<int>(sum & 0xFFFFu) + min(static_cast<int>(sum >> 16), stay);
    equal_before += static_cast<int>(sum >> 16);
  }
  if (cluster > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

constexpr int kMoveThreads = 256;
constexpr int kMoveWarps = kMoveThreads / 32;
constexpr int kRowsInFlight = 8;    // per warp, 512 bytes each; with four CTAs on an SM 128 KB are in flight
constexpr int kWideWarps = 16, kWideRows = 16;   // in place with few items: a CTA has its SM to itself
constexpr int kCluster = 8;

// kRowWords: 16-byte words of one token's K row and V row together when it is the same for every lane pattern (head_dim
// 128: 32, one word per lane and row), 0 for any other width.
// kLookup: rows a warp looks up at a time; in place (the K = 128 form) also the rows it has in registers at a time.
template <bool kInPlace, int kRowWords, int kLookup, int kWarps>
__global__ void __launch_bounds__(kWarps * 32, kWarps > kMoveWarps ? 1 : 4) MoveKernel(const Params p, int parts) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int seq = blockIdx.x / parts, part = blockIdx.x % parts, head = blockIdx.y;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n = min(CachedTokens(p, seq), p.budget);
  // the old length may sit in the same place: cut to the budget a second time it stays what it is
  if (part == 0 && head == 0 && threadIdx.x == 0) p.new_lens[seq] = n;
  const int32_t* table = p.tables + static_cast<int64_t>(seq) * p.max_blocks;
  const int32_t* dst = p.dst_tables + static_cast<int64_t>(seq) * p.dst_max_blocks;
  const int32_t* kept = p.kept + (static_cast<int64_t>(seq) * p.kv_heads + head) * p.budget;
  const int words = p.head_dim / 8;                                        // 16-byte words of a K row
  const int64_t v_words = static_cast<int64_t>(p.kv_heads) * kKvBlock * words;   // from a K row to its V row
  uint4* pool = reinterpret_cast<uint4*>(p.pool);
  auto row_index = [&](int64_t block, int t) { return ((block * 2 * p.kv_heads + head) * kKvBlock + (t & (kKvBlock - 1))) * words; };
  auto weight_index = [&](int64_t block, int t) { return (block * p.kv_heads + head) * kKvBlock + (t & (kKvBlock - 1)); };

  // Rows a warp looks up and moves per round. In place all of them must be in registers before the first is written;
  // with one row per warp that holds for any width, since a word only ever moves to the same word of another row.
  constexpr int kRows = !kInPlace || kRowWords == 32 ? kLookup : 1;
  constexpr int kFlight = kInPlace ? kRows : kRowsInFlight;
  const int round = parts * kWarps * kRows;
  for (int j0 = 0; j0 < n; j0 += round) {
    const int first = j0 + (part * kWarps + warp) * kRows;
    const int rows = max(0, min(kRows, n - first));
    int64_t from = 0, to = 0, weight_to = 0;
    float weight = 0.0f;
    bool moves = false;
    if (lane < rows) {
      const int j = first + lane, t = kept[j];
      moves = !(kInPlace && t == j);
      const int64_t from_block = table[t >> kKvBlockShift], to_block = dst[j >> kKvBlockShift];
      from = row_index(from_block, t);
      to = row_index(to_block, j);
      weight = p.weights[weight_index(from_block, t)];
      weight_to = weight_index(to_block, j);
    }
    const uint32_t moving = __ballot_sync(0xffffffffu, moves);
    if (kRowWords == 32) {
      const int64_t mine = lane < 16 ? lane : v_words + lane - 16;   // this lane's word of a row: K, then V
#pragma unroll
      for (int r0 = 0; r0 < kRows; r0 += kFlight) {
        uint4 v[kFlight];
#pragma unroll
        for (int r = 0; r < kFlight; ++r) {
          const int64_t src = __shfl_sync(0xffffffffu, from, r0 + r);
          if ((moving >> (r0 + r)) & 1) v[r] = pool[src + mine];
        }
        if (kInPlace) {   // all rows of the round are in registers, over the whole cluster, before any is written
          asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
          asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        }
#pragma unroll
        for (int r = 0; r < kFlight; ++r) {
          const int64_t d = __shfl_sync(0xffffffffu, to, r0 + r);
          if ((moving >> (r0 + r)) & 1) pool[d + mine] = v[r];
        }
      }
    } else {
      // any other width: the words of the warp's rows dealt to its lanes, four per lane at a time
      const int row_words = 2 * words;
      const int total = kRows * row_words;
#pragma unroll 1
      for (int w0 = 0; w0 < total; w0 += 32 * 4) {
        uint4 v[4];
        int64_t d[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int w = w0 + i * 32 + lane, r = min(w / row_words, 31), x = w - r * row_words;
          const int64_t off = x < words ? x : v_words + x - words;
          const int64_t src = __shfl_sync(0xffffffffu, from, r) + off;
          d[i] = __shfl_sync(0xffffffffu, to, r) + off;
          if (w >= total || !((moving >> r) & 1)) d[i] = -1;
          if (d[i] >= 0) v[i] = pool[src];
        }
        if (kInPlace) {
          asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
          asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (d[i] >= 0) pool[d[i]] = v[i];
      }
    }
    if (moves) p.weights[weight_to] = weight;
  }
  // Under the overlap option a decode launch behind this one requests pages and reads lengths before its own wait. So
  // dependents are released by each block's last act, when its writes are done, and not at its start. The option is the
  // launching host's state when it comes to the DECODE launch, which this one cannot know: it always holds. (Released at
  // the start: 8.6 in place of 8.8 us for one sequence of 1100 tokens to 1024, 54.6 in place of 56.5 for 64 to 2048.)
  // Those pages are fetched by tensor copies, which go by the asynchronous proxy: the first fence orders the block's rows
  // for them, on the side that wrote them. (On the reading side as well it costs every decode launch 0.3 us.)
  __syncthreads();
  if (threadIdx.x == 0) {
    asm volatile("fence.proxy.async;" ::: "memory");
    __threadfence();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  }
}

// First use on a device: the selection's shared memory.
constexpr int kMaxDevices = 64;
bool g_ready[kMaxDevices];
std::mutex g_mutex;
int EnsureReady(const char* fn) {
  bool& ready = g_ready[CurrentDeviceIndex()];
  std::lock_guard<std::mutex> lock(g_mutex);
  if (ready) return RL_OK;
  cudaError_t e = cudaFuncSetAttribute(SelectKernel<1024>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxCachedKeys * 4);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(SelectKernel<512>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxCachedKeys * 4);
  if (e != cudaSuccess) return Fail(static_cast<int>(e), "%s: shared-memory opt-in: %s", fn, cudaGetErrorString(e));
  ready = true;
  return RL_OK;
}

}  // namespace evict
int KvEvictInit() { return evict::EnsureReady("kv_evict"); }
}  // namespace rl

extern "C" int rl_launch_kv_evict(void* kv_pool_layer, float* weights, const int32_t* block_tables,
                                  int32_t max_blocks_per_seq, const int32_t* dst_block_tables,
                                  int32_t dst_max_blocks_per_seq, const int32_t* seq_lens, int32_t* new_seq_lens,
                                  int32_t* kept, int32_t num_seqs, int32_t num_kv_heads, int32_t head_dim,
                                  int32_t budget, int32_t sinks, int32_t recent, void* stream) {
  using namespace rl;
  using namespace rl::evict;
  constexpr const char* fn = "kv_evict";
  if (num_seqs <= 0) return RL_OK;
  if (!kv_pool_layer || !weights || !block_tables || !dst_block_tables || !seq_lens || !new_seq_lens || !kept)
    return Fail(RL_E_NULL_POINTER, "%s: null device pointer", fn);
  if (num_kv_heads < 1 || num_kv_heads > 65535 || head_dim < 8 || head_dim > 1024 || head_dim % 8 != 0)
    return Fail(RL_E_BAD_SHAPE, "%s: 1 to 65535 KV heads, head_dim a multiple of 8 up to 1024", fn);
  if (max_blocks_per_seq < 1 || dst_max_blocks_per_seq < 1)
    return Fail(RL_E_BAD_SHAPE, "%s: max_blocks_per_seq must be >= 1", fn);
  if (max_blocks_per_seq > (1 << 26) || dst_max_blocks_per_seq > (1 << 26))
    return Fail(RL_E_TOO_LARGE, "%s: at most 2^26 blocks per sequence", fn);
  if (budget < 1 || sinks < 0 || recent < 0 || static_cast<int64_t>(sinks) + recent > budget)
    return Fail(RL_E_BAD_SHAPE, "%s: budget >= 1, sinks and recent >= 0 and together within the budget", fn);
  const int32_t cover = dst_max_blocks_per_seq < max_blocks_per_seq ? dst_max_blocks_per_seq : max_blocks_per_seq;
  if (cover < max_blocks_per_seq && static_cast<int64_t>(cover) * kKvBlock < budget)
    return Fail(RL_E_BAD_SHAPE, "%s: the destination table row does not cover what a sequence keeps", fn);
  if (dst_block_tables == block_tables && dst_max_blocks_per_seq != max_blocks_per_seq)
    return Fail(RL_E_BAD_SHAPE, "%s: in place, both tables have the same row length", fn);
  if (!Aligned16(kv_pool_layer) || !Aligned16(weights))
    return Fail(RL_E_BAD_SHAPE, "%s: the pool slice and the weights must be 16-byte aligned", fn);
  if (num_seqs > INT32_MAX / kCluster || budget > (1 << 30)) return Fail(RL_E_TOO_LARGE, "%s: at most 2^28 sequences and a budget of 2^30", fn);
  const int64_t tokens = static_cast<int64_t>(max_blocks_per_seq) * kKvBlock;
  Params p;
  p.pool = static_cast<half*>(kv_pool_layer);
  p.weights = weights;
  p.tables = block_tables;
  p.dst_tables = dst_block_tables;
  p.seq_lens = seq_lens;
  p.new_lens = new_seq_lens;
  p.kept = kept;
  p.max_blocks = max_blocks_per_seq;
  p.dst_max_blocks = dst_max_blocks_per_seq;
  p.kv_heads = num_kv_heads;
  p.head_dim = head_dim;
  p.budget = budget;
  p.sinks = sinks;
  p.recent = recent;
  const int64_t items = static_cast<int64_t>(num_seqs) * num_kv_heads;
  p.cached_keys = static_cast<int>(tokens < kMaxCachedKeys ? tokens : kMaxCachedKeys);
  const int rc = EnsureReady(fn);
  if (rc != RL_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // A cluster per item as far as the SMs go round and each CTA still has a few thousand tokens (as long as the table
  // says the sequences may be).
  const int sm_count = CurrentDeviceFacts().sm_count;
  int cluster = 1;
  while (cluster < kMaxSelectCluster && 2 * cluster * items <= sm_count && tokens / (2 * cluster) >= 2048) cluster *= 2;
  // More items than SMs: half the threads, so that two CTAs share an SM and wait for their loads side by side (57 x 8 items of
  // 425-9779 tokens: 27.0 us with the move, with 1024 threads each 32.6) - as long as the table's width lets the keys of two
  // into its shared memory. Wider ones have an SM each in either form, and then all threads help (20 x 8 items of 30000-32768:
  // 47.7 us, with 512 threads 58.2; the 57 x 8 in a table of 32768: 32.8 and 34.0).
  const bool crowded = items > sm_count && p.cached_keys <= kPairKeys;
  const size_t key_bytes = static_cast<size_t>(p.cached_keys) * 4;
  const dim3 select_grid(static_cast<unsigned>(num_seqs) * cluster, num_kv_heads);
  cudaError_t e = crowded ? LaunchDependent(SelectKernel<512>, select_grid, dim3(512), key_bytes, 1, s, p, 1)
                          : LaunchDependent(SelectKernel<1024>, select_grid, dim3(1024), key_bytes, cluster, s, p, cluster);
  if (e != cudaSuccess) return Fail(static_cast<int>(e), "%s: %s", fn, cudaGetErrorString(e));
  const bool in_place = dst_block_tables == block_tables;
  // Out of place a warp looks 32 rows up and moves them eight at a time - or, while all rows then still fit the machine
  // at once, only eight, so that no row waits for another.
  const int64_t longest = tokens < budget ? tokens : budget;
  const int sms = CurrentDeviceFacts().sm_count;
  const bool few = items * longest <= 4LL * sms * kMoveWarps * kRowsInFlight;
  const int rows = few ? kRowsInFlight : 32;
  const int64_t most = (longest + kMoveWarps * rows - 1) / (kMoveWarps * rows);
  const int64_t fair = (16LL * sms + items - 1) / items;
  // In place a cluster's round is all that its registers hold. While every item's cluster of at least four CTAs has SMs to itself,
  // 256 rows in the registers of each CTA, so up to 2048 a round; where the items fill the machine several times over, small CTAs, four
  // to an SM, whose rounds overlap (one sequence of 32768 tokens to 8192: 36.0 us wide, 46.9 small; 5 x 4 items of 16000-32768 to 4099,
  // clusters of four: 42.3 against 50.0; 64 sequences to 2048 stay small: 52.6). And no more CTAs than one round of the longest
  // item fills (57 x 8 items to 12 tokens: 26.4 us, in clusters of eight 39.4). (Both sides from when the move released its
  // dependents at its start; the forms chosen now take 36.4, 42.8, 54.6 and 27.1 us, one launch behind the other.)
  int cluster_size = kCluster;
  while (cluster_size > 4 && items * cluster_size > sms) cluster_size /= 2;
  const bool wide = in_place && items * cluster_size <= sms;
  if (!wide) cluster_size = kCluster;
  const int64_t cta_rows = (wide ? kWideWarps : kMoveWarps) * (head_dim != 128 ? 1 : wide ? kWideRows : kRowsInFlight);
  while (cluster_size > 1 && cta_rows * (cluster_size / 2) >= longest) cluster_size /= 2;
  const int parts = in_place ? cluster_size : static_cast<int>(most < fair ? most : fair);
  auto kernel = head_dim == 128
                    ? (wide ? MoveKernel<true, 32, kWideRows, kWideWarps> : in_place ? MoveKernel<true, 32, kRowsInFlight, kMoveWarps>
                       : few ? MoveKernel<false, 32, kRowsInFlight, kMoveWarps> : MoveKernel<false, 32, 32, kMoveWarps>)
                    : (wide ? MoveKernel<true, 0, 0, kWideWarps> : in_place ? MoveKernel<true, 0, 0, kMoveWarps>
                       : few ? MoveKernel<false, 0, kRowsInFlight, kMoveWarps> : MoveKernel<false, 0, 32, kMoveWarps>);
  e = LaunchDependent(kernel, dim3(static_cast<unsigned>(num_seqs) * parts, num_kv_heads), dim3(wide ? kWideWarps * 32 : kMoveThreads), 0,
                      in_place ? parts : 1, s, p, parts);
  if (e != cudaSuccess) return Fail(static_cast<int>(e), "%s (move): %s", fn, cudaGetErrorString(e));
  return LaunchStatus(fn);
}
