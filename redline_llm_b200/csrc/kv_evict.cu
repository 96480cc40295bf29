// Eviction from the paged cache by accumulated attention weight, for sm_100a (B200). Per sequence and KV head: a
// cache of L tokens shrinks to L' = min(L, budget); the first `sinks` and the last `recent` tokens stay, and of the
// rest the budget - sinks - recent with the largest weight (equal weights: the lower position stays first; a NaN
// counts below every number). Kept tokens move, in cache order, to slots 0 .. L'-1 of the destination table's pages,
// K row, V row and weight together.
//
// Two kernels. What bounds them: the selection is a chain of short dependent passes (latency), the move is a copy of
// the kept rows (HBM).
//  * Select, one CTA per (sequence, KV head): weights become integers that compare the same way and stay in shared
//    memory; a radix select of three digits (11, 11, 10 bits) finds the weight of the last kept token - a histogram per
//    digit, its suffix sums over the block, and on to the digit below among the keys that share the prefix; then one
//    ordered sweep writes the kept positions, each warp a stretch of the sequence, ballots giving the ranks.
//  * Move, 32 rows per warp: a lane looks up one row's source and destination, then the warp copies the rows 16 bytes a
//    lane, sixteen rows in flight. In place a cluster of eight CTAs walks a (sequence, head) in cache order, every row of a round
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

constexpr int kSelectThreads = 1024;
constexpr int kSelectWarps = kSelectThreads / 32;
constexpr int kBins = 2048;
constexpr int kMaxCachedKeys = 48 * 1024;   // 192 KB

__global__ void __launch_bounds__(kSelectThreads) SelectKernel(const Params p) {
  extern __shared__ __align__(16) uint32_t keys[];
  __shared__ int bins[kBins];
  __shared__ int warp_sum[kSelectWarps], warp_equal[kSelectWarps];
  __shared__ int found_bin, found_above, found_count;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int seq = blockIdx.x, head = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int len = CachedTokens(p, seq);
  const int n = min(len, p.budget);
  const int32_t* table = p.tables + static_cast<int64_t>(seq) * p.max_blocks;
  int32_t* kept = p.kept + (static_cast<int64_t>(seq) * p.kv_heads + head) * p.budget;
  for (int j = n + tid; j < p.budget; j += kSelectThreads) kept[j] = -1;
  if (len <= p.budget) {
    for (int j = tid; j < n; j += kSelectThreads) kept[j] = j;
    return;
  }
  // candidates are tokens [a, b); their keys are handled four at a time from a4 on (four neighbours share a page)
  const int a = p.sinks, b = len - p.recent, a4 = a & ~3;
  const int quads = (b - a4 + 3) >> 2;
  const bool cached = quads * 4 <= p.cached_keys;
  auto load_quad = [&](int i) {
    const int t = a4 + 4 * i;
    const int64_t block = table[t >> kKvBlockShift];
    const float4 w = *reinterpret_cast<const float4*>(p.weights + (block * p.kv_heads + head) * kKvBlock + (t & (kKvBlock - 1)));
    return make_uint4(OrderKey(w.x), OrderKey(w.y), OrderKey(w.z), OrderKey(w.w));
  };
  auto quad = [&](int i) { return cached ? reinterpret_cast<const uint4*>(keys)[i] : load_quad(i); };
  auto clear_bins = [&]() {
    for (int i = tid; i < kBins; i += kSelectThreads) bins[i] = 0;
  };
  // every candidate key of this thread's quads
  auto for_each = [&](auto&& quad_of, auto&& use) {
#pragma unroll 4
    for (int i = tid; i < quads; i += kSelectThreads) {
      const uint4 k = quad_of(i);
      const int t = a4 + 4 * i;
      if (t >= a && t < b) use(k.x);
      if (t + 1 >= a && t + 1 < b) use(k.y);
      if (t + 2 >= a && t + 2 < b) use(k.z);
      if (t + 3 >= a && t + 3 < b) use(k.w);
    }
  };

  // thr: tokens with a larger key stay, and the first `ties` of those whose key equals it
  uint32_t thr = 0xFFFFFFFFu;   // no weight has this key
  int ties = 0;
  int need = p.budget - p.sinks - p.recent;
  if (need > 0) {
    clear_bins();
    __syncthreads();
    for_each([&](int i) {
      const uint4 k = load_quad(i);
      if (cached) reinterpret_cast<uint4*>(keys)[i] = k;
      return k;
    }, [&](uint32_t k) { atomicAdd(&bins[k >> 21], 1); });
    uint32_t prefix = 0;
    int shift = 21;   // of the digit in hand; the digits above it equal `prefix`
#pragma unroll 1
    while (true) {
      __syncthreads();
      // the bin that holds the need-th largest key: thread i sums bins 2047 - 2i and 2046 - 2i, from the top down
      const int hi = bins[kBins - 1 - 2 * tid], lo = bins[kBins - 2 - 2 * tid];
      int incl = hi + lo;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl += v;
      }
      if (lane == 31) warp_sum[warp] = incl;
      __syncthreads();
      int before = warp_sum[lane];   // lane w: the sum of warp w's bins
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, before, off);
        if (lane >= off) before += v;
      }
      const int passed = __shfl_sync(0xffffffffu, before, warp > 0 ? warp - 1 : 0);
      const int above = (warp > 0 ? passed : 0) + incl - hi - lo;
      if (above < need && above + hi + lo >= need) {
        const bool upper = above + hi >= need;
        found_bin = kBins - 1 - 2 * tid - (upper ? 0 : 1);
        found_above = above + (upper ? 0 : hi);
        found_count = upper ? hi : lo;
      }
      __syncthreads();
      need -= found_above;
      prefix |= static_cast<uint32_t>(found_bin) << shift;
      if (found_count == need) {   // all of this bin stay: whatever is below it does not
        thr = prefix - 1;          // (never below 0: some candidate is left out)
        break;
      }
      if (shift == 0) {
        thr = prefix;
        ties = need;
        break;
      }
      const int above_digit = shift;
      shift = shift == 21 ? 10 : 0;
      const uint32_t digit_mask = shift == 10 ? 0x7FFu : 0x3FFu;
      __syncthreads();
      clear_bins();
      __syncthreads();
      for_each(quad, [&](uint32_t k) {
        if (((k ^ prefix) >> above_digit) == 0) atomicAdd(&bins[(k >> shift) & digit_mask], 1);
      });
    }
  }

  // ---- the kept positions in cache order: each warp a stretch of the sequence
  __syncthreads();
  const int stretch = ((len + kSelectThreads - 1) / kSelectThreads) * 32;
  const int t_begin = min(len, warp * stretch), t_end = min(len, t_begin + stretch);
  auto key_at = [&](int t) -> uint32_t {
    if (cached) return keys[t - a4];
    const int64_t block = table[t >> kKvBlockShift];
    return OrderKey(p.weights[(block * p.kv_heads + head) * kKvBlock + (t & (kKvBlock - 1))]);
  };
  // whether token t stays in any case, and whether it is one of the equals
  auto judge = [&](int t, bool& sure, bool& equal) {
    sure = equal = false;
    if (t < t_end) {
      if (t < a || t >= b) {
        sure = true;
      } else if (thr != 0xFFFFFFFFu) {
        const uint32_t k = key_at(t);
        sure = k > thr;
        equal = k == thr && ties > 0;
      }
    }
  };
  int n_sure = 0, n_equal = 0;
#pragma unroll 4
  for (int t0 = t_begin; t0 < t_end; t0 += 32) {
    bool sure, equal;
    judge(t0 + lane, sure, equal);
    n_sure += __popc(__ballot_sync(0xffffffffu, sure));
    n_equal += __popc(__ballot_sync(0xffffffffu, equal));
  }
  if (lane == 0) {
    warp_sum[warp] = n_sure;
    warp_equal[warp] = n_equal;
  }
  __syncthreads();
  int sure_before = lane < warp ? warp_sum[lane] : 0, equal_before = lane < warp ? warp_equal[lane] : 0;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    sure_before += __shfl_xor_sync(0xffffffffu, sure_before, off);
    equal_before += __shfl_xor_sync(0xffffffffu, equal_before, off);
  }
  const uint32_t below = (1u << lane) - 1u;
  int at = sure_before + min(equal_before, ties);
#pragma unroll 2
  for (int t0 = t_begin; t0 < t_end; t0 += 32) {
    bool sure, equal;
    judge(t0 + lane, sure, equal);
    const uint32_t equals = __ballot_sync(0xffffffffu, equal);
    const bool keep = sure || (equal && equal_before + __popc(equals & below) < ties);
    const uint32_t keeps = __ballot_sync(0xffffffffu, keep);
    if (keep) kept[at + __popc(keeps & below)] = t0 + lane;
    at += __popc(keeps);
    equal_before += __popc(equals);
  }
}

constexpr int kMoveThreads = 256;
constexpr int kMoveWarps = kMoveThreads / 32;
constexpr int kRowsInFlight = 16;
constexpr int kCluster = 8;

// kRowWords: 16-byte words of one token's K row and V row together when it is the same for every lane pattern (head_dim
// 128: 32, one word per lane and row), 0 for any other width.
template <bool kInPlace, int kRowWords>
__global__ void __launch_bounds__(kMoveThreads) MoveKernel(const Params p, int parts) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
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
  constexpr int kRows = !kInPlace ? 32 : kRowWords == 32 ? kRowsInFlight : 1;
  const int round = parts * kMoveWarps * kRows;
  for (int j0 = 0; j0 < n; j0 += round) {
    const int first = j0 + (part * kMoveWarps + warp) * kRows;
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
      for (int r0 = 0; r0 < kRows; r0 += kRowsInFlight) {
        uint4 v[kRowsInFlight];
#pragma unroll
        for (int r = 0; r < kRowsInFlight; ++r) {
          const int64_t src = __shfl_sync(0xffffffffu, from, r0 + r);
          if ((moving >> (r0 + r)) & 1) v[r] = pool[src + mine];
        }
        if (kInPlace) {   // all rows of the round are in registers, over the whole cluster, before any is written
          asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
          asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        }
#pragma unroll
        for (int r = 0; r < kRowsInFlight; ++r) {
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
}

// First use on a device: the selection's shared memory.
constexpr int kMaxDevices = 64;
bool g_ready[kMaxDevices];
std::mutex g_mutex;
int EnsureReady(const char* fn) {
  bool& ready = g_ready[CurrentDeviceIndex()];
  std::lock_guard<std::mutex> lock(g_mutex);
  if (ready) return RL_OK;
  const cudaError_t e = cudaFuncSetAttribute(SelectKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxCachedKeys * 4);
  if (e != cudaSuccess) return Fail(static_cast<int>(e), "%s: shared-memory opt-in: %s", fn, cudaGetErrorString(e));
  ready = true;
  return RL_OK;
}

}  // namespace evict
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
  if (num_seqs > INT32_MAX / kCluster) return Fail(RL_E_TOO_LARGE, "%s: too many sequences", fn);
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
  p.cached_keys = static_cast<int>(tokens < kMaxCachedKeys ? tokens : kMaxCachedKeys);
  const int rc = EnsureReady(fn);
  if (rc != RL_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = LaunchDependent(SelectKernel, dim3(num_seqs, num_kv_heads), dim3(kSelectThreads),
                                  static_cast<size_t>(p.cached_keys) * 4, 1, s, p);
  if (e != cudaSuccess) return Fail(static_cast<int>(e), "%s: %s", fn, cudaGetErrorString(e));
  const bool in_place = dst_block_tables == block_tables;
  const int64_t most = ((tokens < budget ? tokens : budget) + kMoveWarps * 32 - 1) / (kMoveWarps * 32);
  const int64_t items = static_cast<int64_t>(num_seqs) * num_kv_heads;
  const int64_t fair = (16LL * CurrentDeviceFacts().sm_count + items - 1) / items;
  const int parts = in_place ? kCluster : static_cast<int>(most < fair ? most : fair);
  const bool plain = head_dim == 128;
  auto kernel = in_place ? (plain ? MoveKernel<true, 32> : MoveKernel<true, 0>) : (plain ? MoveKernel<false, 32> : MoveKernel<false, 0>);
  e = LaunchDependent(kernel, dim3(static_cast<unsigned>(num_seqs) * parts, num_kv_heads), dim3(kMoveThreads), 0,
                      in_place ? kCluster : 1, s, p, parts);
  if (e != cudaSuccess) return Fail(static_cast<int>(e), "%s (move): %s", fn, cudaGetErrorString(e));
  return LaunchStatus(fn);
}
