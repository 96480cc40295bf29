// Eviction from the paged cache by accumulated attention weight, for sm_100a (B200). Per sequence and KV head: a
// cache of L tokens shrinks to L' = min(L, budget); the first `sinks` and the last `recent` tokens stay, and of the
// rest the budget - sinks - recent with the largest weight (equal weights: the lower position stays first; a NaN
// counts below every number). Kept tokens move, in cache order, to slots 0 .. L'-1 of the destination table's pages,
// K row, V row and weight together.
//
// Two kernels: the first finds the kept positions, the second moves the rows.
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
};

// Weights as unsigned integers that compare the same way: 0 for a NaN, -0 like +0.
__device__ __forceinline__ uint32_t OrderKey(float w) {
  if (w != w) return 0u;
  const uint32_t b = __float_as_uint(w + 0.0f);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

constexpr int kThreads = 256;

__device__ __forceinline__ int BlockSum(int v, int* scratch) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  int sum = 0;
  for (int w = 0; w < kThreads / 32; ++w) sum += scratch[w];
  __syncthreads();
  return sum;
}

// One CTA per (sequence, KV head): the threshold by bisection over the key's bits, then an ordered sweep.
__global__ void __launch_bounds__(kThreads) SelectKernel(const Params p) {
  __shared__ int scratch[kThreads / 32];
  const int seq = blockIdx.x, head = blockIdx.y, tid = threadIdx.x;
  const int len = max(0, min(p.seq_lens[seq], p.max_blocks * kKvBlock));
  const int n = min(len, p.budget);
  const int32_t* table = p.tables + static_cast<int64_t>(seq) * p.max_blocks;
  int32_t* kept = p.kept + (static_cast<int64_t>(seq) * p.kv_heads + head) * p.budget;
  for (int j = n + tid; j < p.budget; j += kThreads) kept[j] = -1;
  if (len <= p.budget) {
    for (int j = tid; j < n; j += kThreads) kept[j] = j;
    return;
  }
  const int a = p.sinks, b = len - p.recent, need = p.budget - p.sinks - p.recent;
  auto key = [&](int t) {
    const int64_t block = table[t >> kKvBlockShift];
    return OrderKey(p.weights[(block * p.kv_heads + head) * kKvBlock + (t & (kKvBlock - 1))]);
  };
  uint32_t thr = 0;   // the largest key that at least `need` candidates reach
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t probe = thr | (1u << bit);
    int c = 0;
    for (int t = a + tid; t < b; t += kThreads) c += key(t) >= probe;
    if (BlockSum(c, scratch) >= need && need > 0) thr = probe;
  }
  int above = 0;
  for (int t = a + tid; t < b; t += kThreads) above += key(t) > thr;
  int ties = need - BlockSum(above, scratch);   // how many of the keys equal to the threshold stay
  int at = 0;
  if (tid == 0) {
    for (int t = 0; t < len; ++t) {
      bool keep = t < a || t >= b;
      if (!keep) {
        const uint32_t k = key(t);
        keep = need > 0 && k > thr;
        if (!keep && need > 0 && k == thr && ties > 0) {
          keep = true;
          --ties;
        }
      }
      if (keep) kept[at++] = t;
    }
  }
}

// One CTA per (sequence, KV head), 16 rows at a time in cache order: all of them are read before any is written, so
// source and destination may be the same pages (a row never moves to a higher slot than its own).
__global__ void __launch_bounds__(kThreads) MoveKernel(const Params p) {
  const int seq = blockIdx.x, head = blockIdx.y, tid = threadIdx.x;
  const int len = max(0, min(p.seq_lens[seq], p.max_blocks * kKvBlock));
  const int n = min(len, p.budget);
  const int32_t* table = p.tables + static_cast<int64_t>(seq) * p.max_blocks;
  const int32_t* dst = p.dst_tables + static_cast<int64_t>(seq) * p.dst_max_blocks;
  const int32_t* kept = p.kept + (static_cast<int64_t>(seq) * p.kv_heads + head) * p.budget;
  const int words = p.head_dim / 8;
  auto row = [&](int64_t block, int kv, int t) {
    return p.pool + (((block * 2 + kv) * p.kv_heads + head) * kKvBlock + (t & (kKvBlock - 1))) * p.head_dim;
  };
  for (int j = 0; j < n; ++j) {
    const int t = kept[j];
    const int64_t from = table[t >> kKvBlockShift], to = dst[j >> kKvBlockShift];
    uint4 v[2];
    float w = 0.0f;
    for (int kv = 0; kv < 2; ++kv)
      if (tid < words) v[kv] = Ldg16(row(from, kv, t) + tid * 8);
    if (tid == 0) w = p.weights[(from * p.kv_heads + head) * kKvBlock + (t & (kKvBlock - 1))];
    __syncthreads();
    for (int kv = 0; kv < 2; ++kv)
      if (tid < words) Stg16(row(to, kv, j) + tid * 8, v[kv]);
    if (tid == 0) p.weights[(to * p.kv_heads + head) * kKvBlock + (j & (kKvBlock - 1))] = w;
    __syncthreads();
  }
}

__global__ void LensKernel(const Params p, int num_seqs) {
  const int s = blockIdx.x * blockDim.x + threadIdx.x;
  if (s < num_seqs) p.new_lens[s] = min(max(0, min(p.seq_lens[s], p.max_blocks * kKvBlock)), p.budget);
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
  if (!Aligned16(kv_pool_layer) || (reinterpret_cast<uintptr_t>(weights) & 3))
    return Fail(RL_E_BAD_SHAPE, "%s: the pool slice must be 16-byte, the weights 4-byte aligned", fn);
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
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  SelectKernel<<<dim3(num_seqs, num_kv_heads), kThreads, 0, s>>>(p);
  MoveKernel<<<dim3(num_seqs, num_kv_heads), kThreads, 0, s>>>(p);
  LensKernel<<<(num_seqs + 255) / 256, 256, 0, s>>>(p, num_seqs);
  return LaunchStatus(fn);
}
