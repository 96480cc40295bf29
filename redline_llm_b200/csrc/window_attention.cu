// Attention over a bounded part of the paged cache, for sm_100a (B200): a query at position p of its sequence sees
// the first `sinks` tokens and the last `window` tokens up to and including p,
//   V(p) = { t <= p : t < sinks or t > p - window },   out = sum_V softmax(q.k * scale) v,
// for one new token per sequence (decode) and for the rows of a prompt chunk; and decode attention that also adds
// up, per cached token and KV head, the probability the token received from the query heads of its group.
#include "common.cuh"

namespace rl {
namespace wattn {

constexpr int kHeadDim = 128;
constexpr int kMaxGroup = 8;        // query heads per KV head
constexpr int kMaxKvHeads = 8;
constexpr int kMaxBlocks = 1 << 26; // token positions stay inside 31 bits

struct Params {
  half* out;
  int64_t out_stride;
  const half* q;
  int64_t q_stride;
  const half* pool;
  const int32_t* tables;
  const int32_t* seq_lens;  // null: the rows of one prompt chunk, row i at position chunk_start + i
  int chunk_start;
  int rows;
  int max_blocks;
  int kv_heads;
  int group;
  float scale_log2e;
  int window;
  int sinks;
  float* weights;
  float* stats;  // [rows][q_heads][2]: log2-domain maximum, 1 / sum
};

__device__ __forceinline__ const half* TokenRow(const Params& p, const int32_t* table, int t, int kv, int head) {
  const int64_t block = table[t >> kKvBlockShift];
  return p.pool + (((block * 2 + kv) * p.kv_heads + head) * kKvBlock + (t & (kKvBlock - 1))) * kHeadDim;
}

__device__ __forceinline__ float Dot(const float (&qv)[4], const half* k, int lane) {
  const uint2 raw = *reinterpret_cast<const uint2*>(k + lane * 4);
  const float2 a = __half22float2(AsHalf2(raw.x)), b = __half22float2(AsHalf2(raw.y));
  float dot = qv[0] * a.x + qv[1] * a.y + qv[2] * b.x + qv[3] * b.y;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, off);
  return dot;
}

// One warp per (row, query head): online softmax over the visible tokens.
__global__ void __launch_bounds__(32) RowsKernel(const Params p) {
  const int row = blockIdx.x, qh = blockIdx.y, lane = threadIdx.x, head = qh / p.group;
  const int len = p.seq_lens ? min(p.seq_lens[row], p.max_blocks * kKvBlock) : p.chunk_start + row + 1;
  if (len <= 0) return;
  const int32_t* table = p.tables + (p.seq_lens ? static_cast<int64_t>(row) * p.max_blocks : 0);
  float qv[4];
  for (int i = 0; i < 4; ++i) qv[i] = __half2float(p.q[row * p.q_stride + qh * kHeadDim + lane * 4 + i]);
  const int w0 = max(0, len - p.window), s1 = min(p.sinks, w0);
  float m = -INFINITY, l = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int i = 0; i < s1 + len - w0; ++i) {
    const int t = i < s1 ? i : i - s1 + w0;
    const float s = Dot(qv, TokenRow(p, table, t, 0, head), lane) * p.scale_log2e;
    const float n = fmaxf(m, s), keep = exp2f(m - n), e = exp2f(s - n);
    const half* v = TokenRow(p, table, t, 1, head) + lane * 4;
    m = n;
    l = l * keep + e;
    for (int d = 0; d < 4; ++d) acc[d] = fmaf(e, __half2float(v[d]), acc[d] * keep);
  }
  for (int d = 0; d < 4; ++d) p.out[row * p.out_stride + qh * kHeadDim + lane * 4 + d] = __float2half_rn(acc[d] / l);
  if (p.stats && lane == 0) {
    float* st = p.stats + (static_cast<int64_t>(row) * gridDim.y + qh) * 2;
    st[0] = m;
    st[1] = 1.0f / l;
  }
}

// One warp per (sequence, KV head, page): the probabilities of the group's heads, summed per token.
__global__ void __launch_bounds__(32) WeightsKernel(const Params p) {
  const int seq = blockIdx.x, head = blockIdx.y, lane = threadIdx.x;
  const int len = min(p.seq_lens[seq], p.max_blocks * kKvBlock);
  const int32_t* table = p.tables + static_cast<int64_t>(seq) * p.max_blocks;
  for (int t = blockIdx.z; t < len; t += gridDim.z) {
    float sum = 0.0f;
    for (int g = 0; g < p.group; ++g) {
      const int qh = head * p.group + g;
      float qv[4];
      for (int i = 0; i < 4; ++i) qv[i] = __half2float(p.q[seq * p.q_stride + qh * kHeadDim + lane * 4 + i]);
      const float* st = p.stats + (static_cast<int64_t>(seq) * p.kv_heads * p.group + qh) * 2;
      sum += exp2f(Dot(qv, TokenRow(p, table, t, 0, head), lane) * p.scale_log2e - st[0]) * st[1];
    }
    if (lane == 0) {
      float* w = p.weights + (static_cast<int64_t>(table[t >> kKvBlockShift]) * p.kv_heads + head) * kKvBlock + (t & (kKvBlock - 1));
      *w = t == len - 1 ? sum : *w + sum;
    }
  }
}

// ----------------------------------------------------------- host side

size_t StatsBytes(int num_seqs, int q_heads) { return static_cast<size_t>(num_seqs) * q_heads * 2 * sizeof(float); }

int CheckCommon(const char* fn, const void* out, int64_t out_stride, const void* q, int64_t q_stride, const void* pool,
                const void* tables, int max_blocks, int q_heads, int kv_heads, int head_dim, float scale) {
  if (!out || !q || !pool || !tables) return Fail(RL_E_NULL_POINTER, "%s: null device pointer", fn);
  if (head_dim != kHeadDim) return Fail(RL_E_BAD_SHAPE, "%s: head_dim must be 128", fn);
  if (kv_heads < 1 || kv_heads > kMaxKvHeads || q_heads < kv_heads || q_heads % kv_heads != 0 ||
      q_heads / kv_heads > kMaxGroup)
    return Fail(RL_E_BAD_SHAPE, "%s: 1 to 8 KV heads with 1 to 8 query heads each", fn);
  if (max_blocks < 1) return Fail(RL_E_BAD_SHAPE, "%s: max_blocks_per_seq must be >= 1", fn);
  if (max_blocks > kMaxBlocks) return Fail(RL_E_TOO_LARGE, "%s: at most 2^26 blocks per sequence", fn);
  const int64_t width = static_cast<int64_t>(q_heads) * head_dim;
  if (q_stride < width || out_stride < width) return Fail(RL_E_BAD_SHAPE, "%s: row stride smaller than the row", fn);
  if (!(scale > 0.0f) || !(scale * 1.4426950408889634f <= 3.402823466e38f))
    return Fail(RL_E_BAD_SHAPE, "%s: scale must be positive and finite", fn);
  if (!Aligned16(pool)) return Fail(RL_E_BAD_SHAPE, "%s: the pool slice must be 16-byte aligned", fn);
  return RL_OK;
}

int CheckWindow(const char* fn, int window, int sinks) {
  if (window < 1 || sinks < 0) return Fail(RL_E_BAD_SHAPE, "%s: window >= 1 and sinks >= 0", fn);
  return RL_OK;
}

int CheckDecode(const char* fn, const void* q, int64_t q_stride, const void* lens, const void* workspace,
                size_t have, size_t need) {
  if (!lens || !workspace) return Fail(RL_E_NULL_POINTER, "%s: null device pointer", fn);
  if ((q_stride & 1) || (reinterpret_cast<uintptr_t>(q) & 3))
    return Fail(RL_E_BAD_SHAPE, "%s: q rows must be 4-byte aligned", fn);
  if (!Aligned16(workspace)) return Fail(RL_E_BAD_SHAPE, "%s: the workspace must be 16-byte aligned", fn);
  if (have < need) return Fail(RL_E_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", fn, have, need);
  return RL_OK;
}

size_t DecodeWorkspace(int num_seqs, int max_blocks, int q_heads, int kv_heads, bool weights) {
  (void)max_blocks, (void)kv_heads, (void)weights;
  return StatsBytes(num_seqs, q_heads) + 256;
}

}  // namespace wattn
}  // namespace rl

extern "C" int rl_window_attention_workspace_bytes(int32_t num_seqs, int32_t max_blocks_per_seq, int32_t num_q_heads,
                                                   int32_t num_kv_heads, int32_t weights, size_t* bytes_out) {
  using namespace rl;
  using namespace rl::wattn;
  if (!bytes_out) return Fail(RL_E_NULL_POINTER, "window_attention_workspace_bytes: null pointer");
  *bytes_out = 0;
  if (num_seqs < 0 || max_blocks_per_seq < 1 || max_blocks_per_seq > kMaxBlocks || num_kv_heads < 1 ||
      num_kv_heads > kMaxKvHeads || num_q_heads < num_kv_heads || num_q_heads % num_kv_heads != 0 ||
      num_q_heads / num_kv_heads > kMaxGroup)
    return Fail(RL_E_BAD_SHAPE, "window_attention_workspace_bytes: not a shape the launchers take");
  *bytes_out = DecodeWorkspace(num_seqs, max_blocks_per_seq, num_q_heads, num_kv_heads, weights != 0);
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
  using namespace rl;
  using namespace rl::wattn;
  constexpr const char* fn = "paged_window_attention_decode";
  if (num_seqs <= 0) return RL_OK;
  int rc = CheckCommon(fn, out, out_row_stride, q, q_row_stride, kv_pool_layer, block_tables, max_blocks_per_seq,
                       num_q_heads, num_kv_heads, head_dim, scale);
  if (rc == RL_OK) rc = CheckWindow(fn, window, sinks);
  if (rc == RL_OK)
    rc = CheckDecode(fn, q, q_row_stride, seq_lens, workspace, workspace_bytes,
                     DecodeWorkspace(num_seqs, max_blocks_per_seq, num_q_heads, num_kv_heads, false));
  if (rc != RL_OK) return rc;
  Params p = {};
  p.out = static_cast<half*>(out);
  p.out_stride = out_row_stride;
  p.q = static_cast<const half*>(q);
  p.q_stride = q_row_stride;
  p.pool = static_cast<const half*>(kv_pool_layer);
  p.tables = block_tables;
  p.seq_lens = seq_lens;
  p.max_blocks = max_blocks_per_seq;
  p.kv_heads = num_kv_heads;
  p.group = num_q_heads / num_kv_heads;
  p.scale_log2e = scale * 1.4426950408889634f;
  p.window = window;
  p.sinks = sinks;
  RowsKernel<<<dim3(num_seqs, num_q_heads), 32, 0, static_cast<cudaStream_t>(stream)>>>(p);
  return LaunchStatus(fn);
}

extern "C" int rl_launch_paged_attention_decode_weights(void* out, int64_t out_row_stride, const void* q,
                                                        int64_t q_row_stride, const void* kv_pool_layer,
                                                        const int32_t* block_tables, const int32_t* seq_lens,
                                                        int32_t num_seqs, int32_t max_blocks_per_seq,
                                                        int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                                                        float scale, float* weights, void* workspace,
                                                        size_t workspace_bytes, void* stream) {
  using namespace rl;
  using namespace rl::wattn;
  constexpr const char* fn = "paged_attention_decode_weights";
  if (num_seqs <= 0) return RL_OK;
  int rc = CheckCommon(fn, out, out_row_stride, q, q_row_stride, kv_pool_layer, block_tables, max_blocks_per_seq,
                       num_q_heads, num_kv_heads, head_dim, scale);
  if (rc == RL_OK && !weights) rc = Fail(RL_E_NULL_POINTER, "%s: null device pointer", fn);
  if (rc == RL_OK && (reinterpret_cast<uintptr_t>(weights) & 3))
    rc = Fail(RL_E_BAD_SHAPE, "%s: the weights must be 4-byte aligned", fn);
  if (rc == RL_OK)
    rc = CheckDecode(fn, q, q_row_stride, seq_lens, workspace, workspace_bytes,
                     DecodeWorkspace(num_seqs, max_blocks_per_seq, num_q_heads, num_kv_heads, true));
  if (rc != RL_OK) return rc;
  Params p = {};
  p.out = static_cast<half*>(out);
  p.out_stride = out_row_stride;
  p.q = static_cast<const half*>(q);
  p.q_stride = q_row_stride;
  p.pool = static_cast<const half*>(kv_pool_layer);
  p.tables = block_tables;
  p.seq_lens = seq_lens;
  p.max_blocks = max_blocks_per_seq;
  p.kv_heads = num_kv_heads;
  p.group = num_q_heads / num_kv_heads;
  p.scale_log2e = scale * 1.4426950408889634f;
  p.window = INT32_MAX;
  p.weights = weights;
  p.stats = reinterpret_cast<float*>(static_cast<char*>(workspace) + 256);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  RowsKernel<<<dim3(num_seqs, num_q_heads), 32, 0, s>>>(p);
  WeightsKernel<<<dim3(num_seqs, num_kv_heads, 64), 32, 0, s>>>(p);
  return LaunchStatus(fn);
}
