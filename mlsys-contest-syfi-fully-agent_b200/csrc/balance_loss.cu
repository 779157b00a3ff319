// Balance loss of a routing, per sequence, with per-expert counts, and its gradient for the router's logits.
//
// s = sigmoid(z) or exp(z), p_ti = s_ti / sum_j s_tj.  For a sequence with n counted tokens whose K selections are
// topk_idx, c_i = selections of expert i:
//     loss = alpha E / (K n^2) sum_i c_i sum_t p_ti
// (the mean over the tokens of p, times the frequencies E c_i / (K n), times alpha), and with the counts held constant
//     dloss/dz_ti = alpha E / (K n^2) d_ti (c_i - sum_j c_j p_tj),    d = p (1 - s) for sigmoid, p for softmax.
// A row whose scores are all zero (every logit -inf) has p = 0 and no gradient.
//
// One warp takes a token: lane l holds experts l, l + 32, ...  The token axis is cut into equal chunks, one CTA each; a
// CTA walks through the sequences that meet its chunk.  What lies inside the chunk is finished there; a sequence that
// crosses a border leaves one partial row per chunk, which balance_join_kernel adds in chunk order (no floating-point
// atomics: the same bits every time).  Counts are integers.
#include "elem_device.cuh"

namespace moe {
namespace {

constexpr int kMaxExperts = 1024;
constexpr int kChunkWarps = 8;
constexpr int kMinChunk = 32;          // tokens; smaller batches stay in one CTA, which needs no second launch
constexpr int kMaxChunks = 4 * kNumSMs;

struct BalanceArgs {
  const void* logits;
  int64_t stride;                      // elements between rows
  const int* topk_idx;                 // [T, K]
  const int* cu;                       // [S + 1] or null: one sequence of T tokens
  const uint8_t* mask;                 // [T] or null
  int T, E, K, S, softmax;
  int chunk, n_chunks;
  float alpha;
  float* loss;                         // [S]
  int *counts, *tokens;                // [S, E], [S]
  // partial results of sequences that cross a chunk border: slot 0 = began before the chunk, 1 = goes on after it
  float* part_p;                       // [n_chunks][2][E]
  int *part_c, *part_n;                // [n_chunks][2][E], [n_chunks][2]
  int* tail;                           // [n_chunks] sequence that begins in the chunk and goes on after it, or -1
  // backward
  const float* grad_loss;              // [S]
  void* grad;                          // [T, E]
};

// Border i of the packed sequences, whatever the caller's array holds inside the batch.
__device__ __forceinline__ int border(const BalanceArgs& a, int i) {
  if (!a.cu) return i == 0 ? 0 : a.T;
  return min(max(__ldg(a.cu + i), 0), a.T);
}

// Number of sequences that begin before token t (borders ascend), by a 32-way search of the calling warp.
__device__ __forceinline__ int begun_before(const BalanceArgs& a, int t, int lane) {
  int lo = 0, hi = a.S;
  while (lo < hi) {
    const int step = (hi - lo + 31) / 32;
    const int i = lo + lane * step;
    const int k = __popc(__ballot_sync(0xFFFFFFFFu, i < hi && border(a, i) < t));
    if (k == 0) return lo;
    hi = min(hi, lo + k * step);
    lo += (k - 1) * step + 1;
  }
  return lo;
}

// Probabilities of a row, zero where the row has none, and in s what the slope dp/dz needs beside them: 1 - sigmoid(z)
// (1 for a softmax), formed as e^-z sigmoid(z) where 1 - sigmoid(z) would cancel.
template <typename T, int EPL>
__device__ __forceinline__ void probabilities(const BalanceArgs& a, int t, int lane, float (&s)[EPL], float (&p)[EPL]) {
  const T* row = static_cast<const T*>(a.logits) + t * a.stride;
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int e = i * 32 + lane;
    s[i] = e < a.E ? to_f32<T>(row[e]) : -INFINITY;
    top = s[i] > top || s[i] != s[i] ? s[i] : top;       // a NaN stays
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    const float o = __shfl_xor_sync(0xFFFFFFFFu, top, d);
    top = o > top || o != o ? o : top;
  }
  float sum = 0.0f;
  // sigmoid(z) is e^z to fp32 below -60, and would lose its bits below -87: such a row is shifted like a softmax's
  const bool shifted = a.softmax || top < -60.0f;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const float z = s[i];
    const float x = expf(shifted ? z - top : -z);
    p[i] = shifted ? (z == -INFINITY ? 0.0f : x) : 1.0f / (1.0f + x);
    s[i] = shifted ? 1.0f : z > 0.0f ? x * p[i] : 1.0f - p[i];
    sum += p[i];
  }
  sum = warp_sum(sum);
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
  for (int i = 0; i < EPL; ++i) p[i] *= inv;
}

template <typename T, int EPL>
__global__ void __launch_bounds__(32 * kChunkWarps) balance_chunk_kernel(BalanceArgs a) {
  griddep_launch_dependents();
  griddep_wait();
  extern __shared__ float sh[];
  float* sums = sh;                                              // [kChunkWarps][EPL * 32]
  int* hist = reinterpret_cast<int*>(sh + kChunkWarps * EPL * 32);  // [EPL * 32]
  __shared__ float red[32];
  __shared__ int n_valid;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x;
  const int t0 = c * a.chunk, t1 = min(a.T, t0 + a.chunk);
  const bool last = c == a.n_chunks - 1;
  const int first = begun_before(a, t0, lane);
  const int end = last ? a.S : begun_before(a, t1, lane);
  int tail = -1;
  for (int q = first > 0 ? first - 1 : 0; q < end; ++q) {
    const int b0 = border(a, q), b1 = max(border(a, q + 1), b0);
    const bool head = q < first;
    if (head && b1 <= t0) continue;
    const int lo = max(b0, t0), hi = min(b1, t1);
    for (int e = threadIdx.x; e < a.E; e += blockDim.x) hist[e] = 0;
    if (threadIdx.x == 0) n_valid = 0;
    __syncthreads();
    float acc[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) acc[i] = 0.0f;
    int n = 0;
    for (int t = lo + w; t < hi; t += kChunkWarps) {
      if (a.mask && !a.mask[t]) continue;
      float s[EPL], p[EPL];
      probabilities<T, EPL>(a, t, lane, s, p);
#pragma unroll
      for (int i = 0; i < EPL; ++i) acc[i] += p[i];
      for (int k = lane; k < a.K; k += 32) {
        const int e = a.topk_idx[static_cast<int64_t>(t) * a.K + k];
        if (e >= 0 && e < a.E) atomicAdd(hist + e, 1);
      }
      ++n;
    }
#pragma unroll
    for (int i = 0; i < EPL; ++i) sums[(w * EPL + i) * 32 + lane] = acc[i];
    if (lane == 0) atomicAdd(&n_valid, n);
    __syncthreads();
    const bool whole = !head && b1 <= t1;
    const int slot = c * 2 + (head ? 0 : 1);
    float dot[1] = {0.0f};
    for (int e = threadIdx.x; e < a.E; e += blockDim.x) {
      float p = 0.0f;
#pragma unroll
      for (int v = 0; v < kChunkWarps; ++v) p += sums[v * EPL * 32 + e];
      if (whole) {
        a.counts[static_cast<int64_t>(q) * a.E + e] = hist[e];
        dot[0] += static_cast<float>(hist[e]) * p;
      } else {
        a.part_p[static_cast<int64_t>(slot) * a.E + e] = p;
        a.part_c[static_cast<int64_t>(slot) * a.E + e] = hist[e];
      }
    }
    if (whole) block_sum(dot, red);
    if (threadIdx.x == 0) {
      const float n_all = static_cast<float>(n_valid);
      if (whole) {
        a.tokens[q] = n_valid;
        a.loss[q] = n_valid ? a.alpha * a.E / a.K * (dot[0] / n_all / n_all) : 0.0f;
      } else {
        a.part_n[slot] = n_valid;
      }
    }
    if (!head && b1 > t1) tail = q;
    __syncthreads();
  }
  if (threadIdx.x == 0) a.tail[c] = tail;
}

// CTA c finishes the sequence that begins in chunk c and goes on after it, if there is one.
__global__ void __launch_bounds__(1024) balance_join_kernel(BalanceArgs a) {
  griddep_launch_dependents();
  griddep_wait();
  __shared__ float red[32];
  const int c = blockIdx.x, q = a.tail[c];
  if (q < 0) return;
  const int last = (max(border(a, q + 1), 1) - 1) / a.chunk;
  float dot[1] = {0.0f};
  for (int e = threadIdx.x; e < a.E; e += blockDim.x) {
    float p = a.part_p[static_cast<int64_t>(2 * c + 1) * a.E + e];
    int n = a.part_c[static_cast<int64_t>(2 * c + 1) * a.E + e];
#pragma unroll 4
    for (int k = c + 1; k <= last; ++k) {
      p += a.part_p[static_cast<int64_t>(2 * k) * a.E + e];
      n += a.part_c[static_cast<int64_t>(2 * k) * a.E + e];
    }
    a.counts[static_cast<int64_t>(q) * a.E + e] = n;
    dot[0] += static_cast<float>(n) * p;
  }
  block_sum(dot, red);
  if (threadIdx.x == 0) {
    int n = a.part_n[2 * c + 1];
    for (int k = c + 1; k <= last; ++k) n += a.part_n[2 * k];
    a.tokens[q] = n;
    a.loss[q] = n ? a.alpha * a.E / a.K * (dot[0] / n / n) : 0.0f;
  }
}

// One warp per token.  The counts enter less their mean K n / E (rounded: an exact integer difference), which leaves the
// gradient as it is, because sum p = 1, and keeps its difference from cancelling when the counts are nearly even.
template <typename T, int EPL>
__global__ void __launch_bounds__(32 * kChunkWarps) balance_backward_kernel(BalanceArgs a) {
  griddep_launch_dependents();
  griddep_wait();
  const int lane = threadIdx.x & 31;
  const int warps = gridDim.x * kChunkWarps, warp = blockIdx.x * kChunkWarps + (threadIdx.x >> 5);
  const int per = (a.T + warps - 1) / warps;
  const int t0 = warp * per, t1 = min(a.T, t0 + per);
  int q = -1, b0 = 0, b1 = -1;       // sequence of the counts in registers and its borders
  float c[EPL], factor = 0.0f;
  for (int t = t0; t < t1; ++t) {
    if (t < b0 || t >= b1) {
      q = begun_before(a, t + 1, lane) - 1;
      b0 = b1 = 0;
      if (q >= 0) {
        b0 = border(a, q);
        b1 = border(a, q + 1);
      }
      if (t >= b0 && t < b1) {
        const int n = max(a.tokens[q], 1);
        const int mean = static_cast<int>(static_cast<int64_t>(a.K) * n / a.E);
        factor = a.grad_loss[q] * (a.alpha * a.E / a.K) / n / n;
#pragma unroll
        for (int i = 0; i < EPL; ++i) {
          const int e = i * 32 + lane;
          c[i] = e < a.E ? static_cast<float>(a.counts[static_cast<int64_t>(q) * a.E + e] - mean) : 0.0f;
        }
      }
    }
    T* out = static_cast<T*>(a.grad) + static_cast<int64_t>(t) * a.E;
    const bool live = t >= b0 && t < b1 && !(a.mask && !a.mask[t]);
    float s[EPL], p[EPL];
    float dot = 0.0f;
    if (live) {
      probabilities<T, EPL>(a, t, lane, s, p);
#pragma unroll
      for (int i = 0; i < EPL; ++i) dot += c[i] * p[i];
      dot = warp_sum(dot);
    }
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const int e = i * 32 + lane;
      if (e < a.E) out[e] = from_f32<T>(live ? factor * (p[i] * s[i]) * (c[i] - dot) : 0.0f);
    }
  }
}

// Tokens of a chunk: a batch of up to kMinChunk stays whole; a longer one gives at most kMaxChunks chunks.
int chunk_tokens(int T) {
  const int least = (T + kMaxChunks - 1) / kMaxChunks;
  return least > kMinChunk ? least : kMinChunk;
}
int chunk_count(int T) { return T > 0 ? (T + chunk_tokens(T) - 1) / chunk_tokens(T) : 1; }

template <typename T, int EPL>
cudaError_t launch_chunks(const BalanceArgs& a, bool backward, cudaStream_t stream) {
  if (backward) {
    const int ctas = (a.T + kChunkWarps - 1) / kChunkWarps;
    return launch_pdl(balance_backward_kernel<T, EPL>, dim3(ctas < 8 * kNumSMs ? ctas : 8 * kNumSMs), dim3(32 * kChunkWarps),
                      0, stream, a);
  }
  const size_t smem = static_cast<size_t>(kChunkWarps + 1) * EPL * 32 * 4;
  return launch_pdl(balance_chunk_kernel<T, EPL>, dim3(a.n_chunks), dim3(32 * kChunkWarps), smem, stream, a);
}

template <typename T>
cudaError_t launch_chunks(const BalanceArgs& a, bool backward, cudaStream_t stream) {
  const int per_lane = (a.E + 31) / 32;
  if (per_lane <= 2) return launch_chunks<T, 2>(a, backward, stream);
  if (per_lane <= 4) return launch_chunks<T, 4>(a, backward, stream);
  if (per_lane <= 8) return launch_chunks<T, 8>(a, backward, stream);
  if (per_lane <= 16) return launch_chunks<T, 16>(a, backward, stream);
  return launch_chunks<T, 32>(a, backward, stream);
}

cudaError_t launch_balance(const BalanceArgs& a, int dtype, bool backward, cudaStream_t stream) {
  if (dtype == MOE_B200_F32) return launch_chunks<float>(a, backward, stream);
  if (dtype == MOE_B200_BF16) return launch_chunks<__nv_bfloat16>(a, backward, stream);
  return launch_chunks<__half>(a, backward, stream);
}

bool bad_common(int T, int E, int K, int S, int dtype, int scoring, const int32_t* cu_seqlens) {
  return T < 0 || E < 1 || E > kMaxExperts || K < 1 || K > E || S < 0 || (!cu_seqlens && S != 1) || dtype < MOE_B200_F32 ||
         dtype > MOE_B200_F16 || scoring < MOE_B200_SCORE_SIGMOID || scoring > MOE_B200_SCORE_SOFTMAX;
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" size_t moe_fp8_block_scale_balance_loss_workspace_bytes(int T, int E) {
  if (T < 0 || E < 1 || E > kMaxExperts) return 0;
  return static_cast<size_t>(chunk_count(T)) * (4 * static_cast<size_t>(E) + 3) * 4;
}

extern "C" int moe_fp8_block_scale_balance_loss(const void* logits, int64_t logits_stride, int dtype, const int32_t* topk_idx,
                                                int T, int E, int K, const int32_t* cu_seqlens, int S,
                                                const uint8_t* token_mask, int scoring, float alpha, float* loss,
                                                int32_t* counts, int32_t* tokens, void* workspace, size_t workspace_bytes,
                                                void* stream_v) {
  if (bad_common(T, E, K, S, dtype, scoring, cu_seqlens)) return MOE_B200_EINVAL;
  if (S == 0) return MOE_B200_OK;
  if ((T > 0 && (!logits || !topk_idx)) || !loss || !counts || !tokens || !workspace || !aligned(workspace, 4))
    return MOE_B200_EINVAL;
  if (workspace_bytes < moe_fp8_block_scale_balance_loss_workspace_bytes(T, E)) return MOE_B200_EWORKSPACE;
  BalanceArgs a = {};
  a.logits = logits; a.stride = logits_stride; a.topk_idx = topk_idx; a.cu = cu_seqlens; a.mask = token_mask;
  a.T = T; a.E = E; a.K = K; a.S = S; a.softmax = scoring == MOE_B200_SCORE_SOFTMAX;
  a.chunk = chunk_tokens(T); a.n_chunks = chunk_count(T);
  a.alpha = alpha; a.loss = loss; a.counts = counts; a.tokens = tokens;
  const size_t rows = static_cast<size_t>(a.n_chunks) * 2 * E;
  a.part_p = static_cast<float*>(workspace);
  a.part_c = reinterpret_cast<int*>(a.part_p + rows);
  a.part_n = a.part_c + rows;
  a.tail = a.part_n + 2 * a.n_chunks;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  cudaError_t e = launch_balance(a, dtype, false, stream);
  if (e == cudaSuccess && a.n_chunks > 1)
    e = launch_pdl(balance_join_kernel, dim3(a.n_chunks - 1), dim3(E < 1024 ? (E + 31) / 32 * 32 : 1024), 0, stream, a);
  return launch_status(e, a.n_chunks > 1 ? 2 : 1);
}

extern "C" int moe_fp8_block_scale_balance_loss_backward(const float* grad_loss, const void* logits, int64_t logits_stride,
                                                         int dtype, const int32_t* counts, const int32_t* tokens, int T,
                                                         int E, int K, const int32_t* cu_seqlens, int S,
                                                         const uint8_t* token_mask, int scoring, float alpha,
                                                         void* grad_logits, void* stream_v) {
  if (bad_common(T, E, K, S, dtype, scoring, cu_seqlens)) return MOE_B200_EINVAL;
  if (T == 0) return MOE_B200_OK;
  if (!logits || !grad_logits || (S > 0 && (!grad_loss || !counts || !tokens))) return MOE_B200_EINVAL;
  BalanceArgs a = {};
  a.logits = logits; a.stride = logits_stride; a.cu = cu_seqlens; a.mask = token_mask;
  a.T = T; a.E = E; a.K = K; a.S = S; a.softmax = scoring == MOE_B200_SCORE_SOFTMAX;
  a.alpha = alpha; a.counts = const_cast<int*>(counts); a.tokens = const_cast<int*>(tokens);
  a.grad_loss = grad_loss; a.grad = grad_logits;
  return launch_status(launch_balance(a, dtype, true, static_cast<cudaStream_t>(stream_v)), 1);
}
