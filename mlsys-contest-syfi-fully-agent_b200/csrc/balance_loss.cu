// Balance loss of a routing, per sequence, with per-expert counts, and its gradient for the router's logits.
//
// s = sigmoid(z) or exp(z), p_ti = s_ti / sum_j s_tj.  For a sequence with n counted tokens whose K selections are
// topk_idx, c_i = selections of expert i:
//     loss = alpha E / (K n^2) sum_i c_i sum_t p_ti
// (the mean over the tokens of p, times the frequencies E c_i / (K n), times alpha), and with the counts held constant
//     dloss/dz_ti = alpha E / (K n^2) d_ti (c_i - sum_j c_j p_tj),    d = p (1 - s) for sigmoid, p for softmax.
// A row whose scores are all zero (every logit -inf) has p = 0 and no gradient.
//
// Forward: the token axis is cut into equal chunks, one CTA of up to 32 warps each, a warp per token.  A sequence of up to 8
// tokens inside the chunk is one warp's work from its probabilities to its loss; a longer one is the whole CTA's.  What
// lies inside the chunk is finished there; a sequence that crosses a border leaves one partial row per chunk, which
// balance_join_kernel adds in chunk order (no floating-point atomics: the same bits every time).  Counts are integers.
// Bound by latency (search of the borders, load, reductions) up to some thousand tokens and by the exponentials and
// their reductions beyond; a row is loaded while the one before is worked on.
// Measured, 256 experts, fp32: 16 tokens 4.7 us, 16384 tokens 17 us (two launches; 172 us when one CTA added 512 partial
// rows in turn), 4099 tokens in 700 sequences of 160 experts 23 us; gradient of 8191 ragged bf16 tokens 9 us.
#include "elem_device.cuh"

namespace moe {
namespace {

constexpr int kMaxExperts = 1024;
// Warps of a chunk's CTA: what the registers of its lanes' experts leave.
__host__ __device__ constexpr int chunk_warps(int per_lane) { return per_lane <= 8 ? 32 : per_lane <= 16 ? 16 : 8; }
constexpr int kMinChunk = 32;          // tokens; smaller batches stay in one CTA, which needs no second launch
constexpr int kSumTokens = 256;        // tokens that a warp adds up in a row at most: off by 256 * 2^-24 / 2 of the sum
constexpr int kShort = 8;              // longest sequence that one warp takes
constexpr int kBackWarps = 8;

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

// Expert of a lane's i-th value: neighbours where a row can be read 16 bytes at a time, else 32 apart.
template <typename T, bool VEC>
__device__ __forceinline__ int expert_of(int i, int lane) {
  constexpr int kRun = VEC ? 16 / static_cast<int>(sizeof(T)) : 1;
  return (i / kRun * 32 + lane) * kRun + i % kRun;
}

// A lane's values of a row as they are in memory.
template <typename T, int EPL, bool VEC>
struct alignas(VEC ? 16 : sizeof(T)) Raw {
  T v[EPL];
};
template <typename T, int EPL, bool VEC>
__device__ __forceinline__ void load_row(const BalanceArgs& a, int t, int lane, Raw<T, EPL, VEC>& r) {
  const T* row = static_cast<const T*>(a.logits) + t * a.stride;
  constexpr int kRun = VEC ? 16 / static_cast<int>(sizeof(T)) : 1;
#pragma unroll
  for (int i = 0; i < EPL; i += kRun) {
    const int e = expert_of<T, VEC>(i, lane);
    if (e >= a.E) continue;
    if (VEC) *reinterpret_cast<uint4*>(r.v + i) = *reinterpret_cast<const uint4*>(row + e);
    else r.v[i] = row[e];
  }
}

// Probabilities of a row, zero where the row has none, and (SLOPE) what dp/dz needs beside them: 1 - sigmoid(z) (1 for a
// softmax), formed as e^-z sigmoid(z) where 1 - sigmoid(z) would cancel.
template <typename T, int EPL, bool VEC, bool SLOPE>
__device__ __forceinline__ void probabilities(const BalanceArgs& a, const Raw<T, EPL, VEC>& r, int lane, float (&p)[EPL], float (&slope)[EPL]) {
  float sum = 0.0f;
  if (!a.softmax) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const float z = expert_of<T, VEC>(i, lane) < a.E ? to_f32<T>(r.v[i]) : -INFINITY;
      const float x = expf(-z);
      p[i] = __fdividef(1.0f, 1.0f + x);                 // 2 units in the last place at most
      if (x > 0x1p125f) p[i] = 0.0f;                     // beyond the fast division's range; the row is shifted if it matters
      if (SLOPE) slope[i] = z > 0.0f ? x * p[i] : 1.0f - p[i];
      sum += p[i];
    }
    sum = warp_sum(sum);
  }
  // sigmoid(z) is e^z to fp32 below -60 and loses its bits below -87: a row with nothing larger (or a NaN) is shifted by
  // its largest value like a softmax's
  if (a.softmax || !(sum > 0x1p-80f)) {
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      p[i] = expert_of<T, VEC>(i, lane) < a.E ? to_f32<T>(r.v[i]) : -INFINITY;
      top = fmaxf(top, p[i]);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      p[i] = p[i] == -INFINITY ? 0.0f : expf(p[i] - top);
      if (SLOPE) slope[i] = 1.0f;
      sum += p[i];
    }
    sum = warp_sum(sum);
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
  for (int i = 0; i < EPL; ++i) p[i] *= inv;
}

// Tokens first, first + step, ... below end: adds their probabilities to acc and their selections to hist (shared
// memory); returns how many counted.
template <typename T, int EPL, bool VEC>
__device__ __forceinline__ int add_tokens(const BalanceArgs& a, int first, int end, int step, int lane, float (&acc)[EPL], int* hist) {
  int n = 0;
  Raw<T, EPL, VEC> next;
  int next_e = -1;                               // the lane's selection; more than 32 of them are read where they count
  bool next_live = false;
  auto fetch = [&](int t) {
    next_live = t < end && (!a.mask || a.mask[t]);
    if (!next_live) return;
    load_row(a, t, lane, next);
    if (lane < a.K) next_e = a.topk_idx[static_cast<int64_t>(t) * a.K + lane];
  };
  fetch(first);
  for (int t = first; t < end; t += step) {
    const Raw<T, EPL, VEC> now = next;
    const int e = next_e;
    const bool live = next_live;
    fetch(t + step);
    if (!live) continue;
    if (e >= 0 && e < a.E) atomicAdd(hist + e, 1);
    for (int k = lane + 32; k < a.K; k += 32) {
      const int more = a.topk_idx[static_cast<int64_t>(t) * a.K + k];
      if (more >= 0 && more < a.E) atomicAdd(hist + more, 1);
    }
    float p[EPL], none[EPL];
    probabilities<T, EPL, VEC, false>(a, now, lane, p, none);
#pragma unroll
    for (int i = 0; i < EPL; ++i) acc[i] += p[i];
    ++n;
  }
  return n;
}

__device__ __forceinline__ float loss_of(const BalanceArgs& a, float dot, int n) {
  return n ? a.alpha * a.E / a.K * (dot / n / n) : 0.0f;
}

template <typename T, int EPL, bool VEC>
__global__ void __launch_bounds__(32 * chunk_warps(EPL)) balance_chunk_kernel(BalanceArgs a) {
  constexpr int kChunkWarps = chunk_warps(EPL);
  griddep_launch_dependents();
  griddep_wait();
  extern __shared__ float sums[];                // [kChunkWarps][E]: sums of the warps, or a histogram for each
  int* const hists = reinterpret_cast<int*>(sums);
  int* const hist = hists + kChunkWarps * a.E;   // [E] of the whole CTA
  __shared__ float red[32];
  __shared__ int n_valid, found[2];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x;
  const int t0 = c * a.chunk, t1 = min(a.T, t0 + a.chunk);
  const bool last = c == a.n_chunks - 1;
  if (w < 2) {
    const int s = w == 0 ? begun_before(a, t0, lane) : last ? a.S : begun_before(a, t1, lane);
    if (lane == 0) found[w] = s;
  }
  __syncthreads();
  const int first = found[0], end = found[1];    // sequences that begin in the chunk

  // short ones inside the chunk: a warp each
  for (int q = first + w; q < end; q += kChunkWarps) {
    const int b0 = border(a, q), b1 = max(border(a, q + 1), b0);
    if (b1 > t1 || b1 - b0 > kShort) continue;
    int* const mine = hists + w * a.E;
    for (int e = lane; e < a.E; e += 32) mine[e] = 0;
    __syncwarp();
    float acc[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) acc[i] = 0.0f;
    const int n = add_tokens<T, EPL, VEC>(a, b0, b1, 1, lane, acc, mine);
    __syncwarp();
    float dot = 0.0f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const int e = expert_of<T, VEC>(i, lane);
      if (e < a.E) dot += static_cast<float>(mine[e]) * acc[i];
    }
    for (int e = lane; e < a.E; e += 32) a.counts[static_cast<int64_t>(q) * a.E + e] = mine[e];
    dot = warp_sum(dot);
    if (lane == 0) {
      a.tokens[q] = n;
      a.loss[q] = loss_of(a, dot, n);
    }
    __syncwarp();
  }

  // the others, all warps together; the first of them may have begun before the chunk
  int tail = -1;
  for (int q = first > 0 ? first - 1 : 0; q < end; ++q) {
    const int b0 = border(a, q), b1 = max(border(a, q + 1), b0);
    const bool head = q < first;
    if (head ? b1 <= t0 : b1 <= t1 && b1 - b0 <= kShort) continue;
    const int lo = max(b0, t0), hi = min(b1, t1);
    __syncthreads();
    for (int e = threadIdx.x; e < a.E; e += blockDim.x) hist[e] = 0;
    if (threadIdx.x == 0) n_valid = 0;
    __syncthreads();
    float acc[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) acc[i] = 0.0f;
    const int n = add_tokens<T, EPL, VEC>(a, lo + w, hi, kChunkWarps, lane, acc, hist);
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const int e = expert_of<T, VEC>(i, lane);
      if (e < a.E) sums[w * a.E + e] = acc[i];
    }
    if (lane == 0) atomicAdd(&n_valid, n);
    __syncthreads();
    const bool whole = !head && b1 <= t1;
    const int slot = c * 2 + (head ? 0 : 1);
    const int used = min(kChunkWarps, hi - lo);  // warps that had a token
    float dot[1] = {0.0f};
    for (int e = threadIdx.x; e < a.E; e += blockDim.x) {
      float p = 0.0f;
#pragma unroll 8
      for (int v = 0; v < used; ++v) p += sums[v * a.E + e];
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
      if (whole) {
        a.tokens[q] = n_valid;
        a.loss[q] = loss_of(a, dot[0], n_valid);
      } else {
        a.part_n[slot] = n_valid;
      }
    }
    if (!head && b1 > t1) tail = q;
  }
  if (threadIdx.x == 0) a.tail[c] = tail;
}

// Rows of a strip of the join that are added up plainly; more of them, which only batches beyond a million tokens have, with
// what the additions lose kept beside the sum (16384 tokens take 18.4 us that way and 17.4 without).
constexpr int kJoinRows = 148;

// CTA c finishes the sequence that begins in chunk c and goes on after it, if there is one.  Strips of the partial rows
// are added side by side and joined in order.
__global__ void __launch_bounds__(1024) balance_join_kernel(BalanceArgs a) {
  griddep_launch_dependents();
  griddep_wait();
  __shared__ float red[32], strip_p[1024], strip_lost[1024];
  __shared__ int strip_c[1024], n_all;
  const int c = blockIdx.x, q = a.tail[c];
  if (q < 0) return;
  const int last = (max(border(a, q + 1), 1) - 1) / a.chunk;
  const int padded = (a.E + 31) / 32 * 32, strips = 1024 / padded;
  const int strip = threadIdx.x / padded, e = threadIdx.x - strip * padded;
  if (threadIdx.x == 0) n_all = 0;
  __syncthreads();
  float p = 0.0f, lost = 0.0f;
  int n = 0;
  if (strip < strips && e < a.E) {
    const int per = (last - c + strips) / strips;                    // rows c .. last
    const int k0 = c + strip * per, k1 = min(last + 1, k0 + per);
    auto at = [&](int k) { return static_cast<int64_t>(2 * k + (k == c ? 1 : 0)) * a.E + e; };
    if (k1 - k0 <= kJoinRows) {
#pragma unroll 8
      for (int k = k0; k < k1; ++k) {
        p += a.part_p[at(k)];
        n += a.part_c[at(k)];
      }
    } else {
#pragma unroll 4
      for (int k = k0; k < k1; ++k) {
        add_exactly(p, lost, a.part_p[at(k)]);
        n += a.part_c[at(k)];
      }
    }
  }
  strip_p[threadIdx.x] = p;
  strip_lost[threadIdx.x] = lost;
  strip_c[threadIdx.x] = n;
  for (int k = c + threadIdx.x; k <= last; k += blockDim.x) atomicAdd(&n_all, a.part_n[2 * k + (k == c ? 1 : 0)]);
  __syncthreads();
  float dot[1] = {0.0f};
  if (threadIdx.x < a.E) {
    p = lost = 0.0f;
    n = 0;
    for (int s = 0; s < strips; ++s) {
      add_exactly(p, lost, strip_p[s * padded + threadIdx.x]);
      lost += strip_lost[s * padded + threadIdx.x];
      n += strip_c[s * padded + threadIdx.x];
    }
    a.counts[static_cast<int64_t>(q) * a.E + threadIdx.x] = n;
    dot[0] = static_cast<float>(n) * joined(p, lost);
  }
  block_sum(dot, red);
  if (threadIdx.x == 0) {
    a.tokens[q] = n_all;
    a.loss[q] = loss_of(a, dot[0], n_all);
  }
}

// A warp takes consecutive tokens.  The counts enter less their mean K n / E (rounded: an exact integer difference),
// which leaves the gradient as it is, because sum p = 1, and keeps its difference from cancelling when the counts are
// nearly even.  Bound by HBM (logits in, gradient out) at many tokens.
template <typename T, int EPL, bool VEC>
__global__ void __launch_bounds__(32 * kBackWarps) balance_backward_kernel(BalanceArgs a) {
  griddep_launch_dependents();
  griddep_wait();
  constexpr int kRun = VEC ? 16 / static_cast<int>(sizeof(T)) : 1;
  const int lane = threadIdx.x & 31;
  const int warps = gridDim.x * kBackWarps, warp = blockIdx.x * kBackWarps + (threadIdx.x >> 5);
  const int per = (a.T + warps - 1) / warps;
  const int t0 = static_cast<int>(min(static_cast<int64_t>(warp) * per, static_cast<int64_t>(a.T))), t1 = min(a.T, t0 + per);
  int q = -1, b0 = 0, b1 = -1;       // sequence of the counts in registers and its borders
  float c[EPL], factor = 0.0f;
  Raw<T, EPL, VEC> next;
  bool next_live = false;
  if (t0 < t1 && (next_live = !a.mask || a.mask[t0])) load_row(a, t0, lane, next);
  for (int t = t0; t < t1; ++t) {
    const Raw<T, EPL, VEC> now = next;
    const bool unmasked = next_live;
    if (t + 1 < t1 && (next_live = !a.mask || a.mask[t + 1])) load_row(a, t + 1, lane, next);
    if (unmasked && (t < b0 || t >= b1)) {
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
          const int e = expert_of<T, VEC>(i, lane);
          c[i] = e < a.E ? static_cast<float>(a.counts[static_cast<int64_t>(q) * a.E + e] - mean) : 0.0f;
        }
      }
    }
    T* out = static_cast<T*>(a.grad) + static_cast<int64_t>(t) * a.E;
    Raw<T, EPL, VEC> result;
    if (unmasked && t >= b0 && t < b1) {
      float p[EPL], slope[EPL];
      float dot = 0.0f;
      probabilities<T, EPL, VEC, true>(a, now, lane, p, slope);
#pragma unroll
      for (int i = 0; i < EPL; ++i) dot += c[i] * p[i];
      dot = warp_sum(dot);
#pragma unroll
      for (int i = 0; i < EPL; ++i) result.v[i] = from_f32<T>(factor * (p[i] * slope[i]) * (c[i] - dot));
    } else {
#pragma unroll
      for (int i = 0; i < EPL; ++i) result.v[i] = from_f32<T>(0.0f);
    }
#pragma unroll
    for (int i = 0; i < EPL; i += kRun) {
      const int e = expert_of<T, VEC>(i, lane);
      if (e >= a.E) continue;
      if (VEC) *reinterpret_cast<uint4*>(out + e) = *reinterpret_cast<const uint4*>(result.v + i);
      else out[e] = result.v[i];
    }
  }
}

// Tokens of a chunk: a batch of up to kMinChunk stays whole; a longer one gives at most one chunk per SM, a very long one
// several, so that no warp has more than kSumTokens of them.
int chunk_tokens(int T, int E) {
  const int most = kSumTokens * (E <= 256 ? chunk_warps(8) : chunk_warps(32));
  const int waves = static_cast<int>((T + int64_t(kNumSMs) * most - 1) / (int64_t(kNumSMs) * most));
  const int chunks = kNumSMs * (waves > 0 ? waves : 1), least = static_cast<int>((T + int64_t(chunks) - 1) / chunks);
  return least > kMinChunk ? least : kMinChunk;
}
int chunk_count(int T, int E) { return T > 0 ? (T - 1) / chunk_tokens(T, E) + 1 : 1; }

template <typename T, int EPL, bool VEC>
cudaError_t launch_chunks(const BalanceArgs& a, bool backward, cudaStream_t stream) {
  if (backward) {
    const int ctas = (a.T + kBackWarps - 1) / kBackWarps;
    return launch_pdl(balance_backward_kernel<T, EPL, VEC>, dim3(ctas < 8 * kNumSMs ? ctas : 8 * kNumSMs), dim3(32 * kBackWarps), 0,
                      stream, a);
  }
  constexpr int kChunkWarps = chunk_warps(EPL);
  const size_t smem = static_cast<size_t>(kChunkWarps + 1) * a.E * 4;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_smem(balance_chunk_kernel<T, EPL, VEC>, (kChunkWarps + 1) * EPL * 32 * 4, done);
  if (e != cudaSuccess) return e;
  return launch_pdl(balance_chunk_kernel<T, EPL, VEC>, dim3(a.n_chunks), dim3(32 * kChunkWarps), smem, stream, a);
}

template <typename T>
cudaError_t launch_chunks(const BalanceArgs& a, bool backward, cudaStream_t stream) {
  constexpr int kRun = 16 / static_cast<int>(sizeof(T));
  const bool vec = a.E % kRun == 0 && a.stride % kRun == 0 && aligned(a.logits, 16) && (!backward || aligned(a.grad, 16));
  const int per_lane = (a.E + 31) / 32;
  if (vec) {
    if (per_lane <= 8) return launch_chunks<T, 8, true>(a, backward, stream);
    if (per_lane <= 16) return launch_chunks<T, 16, true>(a, backward, stream);
    return launch_chunks<T, 32, true>(a, backward, stream);
  }
  if (per_lane <= 2) return launch_chunks<T, 2, false>(a, backward, stream);
  if (per_lane <= 8) return launch_chunks<T, 8, false>(a, backward, stream);
  // 257 to 512 experts too: a kernel between the two was not measured
  return launch_chunks<T, 32, false>(a, backward, stream);
}

cudaError_t launch_balance(const BalanceArgs& a, int dtype, bool backward, cudaStream_t stream) {
  if (dtype == MOE_B200_F32) return launch_chunks<float>(a, backward, stream);
  if (dtype == MOE_B200_BF16) return launch_chunks<__nv_bfloat16>(a, backward, stream);
  return launch_chunks<__half>(a, backward, stream);
}

bool bad_common(int T, int E, int K, int S, int dtype, int scoring, const int32_t* cu_seqlens) {
  return T < 0 || T > (1 << 30) || S > (1 << 30) || E < 1 || E > kMaxExperts || K < 1 || K > E || S < 0 || (!cu_seqlens && S != 1) || dtype < MOE_B200_F32 ||
         dtype > MOE_B200_F16 || scoring < MOE_B200_SCORE_SIGMOID || scoring > MOE_B200_SCORE_SOFTMAX;
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" size_t moe_fp8_block_scale_balance_loss_workspace_bytes(int T, int E) {
  if (T < 0 || E < 1 || E > kMaxExperts) return 0;
  return static_cast<size_t>(chunk_count(T, E)) * (4 * static_cast<size_t>(E) + 3) * 4;
}

extern "C" int moe_fp8_block_scale_balance_loss(const void* logits, int64_t logits_stride, int dtype, const int32_t* topk_idx,
                                                int T, int E, int K, const int32_t* cu_seqlens, int S,
                                                const uint8_t* token_mask, int scoring, float alpha, float* loss,
                                                int32_t* counts, int32_t* tokens, void* workspace, size_t workspace_bytes,
                                                void* stream_v) {
  if (bad_common(T, E, K, S, dtype, scoring, cu_seqlens)) return MOE_B200_EINVAL;
  if (S == 0) return MOE_B200_OK;
  if ((T > 0 && (!logits || !topk_idx)) || !loss || !counts || !tokens || !workspace || !aligned(workspace, 4) ||
      !aligned(logits, element_size(dtype)) || !aligned(topk_idx, 4) || !aligned(cu_seqlens, 4) || !aligned(loss, 4) ||
      !aligned(counts, 4) || !aligned(tokens, 4))
    return MOE_B200_EINVAL;
  if (workspace_bytes < moe_fp8_block_scale_balance_loss_workspace_bytes(T, E)) return MOE_B200_EWORKSPACE;
  BalanceArgs a = {};
  a.logits = logits; a.stride = logits_stride; a.topk_idx = topk_idx; a.cu = cu_seqlens; a.mask = token_mask;
  a.T = T; a.E = E; a.K = K; a.S = S; a.softmax = scoring == MOE_B200_SCORE_SOFTMAX;
  a.chunk = chunk_tokens(T, E); a.n_chunks = chunk_count(T, E);
  a.alpha = alpha; a.loss = loss; a.counts = counts; a.tokens = tokens;
  const size_t rows = static_cast<size_t>(a.n_chunks) * 2 * E;
  a.part_p = static_cast<float*>(workspace);
  a.part_c = reinterpret_cast<int*>(a.part_p + rows);
  a.part_n = a.part_c + rows;
  a.tail = a.part_n + 2 * a.n_chunks;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  cudaError_t e = launch_balance(a, dtype, false, stream);
  if (e == cudaSuccess && a.n_chunks > 1)
    e = launch_pdl(balance_join_kernel, dim3(a.n_chunks - 1), dim3(1024), 0, stream, a);
  return launch_status(e, a.n_chunks > 1 ? 2 : 1);
}

extern "C" int moe_fp8_block_scale_balance_loss_backward(const float* grad_loss, const void* logits, int64_t logits_stride,
                                                         int dtype, const int32_t* counts, const int32_t* tokens, int T,
                                                         int E, int K, const int32_t* cu_seqlens, int S,
                                                         const uint8_t* token_mask, int scoring, float alpha,
                                                         void* grad_logits, void* stream_v) {
  if (bad_common(T, E, K, S, dtype, scoring, cu_seqlens)) return MOE_B200_EINVAL;
  if (T == 0) return MOE_B200_OK;
  if (!logits || !grad_logits || (S > 0 && (!grad_loss || !counts || !tokens)) || !aligned(logits, element_size(dtype)) ||
      !aligned(grad_logits, element_size(dtype)) || !aligned(cu_seqlens, 4) || !aligned(grad_loss, 4) || !aligned(counts, 4) ||
      !aligned(tokens, 4))
    return MOE_B200_EINVAL;
  BalanceArgs a = {};
  a.logits = logits; a.stride = logits_stride; a.cu = cu_seqlens; a.mask = token_mask;
  a.T = T; a.E = E; a.K = K; a.S = S; a.softmax = scoring == MOE_B200_SCORE_SOFTMAX;
  a.alpha = alpha; a.counts = const_cast<int*>(counts); a.tokens = const_cast<int*>(tokens);
  a.grad_loss = grad_loss; a.grad = grad_logits;
  return launch_status(launch_balance(a, dtype, true, static_cast<cudaStream_t>(stream_v)), 1);
}
