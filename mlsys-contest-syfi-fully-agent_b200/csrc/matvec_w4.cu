// Matrix-vector products with 4-bit weights and group scales, for decode-sized batches, dense or by chosen experts:
//     out[r, n] = sum_k x[row(r), k] (q[e(r), n, k] - z[e(r), n, k / G]) scale[e(r), n, k / G]
// q: two values a byte, the even k in the low half; z: 8 without a table.  Pair r = (token, choice) reads row r / per_row
// of x and expert experts[r]; a pair whose expert is not held here gives a zero row.
//
// Bound by the weights, which are read once per (expert, up to 8 or 16 rows), and next by the instructions that unpack
// them.  The products run on mma.sync m16n8k16 with the weights as the 16-row operand, which a lane builds in registers
// from the bytes it loaded itself: such an operand never passes through shared memory or tensor memory, and with at most
// 16 columns per weight the tensor pipe is idle most of the time anyway.  A lane's 16 (8, 4) bytes of a group of 128 (64,
// 32) weights feed eight (four, two) products in whatever order of k suits the unpacking; x is staged in shared memory in
// that same order.
//
// Unpacking begins with one AND per pair: a floating-point format's codes are linear up to twice its smallest normal number,
// so a half word with only a 4-bit field set is q or 16 q times the smallest subnormal (2^-24 in fp16, 2^-133 in bf16).  The
// fields at bit 0 and at bit 4 go to accumulators of their own.  Products and sums are fp32; the scale multiplies a group's
// fp32 sum.  What happens to the zero point depends on the result's type:
// * fp32 results (EXACT): one packed multiply-add per pair,  code * 2^127 - z 2^-6  (bf16; 2^15 and 2^-9 in fp16), makes it
//   (q - z) times a power of two, exactly, so the error goes with sum |(q - z) x| however close to the zero point the weights
//   are.
// * 16-bit results: the tensor cores multiply the codes themselves, exactly, and per group  sum (q - z) x = sum q x - z sum x,
//   with sum x from the staging.  The error goes with sum |q x|, 2^-24 of it in each addition, which the result's own
//   rounding of 2^-9 or 2^-12 hides.  bf16 activations are staged times 2^64 so that the products are normal fp32 numbers
//   (|x| < 2^63; below 2^-57 they keep an absolute 2^-80).  The multiply-adds would cost one token through eight 4096 x 7168
//   experts 35.1 us instead of 31.9, and sixteen tokens through 32 of them 120 instead of 108.
//
// One persistent CTA per SM takes a contiguous run of items (expert and up to 8 or 16 of its rows, 16 weight rows), stages
// the rows of x that the expert has, and its sixteen warps stream weights through rings of their own (cp.async, two
// stages of 16 rows x 256 columns a warp, 64 KB in flight per SM), which run on across items.  A warp has an item to
// itself, or several warps share its K when there are too few items; then their sums meet in shared memory in a fixed
// order.  (A ring in registers waits for its newest loads with its oldest: 97 us where this takes 31.)
// Measured, bf16, groups of 128: one token through eight 4096 x 7168 experts 32 us (3.7 TB/s of weights), sixteen tokens'
// second products through 7168 x 2048 experts 57 us (3.8 TB/s), sixteen tokens through all 32 first ones 110 us (4.4 TB/s);
// half of the issue slots are taken, and what is left is the latency of unpacking and products with four warps on each
// quarter of an SM.  Deeper rings change nothing, 24 warps of 80 registers take 39 us instead of 32.
#include <limits.h>

#include "elem_device.cuh"

namespace moe {
namespace {

constexpr int kMaxPairs = 256;
constexpr int kMaxMatvecExperts = 1024;
constexpr int kLogWarps = 4, kWarps = 1 << kLogWarps;
constexpr int kThreads = 32 * kWarps;
constexpr int kDepth = 2;                  // stages of a warp's ring
constexpr int kStep = 256;                 // columns of a stage
constexpr int kTile = 16;                  // weight rows of an item
constexpr int kSumSteps = 128;             // steps whose sums are added up in fp32 at most: off by 2^-17 of the terms
constexpr int kSmemMost = 227 * 1024;

struct MatvecArgs {
  const void* x;
  int64_t x_stride;
  const uint8_t* q;          // [E, N, K / 2]
  const void* scale;         // [E, N, K / G]
  const uint8_t* zero;       // [E, N, K / G] or null
  const int* experts;        // [pairs] or null
  int pairs, per_row, E, N, K, scale_f32, out_f32;
  int x_cols;                // rows of x that are staged at most
  int slice_most;            // steps of 256 columns staged at a time at most
  int x_chunks;              // 16-byte chunks for staged x: a job with fewer rows stages more steps at a time
  void* out;                 // [pairs, N]
};

template <typename T> struct Mma;
template <> struct Mma<__nv_bfloat16> {
  static constexpr float kUnit = 0x1p69f;              // undoes 2^-133 of the codes and 2^64 of x
  static constexpr float kExactUnit = 0x1p6f;          // undoes 2^-6 of q - z
  static constexpr uint32_t kEven = 0x7F007F00u, kOdd = 0x7D007D00u, kMinus = 0xFF00FF00u, kEight = 0xBE00BE00u;   // 2^127, 2^123, -2^127, -8 2^-6
  static __device__ __forceinline__ uint32_t fma(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
  }
  static __device__ __forceinline__ uint32_t staged(uint32_t v) {
    const __nv_bfloat162 r = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&v), __floats2bfloat162_rn(0x1p64f, 0x1p64f));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ float2 widen(uint32_t v) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u)); }
  static __device__ __forceinline__ void run(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
  }
};
template <> struct Mma<__half> {
  static constexpr float kUnit = 0x1p24f;
  static constexpr float kExactUnit = 0x1p9f;
  static constexpr uint32_t kEven = 0x78007800u, kOdd = 0x68006800u, kMinus = 0xF800F800u, kEight = 0xA400A400u;   // 2^15, 2^11, -2^15, -8 2^-9
  static __device__ __forceinline__ uint32_t fma(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
  }
  static __device__ __forceinline__ uint32_t staged(uint32_t v) { return v; }
  static __device__ __forceinline__ float2 widen(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
  static __device__ __forceinline__ void run(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
  }
};

template <int W> struct Words;             // W words of eight weights
template <> struct Words<4> { using Type = uint4; };
template <> struct Words<2> { using Type = uint2; };
template <> struct Words<1> { using Type = uint32_t; };

// A stage: 16 rows of 128 bytes of weights (16-byte chunks swizzled by row, so that 4-, 8- and 16-byte reads of eight rows
// are free of bank conflicts), then per row the aligned words that hold its scales, then those with its zero points.
template <int G, bool ZERO> struct Stage {
  static constexpr int kGroups = kStep / G;
  static constexpr int kScaleWords = kGroups;                        // fp32: one each; 16 bits: kGroups / 2 + 1 at most
  static constexpr int kZeroWords = ZERO ? (kGroups + 6) / 4 : 0;
  static constexpr int kScales = kTile * kStep / 2, kZeros = kScales + kTile * 4 * kScaleWords;
  static constexpr int kBytes = kZeros + kTile * 4 * kZeroWords;
};
__device__ __forceinline__ int swizzle(int row) { return (row & 1) << 2 | (row & 2) | ((row >> 2) & 1); }

// The batch by experts: rows that chose the same expert, in batches of a column tile.
struct Jobs {
  int list[kMaxPairs];       // pairs, by expert in order of first appearance, ascending inside
  int expert[kMaxPairs], first[kMaxPairs], cols[kMaxPairs];   // of a job: its expert, first entry of list, entries
  int n;
  uint32_t missing[kMaxPairs / 32];   // pairs whose expert is not held here
};

// Fills `jobs` from experts[]; every CTA does it for itself (a few hundred cycles).  `table` has an entry per expert.
__device__ __forceinline__ void find_jobs(const MatvecArgs& a, int max_cols, Jobs& jobs, int* table, int* scan) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int e = -1;
  if (tid < a.pairs) e = a.experts ? a.experts[tid] : 0;
  const bool held = e >= 0 && e < a.E;
  if (held) table[e] = 0;
  if (warp < kMaxPairs / 32) {
    const uint32_t none = __ballot_sync(0xFFFFFFFFu, tid < a.pairs && !held);
    if (lane == 0) jobs.missing[warp] = none;
  }
  __syncthreads();
  // place among the pairs of the same expert: warp after warp, so that the order is the pairs' own
  const uint32_t peers = __match_any_sync(0xFFFFFFFFu, held ? e : -1);
  const int below = __popc(peers & ((1u << lane) - 1));
  int place = 0;
  for (int w = 0; w < (a.pairs + 31) / 32; ++w) {
    if (warp == w && held) place = table[e] + below;
    __syncthreads();
    if (warp == w && held && below == 0) table[e] += __popc(peers);
    __syncthreads();
  }
  // the first pair of an expert opens its jobs; entries and jobs before them by a scan over the CTA, both in one word
  const int count = held && place == 0 ? table[e] : 0;
  const int opened = (count + max_cols - 1) / max_cols;
  int before = count | opened << 16;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xFFFFFFFFu, before, d);
    if (lane >= d) before += o;
  }
  if (lane == 31) scan[warp] = before;
  __syncthreads();
  before -= count | opened << 16;
  for (int w = 0; w < warp; ++w) before += scan[w];
  if (tid == kThreads - 1) jobs.n = (before >> 16) + opened;
  if (count) {
    const int first = before & 0xFFFF;
    table[e] = first;
    for (int j = 0; j < opened; ++j) {
      const int at = (before >> 16) + j;
      jobs.expert[at] = e;
      jobs.first[at] = first + j * max_cols;
      jobs.cols[at] = min(max_cols, count - j * max_cols);
    }
  }
  __syncthreads();
  if (held) jobs.list[table[e] + place] = tid;
  __syncthreads();
}

template <typename T, bool EXACT>
__device__ __forceinline__ void store_result(const MatvecArgs& a, int pair, int n, float v) {
  const int64_t at = static_cast<int64_t>(pair) * a.N + n;
  if (EXACT) static_cast<float*>(a.out)[at] = v;
  else static_cast<T*>(a.out)[at] = from_f32<T>(v);
}

// total += the products of a stage, 16 rows and 256 columns with USED of NT column tiles, times 1 / kUnit (kExactUnit).
template <typename T, int G, int USED, int NT, bool ZERO, bool EXACT>
__device__ __forceinline__ void step(const MatvecArgs& a, const uint8_t* stage, const uint8_t* const (&x_at)[NT], const float* xs_at,
                                     int u, const int (&s_at)[2], const int (&z_low)[2], int gid, int quad, float (&total)[NT][4]) {
  using S = Stage<G, ZERO>;
  constexpr int W = G / 32;                        // words of a lane per row and group
  // the scales of the lane's two rows; groups behind K have zeros for x and q and need a finite scale
  float scale[S::kGroups][2];
  if (a.scale_f32) {
#pragma unroll
    for (int gi = 0; gi < S::kGroups; ++gi)
#pragma unroll
      for (int h = 0; h < 2; ++h) scale[gi][h] = *reinterpret_cast<const float*>(stage + s_at[h] + gi * 4);
  } else {
#pragma unroll
    for (int gi = 0; gi < S::kGroups; ++gi)
#pragma unroll
      for (int h = 0; h < 2; ++h) scale[gi][h] = to_f32<T>(*reinterpret_cast<const T*>(stage + s_at[h] + gi * 2));
  }
  if ((u + 1) * kStep > a.K) {
#pragma unroll
    for (int gi = 1; gi < S::kGroups; ++gi)
      if (u * kStep + gi * G >= a.K) scale[gi][0] = scale[gi][1] = 0.0f;
  }
  float of_step[USED][4] = {};                     // many small groups: a sum of their own, which makes the long one shorter
  auto sum = [&](int t, int i) -> float& { return G < 128 ? of_step[t][i] : total[t][i]; };
#pragma unroll
  for (int gi = 0; gi < S::kGroups; ++gi) {
    typename Words<W>::Type w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      // the lane's W words of the group: byte gi * G / 2 + quad * 4 W of the row
      const int r = gid + 8 * h, byte = gi * (G / 2) + quad * (4 * W);
      w[h] = *reinterpret_cast<const typename Words<W>::Type*>(stage + r * (kStep / 2) + ((byte >> 4) ^ swizzle(r)) * 16 + (byte & 15));
    }
    uint32_t minus[2];                             // EXACT: -z of the lane's two rows, in the operands' unit
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      minus[h] = Mma<T>::kEight;
      if (ZERO && EXACT) {
        const uint32_t z = stage[S::kZeros + (gid + 8 * h) * 4 * S::kZeroWords + ((z_low[h] + u * S::kGroups) & 3) + gi];
        minus[h] = Mma<T>::fma(z | z << 16, Mma<T>::kMinus, 0u);
      }
    }
    float even[USED][4] = {}, odd[USED][4] = {};   // sums over the fields at bit 0 and at bit 4 of a byte
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const uint32_t lo = reinterpret_cast<const uint32_t*>(&w[0])[j];
      const uint32_t hi = reinterpret_cast<const uint32_t*>(&w[1])[j];
      uint32_t fe[4] = {lo & 0x000F000Fu, hi & 0x000F000Fu, (lo >> 8) & 0x000F000Fu, (hi >> 8) & 0x000F000Fu};
      uint32_t fo[4] = {lo & 0x00F000F0u, hi & 0x00F000F0u, (lo >> 8) & 0x00F000F0u, (hi >> 8) & 0x00F000F0u};
      if (EXACT) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          fe[i] = Mma<T>::fma(fe[i], Mma<T>::kEven, minus[i & 1]);
          fo[i] = Mma<T>::fma(fo[i], Mma<T>::kOdd, minus[i & 1]);
        }
      }
#pragma unroll
      for (int t = 0; t < USED; ++t) {
        const uint4 b = *reinterpret_cast<const uint4*>(x_at[t] + gi * (2 * G) + 64 * j);
        Mma<T>::run(even[t], fe, b.x, b.y, even[t]);
        Mma<T>::run(odd[t], fo, b.z, b.w, odd[t]);
      }
    }
    if constexpr (EXACT) {
#pragma unroll
      for (int t = 0; t < USED; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum(t, i) += (even[t][i] + odd[t][i]) * scale[gi][i >> 1];
    } else {
      float2 xt[USED];
#pragma unroll
      for (int t = 0; t < USED; ++t) xt[t] = *reinterpret_cast<const float2*>(xs_at + gi * (8 * NT) + 8 * t);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = gid + 8 * h;
        float zero = 8.0f;
        if (ZERO) zero = static_cast<float>(stage[S::kZeros + r * 4 * S::kZeroWords + ((z_low[h] + u * S::kGroups) & 3) + gi]);
#pragma unroll
        for (int t = 0; t < USED; ++t) {
          sum(t, 2 * h) += (even[t][2 * h] + 0.0625f * odd[t][2 * h] - zero * xt[t].x) * scale[gi][h];
          sum(t, 2 * h + 1) += (even[t][2 * h + 1] + 0.0625f * odd[t][2 * h + 1] - zero * xt[t].y) * scale[gi][h];
        }
      }
    }
  }
  if (G < 128) {
#pragma unroll
    for (int t = 0; t < USED; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) total[t][i] += of_step[t][i];
  }
}

// Where a warp is in its sequence of (job, round, slice, step).
struct Cursor {
  int job, round, slice, u, end;
  int tile, tile_end;        // first tile of the CTA's run in this job and the one behind its last
  int lw;                    // log2 of the warps that share an item of the run
  int slice_steps, slices;   // of x
};

// G: group size.  NT: token tiles of eight columns.  ZERO: a table of zero points.  EXACT: fp32 results.
template <typename T, int G, int NT, bool ZERO, bool EXACT>
__global__ void __launch_bounds__(kThreads, 1) matvec_w4_kernel(MatvecArgs a) {
  using S = Stage<G, ZERO>;
  constexpr int W = G / 32, kCols = 8 * NT;
  extern __shared__ __align__(16) uint8_t smem[];  // rings of the warps, staged x, a group of zeros, sums of x (!EXACT)
  __shared__ float red[2][kWarps][kCols][kTile + 4];
  __shared__ Jobs jobs;
  __shared__ int scan[kWarps];
  __shared__ const T* x_from[kCols];
  static_assert(sizeof(red) >= kMaxMatvecExperts * sizeof(int), "find_jobs' table lies in red");
  griddep_launch_dependents();
  griddep_wait();

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gid = lane >> 2, quad = lane & 3;
  uint4* const xs = reinterpret_cast<uint4*>(smem + kWarps * kDepth * S::kBytes);
  uint4* const none = xs + a.x_chunks;             // what lanes without a column multiply
  float* const xsum = reinterpret_cast<float*>(none + kStep / 8);   // [groups of a slice][kCols]
  const uint32_t ring = smem_address(smem) + warp * kDepth * S::kBytes;
  if (tid < kStep / 8) none[tid] = make_uint4(0u, 0u, 0u, 0u);
  find_jobs(a, a.x_cols, jobs, reinterpret_cast<int*>(red), scan);
  for (int w = 0; w < kMaxPairs / 32; ++w) {
    for (uint32_t left = jobs.missing[w]; left != 0; left &= left - 1) {
      const int p = w * 32 + __ffs(left) - 1;
      for (int n = blockIdx.x * kThreads + tid; n < a.N; n += gridDim.x * kThreads) store_result<T, EXACT>(a, p, n, 0.0f);
    }
  }

  if (jobs.n == 0) return;                         // none of the batch's experts is held here: a batch of zero rows

  const int steps = (a.K + kStep - 1) / kStep, groups = a.K / G, tiles = (a.N + kTile - 1) / kTile;
  const int64_t items = static_cast<int64_t>(jobs.n) * tiles;
  // The CTA's run of items.  A run that goes on into the next job stages x twice and ends two rounds with idle warps, so
  // with few jobs every CTA stays in one of them; with many, equal runs matter more.
  int item0, item1;
  if (jobs.n * 4 <= gridDim.x) {
    const int g = gridDim.x, job = blockIdx.x * jobs.n / g;
    const int lo = (job * g + jobs.n - 1) / jobs.n, n = ((job + 1) * g + jobs.n - 1) / jobs.n - lo, i = blockIdx.x - lo;
    item0 = job * tiles + static_cast<int>(static_cast<int64_t>(tiles) * i / n);
    item1 = job * tiles + static_cast<int>(static_cast<int64_t>(tiles) * (i + 1) / n);
  } else {
    item0 = static_cast<int>(items * blockIdx.x / gridDim.x);
    item1 = static_cast<int>(items * (blockIdx.x + 1) / gridDim.x);
  }
  if (item0 == item1) return;
  const int last_job = (item1 - 1) / tiles;

  auto open_job = [&](Cursor& c) {
    c.slice_steps = min(a.slice_most, (a.x_chunks / jobs.cols[c.job] - 4) / (kStep / 8));
    c.slices = (steps + c.slice_steps - 1) / c.slice_steps;
    c.tile = max(item0 - c.job * tiles, 0);
    c.tile_end = min(item1 - c.job * tiles, tiles);
    // the fewest steps until the last warp is done with the run, with about a step's time for a join
    int best = INT_MAX;
#pragma unroll
    for (int k = 0; k <= kLogWarps; ++k) {
      const int cost = ((c.tile_end - c.tile + (kWarps >> k) - 1) >> (kLogWarps - k)) * (((steps + (1 << k) - 1) >> k) + (k > 0 ? 1 : 0));
      if (cost < best) {
        best = cost;
        c.lw = k;
      }
    }
  };
  auto tile_of = [&](const Cursor& c) { return c.tile + (c.round << (kLogWarps - c.lw)) + (warp >> c.lw); };
  auto open = [&](Cursor& c) {                     // the warp's steps in (job, round, slice)
    const int s0 = c.slice * c.slice_steps, s1 = min(steps, s0 + c.slice_steps), per = (s1 - s0 + (1 << c.lw) - 1) >> c.lw;
    c.u = min(s1, s0 + (warp & ((1 << c.lw) - 1)) * per);
    c.end = tile_of(c) < c.tile_end ? min(s1, c.u + per) : c.u;
  };

  // ---- loads, which run kDepth steps ahead
  Cursor ld = {item0 / tiles, 0, 0, 0, 0, 0, 0, 0, 0, 0};
  const int row8 = lane >> 3, chunk8 = lane & 7;   // a copy instruction takes four rows of 128 bytes
  const uint8_t* ld_q[4];                          // the lane's chunk of rows row8, row8 + 4, ...
  uintptr_t ld_s, ld_z;                            // scales and zeros of row lane % 16
  const int scale_size = a.scale_f32 ? 4 : 2;
  uint32_t to_q[4];                                // where the chunks go in a stage
#pragma unroll
  for (int i = 0; i < 4; ++i) to_q[i] = (row8 + 4 * i) * (kStep / 2) + (chunk8 ^ swizzle(row8 + 4 * i)) * 16;
  auto rows_of = [&]() {
    const int n = tile_of(ld) * kTile;
    const int64_t base = static_cast<int64_t>(jobs.expert[ld.job]) * a.N;
    // rows behind the last read the last one and are not stored
#pragma unroll
    for (int i = 0; i < 4; ++i) ld_q[i] = a.q + (base + min(n + row8 + 4 * i, a.N - 1)) * (a.K / 2) + chunk8 * 16;
    const int64_t row = (base + min(n + (lane & 15), a.N - 1)) * groups;
    ld_s = reinterpret_cast<uintptr_t>(a.scale) + row * scale_size;
    ld_z = reinterpret_cast<uintptr_t>(a.zero) + row;
  };
  auto load = [&](uint32_t stage) {
    while (ld.u >= ld.end && ld.job <= last_job) {
      if (++ld.slice == ld.slices) {
        ld.slice = 0;
        ++ld.round;
        if (ld.tile + (ld.round << (kLogWarps - ld.lw)) >= ld.tile_end) {
          ld.round = 0;
          if (++ld.job > last_job) break;
          open_job(ld);
        }
      }
      open(ld);
      if (ld.u < ld.end) rows_of();
    }
    if (ld.job <= last_job) {
      const bool there = ld.u * kStep + chunk8 * 32 < a.K;
#pragma unroll
      for (int i = 0; i < 4; ++i) copy16(stage + to_q[i], ld_q[i] + ld.u * (kStep / 2), there);
      // aligned words around the row's scales; a word behind the last needed byte is not read
      const int r = lane & 15, n_groups = min(S::kGroups, groups - ld.u * S::kGroups);
      const int words = (static_cast<int>(ld_s & 3) + n_groups * scale_size + 3) / 4;
      const uintptr_t from = (ld_s & ~uintptr_t(3)) + ld.u * (S::kGroups * scale_size);
#pragma unroll
      for (int i = 0; i < S::kScaleWords / 2; ++i) {
        const int word = 2 * i + (lane >> 4);
        if (word < words)
          copy4(stage + S::kScales + (r * S::kScaleWords + word) * 4, reinterpret_cast<const void*>(from + 4 * word));
      }
      if (ZERO) {
        const uintptr_t z = ld_z + ld.u * S::kGroups;
#pragma unroll
        for (int i = 0; i < (S::kZeroWords + 1) / 2; ++i) {
          const int word = 2 * i + (lane >> 4);
          const uintptr_t at = (z & ~uintptr_t(3)) + 4 * word;
          if (word < S::kZeroWords && at < z + n_groups)
            copy4(stage + S::kZeros + (r * S::kZeroWords + word) * 4, reinterpret_cast<const void*>(at));
        }
      }
      ++ld.u;
    }
    copies_close();
  };
  open_job(ld);
  open(ld);
  if (ld.u < ld.end) rows_of();
#pragma unroll
  for (int i = 0; i < kDepth; ++i) load(ring + i * S::kBytes);

  // ---- products
  int slot = 0, par = 0;
  Cursor at = {item0 / tiles, 0, 0, 0, 0, 0, 0, 0, 0, 0};
  for (; at.job <= last_job; ++at.job) {
    open_job(at);
    const int cols = jobs.cols[at.job], first = jobs.first[at.job], wk = 1 << at.lw, at_once = kWarps >> at.lw;
    const int x_row = at.slice_steps * (kStep / 8) + 4;   // 16-byte chunks between staged rows: 64 bytes apart in the banks
    for (at.round = 0; at.tile + at.round * at_once < at.tile_end; ++at.round) {
      const int n0 = tile_of(at) * kTile;
      float sum[NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[t][i] = 0.0f;

      for (at.slice = 0; at.slice < at.slices; ++at.slice) {
        const int s0 = at.slice * at.slice_steps, s1 = min(steps, s0 + at.slice_steps);
        if (at.round == 0 || at.slices > 1) {
          // stage x: a 16-byte chunk holds eight k, stored as the pairs (0, 4), (2, 6), (1, 5), (3, 7); chunk j of quad
          // lane t of a group lies at 4 j + t
          __syncthreads();
          const int chunks = (s1 - s0) * (kStep / 8), held = (min(a.K, s1 * kStep) - s0 * kStep) / 8;   // zeros behind K
          if (tid < cols)
            x_from[tid] = static_cast<const T*>(a.x) + (jobs.list[first + tid] / a.per_row) * a.x_stride + static_cast<int64_t>(s0) * kStep;
          __syncthreads();
          for (int i = tid; i < chunks; i += kThreads) {
            const int in = i % (G / 8), to = i - in + (in % W) * 4 + in / W;
#pragma unroll 4
            for (int c = 0; c < cols; ++c) {
              uint4 v = make_uint4(0u, 0u, 0u, 0u);
              if (i < held) v = __ldg(reinterpret_cast<const uint4*>(x_from[c]) + i);
              const uint4 pairs = make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.y, v.w, 0x5410),
                                             __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x7632));
              if constexpr (EXACT) {
                xs[c * x_row + to] = pairs;
              } else {
                xs[c * x_row + to] = make_uint4(Mma<T>::staged(pairs.x), Mma<T>::staged(pairs.y), Mma<T>::staged(pairs.z), Mma<T>::staged(pairs.w));
                const float2 p = Mma<T>::widen(v.x), q = Mma<T>::widen(v.y), r = Mma<T>::widen(v.z), t = Mma<T>::widen(v.w);
                float total = ((p.x + p.y) + (q.x + q.y)) + ((r.x + r.y) + (t.x + t.y));
#pragma unroll
                for (int d = G / 16; d > 0; d >>= 1) total += __shfl_xor_sync(0xFFFFFFFFu, total, d);
                if (in == 0) xsum[i / (G / 8) * kCols + c] = total * (1.0f / Mma<T>::kUnit);
              }
            }
          }
          __syncthreads();
        }
        open(at);
        const int64_t row = static_cast<int64_t>(jobs.expert[at.job]) * a.N;
        // where the scales of the lane's two rows are in a stage (the same in every step: a step's scales are a multiple of
        // four bytes), and the low address bits of their zeros
        int s_at[2], z_low[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t r = static_cast<uint32_t>(row + min(n0 + gid + 8 * h, a.N - 1)) * static_cast<uint32_t>(groups);
          s_at[h] = S::kScales + (gid + 8 * h) * 4 * S::kScaleWords +
                    static_cast<int>((static_cast<uint32_t>(reinterpret_cast<uintptr_t>(a.scale)) + r * scale_size) & 3);
          z_low[h] = ZERO ? static_cast<int>(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(a.zero)) + r) : 0;
        }
        const uint8_t* x_at[NT];                   // lanes without a column stay on the zeros
        int x_step[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const bool has = 8 * t + gid < cols;
          x_at[t] = reinterpret_cast<const uint8_t*>((has ? xs + (8 * t + gid) * x_row + (at.u - s0) * (kStep / 8) : none) + quad);
          x_step[t] = has ? 2 * kStep : 0;
        }
        for (; at.u < at.end; ++at.u) {
          const uint8_t* const stage = smem + (warp * kDepth + slot) * S::kBytes;
          copies_wait<kDepth - 1>();
          __syncwarp();
          const float* const xs_at = xsum + (at.u - s0) * (S::kGroups * kCols) + 2 * quad;
          if (NT == 1 || cols <= 8) step<T, G, 1, NT, ZERO, EXACT>(a, stage, x_at, xs_at, at.u, s_at, z_low, gid, quad, sum);
          else step<T, G, NT, NT, ZERO, EXACT>(a, stage, x_at, xs_at, at.u, s_at, z_low, gid, quad, sum);
#pragma unroll
          for (int t = 0; t < NT; ++t) x_at[t] += x_step[t];
          __syncwarp();
          load(ring + slot * S::kBytes);
          slot = slot + 1 == kDepth ? 0 : slot + 1;
        }
        if (steps > kSumSteps) {
          // A long K comes in slices of up to kSumSteps: their sums meet in the thread's own places of `red`, with what the
          // additions lose.  The barriers in front of every slice's x end the reads of the round before.
          float *const all = &red[0][warp][0][0] + lane, *const lost = &red[1][warp][0][0] + lane;
          static_assert(4 * NT * 32 <= kCols * (kTile + 4), "a warp's part of red holds its threads' sums");
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int i = (4 * t + k) * 32;
              float v = at.slice > 0 ? all[i] : 0.0f, low = at.slice > 0 ? lost[i] : 0.0f;
              add_exactly(v, low, sum[t][k]);
              const bool done = at.slice == at.slices - 1;
              sum[t][k] = done ? joined(v, low) : 0.0f;
              if (done) continue;
              all[i] = v;
              lost[i] = low;
            }
          __syncwarp();
        }
      }

#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int k = 0; k < 4; ++k) sum[t][k] *= EXACT ? Mma<T>::kExactUnit : Mma<T>::kUnit;
      if (wk == 1) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int c = 8 * t + 2 * quad + (k & 1), n = n0 + gid + 8 * (k >> 1);
            if (c < cols && n < a.N && tile_of(at) < at.tile_end) store_result<T, EXACT>(a, jobs.list[first + c], n, sum[t][k]);
          }
      } else {
        // join the parts in order; the two halves of `red` alternate, so the one barrier of a round also ends the reads
        // of the round before
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int k = 0; k < 4; ++k) red[par][warp][8 * t + 2 * quad + (k & 1)][gid + 8 * (k >> 1)] = sum[t][k];
        __syncthreads();
        const int here = min(at_once, at.tile_end - at.tile - at.round * at_once);
        for (int i = tid; i < here * cols * kTile; i += kThreads) {
          const int r = i % kTile, c = i / kTile % cols, l = i / kTile / cols;
          float v = 0.0f;
          for (int k = 0; k < wk; ++k) v += red[par][l * wk + k][c][r];
          const int n = (at.tile + at.round * at_once + l) * kTile + r;
          if (n < a.N) store_result<T, EXACT>(a, jobs.list[first + c], n, v);
        }
        par ^= 1;
      }
    }
  }
}

template <typename T, int G, int NT, bool ZERO, bool EXACT>
cudaError_t launch_kernel(MatvecArgs a, cudaStream_t stream) {
  constexpr size_t kRing = static_cast<size_t>(kWarps) * kDepth * Stage<G, ZERO>::kBytes;
  constexpr size_t kStatic = sizeof(float) * 2 * kWarps * 8 * NT * (kTile + 4) + sizeof(Jobs) + 4 * kWarps + 8 * 8 * NT;
  constexpr size_t kX = kSmemMost - kRing - kStatic - 1024 - kStep * 2;      // for staged x and its group sums
  const auto kernel = matvec_w4_kernel<T, G, NT, ZERO, EXACT>;
  const int rows = a.pairs / a.per_row;             // a row that names an expert twice gives it a second job
  a.x_cols = rows < 8 * NT ? rows : 8 * NT;
  const int steps = (a.K + kStep - 1) / kStep;
  // steps that fit for one row, the sums of their groups, and the rest for staged rows, as much of it as the call can use
  constexpr size_t kSums = EXACT ? 0 : static_cast<size_t>(kStep / G) * 8 * NT * 4;
  const int most = min(static_cast<int>((kX - 64) / (kStep * 2 + kSums)), kSumSteps);
  a.slice_most = steps < most ? steps : most;
  size_t room = kX - a.slice_most * kSums;
  const size_t useful = static_cast<size_t>(a.x_cols) * (a.slice_most * kStep * 2 + 64);
  if (room > useful) room = useful;
  a.x_chunks = static_cast<int>(room / 16);
  const size_t smem = kRing + static_cast<size_t>(a.x_chunks) * 16 + kStep * 2 + a.slice_most * kSums;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_smem(kernel, kRing + kX + kStep * 2, done);
  if (e != cudaSuccess) return e;
  const int64_t items = static_cast<int64_t>((a.N + kTile - 1) / kTile) * a.pairs;
  return launch_pdl(kernel, dim3(static_cast<unsigned>(items < kNumSMs ? items : kNumSMs)), dim3(kThreads), smem, stream, a);
}

template <typename T, int G, int NT>
cudaError_t launch_kernel(const MatvecArgs& a, cudaStream_t stream) {
  if (a.zero) return a.out_f32 ? launch_kernel<T, G, NT, true, true>(a, stream) : launch_kernel<T, G, NT, true, false>(a, stream);
  return a.out_f32 ? launch_kernel<T, G, NT, false, true>(a, stream) : launch_kernel<T, G, NT, false, false>(a, stream);
}

template <typename T, int NT>
cudaError_t launch_group(const MatvecArgs& a, int G, cudaStream_t stream) {
  if (G == 128) return launch_kernel<T, 128, NT>(a, stream);
  if (G == 64) return launch_kernel<T, 64, NT>(a, stream);
  return launch_kernel<T, 32, NT>(a, stream);
}

template <typename T>
cudaError_t launch_matvec(const MatvecArgs& a, int G, cudaStream_t stream) {
  // One tile of eight columns where no expert can have more rows (a row chooses an expert once), and where at most four of
  // them are expected: an expert that has more all the same is read twice.
  const bool one = a.pairs / a.per_row <= 8 || (a.experts && a.pairs <= 4 * a.E);
  return one ? launch_group<T, 1>(a, G, stream) : launch_group<T, 2>(a, G, stream);
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" int moe_fp8_block_scale_matvec_w4(const void* x, int64_t x_stride, int dtype, const uint8_t* qweight,
                                             const void* scale, int scale_f32, const uint8_t* zero, const int32_t* experts,
                                             int pairs, int pairs_per_row, int E, int N, int K, int G, void* out,
                                             int out_f32, void* stream_v) {
  if (pairs < 0 || pairs > kMaxPairs || pairs_per_row < 1 || pairs % pairs_per_row != 0 || E < 1 || E > kMaxMatvecExperts ||
      N < 1 || N > (1 << 22) || K < 1 || K > (1 << 20) || (G != 32 && G != 64 && G != 128) || K % G != 0 || (dtype != MOE_B200_BF16 && dtype != MOE_B200_F16) ||
      (!experts && (E != 1 || pairs_per_row != 1)))
    return MOE_B200_EINVAL;
  if (pairs == 0) return MOE_B200_OK;
  if (!x || !qweight || !scale || !out || !aligned(scale, scale_f32 ? 4 : 2) || !aligned(out, out_f32 ? 4 : 2) || !aligned(experts, 4) || !aligned(x, 16) || (pairs > pairs_per_row && x_stride % 8 != 0) || !aligned(qweight, 16))
    return MOE_B200_EINVAL;
  MatvecArgs a = {x, x_stride, qweight, scale, zero, experts, pairs, pairs_per_row, E, N, K, scale_f32, out_f32, 1, 0, 0, out};
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  const cudaError_t e = dtype == MOE_B200_BF16 ? launch_matvec<__nv_bfloat16>(a, G, stream) : launch_matvec<__half>(a, G, stream);
  return launch_status(e, 1);
}
