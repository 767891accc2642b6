// Picks one token per row of logits from a uniform number given for the row: temperature, top-k, top-p, min-p.
//
// With x the row (NaN counts as -inf), m its maximum and T the temperature, a token's mass is w = exp((x - m) / T).  The tokens
// are ordered by descending x, ties by ascending index, and the first K of them are kept: K is at most k (top-k), at most the
// shortest prefix whose mass reaches p times that of the first k (top-p), and at most the number of tokens with w >= min_p.  The pick
// is the lowest index at which the running sum of kept masses, in the order of the indices, exceeds u times their total.
//
// Masses are whole numbers: round(w * 2^45), at most 2^18 of them in 64 bits.  A sum of whole numbers does not depend on its
// order, so histograms may be filled by atomics and a row's pick is the same whatever CTA, warp or lane adds first; the rounding
// moves a border of the cumulative distribution by 2^-46 a token, where 32-bit floating sums would move it by up to 2^-24 of the total,
// more than a token in the tail of a large vocabulary has.
//
// A cluster of CTAs takes a row, as many as leave every row's CTAs resident together.  A row crosses HBM once, and is in L1 or L2 when it
// is read again: twice in all for the plain draw, min-p, top-k up to 1280 (768 with one CTA a row; with top-p or not) and top-p alone; three to six times for larger k, for top-p
// behind them, at temperatures below 0.16 or where its window misses; and six times more for each threshold that search finds.  (Rows kept in shared memory as fp32 needed clusters of eight for 151,936 tokens, so 128
// rows four waves of CTAs in lockstep: 76 us for the plain draw and 88 with top-k, where two CTAs a row without it take 52 and 38.)
// A threshold (of top-k, of top-p) is found by narrowing down: a histogram of counts over the distance to the maximum, then, where
// the tokens up to the border's bin are few, a list of them that one CTA sorts and finishes; else a list of the border's bins alone.  Rows
// whose border lies among more (nearly) equal values than a list holds go through eight-bit histograms of the keys (search).  Top-p alone, the
// common case, has its histogram from the first pass, while the row crosses HBM: its bins lie on a ring and need no maximum.
//
// Measured, us a call in a graph with fp32 rows of 151,936 tokens out of HBM, one / 32 / 128 of them (12 us of HBM): plain draw 14 / 21 / 53, min-p 12 / 16 / 34, top-k
// 50 with top-p 19 / 25 / 41, top-p alone 31 / 43 / 88.  Few rows: the chain of reductions across the cluster, 1 to 2 us each.  Many: no unit is full (issue
// slots 49 to 60 %, fp64 12 to 21 %); it is 32 instructions for a token's mass (a power of two in 64 bits, rounded to a whole number) of every token within
// SPAN of the maximum - the plain draw and top-p have one such pass; min-p and top-k compare in 32 bits and leave few tokens to weigh - and their
// latency at two CTAs an SM, whose 64 registers a thread spill (some 850 bytes of loads in the whole kernel; 110 to 130 with one CTA an SM).
// The other ways, one / 128 rows: top-k 5000 34 / 105, with top-p 51 / 175; top-p at temperature 0.1 71 / 246; normal logits of deviation 0.05, top-p 119 / 485, top-k
// 5000 with top-p 236 / 1233; all logits equal, top-p 2300 / 13,100, top-k 5000 with top-p 3300 / 14,200: search adds 64-bit numbers to one bin of a histogram, one behind the
// other (a sort of 128 such rows takes 6000).
#ifndef QMK_SAMPLING_CUH_
#define QMK_SAMPLING_CUH_

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace qmk_sample {

namespace cg = cooperative_groups;

constexpr int THREADS = 512, WARPS = THREADS / 32;
constexpr int MAX_VOCAB = 1 << 18;               // masses of at most 2^45 in 63 bits
constexpr int MAX_CLUSTER = 8;
constexpr int GROUPS = (MAX_VOCAB / 4 + 1 + WARPS * 32 - 1) / (WARPS * 32);   // of 128 tokens, in a warp's range of a row: at most
constexpr int BINS = 2048;                       // of the distance to the maximum: 4 per thread
constexpr float SPAN = 32.5f;                    // times the temperature: masses further below the maximum round to nothing (e^-32.5 < 2^-46)
constexpr int MASS_BINS = 6 * THREADS;           // of masses, 2^(1/64) wide, down to 2^-48: 6 per thread
constexpr double ONE = 8192.0;                   // a mass of its bin's middle in a histogram of masses: 2^18 of them fit 32 bits
constexpr int KEY_BINS = 256;                    // of a histogram of keys: eight bits
constexpr int LIST = 2048;                       // tokens that one CTA sorts: EACH per thread
constexpr int STEPS = 64, COLUMNS = 16;            // of the table of powers, see power_polynomial
constexpr int TURN = 3;                           // fours that a thread has in each of two turns of its ring
constexpr int NO_TOKEN = 0x7fffffff;             // pick of a row without a largest value, as in the greedy steps
constexpr float LARGEST_UNIFORM = 0x1.fffffep-1f;
constexpr float LARGEST_TEMPERATURE = 0x1p100f;  // (SPAN temperatures and the products with it stay finite)
constexpr int RING = 4096;                       // bins of the first pass' counts
constexpr float AROUND = 64.0f, SPAN_AROUND = 34.0f;     // logits, or temperatures where those are more, once round them: more than 1.01 SPAN and the rounding
constexpr float COUNT = 8192.0f;                 // a token in the middle of its bin there: 2^18 of them fit 32 bits
constexpr int WINDOW = 200;                      // tokens to either side of the border that these counts suggest
constexpr int EACH = LIST / THREADS;
static_assert(BINS == 4 * THREADS && LIST == 4 * THREADS, "bins and list entries per thread");

struct Params {
  const void *logits;
  long long row_stride;                          // elements
  int vocab;
  const float *uniforms;
  const float *temperatures, *top_ps, *min_ps;   // per row, or null: the scalar for all
  const int *top_ks;
  float temperature, top_p, min_p;
  int top_k;
  int *tokens;
  float *logprobs;                               // may be null
};

// (sampling_launch.cuh)
cudaError_t launch_fp32(const Params &p, int rows, cudaStream_t stream);
cudaError_t launch_fp16(const Params &p, int rows, cudaStream_t stream);
cudaError_t launch_bf16(const Params &p, int rows, cudaStream_t stream);

struct __align__(16) Shared {
  unsigned int counts[RING];                     // this CTA's histogram, read by the cluster: of tokens (BINS) or of masses (MASS_BINS, RING)
  union {
    unsigned long long keys[2][KEY_BINS];    // search: histograms in turn, one is read while the next is filled
    unsigned long long sorted[LIST];
  };
  unsigned long long list[LIST];                 // this CTA's candidates
  double powers[STEPS * COLUMNS];                // 2^(j / 64), a column for each lane of half a warp
  unsigned long long warp[WARPS], warp_kept[WARPS], group[GROUPS];
  unsigned long long inbox[16][MAX_CLUSTER];     // one row per exchange of the cluster, see gather
  unsigned long long found[4], border[6];
  unsigned long long threshold;                  // written by the CTA that finds it
  int listed, collected;
};

static_assert(sizeof(Shared) % 16 == 0 && offsetof(Shared, keys) % 16 == 0, "vector accesses");

// Order of the values as whole numbers: larger value, larger key, zeros of both signs the same.  (x is not NaN.)
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
// A logit that is no number is left as it is by the loads: maxima pass over it and no comparison holds for it.
__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename V>
__device__ __forceinline__ V warp_sum(V v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A token's place in the order, larger is earlier: the key, then the lower index.
__device__ __forceinline__ unsigned long long place_of(float x, int index) {
  return (static_cast<unsigned long long>(key_of(x)) << 32) | static_cast<uint32_t>(~index);
}
__device__ __forceinline__ float value_of(unsigned long long place) {
  const uint32_t k = static_cast<uint32_t>(place >> 32);
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
__device__ __forceinline__ int index_of(unsigned long long place) { return static_cast<int>(~static_cast<uint32_t>(place)); }

// 2^(y / 64) for whole-number and fractional parts y = 64 n + j + r, |r| <= 1/2: 2^n times a table's 2^(j / 64) times 1 + r times the polynomial that agrees with
// (2^(r / 64) - 1) / r in four Chebyshev nodes (relative error 5e-15, the table's 2^-53).  A table halves the fp64 instructions, which the sums of
// masses are bound by: 15 a token without it, 9 with it.  Every half of a warp has columns of its own, so that lookups never collide.
__device__ __forceinline__ double power_polynomial(double r) {
  double q = 5.732857292414682e-10;
  q = fma(q, r, 2.1173168200092995e-07);
  q = fma(q, r, 5.864904955054418e-05);
  q = fma(q, r, 0.010830424696239445);
  return fma(q, r, 1.0);
}
// round(w * 2^45) for w in [0, 1] from w + 2^7, whose last bit is 2^-45
__device__ __forceinline__ unsigned long long mass_of(double w_and_128) {
  return static_cast<unsigned long long>(__double_as_longlong(w_and_128)) - 0x4060000000000000ull;
}

// Bitonic sort of `size` entries (a power of two, 32 to LIST), largest first, by the whole CTA; a short one by its first warp.
__device__ __forceinline__ void sort_descending(unsigned long long *v, int size, int tid) {
  __syncthreads();
  const bool short_one = size <= 64;
  if (!short_one || tid < 32) {
    for (int block = 2; block <= size; block <<= 1)
      for (int step = block >> 1; step > 0; step >>= 1) {
        for (int pair = tid; pair < size >> 1; pair += THREADS) {
          const int i = 2 * pair - (pair & (step - 1)), j = i + step;
          const unsigned long long a = v[i], b = v[j];
          if ((a < b) == ((i & block) == 0)) { v[i] = b; v[j] = a; }
        }
        if (short_one) __syncwarp(); else __syncthreads();
      }
  }
  __syncthreads();
}

// Four logits from an address that is a multiple of their size
__device__ __forceinline__ float4 load_four(const float *p) { return *reinterpret_cast<const float4 *>(p); }
__device__ __forceinline__ float4 load_four(const __half *p) {
  const uint2 a = *reinterpret_cast<const uint2 *>(p);
  const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&a.x)), g = __half22float2(*reinterpret_cast<const __half2 *>(&a.y));
  return make_float4(f.x, f.y, g.x, g.y);
}
__device__ __forceinline__ float4 load_four(const __nv_bfloat16 *p) {
  const uint2 a = *reinterpret_cast<const uint2 *>(p);
  return make_float4(__uint_as_float(a.x << 16), __uint_as_float(a.x & 0xffff0000u), __uint_as_float(a.y << 16), __uint_as_float(a.y & 0xffff0000u));
}
// ... to shared memory, on their way until the thread waits for them
template <typename T>
__device__ __forceinline__ void copy_four(unsigned char *to, const T *from) {
  const uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(to));
  if (sizeof(T) == 4) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(from) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(from) : "memory");
}

// AN_SM: CTAs of an SM.  One has twice the registers (few rows), two hide each other's waits.
template <typename T, int AN_SM>
__global__ void __launch_bounds__(THREADS, AN_SM) sample_rows(const Params p) {
  extern __shared__ __align__(16) unsigned char smem[];
  Shared &s = *reinterpret_cast<Shared *>(smem);
  unsigned char *const ring = smem + sizeof(Shared);
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int row = static_cast<int>(blockIdx.x) / ranks, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // Tokens go in fours, each four within one aligned piece of memory: the first and the last of a row may be in part outside (-inf).  This CTA's
  // fours are [0, n4), four i begins with token first + 4 i; a warp has a range of them, in groups of 32 (128 tokens), of a group a thread has one.
  const T *const src = static_cast<const T *>(p.logits) + row * p.row_stride;
  const int off = static_cast<int>(reinterpret_cast<unsigned long long>(src) / sizeof(T) & 3), fours = (p.vocab + off + 3) >> 2;
  const int per_rank = (fours + ranks - 1) / ranks, first = 4 * rank * per_rank - off, n4 = max(0, min(per_rank, fours - rank * per_rank));
  const int seg = (n4 + WARPS * 32 - 1) / (WARPS * 32) * 32, seg_lo = min(n4, warp * seg), seg_hi = min(n4, seg_lo + seg);
  const int whole_lo = first < 0 ? 1 : 0, whole_hi = first + 4 * n4 > p.vocab ? n4 - 1 : n4;        // fours [whole_lo, whole_hi) are all inside
  bool infinite = false;                         // the largest value is: it counts as 0 and everything else as -inf
  auto counted = [&](float4 v) {
    if (infinite) v = make_float4(v.x == INFINITY ? 0.0f : -INFINITY, v.y == INFINITY ? 0.0f : -INFINITY, v.z == INFINITY ? 0.0f : -INFINITY, v.w == INFINITY ? 0.0f : -INFINITY);
    return v;
  };
  auto fetch = [&](int i) {
    const int at = first + 4 * i;
    if (i >= whole_lo && i < whole_hi) return counted(load_four(src + at));
    return counted(make_float4(at >= 0 ? as_float(src[at]) : -INFINITY, at + 1 >= 0 && at + 1 < p.vocab ? as_float(src[at + 1]) : -INFINITY,
                               at + 2 >= 0 && at + 2 < p.vocab ? as_float(src[at + 2]) : -INFINITY, at + 3 < p.vocab ? as_float(src[at + 3]) : -INFINITY));
  };
  // f(values, four, which of 0 .. TURN - 1 in turn) for this thread's fours.  A thread copies them to slots of its own in shared memory, TURN at a time, the
  // next ones under way while these are worked on.
  auto walk = [&](auto &&f) {
    constexpr int SLOT = THREADS * 4 * sizeof(T);
    int i = seg_lo + lane;
    if (seg_lo < whole_lo && seg_lo < seg_hi) {  // (the row's first four, not all of it inside: its group by itself)
      if (i < seg_hi) f(fetch(i), i, 0);
      i += 32;
    }
    const int whole = min(seg_hi, whole_hi), steps = whole > i ? (whole - i + 31) >> 5 : 0;      // (of this thread)
    const T *from = src + (first + 4 * i);
    unsigned char *slots = ring + tid * (4 * sizeof(T));
    auto copy = [&](int k, unsigned char *to) {
#pragma unroll
      for (int j = 0; j < TURN; ++j)
        if (k + j < steps) copy_four(to + j * SLOT, from + 128 * (k + j));
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    copy(0, slots);
    copy(TURN, slots + TURN * SLOT);
    int k = 0;
    unsigned char *here = slots, *there = slots + TURN * SLOT;
    for (; k + TURN <= steps; k += TURN) {
      asm volatile("cp.async.wait_group 1;" ::: "memory");
#pragma unroll
      for (int j = 0; j < TURN; ++j) f(counted(load_four(reinterpret_cast<const T *>(here + j * SLOT))), i + 32 * (k + j), j);
      copy(k + 2 * TURN, here);
      unsigned char *const next = there;
      there = here;
      here = next;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
    for (int j = 0; j < TURN - 1; ++j)
      if (k + j < steps) f(counted(load_four(reinterpret_cast<const T *>(here + j * SLOT))), i + 32 * (k + j), j);
    i += 32 * steps;
    if (i < seg_hi) f(fetch(i), i, 0);           // (the row's last four)
    __syncwarp();
  };
  const float asked = p.temperatures ? p.temperatures[row] : p.temperature, temperature = fminf(asked, LARGEST_TEMPERATURE);
  const float top_p = p.top_ps ? p.top_ps[row] : p.top_p, min_p = p.min_ps ? p.min_ps[row] : p.min_p;
  const int top_k = p.top_ks ? p.top_ks[row] : p.top_k;
  const float u_raw = p.uniforms[row];
  const double u = u_raw >= 0.0f ? fminf(u_raw, LARGEST_UNIFORM) : 0.0f;
  const double slope = STEPS * 1.4426950408889634 / static_cast<double>(temperature);       // 64ths of powers of two per unit of a logit
  const double least = min_p > 0.0f ? static_cast<double>(min_p) : 0.0, log_least = least > 0.0 ? log(least) : 0.0;
  int exchange = 0;                              // rows of Shared::inbox are used in turn
  cluster.barrier_arrive();                      // (waited for in front of the first store to another CTA)

  // One value of every CTA to every CTA, in the order of the ranks; what the CTA wrote before is there for the others behind it.  (Written
  // to the others, whose threads read their own shared memory: eight loads from other SMs one behind the other took 2 us.)
  auto gather = [&](unsigned long long mine, auto &&take) {
    const int slot = exchange++ & 15;
    if (tid < ranks) *cluster.map_shared_rank(&s.inbox[slot][rank], tid) = mine;
    cluster.sync();
    for (int r = 0; r < ranks; ++r) take(r, s.inbox[slot][r]);
  };
  // sum over the CTA, to all threads; `before`: of the threads in front of this one
  auto block_sum = [&](unsigned long long v) {
    v = warp_sum(v);
    __syncthreads();
    if (lane == 0) s.warp[warp] = v;
    __syncthreads();
    unsigned long long total = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) total += s.warp[w];
    return total;
  };
  auto block_scan = [&](unsigned long long v, unsigned long long &before) {
    unsigned long long run = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long up = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += up;
    }
    __syncthreads();
    if (lane == 31) s.warp[warp] = run;
    __syncthreads();
    unsigned long long total = 0, ahead = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      ahead += w < warp ? s.warp[w] : 0;
      total += s.warp[w];
    }
    before = ahead + run - v;
    return total;
  };

  // ---- the row, once; its largest value and where that is first
  for (int b = tid; b < RING / 4; b += THREADS) reinterpret_cast<uint4 *>(s.counts)[b] = make_uint4(0, 0, 0, 0);
  if (tid == 0) { s.listed = 0; s.collected = 0; }
  for (int i = tid; i < STEPS * COLUMNS; i += THREADS) s.powers[i] = exp2(static_cast<double>(i / COLUMNS) / STEPS);      // (read behind the first barrier)
  float high[TURN] = {-INFINITY, -INFINITY, -INFINITY};          // the largest values of three parts of what this thread has seen
  // Top-p alone: a histogram, too, over the value's place on a ring of bins, which needs no maximum (near_border), of masses in units of
  // the bin's middle.  What is further below the thread's maximum so far than any mass reaches is left out.
  const float grain = RING / fmaxf(AROUND, SPAN_AROUND * temperature), step = 1.0f / (grain * temperature);      // bins per logit, a bin's width in temperatures
  const bool counting = top_p < 1.0f && !(top_k > 0 && top_k < p.vocab) && asked > 0.0f && step < 0.1f;
  auto ring_bin = [&](float v) { return __float_as_int(fmaf(v, grain, 12582912.0f)); };      // (1.5 * 2^23: the nearest whole number in the low bits)
  auto count = [&](float v) {
    const float b = fmaf(v, grain, 12582912.0f), r = fmaf(v, grain, 12582912.0f - b) * step;
    atomicAdd(&s.counts[__float_as_int(b) & (RING - 1)], static_cast<unsigned int>(__float_as_int(fmaf(fmaf(r, 0.5f, 1.0f) * r, COUNT, 8388608.0f + COUNT)) & 0x3fff));
  };
  if (counting) {
    __syncthreads();                             // (the counts are 0)
    walk([&](float4 v, int, int j) {
      high[j] = fmaxf(fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)), high[j]);
      const float low = fmaxf(fmaf(-1.01f * SPAN, temperature, high[j]), -3.4e38f);
      if (v.x >= low && v.y >= low && v.z >= low && v.w >= low) {      // (nearly always)
        count(v.x); count(v.y); count(v.z); count(v.w);
        return;
      }
      if (v.x >= low) count(v.x);
      if (v.y >= low) count(v.y);
      if (v.z >= low) count(v.z);
      if (v.w >= low) count(v.w);
    });
  } else {
    walk([&](float4 v, int, int j) { high[j] = fmaxf(fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)), high[j]); });
  }
  float top;
  {
    uint32_t best = __reduce_max_sync(0xffffffffu, key_of(fmaxf(fmaxf(high[0], high[1]), high[2])));
    if (lane == 0) s.warp[warp] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w) best = max(best, static_cast<uint32_t>(s.warp[w]));
    const uint32_t mine = best;
    cluster.barrier_wait();
    gather(mine, [&](int, unsigned long long v) { best = max(best, static_cast<uint32_t>(v)); });
    top = value_of(static_cast<unsigned long long>(best) << 32);
  }
  // every token of this CTA: f(value, index)
  auto each = [&](auto &&f) {
    walk([&](float4 v, int i, int) {
      const int at = first + 4 * i;
      f(v.x, at); f(v.y, at + 1); f(v.z, at + 2); f(v.w, at + 3);
    });
  };
  // the same where f has nothing to do for values below `bound`, which most are
  auto each_from = [&](float bound, auto &&f) {
    walk([&](float4 v, int i, int) {
      if (!(fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) >= bound)) return;
      const int at = first + 4 * i;
      f(v.x, at); f(v.y, at + 1); f(v.z, at + 2); f(v.w, at + 3);
    });
  };
  const bool empty = top == -INFINITY;
  if (empty || !(asked > 0.0f) || top_k == 1 || min_p > 1.0f) {      // (no mass is above that of the largest value: the first of the order stays alone)
    uint32_t at = 0xffffffffu;
    if (!empty) each_from(top, [&](float v, int i) { if (v == top) at = min(at, static_cast<uint32_t>(i)); });
    at = __reduce_min_sync(0xffffffffu, at);
    if (lane == 0) s.warp[warp] = at;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w) at = min(at, static_cast<uint32_t>(s.warp[w]));
    const uint32_t mine = at;
    gather(mine, [&](int, unsigned long long v) { at = min(at, static_cast<uint32_t>(v)); });
    if (rank == 0 && tid == 0) {
      p.tokens[row] = empty ? NO_TOKEN : static_cast<int>(at);
      if (p.logprobs) p.logprobs[row] = empty ? NAN : 0.0f;
    }
    cluster.sync();                              // (nobody leaves while its shared memory is read)
    return;
  }
  if (top == INFINITY) {                         // infinite logits share the mass, whatever the others are
    infinite = true;
    top = 0.0f;
#pragma unroll
    for (int j = 0; j < TURN; ++j) high[j] = high[j] == INFINITY ? 0.0f : -INFINITY;
  }

  const double top64 = top;
  const float nothing = fmaf(-1.01f * SPAN, temperature, top);      // below it masses round to 0 (and the exponent of 2 may be any)
  const double *const powers = s.powers + (lane & (COLUMNS - 1));
  // 2^n 2^(j / 64) and the polynomial whose product is the mass of v
  auto factors = [&](float v, double &power, int &k) {
    constexpr double magic = 6755399441055744.0;             // 1.5 * 2^52: the sum's low word is the nearest whole number
    const double d = static_cast<double>(v) - top64, y = fma(d, slope, magic);
    k = __double2loint(y);
    const double p = powers[(k & (STEPS - 1)) * COLUMNS];
    power = __hiloint2double(__double2hiint(p) + ((k >> 6) << 20), __double2loint(p));
    return power_polynomial(fma(d, slope, -(y - magic)));
  };
  auto weight = [&](float v) { double power; int k; const double q = factors(v, power, k); return power * q; };
  // ... and the bin of masses, 64ths of a power of two below the maximum, with the mass in units of its bin's middle (ONE)
  auto mass_and_bin = [&](float v, int &bin, unsigned int &units) {      // (chosen behind the arithmetic: four tokens' run side by side)
    double power;
    int k;
    const double q = factors(v, power, k);
    const unsigned long long m = mass_of(fma(power, q, 128.0));
    units = static_cast<unsigned int>(__double2loint(fma(q, ONE, 4503599627370496.0)));
    bin = v >= nothing ? -k : MASS_BINS;
    return v >= nothing ? m : 0ull;
  };
  auto mass = [&](float v) { int bin; unsigned int units; return mass_and_bin(v, bin, units); };
  auto mass_bin = [&](float v) { return v >= nothing ? -__double2loint(fma(static_cast<double>(v) - top64, slope, 6755399441055744.0)) : MASS_BINS; };
  // no value of the bins 0 .. j of masses is below this
  auto mass_bound = [&](int j) { return top - (static_cast<float>(j) + 0.51f) * temperature * (0.6931472f / STEPS) * (1.0f + 1e-5f) - 1e-6f * fabsf(top); };
  // min_p: a bound for the values that stay, a little low, and the mass of those that do
  const float least_value = least > 0.0 ? static_cast<float>(top64 + log_least * static_cast<double>(temperature) * (1.0 + 1e-6) - 1e-6 * fabs(top64)) : -INFINITY;
  auto above_least = [&](float v) {
    const unsigned long long m = mass(v);
    return weight(v) >= least || v == top ? m : 0ull;
  };
  const double share = top_p > 0.0f ? static_cast<double>(top_p) : 0.0;
  auto share_of = [&](unsigned long long total) {        // of the ranks, those in front of which the mass is below this stay
    const unsigned long long t = __double2ull_ru(share * __ull2double_rn(total));
    return t < 1 ? 1ull : t < total ? t : total;
  };
  auto draw_from = [&](unsigned long long total) { return __double2ull_rd(u * __ull2double_rn(total)); };
  auto write = [&](int index, float v, unsigned long long total) {
    p.tokens[row] = index;
    const double z = v == top ? 0.0 : (static_cast<double>(v) - static_cast<double>(top)) / static_cast<double>(temperature);
    if (p.logprobs) p.logprobs[row] = static_cast<float>(z - log(__ull2double_rn(total) * 0x1p-45));
  };
  // The lowest index of the row at which the running sum of `value` exceeds `target(total)`; one thread calls found(index, x, total).
  // Values below `bound` have none.  find: the same where the sums of the warps' ranges are in `sums` and `mine` is the CTA's.
  auto four = [&](float bound, auto &&value, int i, unsigned long long (&v)[4], const float4 f) {
    const int at = first + 4 * i;
    v[0] = v[1] = v[2] = v[3] = 0;
    if (!(fmaxf(fmaxf(f.x, f.y), fmaxf(f.z, f.w)) >= bound)) return;
    v[0] = value(f.x, at); v[1] = value(f.y, at + 1); v[2] = value(f.z, at + 2); v[3] = value(f.w, at + 3);
  };
  auto warp_scan = [&](unsigned long long v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long up = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += up;
    }
    return v;
  };
  auto find = [&](unsigned long long mine, const unsigned long long *sums, float bound, auto &&value, auto &&target, auto &&found) {
    unsigned long long before = 0, total = 0, v[4];
    float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    gather(mine, [&](int r, unsigned long long c) { before += r < rank ? c : 0; total += c; });
    const unsigned long long want = target(total);
    if (!(before <= want && want < before + mine)) return;     // (the same for every thread of the CTA)
    int w = 0;
    for (; w < WARPS - 1 && before + sums[w] <= want; ++w) before += sums[w];
    const int lo = min(n4, w * seg), hi = min(n4, lo + seg), groups = (hi - lo + 31) >> 5;
    for (int g = warp; g < groups; g += WARPS) {
      v[0] = v[1] = v[2] = v[3] = 0;
      if (lo + 32 * g + lane < hi) four(bound, value, lo + 32 * g + lane, v, fetch(lo + 32 * g + lane));
      const unsigned long long sum = warp_sum((v[0] + v[1]) + (v[2] + v[3]));
      if (lane == 0) s.group[g] = sum;
    }
    __syncthreads();
    if (warp != 0) return;
    int g = 0;
    for (int g0 = 0; g0 < groups; g0 += 32) {                  // the group
      const unsigned long long sum = g0 + lane < groups ? s.group[g0 + lane] : 0, run = warp_scan(sum);
      const unsigned int over = __ballot_sync(0xffffffffu, want < before + run);
      if (over) {
        g = g0 + __ffs(over) - 1;
        before += __shfl_sync(0xffffffffu, run - sum, __ffs(over) - 1);
        break;
      }
      before += __shfl_sync(0xffffffffu, run, 31);
    }
    v[0] = v[1] = v[2] = v[3] = 0;
    const int i = lo + 32 * g + lane;
    if (i < hi) { f = fetch(i); four(bound, value, i, v, f); }
    const unsigned long long own = (v[0] + v[1]) + (v[2] + v[3]);
    before += warp_scan(own) - own;
    const float x[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (before <= want && want < before + v[j]) found(first + 4 * i + j, x[j], total);
      before += v[j];
    }
  };
  auto pick = [&](float bound, auto &&value, auto &&target, auto &&found) {
    unsigned long long sum = 0;
    walk([&](float4 f, int i, int) {
      unsigned long long v[4];
      four(bound, value, i, v, f);
      sum += (v[0] + v[1]) + (v[2] + v[3]);
    });
    find(block_sum(sum), s.warp, bound, value, target, found);
  };

  // s.sorted[0 .. count) to descending order, by `key`, a number that does not grow along it: entries go to 2048 buckets between the largest and the
  // smallest key, and each finds its place among its bucket's few.  (With a bitonic sort of 2048, a row of 151,936 tokens with top-k 1000 and
  // top-p took 40 us; it takes 20.)  Crowded buckets and short lists
  // are left to the bitonic sort.
  auto sort_by = [&](int count, auto &&key) {
    int size = 32;
    while (size < count) size <<= 1;
    if (size > 32) {
      unsigned long long c[EACH];
      float k[EACH], high = -INFINITY, low = INFINITY;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < EACH; ++j) {
        const int i = tid + j * THREADS;
        c[j] = i < count ? s.sorted[i] : 0;
        k[j] = i < count ? key(c[j]) : 0.0f;
        if (i < count) { high = fmaxf(high, k[j]); low = fminf(low, k[j]); }
        s.counts[i] = 0;
      }
      const uint32_t up = __reduce_max_sync(0xffffffffu, key_of(high)), down = __reduce_min_sync(0xffffffffu, key_of(low));
      if (lane == 0) s.warp[warp] = (static_cast<unsigned long long>(up) << 32) | down;
      __syncthreads();
      uint32_t top_key = 0, low_key = 0xffffffffu;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) { top_key = max(top_key, static_cast<uint32_t>(s.warp[w] >> 32)); low_key = min(low_key, static_cast<uint32_t>(s.warp[w])); }
      high = value_of(static_cast<unsigned long long>(top_key) << 32);
      low = value_of(static_cast<unsigned long long>(low_key) << 32);
      const float scale = high > low ? (BINS - 1) / (high - low) : 0.0f;
      int b[EACH], slot[EACH];
#pragma unroll
      for (int j = 0; j < EACH; ++j) {
        b[j] = min(max(static_cast<int>((high - k[j]) * scale), 0), BINS - 1);
        slot[j] = tid + j * THREADS < count ? static_cast<int>(atomicAdd(&s.counts[b[j]], 1u)) : 0;
      }
      __syncthreads();
      const uint4 n4_ = reinterpret_cast<const uint4 *>(s.counts)[tid];
      unsigned long long before;
      block_scan(static_cast<unsigned long long>(n4_.x) + n4_.y + n4_.z + n4_.w, before);
      const uint32_t at = static_cast<uint32_t>(before);
      reinterpret_cast<uint4 *>(s.counts)[tid] = make_uint4(at, at + n4_.x, at + n4_.x + n4_.y, at + n4_.x + n4_.y + n4_.z);
      const bool crowded = __syncthreads_or(max(max(n4_.x, n4_.y), max(n4_.z, n4_.w)) > 256);
      if (!crowded) {
#pragma unroll
        for (int j = 0; j < EACH; ++j)
          if (tid + j * THREADS < count) s.sorted[s.counts[b[j]] + slot[j]] = c[j];
        __syncthreads();
        int place[EACH];
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
          place[j] = 0;
          if (tid + j * THREADS < count) {
            const int from = static_cast<int>(s.counts[b[j]]), to = b[j] + 1 < BINS ? static_cast<int>(s.counts[b[j] + 1]) : count;
            place[j] = from;
            for (int i = from; i < to; ++i) place[j] += s.sorted[i] > c[j];
          }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < EACH; ++j)
          if (tid + j * THREADS < count) s.sorted[place[j]] = c[j];
        __syncthreads();
        return;
      }
    }
    for (int i = count + tid; i < size; i += THREADS) s.sorted[i] = 0;
    sort_descending(s.sorted, size, tid);
  };

  // Candidates: to the CTA's own list, then (collect) to rank 0's, in any order, where they are sorted, largest first.  Their number in all;
  // more than LIST: nothing is sorted.  The others have nothing more to give rank 0 then and may leave.
  auto list = [&](float v, int i) {
    const int at = atomicAdd(&s.listed, 1);
    if (at < LIST) s.list[at] = place_of(v, i);
  };
  auto collect = [&]() {
    __syncthreads();
    const int mine = s.listed;
    if (tid == 0) s.found[3] = mine > 0 ? atomicAdd(cluster.map_shared_rank(&s.collected, 0), mine) : 0;
    __syncthreads();
    const unsigned long long base = s.found[3];
    if (mine > 0 && base + mine <= LIST) {
      unsigned long long *const to = cluster.map_shared_rank(s.sorted, 0) + base;
      for (int i = tid; i < mine; i += THREADS) to[i] = s.list[i];
    }
    int total = 0;
    gather(mine, [&](int, unsigned long long c) { total += static_cast<int>(c); });
    if (rank == 0 && total <= LIST) sort_by(total, [](unsigned long long place) { return value_of(place); });
    return total;
  };
  // rank 0: the threshold behind the sorted candidate number `count` (from 1 on), to every CTA
  auto announce = [&](int count) {
    const unsigned long long at = s.sorted[count - 1];
    if (tid < ranks) *cluster.map_shared_rank(&s.threshold, tid) = at;
  };
  // Rank 0, where the list holds every token that may stay: the first k of it, of those the ones that top-p (`want`: their mass, 0 where it is
  // a share of the list's) and min_p leave, then these by index and the pick among them.
  auto finish_list = [&](int total, unsigned long long k, unsigned long long want) {
    const int limit = static_cast<int>(min(static_cast<unsigned long long>(total), k));
    unsigned long long c[EACH], m[EACH], before, sum = 0;
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      c[j] = EACH * tid + j < limit ? s.sorted[EACH * tid + j] : 0;
      m[j] = EACH * tid + j < limit ? mass(value_of(c[j])) : 0;
      sum += m[j];
    }
    const unsigned long long all = block_scan(sum, before);
    if (top_p < 1.0f) want = want ? want : share_of(all); else want = ~0ull;
    int stay = 0;
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      const bool keep = EACH * tid + j < limit && before < want && (EACH * tid + j == 0 || least == 0.0 || above_least(value_of(c[j])));
      stay += __syncthreads_count(keep);
      before += m[j];
    }
#pragma unroll
    for (int j = 0; j < EACH; ++j)                // the halves change places: by index, the lowest (its complement the largest) first
      if (EACH * tid + j < stay) s.sorted[EACH * tid + j] = (c[j] << 32) | (c[j] >> 32);
    sort_by(stay, [](unsigned long long swapped) { return -static_cast<float>(~static_cast<uint32_t>(swapped >> 32)); });
    sum = 0;
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      c[j] = EACH * tid + j < stay ? s.sorted[EACH * tid + j] : 0;
      c[j] = (c[j] << 32) | (c[j] >> 32);
      m[j] = EACH * tid + j < stay ? mass(value_of(c[j])) : 0;
      sum += m[j];
    }
    const unsigned long long kept = block_scan(sum, before), at = draw_from(kept);
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      if (before <= at && at < before + m[j]) write(index_of(c[j]), value_of(c[j]), kept);
      before += m[j];
    }
  };

  // The place behind which the running sum of `value`, in the order, reaches target(total): eight bits of the key at a time, then the
  // ties by index.  `value` is 0 for tokens that are out already, and the same for equal values.
  auto search = [&](auto &&value, auto &&target) -> unsigned long long {
    uint32_t prefix = 0;
    unsigned long long want = 0, before = 0;
    cluster.sync();                              // (the space of the histograms was another's)
    for (int shift = 24, turn = 0; shift >= 0; shift -= 8, ++turn) {
      unsigned long long *const hist = s.keys[turn & 1];
      if (tid < KEY_BINS) hist[tid] = 0;
      __syncthreads();
      each([&](float v, int i) {
        if (!(v == v)) return;
        const uint32_t k = key_of(v);
        if (shift < 24 && (k >> (shift + 8)) != prefix) return;
        if (i < 0 || i >= p.vocab) return;
        const unsigned long long c = value(v, i);
        if (c) atomicAdd(&hist[(k >> shift) & (KEY_BINS - 1)], c);
      });
      cluster.sync();
      unsigned long long c = 0, ahead;
      const int bin = KEY_BINS - 1 - tid;
      if (tid < KEY_BINS) {
#pragma unroll
        for (int r = 0; r < MAX_CLUSTER; ++r) c += r < ranks ? cluster.map_shared_rank(hist, r)[bin] : 0;
      }
      const unsigned long long total = block_scan(c, ahead);
      if (shift == 24) want = target(total);
      if (tid == 0) s.found[0] = s.found[1] = 0;
      __syncthreads();
      if (before + ahead < want && want <= before + ahead + c) { s.found[0] = bin; s.found[1] = before + ahead; }
      __syncthreads();
      prefix = (prefix << 8) | static_cast<uint32_t>(s.found[0]);
      before = s.found[1];
    }
    // tokens of the border's value: as many as the sum in front of them leaves room for
    if (tid == 0) s.threshold = 0;
    const uint32_t key = prefix;
    unsigned long long one = 0;
    each([&](float v, int i) { if (i >= 0 && i < p.vocab && v == v && key_of(v) == key) { const unsigned long long c = value(v, i); one = c > one ? c : one; } });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { const unsigned long long other = __shfl_xor_sync(0xffffffffu, one, o); one = other > one ? other : one; }
    __syncthreads();
    if (lane == 0) s.warp[warp] = one;
    __syncthreads();
    for (int w = 0; w < WARPS; ++w) one = s.warp[w] > one ? s.warp[w] : one;
    const unsigned long long mine = one;
    gather(mine, [&](int, unsigned long long v) { one = v > one ? v : one; });
    const unsigned long long room = one ? (want - before + one - 1) / one : 1;
    pick(-INFINITY, [&](float v, int i) -> unsigned long long { return i >= 0 && i < p.vocab && v == v && key_of(v) == key && value(v, i) != 0; },
         [&](unsigned long long) { return room - 1; },
         [&](int i, float v, unsigned long long) { for (int r = 0; r < ranks; ++r) *cluster.map_shared_rank(&s.threshold, r) = place_of(v, i); });
    cluster.sync();
    return s.threshold;
  };

  // Bins of the distance to the maximum, bin j around j / per_bin.  Differences, products and rounding are monotonous, so a bin is a
  // range of the order.
  const float per_bin = fminf(static_cast<float>(BINS) / (SPAN * temperature), 3e38f);
  auto bin_of = [&](float v) {                   // BINS or more: out
    const float b = fmaf(top - v, per_bin, 8388608.0f);        // (the last bit is 1: rounded to the nearest whole number)
    return b < 8388608.0f + BINS ? static_cast<int>(__float_as_uint(b) & 0xffffu) : BINS;
  };
  // no value of the bins 0 .. j is below this
  auto bound_of = [&](int j) { return top - (static_cast<float>(j) + 0.51f) / per_bin * (1.0f + 1e-5f) - 1e-6f * fabsf(top); };
  auto clear_counts = [&]() { for (int b = tid; b < RING / 4; b += THREADS) reinterpret_cast<uint4 *>(s.counts)[b] = make_uint4(0, 0, 0, 0); };
  // The cluster's histogram: a CTA adds up its share of the bins, of which a thread has up to six, one behind the other.  (Every CTA reading
  // all of the others' bins took 10 us.)
  struct Share { unsigned int c[6]; int bin, mine; };
  auto share_of_bins = [&](int bins) {
    Share h;
    const int all = bins / ranks, each_ = (all + THREADS - 1) / THREADS;
    h.bin = rank * all + tid * each_;
    h.mine = max(0, min(each_, all - tid * each_));
#pragma unroll
    for (int j = 0; j < 6; ++j) {
      h.c[j] = 0;
      if (j < h.mine) {
#pragma unroll
        for (int r = 0; r < MAX_CLUSTER; ++r) h.c[j] += r < ranks ? cluster.map_shared_rank(s.counts, r)[h.bin + j] : 0;
      }
    }
    return h;
  };
  // The bin in which the running count reaches k, the counts in front of it and up to it, to every CTA (Shared::border); returns the count of all.
  auto count_border = [&](unsigned long long k) {
    const Share h = share_of_bins(BINS);
    unsigned long long before, front = 0, total = 0, sum = 0;
#pragma unroll
    for (int j = 0; j < 6; ++j) sum += h.c[j];
    const unsigned long long mine = block_scan(sum, before);
    gather(mine, [&](int r, unsigned long long v) { front += r < rank ? v : 0; total += v; });
    before += front;
#pragma unroll
    for (int j = 0; j < 6; ++j) {
      if (j < h.mine && before < k && k <= before + h.c[j])
        for (int r = 0; r < ranks; ++r) {
          unsigned long long *const to = cluster.map_shared_rank(s.border, r);
          to[0] = h.bin + j;
          to[1] = before;
          to[2] = before + h.c[j];
        }
      before += h.c[j];
    }
    cluster.sync();
    return total;
  };

  // Kept: tokens whose place is not below the threshold.
  float kept_value = -INFINITY;
  int kept_index = 0x7fffffff;
  bool cut = false;
  auto cut_at = [&](unsigned long long place) { kept_value = value_of(place); kept_index = index_of(place); cut = true; };
  auto kept = [&](float v, int i) { return v > kept_value || (v == kept_value && i <= kept_index); };
  if (top_k > 0 && top_k < p.vocab) {
    const unsigned long long k = static_cast<unsigned long long>(top_k);
    // Few: the largest values of the threads' parts are k tokens at least down to some bin, which leaves out most others without a look at them.
    if (top_k <= LIST * 5 / 8 && top_k * 2 <= min(TURN * ranks * THREADS, fours)) {
#pragma unroll
      for (int j = 0; j < TURN; ++j) {
        const int b = bin_of(high[j]);
        if (b < BINS) atomicAdd(&s.counts[b], 1u);
      }
      cluster.sync();
      const int border = count_border(k) < k ? BINS - 1 : static_cast<int>(s.border[0]);
      each_from(bound_of(border), [&](float v, int i) { if (bin_of(v) <= border) list(v, i); });
      const int total = collect();
      if (total <= LIST) {
        if (rank == 0) finish_list(total, k, 0);
        return;
      }
      clear_counts();
      if (tid == 0) { s.listed = 0; s.collected = 0; }
      cluster.sync();
    }
    each([&](float v, int) { const int b = bin_of(v); if (b < BINS) atomicAdd(&s.counts[b], 1u); });
    cluster.sync();
    if (count_border(k) > k) {                   // (otherwise every token that has a mass stays)
      const int border = static_cast<int>(s.border[0]);
      const unsigned long long above = s.border[1], up_to = s.border[2];
      if (up_to <= LIST) {
        each_from(bound_of(border), [&](float v, int i) { if (bin_of(v) <= border) list(v, i); });
        const int total = collect();
        if (rank == 0) finish_list(total, k, 0);
        return;
      }
      if (up_to - above <= LIST) {
        each_from(bound_of(border), [&](float v, int i) { if (bin_of(v) == border) list(v, i); });
        collect();
        if (rank == 0) announce(static_cast<int>(k - above));
        cluster.sync();
        cut_at(s.threshold);
      } else {
        cut_at(search([&](float, int) { return 1ull; }, [&](unsigned long long) { return k; }));
      }
    }
    cluster.sync();
    clear_counts();
    if (tid == 0) { s.listed = 0; s.collected = 0; }
    cluster.sync();                              // (rank 0's counter is the others')
  }
  // Where the border of top-p lies in the sorted list, `front` being the mass in front of the list's tokens; then the pick, where min_p takes nothing
  // away.  `mine`, `range`: the masses in front of them of this CTA and of this warp's range.
  auto settle = [&](unsigned long long front, unsigned long long mine, unsigned long long range, unsigned long long want) {
    const int listed = collect();
    if (rank == 0) {                             // how many of them stay
      unsigned long long w[EACH], before, all = 0;
#pragma unroll
      for (int j = 0; j < EACH; ++j) {
        w[j] = EACH * tid + j < listed ? mass(value_of(s.sorted[EACH * tid + j])) : 0;
        all += w[j];
      }
      block_scan(all, before);
      before += front;
      int stay = 0;
#pragma unroll
      for (int j = 0; j < EACH; ++j) {
        stay += __syncthreads_count(EACH * tid + j < listed && before < want);
        before += w[j];
      }
      announce(max(stay, 1));
    }
    cluster.sync();
    cut_at(s.threshold);
    if (least > 0.0 && weight(kept_value) < least) return false;
    if (lane == 0) s.warp_kept[warp] = range;    // the ranges' sums are there but for the listed tokens that stay
    __syncthreads();
    unsigned long long sum = 0;
    for (int i = tid; i < s.listed; i += THREADS) {
      const float v = value_of(s.list[i]);
      const int at = index_of(s.list[i]);
      const unsigned long long m = kept(v, at) ? mass(v) : 0;
      sum += m;
      if (m) atomicAdd(&s.warp_kept[((at - first) >> 2) / seg], m);
    }
    find(mine + block_sum(sum), s.warp_kept, kept_value, [&](float v, int i) -> unsigned long long { const unsigned long long m = mass(v); return kept(v, i) ? m : 0ull; }, draw_from, write);
    cluster.sync();
    return true;
  };
  // Three sums over the CTA, and over the cluster with those of the ranks in front.
  auto three_sums = [&](const unsigned long long (&v)[3], unsigned long long (&total)[3], unsigned long long (&front)[3]) {
    const int slot = exchange;
    exchange += 3;
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      if (tid < ranks) *cluster.map_shared_rank(&s.inbox[(slot + j) & 15][rank], tid) = v[j];
      total[j] = front[j] = 0;
    }
    cluster.sync();
    for (int r = 0; r < ranks; ++r)
#pragma unroll
      for (int j = 0; j < 3; ++j) {
        const unsigned long long c = s.inbox[(slot + j) & 15][r];
        front[j] += r < rank ? c : 0;
        total[j] += c;
      }
  };
  // Top-p from the counts of the first pass: they say near which token the border is.  One pass adds up the
  // masses, of all and of those in front of the WINDOW tokens to either side of it, which it lists; if the border is among them, the sums say
  // so, and the rest is as exact as without the counts.  (128 rows of 151,936 tokens: 133 us by the bins of masses below, 86 so; with p = 0.999 384 and 89.)
  enum { ELSEWHERE, LISTED, WRITTEN };
  unsigned long long front_mass = 0, front_mine = 0, front_range = 0, want_mass = 0;         // for settle, where the border's tokens are listed
  auto near_border = [&]() -> int {
    const int top_bin = ring_bin(top);
    const int all = RING / ranks, each_ = max(all / THREADS, 1), mine = tid * each_ < all ? each_ : 0, at0 = rank * all + tid * each_;
    uint32_t *const units = reinterpret_cast<uint32_t *>(s.sorted) + tid * each_;        // the cluster's, of this thread's bins
    static_assert(RING * sizeof(uint32_t) <= sizeof(s.sorted), "a CTA's share of the ring");
    auto tokens = [&](int j) { return static_cast<unsigned long long>((units[j] + static_cast<uint32_t>(COUNT / 2)) / static_cast<uint32_t>(COUNT)); };
    auto estimate = [&](int j) { return __float2ull_rn(static_cast<float>(units[j]) * exp2f(27.0f - static_cast<float>(at0 + j) * (step * 1.4426950f))); };
    unsigned long long sums[3] = {0, 0, 0}, before[2], total[3], front[3];
#pragma unroll 1
    for (int j = 0; j < mine; ++j) {
      uint32_t c = 0;
#pragma unroll
      for (int r = 0; r < MAX_CLUSTER; ++r) c += r < ranks ? cluster.map_shared_rank(s.counts, r)[(top_bin - at0 - j) & (RING - 1)] : 0;
      units[j] = c;
      sums[0] += tokens(j);
      sums[1] += estimate(j);
    }
    if (tid == 0) { s.border[0] = 0; s.border[1] = 0; s.border[2] = RING - 1; s.border[3] = 0; s.border[4] = ~0ull; }
    const unsigned long long own_tokens = sums[0], own_estimate = sums[1];
    sums[0] = block_scan(own_tokens, before[0]);
    sums[1] = block_scan(own_estimate, before[1]);
    three_sums(sums, total, front);
    const unsigned long long target = share_of(total[1]), n0 = front[0] + before[0];
    {
      unsigned long long run = front[1] + before[1], n = n0;
      if (run < target && target <= run + own_estimate)
#pragma unroll 1
        for (int j = 0; j < mine; ++j) {
          const unsigned long long e = estimate(j), c = tokens(j);
          if (run < target && target <= run + e) {
            const unsigned long long centre = n + static_cast<unsigned long long>(__ull2double_rn(c) * (__ull2double_rn(target - run) / __ull2double_rn(e)));
            for (int r = 0; r < ranks; ++r) cluster.map_shared_rank(s.border, r)[1] = centre;
          }
          run += e;
          n += c;
        }
    }
    cluster.sync();
    const unsigned long long centre = s.border[1], from_ = centre > 512 ? centre - WINDOW : 0, to_ = centre + WINDOW;   // (not many: all in front, too)
    if ((n0 < from_ && from_ <= n0 + own_tokens) || (n0 < to_ && to_ <= n0 + own_tokens)) {
      unsigned long long n = n0;
#pragma unroll 1
      for (int j = 0; j < mine; ++j) {
        const unsigned long long c = tokens(j);
        if (n < from_ && from_ <= n + c)
          for (int r = 0; r < ranks; ++r) { unsigned long long *const to = cluster.map_shared_rank(s.border, r); to[0] = at0 + j; to[3] = n; }
        if (n < to_ && to_ <= n + c)
          for (int r = 0; r < ranks; ++r) { unsigned long long *const to = cluster.map_shared_rank(s.border, r); to[2] = at0 + j; to[4] = n + c; }
        n += c;
      }
    }
    cluster.sync();
    const int lo = static_cast<int>(s.border[0]), hi = static_cast<int>(s.border[2]);
    if (min(s.border[4], total[0]) - s.border[3] > LIST * 7 / 8) return ELSEWHERE;        // (bins of many tokens; the counts are up to a tenth low)
    const int lo_bin = top_bin - lo, hi_bin = top_bin - hi;    // as ring_bin gives them: larger in front (tokens without a mass anywhere)
    const unsigned int width = static_cast<unsigned int>(lo_bin - hi_bin);
    unsigned long long v_sum[3] = {0, 0, 0};     // of all, in front of the window, in it
    walk([&](float4 v4, int i, int) {
      const float v[4] = {v4.x, v4.y, v4.z, v4.w};
      unsigned long long m[4];
      int b[4];
      bool at_border = false;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        m[j] = mass(v[j]);
        b[j] = ring_bin(v[j]);
        v_sum[0] += m[j];
        v_sum[1] += b[j] > lo_bin ? m[j] : 0;
        at_border = at_border || static_cast<unsigned int>(b[j] - hi_bin) <= width;
      }
      if (at_border) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (static_cast<unsigned int>(b[j] - hi_bin) <= width && v[j] >= nothing) { v_sum[2] += m[j]; list(v[j], first + 4 * i + j); }
      }
    });
    const unsigned long long range = warp_sum(v_sum[1]);
    const unsigned long long own[3] = {block_sum(v_sum[0]), block_sum(v_sum[1]), block_sum(v_sum[2])};
    three_sums(own, total, front);
    const unsigned long long want = share_of(total[0]);
    if (!(total[1] < want && want <= total[1] + total[2])) return ELSEWHERE;
    if (lo == 0) {
      const int listed = collect();
      if (rank == 0) finish_list(listed, ~0ull, want);
      return WRITTEN;
    }
    front_mass = total[1];
    front_mine = own[1];
    front_range = range;
    want_mass = want;
    return LISTED;
  };
  bool listed_border = false;
  if (counting) {
    int how = ELSEWHERE;
    // (bins of whole numbers that floats hold: then those of the massive tokens are in the order of the values, and none of them round the ring)
    if (!infinite && fabsf(top) * grain < 2097152.0f) how = near_border();
    if (how == WRITTEN) return;
    listed_border = how == LISTED;
    if (!listed_border) {
      cluster.sync();                            // (what the others read or write here has been)
      clear_counts();
      if (tid == 0) { s.listed = 0; s.collected = 0; }
      cluster.sync();
    }
  }
  if (top_p < 1.0f && !listed_border) {
    unsigned long long sum = 0;
    walk([&](float4 v4, int i, int) {              // (four tokens' arithmetic side by side, then the atomics)
      const float v[4] = {v4.x, v4.y, v4.z, v4.w};
      unsigned int units[4];
      int b[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        unsigned long long m = mass_and_bin(v[j], b[j], units[j]);
        if (cut && !kept(v[j], first + 4 * i + j)) { b[j] = MASS_BINS; m = 0; }
        sum += m;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (b[j] < MASS_BINS) atomicAdd(&s.counts[b[j]], units[j]);
    });
    // (as long as nobody finds them: the first bin with nothing in front, the last with everything up to it)
    if (tid == 0) { s.border[0] = 0; s.border[1] = 0; s.border[2] = MASS_BINS - 1; s.border[3] = ~0ull; }
    const unsigned long long own = block_sum(sum);
    unsigned long long total = 0;
    gather(own, [&](int, unsigned long long v) { total += v; });
    const unsigned long long want = share_of(total);
    // The border's bin, or a few that it may be in: units are rounded (6.1e-5 of them; the middle's power adds 2^-21), masses by 2^-46 each.
    const Share h = share_of_bins(MASS_BINS);
    unsigned long long low[6], high_[6], below, ahead, units_before, lows = 0, highs = 0, units_sum = 0;
#pragma unroll
    for (int j = 0; j < 6; ++j) {
      const double middle = exp2f(static_cast<float>(-(h.bin + j)) / STEPS), n_ = h.c[j] * (1.0 / ONE);
      low[j] = __double2ull_rd(n_ * fmax(middle * (1.0 - 6.5e-5) - 0x1.1p-46, 0.0) * 0x1p45);
      high_[j] = __double2ull_ru(n_ * (middle * (1.0 + 6.5e-5) + 0x1.1p-46) * 0x1p45);
      lows += low[j];
      highs += high_[j];
      units_sum += h.c[j];
    }
    const unsigned long long all_low = block_scan(lows, below), all_high = block_scan(highs, ahead), all_units = block_scan(units_sum, units_before);
    {
      const int slot = exchange;                 // three sums at once
      exchange += 3;
      if (tid < ranks) {
        *cluster.map_shared_rank(&s.inbox[slot & 15][rank], tid) = all_low;
        *cluster.map_shared_rank(&s.inbox[(slot + 1) & 15][rank], tid) = all_high;
        *cluster.map_shared_rank(&s.inbox[(slot + 2) & 15][rank], tid) = all_units;
      }
      cluster.sync();
      for (int r = 0; r < rank; ++r) { below += s.inbox[slot & 15][r]; ahead += s.inbox[(slot + 1) & 15][r]; units_before += s.inbox[(slot + 2) & 15][r]; }
    }
#pragma unroll
    for (int j = 0; j < 6; ++j) {
      if (j < h.mine) {
        if (ahead < want && want <= ahead + high_[j])
          for (int r = 0; r < ranks; ++r) { unsigned long long *const to = cluster.map_shared_rank(s.border, r); to[0] = h.bin + j; to[1] = units_before; }
        if (below < want && want <= below + low[j])
          for (int r = 0; r < ranks; ++r) { unsigned long long *const to = cluster.map_shared_rank(s.border, r); to[2] = h.bin + j; to[3] = units_before + h.c[j]; }
      }
      ahead += high_[j];
      below += low[j];
      units_before += h.c[j];
    }
    cluster.sync();
    const int lo = static_cast<int>(s.border[0]), hi = static_cast<int>(s.border[2]);
    // (a token is 0.994 ONE at least)
    const unsigned long long most = static_cast<unsigned long long>(0.99 * ONE) * LIST, units_to = s.border[3];
    const bool few = units_to <= most, few_at_border = units_to - s.border[1] <= most;
    if (few) {
      each_from(mass_bound(hi), [&](float v, int i) { if (mass_bin(v) <= hi && kept(v, i)) list(v, i); });
      const int listed = collect();
      if (rank == 0) finish_list(listed, ~0ull, want);
      return;
    }
    // The mass in front of the border's bins, exactly, and their tokens.
    unsigned long long front = 0;
    sum = 0;
    const float from = mass_bound(hi);
    walk([&](float4 v4, int i, int) {
      if (!(fmaxf(fmaxf(v4.x, v4.y), fmaxf(v4.z, v4.w)) >= from)) return;
      const float v[4] = {v4.x, v4.y, v4.z, v4.w};
      bool at_border = false;
      int b[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        unsigned int units;
        const unsigned long long m = mass_and_bin(v[j], b[j], units);
        if (b[j] > hi || (cut && !kept(v[j], first + 4 * i + j))) b[j] = MASS_BINS;
        sum += b[j] < lo ? m : 0;
        at_border = at_border || (b[j] >= lo && b[j] < MASS_BINS);
      }
      if (at_border && few_at_border) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (b[j] >= lo && b[j] < MASS_BINS) list(v[j], first + 4 * i + j);
      }
    });
    const unsigned long long mine = block_sum(sum), range = warp_sum(sum);
    gather(mine, [&](int, unsigned long long v) { front += v; });
    if (few_at_border) {
      front_mass = front;
      front_mine = mine;
      front_range = range;
      want_mass = want;
      listed_border = true;
    } else {                                     // (many equal values, or a very flat row)
      cut_at(search([&](float v, int i) { const int b = mass_bin(v); return b >= lo && b <= hi && kept(v, i) ? mass(v) : 0ull; },
                    [&](unsigned long long) { return want - front; }));
    }
  }
  if (listed_border && settle(front_mass, front_mine, front_range, want_mass)) return;
  if (cut || least > 0.0)
    pick(fmaxf(kept_value, least_value), [&](float v, int i) -> unsigned long long { const unsigned long long m = above_least(v); return kept(v, i) ? m : 0ull; }, draw_from, write);
  else
    pick(-INFINITY, [&](float v, int) { return mass(v); }, draw_from, write);
  cluster.sync();
}

}  // namespace qmk_sample
#endif  // QMK_SAMPLING_CUH_
