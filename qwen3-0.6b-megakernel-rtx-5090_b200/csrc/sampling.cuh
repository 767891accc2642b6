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
// A cluster of CTAs takes a row and keeps it in shared memory as fp32: the row crosses HBM once, however often it is looked at.
#ifndef QMK_SAMPLING_CUH_
#define QMK_SAMPLING_CUH_

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace qmk_sample {

namespace cg = cooperative_groups;

constexpr int THREADS = 512, WARPS = THREADS / 32;
constexpr int MAX_VOCAB = 1 << 18;               // masses of at most 2^45 in 63 bits
constexpr int MAX_CLUSTER = 8;
constexpr int BINS = 256;                        // of a histogram: eight bits of the key
constexpr int NO_TOKEN = 0x7fffffff;             // pick of a row without a largest value, as in the greedy steps
constexpr float LARGEST_UNIFORM = 0x1.fffffep-1f;

struct Params {
  const void *logits;
  long long row_stride;                          // elements
  int vocab, slice;                              // slice: tokens a CTA of the cluster keeps
  const float *uniforms;
  const float *temperatures, *top_ps, *min_ps;   // per row, or null: the scalar for all
  const int *top_ks;
  float temperature, top_p, min_p;
  int top_k;
  int *tokens;
  float *logprobs;                               // may be null
};

struct Shared {
  unsigned long long mass[2][BINS];              // histograms, in turn: one is read by the cluster while the next is filled
  unsigned long long sum[BINS];                  // the cluster's
  unsigned long long warp[WARPS];
  unsigned long long cta[8];                     // one slot per exchange of the cluster, see Row
  unsigned long long found[3];
  int cut;
};

// Order of the values as whole numbers: larger value, larger key.  (x is not NaN, zeros are +0.)
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x);
  return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float clean(float x) { return x == x ? x + 0.0f : -INFINITY; }
__device__ __forceinline__ float load_logit(const float *p) { return clean(*p); }
__device__ __forceinline__ float load_logit(const __half *p) { return clean(__half2float(*p)); }
__device__ __forceinline__ float load_logit(const __nv_bfloat16 *p) { return clean(__bfloat162float(*p)); }

template <typename V>
__device__ __forceinline__ V warp_sum(V v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// What is kept: values above a threshold, and of those equal to it the ones up to an index.
struct Kept {
  uint32_t key;
  int cut;
  __device__ __forceinline__ bool operator()(uint32_t k, int i) const { return k > key || (k == key && i <= cut); }
};

template <typename T>
__global__ void __launch_bounds__(THREADS) sample_rows(const Params p) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  Shared &s = *reinterpret_cast<Shared *>(smem_raw);
  float *const x = reinterpret_cast<float *>(smem_raw + sizeof(Shared));
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int row = static_cast<int>(blockIdx.x) / ranks, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int first = rank * p.slice, n = max(0, min(p.slice, p.vocab - first));     // this CTA's tokens [first, first + n)
  const float temperature = p.temperatures ? p.temperatures[row] : p.temperature;
  const float top_p = p.top_ps ? p.top_ps[row] : p.top_p, min_p = p.min_ps ? p.min_ps[row] : p.min_p;
  const int top_k = p.top_ks ? p.top_ks[row] : p.top_k;
  const float u_raw = p.uniforms[row];
  const float u = u_raw >= 0.0f ? fminf(u_raw, LARGEST_UNIFORM) : 0.0f;
  int exchange = 0;                              // slots of Shared::cta are used in turn

  // one value of every CTA to every CTA, in the order of the ranks
  auto gather = [&](unsigned long long mine, auto &&take) {
    const int slot = exchange++ & 7;
    if (tid == 0) s.cta[slot] = mine;
    cluster.sync();
    for (int r = 0; r < ranks; ++r) take(r, *cluster.map_shared_rank(&s.cta[slot], r));
  };
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

  // ---- the row, once; its largest value and where that is first
  unsigned long long best = 0;                   // key, then the index from above
  {
    const T *const src = static_cast<const T *>(p.logits) + row * p.row_stride + first;
    for (int i = tid; i < n; i += THREADS) {
      const float v = load_logit(src + i);
      x[i] = v;
      const unsigned long long c = (static_cast<unsigned long long>(key_of(v)) << 32) | static_cast<uint32_t>(~(first + i));
      best = c > best ? c : best;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
      best = other > best ? other : best;
    }
    if (lane == 0) s.warp[warp] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w) best = s.warp[w] > best ? s.warp[w] : best;
    const unsigned long long mine = best;
    gather(mine, [&](int, unsigned long long v) { best = v > best ? v : best; });
  }
  const uint32_t top_key = static_cast<uint32_t>(best >> 32);
  const int top_index = static_cast<int>(~static_cast<uint32_t>(best));
  const float top = __uint_as_float(top_key & 0x80000000u ? top_key ^ 0x80000000u : ~top_key);
  const bool empty = top == -INFINITY, greedy = !(temperature > 0.0f) || top_k == 1;
  if (empty || greedy) {
    if (rank == 0 && tid == 0) {
      p.tokens[row] = empty ? NO_TOKEN : top_index;
      if (p.logprobs) p.logprobs[row] = empty ? NAN : 0.0f;
    }
    cluster.sync();                              // (nobody leaves while its shared memory is read)
    return;
  }

  // (a row with infinite logits: they share the mass alone)
  auto exponent = [&](float v) { return v == top ? 0.0 : top == INFINITY ? -INFINITY : (static_cast<double>(v) - static_cast<double>(top)) / static_cast<double>(temperature); };
  auto weight = [&](float v) { return v == -INFINITY ? 0.0 : exp(exponent(v)); };
  auto mass_of = [&](float v) { return static_cast<unsigned long long>(__double2ull_rn(weight(v) * 0x1p45)); };

  // The lowest index of the row at which the running sum of `value` exceeds `target(total)`; the CTA that holds it calls found(index, value, total).
  auto pick = [&](auto &&value, auto &&target, auto &&found) {
    const int seg = (n + WARPS - 1) / WARPS, lo = min(n, warp * seg), hi = min(n, lo + seg);   // a warp, a range of the indices
    unsigned long long sum = 0;
    for (int i = lo + lane; i < hi; i += 32) sum += value(i);
    const unsigned long long mine = block_sum(sum);
    unsigned long long before = 0, total = 0;
    gather(mine, [&](int r, unsigned long long v) { before += r < rank ? v : 0; total += v; });
    const unsigned long long want = target(total);
    if (before <= want && want < before + mine) {          // (the same for every thread of the CTA)
      unsigned long long at = before;
      int w = 0;
      for (; w < WARPS - 1 && at + s.warp[w] <= want; ++w) at += s.warp[w];
      if (warp == w) {
        bool done = false;
        for (int i0 = lo; i0 < hi && !done; i0 += 32) {
          const int i = i0 + lane;
          const unsigned long long v = i < hi ? value(i) : 0;
          unsigned long long run = v;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long up = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += up;
          }
          const unsigned int over = __ballot_sync(0xffffffffu, at + run > want);
          if (over) {
            if (lane == __ffs(over) - 1) found(i, total);
            done = true;
          }
          at += __shfl_sync(0xffffffffu, run, 31);
        }
      }
    }
  };

  // The threshold behind which the running sum of `value`, in the order of the values, reaches target(total): eight bits of the
  // key at a time, then the ties.  `value(i)` is 0 for tokens that are out already.
  int turn = 0;
  auto search = [&](auto &&value, auto &&target) -> Kept {
    uint32_t prefix = 0;
    unsigned long long want = 0, before = 0;
    bool everything = false;
    for (int shift = 24; shift >= 0 && !everything; shift -= 8) {
      unsigned long long *const hist = s.mass[turn & 1];
      for (int b = tid; b < BINS; b += THREADS) hist[b] = 0;
      __syncthreads();
      for (int i = tid; i < n; i += THREADS) {
        const uint32_t k = key_of(x[i]);
        if (shift < 24 && (k >> (shift + 8)) != prefix) continue;
        const unsigned long long v = value(i);
        if (v) atomicAdd(&hist[(k >> shift) & (BINS - 1)], v);
      }
      cluster.sync();
      for (int b = tid; b < BINS; b += THREADS) {
        unsigned long long v = 0;
        for (int r = 0; r < ranks; ++r) v += cluster.map_shared_rank(hist, r)[b];
        s.sum[b] = v;
      }
      __syncthreads();
      if (tid == 0) {
        unsigned long long total = 0, at = before;
        for (int b = 0; b < BINS; ++b) total += s.sum[b];
        if (shift == 24) want = target(total);
        int b = BINS - 1;
        while (b > 0 && at + s.sum[b] < want) at += s.sum[b--];
        s.found[0] = at + s.sum[b] < want ? ~0ull : b;     // fewer in all: everything stays
        s.found[1] = at;
        s.found[2] = want;
      }
      __syncthreads();
      everything = s.found[0] == ~0ull;
      prefix = (prefix << 8) | static_cast<uint32_t>(s.found[0]);
      before = s.found[1];
      want = s.found[2];
      ++turn;
    }
    if (everything) return Kept{0u, 0x7fffffff};
    // tokens of the threshold's value, as many as the sum before them leaves room for
    if (tid == 0) s.cut = 0x7fffffff;
    const uint32_t key = prefix;
    unsigned long long each = 0;
    for (int i = tid; i < n; i += THREADS)
      if (key_of(x[i]) == key) { const unsigned long long v = value(i); each = v > each ? v : each; }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { const unsigned long long other = __shfl_xor_sync(0xffffffffu, each, o); each = other > each ? other : each; }
    __syncthreads();
    if (lane == 0) s.warp[warp] = each;
    __syncthreads();
    for (int w = 0; w < WARPS; ++w) each = s.warp[w] > each ? s.warp[w] : each;
    gather(each, [&](int, unsigned long long v) { each = v > each ? v : each; });
    const unsigned long long room = each ? (want - before + each - 1) / each : 1;
    pick([&](int i) -> unsigned long long { return key_of(x[i]) == key && value(i) != 0; }, [&](unsigned long long) { return room - 1; },
         [&](int i, unsigned long long) { for (int r = 0; r < ranks; ++r) *cluster.map_shared_rank(&s.cut, r) = first + i; });
    cluster.sync();
    return Kept{key, s.cut};
  };

  Kept kept{0u, 0x7fffffff};
  if (top_k > 0 && top_k < p.vocab)
    kept = search([&](int) { return 1ull; }, [&](unsigned long long) { return static_cast<unsigned long long>(top_k); });
  if (top_p < 1.0f) {
    const Kept by_k = kept;
    const double share = top_p > 0.0f ? static_cast<double>(top_p) : 0.0;
    kept = search([&](int i) { return by_k(key_of(x[i]), first + i) ? mass_of(x[i]) : 0ull; },
                  [&](unsigned long long total) { const unsigned long long t = __double2ull_ru(share * __ull2double_rn(total)); return t < 1 ? 1ull : t < total ? t : total; });
  }
  const double least = min_p > 0.0f ? static_cast<double>(min_p) : 0.0;
  pick([&](int i) -> unsigned long long {
         const float v = x[i];
         return kept(key_of(v), first + i) && (weight(v) >= least || v == top) ? mass_of(v) : 0ull;
       },
       [&](unsigned long long total) { return __double2ull_rd(static_cast<double>(u) * __ull2double_rn(total)); },
       [&](int i, unsigned long long total) {
         p.tokens[row] = first + i;
         if (p.logprobs) p.logprobs[row] = static_cast<float>(exponent(x[i]) - log(__ull2double_rn(total) * 0x1p-45));
       });
  cluster.sync();
}

}  // namespace qmk_sample
#endif  // QMK_SAMPLING_CUH_
