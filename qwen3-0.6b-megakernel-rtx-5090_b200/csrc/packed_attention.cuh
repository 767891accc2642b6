// Attention of one new token per sequence over a packed cache (packed_cache.cuh): out = softmax(scale * q . k) v, k and v the rows' values.
//
// A CTA takes a query head of a sequence; eight lanes share a row, every eighth of a warp has a running maximum, sum and output of its own, joined at the end.
#ifndef QMK_PACKED_ATTENTION_CUH_
#define QMK_PACKED_ATTENTION_CUH_

#include "packed_cache.cuh"

namespace qmk_packed {

constexpr int MAX_GROUP = 16;                    // query heads per kv head
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

struct AttendParams {
  Caches caches;
  const void *q;
  long long q_seq, q_head;                       // strides, in elements
  int q_heads, group;
  const int *lens;
  float scale_log2;                              // scale * log2 e
  void *out;                                     // [seq][q_head][DIM]
  float *lse;
};

template <typename T, int DIM, int BITS>
__global__ void __launch_bounds__(128) attend_rows(const __grid_constant__ AttendParams p) {
  constexpr int EIGHTS = 16, E = DIM / 8, N = DIM * BITS / 256;
  __shared__ float sm[EIGHTS], sl[EIGHTS], sa[EIGHTS][DIM];
  const int g = threadIdx.x & 7, eighth = threadIdx.x >> 3, b = blockIdx.x / p.q_heads, head = blockIdx.x % p.q_heads;
  const int n = min(max(p.lens[b], 0), p.caches.rows);
  const T *const q = static_cast<const T *>(p.q) + b * p.q_seq + head * p.q_head;
  const long long base = head / p.group * p.caches.head;
  const unsigned char *const kc = p.caches.k[b] + base, *const vc = p.caches.v[b] + base;
  float qv[E], acc[E], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    qv[i] = static_cast<float>(q[DIM / 4 * (i / (E / 4)) + DIM / 32 * g + i % (E / 4)]) * p.scale_log2;
    acc[i] = 0.0f;
  }
  for (int first = 0; first < n; first += EIGHTS) {        // (the same for the CTA)
    const int row = first + eighth;
    const bool there = row < n;
    const long long off = there ? row * p.caches.row : 0;
    uint32_t kw[N], vw[N];
    __half kp[8], vp[8];
    load_codes<DIM, BITS>(kc + off, g, there, kw);
    load_codes<DIM, BITS>(vc + off, g, there, vw);
    *reinterpret_cast<uint4 *>(kp) = __ldg(reinterpret_cast<const uint4 *>(kc + off + DIM * BITS / 8));
    *reinterpret_cast<uint4 *>(vp) = __ldg(reinterpret_cast<const uint4 *>(vc + off + DIM * BITS / 8));
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) s = fmaf(qv[i], value_of<DIM, BITS>(kw, kp, i / (E / 4), i % (E / 4)), s);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (!there) continue;
    const float top = fmaxf(m, s), sub = top == -INFINITY ? 0.0f : top, old = exp2f(m - sub), w = exp2f(s - sub);
    m = top;
    l = fmaf(l, old, w);
#pragma unroll
    for (int i = 0; i < E; ++i) acc[i] = fmaf(w, value_of<DIM, BITS>(vw, vp, i / (E / 4), i % (E / 4)), acc[i] * old);
  }
  if (g == 0) { sm[eighth] = m; sl[eighth] = l; }
#pragma unroll
  for (int i = 0; i < E; ++i) sa[eighth][DIM / 4 * (i / (E / 4)) + DIM / 32 * g + i % (E / 4)] = acc[i];
  __syncthreads();
  if (threadIdx.x >= DIM) return;
  float top = -INFINITY, total = 0.0f, out = 0.0f;
  for (int i = 0; i < EIGHTS; ++i) top = fmaxf(top, sm[i]);
  for (int i = 0; i < EIGHTS; ++i) {
    const float f = sm[i] == -INFINITY ? (sl[i] == 0.0f ? 0.0f : 1.0f) : exp2f(sm[i] - top);   // (a sum that is no number stays one)
    total = fmaf(sl[i], f, total);
    out = fmaf(sa[i][threadIdx.x], f, out);
  }
  static_cast<T *>(p.out)[static_cast<size_t>(blockIdx.x) * DIM + threadIdx.x] = static_cast<T>(total == 0.0f ? 0.0f : out / total);
  if (p.lse && threadIdx.x == 0) p.lse[blockIdx.x] = total == 0.0f ? -INFINITY : top * LN2 + logf(total);
}

}  // namespace qmk_packed
#endif  // QMK_PACKED_ATTENTION_CUH_
