// Attention of one new token per sequence over cache rows that all sequences share (a prefix) and rows of their own.
//
// out = softmax(scale * q . k) v over the prefix rows and the sequence's own ones.  The prefix is the same for all sequences, so
// its scores are matrix products: the queries of all sequences that read a kv head are the rows of one operand, the
// prefix rows cross HBM once for all of them instead of once for each.  A softmax over a split range is joined from partial
// states - the maximum M, the sum L of 2^(s - M) and the unnormalised output A of each part, all fp32 - as sum(2^(M_i - M) A_i) /
// sum(2^(M_i - M) L_i), so the prefix may be split over many CTAs and the own rows handled by others.  A part whose scores are all -inf
// has M = -inf and L = 0 and weighs nothing.
//
// An item is a block of query rows against a range of cache rows of one kv head: (row tile, kv head, prefix range) or (sequence, kv
// head, range of own rows).  Three or two launches: the items' states (up to 32 query rows of a kv head here, more in shared_prefix_tcgen05.cuh with the
// own rows' kernel behind it), then the join.  Each starts early, behind the last CTAs of the one before, and waits where it has to (programmatic dependent
// launch).
//
// Measured, caches cold, 16 query heads on 8 kv heads of 128 dims: attend_parts with 8 sequences and 32,768 shared rows 25.5 us, 5.3 TB/s, bound by
// HBM and the ramp of the CTAs' first tiles; own_parts with 64 sequences of 512 own rows 16.5 us, 4.1 TB/s; join_parts 6 to 10 us, the latency of two
// dependent loads and of the launch.
#ifndef QMK_SHARED_PREFIX_ATTENTION_CUH_
#define QMK_SHARED_PREFIX_ATTENTION_CUH_

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace qmk_spa {

constexpr int MAX_SEQS = 128;
constexpr int MAX_GROUP = 16;                    // query heads per kv head: one m16 tile of a sequence's own rows
constexpr int THREADS = 128, WARPS = 4;
constexpr int KEYS = 64;                         // cache rows per tile
constexpr int STAGES = 3;
constexpr int OWN_RANGE = 256, OWN_PARTS = 16;   // own rows per item, more where a cache has more than OWN_PARTS such ranges
constexpr int OWN_STAGES = 2;
constexpr int own_warps(int dim) { return dim == 64 ? 4 : 2; }               // of own_parts: tiles of 16 KB
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

struct Params {
  const void *q;
  long long q_seq, q_head;                       // strides, in elements
  int seqs, group, q_heads, kv_heads;
  const void *k_prefix, *v_prefix;
  long long prefix_row, prefix_head;
  int prefix_len, prefix_parts, prefix_range, row_tiles;   // range: prefix rows per item, a multiple of KEYS
  int prefix_items;                              // of attend_parts
  long long own_row, own_head;
  int own_rows, own_parts, own_range;            // range: a multiple of 64
  const int *own_lens;
  int own_bias;                                  // added to own_lens
  float scale_log2;                              // scale * log2 e
  float *part_out;                               // [part][seq][q_head][dim]
  float2 *part_ml;                               // [part][seq][q_head]
  void *out;
  float *lse;
  const void *k_own[MAX_SEQS], *v_own[MAX_SEQS];
};

__device__ __forceinline__ void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ uint32_t s32(const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// 16 bytes to shared memory; zeros where there is no row
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
template <typename T> struct Half;
template <> struct Half<__half> {
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
  static __device__ __forceinline__ __half from(float a) { return __float2half_rn(a); }
  // Weights are rounded to the operand type, once, because the tensor cores multiply 16-bit operands by values of 16 bits only; the sum of the weights, the
  // outputs and the joined states stay fp32.  Each weight is off by at most 2^-11 of itself in fp16 (2^-8 in bf16), as much as the output's own rounding, so the
  // error against 64 bits grows by 1.4 at most where many weights count (16,384 equal-sized ones: 2.8e-4 of the outputs' size, with fp32 weights 2.1e-4).
  // They are at most 2^P_SHIFT: rounding 2^-11 of the value down to 2^-14, and so for weights of 2^-26 of the row's largest on.
  static constexpr float P_SHIFT = 12.0f;
  static constexpr bool BF16 = false;
};
template <> struct Half<__nv_bfloat16> {
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
  static __device__ __forceinline__ __nv_bfloat16 from(float a) { return __float2bfloat16_rn(a); }
  static constexpr float P_SHIFT = 0.0f;
  static constexpr bool BF16 = true;
};

// mma.sync tiles: MT warps side by side own 16 query rows each, the 4 / MT groups of warps take the tile's cache rows in turn; every
// warp has a running maximum, sum and output of its own.
template <typename T, int D, int MT>
__device__ __forceinline__ void item_mma(const Params &p, unsigned char *smem, int part, int kv_head, int row0, int live_rows,
                                         const T *kp, const T *vp, long long row_stride, int nrows) {
  constexpr int KG = WARPS / MT, WK = KEYS / KG;           // groups of warps over the cache rows, rows a group takes of a tile
  constexpr int CHUNKS = D / 8, ROW_BYTES = D * 2, TILE = KEYS * ROW_BYTES;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, mt = warp % MT, kg = warp / MT;
  const int quad = lane & 3, rq = lane >> 2;
  const uint32_t base = s32(smem);
  // query fragments straight from global memory: row r of the tile is head r % group of sequence r / group (own rows: one sequence)
  uint32_t qa[D / 16][4];
  {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int r = row0 + mt * 16 + rq + 8 * half;
      const bool live = mt * 16 + rq + 8 * half < live_rows;
      const int b = r / p.group, h = kv_head * p.group + r % p.group;
      const T *src = static_cast<const T *>(p.q) + (live ? b * p.q_seq + h * p.q_head : 0);
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        qa[ks][half] = live ? *reinterpret_cast<const uint32_t *>(src + ks * 16 + quad * 2) : 0u;
        qa[ks][2 + half] = live ? *reinterpret_cast<const uint32_t *>(src + ks * 16 + 8 + quad * 2) : 0u;
      }
    }
  }
  float acc[D / 8][4];
#pragma unroll
  for (int t = 0; t < D / 8; ++t) { acc[t][0] = 0.f; acc[t][1] = 0.f; acc[t][2] = 0.f; acc[t][3] = 0.f; }
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  const int tiles = (nrows + KEYS - 1) / KEYS;
  auto load = [&](int t) {
    if (t < tiles) {
      const uint32_t dst = base + (t % STAGES) * 2 * TILE;
#pragma unroll
      for (int i = tid; i < KEYS * CHUNKS; i += THREADS) {
        const int r = i / CHUNKS, c = i % CHUNKS, row = t * KEYS + r;
        const bool there = row < nrows;
        const long long off = (there ? row : 0) * row_stride + c * 8;
        const uint32_t at = r * ROW_BYTES + ((c ^ (r & 7)) << 4);
        copy16(dst + at, kp + off, there);
        copy16(dst + TILE + at, vp + off, there);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int t = 0; t < STAGES - 1; ++t) load(t);
  for (int t = 0; t < tiles; ++t) {
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    __syncthreads();                                       // tile t is there, tile t - 1 has been read
    load(t + STAGES - 1);
    const uint32_t kt = base + (t % STAGES) * 2 * TILE, vt = kt + TILE;
    float sc[WK / 8][4];
#pragma unroll
    for (int n = 0; n < WK / 8; ++n) { sc[n][0] = 0.f; sc[n][1] = 0.f; sc[n][2] = 0.f; sc[n][3] = 0.f; }
#pragma unroll
    for (int n = 0; n < WK / 16; ++n) {
      const int r = kg * WK + n * 16 + (lane & 7) + (lane >> 4) * 8;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        uint32_t b[4];
        ldsm4(kt + r * ROW_BYTES + (((2 * ks + ((lane >> 3) & 1)) ^ (r & 7)) << 4), b);
        Half<T>::mma(sc[2 * n], qa[ks], b[0], b[1]);
        Half<T>::mma(sc[2 * n + 1], qa[ks], b[2], b[3]);
      }
    }
    const int key0 = t * KEYS + kg * WK;
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < WK / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float v = key0 + n * 8 + quad * 2 + (i & 1) < nrows ? sc[n][i] * p.scale_log2 : -INFINITY;
        sc[n][i] = v;
        mx[i >> 1] = fmaxf(mx[i >> 1], v);
      }
    float sub[2], corr[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
      mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
      const float mn = fmaxf(m[h], mx[h]);
      sub[h] = mn == -INFINITY ? 0.f : mn;                 // nothing seen yet: 2^(-inf - 0) = 0, not NaN
      corr[h] = exp2f(m[h] - sub[h]);
      m[h] = mn;
      sub[h] -= Half<T>::P_SHIFT;
      l[h] *= corr[h];
    }
#pragma unroll
    for (int n = 0; n < WK / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sc[n][i] = exp2f(sc[n][i] - sub[i >> 1]);
        l[i >> 1] += sc[n][i];
      }
#pragma unroll
    for (int t2 = 0; t2 < D / 8; ++t2) { acc[t2][0] *= corr[0]; acc[t2][1] *= corr[0]; acc[t2][2] *= corr[1]; acc[t2][3] *= corr[1]; }
#pragma unroll
    for (int n = 0; n < WK / 16; ++n) {
      const uint32_t pa[4] = {Half<T>::pack(sc[2 * n][0], sc[2 * n][1]), Half<T>::pack(sc[2 * n][2], sc[2 * n][3]),
                              Half<T>::pack(sc[2 * n + 1][0], sc[2 * n + 1][1]), Half<T>::pack(sc[2 * n + 1][2], sc[2 * n + 1][3])};
      const int r = kg * WK + n * 16 + (lane & 15);
#pragma unroll
      for (int dp = 0; dp < D / 16; ++dp) {
        uint32_t b[4];
        ldsm4_trans(vt + r * ROW_BYTES + (((2 * dp + (lane >> 4)) ^ (r & 7)) << 4), b);
        Half<T>::mma(acc[2 * dp], pa, b[0], b[1]);
        Half<T>::mma(acc[2 * dp + 1], pa, b[2], b[3]);
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
  }
  __syncthreads();                                         // the ring is free: the groups' states are joined in it
  constexpr int PITCH = D + 4;                             // floats between rows
  float *const so = reinterpret_cast<float *>(smem);       // [KG][MT * 16][PITCH]
  float2 *const sml = reinterpret_cast<float2 *>(so + KG * MT * 16 * PITCH);
  {
    float *const mine = so + (kg * MT + mt) * 16 * PITCH;
#pragma unroll
    for (int t = 0; t < D / 8; ++t) {
      *reinterpret_cast<float2 *>(mine + rq * PITCH + t * 8 + quad * 2) = make_float2(acc[t][0], acc[t][1]);
      *reinterpret_cast<float2 *>(mine + (rq + 8) * PITCH + t * 8 + quad * 2) = make_float2(acc[t][2], acc[t][3]);
    }
    if (quad == 0) {
      sml[(kg * MT + mt) * 16 + rq] = make_float2(m[0], l[0]);
      sml[(kg * MT + mt) * 16 + rq + 8] = make_float2(m[1], l[1]);
    }
  }
  __syncthreads();
  const size_t rows_all = static_cast<size_t>(p.seqs) * p.q_heads;
  for (int i = tid; i < MT * 16 * (D / 4); i += THREADS) {
    const int r = i / (D / 4), c = i % (D / 4) * 4;
    if (r >= live_rows) continue;
    float M = -INFINITY;
#pragma unroll
    for (int g = 0; g < KG; ++g) M = fmaxf(M, sml[g * MT * 16 + r].x);
    float L = 0.f;
    float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int g = 0; g < KG; ++g) {
      const float2 ml = sml[g * MT * 16 + r];
      const float f = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : exp2f(ml.x - M);
      const float4 a = *reinterpret_cast<const float4 *>(so + (g * MT * 16 + r) * PITCH + c);
      L += ml.y * f;
      A.x += a.x * f; A.y += a.y * f; A.z += a.z * f; A.w += a.w * f;
    }
    const int b = (row0 + r) / p.group, h = kv_head * p.group + (row0 + r) % p.group;
    const size_t at = part * rows_all + static_cast<size_t>(b) * p.q_heads + h;
    *reinterpret_cast<float4 *>(p.part_out + at * D + c) = A;
    if (c == 0) p.part_ml[at] = make_float2(M, L);
  }
}

// A sequence's own rows against its query heads of a kv head (NT blocks of eight).  Turned round: cache rows are the 16 rows of an mma.sync tile
// and heads its eight columns, scores = K q^T and out^T = V^T p^T, so two heads cost half the products and a third of the registers that 16 query rows
// would.  A warp takes 16 of a tile's rows; p^T becomes an operand by transposing 8 x 8 blocks in registers.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <typename T, int D, int NT, int W>
struct OwnRows {
  static constexpr int ROWS = 16 * W;                      // of a tile, 16 for each of W warps
  static constexpr int CHUNKS = D / 8, ROW_BYTES = D * 2, TILE = ROWS * ROW_BYTES, PITCH = D + 4, HEADS = NT * 8;
  static constexpr int STATE_BYTES = W * HEADS * (PITCH * 4 + 8);            // of the warps' states, where they are joined
  uint32_t qb[NT][D / 16][2];
  float acc[NT][D / 16][4], m[NT][2], l[NT][2];            // heads 2 quad and 2 quad + 1 of each block

  static __device__ __forceinline__ void load(const Params &p, uint32_t dst, const T *kp, const T *vp, int t, int nrows) {
#pragma unroll
    for (int i = threadIdx.x; i < ROWS * CHUNKS; i += 32 * W) {
      const int r = i / CHUNKS, c = i % CHUNKS, row = t * ROWS + r;
      const bool there = row < nrows;
      const long long off = (there ? row : 0) * p.own_row + c * 8;
      const uint32_t at = r * ROW_BYTES + ((c ^ (r & 7)) << 4);
      copy16(dst + at, kp + off, there);
      copy16(dst + TILE + at, vp + off, there);
    }
  }
  __device__ __forceinline__ void begin(const Params &p, int kv_head, int b) {
    const int lane = threadIdx.x & 31, quad = lane & 3, rq = lane >> 2;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const bool live = nt * 8 + rq < p.group;
      const T *src = static_cast<const T *>(p.q) + b * p.q_seq + (kv_head * p.group + (live ? nt * 8 + rq : 0)) * p.q_head + quad * 2;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        qb[nt][ks][0] = live ? *reinterpret_cast<const uint32_t *>(src + ks * 16) : 0u;
        qb[nt][ks][1] = live ? *reinterpret_cast<const uint32_t *>(src + ks * 16 + 8) : 0u;
      }
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int t = 0; t < D / 16; ++t) { acc[nt][t][0] = 0.f; acc[nt][t][1] = 0.f; acc[nt][t][2] = 0.f; acc[nt][t][3] = 0.f; }
    }
  }
  // this warp's 16 rows of tile t
  __device__ __forceinline__ void tile(const Params &p, uint32_t kt, int t, int nrows) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rq = lane >> 2, key0 = t * ROWS + warp * 16;
    const uint32_t vt = kt + TILE;
    if (key0 >= nrows) return;                             // (the same for the warp)
    float sc[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) { sc[nt][0] = 0.f; sc[nt][1] = 0.f; sc[nt][2] = 0.f; sc[nt][3] = 0.f; }
    const int kr = warp * 16 + (lane & 15);
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      uint32_t a[4];
      ldsm4(kt + kr * ROW_BYTES + (((2 * ks + (lane >> 4)) ^ (kr & 7)) << 4), a);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) Half<T>::mma(sc[nt], a, qb[nt][ks][0], qb[nt][ks][1]);
    }
    uint32_t pb[NT][2];
    const bool top_row = key0 + rq < nrows, low_row = key0 + rq + 8 < nrows;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 4; ++i) sc[nt][i] = (i < 2 ? top_row : low_row) ? sc[nt][i] * p.scale_log2 : -INFINITY;
      float corr[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float mx = fmaxf(sc[nt][h], sc[nt][2 + h]);
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float mn = fmaxf(m[nt][h], mx);
        float sub = mn == -INFINITY ? 0.f : mn;            // scores of -inf only: 2^(-inf - 0) = 0, not NaN
        corr[h] = exp2f(m[nt][h] - sub);
        m[nt][h] = mn;
        sub -= Half<T>::P_SHIFT;
        sc[nt][h] = exp2f(sc[nt][h] - sub);
        sc[nt][2 + h] = exp2f(sc[nt][2 + h] - sub);
        l[nt][h] = l[nt][h] * corr[h] + (sc[nt][h] + sc[nt][2 + h]);
      }
      pb[nt][0] = transposed(Half<T>::pack(sc[nt][0], sc[nt][1]));
      pb[nt][1] = transposed(Half<T>::pack(sc[nt][2], sc[nt][3]));
#pragma unroll
      for (int t2 = 0; t2 < D / 16; ++t2) { acc[nt][t2][0] *= corr[0]; acc[nt][t2][1] *= corr[1]; acc[nt][t2][2] *= corr[0]; acc[nt][t2][3] *= corr[1]; }
    }
    const int vr = warp * 16 + (lane & 7) + 8 * (lane >> 4);
#pragma unroll
    for (int dp = 0; dp < D / 16; ++dp) {
      uint32_t a[4];
      ldsm4_trans(vt + vr * ROW_BYTES + (((2 * dp + ((lane >> 3) & 1)) ^ (vr & 7)) << 4), a);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) Half<T>::mma(acc[nt][dp], a, pb[nt][0], pb[nt][1]);
    }
  }
  // The warps' states, joined in `smem` (STATE_BYTES, free when this is called), to the workspace.
  __device__ __forceinline__ void end(const Params &p, unsigned char *smem, int part, int kv_head, int b) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, quad = lane & 3, rq = lane >> 2;
    float *const so = reinterpret_cast<float *>(smem);     // [warp][head][PITCH]
    float2 *const sml = reinterpret_cast<float2 *>(so + W * HEADS * PITCH);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[nt][h] += __shfl_xor_sync(0xffffffffu, l[nt][h], o);
        float *const mine = so + (warp * HEADS + nt * 8 + quad * 2 + h) * PITCH + rq;
#pragma unroll
        for (int t = 0; t < D / 16; ++t) { mine[t * 16] = acc[nt][t][h]; mine[t * 16 + 8] = acc[nt][t][2 + h]; }
        if (rq == 0) sml[warp * HEADS + nt * 8 + quad * 2 + h] = make_float2(m[nt][h], l[nt][h]);
      }
    }
    __syncthreads();
    const size_t at0 = (static_cast<size_t>(part) * p.seqs + b) * p.q_heads + kv_head * p.group;
    for (int i = tid; i < p.group * (D / 4); i += 32 * W) {
      const int h = i / (D / 4), c = i % (D / 4) * 4;
      float M = -INFINITY, L = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) M = fmaxf(M, sml[w * HEADS + h].x);
      float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float2 ml = sml[w * HEADS + h];
        const float f = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : exp2f(ml.x - M);
        const float4 a = *reinterpret_cast<const float4 *>(so + (w * HEADS + h) * PITCH + c);
        L += ml.y * f;
        A.x += a.x * f; A.y += a.y * f; A.z += a.z * f; A.w += a.w * f;
      }
      *reinterpret_cast<float4 *>(p.part_out + (at0 + h) * D + c) = A;
      if (c == 0) p.part_ml[at0 + h] = make_float2(M, L);
    }
  }
};
// An own item: (kv head, sequence, range)
struct OwnItem { int kv, b, own; };
__device__ __forceinline__ OwnItem own_item(const Params &p, int id) { return OwnItem{id % p.kv_heads, id / p.kv_heads % p.seqs, id / (p.kv_heads * p.seqs)}; }
__device__ __forceinline__ int own_len(const Params &p, int b) { return static_cast<int>(min(max(static_cast<long long>(p.own_lens[b]) + p.own_bias, 0ll), static_cast<long long>(p.own_rows))); }
template <typename T>
__device__ __forceinline__ const T *own_base(const Params &p, const void *const *caches, const OwnItem &it) {
  return static_cast<const T *>(caches[it.b]) + static_cast<size_t>(it.kv) * p.own_head + static_cast<size_t>(it.own) * p.own_range * p.own_row;
}
template <typename T, int D, int NT, int W>
__device__ __forceinline__ void own_cta(const Params &p, unsigned char *smem, int id) {
  using Own = OwnRows<T, D, NT, W>;
  const OwnItem it = own_item(p, id);
  const int n = min(p.own_range, own_len(p, it.b) - it.own * p.own_range), tiles = (n + Own::ROWS - 1) / Own::ROWS;
  if (n <= 0) return;                                      // (join_parts goes by the length too)
  const T *const kp = own_base<T>(p, p.k_own, it), *const vp = own_base<T>(p, p.v_own, it);
  auto load = [&](int t) {
    if (t < tiles) Own::load(p, s32(smem) + (t % OWN_STAGES) * 2 * Own::TILE, kp, vp, t, n);
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int t = 0; t < OWN_STAGES; ++t) load(t);
  Own own;
  own.begin(p, it.kv, it.b);
  for (int t = 0; t < tiles; ++t) {
    asm volatile("cp.async.wait_group %0;" ::"n"(OWN_STAGES - 1) : "memory");
    __syncthreads();
    own.tile(p, s32(smem) + (t % OWN_STAGES) * 2 * Own::TILE, t, n);
    __syncthreads();                                       // the tile has been read
    load(t + OWN_STAGES);
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  own.end(p, smem, p.prefix_parts + it.own, it.kv, it.b);
}

// Few query rows: prefix items first, they are the longest, then the own ones.
template <typename T, int D, int MT, int NT>
__global__ void __launch_bounds__(THREADS) attend_parts(const __grid_constant__ Params p) {
  extern __shared__ __align__(128) unsigned char smem[];
  pdl_wait();
  pdl_trigger();
  const int id = static_cast<int>(blockIdx.x);
  if (id >= p.prefix_items) { own_cta<T, D, NT, WARPS>(p, smem, id - p.prefix_items); return; }
  const int kv = id % p.kv_heads, tile = id / p.kv_heads % p.row_tiles, part = id / (p.kv_heads * p.row_tiles);
  const int first = part * p.prefix_range, n = min(p.prefix_range, p.prefix_len - first);
  const int row0 = tile * MT * 16, live = min(MT * 16, p.seqs * p.group - row0);
  const size_t off = static_cast<size_t>(kv) * p.prefix_head + static_cast<size_t>(first) * p.prefix_row;
  item_mma<T, D, MT>(p, smem, part, kv, row0, live, static_cast<const T *>(p.k_prefix) + off, static_cast<const T *>(p.v_prefix) + off, p.prefix_row, n);
}
// Many: the own rows alone, launched behind prefix_parts_tc, which has waited for what is read here: they start on the SMs that it does not use or has
// left - no CTA of this kernel fits beside one of it, which has 168 x 384 registers and with 128 dims 229,632 bytes of shared memory - and end behind
// it.  Small CTAs, six an SM: what one waits for (its length, the queries, the first rows, its warps at the end) passes under the others.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(32 * own_warps(D), D == 64 ? 4 : 6) own_parts(const __grid_constant__ Params p) {
  extern __shared__ __align__(128) unsigned char smem[];
  pdl_trigger();
  own_cta<T, D, NT, own_warps(D)>(p, smem, static_cast<int>(blockIdx.x));
  pdl_wait();
}

// A CTA joins the parts of a (sequence, query head): a warp takes every fourth part.
template <typename T, int D>
__global__ void __launch_bounds__(128) join_parts(const __grid_constant__ Params p) {
  constexpr int E = D / 32, AHEAD = 8;
  __shared__ float sm[4], sl[4];
  __shared__ __align__(16) float sa[4][D];
  // Own ranges behind a sequence's length have no state.  (The lengths were there before the kernels were launched that this one follows; read while
  // they run.)
  const int parts = p.prefix_parts + (p.own_parts ? (own_len(p, static_cast<int>(blockIdx.x) / p.q_heads) + p.own_range - 1) / p.own_range : 0);
  pdl_wait();
  pdl_trigger();
  const int rows = p.seqs * p.q_heads, row = static_cast<int>(blockIdx.x), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float M = -INFINITY, L = 0.f, A[E];
#pragma unroll
  for (int i = 0; i < E; ++i) A[i] = 0.f;
  auto take = [&](int i0) {                                // up to eight parts, their outputs asked for with their maxima
    float v[AHEAD][E];
    float2 ml[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      ml[j] = make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int k = 0; k < E; ++k) v[j][k] = 0.f;
      if (i0 + 4 * j < parts) {
        const size_t at = static_cast<size_t>(i0 + 4 * j) * rows + row;
        ml[j] = p.part_ml[at];
        const float *src = p.part_out + at * D + lane * E;
        if (E == 4) { const float4 a = *reinterpret_cast<const float4 *>(src); v[j][0] = a.x; v[j][1] = a.y; v[j][E - 2] = a.z; v[j][E - 1] = a.w; }
        else { const float2 a = *reinterpret_cast<const float2 *>(src); v[j][0] = a.x; v[j][1] = a.y; }
      }
    }
    float top = M;
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) top = fmaxf(top, ml[j].x);
    const float f0 = M == -INFINITY ? 0.f : exp2f(M - top);
    M = top;
    L *= f0;
#pragma unroll
    for (int k = 0; k < E; ++k) A[k] *= f0;
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      // (scores of -inf alone: nothing; a maximum of -inf with a sum that is no number: the result is none)
      const float f = ml[j].x == -INFINITY ? (ml[j].y == 0.f ? 0.f : 1.f) : exp2f(ml[j].x - top);
      L = fmaf(ml[j].y, f, L);
#pragma unroll
      for (int k = 0; k < E; ++k) A[k] = fmaf(v[j][k], f, A[k]);
    }
  };
  for (int i0 = warp; i0 < parts; i0 += 4 * AHEAD) take(i0);
  if (lane == 0) { sm[warp] = M; sl[warp] = L; }
#pragma unroll
  for (int k = 0; k < E; ++k) sa[warp][lane * E + k] = A[k];
  __syncthreads();
  const int d = threadIdx.x;
  if (d >= D) return;
  const float top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  float total = 0.f, out = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float f = sm[w] == -INFINITY ? (sl[w] == 0.f ? 0.f : 1.f) : exp2f(sm[w] - top);
    total = fmaf(sl[w], f, total);
    out = fmaf(sa[w][d], f, out);
  }
  static_cast<T *>(p.out)[static_cast<size_t>(row) * D + d] = Half<T>::from(total == 0.f ? 0.f : out / total);
  if (p.lse && d == 0) p.lse[row] = total == 0.f ? -INFINITY : (top - Half<T>::P_SHIFT) * LN2 + logf(total);
}

}  // namespace qmk_spa
#endif  // QMK_SHARED_PREFIX_ATTENTION_CUH_
