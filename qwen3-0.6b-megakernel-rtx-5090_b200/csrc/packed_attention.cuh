// Attention of one new token per sequence over a packed cache (packed_cache.cuh): out = softmax(scale * q . k) v, k and v the rows' values.
//
// With c(d) = n - M the codes around their middle, b(d) the quarter of dimension d, s and z a row's scales and centres:
//   q . k = sum_b s_b (sum_{d in b} q_d n_d - M Q_b) + sum_b z_b Q_b,   Q_b = sum_{d in b} q_d,
//   out_d = sum_r p_r z_{r,b(d)} + sum_r (p_r s_{r,b(d)}) c_{r,d},
// so codes enter the products as they are: n as the fp16 number n 2^-24 is its own bit pattern, and masking four bits of each half of a word makes two
// operands at once.  Rows of the cache are the 16 rows of an mma.sync tile and query heads its eight columns (NT blocks of them).  Scores: codes times queries, one
// sum for each quarter, which starts at -M Q_b; out^T: codes times weights times scales.  Weights are carried as two fp16 numbers and the product with a
// scale is rounded once, to fp16: as much as the rounding of an fp16 output; sums, softmax statistics and outputs are fp32.
//
// Work: tiles of 32 rows of a (sequence, kv head), all in one line; each warp takes an equal stretch of it, whatever the sequences' lengths, with a ring of copies
// of its own.  A stretch that holds a whole item writes its output; parts of an item leave their states - the maximum, the sum and the unnormalised output -
// in the workspace, and a second launch joins them.
#ifndef QMK_PACKED_ATTENTION_CUH_
#define QMK_PACKED_ATTENTION_CUH_

#include "packed_cache.cuh"

namespace qmk_packed {

constexpr int MAX_GROUP = 16;                    // query heads per kv head
constexpr int TILE = 32;                         // rows
constexpr int WARPS = 4, SMS = 148;
// CTAs on an SM: what registers allow (168 a thread, 255 with two blocks of heads); tiles of a warp's ring: what their shared memory does
constexpr int ctas_per_sm(int blocks) { return blocks == 1 ? 3 : 2; }
constexpr int stages(int blocks, int row_bytes) {
  const int fit = 225 * 1024 / (ctas_per_sm(blocks) * WARPS * 2 * TILE * row_bytes);
  return fit < 4 ? fit : 4;
}
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
// Weights are 2^SHIFT at the row's maximum, up to 2^(SHIFT + SLACK) where that has risen since it was last looked at: fp16 has 11 bits of them down to 2^-21 of
// the largest.
constexpr float SHIFT = 7.0f, SLACK = 8.0f;

struct AttendParams {
  Caches caches;
  const void *q;
  long long q_seq, q_head;                       // strides, in elements
  int q_heads, group;
  const int *lens;
  float scale_log2;                              // scale * log2 e
  int warps;                                     // of the launch
  float *part_out;                               // [2 warps][group][DIM]
  float2 *part_ml;                               // [2 warps][group]
  void *out;                                     // [seq][q_head][DIM]
  float *lse;
};

__device__ __forceinline__ void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool there) {         // zeros where there is no row
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, float c0, float c1, float c2, float c3) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ void mma_k8(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5}, {%6}, {%7, %7, %7, %7};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(b0), "f"(0.0f));
}
__device__ __forceinline__ uint32_t pack2(float a, float b) { return bits_of(__floats2half2_rn(a, b)); }
__device__ __forceinline__ __half2 h2(uint32_t x) { return from_bits<__half2>(x); }
__device__ __forceinline__ float power2(int e) { return __int_as_float((e + 127) << 23); }    // e in [-126, 127]
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Words of shared memory
template <int N> __device__ __forceinline__ void lds(uint32_t at, uint32_t (&w)[N]) {
  if constexpr (N == 4) asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
  else if constexpr (N == 2) asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at) : "memory");
  else asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0]) : "r"(at) : "memory");
}
__device__ __forceinline__ uint32_t lds16(uint32_t at) {
  unsigned short h;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(at) : "memory");
  return h;
}

// Codes of quarter b of two chunks (DIM/8 codes each), the first in the lower halves: x[j] = (a_j, b_j) as fp16 numbers of 2^-24, of 4-bit codes every second of
// 2^-20.
template <int DIM, int BITS>
__device__ __forceinline__ void expand(const uint32_t (&a)[DIM * BITS / 256], const uint32_t (&c)[DIM * BITS / 256], int b, uint32_t (&x)[DIM / 32]) {
  if constexpr (BITS == 4 && DIM == 64) {
    const uint32_t w = __byte_perm(a[0], c[0], b | b << 4 | (4 + b) << 8 | (4 + b) << 12);
    x[0] = w & 0x000f000fu;
    x[1] = w & 0x00f000f0u;
  } else if constexpr (BITS == 4) {
    const uint32_t w = __byte_perm(a[b / 2], c[b / 2], b % 2 ? 0x7632 : 0x5410), u = w >> 8;
    x[0] = w & 0x000f000fu;
    x[1] = w & 0x00f000f0u;
    x[2] = u & 0x000f000fu;
    x[3] = u & 0x00f000f0u;
  } else if constexpr (DIM == 64) {
    const uint32_t w = __byte_perm(a[b / 2], c[b / 2], b % 2 ? 0x7632 : 0x5410);
    x[0] = w & 0x00ff00ffu;
    x[1] = w >> 8 & 0x00ff00ffu;
  } else {
    const uint32_t w = __byte_perm(a[b], c[b], 0x5410), u = __byte_perm(a[b], c[b], 0x7632);
    x[0] = w & 0x00ff00ffu;
    x[1] = w >> 8 & 0x00ff00ffu;
    x[2] = u & 0x00ff00ffu;
    x[3] = u >> 8 & 0x00ff00ffu;
  }
}

// The line of tiles: sequence by sequence, kv head by kv head.
struct Line {
  int total;                                     // tiles
  int before[MAX_SEQS];                          // tiles in front of a sequence
};
__device__ __forceinline__ int seen_rows(const AttendParams &p, int b) { return min(max(p.lens[b], 0), p.caches.rows); }
__device__ __forceinline__ int tiles_of(int rows) { return (rows + TILE - 1) / TILE; }
// (a sequence to each of the first threads; in front of a barrier of the caller's)
__device__ __forceinline__ void make_line(const AttendParams &p, Line &line, int (&sums)[MAX_SEQS / 32]) {
  const int i = threadIdx.x, lane = i & 31;
  int n = i < p.caches.seqs ? tiles_of(seen_rows(p, i)) * p.caches.kv_heads : 0;
  const int own = n;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, n, o);
    if (lane >= o) n += up;
  }
  if (lane == 31 && i < MAX_SEQS) sums[i >> 5] = n;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < MAX_SEQS / 32; ++w)
    if (w < (i >> 5)) n += sums[w];
  if (i < MAX_SEQS) line.before[i] = n - own;
  if (i == MAX_SEQS - 1) line.total = n;
}
// Stretch r of `parts` equal ones begins at tile total * r / parts; the stretch that holds tile t
__device__ __forceinline__ int begin_of(int total, int parts, int r) { return static_cast<int>(static_cast<long long>(total) * r / parts); }
__device__ __forceinline__ int part_of(int total, int parts, int t) { return static_cast<int>(((t + 1ll) * parts - 1) / total); }

// A place in the line
struct Place {
  int b, head, tile, tiles, rows;
  __device__ __forceinline__ void sequence(const AttendParams &p, int at) {
    b = at;
    rows = b < p.caches.seqs ? seen_rows(p, b) : 0;
    tiles = tiles_of(rows);
  }
  __device__ __forceinline__ void start(const AttendParams &p, const Line &line, int t) {
    int low = 0, high = p.caches.seqs - 1;       // the last sequence that begins at t or before, and has tiles
    while (low < high) {
      const int mid = (low + high + 1) / 2;
      if (line.before[mid] <= t) low = mid; else high = mid - 1;
    }
    sequence(p, low);
    const int i = t - line.before[low];
    head = i / tiles;
    tile = i - head * tiles;
  }
  __device__ __forceinline__ void next(const AttendParams &p) {
    if (++tile < tiles) return;
    tile = 0;
    if (++head < p.caches.kv_heads) return;
    head = 0;
    do sequence(p, b + 1); while (tiles == 0 && b < p.caches.seqs);
  }
};

template <typename T, int DIM, int BITS, int NT>
struct Attend {
  static constexpr int ROW = ROW_BYTES<DIM, BITS>, CODES = ROW - TRAILER, PIECES = ROW / 16;
  static constexpr int CHUNK = CODES / 8, N = CHUNK / 4, J = DIM / 32, STEPS = J / 2;       // bytes and words of a chunk; codes of a quarter in it; k steps of a quarter
  static constexpr int STAGE = 2 * TILE * ROW;                                              // keys, then values
  static constexpr int STAGES = stages(NT, ROW), SMEM = WARPS * STAGES * STAGE;
  static constexpr float M = 1 << (BITS - 1), UNIT = 0x1p-24f;
  static constexpr bool SPREAD = BITS == 8 && DIM == 128;                                   // a lane's two chunks of keys: four apart, or one behind the other

  uint32_t qb[NT][4][STEPS][2], qz[NT];          // queries; sums over quarters, as upper and lower fp16 parts
  float start[NT][4][2], factor[NT][2];          // -M Q_b, and scale * log2 e over the queries' power of two, of heads 2 t and 2 t + 1
  float acc[NT][4][STEPS][4], zacc[NT][4], m[NT][2], l[NT][2];
  __half2 f01, f23;                              // powers of two that take the quarters' scales of values to 1 or below

  static __device__ __forceinline__ void load(const AttendParams &p, const Place &at, uint32_t dst, int lane) {
    const long long base = static_cast<long long>(at.head) * p.caches.head + static_cast<long long>(at.tile) * TILE * p.caches.row;
    const unsigned char *const k = p.caches.k[at.b] + base, *const v = p.caches.v[at.b] + base;
    const int pieces = min(at.rows - at.tile * TILE, TILE) * PIECES;
    if (p.caches.row == ROW) {                   // rows right behind one another
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const int piece = lane + 32 * i;
        const bool there = piece < pieces;
        const int off = there ? piece * 16 : 0;
        copy16(dst + piece * 16, k + off, there);
        copy16(dst + TILE * ROW + piece * 16, v + off, there);
      }
    } else {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const int piece = lane + 32 * i;
        const bool there = piece < pieces;
        const long long off = there ? piece / PIECES * p.caches.row + piece % PIECES * 16 : 0;
        copy16(dst + piece * 16, k + off, there);
        copy16(dst + TILE * ROW + piece * 16, v + off, there);
      }
    }
  }

  // The queries of an item, and nothing seen yet
  __device__ __forceinline__ void begin(const AttendParams &p, int b, int kv_head, int lane) {
    const int t = lane & 3, g = lane >> 2;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const bool live = nt * 8 + g < p.group;
      const T *const q = static_cast<const T *>(p.q) + b * p.q_seq + (kv_head * p.group + (live ? nt * 8 + g : 0)) * p.q_head;
      float x[4][2 * J], top = 0.0f;             // of the lane's two chunks
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int j = 0; j < J; ++j) {
            const int chunk = SPREAD ? t + 4 * c : 2 * t + c;
            x[i][c * J + j] = live ? static_cast<float>(q[DIM / 4 * i + DIM / 32 * chunk + j]) : 0.0f;
            top = fmaxf(top, fabsf(x[i][c * J + j]));
          }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // taken to at most 2^9, so that sums over a quarter stay in fp16 and entries lose bits from 2^-29 of the largest on
      int e = static_cast<int>(__float_as_uint(top) >> 23) - 126;        // top < 2^e
      e = top == 0.0f || top == INFINITY ? 9 : e;
      const int up = min(max(9 - e, -126), 126);
      const float by = power2(up);
      float sum[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sum[i] = 0.0f;
#pragma unroll
        for (int j = 0; j < 2 * J; ++j) { x[i][j] *= by; sum[i] += x[i][j]; }
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
#pragma unroll
        for (int u = 0; u < STEPS; ++u) {
          qb[nt][i][u][0] = pack2(x[i][2 * u], x[i][J + 2 * u]);
          qb[nt][i][u][1] = pack2(x[i][2 * u + 1] * (BITS == 4 ? 0.0625f : 1.0f), x[i][J + 2 * u + 1] * (BITS == 4 ? 0.0625f : 1.0f));
        }
      }
      // columns 2 t and 2 t + 1 of the sums: lanes 8 t and 8 t + 4
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        start[nt][i][0] = -M * UNIT * __shfl_sync(0xffffffffu, sum[i], 8 * t);
        start[nt][i][1] = -M * UNIT * __shfl_sync(0xffffffffu, sum[i], 8 * t + 4);
      }
      const float down = p.scale_log2 * power2(-up);
      factor[nt][0] = __shfl_sync(0xffffffffu, down, 8 * t);
      factor[nt][1] = __shfl_sync(0xffffffffu, down, 8 * t + 4);
      const float s0 = t & 1 ? sum[2] : sum[0], s1 = t & 1 ? sum[3] : sum[1];
      const uint32_t upper = pack2(s0, s1);
      const float2 back = __half22float2(h2(upper));
      qz[nt] = t < 2 ? upper : pack2(s0 - back.x, s1 - back.y);
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        zacc[nt][i] = 0.0f;
#pragma unroll
        for (int u = 0; u < STEPS; ++u) { acc[nt][i][u][0] = 0.0f; acc[nt][i][u][1] = 0.0f; acc[nt][i][u][2] = 0.0f; acc[nt][i][u][3] = 0.0f; }
      }
    }
    f01 = f23 = __float2half2_rn(0x1p15f);
  }

  // Scores of 16 rows, in powers of two: rows g and g + 8, heads 2 t and 2 t + 1
  __device__ __forceinline__ void scores(uint32_t kt, int lane, float (&x)[NT][4]) const {
    const int t = lane & 3, g = lane >> 2;
    uint32_t w[2][2][N];                         // row, chunk
    float s[2][4];
    uint32_t z[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint32_t at = kt + (g + 8 * r) * ROW;
      if constexpr (SPREAD) {
        lds<N>(at + t * CHUNK, w[r][0]);
        lds<N>(at + (t + 4) * CHUNK, w[r][1]);
      } else {
        uint32_t both[2 * N];
        lds<2 * N>(at + 2 * t * CHUNK, both);
#pragma unroll
        for (int i = 0; i < N; ++i) { w[r][0][i] = both[i]; w[r][1][i] = both[N + i]; }
      }
      uint32_t sw[2], zw[1];
      lds<2>(at + CODES, sw);
      lds<1>(at + CODES + 8 + 4 * (t & 1), zw);
      const float2 s01 = __half22float2(h2(sw[0])), s23 = __half22float2(h2(sw[1]));
      s[r][0] = s01.x; s[r][1] = s01.y; s[r][2] = s23.x; s[r][3] = s23.y;
      z[r] = zw[0];
    }
    float y[NT][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t top[J], low[J];
      expand<DIM, BITS>(w[0][0], w[0][1], i, top);
      expand<DIM, BITS>(w[1][0], w[1][1], i, low);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float c[4];
        mma(c, top[0], low[0], top[1], low[1], qb[nt][i][0][0], qb[nt][i][0][1], start[nt][i][0], start[nt][i][1], start[nt][i][0], start[nt][i][1]);
        if constexpr (STEPS == 2) mma(c, top[J - 2], low[J - 2], top[J - 1], low[J - 1], qb[nt][i][STEPS - 1][0], qb[nt][i][STEPS - 1][1], c[0], c[1], c[2], c[3]);
#pragma unroll
        for (int e = 0; e < 4; ++e) y[nt][e] = i == 0 ? c[e] * s[e / 2][0] : fmaf(c[e], s[e / 2][i], y[nt][e]);
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float c[4];
      mma_k8(c, z[0], z[1], qz[nt]);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[nt][e] = fmaf(y[nt][e], factor[nt][e % 2] * 0x1p24f, c[e] * factor[nt][e % 2]);
    }
  }

  // Weights of 16 rows (upper and lower parts, rows 2 t, 2 t + 1 and those + 8 of head g) times their values
  __device__ __forceinline__ void weigh(uint32_t vt, int lane, const uint32_t (&hi)[NT][2], const uint32_t (&lo)[NT][2]) {
    const int t = lane & 3, g = lane >> 2;
    uint32_t w[4][N], s[4][2], z[2];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint32_t at = vt + (2 * t + (r & 1) + 8 * (r >> 1)) * ROW;
      lds<N>(at + g * CHUNK, w[r]);
      lds<2>(at + CODES, s[r]);
      s[r][0] = bits_of(__hmul2(h2(s[r][0]), f01));
      s[r][1] = bits_of(__hmul2(h2(s[r][1]), f23));
      const uint32_t one = lds16(at + CODES + 8 + 2 * (g & 3));
      z[r >> 1] = r & 1 ? z[r >> 1] | one << 16 : one;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t first[J], second[J], pb[NT][2];
      const uint32_t sel = i % 2 ? 0x7632 : 0x5410;
      const __half2 s0 = h2(__byte_perm(s[0][i / 2], s[1][i / 2], sel)), s1 = h2(__byte_perm(s[2][i / 2], s[3][i / 2], sel));
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        pb[nt][0] = bits_of(__hfma2(h2(hi[nt][0]), s0, __hmul2(h2(lo[nt][0]), s0)));
        pb[nt][1] = bits_of(__hfma2(h2(hi[nt][1]), s1, __hmul2(h2(lo[nt][1]), s1)));
      }
      expand<DIM, BITS>(w[0], w[1], i, first);
      expand<DIM, BITS>(w[2], w[3], i, second);
#pragma unroll
      for (int j = 0; j < J; ++j) {              // (exact: whole multiples of 2^-24)
        const __half2 middle = __float2half2_rn(-M * UNIT * (BITS == 4 && j % 2 ? 16.0f : 1.0f));
        first[j] = bits_of(__hadd2(h2(first[j]), middle));
        second[j] = bits_of(__hadd2(h2(second[j]), middle));
      }
#pragma unroll
      for (int u = 0; u < STEPS; ++u)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float (&c)[4] = acc[nt][i][u];
          mma(c, first[2 * u], first[2 * u + 1], second[2 * u], second[2 * u + 1], pb[nt][0], pb[nt][1], c[0], c[1], c[2], c[3]);
        }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float (&c)[4] = zacc[nt];
      mma(c, z[0], z[0], z[1], z[1], hi[nt][0], hi[nt][1], c[0], c[1], c[2], c[3]);
      mma(c, z[0], z[0], z[1], z[1], lo[nt][0], lo[nt][1], c[0], c[1], c[2], c[3]);
    }
  }

  // A tile, of which `rows` rows (32 or fewer) are there
  __device__ __forceinline__ void tile(uint32_t kt, int rows, int lane) {
    const int g = lane >> 2;
    const uint32_t vt = kt + TILE * ROW;
    float x[2][NT][4];
    scores(kt, lane, x[0]);
    scores(kt + 16 * ROW, lane, x[1]);
    if (rows < TILE) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (16 * h + g + 8 * (e / 2) >= rows) x[h][nt][e] = -INFINITY;
    }
    // the maximum moves when a score is SLACK above it
    bool rises = false;
    float top[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        top[nt][e] = fmaxf(fmaxf(x[0][nt][e], x[0][nt][e + 2]), fmaxf(x[1][nt][e], x[1][nt][e + 2]));
        rises |= top[nt][e] > m[nt][e] + SLACK;
      }
    if (__any_sync(0xffffffffu, rises)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float v = top[nt][e];
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
          v = fmaxf(v, m[nt][e]);
          const float f = v == -INFINITY ? 1.0f : exp2_fast(m[nt][e] - v);
          m[nt][e] = v;
          l[nt][e] *= f;
          zacc[nt][e] *= f;
          zacc[nt][e + 2] *= f;
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int u = 0; u < STEPS; ++u) { acc[nt][i][u][e] *= f; acc[nt][i][u][e + 2] *= f; }
        }
    }
    // the scales of values: a row to a lane
    {
      uint32_t s[2];
      lds<2>(vt + lane * ROW + CODES, s);
      const __half2 over = __hmax2(__hmul2(h2(s[0]), f01), __hmul2(h2(s[1]), f23));
      if (__any_sync(0xffffffffu, __low2float(over) > 1.0f || __high2float(over) > 1.0f)) {
        __half2 a = h2(s[0]), c = h2(s[1]);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          a = __hmax2(a, h2(__shfl_xor_sync(0xffffffffu, bits_of(a), o)));
          c = __hmax2(c, h2(__shfl_xor_sync(0xffffffffu, bits_of(c), o)));
        }
        const float2 a2 = __half22float2(a), c2 = __half22float2(c), f2 = __half22float2(f01), g2 = __half22float2(f23);
        const float most[4] = {a2.x, a2.y, c2.x, c2.y}, old[4] = {f2.x, f2.y, g2.x, g2.y};
        float now[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // the power of two that takes `most` into (1/2, 1]
          const int e = static_cast<int>((__float_as_uint(most[i]) + 0x7fffffu) >> 23) - 127;
          now[i] = fminf(old[i], power2(min(max(-e, -14), 15)));
          const float f = now[i] / old[i];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int u = 0; u < STEPS; ++u) { acc[nt][i][u][0] *= f; acc[nt][i][u][1] *= f; acc[nt][i][u][2] *= f; acc[nt][i][u][3] *= f; }
        }
        f01 = __floats2half2_rn(now[0], now[1]);
        f23 = __floats2half2_rn(now[2], now[3]);
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t hi[NT][2], lo[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float at = m[nt][e % 2];
          w[e] = exp2_fast(x[h][nt][e] - ((at == -INFINITY ? 0.0f : at) - SHIFT));
          l[nt][e % 2] += w[e];
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint32_t upper = pack2(w[2 * r], w[2 * r + 1]);
          const float2 back = __half22float2(h2(upper));
          hi[nt][r] = transposed(upper);
          lo[nt][r] = transposed(pack2(w[2 * r] - back.x, w[2 * r + 1] - back.y));
        }
      }
      weigh(vt + 16 * h * ROW, lane, hi, lo);
    }
  }

  // The state of a part to the workspace (slot >= 0), or the output of a whole item
  __device__ __forceinline__ void end(const AttendParams &p, int b, int kv_head, int slot, int lane) {
    const int t = lane & 3, g = lane >> 2;
    const float2 f2 = __half22float2(f01), g2 = __half22float2(f23);
    const float inverse[4] = {1.0f / f2.x / UNIT, 1.0f / f2.y / UNIT, 1.0f / g2.x / UNIT, 1.0f / g2.y / UNIT};
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float total = l[nt][e];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        float v[4][J];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float z = __shfl_sync(0xffffffffu, zacc[nt][e], 4 * i + t);
#pragma unroll
          for (int j = 0; j < J; ++j) v[i][j] = fmaf(acc[nt][i][j / 2][e + 2 * (j % 2)], inverse[i] * (BITS == 4 && j % 2 ? 0.0625f : 1.0f), z);
        }
        const int h = nt * 8 + 2 * t + e;
        if (h >= p.group) continue;
        if (slot >= 0) {
          const size_t at = static_cast<size_t>(slot) * p.group + h;
          if (g == 0) p.part_ml[at] = make_float2(m[nt][e], total);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float *const to = p.part_out + at * DIM + DIM / 4 * i + J * g;
            if constexpr (J == 4) *reinterpret_cast<float4 *>(to) = make_float4(v[i][0], v[i][1], v[i][J - 2], v[i][J - 1]);
            else *reinterpret_cast<float2 *>(to) = make_float2(v[i][0], v[i][1]);
          }
        } else {
          const size_t at = static_cast<size_t>(b) * p.q_heads + kv_head * p.group + h;
          if (g == 0 && p.lse) p.lse[at] = total == 0.0f ? -INFINITY : (m[nt][e] - SHIFT) * LN2 + logf(total);
          const float by = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            T *const to = static_cast<T *>(p.out) + at * DIM + DIM / 4 * i + J * g;
            T o[J];
#pragma unroll
            for (int j = 0; j < J; ++j) o[j] = static_cast<T>(v[i][j] * by);
            if constexpr (J == 4) *reinterpret_cast<uint2 *>(to) = *reinterpret_cast<const uint2 *>(o);
            else *reinterpret_cast<uint32_t *>(to) = *reinterpret_cast<const uint32_t *>(o);
          }
        }
      }
  }
};

template <typename T, int DIM, int BITS, int NT>
__global__ void __launch_bounds__(WARPS * 32, ctas_per_sm(NT)) attend_tiles(const __grid_constant__ AttendParams p) {
  using A = Attend<T, DIM, BITS, NT>;
  constexpr int STAGES = A::STAGES;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ Line line;
  __shared__ int sums[MAX_SEQS / 32];
  pdl_wait();
  pdl_trigger();
  make_line(p, line, sums);
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = warp * gridDim.x + blockIdx.x, parts = min(p.warps, line.total);          // (few stretches: on as many SMs)
  if (r >= parts) return;
  const int first = begin_of(line.total, parts, r), last = begin_of(line.total, parts, r + 1);
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * (STAGES * A::STAGE);
  Place ahead, now;
  now.start(p, line, first);
  ahead = now;
  int fetched = first;
  auto fetch = [&]() {
    if (fetched < last) {
      A::load(p, ahead, ring + (fetched - first) % STAGES * A::STAGE, lane);
      ahead.next(p);
    }
    ++fetched;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) fetch();
  A a;
  a.begin(p, now.b, now.head, lane);
  int began = now.tile;
  for (int i = first; i < last; ++i) {
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    __syncwarp();                                // every lane's copies of tile i are there, and tile i - 1 has been read
    fetch();
    a.tile(ring + (i - first) % STAGES * A::STAGE, min(now.rows - now.tile * TILE, TILE), lane);
    const bool done = now.tile == now.tiles - 1;
    if (done || i == last - 1) {
      const bool whole = done && began == 0;
      a.end(p, now.b, now.head, whole ? -1 : 2 * r + (began == 0 && i - first > now.tile), lane);
    }
    if (i == last - 1) break;
    now.next(p);
    if (done) {
      a.begin(p, now.b, now.head, lane);
      began = 0;
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// A CTA joins the parts of a (sequence, query head): a warp takes every JOIN_WARPS-th, eight at a time.
constexpr int JOIN_WARPS = 8;
template <typename T, int DIM>
__global__ void __launch_bounds__(JOIN_WARPS * 32) join_stretches(const __grid_constant__ AttendParams p) {
  constexpr int E = DIM / 32, AHEAD = 8;
  __shared__ Line line;
  __shared__ int sums[MAX_SEQS / 32];
  __shared__ float sm[JOIN_WARPS], sl[JOIN_WARPS];
  __shared__ __align__(16) float sa[JOIN_WARPS][DIM];
  const int b = static_cast<int>(blockIdx.x) / p.q_heads, head = static_cast<int>(blockIdx.x) % p.q_heads, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // (the lengths were there before the kernel that this one follows)
  make_line(p, line, sums);
  __syncthreads();
  const int tiles = tiles_of(seen_rows(p, b));
  const size_t row = blockIdx.x;
  if (tiles == 0) {
    pdl_wait();
    if (threadIdx.x < DIM) static_cast<T *>(p.out)[row * DIM + threadIdx.x] = static_cast<T>(0.0f);
    if (threadIdx.x == 0 && p.lse) p.lse[row] = -INFINITY;
    return;
  }
  const int parts = min(p.warps, line.total), t0 = line.before[b] + head / p.group * tiles;
  const int r0 = part_of(line.total, parts, t0), r1 = part_of(line.total, parts, t0 + tiles - 1);
  pdl_wait();
  if (r0 == r1) return;                          // (written there)
  const bool inside = begin_of(line.total, parts, r0) < t0;
  float M = -INFINITY, L = 0.0f, A[E];
#pragma unroll
  for (int i = 0; i < E; ++i) A[i] = 0.0f;
  // (a maximum of -inf: nothing seen, or a sum that is no number and stays one)
  auto weight = [](float m, float l, float top) { return m == -INFINITY ? (l == 0.0f ? 0.0f : 1.0f) : exp2f(m - top); };
  for (int first = r0 + warp; first <= r1; first += JOIN_WARPS * AHEAD) {
    float v[AHEAD][E];
    float2 ml[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int r = first + i * JOIN_WARPS;
      ml[i] = make_float2(-INFINITY, 0.0f);
#pragma unroll
      for (int k = 0; k < E; ++k) v[i][k] = 0.0f;
      if (r <= r1) {
        const size_t at = static_cast<size_t>(2 * r + (r == r0 && inside)) * p.group + head % p.group;
        ml[i] = p.part_ml[at];
        const float *const src = p.part_out + at * DIM + lane * E;
        if constexpr (E == 4) { const float4 a = *reinterpret_cast<const float4 *>(src); v[i][0] = a.x; v[i][1] = a.y; v[i][E - 2] = a.z; v[i][E - 1] = a.w; }
        else { const float2 a = *reinterpret_cast<const float2 *>(src); v[i][0] = a.x; v[i][1] = a.y; }
      }
    }
    float top = M;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) top = fmaxf(top, ml[i].x);
    const float f0 = weight(M, L, top);
    M = top;
    L *= f0;
#pragma unroll
    for (int k = 0; k < E; ++k) A[k] *= f0;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const float f = weight(ml[i].x, ml[i].y, top);
      L = fmaf(ml[i].y, f, L);
#pragma unroll
      for (int k = 0; k < E; ++k) A[k] = fmaf(v[i][k], f, A[k]);
    }
  }
  if (lane == 0) { sm[warp] = M; sl[warp] = L; }
#pragma unroll
  for (int i = 0; i < E; ++i) sa[warp][lane * E + i] = A[i];
  __syncthreads();
  if (threadIdx.x >= DIM) return;
  float top = -INFINITY, total = 0.0f, out = 0.0f;
#pragma unroll
  for (int w = 0; w < JOIN_WARPS; ++w) top = fmaxf(top, sm[w]);
#pragma unroll
  for (int w = 0; w < JOIN_WARPS; ++w) {
    const float f = weight(sm[w], sl[w], top);
    total = fmaf(sl[w], f, total);
    out = fmaf(sa[w][threadIdx.x], f, out);
  }
  static_cast<T *>(p.out)[row * DIM + threadIdx.x] = static_cast<T>(total == 0.0f ? 0.0f : out / total);
  if (p.lse && threadIdx.x == 0) p.lse[row] = total == 0.0f ? -INFINITY : (top - SHIFT) * LN2 + logf(total);
}

}  // namespace qmk_packed
#endif  // QMK_PACKED_ATTENTION_CUH_
