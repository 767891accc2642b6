// Attention of one new token per sequence over a packed cache (packed_cache.cuh): out = softmax(scale * q . k) v, k and v the rows' values.
//
// With n the codes, M = 2^(BITS - 1), b(d) the quarter of dimension d, s and z a row's scales and centres:
//   q . k = sum_b s_b (sum_{d in b} q_d n_d - M Q_b) + sum_b z_b Q_b,   Q_b = sum_{d in b} q_d,
//   out_d = sum_r p_r z_{r,b(d)} + sum_r (p_r s_{r,b(d)}) n_{r,d} - M sum_r (p_r s_{r,b(d)}),
// so codes enter the products as they are: the number n 2^-24 is the fp16 pattern n (of 4 bits 16 n, 2^-20 each), and masking some bits of both halves of a word makes two operands.  Rows
// of the cache are the 16 rows of an mma.sync tile, query heads its eight columns; a row's trailer, 16 bytes, is a row of an 8 x 8 tile, so ldmatrix makes the operands of the sums over
// centres.  tcgen05 could have rows of the cache, or dimensions, as its M too, but takes that operand from shared or tensor memory: codes would be expanded into it, 512 bytes a row of keys
// and values of 128 dims, by estimate 4 cycles of an SM's shared memory a row or 90 us of the 187 of 96 sequences of 8192 rows, besides reading it; mma.sync takes them from the
// registers in which they are expanded.
//
// Roundings: queries are taken to fp16 times a power of two (Tiles::lift).  Weights and their products with scales are carried as two fp16 numbers each, because the tensor cores multiply
// 16-bit numbers: over many outputs the error against 64 bits is that of rounding the exact result (1.06 to 1.36 times with one number a product, which took 16 of up to 2048
// rows 12.8 us, 128 of up to 8192 122, 96 of 8192 160 and 32 of up to 4096 with sixteen heads a kv head 23.5, where two took 13.6, 125, 175 and 27.9).  So for bf16 outputs: with one number each
// an output whose terms cancel is off by up to 2^-10 of these.  Sums, softmax statistics and outputs are fp32.  Every second 16 rows go in as 2^BITS - 1 - n with the
// weights' sign turned (the same instructions): the running sums stay around zero, whose size the accumulator's truncation goes by.
//
// Work: tiles of 32 rows, a tile to a warp, each with a ring of copies of its own (cp.async: no waits but for its own copies).  attend_items: a cluster of CTAs has a (sequence, kv
// head) and joins its states - the maximum, the sum and the unnormalised output - in shared memory.  attend_tiles: the tiles of all items in one line, of which
// each warp takes an equal stretch, whatever the sequences' lengths; a stretch that holds a whole item writes its output, parts of items leave their states in the workspace,
// and a second launch joins them.  Of few long items each is shared by many clusters of attend_items, which leave a state each.
//
// Measured in a graph, caches cold: 96 sequences of 8192 rows, two heads on each of eight kv heads, 4 bits: 187 us, 5.4 TB/s, 0.82 of the copy rate, with 291 warp
// instructions for 16 rows: HBM and the issue of instructions; 64 of up to 4096 in 8 bits 57, 0.82.  32 of 8192 rows (336 MB) with 2 / 4 / 8 / 16 query heads a kv head: 70 / 78 / 93 / 161,
// attend_tiles alone under the profiler 72 / 81 / 93 / 160: instructions (291 / 321 / 359 / 509 for 16 rows, issued in 56 / 54 / 53 / 44 % of the cycles; four or three warps a scheduler,
// waits for the ALU and fixed latencies), with 16 also 255 registers and two warps a scheduler.  The joins: 4 to 6 us.
#ifndef QMK_PACKED_ATTENTION_CUH_
#define QMK_PACKED_ATTENTION_CUH_

#include "packed_cache.cuh"

namespace qmk_packed {

constexpr int MAX_GROUP = 16;                    // query heads per kv head
constexpr int TILE = 32;                         // rows
constexpr int WARPS = 4, SMS = 148;
// How a tile is taken: by one or two query heads (PAIR), three or four (QUAD), blocks of up to eight (ONE, TWO)
enum Way { PAIR, QUAD, ONE, TWO };
__host__ __device__ constexpr Way way_of(int group) { return group <= 2 ? PAIR : group <= 4 ? QUAD : group <= 8 ? ONE : TWO; }
// CTAs on an SM: four where 128 registers do and a tile has at most 5 KB, three of 168, or two of 255.  Four against three, us: 96 sequences of 8192 rows 187 and 188 (PAIR), 128 of up
// to 256 17.4 and 20.8; four heads a kv head (QUAD), 64 of up to 512 rows 15.1 and 18.5, one of 32,768 19.3 and 19.9, 64 of up to 4096 51.2 and 48.4; ONE with 128 dims spills in 128
// registers: 64 of up to 4096, eight heads a kv head, 43.4 and 37.6.
__host__ __device__ constexpr int ctas_per_sm(Way way, int dim, int bits) { return way == TWO ? 2 : bits * dim <= 512 && (way != ONE || dim == 64) ? 4 : 3; }
// (228 KB an SM; of a CTA 1 KB is the system's, 1.25 KB the line's)
constexpr int warp_bytes(int ctas) { return (228 * 1024 - ctas * 2304) / (ctas * WARPS); }
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
// Weights are 2^SHIFT at the row's maximum, up to 2^(SHIFT + SLACK) where that has risen since it was last looked at: fp16 has 11 bits of them down to 2^-21 of
// the largest.
constexpr float SHIFT = 7.0f, SLACK = 8.0f;
constexpr float NOTHING = -3.0e38f;              // the maximum while no score has been seen: the first one rises (times 2^-120 it is -256 below), -inf stays that
// The largest factor (scores are below 2^12 in their units, so products stay finite).  One that is cut to it makes the same weights: scores that differ do so by 2^-72 at least, and
// that times 2^112 leaves the largest alone.
constexpr float MOST = 0x1p112f;

struct AttendParams {
  Caches caches;
  const void *q;
  long long q_seq, q_head;                       // strides, in elements
  int q_heads, group;
  const int *lens;
  float scale_log2;                              // scale * log2 e
  int ranks;                                     // where items have clusters of their own: log2 of the CTAs that share one, + 1; else 0
  int splits;                                    // the clusters of an item, at most
  int warps;                                     // parts that are left for a second launch, at most: of warps, or of clusters (0: none)
  float *part_out;                               // [2 warps][group][DIM], every second one unused where clusters make them
  float2 *part_ml;                               // [2 warps][group]
  void *out;                                     // [seq][q_head][DIM]
  float *lse;
};

__device__ __forceinline__ void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool there) {         // zeros where there is no row
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void *src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, float c0, float c1, float c2, float c3) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
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
// The trailers of 16 rows as 8 x 8 tiles that make an operand of a product: row g's entries 2 t and 2 t + 1 and row g + 8's, twice; transposed: entry g of rows
// 2 t and 2 t + 1, twice, and of rows 2 t + 8 and 2 t + 9, twice.
template <bool TRANSPOSED, int ROW> __device__ __forceinline__ void trailers(uint32_t first, int lane, uint32_t (&w)[4]) {
  if constexpr (TRANSPOSED) {
    const uint32_t at = first + ((lane & 7) + (lane >> 4) * 8) * ROW;
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
  } else {
    const uint32_t at = first + (lane & 15) * ROW;
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
  }
}

// (as a multiplication, whose pipe has room where that of shifts and masks has not: 128 sequences of up to 8192 rows 133.2 us, by a shift 135.0)
__device__ __forceinline__ uint32_t times16(uint32_t x) {
  uint32_t y;
  asm("mad.lo.u32 %0, %1, %2, 0;" : "=r"(y) : "r"(x), "r"(16u));
  return y;
}
// Codes of quarter b of two chunks (DIM/8 codes each), the first in the lower halves: x[j] = (a_j, b_j) as fp16 numbers of UNIT (2^-24; 4-bit codes of 2^-20); FLIP:
// 2^BITS - 1 less the code.  These numbers have fp16's smallest exponent, by which the tensor cores line products up: codes of 4 bits in the lowest places would keep four bits less
// of them, so that sums of a few rows were off by up to 2^-17 of their terms, scores by 2^-20.
template <int DIM, int BITS, bool FLIP = false>
__device__ __forceinline__ void expand(const uint32_t (&a)[DIM * BITS / 256], const uint32_t (&c)[DIM * BITS / 256], int b, uint32_t (&x)[DIM / 32]) {
  constexpr uint32_t ALL = FLIP ? 0xffffffffu : 0u;
  if constexpr (BITS == 4 && DIM == 64) {
    const uint32_t w = __byte_perm(a[0], c[0], b | b << 4 | (4 + b) << 8 | (4 + b) << 12);
    x[0] = (times16(w) ^ ALL) & 0x00f000f0u;
    x[1] = (w ^ ALL) & 0x00f000f0u;
  } else if constexpr (BITS == 4) {
    const uint32_t w = __byte_perm(a[b / 2], c[b / 2], b % 2 ? 0x7632 : 0x5410), u = w >> 8;
    x[0] = (times16(w) ^ ALL) & 0x00f000f0u;
    x[1] = (w ^ ALL) & 0x00f000f0u;
    x[2] = (times16(u) ^ ALL) & 0x00f000f0u;
    x[3] = (u ^ ALL) & 0x00f000f0u;
  } else if constexpr (DIM == 64) {
    const uint32_t w = __byte_perm(a[b / 2], c[b / 2], b % 2 ? 0x7632 : 0x5410), u = w >> 8;
    x[0] = (w ^ ALL) & 0x00ff00ffu;
    x[1] = (u ^ ALL) & 0x00ff00ffu;
  } else {
    const uint32_t w = __byte_perm(a[b], c[b], 0x5410), u = __byte_perm(a[b], c[b], 0x7632), w8 = w >> 8, u8 = u >> 8;
    x[0] = (w ^ ALL) & 0x00ff00ffu;
    x[1] = (w8 ^ ALL) & 0x00ff00ffu;
    x[2] = (u ^ ALL) & 0x00ff00ffu;
    x[3] = (u8 ^ ALL) & 0x00ff00ffu;
  }
}

// The line of tiles: sequence by sequence, kv head by kv head.
struct Line {
  int total;                                     // tiles
  int before[MAX_SEQS], rows[MAX_SEQS];          // tiles in front of a sequence, rows that it sees
};
__device__ __forceinline__ int seen_rows(const AttendParams &p, int b) { return min(max(p.lens[b], 0), p.caches.rows); }
__device__ __forceinline__ int tiles_of(int rows) { return (rows + TILE - 1) / TILE; }
// (a sequence to each of the first threads; in front of a barrier of the caller's)
__device__ __forceinline__ void make_line(const AttendParams &p, Line &line, int (&sums)[MAX_SEQS / 32]) {
  const int i = threadIdx.x, lane = i & 31;
  const int rows = i < p.caches.seqs ? seen_rows(p, i) : 0, own = tiles_of(rows) * p.caches.kv_heads;
  int n = own;
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
  if (i < MAX_SEQS) { line.before[i] = n - own; line.rows[i] = rows; }
  if (i == MAX_SEQS - 1) line.total = n;
}
// Stretch r of `parts` equal ones begins at tile total * r / parts; the stretch that holds tile t
__device__ __forceinline__ int begin_of(int total, int parts, int r) { return static_cast<int>(static_cast<long long>(total) * r / parts); }
__device__ __forceinline__ int part_of(int total, int parts, int t) { return static_cast<int>(((t + 1ll) * parts - 1) / total); }

// A place in the line
struct Place {
  int b, head, tile, tiles, rows;
  __device__ __forceinline__ void sequence(const Line &line, int at) {
    b = at;
    rows = b < MAX_SEQS ? line.rows[b] : 0;
    tiles = tiles_of(rows);
  }
  __device__ __forceinline__ void start(const AttendParams &p, const Line &line, int t) {
    int low = 0, high = p.caches.seqs - 1;       // the last sequence that begins at t or before, and has tiles
    while (low < high) {
      const int mid = (low + high + 1) / 2;
      if (line.before[mid] <= t) low = mid; else high = mid - 1;
    }
    sequence(line, low);
    const int i = t - line.before[low];
    head = i / tiles;
    tile = i - head * tiles;
  }
};

// An item on a warp's way along the line, and how many of its rows are left
struct Item {
  int b, head, left;
  __device__ __forceinline__ void next(const AttendParams &p, const Line &line) {
    if (++head == p.caches.kv_heads) {
      head = 0;
      do ++b; while (b < p.caches.seqs && line.rows[b] == 0);
    }
    left = b < p.caches.seqs ? line.rows[b] : 0;
  }
};
// Where its next tile is copied from: the lane's first 16 bytes of it
struct Source {
  const unsigned char *k, *v;
  __device__ __forceinline__ void at(const AttendParams &p, const Item &item, int tile, int lane) {
    const long long base = static_cast<long long>(item.head) * p.caches.head + static_cast<long long>(tile) * TILE * p.caches.row + lane * 16;
    k = p.caches.k[item.b] + base;
    v = p.caches.v[item.b] + base;
  }
  __device__ __forceinline__ void next(const AttendParams &p) { k += TILE * p.caches.row; v += TILE * p.caches.row; }
};

// DIM/32 values of a row side by side
template <int DIM> __device__ __forceinline__ void store_part(float *to, const float (&v)[DIM / 32]) {
  if constexpr (DIM == 128) *reinterpret_cast<float4 *>(to) = make_float4(v[0], v[1], v[DIM / 32 - 2], v[DIM / 32 - 1]);
  else *reinterpret_cast<float2 *>(to) = make_float2(v[0], v[1]);
}
template <typename T, int DIM> __device__ __forceinline__ void store_out(T *to, const float (&v)[DIM / 32], float by) {
  T o[DIM / 32];
#pragma unroll
  for (int j = 0; j < DIM / 32; ++j) o[j] = static_cast<T>(v[j] * by);
  if constexpr (DIM == 128) *reinterpret_cast<uint2 *>(to) = make_uint2(*reinterpret_cast<const uint32_t *>(o), *reinterpret_cast<const uint32_t *>(o + DIM / 32 - 2));
  else *reinterpret_cast<uint32_t *>(to) = *reinterpret_cast<const uint32_t *>(o);
}

// What the ways to take a tile have in common.
template <int DIM, int BITS, Way WAY, int HEADS>
struct Tiles {
  static constexpr int CTAS = ctas_per_sm(WAY, DIM, BITS), HEAD_DIM = DIM;
  static constexpr int ROW = ROW_BYTES<DIM, BITS>, CODES = ROW - TRAILER, PIECES = ROW / 16;
  static constexpr int CHUNK = CODES / 8, N = CHUNK / 4, J = DIM / 32, STEPS = J / 2;       // bytes and words of a chunk; codes of a quarter in it; k steps of a quarter
  static constexpr int STAGE = 2 * TILE * ROW;                                              // keys, then values
  static constexpr int FIT = warp_bytes(CTAS) / STAGE, STAGES = FIT < 4 ? FIT : 4;
  // Queries of the next item, copied with its first rows; where a warp's shared memory has room
  static constexpr int QUERIES = STAGES * STAGE + HEADS * DIM * 2 <= warp_bytes(CTAS) ? HEADS * DIM * 2 : 0;
  static constexpr int QUERY_STRIDE = DIM, WARP_SMEM = STAGES * STAGE + QUERIES, SMEM = WARPS * WARP_SMEM;
  static_assert(STAGES * STAGE >= HEADS * (DIM * 4 + 8), "a warp's state fits its ring");
  static constexpr float M = 1 << (BITS - 1), UNIT = BITS == 4 ? 0x1p-20f : 0x1p-24f;
  // What the codes (the flipped ones) are above the numbers they stand for, negative, as pairs of fp16 numbers
  static constexpr uint32_t MIDDLE = BITS == 4 ? 0xc800c800u : 0xd800d800u, MIDDLE_FLIPPED = BITS == 4 ? 0xc700c700u : 0xd7f0d7f0u;         // -8, -128; -7, -127
  static constexpr bool SPREAD = BITS == 8 && DIM == 128;                                   // a lane's two chunks of keys: four apart, or one behind the other
  static __device__ __forceinline__ int chunk_of(int t, int c) { return SPREAD ? t + 4 * c : 2 * t + c; }

  static __device__ __forceinline__ void load(const AttendParams &p, const Source &from, int rows, uint32_t dst, int lane) {
    if (p.caches.row == ROW && rows >= TILE) {   // rows right behind one another, all there
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        copy16(dst + lane * 16 + 512 * i, from.k + 512 * i);
        copy16(dst + lane * 16 + TILE * ROW + 512 * i, from.v + 512 * i);
      }
    } else {
      const unsigned char *const k = from.k - lane * 16, *const v = from.v - lane * 16;
      const int pieces = min(rows, TILE) * PIECES;
#pragma unroll 1
      for (int i = 0; i < PIECES; ++i) {
        const int piece = lane + 32 * i;
        const bool there = piece < pieces;
        const long long off = there ? piece / PIECES * p.caches.row + piece % PIECES * 16 : 0;
        copy16(dst + piece * 16, k + off, there);
        copy16(dst + TILE * ROW + piece * 16, v + off, there);
      }
    }
  }
  // The queries of an item, one head behind the other
  template <typename T>
  static __device__ __forceinline__ void load_queries(const AttendParams &p, const Item &at, uint32_t dst, int lane) {
    const T *const q = static_cast<const T *>(p.q) + at.b * p.q_seq + static_cast<long long>(at.head) * p.group * p.q_head;
    for (int i = lane; i < p.group * (DIM / 8); i += 32) copy16(dst + i * 16, q + i / (DIM / 8) * p.q_head + i % (DIM / 8) * 8);
  }
  // The lane's two chunks of keys of row g
  static __device__ __forceinline__ void keys(uint32_t row, int t, uint32_t (&w)[2][N]) {
    if constexpr (SPREAD) {
      lds<N>(row + t * CHUNK, w[0]);
      lds<N>(row + (t + 4) * CHUNK, w[1]);
    } else {
      uint32_t both[2 * N];
      lds<2 * N>(row + 2 * t * CHUNK, both);
#pragma unroll
      for (int i = 0; i < N; ++i) { w[0][i] = both[i]; w[1][i] = both[N + i]; }
    }
  }
  // The power of two that queries of which the largest is `top` are multiplied with: to at most 2^TOP, so that M times the sum over a quarter stays in fp16.  An entry
  // is off by 2^-25 of the largest at most: those below about 2^-14 of it may lose bits.
  static constexpr int TOP = BITS == 4 ? 5 : 1;
  static __device__ __forceinline__ int lift(float top) {
    const int e = static_cast<int>(__float_as_uint(top) >> 23) - 126;      // top < 2^e
    return top == 0.0f || top == INFINITY ? 0 : min(max(TOP - e, -126), 126);
  }
  // What a score is multiplied by (a factor of 0 would make no number of the scores of rows that are not there, -inf)
  static __device__ __forceinline__ float factor_of(const AttendParams &p, int lifted) { return fminf(fmaxf(fabsf(p.scale_log2) * power2(-lifted) / UNIT, 0x1p-120f), MOST); }
  // The score, times log2 e, whose weight is 1 where that of the maximum is 2^SHIFT; at most the largest number.  Of a head whose factor was cut to MOST by what that would have been
  template <typename T>
  static __device__ __forceinline__ float level_of(const AttendParams &p, float m, float factor, int b, int q_head) {
    if (factor < MOST || isinf(m)) return fmaf(m, factor, -SHIFT);
    const T *const q = static_cast<const T *>(p.q) + b * p.q_seq + q_head * p.q_head;
    float top = 0.0f;
    for (int d = 0; d < DIM; ++d) top = fmaxf(top, fabsf(static_cast<float>(q[d])));
    const double x = static_cast<double>(m) * fabsf(p.scale_log2) * power2(-lift(top)) / UNIT;
    return static_cast<float>(fmin(fmax(x, -3.4e38), 3.4e38));
  }
  // The power of two that takes a scale into (1/2, 1], at most `old`
  static __device__ __forceinline__ float taken(float most, float old) {
    const int e = static_cast<int>((__float_as_uint(fmaxf(most, 0.0f)) + 0x7fffffu) >> 23) - 127;
    return fminf(old, power2(min(max(-e, -14), 15)));
  }
  // Two rows' weights times scales, all as upper and lower fp16 parts
  template <bool FLIP>
  static __device__ __forceinline__ void times(uint32_t hi, uint32_t lo, __half2 scales, uint32_t &upper, uint32_t &lower) {
    const __half2 s = FLIP ? __hneg2(scales) : scales, first = __hmul2(h2(hi), s);
    upper = bits_of(first);
    lower = bits_of(__hfma2(h2(lo), s, __hfma2(h2(hi), s, __hneg2(first))));
  }
  // The same where one of the powers of two is below 1, a scale above 1 having been seen: fp16 might not hold small scales times it, so they come as they are and it apart
  template <bool FLIP>
  static __device__ __forceinline__ void times(uint32_t hi, uint32_t lo, __half2 scales, float power, uint32_t &upper, uint32_t &lower) {
    const float2 a = __half22float2(h2(hi)), b = __half22float2(h2(lo)), s = __half22float2(scales);
    const float by = FLIP ? -power : power, x = (a.x + b.x) * s.x * by, y = (a.y + b.y) * s.y * by;
    upper = pack2(x, y);
    const float2 back = __half22float2(h2(upper));
    lower = pack2(x - back.x, y - back.y);
  }
};

// A tile where all of a thread's columns are of one query head; `rows` rows of it are there (32 or more: all).
template <int ROW, typename A>
__device__ __forceinline__ void take_tile(A &a, uint32_t kt, int rows, int lane) {
  const int g = lane >> 2;
  const uint32_t vt = kt + TILE * ROW;
  float x[2][2];
  a.scores(kt, lane, x[0]);
  a.scores(kt + 16 * ROW, lane, x[1]);
  if (rows < TILE) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (8 * e + g >= rows) x[e / 2][e % 2] = -INFINITY;
  }
  // the maximum moves when a score is SLACK above it
  float v = fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[1][0], x[1][1]));
  if (__any_sync(0xffffffffu, (v - a.m) * a.factor > SLACK)) {
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    v = fmaxf(v, a.m);
    a.scale(exp2_fast((a.m - v) * a.factor));
    a.m = v;
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t hi[2], lo[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float w = exp2_fast(fmaf(x[h][r] - a.m, a.factor, SHIFT));
      a.l += w;
      const uint32_t upper = pack2(w, w);
      const float rest = w - __low2float(h2(upper));
      hi[r] = transposed(upper);
      lo[r] = transposed(pack2(rest, rest));
    }
    if (h == 0) a.template weigh<false>(vt, lane, hi, lo);
    else a.template weigh<true>(vt + 16 * ROW, lane, hi, lo);
  }
}

// One or two query heads: each takes four of the eight columns, one for each quarter of the dimensions.  Keys: queries are zero outside their column's
// quarter, so one product over all codes has the quarters' sums side by side, each is scaled once, and pairs of codes need not be of one quarter; values: the weights'
// scales are the columns', one operand for all dimensions, of whose columns each quarter of the output keeps its own.
template <typename T, int DIM, int BITS>
struct AttendPair : Tiles<DIM, BITS, PAIR, 2> {
  using Value = T;
  using Base = Tiles<DIM, BITS, PAIR, 2>;
  using Base::ROW; using Base::CODES; using Base::N; using Base::J; using Base::STEPS; using Base::M; using Base::UNIT; using Base::CHUNK;
  static constexpr int PAIRS = 16 / BITS, KSTEPS = N * PAIRS;               // operand words of a word of codes; k steps of a row of keys

  uint32_t qb[KSTEPS][2], qz[2];                 // queries; sums over quarters, as upper and lower fp16 parts
  float factor, m, l;                            // what a score is multiplied by, the largest score, the sum of weights
  float acc[4][STEPS][4], sums[4], zacc[4];      // out^T, quarter by quarter; what is to be taken off; sums of weights times centres (lanes g >= 4: of quarter g - 4)
  __half2 f;                                     // power of two that takes quarter g & 3's scales of values to 1 or below
  bool wide;                                     // whether one of these is below 1

  __device__ __forceinline__ void begin(const AttendParams &p, const T *queries, long long stride, int lane) {
    const int t = lane & 3, g = lane >> 2, h = g >> 2, quarter = g & 3;
    const bool live = h < p.group;
    const T *const q = queries + (live ? h : 0) * stride + DIM / 4 * quarter;
    float x[2][J], top = 0.0f;
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int j = 0; j < J; ++j) {
        x[c][j] = live ? static_cast<float>(q[DIM / 32 * Base::chunk_of(t, c) + j]) : 0.0f;
        top = fmaxf(top, fabsf(x[c][j]));
      }
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const int up = Base::lift(top);
    const float by = copysignf(power2(up), p.scale_log2);
    float sum = 0.0f;
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int j = 0; j < J; ++j) { x[c][j] *= by; sum += x[c][j]; }
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    // operand word i of the row: codes PAIRS / 2 ... of a word, the lower and the upper half's
#pragma unroll
    for (int i = 0; i < 2 * KSTEPS; ++i) {
      const int c = i / KSTEPS, low = i % KSTEPS / PAIRS * (2 * PAIRS) + i % PAIRS, high = low + PAIRS;
      qb[i / 2][i % 2] = pack2(quarter == low / J ? x[c][low % J] : 0.0f, quarter == high / J ? x[c][high % J] : 0.0f);
    }
    const float coefficient = t < 2 ? -M * sum : sum;
    const bool even = quarter == (2 * t & 3), odd = quarter == (2 * t & 3) + 1;
    const __half upper = __float2half_rn(coefficient);
    const float rest = coefficient - __half2float(upper);
    qz[0] = pack2(even ? __half2float(upper) : 0.0f, odd ? __half2float(upper) : 0.0f);
    qz[1] = pack2(even ? rest : 0.0f, odd ? rest : 0.0f);
    factor = __shfl_sync(0xffffffffu, Base::factor_of(p, up), t < 2 ? 0 : 16);
    m = NOTHING;
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sums[i] = zacc[i] = 0.0f;
#pragma unroll
      for (int u = 0; u < STEPS; ++u) { acc[i][u][0] = 0.0f; acc[i][u][1] = 0.0f; acc[i][u][2] = 0.0f; acc[i][u][3] = 0.0f; }
    }
    f = __float2half2_rn(0x1p15f);
    wide = false;
  }

  // Scores of rows g and g + 8 of 16, times the power of two, head t / 2
  __device__ __forceinline__ void scores(uint32_t kt, int lane, float (&y)[2]) const {
    const int t = lane & 3, g = lane >> 2;
    uint32_t w[2][2][N], pair[4];
    trailers<false, ROW>(kt + CODES, lane, pair);
    Base::keys(kt + g * ROW, t, w[0]);
    Base::keys(kt + (g + 8) * ROW, t, w[1]);
    float c[4], z[4];
    mma(z, pair[0], pair[1], pair[2], pair[3], qz[0], qz[1], 0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) {
      uint32_t x[2][PAIRS];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint32_t word = w[r][i / N][i % N];
        if constexpr (BITS == 4) {
          x[r][0] = times16(word) & 0x00f000f0u;
          x[r][1] = word & 0x00f000f0u;
          x[r][PAIRS - 2] = times16(word >> 8) & 0x00f000f0u;
          x[r][PAIRS - 1] = word >> 8 & 0x00f000f0u;
        } else {
          x[r][0] = word & 0x00ff00ffu;
          x[r][1] = word >> 8 & 0x00ff00ffu;
        }
      }
#pragma unroll
      for (int u = 0; u < PAIRS / 2; ++u) {
        const uint32_t (&b)[2] = qb[i * (PAIRS / 2) + u];
        if (i == 0 && u == 0) mma(c, x[0][0], x[1][0], x[0][1], x[1][1], b[0], b[1], 0.0f, 0.0f, 0.0f, 0.0f);
        else mma(c, x[0][2 * u], x[1][2 * u], x[0][2 * u + 1], x[1][2 * u + 1], b[0], b[1], c[0], c[1], c[2], c[3]);
      }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float2 s = __half22float2(h2(__shfl_sync(0xffffffffu, pair[r], lane & ~2)));
      const float v = fmaf(c[2 * r], s.x, z[2 * r] * UNIT) + fmaf(c[2 * r + 1], s.y, z[2 * r + 1] * UNIT);
      y[r] = v + __shfl_xor_sync(0xffffffffu, v, 1);
    }
  }

  // A scale exceeds 1: the powers of two follow
  __device__ __forceinline__ void rescale(int lane, const uint32_t (&raw)[4]) {
    const __half2 top = __hmax2(h2(raw[0]), h2(raw[2]));
    float most = fmaxf(__low2float(top), __high2float(top));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
    most = __shfl_sync(0xffffffffu, most, lane & 15);                       // (of quarter g & 3)
    const float old = __low2float(f), now = Base::taken(most, old), by = now / old;
    f = __float2half2_rn(now);
    wide = __any_sync(0xffffffffu, now < 1.0f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float r = __shfl_sync(0xffffffffu, by, 4 * i);
#pragma unroll
      for (int u = 0; u < STEPS; ++u) { acc[i][u][0] *= r; acc[i][u][1] *= r; acc[i][u][2] *= r; acc[i][u][3] *= r; }
    }
    // (columns 2 t and 2 t + 1: quarters 2 t & 3 and the next)
    const float r0 = __shfl_sync(0xffffffffu, by, 8 * (lane & 1)), r1 = __shfl_sync(0xffffffffu, by, 8 * (lane & 1) + 4);
    sums[0] *= r0; sums[1] *= r1; sums[2] *= r0; sums[3] *= r1;
  }

  // Weights of 16 rows (upper and lower parts, rows 2 t, 2 t + 1 and those + 8 of column g) times their values
  template <bool FLIP>
  __device__ __forceinline__ void weigh(uint32_t vt, int lane, const uint32_t (&hi)[2], const uint32_t (&lo)[2]) {
    constexpr uint32_t MIDDLE = FLIP ? Base::MIDDLE_FLIPPED : Base::MIDDLE;
    const int t = lane & 3, g = lane >> 2;
    uint32_t raw[4], w[4][N], pb[2], pl[2];
    trailers<true, ROW>(vt + CODES, lane, raw);
#pragma unroll
    for (int r = 0; r < 4; ++r) lds<N>(vt + (2 * t + (r & 1) + 8 * (r >> 1)) * ROW + g * CHUNK, w[r]);
    const uint32_t r0 = __shfl_sync(0xffffffffu, raw[0], lane & 15), r1 = __shfl_sync(0xffffffffu, raw[2], lane & 15);
    __half2 s0 = __hmul2(h2(r0), f), s1 = __hmul2(h2(r1), f);
    if (__any_sync(0xffffffffu, !__hble2(__hmax2(s0, s1), __float2half2_rn(1.0f)))) {
      rescale(lane, raw);
      s0 = __hmul2(h2(r0), f);
      s1 = __hmul2(h2(r1), f);
    }
    Base::template times<FLIP>(hi[0], lo[0], s0, pb[0], pl[0]);
    Base::template times<FLIP>(hi[1], lo[1], s1, pb[1], pl[1]);
    if (wide) {
      Base::template times<FLIP>(hi[0], lo[0], h2(r0), __low2float(f), pb[0], pl[0]);
      Base::template times<FLIP>(hi[1], lo[1], h2(r1), __low2float(f), pb[1], pl[1]);
    }
    mma(sums, MIDDLE, MIDDLE, MIDDLE, MIDDLE, pb[0], pb[1], sums[0], sums[1], sums[2], sums[3]);
    mma(sums, MIDDLE, MIDDLE, MIDDLE, MIDDLE, pl[0], pl[1], sums[0], sums[1], sums[2], sums[3]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t first[J], second[J];
      expand<DIM, BITS, FLIP>(w[0], w[1], i, first);
      expand<DIM, BITS, FLIP>(w[2], w[3], i, second);
#pragma unroll
      for (int u = 0; u < STEPS; ++u) {
        float (&c)[4] = acc[i][u];
        mma(c, first[2 * u], first[2 * u + 1], second[2 * u], second[2 * u + 1], pb[0], pb[1], c[0], c[1], c[2], c[3]);
        mma(c, first[2 * u], first[2 * u + 1], second[2 * u], second[2 * u + 1], pl[0], pl[1], c[0], c[1], c[2], c[3]);
      }
    }
    mma(zacc, raw[0], raw[1], raw[2], raw[3], hi[0], hi[1], zacc[0], zacc[1], zacc[2], zacc[3]);
    mma(zacc, raw[0], raw[1], raw[2], raw[3], lo[0], lo[1], zacc[0], zacc[1], zacc[2], zacc[3]);
  }

  // All there is of the head scaled: its maximum has moved
  __device__ __forceinline__ void scale(float by) {
    l *= by;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sums[i] *= by;
      zacc[i] *= by;
#pragma unroll
      for (int u = 0; u < STEPS; ++u) { acc[i][u][0] *= by; acc[i][u][1] *= by; acc[i][u][2] *= by; acc[i][u][3] *= by; }
    }
  }
  __device__ __forceinline__ void tile(uint32_t kt, int rows, int lane) { take_tile<ROW>(*this, kt, rows, lane); }

  // The state of a part to `state` and `ml`, one head behind the other, or (null) the output of a whole item
  __device__ __forceinline__ void end(const AttendParams &p, int b, int kv_head, float *state, float2 *ml, int lane) {
    const int t = lane & 3, g = lane >> 2, h = t >> 1;
    float total = l;
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    const float by = total == 0.0f ? 0.0f : 1.0f / total;
    const size_t row = static_cast<size_t>(b) * p.q_heads + kv_head * p.group + h;
    const bool live = h < p.group;
    // this lane's columns: quarters 2 t & 3 and the next
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = (2 * t & 3) + e;
      const float z = __shfl_sync(0xffffffffu, zacc[e], 4 * i + 16 + t), inverse = 1.0f / __shfl_sync(0xffffffffu, __low2float(f), 4 * i);
      float v[J];
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const float c = t & 1 ? acc[2 + e][j / 2][e + 2 * (j % 2)] : acc[e][j / 2][e + 2 * (j % 2)];
        v[j] = fmaf(fmaf(c, 1.0f / UNIT, sums[e]), inverse, z);
      }
      if (!live) continue;
      if (state) store_part<DIM>(state + h * DIM + DIM / 4 * i + J * g, v);
      else store_out<T, DIM>(static_cast<T *>(p.out) + row * DIM + DIM / 4 * i + J * g, v, by);
    }
    if (!live || (t & 1) || g) return;
    const float most = total == 0.0f ? -INFINITY : Base::template level_of<T>(p, m, factor, b, kv_head * p.group + h);
    if (state) ml[h] = make_float2(most, total);
    else if (p.lse) p.lse[row] = logf(total) + most * LN2;
  }
};

// Three or four query heads: each takes two of the eight columns, one for each half of the dimensions.  A quarter's products have it in the columns of its half, which
// alone are looked at; two operands of weights times scales, for the even and the odd quarters.
template <typename T, int DIM, int BITS>
struct AttendQuad : Tiles<DIM, BITS, QUAD, 4> {
  using Value = T;
  using Base = Tiles<DIM, BITS, QUAD, 4>;
  using Base::ROW; using Base::CODES; using Base::N; using Base::J; using Base::STEPS; using Base::M; using Base::UNIT; using Base::CHUNK;

  uint32_t qb[2][STEPS][2], qz[2];               // queries of the column's even and odd quarter; sums over quarters, as upper and lower fp16 parts
  float factor, m, l;                            // what a score is multiplied by, the largest score, the sum of weights; of head t
  float acc[4][STEPS][4], sums[2][4], zacc[4];   // out^T, quarter by quarter; what is to be taken off; sums of weights times centres (lanes g >= 4: of quarter g - 4)
  __half2 f;                                     // power of two that takes quarter g & 3's scales of values to 1 or below
  bool wide;                                     // whether one of these is below 1

  __device__ __forceinline__ void begin(const AttendParams &p, const T *queries, long long stride, int lane) {
    const int t = lane & 3, g = lane >> 2, h = g >> 1, half = g & 1;
    const bool live = h < p.group;
    const T *const q = queries + (live ? h : 0) * stride + DIM / 2 * half;
    float x[2][2][J], top = 0.0f;                // of the column's quarters, of the lane's two chunks
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int j = 0; j < J; ++j) {
          x[i][c][j] = live ? static_cast<float>(q[DIM / 4 * i + DIM / 32 * Base::chunk_of(t, c) + j]) : 0.0f;
          top = fmaxf(top, fabsf(x[i][c][j]));
        }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const int up = Base::lift(top);
    const float by = copysignf(power2(up), p.scale_log2);
    float sum[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      sum[i] = 0.0f;
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int j = 0; j < J; ++j) { x[i][c][j] *= by; sum[i] += x[i][c][j]; }
      sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
      sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
#pragma unroll
      for (int u = 0; u < STEPS; ++u) {
        qb[i][u][0] = pack2(x[i][0][2 * u], x[i][1][2 * u]);
        qb[i][u][1] = pack2(x[i][0][2 * u + 1], x[i][1][2 * u + 1]);
      }
    }
    // a trailer's entries 2 t and 2 t + 1: scales (t < 2) or centres of half t & 1
    const float unit = half == (t & 1) ? t < 2 ? -M : 1.0f : 0.0f;
    qz[0] = pack2(unit * sum[0], unit * sum[1]);
    const float2 back = __half22float2(h2(qz[0]));
    qz[1] = pack2(unit * sum[0] - back.x, unit * sum[1] - back.y);
    factor = __shfl_sync(0xffffffffu, Base::factor_of(p, up), 8 * t);
    m = NOTHING;
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sums[0][i] = sums[1][i] = zacc[i] = 0.0f;
#pragma unroll
      for (int u = 0; u < STEPS; ++u) { acc[i][u][0] = 0.0f; acc[i][u][1] = 0.0f; acc[i][u][2] = 0.0f; acc[i][u][3] = 0.0f; }
    }
    f = __float2half2_rn(0x1p15f);
    wide = false;
  }

  // Scores of rows g and g + 8 of 16, times the power of two, head t
  __device__ __forceinline__ void scores(uint32_t kt, int lane, float (&y)[2]) const {
    const int t = lane & 3, g = lane >> 2;
    uint32_t w[2][2][N], pair[4];
    float s[2][4], z[4];
    trailers<false, ROW>(kt + CODES, lane, pair);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint32_t at = kt + (g + 8 * r) * ROW;
      Base::keys(at, t, w[r]);
      uint32_t sw[2];
      lds<2>(at + CODES, sw);
      const float2 s01 = __half22float2(h2(sw[0])), s23 = __half22float2(h2(sw[1]));
      s[r][0] = s01.x; s[r][1] = s01.y; s[r][2] = s23.x; s[r][3] = s23.y;
    }
    mma(z, pair[0], pair[1], pair[2], pair[3], qz[0], qz[1], 0.0f, 0.0f, 0.0f, 0.0f);
    y[0] = (z[0] + z[1]) * UNIT;
    y[1] = (z[2] + z[3]) * UNIT;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t top[J], low[J];
      expand<DIM, BITS>(w[0][0], w[0][1], i, top);
      expand<DIM, BITS>(w[1][0], w[1][1], i, low);
      const uint32_t (&b)[STEPS][2] = qb[i % 2];
      float c[4];
      mma(c, top[0], low[0], top[1], low[1], b[0][0], b[0][1], 0.0f, 0.0f, 0.0f, 0.0f);
      if constexpr (STEPS == 2) mma(c, top[J - 2], low[J - 2], top[J - 1], low[J - 1], b[STEPS - 1][0], b[STEPS - 1][1], c[0], c[1], c[2], c[3]);
      y[0] = fmaf(c[i / 2], s[0][i], y[0]);
      y[1] = fmaf(c[2 + i / 2], s[1][i], y[1]);
    }
  }

  // A scale exceeds 1: the powers of two follow
  __device__ __forceinline__ void rescale(int lane, const uint32_t (&raw)[4]) {
    const __half2 top = __hmax2(h2(raw[0]), h2(raw[2]));
    float most = fmaxf(__low2float(top), __high2float(top));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
    most = __shfl_sync(0xffffffffu, most, lane & 15);                       // (of quarter g & 3)
    const float old = __low2float(f), now = Base::taken(most, old), by = now / old;
    f = __float2half2_rn(now);
    wide = __any_sync(0xffffffffu, now < 1.0f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float r = __shfl_sync(0xffffffffu, by, 4 * i);
      sums[i % 2][i / 2] *= r;
      sums[i % 2][2 + i / 2] *= r;
#pragma unroll
      for (int u = 0; u < STEPS; ++u) { acc[i][u][0] *= r; acc[i][u][1] *= r; acc[i][u][2] *= r; acc[i][u][3] *= r; }
    }
  }

  // Weights of 16 rows (upper and lower parts, rows 2 t, 2 t + 1 and those + 8 of column g) times their values
  template <bool FLIP>
  __device__ __forceinline__ void weigh(uint32_t vt, int lane, const uint32_t (&hi)[2], const uint32_t (&lo)[2]) {
    constexpr uint32_t MIDDLE = FLIP ? Base::MIDDLE_FLIPPED : Base::MIDDLE;
    const int t = lane & 3, g = lane >> 2;
    uint32_t raw[4], w[4][N], pb[2][2], pl[2][2];
    trailers<true, ROW>(vt + CODES, lane, raw);
#pragma unroll
    for (int r = 0; r < 4; ++r) lds<N>(vt + (2 * t + (r & 1) + 8 * (r >> 1)) * ROW + g * CHUNK, w[r]);
    __half2 s0 = __hmul2(h2(raw[0]), f), s1 = __hmul2(h2(raw[2]), f);
    if (__any_sync(0xffffffffu, g < 4 && !__hble2(__hmax2(s0, s1), __float2half2_rn(1.0f)))) {
      rescale(lane, raw);
      s0 = __hmul2(h2(raw[0]), f);
      s1 = __hmul2(h2(raw[2]), f);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {                // quarter 2 (g & 1) + i
      const int from = 8 * (g & 1) + 4 * i + t;
      const __half2 a0 = h2(__shfl_sync(0xffffffffu, bits_of(s0), from)), a1 = h2(__shfl_sync(0xffffffffu, bits_of(s1), from));
      Base::template times<FLIP>(hi[0], lo[0], a0, pb[i][0], pl[i][0]);
      Base::template times<FLIP>(hi[1], lo[1], a1, pb[i][1], pl[i][1]);
    }
    if (wide) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int from = 8 * (g & 1) + 4 * i + t;
        const float power = __shfl_sync(0xffffffffu, __low2float(f), from);
        Base::template times<FLIP>(hi[0], lo[0], h2(__shfl_sync(0xffffffffu, raw[0], from)), power, pb[i][0], pl[i][0]);
        Base::template times<FLIP>(hi[1], lo[1], h2(__shfl_sync(0xffffffffu, raw[2], from)), power, pb[i][1], pl[i][1]);
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float (&c)[4] = sums[i];
      mma(c, MIDDLE, MIDDLE, MIDDLE, MIDDLE, pb[i][0], pb[i][1], c[0], c[1], c[2], c[3]);
      mma(c, MIDDLE, MIDDLE, MIDDLE, MIDDLE, pl[i][0], pl[i][1], c[0], c[1], c[2], c[3]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t first[J], second[J];
      expand<DIM, BITS, FLIP>(w[0], w[1], i, first);
      expand<DIM, BITS, FLIP>(w[2], w[3], i, second);
#pragma unroll
      for (int u = 0; u < STEPS; ++u) {
        float (&c)[4] = acc[i][u];
        mma(c, first[2 * u], first[2 * u + 1], second[2 * u], second[2 * u + 1], pb[i % 2][0], pb[i % 2][1], c[0], c[1], c[2], c[3]);
        mma(c, first[2 * u], first[2 * u + 1], second[2 * u], second[2 * u + 1], pl[i % 2][0], pl[i % 2][1], c[0], c[1], c[2], c[3]);
      }
    }
    mma(zacc, raw[0], raw[1], raw[2], raw[3], hi[0], hi[1], zacc[0], zacc[1], zacc[2], zacc[3]);
    mma(zacc, raw[0], raw[1], raw[2], raw[3], lo[0], lo[1], zacc[0], zacc[1], zacc[2], zacc[3]);
  }

  // All there is of head t scaled: its maximum has moved
  __device__ __forceinline__ void scale(float by) {
    l *= by;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sums[0][i] *= by;
      sums[1][i] *= by;
      zacc[i] *= by;
#pragma unroll
      for (int u = 0; u < STEPS; ++u) { acc[i][u][0] *= by; acc[i][u][1] *= by; acc[i][u][2] *= by; acc[i][u][3] *= by; }
    }
  }
  __device__ __forceinline__ void tile(uint32_t kt, int rows, int lane) { take_tile<ROW>(*this, kt, rows, lane); }

  // The state of a part to `state` and `ml`, one head behind the other, or (null) the output of a whole item
  __device__ __forceinline__ void end(const AttendParams &p, int b, int kv_head, float *state, float2 *ml, int lane) {
    const int t = lane & 3, g = lane >> 2, h = t;
    float total = l;
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    const float by = total == 0.0f ? 0.0f : 1.0f / total;
    const size_t row = static_cast<size_t>(b) * p.q_heads + kv_head * p.group + h;
    const bool live = h < p.group;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float z = __shfl_sync(0xffffffffu, zacc[0], 4 * i + 16 + t), inverse = 1.0f / __shfl_sync(0xffffffffu, __low2float(f), 4 * i);
      float v[J];
#pragma unroll
      for (int j = 0; j < J; ++j)
        v[j] = fmaf(fmaf(acc[i][j / 2][i / 2 + 2 * (j % 2)], 1.0f / UNIT, sums[i % 2][i / 2]), inverse, z);
      if (!live) continue;
      if (state) store_part<DIM>(state + h * DIM + DIM / 4 * i + J * g, v);
      else store_out<T, DIM>(static_cast<T *>(p.out) + row * DIM + DIM / 4 * i + J * g, v, by);
    }
    if (!live || g) return;
    const float most = total == 0.0f ? -INFINITY : Base::template level_of<T>(p, m, factor, b, kv_head * p.group + h);
    if (state) ml[h] = make_float2(most, total);
    else if (p.lse) p.lse[row] = logf(total) + most * LN2;
  }
};

// Up to sixteen query heads, in NT blocks of eight columns.
template <typename T, int DIM, int BITS, int NT>
struct Attend : Tiles<DIM, BITS, NT == 1 ? ONE : TWO, 8 * NT> {
  using Value = T;
  using Base = Tiles<DIM, BITS, NT == 1 ? ONE : TWO, 8 * NT>;
  using Base::ROW; using Base::CODES; using Base::N; using Base::J; using Base::STEPS; using Base::M; using Base::UNIT; using Base::CHUNK;

  uint32_t qb[NT][4][STEPS][2], qz[NT][2];       // queries; sums over quarters, as upper and lower fp16 parts
  float factor[NT][2], m[NT][2], l[NT][2];       // of heads 2 t and 2 t + 1: what a score is multiplied by, the largest score, the sum of weights
  float acc[NT][4][STEPS][4], sums[NT][4][4], zacc[NT][4]; // out^T, quarter by quarter; what is to be taken off; sums of weights times centres (lanes g >= 4: of quarter g - 4)
  __half2 f;                                     // power of two that takes quarter g & 3's scales of values to 1 or below
  bool wide;                                     // whether one of these is below 1

  // An item's queries, `stride` apart (global or shared memory), and nothing seen yet
  __device__ __forceinline__ void begin(const AttendParams &p, const T *queries, long long stride, int lane) {
    const int t = lane & 3, g = lane >> 2;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const bool live = nt * 8 + g < p.group;
      const T *const q = queries + (live ? nt * 8 + g : 0) * stride;
      float x[4][2 * J], top = 0.0f;             // of the lane's two chunks
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int j = 0; j < J; ++j) {
            x[i][c * J + j] = live ? static_cast<float>(q[DIM / 4 * i + DIM / 32 * Base::chunk_of(t, c) + j]) : 0.0f;
            top = fmaxf(top, fabsf(x[i][c * J + j]));
          }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int up = Base::lift(top);
      const float by = copysignf(power2(up), p.scale_log2);
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
          qb[nt][i][u][1] = pack2(x[i][2 * u + 1], x[i][J + 2 * u + 1]);
        }
      }
      // heads 2 t and 2 t + 1: lanes 8 t and 8 t + 4
      const float down = Base::factor_of(p, up);
      factor[nt][0] = __shfl_sync(0xffffffffu, down, 8 * t);
      factor[nt][1] = __shfl_sync(0xffffffffu, down, 8 * t + 4);
      const float by0 = t < 2 ? -M : 1.0f, s0 = by0 * (t & 1 ? sum[2] : sum[0]), s1 = by0 * (t & 1 ? sum[3] : sum[1]);
      const uint32_t upper = pack2(s0, s1);
      const float2 back = __half22float2(h2(upper));
      qz[nt][0] = upper;
      qz[nt][1] = pack2(s0 - back.x, s1 - back.y);
      m[nt][0] = m[nt][1] = NOTHING;
      l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        zacc[nt][i] = 0.0f;
        sums[nt][i][0] = 0.0f; sums[nt][i][1] = 0.0f; sums[nt][i][2] = 0.0f; sums[nt][i][3] = 0.0f;
#pragma unroll
        for (int u = 0; u < STEPS; ++u) { acc[nt][i][u][0] = 0.0f; acc[nt][i][u][1] = 0.0f; acc[nt][i][u][2] = 0.0f; acc[nt][i][u][3] = 0.0f; }
      }
    }
    f = __float2half2_rn(0x1p15f);
    wide = false;
  }

  // Scores of 16 rows, times the power of two: rows g and g + 8, heads 2 t and 2 t + 1
  __device__ __forceinline__ void scores(uint32_t kt, int lane, float (&x)[NT][4]) const {
    const int t = lane & 3, g = lane >> 2;
    uint32_t w[2][2][N], pair[4];                // row, chunk
    float s[2][4];
    trailers<false, ROW>(kt + CODES, lane, pair);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint32_t at = kt + (g + 8 * r) * ROW;
      Base::keys(at, t, w[r]);
      uint32_t sw[2];
      lds<2>(at + CODES, sw);
      const float2 s01 = __half22float2(h2(sw[0])), s23 = __half22float2(h2(sw[1]));
      s[r][0] = s01.x; s[r][1] = s01.y; s[r][2] = s23.x; s[r][3] = s23.y;
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      mma(x[nt], pair[0], pair[1], pair[2], pair[3], qz[nt][0], qz[nt][1], 0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[nt][e] *= UNIT;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t top[J], low[J];
      expand<DIM, BITS>(w[0][0], w[0][1], i, top);
      expand<DIM, BITS>(w[1][0], w[1][1], i, low);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float c[4];
        mma(c, top[0], low[0], top[1], low[1], qb[nt][i][0][0], qb[nt][i][0][1], 0.0f, 0.0f, 0.0f, 0.0f);
        if constexpr (STEPS == 2) mma(c, top[J - 2], low[J - 2], top[J - 1], low[J - 1], qb[nt][i][STEPS - 1][0], qb[nt][i][STEPS - 1][1], c[0], c[1], c[2], c[3]);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[nt][e] = fmaf(c[e], s[e / 2][i], x[nt][e]);
      }
    }
  }

  // A scale exceeds 1: the powers of two follow
  __device__ __forceinline__ void rescale(int lane, const uint32_t (&raw)[4]) {
    const __half2 top = __hmax2(h2(raw[0]), h2(raw[2]));
    float most = fmaxf(__low2float(top), __high2float(top));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
    most = __shfl_sync(0xffffffffu, most, lane & 15);                       // (of quarter g & 3)
    const float old = __low2float(f), now = Base::taken(most, old), by = now / old;
    f = __float2half2_rn(now);
    wide = __any_sync(0xffffffffu, now < 1.0f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float r = __shfl_sync(0xffffffffu, by, 4 * i);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        sums[nt][i][0] *= r; sums[nt][i][1] *= r; sums[nt][i][2] *= r; sums[nt][i][3] *= r;
#pragma unroll
        for (int u = 0; u < STEPS; ++u) { acc[nt][i][u][0] *= r; acc[nt][i][u][1] *= r; acc[nt][i][u][2] *= r; acc[nt][i][u][3] *= r; }
      }
    }
  }

  // Weights of 16 rows (upper and lower parts, rows 2 t, 2 t + 1 and those + 8 of head g) times their values
  template <bool FLIP>
  __device__ __forceinline__ void weigh(uint32_t vt, int lane, const uint32_t (&hi)[NT][2], const uint32_t (&lo)[NT][2]) {
    constexpr uint32_t MIDDLE = FLIP ? Base::MIDDLE_FLIPPED : Base::MIDDLE;
    const int t = lane & 3, g = lane >> 2;
    uint32_t raw[4], w[4][N];
    trailers<true, ROW>(vt + CODES, lane, raw);
#pragma unroll
    for (int r = 0; r < 4; ++r) lds<N>(vt + (2 * t + (r & 1) + 8 * (r >> 1)) * ROW + g * CHUNK, w[r]);
    __half2 s0 = __hmul2(h2(raw[0]), f), s1 = __hmul2(h2(raw[2]), f);
    if (__any_sync(0xffffffffu, g < 4 && !__hble2(__hmax2(s0, s1), __float2half2_rn(1.0f)))) {
      rescale(lane, raw);
      s0 = __hmul2(h2(raw[0]), f);
      s1 = __hmul2(h2(raw[2]), f);
    }
    constexpr int SPAN = NT == 1 ? 4 : 1;        // quarters whose operands are made together, with one look at `wide` (of two blocks of heads one: registers)
#pragma unroll
    for (int first_of = 0; first_of < 4; first_of += SPAN) {
      uint32_t pb[SPAN][NT][2], pl[SPAN][NT][2];
#pragma unroll
      for (int k = 0; k < SPAN; ++k) {
        const int from = 4 * (first_of + k) + t;
        const __half2 a0 = h2(__shfl_sync(0xffffffffu, bits_of(s0), from)), a1 = h2(__shfl_sync(0xffffffffu, bits_of(s1), from));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          Base::template times<FLIP>(hi[nt][0], lo[nt][0], a0, pb[k][nt][0], pl[k][nt][0]);
          Base::template times<FLIP>(hi[nt][1], lo[nt][1], a1, pb[k][nt][1], pl[k][nt][1]);
        }
      }
      if (wide) {
#pragma unroll
        for (int k = 0; k < SPAN; ++k) {
          const int from = 4 * (first_of + k) + t;
          const float power = __shfl_sync(0xffffffffu, __low2float(f), from);
          const __half2 r0 = h2(__shfl_sync(0xffffffffu, raw[0], from)), r1 = h2(__shfl_sync(0xffffffffu, raw[2], from));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            Base::template times<FLIP>(hi[nt][0], lo[nt][0], r0, power, pb[k][nt][0], pl[k][nt][0]);
            Base::template times<FLIP>(hi[nt][1], lo[nt][1], r1, power, pb[k][nt][1], pl[k][nt][1]);
          }
        }
      }
#pragma unroll
      for (int k = 0; k < SPAN; ++k) {
        const int i = first_of + k;
        uint32_t first[J], second[J];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float (&c)[4] = sums[nt][i];
          mma(c, MIDDLE, MIDDLE, MIDDLE, MIDDLE, pb[k][nt][0], pb[k][nt][1], c[0], c[1], c[2], c[3]);
          mma(c, MIDDLE, MIDDLE, MIDDLE, MIDDLE, pl[k][nt][0], pl[k][nt][1], c[0], c[1], c[2], c[3]);
        }
        expand<DIM, BITS, FLIP>(w[0], w[1], i, first);
        expand<DIM, BITS, FLIP>(w[2], w[3], i, second);
#pragma unroll
        for (int u = 0; u < STEPS; ++u)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float (&c)[4] = acc[nt][i][u];
            mma(c, first[2 * u], first[2 * u + 1], second[2 * u], second[2 * u + 1], pb[k][nt][0], pb[k][nt][1], c[0], c[1], c[2], c[3]);
            mma(c, first[2 * u], first[2 * u + 1], second[2 * u], second[2 * u + 1], pl[k][nt][0], pl[k][nt][1], c[0], c[1], c[2], c[3]);
          }
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float (&c)[4] = zacc[nt];
      mma(c, raw[0], raw[1], raw[2], raw[3], hi[nt][0], hi[nt][1], c[0], c[1], c[2], c[3]);
      mma(c, raw[0], raw[1], raw[2], raw[3], lo[nt][0], lo[nt][1], c[0], c[1], c[2], c[3]);
    }
  }

  // A tile, of which `rows` rows are there (32 or more: all)
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
        rises |= (top[nt][e] - m[nt][e]) * factor[nt][e] > SLACK;
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
          const float by = exp2_fast((m[nt][e] - v) * factor[nt][e]);
          m[nt][e] = v;
          l[nt][e] *= by;
          zacc[nt][e] *= by;
          zacc[nt][e + 2] *= by;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            sums[nt][i][e] *= by;
            sums[nt][i][e + 2] *= by;
#pragma unroll
            for (int u = 0; u < STEPS; ++u) { acc[nt][i][u][e] *= by; acc[nt][i][u][e + 2] *= by; }
          }
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
          w[e] = exp2_fast(fmaf(x[h][nt][e] - m[nt][e % 2], factor[nt][e % 2], SHIFT));
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
      if (h == 0) weigh<false>(vt, lane, hi, lo);
      else weigh<true>(vt + 16 * ROW, lane, hi, lo);
    }
  }

  // The state of a part to `state` and `ml`, one head behind the other, or (null) the output of a whole item
  __device__ __forceinline__ void end(const AttendParams &p, int b, int kv_head, float *state, float2 *ml, int lane) {
    const int t = lane & 3, g = lane >> 2;
    float inverse[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) inverse[i] = 1.0f / __shfl_sync(0xffffffffu, __low2float(f), 4 * i);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float total = l[nt][e];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        const int h = nt * 8 + 2 * t + e;
        const float by = total == 0.0f ? 0.0f : 1.0f / total;
        const size_t row = static_cast<size_t>(b) * p.q_heads + kv_head * p.group + h;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float z = __shfl_sync(0xffffffffu, zacc[nt][e], 4 * i + 16 + t);
          float v[J];
#pragma unroll
          for (int j = 0; j < J; ++j)
            v[j] = fmaf(fmaf(acc[nt][i][j / 2][e + 2 * (j % 2)], 1.0f / UNIT, sums[nt][i][e]), inverse[i], z);
          if (h >= p.group) continue;
          if (state) store_part<DIM>(state + h * DIM + DIM / 4 * i + J * g, v);
          else store_out<T, DIM>(static_cast<T *>(p.out) + row * DIM + DIM / 4 * i + J * g, v, by);
        }
        if (h >= p.group || g) continue;
        const float most = total == 0.0f ? -INFINITY : Base::template level_of<T>(p, m[nt][e], factor[nt][e], b, kv_head * p.group + h);
        if (state) ml[h] = make_float2(most, total);
        else if (p.lse) p.lse[row] = logf(total) + most * LN2;
      }
  }
};

template <typename A>
__global__ void __launch_bounds__(WARPS * 32, A::CTAS) attend_tiles(const __grid_constant__ AttendParams p) {
  constexpr int STAGES = A::STAGES;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ Line line;
  __shared__ int sums[MAX_SEQS / 32];
  pdl_wait();
  pdl_trigger();
  make_line(p, line, sums);
  __syncthreads();
  // (a warp's number that the compiler knows to be one for the warp)
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int r = warp * gridDim.x + blockIdx.x, parts = min(p.warps, line.total);          // (few stretches: on as many SMs)
  if (r >= parts) return;
  const int first = begin_of(line.total, parts, r), last = begin_of(line.total, parts, r + 1);
  unsigned char *const own = smem + warp * A::WARP_SMEM;
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(own));
  Place place;
  place.start(p, line, first);
  Item now{place.b, place.head, place.rows - place.tile * TILE}, ahead = now;
  Source source;
  source.at(p, ahead, place.tile, lane);
  int fetched = first, began = first - place.tile, queries_of = -1;         // tiles asked for; the item's first tile; the one whose item's queries wait in shared memory
  uint32_t put = ring, get = ring;
  bool fresh = true;                             // whether the next tile to ask for is the first of its item, or of all
  auto fetch = [&]() {
    if (fetched < last) {
      A::load(p, source, ahead.left, put, lane);
      if (A::QUERIES && fresh && queries_of < 0) {
        A::template load_queries<typename A::Value>(p, ahead, ring + STAGES * A::STAGE, lane);
        queries_of = fetched;
      }
      put = put == ring + (STAGES - 1) * A::STAGE ? ring : put + A::STAGE;
      ahead.left -= TILE;
      fresh = ahead.left <= 0;
      if (fresh && fetched + 1 < last) {
        ahead.next(p, line);
        source.at(p, ahead, 0, lane);
      } else {
        source.next(p);
      }
    }
    ++fetched;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) fetch();
  A a;
  bool begins = true;                            // whether tile i is the first of its item, or of all
  for (int i = first; i < last; ++i) {
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    __syncwarp();                                // every lane's copies of tile i are there, and tile i - 1 has been read
    if (begins) {
      const typename A::Value *q = static_cast<const typename A::Value *>(p.q) + now.b * p.q_seq + static_cast<long long>(now.head) * p.group * p.q_head;
      long long stride = p.q_head;
      if (A::QUERIES && queries_of == i) {
        q = reinterpret_cast<const typename A::Value *>(own + STAGES * A::STAGE);
        stride = A::QUERY_STRIDE;
      }
      a.begin(p, q, stride, lane);
      __syncwarp();                              // (read by all lanes before the next are copied)
      if (queries_of == i) queries_of = -1;
      begins = false;
    }
    fetch();
    a.tile(get, now.left, lane);
    get = get == ring + (STAGES - 1) * A::STAGE ? ring : get + A::STAGE;
    now.left -= TILE;
    if (now.left <= 0 || i == last - 1) {
      const size_t slot = static_cast<size_t>(2 * r + (began > first)) * p.group;
      const bool whole = now.left <= 0 && began >= first;
      a.end(p, now.b, now.head, whole ? nullptr : p.part_out + slot * A::HEAD_DIM, whole ? nullptr : p.part_ml + slot, lane);
      if (i == last - 1) break;
      now.next(p, line);
      began = i + 1;
      begins = true;
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// (a maximum of -inf: nothing seen, or a sum that is no number and stays one)
__device__ __forceinline__ float part_weight(float m, float l, float top) { return m == -INFINITY ? (l == 0.0f ? 0.0f : 1.0f) : exp2f(m - top); }
// Zeros for a sequence's query heads [first, first + n), which see no row
template <typename T>
__device__ __forceinline__ void zero_heads(const AttendParams &p, int dim, int b, int first, int n, int lane) {
  const size_t row = static_cast<size_t>(b) * p.q_heads + first;
  for (int i = lane; i < n * (dim / 8); i += 32) *reinterpret_cast<uint4 *>(static_cast<T *>(p.out) + row * dim + i * 8) = make_uint4(0, 0, 0, 0);
  for (int i = lane; p.lse && i < n; i += 32) p.lse[row + i] = -INFINITY;
}
// Short items, one launch: a cluster of CTAs takes an item, each warp an equal part of its tiles; the states stay in shared memory, where all of the cluster
// can read them, and its warps join them.  Long items, few: `splits` clusters each have an equal part of one (as many as it has tiles, if that is fewer).
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address of `at` in the shared memory of the cluster's CTA `rank`
__device__ __forceinline__ uint32_t of_rank(uint32_t at, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(at), "r"(rank));
  return r;
}
template <int E> __device__ __forceinline__ void ld_cluster(uint32_t at, float (&v)[E]) {
  if constexpr (E == 4) asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(at) : "memory");
  else asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v[0]), "=f"(v[1]) : "r"(at) : "memory");
}
// A cluster's parts: a warp each of 2^shift CTAs, part w warp w >> shift of CTA w & 2^shift - 1 (few tiles: in different CTAs), its first tile.  (A cluster has at most 2^19 / 8.)
__device__ __forceinline__ int begin_of_part(int tiles, int shift, int w) { return tiles * w >> (shift + 2); }
static_assert(WARPS == 4, "a CTA has four of a cluster's parts");
// The states of a cluster's parts, at most 32, joined by warps `mine` and so on; `part`: where the joined state goes, -1 for the output of a whole item.  Unit: DIM /
// GROUPS dimensions of a query head; groups of lanes take every GROUPS-th part, eight or four at a time.
template <typename A, int GROUPS>
__device__ __forceinline__ void join_cluster(const AttendParams &p, const Place &item, int part, int shift, unsigned char *smem, int mine, int lane) {
  using T = typename A::Value;
  constexpr int DIM = A::HEAD_DIM, UNIT_DIMS = DIM / GROUPS, LANES = 32 / GROUPS, E = UNIT_DIMS / LANES, EACH = GROUPS == 1 ? 8 : 4;      // dimensions of a lane
  const int parts = WARPS << shift, group = lane / LANES;
  const uint32_t base = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
  auto part_at = [&](int w) { return of_rank(base + (w >> shift) * A::WARP_SMEM, w & ((1 << shift) - 1)); };
  const bool there = lane < parts && begin_of_part(item.tiles, shift, lane) < begin_of_part(item.tiles, shift, lane + 1);
  const unsigned int any = __ballot_sync(0xffffffffu, there);
  for (int u = mine; u < p.group * GROUPS; u += parts) {
    const int h = u / GROUPS, d = u % GROUPS * UNIT_DIMS + lane % LANES * E;
    float ml[2] = {-INFINITY, 0.0f}, out[E];                                // a part's maximum and sum to a lane
    if (there) ld_cluster<2>(part_at(lane) + p.group * DIM * 4 + h * 8, ml);
    float top = 0.0f, f = 0.0f, total = 0.0f;
#pragma unroll
    for (int k = 0; k < E; ++k) out[k] = 0.0f;
    for (int first = 0; first < parts; first += EACH * GROUPS) {
      float v[EACH][E];
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const int w = first + group + GROUPS * i;
#pragma unroll
        for (int k = 0; k < E; ++k) v[i][k] = 0.0f;
        if (any >> w & 1u) ld_cluster<E>(part_at(w) + (h * DIM + d) * 4, v[i]);
      }
      if (first == 0) {                          // (beside the states)
        top = ml[0];
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        f = part_weight(ml[0], ml[1], top);
        total = ml[1] * f;
#pragma unroll
        for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
      }
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const float by = __shfl_sync(0xffffffffu, f, first + group + GROUPS * i);
#pragma unroll
        for (int k = 0; k < E; ++k) out[k] = fmaf(v[i][k], by, out[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < E; ++k)
#pragma unroll
      for (int o = LANES; o < 32; o <<= 1) out[k] += __shfl_xor_sync(0xffffffffu, out[k], o);
    if (part >= 0) {
      const size_t at = 2ull * part * p.group + h;
      if (lane < LANES) store_part<32 * E>(p.part_out + at * DIM + d, out);
      if (lane == 0 && u % GROUPS == 0) p.part_ml[at] = make_float2(top, total);
      continue;
    }
    const size_t row = static_cast<size_t>(item.b) * p.q_heads + item.head * p.group + h;
    if (lane < LANES) store_out<T, 32 * E>(static_cast<T *>(p.out) + row * DIM + d, out, total == 0.0f ? 0.0f : 1.0f / total);
    if (lane == 0 && u % GROUPS == 0 && p.lse) p.lse[row] = total == 0.0f ? -INFINITY : top * LN2 + logf(total);
  }
}
template <typename A>
__global__ void __launch_bounds__(WARPS * 32, A::CTAS) attend_items(const __grid_constant__ AttendParams p) {
  using T = typename A::Value;
  constexpr int STAGES = A::STAGES, DIM = A::HEAD_DIM;
  extern __shared__ __align__(128) unsigned char smem[];
  pdl_wait();
  pdl_trigger();
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31, rank = cluster_rank();
  const int shift = p.ranks - 1, cluster = static_cast<int>(blockIdx.x) >> shift, item = cluster / p.splits, split = cluster - item * p.splits;
  Place now;
  now.b = item / p.caches.kv_heads;
  now.head = item - now.b * p.caches.kv_heads;
  now.rows = seen_rows(p, now.b);
  now.tiles = tiles_of(now.rows);
  if (now.tiles == 0) {                          // (all of the cluster)
    if (split == 0 && rank == 0 && warp == 0) zero_heads<T>(p, DIM, now.b, now.head * p.group, p.group, lane);
    return;
  }
  const int splits = min(p.splits, now.tiles), begin = begin_of(now.tiles, splits, split);
  if (split >= splits) return;                   // (all of the cluster)
  now.tiles = begin_of(now.tiles, splits, split + 1) - begin;               // the cluster's
  const int mine = (warp << shift) + rank, first = begin + begin_of_part(now.tiles, shift, mine), last = begin + begin_of_part(now.tiles, shift, mine + 1);
  unsigned char *const own = smem + warp * A::WARP_SMEM;
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(own));
  if (first < last) {
    Source source;
    source.at(p, Item{now.b, now.head, 0}, first, lane);
    int fetched = first;
    uint32_t put = ring, get = ring;
    auto fetch = [&]() {
      if (fetched < last) {
        A::load(p, source, now.rows - fetched * TILE, put, lane);
        put = put == ring + (STAGES - 1) * A::STAGE ? ring : put + A::STAGE;
        source.next(p);
      }
      ++fetched;
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) fetch();
    A a;
    a.begin(p, static_cast<const T *>(p.q) + now.b * p.q_seq + static_cast<long long>(now.head) * p.group * p.q_head, p.q_head, lane);
    for (int i = first; i < last; ++i) {
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
      __syncwarp();                              // every lane's copies of tile i are there, and tile i - 1 has been read
      fetch();
      a.tile(get, now.rows - i * TILE, lane);
      get = get == ring + (STAGES - 1) * A::STAGE ? ring : get + A::STAGE;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncwarp();
    float *const state = reinterpret_cast<float *>(own);
    a.end(p, now.b, now.head, state, reinterpret_cast<float2 *>(state + p.group * DIM), lane);
  }
  cluster_sync();
  const int part = splits > 1 ? cluster : -1;    // (one: the whole item)
  // whole heads where there are few parts, or heads enough for the warps; else eighths.  (One CTA, two heads: 128 rows 5.6 us, with eighths 8.7; four CTAs, eight heads:
  // 12.8 and 13.0; eight CTAs, two heads, 1024 rows: 10.8 and 7.2.)
  if (shift < 2 || 2 * p.group >= (WARPS << shift)) join_cluster<A, 1>(p, now, part, shift, smem, mine, lane);
  else join_cluster<A, 8>(p, now, part, shift, smem, mine, lane);
  cluster_sync();                                // (nobody leaves while its states are read)
}

// The join: outputs of items whose parts lie in several stretches, and of sequences without rows.
template <int DIM, int AHEAD>
struct Joined {
  static constexpr int E = DIM / 32;
  float M, L, A[E];                              // dimensions lane * E ... of the warp's parts
  // parts of stretches r0 + from, r0 + from + step, ... up to r1, AHEAD at a time; `inside`: the first is not the first item of its stretch
  __device__ __forceinline__ void take(const AttendParams &p, int r0, int r1, int from, int step, bool inside, int head, int lane) {
    M = -INFINITY;
    L = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) A[i] = 0.0f;
    for (int first = r0 + from; first <= r1; first += step * AHEAD) {
      float v[AHEAD][E];
      float2 ml[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int r = first + i * step;
        ml[i] = make_float2(-INFINITY, 0.0f);
#pragma unroll
        for (int k = 0; k < E; ++k) v[i][k] = 0.0f;
        if (r <= r1) {
          const size_t at = static_cast<size_t>(2 * r + (r == r0 && inside)) * p.group + head;
          ml[i] = p.part_ml[at];
          const float *const src = p.part_out + at * DIM + lane * E;
          if constexpr (E == 4) { const float4 a = *reinterpret_cast<const float4 *>(src); v[i][0] = a.x; v[i][1] = a.y; v[i][E - 2] = a.z; v[i][E - 1] = a.w; }
          else { const float2 a = *reinterpret_cast<const float2 *>(src); v[i][0] = a.x; v[i][1] = a.y; }
        }
      }
      float top = M;
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) top = fmaxf(top, ml[i].x);
      const float f0 = part_weight(M, L, top);
      M = top;
      L *= f0;
#pragma unroll
      for (int k = 0; k < E; ++k) A[k] *= f0;
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const float f = part_weight(ml[i].x, ml[i].y, top);
        L = fmaf(ml[i].y, f, L);
#pragma unroll
        for (int k = 0; k < E; ++k) A[k] = fmaf(v[i][k], f, A[k]);
      }
    }
  }
};
template <typename T>
__device__ __forceinline__ void zero_empty(const AttendParams &p, const Line &line, int dim, int first, int step, int lane) {
  for (int b = first; b < p.caches.seqs; b += step)
    if (line.rows[b] == 0) zero_heads<T>(p, dim, b, 0, p.q_heads, lane);
}
// A warp takes a query head of an item: for items of few parts.
constexpr int FEW = 4;                           // parts asked for together
template <typename T, int DIM>
__global__ void __launch_bounds__(256) join_few(const __grid_constant__ AttendParams p) {
  __shared__ Line line;
  __shared__ int sums[MAX_SEQS / 32];
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31, w = static_cast<int>(blockIdx.x) * 8 + warp, warps = static_cast<int>(gridDim.x) * 8;
  // (the lengths were there before the kernel that this one follows)
  make_line(p, line, sums);
  __syncthreads();
  const int parts = min(p.warps, line.total);
  zero_empty<T>(p, line, DIM, w, warps, lane);
  // unit: a stretch that begins inside an item, as the first to do so, and a query head
  for (int u = w; u < (parts - 1) * p.group; u += warps) {
    const int r = u / p.group + 1, head = u - (r - 1) * p.group, t = begin_of(line.total, parts, r), before = begin_of(line.total, parts, r - 1);
    Place at;
    at.start(p, line, t);
    const int t0 = t - at.tile;
    if (at.tile == 0 || before > t0) continue;
    const int r1 = part_of(line.total, parts, t0 + at.tiles - 1);
    const size_t row = static_cast<size_t>(at.b) * p.q_heads + at.head * p.group + head;
    pdl_wait();                                  // (all the above passes under the other kernel's end)
    Joined<DIM, FEW> j;
    j.take(p, r - 1, r1, 0, 1, before < t0, head, lane);
    store_out<T, DIM>(static_cast<T *>(p.out) + row * DIM + lane * (DIM / 32), j.A, j.L == 0.0f ? 0.0f : 1.0f / j.L);
    if (lane == 0 && p.lse) p.lse[row] = j.L == 0.0f ? -INFINITY : j.M * LN2 + logf(j.L);
  }
  pdl_wait();
}
// A CTA takes a query head of an item, its W warps every W-th part: for items of many.
template <typename T, int DIM, int W, int AHEAD>
__global__ void __launch_bounds__(32 * W) join_many(const __grid_constant__ AttendParams p) {
  constexpr int E = DIM / 32;
  __shared__ Line line;
  __shared__ int sums[MAX_SEQS / 32];
  __shared__ float sm[W], sl[W];
  __shared__ __align__(16) float sa[W][DIM];
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31, row = blockIdx.x, b = row / p.q_heads, head = row - b * p.q_heads;
  int r0, r1;
  bool inside = false;
  if (p.ranks > 0) {                             // (clusters' parts)
    const int item = b * p.caches.kv_heads + head / p.group, splits = min(p.splits, tiles_of(seen_rows(p, b)));
    r0 = item * p.splits;
    r1 = r0 + max(splits, 1) - 1;
  } else {
    make_line(p, line, sums);
    __syncthreads();
    const int parts = min(p.warps, line.total), tiles = tiles_of(line.rows[b]);
    if (tiles == 0) {
      pdl_wait();
      if (head == 0 && warp == 0) zero_empty<T>(p, line, DIM, b, MAX_SEQS, lane);
      return;
    }
    const int t0 = line.before[b] + head / p.group * tiles;
    r0 = part_of(line.total, parts, t0), r1 = part_of(line.total, parts, t0 + tiles - 1);
    inside = begin_of(line.total, parts, r0) < t0;
  }
  pdl_wait();
  if (r0 == r1) return;                          // (written there)
  Joined<DIM, AHEAD> j;
  j.take(p, r0, r1, warp, W, inside, head % p.group, lane);
  if (lane == 0) { sm[warp] = j.M; sl[warp] = j.L; }
#pragma unroll
  for (int i = 0; i < E; ++i) sa[warp][lane * E + i] = j.A[i];
  __syncthreads();
  if (threadIdx.x >= DIM) return;
  float top = -INFINITY, total = 0.0f, sum = 0.0f;
#pragma unroll
  for (int i = 0; i < W; ++i) top = fmaxf(top, sm[i]);
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const float f = part_weight(sm[i], sl[i], top);
    total = fmaf(sl[i], f, total);
    sum = fmaf(sa[i][threadIdx.x], f, sum);
  }
  static_cast<T *>(p.out)[static_cast<size_t>(row) * DIM + threadIdx.x] = static_cast<T>(total == 0.0f ? 0.0f : sum / total);
  if (p.lse && threadIdx.x == 0) p.lse[row] = total == 0.0f ? -INFINITY : top * LN2 + logf(total);
}

}  // namespace qmk_packed
#endif  // QMK_PACKED_ATTENTION_CUH_
