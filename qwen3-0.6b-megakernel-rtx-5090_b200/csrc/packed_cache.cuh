// Caches kept in 4 or 8 bits: the format of a row, rows quantised as they are written, rows read back.
//
// A packed row (what a kv head keeps of a position, DIM = 64 or 128 values) is DIM * BITS / 8 bytes of codes and a trailer of 16 bytes: four fp16 scales
// s and four fp16 centres z, one pair for each quarter b of the dimensions.  With M = 2^(BITS - 1) a code n stands for z + s (n - M);
//   s = fp16((hi - lo) / (2^BITS - 1)),  z = fp16(lo + M s),  n = the whole number nearest to (x - z) / s (ties to even) + M, taken into [0, 2^BITS - 1],
// lo and hi the quarter's least and largest value.  A centre instead of the least value, because the attention multiplies rounded weights by z and
// by s (n - M) apart: both are of the values' own size then, and their errors too.  A quarter with a value that is no number, infinite or
// above 65504 has s = z = NaN, so what it was written from does not read back as something else.
//
// Order of the codes: dimension DIM/4 b + DIM/32 g + j (b < 4, g < 8, j < DIM/32) lies at index DIM/8 g + DIM/32 b + j, 4-bit codes in the low half of
// a byte first.  One of eight lanes that share a row has its DIM/8 codes together then, DIM/32 of each quarter, and in the attention's products a
// lane's codes of one scale are those of one operand tile.
#ifndef QMK_PACKED_CACHE_CUH_
#define QMK_PACKED_CACHE_CUH_

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace qmk_packed {

constexpr int MAX_SEQS = 128;
constexpr int THREADS = 256;
constexpr int TRAILER = 16;
template <int DIM, int BITS> constexpr int ROW_BYTES = DIM * BITS / 8 + TRAILER;

// Caches of all sequences: strides in bytes, rows of a head `row` apart.
struct Caches {
  int seqs, kv_heads, rows;
  long long head, row;
  const unsigned char *k[MAX_SEQS], *v[MAX_SEQS];
};
struct RowParams {
  Caches caches;
  void *k, *v;                                   // the rows: strides in elements
  long long seq, head, row;
  int rows;                                      // of a sequence, in the call
  const int *starts, *lens;                      // may be null: all `start`, all `rows`
  int start;
};

template <typename T> struct Type;
template <> struct Type<__half> {
  static constexpr bool BF16 = false;
  using Two = __half2;
  static __device__ __forceinline__ float2 floats(Two x) { return __half22float2(x); }
  // (a scale that was rounded up may lead a code past the largest fp16 number: that one then, and not infinity)
  static __device__ __forceinline__ uint32_t two(float a, float b) {
    uint32_t r;
    asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
  }
};
template <> struct Type<__nv_bfloat16> {
  static constexpr bool BF16 = true;
  using Two = __nv_bfloat162;
  static __device__ __forceinline__ float2 floats(Two x) { return __bfloat1622float2(x); }
  static __device__ __forceinline__ uint32_t two(float a, float b) {
    const Two r = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&r);
  }
};
template <typename V> __device__ __forceinline__ uint32_t bits_of(V x) { return *reinterpret_cast<const uint32_t *>(&x); }
template <typename V> __device__ __forceinline__ V from_bits(uint32_t x) { return *reinterpret_cast<const V *>(&x); }

// Eight lanes share a row; lane g of them has the codes of dimensions DIM/4 b + DIM/32 g + j.  A row of the call: (sequence, head, row), rows first, so that
// the four rows of a warp lie together in the cache.
struct RowOfCall {
  int b, head, t, at;                            // at: row of the cache
  bool there;
};
__device__ __forceinline__ RowOfCall row_of(const RowParams &p, unsigned int i) {
  RowOfCall r;
  const unsigned int pair = i / static_cast<unsigned int>(p.rows);
  r.t = static_cast<int>(i - pair * p.rows);
  r.b = static_cast<int>(pair / static_cast<unsigned int>(p.caches.kv_heads));
  r.head = static_cast<int>(pair - r.b * static_cast<unsigned int>(p.caches.kv_heads));
  const long long at = static_cast<long long>(p.starts ? p.starts[r.b] : p.start) + r.t;
  r.there = r.t < (p.lens ? p.lens[r.b] : p.rows) && at >= 0 && at < p.caches.rows;
  r.at = static_cast<int>(at);
  return r;
}

// The code of x.  The quotient in fp32 is off by 2^-20 (4 bits; 8: 2^-16) at most; where that may cross a border the exact one decides: difference and
// product of fp16 numbers are exact in 64 bits, and a quotient of them is not within 2^-53 of a border that it is not on.
template <int BITS>
__device__ __forceinline__ uint32_t code_of(float x, float z, float s, float inverse) {
  constexpr float M = 1 << (BITS - 1), NEAR = BITS == 4 ? 0x1p-18f : 0x1p-14f;
  const float t = (x - z) * inverse;
  float n = rintf(t);
  if (fabsf(t - n) > 0.5f - NEAR) n = static_cast<float>(rint((static_cast<double>(x) - static_cast<double>(z)) / static_cast<double>(s)));
  return static_cast<uint32_t>(fminf(fmaxf(n + M, 0.0f), 2.0f * M - 1.0f));
}

// One row of values (at `src`, this lane's DIM/8) to a packed one.
template <typename T, int DIM, int BITS>
__device__ __forceinline__ void pack_row(const uint32_t (&x)[4][DIM / 64], unsigned char *dst, int g, bool there) {
  using Two = typename Type<T>::Two;
  constexpr int W = DIM / 64, CODES = DIM / 8;   // 32-bit words of values in a quarter; codes of the lane
  constexpr float M = 1 << (BITS - 1), LEVELS = (1 << BITS) - 1;
  // least and largest value of the quarters, two in a register, over the eight lanes
  Two lo[2], hi[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    Two l[2], h[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      l[b] = h[b] = from_bits<Two>(x[2 * i + b][0]);
      if (W == 2) { l[b] = __hmin2_nan(l[b], from_bits<Two>(x[2 * i + b][W - 1])); h[b] = __hmax2_nan(h[b], from_bits<Two>(x[2 * i + b][W - 1])); }
    }
    lo[i] = __hmin2_nan(from_bits<Two>(__byte_perm(bits_of(l[0]), bits_of(l[1]), 0x5410)), from_bits<Two>(__byte_perm(bits_of(l[0]), bits_of(l[1]), 0x7632)));
    hi[i] = __hmax2_nan(from_bits<Two>(__byte_perm(bits_of(h[0]), bits_of(h[1]), 0x5410)), from_bits<Two>(__byte_perm(bits_of(h[0]), bits_of(h[1]), 0x7632)));
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
      lo[i] = __hmin2_nan(lo[i], from_bits<Two>(__shfl_xor_sync(0xffffffffu, bits_of(lo[i]), o)));
      hi[i] = __hmax2_nan(hi[i], from_bits<Two>(__shfl_xor_sync(0xffffffffu, bits_of(hi[i]), o)));
    }
  }
  uint32_t words[CODES * BITS / 32];
  uint32_t mine = 0;                             // this lane's 16 bits of the trailer
#pragma unroll
  for (int i = 0; i < CODES * BITS / 32; ++i) words[i] = 0;
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const float2 l2 = Type<T>::floats(lo[b / 2]), h2 = Type<T>::floats(hi[b / 2]);
    const float low = b % 2 ? l2.y : l2.x, high = b % 2 ? h2.y : h2.x;
    const bool good = low >= -65504.0f && high <= 65504.0f;
    const __half sh = good ? __float2half_rn((high - low) / LEVELS) : __ushort_as_half(0x7fff);
    const float s = __half2float(sh);
    const __half zh = good ? __float2half_rn(fmaf(M, s, low)) : __ushort_as_half(0x7fff);
    const float z = __half2float(zh), inverse = s > 0.0f ? 1.0f / s : 0.0f;
    if (g == b) mine = __half_as_ushort(sh);
    if (g == 4 + b) mine = __half_as_ushort(zh);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float2 v = Type<T>::floats(from_bits<Two>(x[b][w]));
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int index = 2 * W * b + 2 * w + j;
        const uint32_t n = inverse > 0.0f ? code_of<BITS>(j ? v.y : v.x, z, s, inverse) : 1u << (BITS - 1);
        words[index * BITS / 32] |= n << (index * BITS % 32);
      }
    }
  }
  if (!there) return;
  unsigned char *const to = dst + g * (CODES * BITS / 8);
  if constexpr (CODES * BITS == 128) *reinterpret_cast<uint4 *>(to) = make_uint4(words[0], words[1], words[2], words[3]);
  else if constexpr (CODES * BITS == 64) *reinterpret_cast<uint2 *>(to) = make_uint2(words[0], words[1]);
  else *reinterpret_cast<uint32_t *>(to) = words[0];
  *reinterpret_cast<unsigned short *>(dst + DIM * BITS / 8 + 2 * g) = static_cast<unsigned short>(mine);
}

// This lane's words of a row of values: two or four at a time of each quarter
template <int DIM>
__device__ __forceinline__ void load_values(const void *src, int g, bool there, uint32_t (&x)[4][DIM / 64]) {
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const char *const at = static_cast<const char *>(src) + (DIM / 4 * b + DIM / 32 * g) * 2;
    if constexpr (DIM == 128) {
      const uint2 w = there ? __ldg(reinterpret_cast<const uint2 *>(at)) : make_uint2(0, 0);
      x[b][0] = w.x;
      x[b][DIM / 64 - 1] = w.y;
    } else {
      x[b][0] = there ? __ldg(reinterpret_cast<const uint32_t *>(at)) : 0u;
    }
  }
}

template <typename T, int DIM, int BITS>
__global__ void __launch_bounds__(THREADS) write_rows(const __grid_constant__ RowParams p, unsigned int count) {
  const int g = threadIdx.x & 7;
  for (unsigned int first = blockIdx.x * (THREADS / 8); first < count; first += gridDim.x * (THREADS / 8)) {
    const unsigned int i = first + (threadIdx.x >> 3);
    const RowOfCall r = row_of(p, i < count ? i : count - 1);
    const bool there = r.there && i < count;
    const long long from = r.b * p.seq + r.head * p.head + r.t * p.row, to = r.head * p.caches.head + r.at * p.caches.row;
    uint32_t k[4][DIM / 64], v[4][DIM / 64];
    load_values<DIM>(static_cast<const T *>(p.k) + from, g, there, k);
    load_values<DIM>(static_cast<const T *>(p.v) + from, g, there, v);
    pack_row<T, DIM, BITS>(k, const_cast<unsigned char *>(p.caches.k[r.b]) + to, g, there);
    pack_row<T, DIM, BITS>(v, const_cast<unsigned char *>(p.caches.v[r.b]) + to, g, there);
  }
}

// This lane's codes of a packed row, as words
template <int DIM, int BITS>
__device__ __forceinline__ void load_codes(const unsigned char *row, int g, bool there, uint32_t (&words)[DIM * BITS / 256]) {
  constexpr int N = DIM * BITS / 256;
  const unsigned char *const at = row + g * (4 * N);
  if constexpr (N == 4) {
    const uint4 w = there ? __ldg(reinterpret_cast<const uint4 *>(at)) : make_uint4(0, 0, 0, 0);
    words[0] = w.x; words[1] = w.y; words[2] = w.z; words[3] = w.w;
  } else if constexpr (N == 2) {
    const uint2 w = there ? __ldg(reinterpret_cast<const uint2 *>(at)) : make_uint2(0, 0);
    words[0] = w.x; words[1] = w.y;
  } else {
    words[0] = there ? __ldg(reinterpret_cast<const uint32_t *>(at)) : 0u;
  }
}
// The value of dimension DIM/4 b + DIM/32 g + j from the lane's words and the trailer
template <int DIM, int BITS>
__device__ __forceinline__ float value_of(const uint32_t (&words)[DIM * BITS / 256], const __half (&pairs)[8], int b, int j) {
  const int at = (DIM / 32 * b + j) * BITS;
  const float n = static_cast<float>(words[at / 32] >> (at % 32) & ((1u << BITS) - 1)) - (1 << (BITS - 1));
  return fmaf(__half2float(pairs[b]), n, __half2float(pairs[4 + b]));
}
template <typename T, int DIM, int BITS>
__device__ __forceinline__ void unpack_row(const unsigned char *row, T *dst, int g, bool there) {
  constexpr int N = DIM * BITS / 256;
  uint32_t words[N];
  load_codes<DIM, BITS>(row, g, there, words);
  const uint4 trailer = there ? __ldg(reinterpret_cast<const uint4 *>(row + DIM * BITS / 8)) : make_uint4(0, 0, 0, 0);
  __half pairs[8];
  *reinterpret_cast<uint4 *>(pairs) = trailer;
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    T *const to = dst + DIM / 4 * b + DIM / 32 * g;
    const uint32_t first = Type<T>::two(value_of<DIM, BITS>(words, pairs, b, 0), value_of<DIM, BITS>(words, pairs, b, 1));
    if constexpr (DIM == 128) {
      const uint32_t second = Type<T>::two(value_of<DIM, BITS>(words, pairs, b, 2), value_of<DIM, BITS>(words, pairs, b, 3));
      *reinterpret_cast<uint2 *>(to) = make_uint2(first, second);
    } else {
      *reinterpret_cast<uint32_t *>(to) = first;
    }
  }
}
template <typename T, int DIM, int BITS>
__global__ void __launch_bounds__(THREADS) read_rows(const __grid_constant__ RowParams p, unsigned int count) {
  const int g = threadIdx.x & 7;
  for (unsigned int first = blockIdx.x * (THREADS / 8); first < count; first += gridDim.x * (THREADS / 8)) {
    const unsigned int i = first + (threadIdx.x >> 3);
    if (i >= count) break;
    const RowOfCall r = row_of(p, i);
    const long long to = r.b * p.seq + r.head * p.head + r.t * p.row, from = r.there ? r.head * p.caches.head + r.at * p.caches.row : 0;
    unpack_row<T, DIM, BITS>(p.caches.k[r.b] + from, static_cast<T *>(p.k) + to, g, r.there);
    unpack_row<T, DIM, BITS>(p.caches.v[r.b] + from, static_cast<T *>(p.v) + to, g, r.there);
  }
}

}  // namespace qmk_packed
#endif  // QMK_PACKED_CACHE_CUH_
