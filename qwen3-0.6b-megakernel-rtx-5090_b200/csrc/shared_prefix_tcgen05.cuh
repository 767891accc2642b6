// The products of the shared prefix on tcgen05 (see shared_prefix_attention.cuh): 128 query rows against a range of prefix rows.
//
// One CTA per (128 rows of queries, kv head, range).  The rows are the query heads of a kv head, sequence by sequence, brought by one tiled
// copy of the queries; keys and values come in tiles of 128 rows.  Barriers, descriptors and roles are those of the prefill's attention
// (attention_tcgen05.cuh): even and odd tiles belong to two chains with four softmax warps (a query row per thread), a score buffer, a P tile and
// an output accumulator each (all of TMEM), so that one chain's round trip - scores read, P stored, P . V - runs beside the other's
// arithmetic; the loads of keys and values, the score products and P . V have an issuing thread each.  Here all queries see all rows, so there is no mask but for the
// prefix's end, and a CTA leaves a partial state (unnormalised output, maximum, sum) instead of the result.  A tile's time is
// the round trip's latency (1800 cycles for a tile of 64 rows).  16,384 rows of 128 dims against 256 query rows of eight kv heads, caches cold: tiles
// of 64 rows 27.6 us, of 128 rows 28.0, of 128 rows with the chains taking turns at the exponentials 26.3, 0.65 PFLOP/s.
// (17 GFLOP at the rate of a large product are 10 us, and so are 67 MB from HBM.)  What bounds it: every product of 128 x 128 x 16 reads 8 KB of operands from shared
// memory, and an SM has 16 exponentials a cycle, 1024 cycles a tile.  Two tiles of query rows a CTA, which read keys half as often, took 33.
//
// The running maximum is raised when it grew by more than 2^3; weights are stored times 2^P_SHIFT (fp16: 2^12, so at most 2^15), which keeps ten
// more bits of the small ones than storing them as they are.
// Waits are bounded.  On a time-out the CTA sets *status = 4 and leaves NaN as the state of its rows, so that the result is NaN.
#ifndef QMK_SHARED_PREFIX_TCGEN05_CUH_
#define QMK_SHARED_PREFIX_TCGEN05_CUH_

#include <cuda.h>

#include "attention_tcgen05.cuh"
#include "shared_prefix_attention.cuh"

namespace qmk_spa {

constexpr int TC_THREADS = qmk_attn::THREADS;
constexpr int TC_ROWS = 128;                                       // prefix rows per tile
constexpr uint32_t BOX_BYTES = 64 * 128, BLOCK_BYTES = 128 * 128;  // [64 rows x 64 dims], [128 rows x 64 dims or keys], swizzled
constexpr float RAISE = 3.0f;                                      // log2
template <int D> constexpr uint32_t tc_tile_bytes() { return (D / 64) * BLOCK_BYTES; }          // of queries, keys, values
template <int D> constexpr size_t tc_smem_bytes() { return 5 * tc_tile_bytes<D>() + 4 * BLOCK_BYTES + 256; }
static_assert(tc_smem_bytes<128>() <= 232448, "shared memory of a CTA");

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *map, int c0, int c1, int c2, int c3, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
               ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar) : "memory");
}

// map_q: {dims, heads of a kv head, kv heads, sequences}, boxes of {64, group, 1, seqs_per_tile}; map_k / map_v: {dims, prefix rows, kv heads}, boxes of
// {64, 64, 1}; 128-byte swizzle, zeros outside.  TEST: the self test's score issuer that stops behind its second tile.
template <typename T, int D, bool TEST = false>
__global__ void __launch_bounds__(TC_THREADS, 1)
prefix_parts_tc(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                const __grid_constant__ Params p, int seqs_per_tile, unsigned int *status, unsigned long long budget_ns) {
  using namespace qmk_gemm;
  using qmk_attn::tma_load_3d;
  using qmk_attn::fast_exp2;
  using qmk_attn::smem_desc_mn_sw128;
  constexpr int HALVES = D / 64, CHAINS = 2;
  constexpr uint32_t OFF_K = tc_tile_bytes<D>(), OFF_V = OFF_K + 2 * tc_tile_bytes<D>(), OFF_P = OFF_V + 2 * tc_tile_bytes<D>(), OFF_BARS = OFF_P + 4 * BLOCK_BYTES;
  constexpr uint32_t FORMAT = Half<T>::BF16 ? (1u << 7) | (1u << 10) : 0u;         // of A and B
  constexpr uint32_t IDESC_S = qmk_attn::IDESC_S2 | FORMAT;        // 128 x 128
  constexpr uint32_t IDESC_PV = (1u << 4) | (1u << 16) | (static_cast<uint32_t>(D >> 3) << 17) | (static_cast<uint32_t>(128 >> 4) << 24) | FORMAT;
  extern __shared__ __align__(1024) unsigned char tc_smem[];
  const uint32_t base = qmk_gemm::s32(tc_smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int id = static_cast<int>(blockIdx.x), kv = id % p.kv_heads, tile = id / p.kv_heads % p.row_tiles, part = id / (p.kv_heads * p.row_tiles);
  const int first = part * p.prefix_range, nrows = min(p.prefix_range, p.prefix_len - first), ntiles = (nrows + TC_ROWS - 1) / TC_ROWS;
  const uint32_t bars = base + OFF_BARS;
  // of chain c
  auto k_full = [&](int c) { return bars + 8u * c; };
  auto k_empty = [&](int c) { return bars + 8u * (2 + c); };
  auto v_full = [&](int c) { return bars + 8u * (4 + c); };
  auto v_empty = [&](int c) { return bars + 8u * (6 + c); };
  auto s_full = [&](int c) { return bars + 8u * (8 + c); };
  auto s_free = [&](int c) { return bars + 8u * (10 + c); };
  auto p_ready = [&](int c) { return bars + 8u * (12 + c); };
  auto pv_done = [&](int c) { return bars + 8u * (14 + c); };
  auto turn = [&](int c) { return bars + 8u * (19 + c); };         // the other chain is through with its exponentials
  const uint32_t q_full = bars + 8u * 16, s_stopped = bars + 8u * 17, pv_stopped = bars + 8u * 18;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(tc_smem + OFF_BARS + 8 * 21);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

  if ((base & 1023u) != 0u) {              // the swizzled tiles need a 1024-byte aligned window: NaN instead of garbage
    const int r = tile * p.group * seqs_per_tile + static_cast<int>(threadIdx.x);
    if (static_cast<int>(threadIdx.x) < p.group * seqs_per_tile && r < p.seqs * p.group)
      p.part_ml[(static_cast<size_t>(part) * p.seqs + r / p.group) * p.q_heads + kv * p.group + r % p.group] = make_float2(NAN, NAN);
    return;
  }
  if (threadIdx.x == 0) {
    for (int c = 0; c < CHAINS; ++c) {
      bar_init(k_full(c), 1); bar_init(k_empty(c), 1); bar_init(v_full(c), 1); bar_init(v_empty(c), 1);
      bar_init(s_full(c), 1); bar_init(s_free(c), 4); bar_init(p_ready(c), 4); bar_init(pv_done(c), 1); bar_init(turn(c), 4);
    }
    bar_init(q_full, 1);
    bar_init(s_stopped, 1);
    bar_init(pv_stopped, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(qmk_gemm::s32(tmem_slot)), "r"(qmk_attn::TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  qmk_gemm::pdl_wait();
  if (warp == 0) __syncwarp();
  auto load_tile = [&](bool is_v, int j) {
    const int c = j & 1;
    const uint32_t full = is_v ? v_full(c) : k_full(c), to = base + (is_v ? OFF_V : OFF_K) + c * tc_tile_bytes<D>();
    const CUtensorMap *const map = is_v ? &map_v : &map_k;
    bar_expect_tx(full, tc_tile_bytes<D>());
#pragma unroll
    for (int h = 0; h < HALVES; ++h)
#pragma unroll
      for (int r = 0; r < 2; ++r) tma_load_3d(to + h * BLOCK_BYTES + r * BOX_BYTES, map, 64 * h, first + j * TC_ROWS + 64 * r, kv, full);
  };
  const int k_prefilled = ntiles < 2 ? ntiles : 2;
  if (warp == 0 && elect_one()) {          // (rows of the tile that the box does not cover hold what was there: they stay in their own rows)
    bar_expect_tx(q_full, static_cast<uint32_t>(HALVES) * 128u * static_cast<uint32_t>(p.group * seqs_per_tile));
#pragma unroll
    for (int h = 0; h < HALVES; ++h) tma_load_4d(base + h * BLOCK_BYTES, &map_q, 64 * h, 0, kv, tile * seqs_per_tile, q_full);
    for (int j = 0; j < k_prefilled; ++j) load_tile(false, j);
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  qmk_gemm::pdl_trigger();
  const uint32_t tmem_base = *tmem_slot, tmem_o0 = tmem_base + 256u;

  if (warp == 0 || warp == 3 + 4 * CHAINS) {
    if (elect_one()) {                     // ---- producers: the K ring (warp 0) and the V ring
      const bool is_v = warp != 0;
      int issued = is_v ? 0 : k_prefilled;
      for (int j = issued; j < ntiles; ++j) {
        if (j >= 2 && !bar_wait(is_v ? v_empty(j & 1) : k_empty(j & 1), ((j >> 1) - 1) & 1, abort_flag, status, budget_ns)) break;
        if (*abort_flag) break;
        load_tile(is_v, j);
        issued = j + 1;
      }
      if (*abort_flag)
        for (int j = (issued > 2 ? issued - 2 : 0); j < issued; ++j) bar_drain(is_v ? v_full(j & 1) : k_full(j & 1), (j >> 1) & 1, budget_ns);
    }
  } else if (warp == 1) {
    if (elect_one()) {                     // ---- scores
      for (int j = 0; j < ntiles; ++j) {
        const int c = j & 1, n = j >> 1;
        bool ok = (j > 0 || bar_wait(q_full, 0, abort_flag, status, budget_ns)) && bar_wait(k_full(c), n & 1, abort_flag, status, budget_ns) &&
                  (n == 0 || bar_wait(s_free(c), (n - 1) & 1, abort_flag, status, budget_ns));
        if (TEST && j == 2) ok = bar_wait(s_stopped, 0, abort_flag, status, budget_ns);      // (nothing arrives)
        if (!ok) {                         // the products issued end, and so do the copies that the loader may have asked for
          bar_drain(q_full, 0, budget_ns);
          mma_commit(s_stopped);
          bar_drain(s_stopped, 0, budget_ns);
          for (int i = j; i < ntiles && i < j + 2; ++i) bar_drain(k_full(i & 1), (i >> 1) & 1, budget_ns);
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
          const uint64_t da = smem_desc_sw128(base + h * BLOCK_BYTES), db = smem_desc_sw128(base + OFF_K + c * tc_tile_bytes<D>() + h * BLOCK_BYTES);
#pragma unroll
          for (int k = 0; k < 4; ++k) mma_f16_ss(tmem_base + 128u * c, da + 2u * k, db + 2u * k, (h > 0 || k > 0) ? 1u : 0u, IDESC_S);
        }
        mma_commit(s_full(c));
        mma_commit(k_empty(c));
      }
    }
  } else if (warp == 2 + 4 * CHAINS) {
    if (elect_one()) {                     // ---- P . V
      for (int j = 0; j < ntiles; ++j) {
        const int c = j & 1, n = j >> 1;
        if (!bar_wait(v_full(c), n & 1, abort_flag, status, budget_ns) || !bar_wait(p_ready(c), n & 1, abort_flag, status, budget_ns)) {
          mma_commit(pv_stopped);
          bar_drain(pv_stopped, 0, budget_ns);
          for (int i = j; i < ntiles && i < j + 2; ++i) bar_drain(v_full(i & 1), (i >> 1) & 1, budget_ns);
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t vt = base + OFF_V + c * tc_tile_bytes<D>(), to = tmem_o0 + 128u * c;
#pragma unroll
        for (int h = 0; h < 2; ++h) {      // 64 keys of P each
          const uint64_t dp = smem_desc_sw128(base + OFF_P + (2 * c + h) * BLOCK_BYTES);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_f16_ss(to, dp + 2u * k, smem_desc_mn_sw128(vt + (4 * h + k) * 16 * 128, BLOCK_BYTES), (n > 0 || h > 0 || k > 0) ? 1u : 0u, IDESC_PV);
        }
        mma_commit(pv_done(c));
        mma_commit(v_empty(c));
      }
    }
  } else {                                 // ---- softmax: chain = warp group, thread = query row = TMEM lane
    const int chain = (warp - 2) >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tmem_o = tmem_o0 + 128u * static_cast<uint32_t>(chain), p_tile = base + OFF_P + static_cast<uint32_t>(chain) * 2 * BLOCK_BYTES;
    const uint32_t tmem_s = tmem_base + 128u * static_cast<uint32_t>(chain) + lane_base;
    const bool negative = p.scale_log2 < 0.0f;
    const float sc = fabsf(p.scale_log2);
    float m_used = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = chain; j < ntiles && ok; j += CHAINS) {
      const int n = j >> 1;
      ok = __all_sync(0xffffffffu, bar_wait(s_full(chain), n & 1, abort_flag, status, budget_ns));
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      uint32_t s[4][32];
#pragma unroll
      for (int b = 0; b < 4; ++b) QMK_TMEM_LD32(s[b], tmem_s + 32u * b);
      asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");     // the scores are in registers: the next product may overwrite them
      __syncwarp();
      if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(s_free(chain)) : "memory");
      if (negative) {
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
          for (int c = 0; c < 32; ++c) s[b][c] ^= 0x80000000u;
      }
      const int left = nrows - j * TC_ROWS;      // rows of this tile that are there (one at least)
      if (left < TC_ROWS) {
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (32 * b + c >= left) s[b][c] = __float_as_uint(-INFINITY);
      }
      float mx4[4];
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        mx4[b] = __uint_as_float(s[b][0]);
#pragma unroll
        for (int c = 1; c < 32; ++c) mx4[b] = fmaxf(mx4[b], __uint_as_float(s[b][c]));
      }
      const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * sc;
      const bool raise = mx > m_used + RAISE;                        // always from -inf, but for scores of -inf
      const float m_new = raise ? mx : m_used, alpha = raise ? exp2f(m_used - m_new) : 1.0f;
      if (n > 0) {
        ok = __all_sync(0xffffffffu, bar_wait(pv_done(chain), (n - 1) & 1, abort_flag, status, budget_ns));
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (__any_sync(0xffffffffu, raise)) {
#pragma unroll 1
          for (int c = 0; c < D / 8; ++c) {      // (eight columns at a time: the scores have the registers)
            uint32_t o[8];
            asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                         : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3]), "=r"(o[4]), "=r"(o[5]), "=r"(o[6]), "=r"(o[7])
                         : "r"(tmem_o + lane_base + static_cast<uint32_t>(c * 8)) : "memory");
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                         ::"r"(tmem_o + lane_base + static_cast<uint32_t>(c * 8)), "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]), "r"(o[4]), "r"(o[5]), "r"(o[6]), "r"(o[7])
                         : "memory");
          }
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        }
      }
      l *= alpha;
      m_used = m_new;
      // The chains take turns at the exponentials, so that one's products run under the other's: side by side in step, both wait for products
      // and then share the units.
      if (chain == 1 || n > 0) {
        ok = __all_sync(0xffffffffu, bar_wait(turn(chain), (chain == 1 ? n : n - 1) & 1, abort_flag, status, budget_ns));
        if (!ok) break;
      }
      const float sub = Half<T>::P_SHIFT - (m_used == -INFINITY ? 0.f : m_used);
      const uint32_t prow = p_tile + static_cast<uint32_t>(row) * 128u, x = static_cast<uint32_t>(row & 7);
      float sum4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int seg = 0; seg < 16; ++seg) {
        uint32_t packed[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int c = seg * 8 + 2 * i;
          const float a = fast_exp2(fmaf(__uint_as_float(s[c >> 5][c & 31]), sc, sub)), b = fast_exp2(fmaf(__uint_as_float(s[c >> 5][(c & 31) + 1]), sc, sub));
          sum4[i] += a + b;
          packed[i] = Half<T>::pack(a, b);
        }
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(prow + (seg >> 3) * BLOCK_BYTES + ((static_cast<uint32_t>(seg & 7) ^ x) << 4)), "r"(packed[0]),
                     "r"(packed[1]), "r"(packed[2]), "r"(packed[3]) : "memory");
      }
      if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(turn(chain ^ 1)) : "memory");
      l += (sum4[0] + sum4[1]) + (sum4[2] + sum4[3]);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(p_ready(chain)) : "memory");
    }
    const int my_tiles = (ntiles - chain + 1) / CHAINS;
    if (ok && my_tiles > 0) ok = __all_sync(0xffffffffu, bar_wait(pv_done(chain), (my_tiles - 1) & 1, abort_flag, status, budget_ns));
    if (!ok) bar_drain(pv_done(chain), (my_tiles - 1) & 1, budget_ns);
    // ---- the two chains' states, joined per row; (maximum, sum) go through the chain's own P tile
    asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(p_tile + static_cast<uint32_t>(row) * 8u), "f"(m_used), "f"(l) : "memory");
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    asm volatile("bar.sync 1, %0;" ::"n"(128 * CHAINS) : "memory");
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    float m_other, l_other;
    asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(m_other), "=f"(l_other)
                 : "r"(base + OFF_P + static_cast<uint32_t>(chain ^ 1) * 2 * BLOCK_BYTES + static_cast<uint32_t>(row) * 8u) : "memory");
    const bool good = ok && !*abort_flag, two = ntiles > 1;
    const float m_a = chain == 0 ? m_used : m_other, l_a = chain == 0 ? l : l_other, m_b = chain == 0 ? m_other : m_used, l_b = chain == 0 ? l_other : l;
    const float m_all = two ? fmaxf(m_a, m_b) : m_a;
    const float fa = m_a == -INFINITY ? 0.f : exp2f(m_a - m_all), fb = !two || m_b == -INFINITY ? 0.f : exp2f(m_b - m_all);
    const int rows = p.group * seqs_per_tile, r = tile * rows + row;
    const bool live = row < rows && r < p.seqs * p.group;
    const size_t at = (static_cast<size_t>(part) * p.seqs + (live ? r / p.group : 0)) * p.q_heads + kv * p.group + (live ? r % p.group : 0);
    float *const dst = p.part_out + at * D + (D / 2) * chain;
    if (live && chain == 0) p.part_ml[at] = good ? make_float2(m_all, l_a * fa + (two ? l_b * fb : 0.f)) : make_float2(NAN, NAN);
    if (good) {
#pragma unroll 1
      for (int c = 0; c < D / 64; ++c) {
        const uint32_t col = static_cast<uint32_t>((D / 2) * chain + 32 * c);
        uint32_t oa[32], ob[32];
        QMK_TMEM_LD32(oa, tmem_o0 + lane_base + col);
        if (two) QMK_TMEM_LD32(ob, tmem_o0 + 128u + lane_base + col);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        if (live) {
#pragma unroll
          for (int i = 0; i < 32; i += 8) {      // (32 bytes at a time: whole sectors)
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              v[k] = __uint_as_float(oa[i + k]) * fa;
              if (two) v[k] = fmaf(__uint_as_float(ob[i + k]), fb, v[k]);
            }
            asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst + 32 * c + i), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]),
                         "f"(v[5]), "f"(v[6]), "f"(v[7]) : "memory");
          }
        }
      }
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(qmk_attn::TMEM_COLS) : "memory");
  }
}

}  // namespace qmk_spa
#endif  // QMK_SHARED_PREFIX_TCGEN05_CUH_
