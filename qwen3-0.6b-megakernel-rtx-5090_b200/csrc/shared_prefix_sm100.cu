// C entry of the attention over a shared prefix (shared_prefix_attention.cuh).
#include "../../include/qwen_megakernel.h"

#include <algorithm>
#include <string>

#include "engine_internal.h"
#include "prefill_sm100.h"
#include "shared_prefix_attention.cuh"
#include "shared_prefix_tcgen05.cuh"

namespace {

using namespace qmk_spa;

constexpr int MAX_ROWS = 1 << 24;                // of a prefix or an own cache

int refuse(const std::string &why) {
  qmk_internal::note_error("qmk_attention_shared_prefix: " + why);
  return QMK_ERR_BAD_ARGUMENT;
}

// What is wrong with sizes; null: nothing
const char *refused_heads(int q_heads, int kv_heads, int head_dim) {
  if (head_dim != 64 && head_dim != 128) return "head_dim must be 64 or 128";
  if (kv_heads < 1 || q_heads < 1 || q_heads % kv_heads || q_heads / kv_heads > MAX_GROUP || q_heads > 1024) return "q_heads must be 1 to 16 times kv_heads, and at most 1024";
  return nullptr;
}
const char *refused_lengths(int prefix_len, int own_rows) {
  return prefix_len < 0 || own_rows < 0 || prefix_len > MAX_ROWS || own_rows > MAX_ROWS ? "a length is negative or above 2^24" : nullptr;
}

// How a call is cut into items.  More than 32 rows of queries against a kv head and 96 M products (rows x prefix rows x kv heads x dims) go through
// tcgen05, 128 rows at a time.  mma.sync against tcgen05, us a call in a graph, the prefix in L2, eight kv heads of 128 dims: 32 query rows each 9.0 and 9.9 with 1000
// prefix rows, 20.4 and 20.2 with 16,384; 40 rows 30.3 and 20.8 with 16,384; 64 rows 9.2 and 10.0 with 200, 15.5 and 14.7 with 4096; 128 rows 16.8 and 16.2 with 1000,
// 52.4 and 24.6 with 16,384.  Four kv heads of 64 dims: 64 rows 8.1 and 9.8 with 4096, 13.4 and 12.5 with 16,384.
struct Split {
  bool tc;
  int row_warps, row_tiles, seqs_per_tile, prefix_parts, prefix_range, own_parts, own_range;
};
constexpr int SMS = 148;
constexpr long long TC_PRODUCTS = 96 << 20;
Split split_of(int seqs, int q_heads, int kv_heads, int head_dim, int prefix_len, int own_rows, bool tc) {
  Split s;
  const int group = q_heads / kv_heads, rows = seqs * group, tiles = (prefix_len + KEYS - 1) / KEYS;
  s.tc = tc && rows > 32 && 1ll * rows * kv_heads * head_dim * prefix_len >= TC_PRODUCTS;
  s.row_warps = rows <= 16 ? 1 : 2;
  s.seqs_per_tile = std::min(128 / group, seqs);
  s.row_tiles = s.tc ? (seqs + s.seqs_per_tile - 1) / s.seqs_per_tile : (rows + 16 * s.row_warps - 1) / (16 * s.row_warps);
  const int items = s.row_tiles * kv_heads, parts = std::max(1, (s.tc ? SMS : 2 * SMS) / items);
  s.prefix_range = std::max(2, ((tiles + parts - 1) / parts + 1) / 2 * 2) * KEYS;      // (whole tiles of prefix_parts_tc)
  s.prefix_parts = (prefix_len + s.prefix_range - 1) / s.prefix_range;
  s.own_range = std::max(OWN_RANGE, (own_rows / OWN_PARTS + 64) / 64 * 64);
  s.own_parts = (own_rows + s.own_range - 1) / s.own_range;
  return s;
}
long long workspace_bytes(const Split &s, int seqs, int q_heads, int head_dim) {
  return 16 + static_cast<long long>(s.prefix_parts + s.own_parts) * seqs * q_heads * (head_dim * 4ll + 8);
}

// Maps of the queries and of the prefix for prefix_parts_tc; false where the strides are none that a map can have.
bool make_maps(CUtensorMap *maps, const Params &p, const Split &s, int head_dim, bool bf16) {
  const unsigned long long dim = head_dim, q_dims[4] = {dim, static_cast<unsigned long long>(p.group), static_cast<unsigned long long>(p.kv_heads), static_cast<unsigned long long>(p.seqs)};
  const unsigned long long q_strides[3] = {2ull * p.q_head, 2ull * p.q_head * p.group, 2ull * p.q_seq};
  const unsigned int q_box[4] = {64, static_cast<unsigned int>(p.group), 1, static_cast<unsigned int>(s.seqs_per_tile)};
  const unsigned long long kv_dims[3] = {dim, static_cast<unsigned long long>(p.prefix_len), static_cast<unsigned long long>(p.kv_heads)};
  const unsigned long long kv_strides[2] = {2ull * p.prefix_row, 2ull * p.prefix_head};
  const unsigned int kv_box[3] = {64, KEYS, 1};
  return qmk_tc::make_map_tiled(maps, bf16, 4, p.q, q_dims, q_strides, q_box) && qmk_tc::make_map_tiled(maps + 1, bf16, 3, p.k_prefix, kv_dims, kv_strides, kv_box) &&
         qmk_tc::make_map_tiled(maps + 2, bf16, 3, p.v_prefix, kv_dims, kv_strides, kv_box);
}

// The waits of prefix_parts_tc, and whether a kernel of the call may start early behind the one before it.
struct Waits {
  unsigned int *status;
  unsigned long long budget_ns;
  bool overlap;
};
template <typename T, int D, int NT>
cudaError_t launch(Params &p, const Split &s, const CUtensorMap *maps, const Waits &waits, cudaStream_t stream) {
  using Own = OwnRows<T, D, NT, own_warps(D)>;
  using Beside = OwnRows<T, D, NT, WARPS>;
  constexpr int own_smem = OWN_STAGES * 2 * Own::TILE, beside_smem = OWN_STAGES * 2 * Beside::TILE, smem = STAGES * 2 * KEYS * D * 2;
  static_assert(own_smem >= Own::STATE_BYTES && beside_smem >= Beside::STATE_BYTES && smem >= WARPS * 16 * (D + 4) * 4 + WARPS * 16 * 8 && smem >= beside_smem,
                "the warps' states fit the rings");
  void (*const kernel)(Params) = s.row_warps == 1 ? attend_parts<T, D, 1, NT> : attend_parts<T, D, 2, NT>;
  cudaError_t e;
  const int prefix_items = s.prefix_parts * s.row_tiles * p.kv_heads, own_items = s.own_parts * p.kv_heads * p.seqs;
  bool dependent = qmk_tc::pdl_active();
  if (s.tc) {
    p.prefix_items = 0;
    e = cudaFuncSetAttribute(prefix_parts_tc<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(tc_smem_bytes<D>()));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(own_parts<T, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, own_smem);
    if (e == cudaSuccess)
      e = qmk_tc::launch_kernel(prefix_parts_tc<T, D>, dim3(prefix_items), dim3(TC_THREADS), tc_smem_bytes<D>(), stream, maps[0], maps[1], maps[2], p,
                                s.seqs_per_tile, waits.status, waits.budget_ns);
    dependent = waits.overlap;                   // (of the launch before, inside this call)
    const qmk_tc::PdlScope scope(dependent);
    if (e == cudaSuccess && own_items > 0) e = qmk_tc::launch_kernel(own_parts<T, D, NT>, dim3(own_items), dim3(32 * own_warps(D)), own_smem, stream, p);
    if (e != cudaSuccess) return e;
  } else if (prefix_items + own_items > 0) {
    p.prefix_items = prefix_items;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess) e = qmk_tc::launch_kernel(kernel, dim3(prefix_items + own_items), dim3(THREADS), prefix_items > 0 ? smem : beside_smem, stream, p);
    if (e != cudaSuccess) return e;
    dependent = waits.overlap;
  }
  const qmk_tc::PdlScope scope(dependent);
  return qmk_tc::launch_kernel(join_parts<T, D>, dim3(p.seqs * p.q_heads), dim3(128), 0, stream, p);
}
template <typename T>
cudaError_t launch(Params &p, const Split &s, int head_dim, const CUtensorMap *maps, const Waits &waits, cudaStream_t stream) {
  if (p.group > 8) return head_dim == 64 ? launch<T, 64, 2>(p, s, maps, waits, stream) : launch<T, 128, 2>(p, s, maps, waits, stream);
  return head_dim == 64 ? launch<T, 64, 1>(p, s, maps, waits, stream) : launch<T, 128, 1>(p, s, maps, waits, stream);
}

}  // namespace

extern "C" long long qmk_attention_shared_prefix_workspace(int num_sequences, int q_heads, int kv_heads, int head_dim, int prefix_len,
                                                           int own_rows) {
  if (num_sequences < 1 || num_sequences > MAX_SEQS || refused_heads(q_heads, kv_heads, head_dim) || refused_lengths(prefix_len, own_rows)) return 0;
  return std::max(workspace_bytes(split_of(num_sequences, q_heads, kv_heads, head_dim, prefix_len, own_rows, true), num_sequences, q_heads, head_dim),
                  workspace_bytes(split_of(num_sequences, q_heads, kv_heads, head_dim, prefix_len, own_rows, false), num_sequences, q_heads, head_dim));
}

extern "C" int qmk_attention_shared_prefix(const qmk_shared_prefix_args *a, cudaStream_t stream) {
  qmk_internal::begin_call();
  if (!a) return refuse("null pointer argument");
  if (a->num_sequences < 1 || a->num_sequences > MAX_SEQS) return refuse("num_sequences must be in [1, 128]");
  if (a->type < 0 || a->type > 1) return refuse("the type is fp16 (0) or bf16 (1)");
  if (const char *why = refused_heads(a->q_heads, a->kv_heads, a->head_dim)) return refuse(why);
  if (const char *why = refused_lengths(a->prefix_len, a->own_rows)) return refuse(why);
  if (!a->q || !a->out || (a->prefix_len > 0 && (!a->k_prefix || !a->v_prefix)) || (a->own_rows > 0 && (a->k_own ? !a->v_own : !a->k_own_base || !a->v_own_base)) || (a->own_rows > 0 && !a->own_lens))
    return refuse("null pointer argument");
  if (!(a->scale > -2.0e38f && a->scale < 2.0e38f)) return refuse("the scale must be finite, and below 2e38");   // (times log2 e too)
  if (a->timeout_ms < 0) return refuse("timeout_ms is negative");
  auto aligned = [](const void *ptr) { return (reinterpret_cast<unsigned long long>(ptr) & 15u) == 0; };
  bool ok = aligned(a->q) && aligned(a->k_prefix) && aligned(a->v_prefix) && aligned(a->out) && (reinterpret_cast<unsigned long long>(a->workspace) & 31u) == 0;
  Params p;
  for (int b = 0; a->own_rows > 0 && b < a->num_sequences; ++b) {
    const long long at = 2 * b * a->own_seq_stride;
    p.k_own[b] = a->k_own ? a->k_own[b] : static_cast<const char *>(a->k_own_base) + at;
    p.v_own[b] = a->k_own ? a->v_own[b] : static_cast<const char *>(a->v_own_base) + at;
    if (!p.k_own[b] || !p.v_own[b]) return refuse("null pointer argument");
    ok = ok && aligned(p.k_own[b]) && aligned(p.v_own[b]);
  }
  if (!ok) return refuse("pointers must be 16-byte aligned, the workspace 32");
  auto odd = [](long long stride, int size) { return size > 1 && stride % 8; };
  if (odd(a->q_seq_stride, a->num_sequences) || odd(a->q_head_stride, a->q_heads) || odd(a->prefix_row_stride, a->prefix_len) || odd(a->prefix_head_stride, a->kv_heads) ||
      odd(a->own_row_stride, a->own_rows) || odd(a->own_head_stride, a->kv_heads))
    return refuse("strides must be multiples of 8 elements");
  if (!a->workspace || a->workspace_bytes < qmk_attention_shared_prefix_workspace(a->num_sequences, a->q_heads, a->kv_heads, a->head_dim, a->prefix_len, a->own_rows))
    return refuse("workspace too small");
  p.q = a->q;
  p.q_seq = a->q_seq_stride;
  p.q_head = a->q_head_stride;
  p.seqs = a->num_sequences;
  p.group = a->q_heads / a->kv_heads;
  p.q_heads = a->q_heads;
  p.kv_heads = a->kv_heads;
  p.k_prefix = a->k_prefix;
  p.v_prefix = a->v_prefix;
  p.prefix_row = a->prefix_row_stride;
  p.prefix_head = a->prefix_head_stride;
  p.prefix_len = a->prefix_len;
  p.own_row = a->own_row_stride;
  p.own_head = a->own_head_stride;
  p.own_rows = a->own_rows;
  p.own_lens = a->own_lens;
  p.own_bias = a->own_lens_add;
  p.scale_log2 = a->scale * LOG2E;
  // (a scale of 0 would turn the masked scores of a last tile, -inf, into NaN there)
  Split s = split_of(p.seqs, p.q_heads, p.kv_heads, a->head_dim, p.prefix_len, p.own_rows, p.scale_log2 != 0.0f);
  CUtensorMap maps[3];
  if (s.tc && !make_maps(maps, p, s, a->head_dim, a->type == 1)) s = split_of(p.seqs, p.q_heads, p.kv_heads, a->head_dim, p.prefix_len, p.own_rows, false);
  p.prefix_parts = s.prefix_parts;
  p.prefix_range = s.prefix_range;
  p.row_tiles = s.row_tiles;
  p.own_parts = s.own_parts;
  p.own_range = s.own_range;
  const long long states = static_cast<long long>(s.prefix_parts + s.own_parts) * p.seqs * p.q_heads;
  p.part_out = static_cast<float *>(a->workspace);
  p.part_ml = reinterpret_cast<float2 *>(p.part_out + states * a->head_dim);
  const Waits waits = {a->status ? a->status : reinterpret_cast<unsigned int *>(p.part_ml + states),      // (in the workspace: for nobody)
                       (a->timeout_ms ? a->timeout_ms : 2000) * 1000000ull, a->no_overlap == 0};
  p.out = a->out;
  p.lse = a->lse;
  const cudaError_t e = a->type == 0 ? launch<__half>(p, s, a->head_dim, maps, waits, stream) : launch<__nv_bfloat16>(p, s, a->head_dim, maps, waits, stream);
  if (e != cudaSuccess) {
    cudaGetLastError();
    qmk_internal::note_error(std::string("qmk_attention_shared_prefix: ") + cudaGetErrorString(e));
    return QMK_ERR_CUDA;
  }
  return QMK_OK;
}

extern "C" int qmk_selftest_shared_prefix_wait_timeout(int budget_us) {
  qmk_internal::begin_call();
  if (budget_us < 1 || budget_us > 1000000) return refuse("budget_us must be in [1, 1e6]");
  // 64 sequences of two heads on each of two kv heads (a tile of 128 query rows), 1024 prefix rows in one range
  constexpr int SEQS = 64, GROUP = 2, KV = 2, HEADS = GROUP * KV, D = 128, ROWS = 1024, STATES = SEQS * HEADS;
  constexpr size_t q_bytes = 2ull * STATES * D, kv_bytes = 2ull * KV * ROWS * D, at_k = q_bytes, at_v = at_k + kv_bytes, at_out = at_v + kv_bytes,
                   at_lse = at_out + q_bytes, at_parts = at_lse + 4ull * STATES, at_ml = at_parts + 4ull * STATES * D, at_status = at_ml + 8ull * STATES,
                   total = at_status + 16;
  unsigned char *buf = nullptr;
  cudaError_t e = cudaMalloc(&buf, total);
  if (e == cudaSuccess) e = cudaMemset(buf, 0, total);
  Params p = {};
  p.q = buf;
  p.q_seq = HEADS * D;
  p.q_head = D;
  p.seqs = SEQS;
  p.group = GROUP;
  p.q_heads = HEADS;
  p.kv_heads = KV;
  p.k_prefix = buf + at_k;
  p.v_prefix = buf + at_v;
  p.prefix_row = D;
  p.prefix_head = ROWS * D;
  p.prefix_len = p.prefix_range = ROWS;
  p.prefix_parts = p.row_tiles = 1;
  p.scale_log2 = 1.0f;
  p.part_out = reinterpret_cast<float *>(buf + at_parts);
  p.part_ml = reinterpret_cast<float2 *>(buf + at_ml);
  p.out = buf + at_out;
  p.lse = reinterpret_cast<float *>(buf + at_lse);
  unsigned int *const status = reinterpret_cast<unsigned int *>(buf + at_status);
  Split s = {};
  s.seqs_per_tile = SEQS;
  CUtensorMap maps[3];
  unsigned int word = 0;
  float lse[STATES];
  __half out[STATES];                       // one dimension of every row
  if (e == cudaSuccess && !make_maps(maps, p, s, D, false)) e = cudaErrorInvalidValue;
  auto *const kernel = prefix_parts_tc<__half, D, true>;
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(tc_smem_bytes<D>()));
  if (e == cudaSuccess) {
    kernel<<<KV, TC_THREADS, tc_smem_bytes<D>()>>>(maps[0], maps[1], maps[2], p, SEQS, status, budget_us * 1000ull);
    join_parts<__half, D><<<STATES, 128>>>(p);
    e = cudaGetLastError();
  }
  if (e == cudaSuccess) e = cudaMemcpy(&word, status, 4, cudaMemcpyDeviceToHost);
  if (e == cudaSuccess) e = cudaMemcpy(lse, p.lse, sizeof(lse), cudaMemcpyDeviceToHost);
  if (e == cudaSuccess) e = cudaMemcpy2D(out, 2, p.out, 2 * D, 2, STATES, cudaMemcpyDeviceToHost);
  cudaFree(buf);
  if (e != cudaSuccess) {
    cudaGetLastError();
    qmk_internal::note_error(std::string("self test of the attention over a shared prefix: ") + cudaGetErrorString(e));
    return QMK_ERR_CUDA;
  }
  for (int i = 0; i < STATES; ++i)
    if (lse[i] == lse[i] || !__hisnan(out[i])) return QMK_OK;
  return static_cast<int>(word);
}
