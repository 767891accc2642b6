// C entries of the packed caches (packed_cache.cuh) and of the attention over them (packed_attention.cuh).
#include "../../include/qwen_megakernel.h"

#include <algorithm>
#include <atomic>
#include <string>

#include "engine_internal.h"
#include "packed_attention.cuh"
#include "packed_cache.cuh"
#include "prefill_sm100.h"

namespace {

using namespace qmk_packed;

constexpr int MAX_ROWS = 1 << 24;                // of a cache
constexpr int MAX_HEADS = 1024;
constexpr long long MAX_TILES = 0x7ffffff0;       // of all sequences and heads: a warp counts up to three past its last one
constexpr int MAX_RANKS = 4;                     // clusters of 2^(4 - 1) CTAs

int refuse(const char *who, const std::string &why) {
  qmk_internal::note_error(std::string(who) + ": " + why);
  return QMK_ERR_BAD_ARGUMENT;
}
int answer(const char *who, cudaError_t e) {
  if (e == cudaSuccess) return QMK_OK;
  cudaGetLastError();
  qmk_internal::note_error(std::string(who) + ": " + cudaGetErrorString(e));
  return QMK_ERR_CUDA;
}
bool odd(const void *ptr) { return (reinterpret_cast<unsigned long long>(ptr) & 15u) != 0; }
bool odd(long long stride, int size, int of) { return size > 1 && stride % of; }

// What is wrong with a cache; null: nothing, and `c` says where it is
const char *read_cache(const qmk_packed_cache *a, Caches *c) {
  if (!a) return "null pointer argument";
  if (a->bits != 4 && a->bits != 8) return "bits must be 4 or 8";
  if (a->head_dim != 64 && a->head_dim != 128) return "head_dim must be 64 or 128";
  if (a->num_sequences < 1 || a->num_sequences > MAX_SEQS) return "num_sequences must be in [1, 128]";
  if (a->kv_heads < 1 || a->kv_heads > MAX_HEADS) return "kv_heads must be in [1, 1024]";
  if (a->rows < 0 || a->rows > MAX_ROWS) return "rows must be in [0, 2^24]";
  if (a->rows > 0 && (a->k ? !a->v : !a->k_base || !a->v_base)) return "null pointer argument";
  if (odd(a->seq_stride, a->num_sequences, 16) || odd(a->head_stride, a->kv_heads, 16) || odd(a->row_stride, a->rows, 16)) return "a cache's strides must be multiples of 16 bytes";
  if (a->rows > 1 && a->row_stride < a->head_dim * a->bits / 8 + TRAILER) return "rows of a cache overlap: the row stride is below a row's bytes";
  c->seqs = a->num_sequences;
  c->kv_heads = a->kv_heads;
  c->rows = a->rows;
  c->head = a->head_stride;
  c->row = a->row_stride;
  for (int b = 0; b < a->num_sequences; ++b) {
    c->k[b] = c->v[b] = nullptr;
    if (a->rows == 0) continue;                  // (no address is looked at)
    c->k[b] = static_cast<const unsigned char *>(a->k ? a->k[b] : static_cast<const char *>(a->k_base) + b * a->seq_stride);
    c->v[b] = static_cast<const unsigned char *>(a->k ? a->v[b] : static_cast<const char *>(a->v_base) + b * a->seq_stride);
    if (!c->k[b] || !c->v[b]) return "null pointer argument";
    if (odd(c->k[b]) || odd(c->v[b])) return "a cache's address must be a multiple of 16";
  }
  return nullptr;
}

// What is wrong with the rows of a call; null: nothing
const char *read_rows_of(const qmk_packed_rows *a, RowParams *p) {
  if (!a) return "null pointer argument";
  if (a->type < 0 || a->type > 1) return "the type is fp16 (0) or bf16 (1)";
  if (a->rows < 0 || a->rows > MAX_ROWS) return "rows must be in [0, 2^24]";
  if (static_cast<long long>(p->caches.seqs) * p->caches.kv_heads * a->rows > 0x7fffffffll) return "2^31 rows of all heads or more";
  if (a->rows > 0 && (!a->k || !a->v)) return "null pointer argument";
  if (odd(a->k) || odd(a->v)) return "the rows' addresses must be multiples of 16";
  if (odd(a->seq_stride, p->caches.seqs, 8) || odd(a->head_stride, p->caches.kv_heads, 8) || odd(a->row_stride, a->rows, 8)) return "the rows' strides must be multiples of 8 elements";
  p->k = a->k;
  p->v = a->v;
  p->seq = a->seq_stride;
  p->head = a->head_stride;
  p->row = a->row_stride;
  p->rows = a->rows;
  p->starts = a->starts;
  p->start = a->start;
  p->lens = a->lens;
  return nullptr;
}

// Rows that a call would write twice whatever its starts and lengths; null: none
const char *shared_rows(const Caches &c) {
  if (c.rows == 0) return nullptr;
  if (c.kv_heads > 1 && c.head == 0) return "heads share a cache's rows: the head stride is 0";
  for (int b = 0; b < c.seqs; ++b)
    if (c.k[b] == c.v[b]) return "keys and values share a cache";
  return nullptr;
}
const char *shared_rows(const RowParams &p) {
  if (p.k == p.v) return "keys and values share rows";
  if ((p.caches.seqs > 1 && p.seq == 0) || (p.caches.kv_heads > 1 && p.head == 0) || (p.rows > 1 && p.row == 0)) return "rows share memory: a stride is 0";
  return nullptr;
}

template <typename T, int DIM, int BITS>
void (*row_kernel(bool write))(RowParams, unsigned int) { return write ? write_rows<T, DIM, BITS> : read_rows<T, DIM, BITS>; }
template <typename T>
void (*row_kernel(bool write, int dim, int bits))(RowParams, unsigned int) {
  if (bits == 4) return dim == 64 ? row_kernel<T, 64, 4>(write) : row_kernel<T, 128, 4>(write);
  return dim == 64 ? row_kernel<T, 64, 8>(write) : row_kernel<T, 128, 8>(write);
}

int rows_call(const char *who, const qmk_packed_cache *cache, const qmk_packed_rows *rows, bool write, cudaStream_t stream) {
  qmk_internal::begin_call();
  RowParams p;
  if (const char *why = read_cache(cache, &p.caches)) return refuse(who, why);
  if (const char *why = read_rows_of(rows, &p)) return refuse(who, why);
  const unsigned int count = static_cast<unsigned int>(p.caches.seqs) * p.caches.kv_heads * p.rows;
  if (count == 0) return QMK_OK;
  if (const char *why = write ? shared_rows(p.caches) : shared_rows(p)) return refuse(who, why);
  p.by_rows.set(p.rows);
  p.by_heads.set(p.caches.kv_heads);
  // (CTAs: 4 x 4096 rows of 8 heads written by four an SM for keys and four for values 20.9 us, by eight 21.1, by sixteen 22.2; 28 x 4096 read by 64 an SM 104, by sixteen 108, by eight 123)
  const unsigned int rows_of_block = THREADS / (write ? 4 : 8), blocks = std::min((count + rows_of_block - 1) / rows_of_block, 148u * (write ? 4 : 64));
  void (*const kernel)(RowParams, unsigned int) = rows->type == 0 ? row_kernel<__half>(write, cache->head_dim, cache->bits) : row_kernel<__nv_bfloat16>(write, cache->head_dim, cache->bits);
  kernel<<<dim3(blocks, write ? 2 : 1), THREADS, 0, stream>>>(p, count);
  return answer(who, cudaGetLastError());
}

// How a call is cut.  Where no warp gets more than ITEM_TILES tiles of caches that are full, a cluster of CTAs takes an item, one launch; up to ITEM_WAVES times as many items
// as are resident together.  Else, of few sequences, as many clusters of two CTAs as are resident together share the items, and a second launch joins what they have
// joined; of more sequences a warp takes a stretch of the line of tiles, all resident together, not more of them than there can be tiles, and a second launch joins.
// Measured in a graph, us, 128 dims, 4 bits, 16 query heads on 8, lengths from 0 up (tiles a warp in brackets).  Stretches against a cluster an item: one sequence of 128 rows
// 6.3 and 5.3; 16 of up to 2048 (4) 15.4 and 14.0; 128 of up to 1024 (8, seven CTAs an SM one after the other) 32.7 and 31.8; 16 of up to 4096 (8) 19.6 and 20.1, of up to 8192
// (16) 27.4 and 31.4 (a cluster has a longest item to wait for, a stretch has not); one of 8192 (8) 13.5 and 12.0, of 32,768 (32) 21.0 and 30.8.  On the host 16 and 11.
// Clusters of 16 CTAs start late: one sequence of 2048 rows 15.5, of eight 6.5.  Stretches against pairs that share: one sequence of 16,384 rows 16.7 and 14.0, of 32,768 21.0
// and 17.9 (16 query heads on 2 21.5 and 16.7), of 131,072 42.5 and 37.5; four of up to 16,384 20.2 and 18.7, all full 26.2 and 24.8; eight of up to 32,768 44 and 54.
// Sharing by single CTAs 19.0 where pairs take 17.9, by four or eight 22; one of 8192 by pairs or by one cluster of eight 12.0.
// The rule sees how long the caches may be, and so does that of the join; lengths are on the device.  Of 128 caches of 8192 rows one full and the others empty takes 77 us, most of
// them join_few's (one warp a head for some 256 parts), where that sequence in a call of its own takes 12; one of 32,768 beside 127 of 200 68.
constexpr int ITEM_TILES = 8, ITEM_WAVES = 4;
constexpr int SHARING_SEQS = 4, SHARING_PAIRS = 8;                          // sequences at most, pairs of an item at least (fewer leave many places of the device empty)
struct Cut {
  int ranks, splits, warps;
};
long long most_tiles(int seqs, int kv_heads, int rows) { return static_cast<long long>(seqs) * kv_heads * ((rows + TILE - 1) / TILE); }
Cut cut_of(int seqs, int kv_heads, int group, int dim, int bits, int rows) {
  const int ctas = SMS * ctas_per_sm(way_of(group), dim, bits), tiles = (rows + TILE - 1) / TILE, items = seqs * kv_heads;
  int ranks = 1;                                 // log2 of a cluster's CTAs, + 1
  while (ranks < MAX_RANKS && (items << ranks) <= ctas && (WARPS << (ranks - 1)) < tiles) ++ranks;
  if (items <= ITEM_WAVES * ctas && tiles <= ITEM_TILES * (WARPS << (ranks - 1))) return Cut{ranks, 1, 0};
  const int pairs = ctas / 2 / items;
  if (seqs <= SHARING_SEQS && pairs >= SHARING_PAIRS) return Cut{2, pairs, items * pairs};
  return Cut{0, 1, static_cast<int>(std::min<long long>(std::max(most_tiles(seqs, kv_heads, rows), 1ll), ctas * WARPS))};
}
long long workspace_bytes(const Cut &cut, int group, int dim) { return 2ll * cut.warps * group * (dim * 4ll + 8); }

// How the parts are joined goes by how many an item has where all stretches or pairs are used: warps (of stretches), or CTAs of four, eight or 32 warps.
template <typename T, int DIM>
cudaError_t launch_join(const AttendParams &p, bool overlap, cudaStream_t stream) {
  const qmk_tc::PdlScope scope(overlap);
  const int rows = p.caches.seqs * p.q_heads, each = p.warps / (p.caches.seqs * p.caches.kv_heads);
  if (each <= FEW && p.ranks == 0) {
    const int units = std::max(p.warps * p.group, p.caches.seqs);
    return qmk_tc::launch_kernel(join_few<T, DIM>, dim3(std::min((units + 7) / 8, 8 * SMS)), dim3(256), 0, stream, p);
  }
  if (each <= 16) return qmk_tc::launch_kernel(join_many<T, DIM, 4, 4>, dim3(rows), dim3(128), 0, stream, p);
  if (each <= 64) return qmk_tc::launch_kernel(join_many<T, DIM, 8, 8>, dim3(rows), dim3(256), 0, stream, p);
  return qmk_tc::launch_kernel(join_many<T, DIM, 32, 8>, dim3(rows), dim3(1024), 0, stream, p);
}

// A kernel's shared memory, once a device (the call takes half a microsecond)
template <typename K>
cudaError_t allow(std::atomic<unsigned long long> &known, K kernel, int bytes) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  const unsigned long long bit = device < 64 ? 1ull << device : 0;
  if (e != cudaSuccess || (known.load() & bit)) return e;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) known |= bit;
  return e;
}
template <typename A>
cudaError_t launch_tiles(const AttendParams &p, cudaStream_t stream) {
  static std::atomic<unsigned long long> tiles_known{0}, items_known{0};
  if (p.ranks == 0) {
    const cudaError_t e = allow(tiles_known, attend_tiles<A>, A::SMEM);
    if (e != cudaSuccess) return e;
    return qmk_tc::launch_kernel(attend_tiles<A>, dim3(std::min(p.warps, SMS * A::CTAS)), dim3(WARPS * 32), A::SMEM, stream, p);         // (a warp of each where there are few)
  }
  const cudaError_t e = allow(items_known, attend_items<A>, A::SMEM);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((p.caches.seqs * p.caches.kv_heads * p.splits) << (p.ranks - 1));
  cfg.blockDim = dim3(WARPS * 32);
  cfg.dynamicSmemBytes = A::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1 << (p.ranks - 1);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = qmk_tc::pdl_active() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, attend_items<A>, p);
}
template <typename T, int DIM, int BITS>
cudaError_t attend(const AttendParams &p, bool overlap, cudaStream_t stream) {
  cudaError_t e = cudaSuccess;
  const bool tiles = p.caches.rows > 0 || p.ranks > 0;
  if (tiles) {
    switch (way_of(p.group)) {
      case PAIR: e = launch_tiles<AttendPair<T, DIM, BITS>>(p, stream); break;
      case QUAD: e = launch_tiles<AttendQuad<T, DIM, BITS>>(p, stream); break;
      case ONE: e = launch_tiles<Attend<T, DIM, BITS, 1>>(p, stream); break;
      case TWO: e = launch_tiles<Attend<T, DIM, BITS, 2>>(p, stream); break;
    }
  }
  return e != cudaSuccess || p.warps == 0 ? e : launch_join<T, DIM>(p, overlap && tiles, stream);    // (alone, it would not wait for the kernel of another call in front of it)
}
template <typename T>
cudaError_t attend(const AttendParams &p, int dim, int bits, bool overlap, cudaStream_t stream) {
  if (bits == 4) return dim == 64 ? attend<T, 64, 4>(p, overlap, stream) : attend<T, 128, 4>(p, overlap, stream);
  return dim == 64 ? attend<T, 64, 8>(p, overlap, stream) : attend<T, 128, 8>(p, overlap, stream);
}

}  // namespace

extern "C" int qmk_write_cache_packed(const qmk_packed_cache *cache, const qmk_packed_rows *rows, cudaStream_t stream) {
  return rows_call("qmk_write_cache_packed", cache, rows, true, stream);
}
extern "C" int qmk_read_cache_packed(const qmk_packed_cache *cache, const qmk_packed_rows *rows, cudaStream_t stream) {
  return rows_call("qmk_read_cache_packed", cache, rows, false, stream);
}

extern "C" long long qmk_attention_packed_cache_workspace(int num_sequences, int q_heads, int kv_heads, int head_dim, int bits, int rows) {
  if (num_sequences < 1 || num_sequences > MAX_SEQS || kv_heads < 1 || kv_heads > MAX_HEADS || q_heads < 1 || q_heads % kv_heads || q_heads / kv_heads > MAX_GROUP ||
      (head_dim != 64 && head_dim != 128) || (bits != 4 && bits != 8) || rows < 0 || rows > MAX_ROWS)
    return -1;
  if (most_tiles(num_sequences, kv_heads, rows) > MAX_TILES) return -1;
  return workspace_bytes(cut_of(num_sequences, kv_heads, q_heads / kv_heads, head_dim, bits, rows), q_heads / kv_heads, head_dim);
}

extern "C" int qmk_attention_packed_cache(const qmk_packed_cache *cache, const qmk_packed_attention *a, cudaStream_t stream) {
  const char *const who = "qmk_attention_packed_cache";
  qmk_internal::begin_call();
  AttendParams p;
  if (const char *why = read_cache(cache, &p.caches)) return refuse(who, why);
  if (!a || !a->q || !a->out || !a->lens) return refuse(who, "null pointer argument");
  if (a->type < 0 || a->type > 1) return refuse(who, "the type is fp16 (0) or bf16 (1)");
  if (a->q_heads < 1 || a->q_heads % cache->kv_heads || a->q_heads / cache->kv_heads > MAX_GROUP) return refuse(who, "q_heads must be 1 to 16 times kv_heads");
  if (most_tiles(cache->num_sequences, cache->kv_heads, cache->rows) > MAX_TILES) return refuse(who, "2^36 rows of all heads (512 less), or more");
  if (!(a->scale > -2.0e38f && a->scale < 2.0e38f)) return refuse(who, "the scale must be finite, and below 2e38");   // (times log2 e too)
  if (odd(a->q) || odd(a->out) || odd(a->workspace)) return refuse(who, "pointers must be 16-byte aligned");
  if (odd(a->q_seq_stride, cache->num_sequences, 8) || odd(a->q_head_stride, a->q_heads, 8)) return refuse(who, "the queries' strides must be multiples of 8 elements");
  p.group = a->q_heads / cache->kv_heads;
  const Cut cut = cut_of(cache->num_sequences, cache->kv_heads, p.group, cache->head_dim, cache->bits, cache->rows);
  if (cut.warps > 0 && (!a->workspace || a->workspace_bytes < workspace_bytes(cut, p.group, cache->head_dim))) return refuse(who, "workspace too small");
  p.q = a->q;
  p.q_seq = a->q_seq_stride;
  p.q_head = a->q_head_stride;
  p.q_heads = a->q_heads;
  p.lens = a->lens;
  p.scale_log2 = a->scale * LOG2E;
  p.ranks = cut.ranks;
  p.splits = cut.splits;
  p.warps = cut.warps;
  p.part_out = static_cast<float *>(a->workspace);
  p.part_ml = reinterpret_cast<float2 *>(p.part_out + 2ll * p.warps * p.group * cache->head_dim);
  p.out = a->out;
  p.lse = a->lse;
  return answer(who, a->type == 0 ? attend<__half>(p, cache->head_dim, cache->bits, a->no_overlap == 0, stream)
                                  : attend<__nv_bfloat16>(p, cache->head_dim, cache->bits, a->no_overlap == 0, stream));
}
