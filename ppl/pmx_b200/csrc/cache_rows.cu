// Moving rows inside the key/value cache after drafted tokens were verified.
//
// Sequence b has stored drafted tokens at rows base, base + 1, ... with base = cachestarts[b] +
// start_pos[b]; the accepted ones, accept_index[accept_starts[b] ..], move to the front:
// row base + i <- row base + accept_index[i], in all layers, keys and values, all reads before all
// writes.  Bound by the bytes of the rows that move.  A column -- the same 16 bytes of every row --
// belongs to one thread, which holds its share of all the rows in registers between the reads and
// the writes: the order needs no barrier, any indices (repeated, descending) are right, and all
// loads of a thread are in flight together.
#include "common.cuh"

namespace pmx {
namespace {

struct CompactArgs {
  char* cache;
  const int64_t *cachestarts, *start_pos, *accept_starts, *accept_index;
  int64_t rows, index_count;
  int64_t row_bytes, layer_bytes, kv_bytes, head_bytes;   // strides
  int layers, heads, chunks;                              // chunks: vectors of a head row
};

template <typename VEC, int N>   // N: rows a thread can hold
__global__ void __launch_bounds__(128) compact_cache_kernel(const CompactArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.y;
  const int64_t col = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (col >= (int64_t)a.layers * 2 * a.heads * a.chunks) return;
  const int64_t first = __ldcg(a.accept_starts + b), last = __ldcg(a.accept_starts + b + 1);
  const int64_t base = __ldcg(a.cachestarts + b) + __ldcg(a.start_pos + b);
  if (first < 0 || last > a.index_count) return;
  const int n = (int)(last - first < N ? last - first : N);
  const int64_t ch = col % a.chunks, hh = col / a.chunks;
  const int64_t h = hh % a.heads, lk = hh / a.heads;
  char* at = a.cache + (lk >> 1) * a.layer_bytes + (lk & 1) * a.kv_bytes + h * a.head_bytes + ch * sizeof(VEC);
  VEC held[N];
  uint64_t moved = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (i < n) {
      const int64_t from = __ldcg(a.accept_index + first + i), src = base + from, dst = base + i;
      // a row that stays, or one outside the cache, is left alone
      if (from >= 0 && from != i && src >= 0 && src < a.rows && dst >= 0 && dst < a.rows) {
        held[i] = __ldcg(reinterpret_cast<const VEC*>(at + src * a.row_bytes));
        moved |= 1ull << i;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (moved >> i & 1) *reinterpret_cast<VEC*>(at + (base + i) * a.row_bytes) = held[i];
}

}  // namespace

int launch_compact_cache(void* cache, const int64_t* cachestarts, const int64_t* start_pos, const int64_t* accept_starts,
                         const int64_t* accept_index, int64_t B, int64_t index_count, int max_accept, int layers,
                         int heads, int D, int64_t rows, int64_t row_stride, int64_t layer_stride, int64_t kv_stride,
                         int64_t head_stride, int dtype, cudaStream_t s) {
  if (!cache || !cachestarts || !start_pos || !accept_starts || !accept_index)
    return fail(PMX_ERR_INVALID_ARGUMENT, "compact_cache: null pointer");
  if (B <= 0 || layers <= 0 || heads <= 0 || D <= 0 || rows <= 0 || max_accept <= 0 || index_count <= 0)
    return fail(PMX_ERR_INVALID_ARGUMENT, "compact_cache: sizes must be positive");
  if (max_accept > 64) return fail(PMX_ERR_UNSUPPORTED, "compact_cache: at most 64 accepted rows a sequence");
  if (B > 65535) return fail(PMX_ERR_UNSUPPORTED, "compact_cache: too many sequences");
  int e;
  switch (dtype) {
    case PMX_DTYPE_F16: case PMX_DTYPE_BF16: e = 2; break;
    case PMX_DTYPE_F32: e = 4; break;
    default: return fail(PMX_ERR_UNSUPPORTED, "compact_cache: unknown dtype %d", dtype);
  }
  // the widest vector that every head row begins on and divides into; 64 rows need the registers
  // that 16-byte vectors would take for 32
  const uint64_t grain = (uint64_t)(row_stride | layer_stride | kv_stride | head_stride | D) * e | reinterpret_cast<uintptr_t>(cache);
  int vec = grain % 16 == 0 ? 16 : grain % 8 == 0 ? 8 : grain % 4 == 0 ? 4 : 2;
  if (max_accept > 32 && vec > 8) vec = 8;
  CompactArgs a{};
  a.cache = (char*)cache;
  a.cachestarts = cachestarts; a.start_pos = start_pos; a.accept_starts = accept_starts; a.accept_index = accept_index;
  a.rows = rows; a.index_count = index_count;
  a.row_bytes = row_stride * e; a.layer_bytes = layer_stride * e; a.kv_bytes = kv_stride * e; a.head_bytes = head_stride * e;
  a.layers = layers; a.heads = heads; a.chunks = D * e / vec;
  const int64_t cols = (int64_t)layers * 2 * heads * a.chunks;
  const int64_t blocks = ceil_div(cols, 128);
  if (blocks > 0x7FFFFFFFll) return fail(PMX_ERR_UNSUPPORTED, "compact_cache: cache too wide");
  const dim3 grid((unsigned)blocks, (unsigned)B), block(128);
  if (vec == 16) {
    if (max_accept <= 8) return launch_pdl_k(compact_cache_kernel<uint4, 8>, grid, block, 0, s, a);
    if (max_accept <= 16) return launch_pdl_k(compact_cache_kernel<uint4, 16>, grid, block, 0, s, a);
    return launch_pdl_k(compact_cache_kernel<uint4, 32>, grid, block, 0, s, a);
  }
  if (vec == 8) return launch_pdl_k(compact_cache_kernel<uint2, 64>, grid, block, 0, s, a);
  if (vec == 4) return launch_pdl_k(compact_cache_kernel<uint32_t, 64>, grid, block, 0, s, a);
  return launch_pdl_k(compact_cache_kernel<uint16_t, 64>, grid, block, 0, s, a);
}

}  // namespace pmx
