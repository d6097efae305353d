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

int launch_compact_cache(const pmx_compact_cache_args& p, cudaStream_t s) {
  if (!p.cache || !p.cachestarts || !p.start_pos || !p.accept_starts || !p.accept_index)
    return fail(PMX_ERR_INVALID_ARGUMENT, "compact_cache: null pointer");
  if (p.sequences <= 0 || p.num_layers <= 0 || p.num_kv_heads <= 0 || p.head_dim <= 0 || p.cache_rows <= 0 ||
      p.max_accept <= 0 || p.index_count <= 0)
    return fail(PMX_ERR_INVALID_ARGUMENT, "compact_cache: sizes must be positive");
  if (p.max_accept > 64) return fail(PMX_ERR_UNSUPPORTED, "compact_cache: at most 64 accepted rows a sequence");
  if (p.sequences > 65535 || p.num_layers > (1 << 20) || p.num_kv_heads > (1 << 20) || p.head_dim > (1 << 20))
    return fail(PMX_ERR_UNSUPPORTED, "compact_cache: sizes beyond what the kernel indexes");
  const int max_accept = (int)p.max_accept;
  int e;
  switch (p.dtype) {
    case PMX_DTYPE_F16: case PMX_DTYPE_BF16: e = 2; break;
    case PMX_DTYPE_F32: e = 4; break;
    default: return fail(PMX_ERR_UNSUPPORTED, "compact_cache: unknown dtype %d", (int)p.dtype);
  }
  // the widest vector that every head row begins on and divides into; 64 rows need the registers
  // that 16-byte vectors would take for 32
  const uint64_t grain = (uint64_t)(p.row_stride | p.layer_stride | p.kv_stride | p.head_stride | p.head_dim) * e |
                         reinterpret_cast<uintptr_t>(p.cache);
  int vec = grain % 16 == 0 ? 16 : grain % 8 == 0 ? 8 : grain % 4 == 0 ? 4 : 2;
  if (max_accept > 32 && vec > 8) vec = 8;
  CompactArgs a{};
  a.cache = (char*)p.cache;
  a.cachestarts = p.cachestarts; a.start_pos = p.start_pos; a.accept_starts = p.accept_starts; a.accept_index = p.accept_index;
  a.rows = p.cache_rows; a.index_count = p.index_count;
  a.row_bytes = p.row_stride * e; a.layer_bytes = p.layer_stride * e; a.kv_bytes = p.kv_stride * e; a.head_bytes = p.head_stride * e;
  a.layers = (int)p.num_layers; a.heads = (int)p.num_kv_heads; a.chunks = (int)p.head_dim * e / vec;
  const int64_t cols = p.num_layers * 2 * p.num_kv_heads * a.chunks;
  const int64_t blocks = ceil_div(cols, 128);
  if (blocks > 0x7FFFFFFFll) return fail(PMX_ERR_UNSUPPORTED, "compact_cache: cache too wide");
  const dim3 grid((unsigned)blocks, (unsigned)p.sequences), block(128);
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
