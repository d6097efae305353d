// Moving rows inside the key/value cache after drafted tokens were verified.
//
// Sequence b has stored drafted tokens at rows base, base + 1, ... with base = cachestarts[b] +
// start_pos[b]; the accepted ones, accept_index[accept_starts[b] ..], move to the front:
// row base + i <- row base + accept_index[i], in all layers, keys and values, all reads before all
// writes.  Bound by the bytes of the rows that move.  A block looks the rows of its sequence up once and then walks
// over columns (the same 16 bytes of every row): a thread has one to four rows and eight of its row's or rows'
// vectors under way, and the block holds all rows of the columns at hand between its reads and its writes, which a
// barrier keeps apart: any indices (repeated, descending) are right.  For 32 sequences of up to 19 rows of 128 KB,
// out of HBM: 31 us; one thread per column with all its rows 50 us (few warps), one vector per thread
// and block 79 us (the look-up's three memory latencies in every block).
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

constexpr int kThreads = 256, kVectors = 8;      // vectors that a thread has under way

// `slots` rows (a power of two) times 256 / slots columns at a time, ROWS rows per thread
template <typename VEC, int ROWS>
__global__ void __launch_bounds__(kThreads) compact_cache_kernel(const CompactArgs a, int slots, int slot_bits) {
  constexpr int GROUPS = kVectors / ROWS;
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.y;
  const int64_t first = __ldcg(a.accept_starts + b), last = __ldcg(a.accept_starts + b + 1);
  const int64_t base = __ldcg(a.cachestarts + b) + __ldcg(a.start_pos + b);
  if (first < 0 || last > a.index_count) return;
  const int n = (int)(last - first < ROWS * slots ? last - first : ROWS * slots);
  const int cols = kThreads >> slot_bits, row = threadIdx.x / cols;
  int64_t src[ROWS], dst[ROWS];                  // byte offsets of this thread's rows
  bool moves[ROWS];
#pragma unroll
  for (int k = 0; k < ROWS; ++k) {
    const int i = row + k * slots;
    const int64_t from = i < n ? __ldcg(a.accept_index + first + i) : -1;
    // a row that stays, or one outside the cache, is left alone
    moves[k] = from >= 0 && from != i && base + from >= 0 && base + from < a.rows && base + i >= 0 && base + i < a.rows;
    src[k] = (base + from) * a.row_bytes;
    dst[k] = (base + i) * a.row_bytes;
  }
  const uint32_t columns = (uint32_t)a.layers * 2 * a.heads * a.chunks, step = gridDim.x * cols;      // below 2^30
  for (uint32_t c0 = blockIdx.x * cols; c0 < columns; c0 += GROUPS * step) {
    VEC held[GROUPS][ROWS];
    char* at[GROUPS];
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      const uint32_t col = c0 + g * step + (threadIdx.x - row * cols);
      const uint32_t hh = col / (uint32_t)a.chunks, ch = col - hh * a.chunks, lk = hh / (uint32_t)a.heads, h = hh - lk * a.heads;
      at[g] = col < columns ? a.cache + (int64_t)(lk >> 1) * a.layer_bytes + (int64_t)(lk & 1) * a.kv_bytes + (int64_t)h * a.head_bytes + (int64_t)(ch * sizeof(VEC)) : nullptr;
#pragma unroll
      for (int k = 0; k < ROWS; ++k)
        if (at[g] && moves[k]) held[g][k] = __ldcg(reinterpret_cast<const VEC*>(at[g] + src[k]));
    }
    __syncthreads();
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
#pragma unroll
      for (int k = 0; k < ROWS; ++k)
        if (at[g] && moves[k]) *reinterpret_cast<VEC*>(at[g] + dst[k]) = held[g][k];
  }
}

template <typename VEC>
int launch_compact_vec(const CompactArgs& a, int max_accept, int64_t B, cudaStream_t s) {
  // a row per thread up to 16 accepted rows (16 columns of 16 bytes: a block still touches whole 256-byte head rows), then two
  // or four
  int bits = 0;
  while (bits < 4 && (1 << bits) < max_accept) ++bits;
  const int slots = 1 << bits;
  const int64_t groups = ceil_div((int64_t)a.layers * 2 * a.heads * a.chunks, kThreads / slots);
  // as many blocks as are resident at once, each with at least one round of loads
  const int64_t most = ceil_div((int64_t)sm_count() * 6, B), rounds = ceil_div(groups, max_accept <= 16 ? 8 : max_accept <= 32 ? 4 : 2);
  const dim3 grid((unsigned)(rounds < most ? rounds : most), (unsigned)B), block(kThreads);
  if (max_accept <= 16) return launch_pdl_k(compact_cache_kernel<VEC, 1>, grid, block, 0, s, a, slots, bits);
  if (max_accept <= 32) return launch_pdl_k(compact_cache_kernel<VEC, 2>, grid, block, 0, s, a, slots, bits);
  return launch_pdl_k(compact_cache_kernel<VEC, 4>, grid, block, 0, s, a, slots, bits);
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
  // the widest vector that every head row begins on and divides into
  const uint64_t grain = (uint64_t)(p.row_stride | p.layer_stride | p.kv_stride | p.head_stride | p.head_dim) * e |
                         reinterpret_cast<uintptr_t>(p.cache);
  const int vec = grain % 16 == 0 ? 16 : grain % 8 == 0 ? 8 : grain % 4 == 0 ? 4 : 2;
  CompactArgs a{};
  a.cache = (char*)p.cache;
  a.cachestarts = p.cachestarts; a.start_pos = p.start_pos; a.accept_starts = p.accept_starts; a.accept_index = p.accept_index;
  a.rows = p.cache_rows; a.index_count = p.index_count;
  a.row_bytes = p.row_stride * e; a.layer_bytes = p.layer_stride * e; a.kv_bytes = p.kv_stride * e; a.head_bytes = p.head_stride * e;
  a.layers = (int)p.num_layers; a.heads = (int)p.num_kv_heads; a.chunks = (int)p.head_dim * e / vec;
  if (p.num_layers * 2 * p.num_kv_heads >= (1 << 30) / a.chunks) return fail(PMX_ERR_UNSUPPORTED, "compact_cache: cache too wide");
  switch (vec) {
    case 16: return launch_compact_vec<uint4>(a, max_accept, p.sequences, s);
    case 8: return launch_compact_vec<uint2>(a, max_accept, p.sequences, s);
    case 4: return launch_compact_vec<uint32_t>(a, max_accept, p.sequences, s);
    default: return launch_compact_vec<uint16_t>(a, max_accept, p.sequences, s);
  }
}

}  // namespace pmx
