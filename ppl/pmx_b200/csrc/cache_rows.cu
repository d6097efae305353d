// Moving rows inside the key/value cache after drafted tokens were verified.
//
// Sequence b has stored drafted tokens at rows base, base + 1, ... with base = cachestarts[b] +
// start_pos[b]; the accepted ones, accept_index[accept_starts[b] ..], move to the front:
// row base + i <- row base + accept_index[i], in all layers, keys and values, all reads before all
// writes.  Bound by the bytes of the rows that move.  A block looks the rows of its sequence up once; its warps then walk
// over columns (the same 16 bytes of every row), and a warp holds all rows of the columns at hand between its reads and its
// writes, eight or sixteen vectors a lane: any indices (repeated, descending) are right, and no warp waits for another.  For
// 32 sequences in 32 layers, out of HBM: 24 us with up to 19 rows of 128 KB, 9.6 us with up to 10; whole blocks that
// read, meet at a barrier and write took 30 and 21 us, one thread per column with all its rows 50 (few warps), one
// vector per thread and block 79 (the look-up's three memory latencies in every block).
#include "common.cuh"

namespace pmx {
namespace {

struct CompactArgs {
  char* cache;
  const int64_t *cachestarts, *start_pos, *accept_starts, *accept_index;
  int64_t rows, index_count;
  int64_t row_bytes, layer_bytes, kv_bytes, head_bytes;   // strides
  int layers, heads, chunks;                              // chunks: vectors of a head row
  int max_accept;                                         // of a sequence; the kernel's variant has vectors for as many rows
};

constexpr int kWarps = 8;
constexpr int kMaxAccept = 64;

// W columns side by side, 32 / W rows to a step; a lane has kVectors vectors under way
template <typename VEC, int W, int kVectors>
__global__ void __launch_bounds__(kWarps * 32) compact_cache_kernel(const __grid_constant__ CompactArgs a) {
  constexpr int R = 32 / W;
  __shared__ int64_t moves[2][kMaxAccept];       // byte offsets from and to which rows move
  __shared__ int count;
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (warp == 0) {
    const int64_t first = __ldcg(a.accept_starts + b), last = __ldcg(a.accept_starts + b + 1);
    const int64_t start = __ldcg(a.cachestarts + b), base = start + __ldcg(a.start_pos + b);
    const int64_t lowest = start > 0 ? start : 0;        // rows in front of it are another sequence's, or none
    const int64_t n = first < 0 || last > a.index_count ? 0 : (last - first < a.max_accept ? last - first : a.max_accept);
    int before = 0;
    for (int i = lane; i < kMaxAccept; i += 32) {
      const int64_t from = i < n ? __ldcg(a.accept_index + first + i) : -1;
      // a row that stays, or one outside the cache or the sequence, is left alone
      const bool on = from >= 0 && from != i && base + from >= lowest && base + from < a.rows && base + i >= lowest && base + i < a.rows;
      const unsigned some = __ballot_sync(0xFFFFFFFFu, on);
      if (on) {
        const int at = before + __popc(some & ((1u << lane) - 1));
        moves[0][at] = (base + from) * a.row_bytes;
        moves[1][at] = (base + i) * a.row_bytes;
      }
      before += __popc(some);
    }
    if (lane == 0) count = before;
  }
  __syncthreads();
  const int m = count, steps = (m + R - 1) / R, row = lane / W;
  if (m == 0) return;
  const uint32_t columns = (uint32_t)a.layers * 2 * a.heads * a.chunks;              // below 2^30
  const uint32_t units = (columns + W - 1) / W, stride = gridDim.x * kWarps;
  uint32_t unit = blockIdx.x * kWarps + warp;
  while (unit < units) {
    VEC held[kVectors];
    char* to[kVectors];
    char* at = nullptr;
    int step = steps;
    const uint32_t full = kVectors / steps;      // units of this round
    uint32_t next = unit;
#pragma unroll
    for (int k = 0; k < kVectors; ++k) {
      to[k] = nullptr;
      if (step == steps) {
        step = 0;
        const uint32_t col = next * W + (lane & (W - 1));
        const uint32_t hh = col / (uint32_t)a.chunks, ch = col - hh * a.chunks, lk = hh / (uint32_t)a.heads, h = hh - lk * a.heads;
        at = next < unit + full * stride && col < columns && next < units
                 ? a.cache + (int64_t)(lk >> 1) * a.layer_bytes + (int64_t)(lk & 1) * a.kv_bytes + (int64_t)h * a.head_bytes + (int64_t)(ch * sizeof(VEC))
                 : nullptr;
        next += stride;
      }
      const int i = step * R + row;
      if (at && i < m) {
        held[k] = __ldcg(reinterpret_cast<const VEC*>(at + moves[0][i]));
        to[k] = at + moves[1][i];
      }
      ++step;
    }
    __syncwarp();                                // all reads of the columns at hand before the writes
#pragma unroll
    for (int k = 0; k < kVectors; ++k)
      if (to[k]) *reinterpret_cast<VEC*>(to[k]) = held[k];
    unit += full * stride;
  }
}

template <typename VEC>
int launch_compact_vec(const CompactArgs& a, int64_t B, cudaStream_t s) {
  // 16 columns side by side are the 256 bytes of a usual head's row; more rows than 16 take twice the registers, more
  // than 32 half the columns.  Up to eight blocks per SM: 26 and 27 us in the case above with twelve and sixteen.
  const int w = a.max_accept <= 32 ? 16 : 8;
  const int64_t blocks = ceil_div(ceil_div((int64_t)a.layers * 2 * a.heads * a.chunks, w), kWarps);
  const int64_t most = ceil_div((int64_t)sm_count() * 8, B);
  const dim3 grid((unsigned)(blocks < most ? blocks : most), (unsigned)B), block(kWarps * 32);
  if (a.max_accept <= 16) return launch_pdl_k(compact_cache_kernel<VEC, 16, 8>, grid, block, 0, s, a);
  if (a.max_accept <= 32) return launch_pdl_k(compact_cache_kernel<VEC, 16, 16>, grid, block, 0, s, a);
  return launch_pdl_k(compact_cache_kernel<VEC, 8, 16>, grid, block, 0, s, a);
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
  a.rows = p.cache_rows; a.index_count = p.index_count; a.max_accept = (int)p.max_accept;
  a.row_bytes = p.row_stride * e; a.layer_bytes = p.layer_stride * e; a.kv_bytes = p.kv_stride * e; a.head_bytes = p.head_stride * e;
  a.layers = (int)p.num_layers; a.heads = (int)p.num_kv_heads; a.chunks = (int)p.head_dim * e / vec;
  if (p.num_layers * 2 * p.num_kv_heads >= (1 << 30) / a.chunks) return fail(PMX_ERR_UNSUPPORTED, "compact_cache: cache too wide");
  switch (vec) {
    case 16: return launch_compact_vec<uint4>(a, p.sequences, s);
    case 8: return launch_compact_vec<uint2>(a, p.sequences, s);
    case 4: return launch_compact_vec<uint32_t>(a, p.sequences, s);
    default: return launch_compact_vec<uint16_t>(a, p.sequences, s);
  }
}

}  // namespace pmx
