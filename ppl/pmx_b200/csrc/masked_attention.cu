// Attention of several new tokens per sequence: packed ragged prompts (prompt_attention) and
// trees of drafted tokens over the key/value cache (tree_cache_attention).
//
//   s_ij = scale q_i . k_j;  with a cap c: s = c tanh(s / c);  with a distance bias: s -= slope_h |i - j|
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(s_ij - max_j s_ij),  over the keys j that i may see;
//   a row that sees no key is zero.
// Prompts: the n queries of a sequence are the last n of its L keys; query i (position i + L - n) sees
// the keys below max(position + 1, prefix), or all L when not causal -- one limit per row, so the
// causal, the prefix and the document mask (a sequence IS a document) need no mask in memory.
// Trees: every drafted token sees the whole cached past and those drafted tokens of its sequence
// whose bit is set in its 64-bit mask.  Their keys and values come from the step's tensors, and are
// stored into the cache on the way.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <type_traits>

#include "common.cuh"
#include "packed_f32.cuh"

namespace pmx {
namespace {

constexpr int kTreeLimit = 64;     // drafted tokens of a sequence: the bits of a mask
constexpr int kMaxHeadDim = 256;

struct KvRows {                    // keys and values of one source, element (row, head, d)
  const void *k, *v;
  int64_t k_row, k_head, v_row, v_head;
  int64_t rows;
};

struct AttnArgs {
  const void* q;                   // [Tq, Hq, D] with strides
  int64_t q_tok, q_head;
  KvRows past, cur;                // prompts use `past` only
  const int64_t* seqstarts;        // [B+1] query rows (and rows of `cur`)
  const int64_t* kvstarts;         // prompts: [B+1] key rows
  const int64_t *cachestarts, *start_pos;   // trees: [B]
  const int64_t* tree_mask;        // trees: [Tq]; null for prompts
  const int64_t* prefix;           // [B] or null
  const float* slopes;             // [Hq] or null
  void* out;                       // [Tq, Hq, D] dense
  int64_t Tq;
  int B, Hq, Hkv, D, max_seqlen, causal;
  float scale, cap;
};

// What a CTA or warp knows of one sequence; every index is clamped to the tensors, so that no
// content of the index arrays reaches outside them.
struct Sequence {
  int64_t q0;      // first query row
  int n;           // queries
  int64_t kv0;     // first row of `past`
  int64_t len;     // keys in `past`
  int64_t store;   // trees: row of `past` that takes the first drafted token's key and value; see stored()
  int64_t shift;   // position of query i among the keys: i + shift
  int64_t prefix;  // keys below it are seen by all queries (0: none)
};

__device__ __forceinline__ int64_t clamp64(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : (v > hi ? hi : v); }

__device__ __forceinline__ Sequence load_sequence(const AttnArgs& a, int b) {
  Sequence s;
  s.q0 = clamp64(__ldcg(a.seqstarts + b), 0, a.Tq);
  const int64_t q1 = clamp64(__ldcg(a.seqstarts + b + 1), s.q0, a.Tq);
  s.n = (int)(q1 - s.q0 < a.max_seqlen ? q1 - s.q0 : a.max_seqlen);
  if (a.tree_mask) {
    // of rows [c, c + p) those that exist; 2^40 is beyond any cache and keeps the sums small
    constexpr int64_t kFar = 1ll << 40;
    const int64_t c = clamp64(__ldcg(a.cachestarts + b), -kFar, kFar);
    s.store = c + clamp64(__ldcg(a.start_pos + b), -kFar, kFar);
    s.kv0 = clamp64(c, 0, a.past.rows);
    s.len = clamp64(s.store, s.kv0, a.past.rows) - s.kv0;
    s.shift = 0;
    s.prefix = 0;
  } else {
    s.kv0 = clamp64(__ldcg(a.kvstarts + b), 0, a.past.rows);
    s.len = clamp64(__ldcg(a.kvstarts + b + 1), s.kv0, a.past.rows) - s.kv0;
    s.store = 0;
    s.shift = s.len - (q1 - s.q0);
    s.prefix = a.prefix ? clamp64(__ldcg(a.prefix + b), 0, s.len) : 0;
  }
  return s;
}

// The row that takes drafted token i's key and value, or -1: rows outside the cache are dropped, and so are those in front of
// their sequence's first (a negative start_pos), which are another's.
__device__ __forceinline__ int64_t stored(const AttnArgs& a, const Sequence& s, int64_t i) {
  const int64_t row = s.store + i;
  return row >= s.kv0 && row < a.past.rows ? row : -1;
}

// keys of `past` that query i sees: the first this many
__device__ __forceinline__ int64_t visible(const AttnArgs& a, const Sequence& s, int64_t i) {
  if (a.tree_mask || !a.causal) return s.len;
  const int64_t own = clamp64(i + s.shift + 1, 0, s.len);
  return own > s.prefix ? own : s.prefix;
}

// ---- one warp per (query, head), any type, head size and alignment -----------------------------
// 32 keys a round: each lane takes the dot product with one key, then the lanes share the head's
// dimensions out for the values.  Keys a query may not see are not touched.
constexpr int kRowWarps = 4;

template <typename T>
__global__ void __launch_bounds__(kRowWarps * 32) attention_row_kernel(const __grid_constant__ AttnArgs a) {
  __shared__ float sq[kRowWarps][kMaxHeadDim];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t item = (int64_t)blockIdx.x * kRowWarps + warp;
  if (item >= a.Tq * a.Hq) return;
  const int64_t t = item / a.Hq;
  const int h = (int)(item - t * a.Hq), hk = h / (a.Hq / a.Hkv);
  int before = 0;
  for (int i = lane; i <= a.B; i += 32) before += __ldcg(a.seqstarts + i) <= t ? 1 : 0;
  const int b = __reduce_add_sync(0xFFFFFFFFu, before) - 1;
  T* out = reinterpret_cast<T*>(a.out) + (t * a.Hq + h) * a.D;
  Sequence s{};
  if (b >= 0 && b < a.B) s = load_sequence(a, b);
  const int64_t i = t - s.q0;
  if (b < 0 || b >= a.B || i >= s.n) {             // a row of no sequence
    for (int d = lane; d < a.D; d += 32) out[d] = Elem<T>::from_f(0.f);
    return;
  }
  const T* q = reinterpret_cast<const T*>(a.q) + t * a.q_tok + (int64_t)h * a.q_head;
  for (int d = lane; d < a.D; d += 32) sq[warp][d] = Elem<T>::to_f(q[d]);
  __syncwarp();
  if (a.tree_mask && h % (a.Hq / a.Hkv) == 0) {    // one head of each group stores the new key and value
    const int64_t row = stored(a, s, i);
    if (row >= 0) {
      const T* kc = reinterpret_cast<const T*>(a.cur.k) + t * a.cur.k_row + (int64_t)hk * a.cur.k_head;
      const T* vc = reinterpret_cast<const T*>(a.cur.v) + t * a.cur.v_row + (int64_t)hk * a.cur.v_head;
      T* kd = reinterpret_cast<T*>(const_cast<void*>(a.past.k)) + row * a.past.k_row + (int64_t)hk * a.past.k_head;
      T* vd = reinterpret_cast<T*>(const_cast<void*>(a.past.v)) + row * a.past.v_row + (int64_t)hk * a.past.v_head;
      for (int d = lane; d < a.D; d += 32) {
        kd[d] = kc[d];
        vd[d] = vc[d];
      }
    }
  }
  float acc[kMaxHeadDim / 32];
#pragma unroll
  for (int r = 0; r < kMaxHeadDim / 32; ++r) acc[r] = 0.f;
  float m = -INFINITY, l = 0.f;
  const float slope = a.slopes ? __ldcg(a.slopes + h) : 0.f;
  const uint64_t bits = a.tree_mask ? (uint64_t)__ldcg(a.tree_mask + t) : 0ull;
  const int64_t limit = visible(a, s, i);
  const int64_t total = a.tree_mask ? limit + s.n : limit;
  for (int64_t j0 = 0; j0 < total; j0 += 32) {
    const int64_t j = j0 + lane;
    const bool is_cur = j >= limit;
    const bool seen = j < total && (!is_cur || (bits >> (j - limit) & 1));
    const KvRows& src = is_cur ? a.cur : a.past;
    const int64_t row = is_cur ? s.q0 + (j - limit) : s.kv0 + j;
    float x = -INFINITY;
    if (seen) {
      const T* k = reinterpret_cast<const T*>(src.k) + row * src.k_row + (int64_t)hk * src.k_head;
      float dot = 0.f;
      for (int d = 0; d < a.D; ++d) dot = fmaf(sq[warp][d], Elem<T>::to_f(k[d]), dot);
      x = dot * a.scale;
      if (a.cap > 0.f) x = a.cap * tanhf(x / a.cap);
      if (a.slopes) {
        const int64_t far = i + s.shift - j;
        x -= slope * (float)(far < 0 ? -far : far);
      }
    }
    float mx = x;
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, o));
    const float m_new = fmaxf(m, mx);
    const float base = m_new == -INFINITY ? 0.f : m_new;
    const float corr = expf(m - base);
    const float p = seen ? expf(x - base) : 0.f;
    l = l * corr + p;                               // each lane's share
    m = m_new;
#pragma unroll
    for (int r = 0; r < kMaxHeadDim / 32; ++r) acc[r] *= corr;
    unsigned todo = __ballot_sync(0xFFFFFFFFu, seen);
    while (todo) {
      const int jj = __ffs(todo) - 1;
      todo &= todo - 1;
      const float pj = __shfl_sync(0xFFFFFFFFu, p, jj);
      const int64_t rj = __shfl_sync(0xFFFFFFFFu, row, jj);
      const bool cj = j0 + jj >= limit;
      const T* v = reinterpret_cast<const T*>(cj ? a.cur.v : a.past.v) + rj * (cj ? a.cur.v_row : a.past.v_row) +
                   (int64_t)hk * (cj ? a.cur.v_head : a.past.v_head);
#pragma unroll
      for (int r = 0; r < kMaxHeadDim / 32; ++r)
        if (lane + 32 * r < a.D) acc[r] = fmaf(pj, Elem<T>::to_f(v[lane + 32 * r]), acc[r]);
    }
  }
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, o);
  const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
  for (int r = 0; r < kMaxHeadDim / 32; ++r)
    if (lane + 32 * r < a.D) out[lane + 32 * r] = Elem<T>::from_f(acc[r] * inv);
}

int launch_rows(const AttnArgs& a, int dtype, const char* name, cudaStream_t s) {
  const int64_t blocks = ceil_div(a.Tq * a.Hq, kRowWarps);
  if (blocks > 0x7FFFFFFFll) return fail(PMX_ERR_UNSUPPORTED, "%s: too many rows", name);
  const dim3 grid((unsigned)blocks), block(kRowWarps * 32);
  switch (dtype) {
    case PMX_DTYPE_F16: return launch_pdl_k(attention_row_kernel<__half>, grid, block, 0, s, a);
    case PMX_DTYPE_BF16: return launch_pdl_k(attention_row_kernel<__nv_bfloat16>, grid, block, 0, s, a);
    default: return launch_pdl_k(attention_row_kernel<float>, grid, block, 0, s, a);
  }
}

#include "tcgen05_common.cuh"
namespace tc {
#include "masked_attention_tc.cuh"
}

}  // namespace

int attention_check(int out[4], cudaStream_t s) {
  PMX_CUDA_OK(cudaMemcpyFromSymbolAsync(out, tc::g_attention_status, sizeof(tc::g_attention_status), 0, cudaMemcpyDeviceToHost, s));
  PMX_CUDA_OK(cudaStreamSynchronize(s));
  if (out[0] == 0) return PMX_OK;
  void* at = nullptr;
  PMX_CUDA_OK(cudaGetSymbolAddress(&at, tc::g_attention_status));
  PMX_CUDA_OK(cudaMemsetAsync(at, 0, sizeof(tc::g_attention_status), s));
  PMX_CUDA_OK(cudaStreamSynchronize(s));
  return fail(PMX_ERR_DEVICE_CHECK, "attention: a wait inside a kernel ran out (role %d, tile %d, CTA %d)", out[1], out[2], out[3]);
}

size_t attention_workspace_bytes(int64_t Tq, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_seqlen,
                                 int64_t max_kvlen, int dtype) {
  return tc::tc_workspace(tc::plan_tc(Tq, B, Hq, Hkv, D, max_seqlen, max_kvlen, dtype), Tq, B, Hq, Hkv, D);
}

// what the two operators share once their own arguments are in place
template <typename P>
int run_attention(AttnArgs& a, const P& p, const char* name, cudaStream_t s) {
  if (p.tokens <= 0 || p.sequences <= 0 || p.num_heads <= 0 || p.num_kv_heads <= 0 || p.head_dim <= 0 ||
      p.max_seqlen <= 0 || p.max_kvlen <= 0 || a.past.rows <= 0 || p.num_heads % p.num_kv_heads)
    return fail(PMX_ERR_INVALID_ARGUMENT, "%s: sizes must be positive and num_heads a multiple of num_kv_heads (tokens=%lld sequences=%lld heads=%lld/%lld)", name, (long long)p.tokens, (long long)p.sequences, (long long)p.num_heads, (long long)p.num_kv_heads);
  if (p.head_dim > kMaxHeadDim) return fail(PMX_ERR_UNSUPPORTED, "%s: head_dim %lld (at most %d)", name, (long long)p.head_dim, kMaxHeadDim);
  if (p.sequences > (1 << 20) || p.num_heads > (1 << 16) || p.tokens > (1ll << 40)) return fail(PMX_ERR_UNSUPPORTED, "%s: too many sequences, heads or tokens", name);
  if (p.dtype != PMX_DTYPE_F16 && p.dtype != PMX_DTYPE_BF16 && p.dtype != PMX_DTYPE_F32)
    return fail(PMX_ERR_UNSUPPORTED, "%s: unknown dtype %d", name, (int)p.dtype);
  a.q = p.query; a.q_tok = p.q_token_stride; a.q_head = p.q_head_stride;
  a.seqstarts = p.seqstarts;
  a.out = p.out; a.Tq = p.tokens; a.B = (int)p.sequences; a.Hq = (int)p.num_heads; a.Hkv = (int)p.num_kv_heads;
  a.D = (int)p.head_dim;
  const int64_t most = p.max_seqlen < p.tokens ? p.max_seqlen : p.tokens;
  a.max_seqlen = (int)(most < 0x7FFFFFFF ? most : 0x7FFFFFFF);
  a.scale = (float)p.scale; a.cap = (float)p.logit_cap;
  if (!(a.scale > 0.f) || a.scale > 3e38f) return fail(PMX_ERR_INVALID_ARGUMENT, "%s: scale must be positive and finite", name);
  if (!(a.cap >= 0.f) || a.cap > 3e38f) return fail(PMX_ERR_INVALID_ARGUMENT, "%s: logit_cap must be finite and not negative", name);
  const tc::TcPlan plan = tc::plan_tc(p.tokens, p.sequences, p.num_heads, p.num_kv_heads, p.head_dim, p.max_seqlen, p.max_kvlen, (int)p.dtype);
  const size_t need = tc::tc_workspace(plan, p.tokens, p.sequences, p.num_heads, p.num_kv_heads, p.head_dim);
  if (need && (!p.workspace || p.workspace_bytes < (int64_t)need))
    return fail(PMX_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, %lld given", name, need, (long long)p.workspace_bytes);
  if (need && !aligned16(p.workspace)) return fail(PMX_ERR_ALIGNMENT, "%s: the workspace must be 16-byte aligned", name);
  bool done;
  const int st = tc::launch_tc(a, plan, (int)p.dtype, name, p.workspace, s, &done);
  return done ? st : launch_rows(a, (int)p.dtype, name, s);
}

int launch_prompt_attention(const pmx_prompt_attention_args& p, cudaStream_t s) {
  const char* name = "prompt_attention";
  if (!p.query || !p.key || !p.value || !p.out || !p.seqstarts || !p.kvstarts) return fail(PMX_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  AttnArgs a{};
  a.past = KvRows{p.key, p.value, p.k_token_stride, p.k_head_stride, p.v_token_stride, p.v_head_stride, p.keys};
  a.kvstarts = p.kvstarts; a.prefix = p.prefix_lens; a.slopes = p.alibi_slopes;
  a.causal = p.is_causal != 0;
  return run_attention(a, p, name, s);
}

int launch_tree_attention(const pmx_tree_attention_args& p, cudaStream_t s) {
  const char* name = "tree_cache_attention";
  if (!p.query || !p.current_key || !p.current_value || !p.out || !p.cache || !p.seqstarts || !p.cachestarts || !p.start_pos || !p.tree_mask)
    return fail(PMX_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  if (p.max_seqlen > kTreeLimit) return fail(PMX_ERR_UNSUPPORTED, "%s: at most %d drafted tokens a sequence", name, kTreeLimit);
  const int e = p.dtype == PMX_DTYPE_F32 ? 4 : 2;
  char* layer = (char*)p.cache + p.layer_offset * e;
  AttnArgs a{};
  a.past = KvRows{layer, layer + p.kv_stride * e, p.row_stride, p.head_stride, p.row_stride, p.head_stride, p.cache_rows};
  a.cur = KvRows{p.current_key, p.current_value, p.k_token_stride, p.k_head_stride, p.v_token_stride, p.v_head_stride, p.tokens};
  a.cachestarts = p.cachestarts; a.start_pos = p.start_pos; a.tree_mask = p.tree_mask;
  return run_attention(a, p, name, s);
}

}  // namespace pmx
