// Rotary positions on packed query and key heads, optionally behind an RMS norm of every head.
//
// For a token at position p and pair i of the first `rotary_dim` values of a head, with
// a = p * f_i:  (x1, x2) -> m (x1 cos a - x2 sin a, x2 cos a + x1 sin a);  the pairs are
// (i, i + rotary_dim/2) or, interleaved, (2i, 2i+1); the other values pass through.  With the
// norm, x is first x * w / sqrt(mean over the head of x^2 + eps).  One rounding, at the store.
//
// Bound by the bytes of the heads, read once and written once: the norm's sum stays inside the
// lanes that hold the head, and no angle comes from memory.  A CTA takes a run of whole tokens:
// its threads first fill a table of cosines and sines in shared memory -- one entry per (token,
// pair), used by all heads of the token -- and then walk the heads, every lane with two 16-byte
// vectors that hold complete pairs.  The angle is taken in turns, p * f_i / (2 pi), in 64 bits, and
// only its distance to the nearest whole turn goes on in 32 bits, so far positions keep the
// precision of near ones (in 32 bits p = 10^6 would already be off by 0.06 rad).
#include "common.cuh"

namespace pmx {
namespace {

constexpr int kRotThreads = 256;
constexpr int kRotMaxPairs = 128;
constexpr int kRotMaxTokens = 8;      // tokens of a CTA

struct RotaryArgs {
  double turns[kRotMaxPairs];         // f_i / (2 pi)
  const void *q, *k;                  // [T, Hq, D], [T, Hkv, D] with strides; k may be null (Hkv = 0)
  const void *qw, *kw;                // [D] norm weights, or null
  void *qo, *ko;                      // dense
  int64_t q_tok, q_head, k_tok, k_head;
  const int64_t *seqstarts, *start_pos, *position_ids;
  int64_t T;
  int B, Hq, Hkv, D, pairs, tokens;   // tokens: of a CTA
  int lanes;                          // vector kernel: lanes per head, a power of two
  float eps, factor;
};

// The position of token t, or false for a token of no sequence.  Called by a whole warp; the
// sequence is the number of starts at or before t, counted by the lanes side by side: one
// memory latency where a binary search would pay one per level.
__device__ __forceinline__ bool token_position(const RotaryArgs& a, int64_t t, int64_t* pos) {
  if (a.position_ids) {
    *pos = __ldcg(a.position_ids + t);
    return true;
  }
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int i = lane; i <= a.B; i += 32) before += __ldcg(a.seqstarts + i) <= t ? 1 : 0;
  before = __reduce_add_sync(0xFFFFFFFFu, before);
  const int b = before - 1;
  if (b < 0 || b >= a.B) return false;
  *pos = __ldcg(a.start_pos + b) + (t - __ldcg(a.seqstarts + b));
  return true;
}

// Fills the CTA's table for its tokens: warp w looks up the tokens w, w + 8, ..., then all threads
// share the entries out.  A token of no sequence gets the rotation by zero and live = false.
__device__ __forceinline__ void fill_table(const RotaryArgs& a, int64_t t0, int n, float* cs, float* sn, double* pos,
                                           bool* live) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = warp; i < n; i += kRotThreads / 32) {
    int64_t p = 0;
    const bool ok = token_position(a, t0 + i, &p);
    if (lane == 0) {
      pos[i] = (double)p;
      live[i] = ok;
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < n * a.pairs; e += kRotThreads) {
    const int i = e / a.pairs, j = e - i * a.pairs;
    double turn = pos[i] * a.turns[j];
    turn -= rint(turn);
    float s, c;
    sincospif(2.0f * (float)turn, &s, &c);
    cs[e] = c * a.factor;
    sn[e] = s * a.factor;
  }
  __syncthreads();
}

// one spelling for both kernels, so that a value does not depend on which of them takes the call
__device__ __forceinline__ void rotate_pair(float& l, float& r, float c, float s) {
  const float x = l, y = r;
  l = fmaf(x, c, -(y * s));
  r = fmaf(y, c, x * s);
}

// VEC kernel: 16-byte vectors of V values.  A lane owns one "unit" of two vectors, (u, u + h) with
// h = rotary_dim/2/V, so that it has both members of its pairs; interleaved pairs and the values
// behind rotary_dim go by two neighbouring vectors.
template <typename T, bool NORM, bool INTERLEAVED>
__global__ void __launch_bounds__(kRotThreads, 4) rotary_vec_kernel(const __grid_constant__ RotaryArgs a) {
  constexpr int V = kVec<T>;
  __shared__ __align__(16) float cs[kRotMaxTokens * kRotMaxPairs], sn[kRotMaxTokens * kRotMaxPairs];
  __shared__ double pos[kRotMaxTokens];
  __shared__ bool live[kRotMaxTokens];
  pdl_launch_dependents();
  pdl_wait();
  const int64_t t0 = (int64_t)blockIdx.x * a.tokens;
  const int n = (int)(a.T - t0 < a.tokens ? a.T - t0 : a.tokens);
  const int lp = a.lanes, u = threadIdx.x & (lp - 1), heads = a.Hq + a.Hkv;
  const int half_vecs = INTERLEAVED ? 0 : a.pairs / V, vecs = a.D / V;
  int v0, v1;
  if (!INTERLEAVED && u < half_vecs) {
    v0 = u;
    v1 = u + half_vecs;
  } else {
    v0 = 2 * u;
    v1 = 2 * u + 1;
  }
  const bool has0 = v0 < vecs, has1 = v1 < vecs;
  uint4 wq0 = make_uint4(0, 0, 0, 0), wq1 = wq0, wk0 = wq0, wk1 = wq0;
  if (NORM) {
    const T *wq = reinterpret_cast<const T*>(a.qw), *wk = reinterpret_cast<const T*>(a.kw);
    if (has0) wq0 = ld_stream16(wq + v0 * V);
    if (has1) wq1 = ld_stream16(wq + v1 * V);
    if (has0 && wk) wk0 = ld_stream16(wk + v0 * V);
    if (has1 && wk) wk1 = ld_stream16(wk + v1 * V);
  }
  fill_table(a, t0, n, cs, sn, pos, live);
  const int items = n * heads, step = kRotThreads / lp;
  for (int it = threadIdx.x / lp; it < ((items + step - 1) / step) * step; it += step) {
    const bool on = it < items;              // the lanes of a warp reduce together
    const int i = on ? it / heads : 0, h = on ? it - i * heads : 0;
    const bool is_k = h >= a.Hq;
    const T* src = is_k ? reinterpret_cast<const T*>(a.k) + (t0 + i) * a.k_tok + (int64_t)(h - a.Hq) * a.k_head
                        : reinterpret_cast<const T*>(a.q) + (t0 + i) * a.q_tok + (int64_t)h * a.q_head;
    uint4 r0 = make_uint4(0, 0, 0, 0), r1 = r0;
    if (on && has0) r0 = ld_stream16(src + v0 * V);
    if (on && has1) r1 = ld_stream16(src + v1 * V);
    const bool rotate = live[i];
    float x0[V], x1[V];
    unpack16<T>(r0, x0);
    unpack16<T>(r1, x1);
    if (NORM) {
      float ss = 0.f;
#pragma unroll
      for (int v = 0; v < V; ++v) ss = fmaf(x0[v], x0[v], fmaf(x1[v], x1[v], ss));
      for (int o = lp / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
      if (rotate) {
        const float inv = 1.0f / sqrtf(ss / (float)a.D + a.eps);
        float w0[V], w1[V];
        const uint4 g0 = is_k ? wk0 : wq0, g1 = is_k ? wk1 : wq1;
        unpack16<T>(g0, w0);
        unpack16<T>(g1, w1);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          x0[v] = x0[v] * inv * w0[v];
          x1[v] = x1[v] * inv * w1[v];
        }
      }
    }
    if (rotate) {
      const float *c = cs + i * a.pairs, *s = sn + i * a.pairs;
      if (!INTERLEAVED) {
        if (u < half_vecs) {
#pragma unroll
          for (int v = 0; v < V; ++v) rotate_pair(x0[v], x1[v], c[u * V + v], s[u * V + v]);
        }
      } else {
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          float(&x)[V] = m ? x1 : x0;
          const int p0 = (m ? v1 : v0) * (V / 2);
          if (p0 < a.pairs) {                // whole vectors: rotary_dim is a multiple of V
#pragma unroll
            for (int v = 0; v < V; v += 2) rotate_pair(x[v], x[v + 1], c[p0 + v / 2], s[p0 + v / 2]);
          }
        }
      }
      r0 = pack16<T>(x0);
      r1 = pack16<T>(x1);
    }
    T* dst = is_k ? reinterpret_cast<T*>(a.ko) + ((t0 + i) * a.Hkv + (h - a.Hq)) * a.D
                  : reinterpret_cast<T*>(a.qo) + ((t0 + i) * a.Hq + h) * a.D;
    if (on && has0) *reinterpret_cast<uint4*>(dst + v0 * V) = r0;
    if (on && has1) *reinterpret_cast<uint4*>(dst + v1 * V) = r1;
  }
}

// Any head size, alignment and stride: one warp per head, one value per lane and access.
template <typename T, bool NORM>
__global__ void __launch_bounds__(kRotThreads) rotary_any_kernel(const __grid_constant__ RotaryArgs a, int interleaved) {
  __shared__ float cs[kRotMaxTokens * kRotMaxPairs], sn[kRotMaxTokens * kRotMaxPairs];
  __shared__ double pos[kRotMaxTokens];
  __shared__ bool live[kRotMaxTokens];
  pdl_launch_dependents();
  pdl_wait();
  const int64_t t0 = (int64_t)blockIdx.x * a.tokens;
  const int n = (int)(a.T - t0 < a.tokens ? a.T - t0 : a.tokens);
  const int lane = threadIdx.x & 31, heads = a.Hq + a.Hkv;
  fill_table(a, t0, n, cs, sn, pos, live);
  for (int it = threadIdx.x >> 5; it < n * heads; it += kRotThreads / 32) {
    const int i = it / heads, h = it - i * heads;
    const bool is_k = h >= a.Hq;
    const T* src = is_k ? reinterpret_cast<const T*>(a.k) + (t0 + i) * a.k_tok + (int64_t)(h - a.Hq) * a.k_head
                        : reinterpret_cast<const T*>(a.q) + (t0 + i) * a.q_tok + (int64_t)h * a.q_head;
    T* dst = is_k ? reinterpret_cast<T*>(a.ko) + ((t0 + i) * a.Hkv + (h - a.Hq)) * a.D
                  : reinterpret_cast<T*>(a.qo) + ((t0 + i) * a.Hq + h) * a.D;
    const T* w = reinterpret_cast<const T*>(is_k ? a.kw : a.qw);
    if (!live[i]) {
      for (int d = lane; d < a.D; d += 32) dst[d] = src[d];
      continue;
    }
    float inv = 1.0f;
    if (NORM) {
      float ss = 0.f;
      for (int d = lane; d < a.D; d += 32) {
        const float x = Elem<T>::to_f(src[d]);
        ss = fmaf(x, x, ss);
      }
      for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
      inv = 1.0f / sqrtf(ss / (float)a.D + a.eps);
    }
    auto value = [&](int d) {
      const float x = Elem<T>::to_f(src[d]);
      return NORM ? x * inv * Elem<T>::to_f(w[d]) : x;
    };
    const float *c = cs + i * a.pairs, *s = sn + i * a.pairs;
    for (int p = lane; p < a.pairs; p += 32) {
      const int d1 = interleaved ? 2 * p : p, d2 = interleaved ? 2 * p + 1 : p + a.pairs;
      float l = value(d1), r = value(d2);
      rotate_pair(l, r, c[p], s[p]);
      dst[d1] = Elem<T>::from_f(l);
      dst[d2] = Elem<T>::from_f(r);
    }
    for (int d = 2 * a.pairs + lane; d < a.D; d += 32) dst[d] = NORM ? Elem<T>::from_f(value(d)) : src[d];
  }
}

template <typename T>
int launch_rotary_t(RotaryArgs& a, bool norm, bool interleaved, cudaStream_t s) {
  constexpr int V = kVec<T>;
  // vectors need whole pairs in a lane's two vectors, and 16-byte rows
  const bool vec = a.D % V == 0 && a.D <= 64 * V && (interleaved ? 2 * a.pairs : a.pairs) % V == 0 && a.q_tok % V == 0 &&
                   a.q_head % V == 0 && aligned16(a.q) && aligned16(a.qo) &&
                   (!a.k || (a.k_tok % V == 0 && a.k_head % V == 0 && aligned16(a.k) && aligned16(a.ko))) &&
                   (!norm || (aligned16(a.qw) && (!a.k || aligned16(a.kw))));
  // one token per CTA while that fills the GPU with CTAs, more after that (the table's set-up is shared)
  int64_t per = a.T / ((int64_t)sm_count() * 8);
  a.tokens = (int)(per < 1 ? 1 : (per > kRotMaxTokens ? kRotMaxTokens : per));
  const int64_t blocks = ceil_div(a.T, a.tokens);
  if (blocks > 0x7FFFFFFFll) return fail(PMX_ERR_UNSUPPORTED, "rotary_embedding: too many tokens");
  const dim3 grid((unsigned)blocks), block(kRotThreads);
  if (vec) {
    const int units = interleaved ? (a.D / V + 1) / 2 : a.pairs / V + (a.D / V - 2 * (a.pairs / V) + 1) / 2;
    a.lanes = 1;
    while (a.lanes < units) a.lanes *= 2;
    if (norm)
      return interleaved ? launch_pdl_k(rotary_vec_kernel<T, true, true>, grid, block, 0, s, a)
                         : launch_pdl_k(rotary_vec_kernel<T, true, false>, grid, block, 0, s, a);
    return interleaved ? launch_pdl_k(rotary_vec_kernel<T, false, true>, grid, block, 0, s, a)
                       : launch_pdl_k(rotary_vec_kernel<T, false, false>, grid, block, 0, s, a);
  }
  return norm ? launch_pdl_k(rotary_any_kernel<T, true>, grid, block, 0, s, a, (int)interleaved)
              : launch_pdl_k(rotary_any_kernel<T, false>, grid, block, 0, s, a, (int)interleaved);
}

}  // namespace

int launch_rotary(const pmx_rotary_args& p, cudaStream_t s) {
  if (!p.query || !p.query_out || !p.frequencies) return fail(PMX_ERR_INVALID_ARGUMENT, "rotary_embedding: null pointer");
  if (p.tokens <= 0 || p.num_heads <= 0 || p.head_dim <= 0 || p.num_kv_heads < 0)
    return fail(PMX_ERR_INVALID_ARGUMENT, "rotary_embedding: tokens, heads and head_dim must be positive");
  if (p.num_heads > (1 << 20) || p.num_kv_heads > (1 << 20) || p.head_dim > (1 << 20) || p.sequences > (1ll << 30))
    return fail(PMX_ERR_UNSUPPORTED, "rotary_embedding: sizes beyond what the kernels index");
  if ((p.num_kv_heads > 0) != (p.key != nullptr) || (p.key && !p.key_out))
    return fail(PMX_ERR_INVALID_ARGUMENT, "rotary_embedding: key, its output and num_kv_heads go together");
  if (!p.position_ids && (!p.seqstarts || !p.start_pos || p.sequences <= 0))
    return fail(PMX_ERR_INVALID_ARGUMENT, "rotary_embedding: positions come from position_ids or from seqstarts and start_pos");
  if (p.rotary_dim <= 0 || p.rotary_dim % 2 || p.rotary_dim > p.head_dim)
    return fail(PMX_ERR_INVALID_ARGUMENT, "rotary_embedding: rotary_dim must be even, positive and at most head_dim");
  if (p.rotary_dim > 2 * kRotMaxPairs) return fail(PMX_ERR_UNSUPPORTED, "rotary_embedding: rotary_dim of at most %d", 2 * kRotMaxPairs);
  if ((p.key_norm_weight != nullptr) != (p.query_norm_weight != nullptr && p.key != nullptr))
    return fail(PMX_ERR_INVALID_ARGUMENT, "rotary_embedding: norm weights are given for query and key, or for neither");
  RotaryArgs a{};
  a.pairs = (int)p.rotary_dim / 2;
  for (int i = 0; i < a.pairs; ++i) a.turns[i] = p.frequencies[i] * 0.15915494309189533577;   // 1 / (2 pi)
  a.q = p.query; a.k = p.key; a.qw = p.query_norm_weight; a.kw = p.key_norm_weight; a.qo = p.query_out; a.ko = p.key_out;
  a.q_tok = p.q_token_stride; a.q_head = p.q_head_stride; a.k_tok = p.k_token_stride; a.k_head = p.k_head_stride;
  a.seqstarts = p.seqstarts; a.start_pos = p.start_pos; a.position_ids = p.position_ids;
  a.T = p.tokens; a.B = (int)p.sequences; a.Hq = (int)p.num_heads; a.Hkv = (int)p.num_kv_heads; a.D = (int)p.head_dim;
  a.eps = (float)p.eps; a.factor = (float)p.factor;
  switch (p.dtype) {
    case PMX_DTYPE_F16: return launch_rotary_t<__half>(a, a.qw != nullptr, p.interleaved != 0, s);
    case PMX_DTYPE_BF16: return launch_rotary_t<__nv_bfloat16>(a, a.qw != nullptr, p.interleaved != 0, s);
    case PMX_DTYPE_F32: return launch_rotary_t<float>(a, a.qw != nullptr, p.interleaved != 0, s);
  }
  return fail(PMX_ERR_UNSUPPORTED, "rotary_embedding: unknown dtype %d", (int)p.dtype);
}

}  // namespace pmx
