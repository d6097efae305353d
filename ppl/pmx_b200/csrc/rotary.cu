// Rotary positions on packed query and key heads, optionally behind an RMS norm of every head.
//
// For a token at position p and pair i of the first `rotary_dim` values of a head, with
// a = p * f_i:  (x1, x2) -> m (x1 cos a - x2 sin a, x2 cos a + x1 sin a);  the pairs are
// (i, i + rotary_dim/2) or, interleaved, (2i, 2i+1); the other values pass through.  With the
// norm, x is first x * w / sqrt(mean over the head of x^2 + eps).  One rounding, at the store.
//
// Bound by the bytes of the heads, read once and written once, if an element costs few instructions and the loads
// never pause.  A warp walks the heads of a run of tokens: its loads go several steps ahead, across heads and tokens,
// into a ring in shared memory (every lane reads back what it fetched itself, so nothing waits for other lanes); the
// cosines and sines of a token are made once, by the warp, and stay in registers for all its heads, with the norm's
// weights multiplied in; the norm's sum stays inside the lanes that hold the head; products go two to an instruction.
// On B200, 16 k tokens of 40 heads of 128 with the norm: 60 us, 5.5 TB/s, 85 % of the measured copy rate.  One token a warp without the ring took 72 us,
// one thread per vector pair with a table per CTA 104 us (barriers and per-thread index arithmetic).
// The angle is taken in turns, p * f_i / (2 pi), in 64 bits, and only its distance to the nearest whole turn goes on
// in 32 bits, so far positions keep the precision of near ones (in 32 bits p = 10^6 would be off by 0.06 rad).
#include <type_traits>

#include "common.cuh"
#include "packed_f32.cuh"

namespace pmx {
namespace {

constexpr int kRotWarps = 4;
constexpr int kRotMaxPairs = 128;
constexpr int kRotRing = 4;           // steps of a warp's ring: 3 KB of loads under way
constexpr int kRotWarpsPerSm = 16;    // 60 us in the case above; 12: 75, 20: 69, 24 (spills): 81; a ring of 6: 62

struct RotaryArgs {
  double turns[kRotMaxPairs];         // f_i / (2 pi)
  const void *q, *k;                  // [T, Hq, D], [T, Hkv, D] with strides; k may be null (Hkv = 0)
  const void *qw, *kw;                // [D] norm weights, or null
  void *qo, *ko;                      // dense
  int64_t q_tok, q_head, k_tok, k_head;
  const int64_t *seqstarts, *start_pos, *position_ids;
  int64_t T;
  int B, Hq, Hkv, D, pairs;
  int tokens, chunks, chunk_heads;    // tokens of a warp; warps that share a token's heads, heads of each
  int lanes;                          // vector kernel: lanes per head, a power of two
  float eps, factor, per_head;        // per_head: 1 / D
};

// The positions of consecutive tokens, for a whole warp.  A token's sequence is the number of starts at or before
// it, counted by the lanes side by side: one memory latency where a binary search would pay one per level.  Inside the
// sequence the position counts on.
struct Positions {
  int64_t pos, end;                   // of the last token asked for; the first token that needs a look-up
  bool live;                          // whether the token belongs to a sequence
  __device__ __forceinline__ void start() { end = -1; }
  __device__ __forceinline__ void at(const RotaryArgs& a, int64_t t) {
    if (a.position_ids) {
      pos = __ldcg(a.position_ids + t);
      live = true;
      return;
    }
    if (t < end) {
      ++pos;
      return;
    }
    int before = 0;
    for (int i = threadIdx.x & 31; i <= a.B; i += 32) before += __ldcg(a.seqstarts + i) <= t ? 1 : 0;
    const int b = __reduce_add_sync(0xFFFFFFFFu, before) - 1;
    live = b >= 0 && b < a.B;
    pos = live ? __ldcg(a.start_pos + b) + (t - __ldcg(a.seqstarts + b)) : 0;
    end = live ? __ldcg(a.seqstarts + b + 1) : t + 1;
  }
};

// Fills the warp's table of cosines and sines for position p.
__device__ __forceinline__ void fill_table(const RotaryArgs& a, int64_t p, float* cs, float* sn) {
  const double pos = (double)p;
  __syncwarp();                       // the table of the token before is read
  for (int j = threadIdx.x & 31; j < a.pairs; j += 32) {
    double turn = pos * a.turns[j];
    turn -= rint(turn);
    float s, c;
    sincospif(2.0f * (float)turn, &s, &c);
    cs[j] = c * a.factor;
    sn[j] = s * a.factor;
  }
  __syncwarp();
}

// Spelt as in the vector kernel: without a norm a value's bits do not depend on which of the two takes the call.  (With one they
// may, by roundings in 32 bits: the vector kernel multiplies the weights into the coefficients.)
__device__ __forceinline__ void rotate_pair(float& l, float& r, float c, float s) {
  const float x = l, y = r;
  l = fmaf(x, c, -(y * s));
  r = fmaf(y, c, x * s);
}

// a 16-byte vector as V/2 pairs, and back with one rounding each
template <typename T>
__device__ __forceinline__ void unpack_pairs(const uint4& v, f32x2 (&x)[kVec<T> / 2]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < kVec<T> / 2; ++i) {
    if constexpr (std::is_same<T, float>::value) {
      x[i] = pair2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      x[i] = pair2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[i] = pair2(f.x, f.y);
    }
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack_pairs(const f32x2 (&x)[kVec<T> / 2]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < kVec<T> / 2; ++i) {
    float lo, hi;
    unpair2(x[i], lo, hi);
    if constexpr (std::is_same<T, float>::value) {
      w[2 * i] = __float_as_uint(lo);
      w[2 * i + 1] = __float_as_uint(hi);
    } else if constexpr (std::is_same<T, __half>::value) {
      const __half2 h = __floats2half2_rn(lo, hi);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ void rot_fetch16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// 16-byte vectors of V values.  A lane owns two vectors of a head that hold complete pairs: (u, u + rotary_dim/2/V), or, for
// interleaved pairs and for the values behind rotary_dim, any two (half of what is there apart).  A step takes
// as many heads as the warp's lanes hold; query heads and key heads take steps of their own.
template <typename T, bool NORM, bool INTERLEAVED>
__global__ void __launch_bounds__(kRotWarps * 32, kRotWarpsPerSm / kRotWarps) rotary_vec_kernel(const __grid_constant__ RotaryArgs a) {
  constexpr int V = kVec<T>, W = V / 2;
  __shared__ __align__(16) uint4 ring[kRotWarps][kRotRing][2][32];
  __shared__ __align__(16) float table[kRotWarps][2][kRotMaxPairs];
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t ta = ((int64_t)blockIdx.x * kRotWarps + warp) * a.tokens;
  if (ta >= a.T) return;
  const int64_t tb = a.T - ta < a.tokens ? a.T : ta + a.tokens;
  const int h0 = blockIdx.y * a.chunk_heads, h1 = min(h0 + a.chunk_heads, a.Hq + a.Hkv);
  const int lp = a.lanes, u = lane & (lp - 1), step = 32 / lp, g = lane / lp;
  // neighbouring lanes take neighbouring vectors: whole sectors per access
  const int half_vecs = INTERLEAVED ? 0 : a.pairs / V, vecs = a.D / V, rest = (vecs - 2 * half_vecs + 1) / 2;
  const bool split = u < half_vecs;
  const int v0 = split ? u : half_vecs + u, v1 = split ? u + half_vecs : v0 + rest;
  const bool has0 = split || u < half_vecs + rest, has1 = has0 && v1 < vecs;
  const int nq = max(0, min(h1, a.Hq) - h0), k_first = max(h0, a.Hq) - a.Hq, nk = max(0, h1 - a.Hq - k_first);
  const int q_steps = (nq + step - 1) / step, steps = q_steps + (nk + step - 1) / step;

  // ---- the loads: one step further every time `fetch` is called
  const T *q_next = reinterpret_cast<const T*>(a.q) + ta * a.q_tok + (int64_t)(h0 + g) * a.q_head;
  const T *k_next = reinterpret_cast<const T*>(a.k) + ta * a.k_tok + (int64_t)(k_first + g) * a.k_head;
  const int64_t q_step = (int64_t)step * a.q_head, k_step = (int64_t)step * a.k_head;
  int64_t fetch_t = ta;
  int fetch_s = 0;
  const T* fetch_at = q_steps ? q_next : k_next;
  uint32_t my_ring = static_cast<uint32_t>(__cvta_generic_to_shared(&ring[warp][0][0][lane]));
  auto fetch = [&](int slot) {
    if (fetch_t < tb) {
      const bool is_k = fetch_s >= q_steps;
      const bool on = is_k ? (fetch_s - q_steps) * step + g < nk : fetch_s * step + g < nq;
      const uint32_t dst = my_ring + slot * 1024;
      if (on && has0) rot_fetch16(dst, fetch_at + v0 * V);
      if (on && has1) rot_fetch16(dst + 512, fetch_at + v1 * V);
      fetch_at += is_k ? k_step : q_step;
      if (++fetch_s == q_steps) fetch_at = k_next;
      if (fetch_s == steps) {
        fetch_s = 0;
        ++fetch_t;
        q_next += a.q_tok;
        k_next += a.k_tok;
        fetch_at = q_steps ? q_next : k_next;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kRotRing - 1; ++i) fetch(i);

  const bool rot0 = INTERLEAVED ? v0 * W < a.pairs : split, rot1 = INTERLEAVED ? v1 * W < a.pairs : split;
  // y0 = x0 * a0 + z0 * b0,  y1 = x1 * a1 + z1 * b1, with z the other member of each value's pair
  f32x2 a0[W], b0[W], a1[W], b1[W];
  auto coefficients = [&](const void* weight) {
    const float *c = table[warp][0] + (INTERLEAVED ? v0 * W : u * V), *s = table[warp][1] + (INTERLEAVED ? v0 * W : u * V);
    const int far = (v1 - v0) * W;            // interleaved: from the first vector's pairs to the second's
#pragma unroll
    for (int i = 0; i < W; ++i) {
      if (!INTERLEAVED) {
        a0[i] = a1[i] = rot0 ? pair2(c[2 * i], c[2 * i + 1]) : pair2(1.f, 1.f);
        b1[i] = rot0 ? pair2(s[2 * i], s[2 * i + 1]) : pair2(0.f, 0.f);
        b0[i] = mul2(b1[i], pair2(-1.f, -1.f));
      } else {
        a0[i] = rot0 ? pair2(c[i], c[i]) : pair2(1.f, 1.f);
        b0[i] = rot0 ? pair2(-s[i], s[i]) : pair2(0.f, 0.f);
        a1[i] = rot1 ? pair2(c[far + i], c[far + i]) : pair2(1.f, 1.f);
        b1[i] = rot1 ? pair2(-s[far + i], s[far + i]) : pair2(0.f, 0.f);
      }
    }
    if (NORM) {
      f32x2 w0[W], w1[W];
      const T* w = reinterpret_cast<const T*>(weight);
      unpack_pairs<T>(has0 ? ld_nc16(w + v0 * V) : make_uint4(0, 0, 0, 0), w0);
      unpack_pairs<T>(has1 ? ld_nc16(w + v1 * V) : make_uint4(0, 0, 0, 0), w1);
#pragma unroll
      for (int i = 0; i < W; ++i) {
        a0[i] = mul2(a0[i], w0[i]);
        a1[i] = mul2(a1[i], w1[i]);
        if (!INTERLEAVED) {
          b0[i] = mul2(b0[i], w1[i]);
          b1[i] = mul2(b1[i], w0[i]);
        } else {
          float l, r;
          unpair2(w0[i], l, r);
          b0[i] = mul2(b0[i], pair2(r, l));
          unpair2(w1[i], l, r);
          b1[i] = mul2(b1[i], pair2(r, l));
        }
      }
    }
  };

  // ---- the heads, in the order of the loads
  Positions where;
  where.start();
  int slot = 0;
  for (int64_t t = ta; t < tb; ++t) {
    where.at(a, t);
    fill_table(a, where.pos, table[warp][0], table[warp][1]);
    const bool live = where.live;
    T* at = q_steps ? reinterpret_cast<T*>(a.qo) + (t * a.Hq + h0 + g) * a.D
                    : reinterpret_cast<T*>(a.ko) + (t * a.Hkv + k_first + g) * a.D;
    if (q_steps) coefficients(a.qw);
    for (int i = 0; i < steps; ++i) {
      const bool is_k = i >= q_steps;
      if (i == q_steps) {
        at = reinterpret_cast<T*>(a.ko) + (t * a.Hkv + k_first + g) * a.D;
        if (NORM || !q_steps) coefficients(a.kw);
      }
      const bool on = is_k ? (i - q_steps) * step + g < nk : i * step + g < nq;
      asm volatile("cp.async.wait_group %0;" ::"n"(kRotRing - 2) : "memory");
      const uint4 raw0 = ring[warp][slot][0][lane], raw1 = ring[warp][slot][1][lane];
      fetch(slot == 0 ? kRotRing - 1 : slot - 1);        // the slot of the step before
      if (++slot == kRotRing) slot = 0;
      uint4 out0 = raw0, out1 = raw1;
      if (NORM || rot0) {
        f32x2 x0[W], x1[W], y0[W], y1[W];
        unpack_pairs<T>(raw0, x0);
        unpack_pairs<T>(raw1, x1);
        if (NORM) {
          // a unit's vectors behind the head's end hold nothing: their share of the sum is left out
          f32x2 s0 = mul2(x0[0], x0[0]), s1 = mul2(x1[0], x1[0]);
#pragma unroll
          for (int j = 1; j < W; ++j) {
            s0 = fma2(x0[j], x0[j], s0);
            s1 = fma2(x1[j], x1[j], s1);
          }
          float p, q, v, w;
          unpair2(s0, p, q);
          unpair2(s1, v, w);
          float ss = (has0 ? p + q : 0.f) + (has1 ? v + w : 0.f);
          for (int o = lp / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
          const float inv = rsqrtf(fmaf(ss, a.per_head, a.eps));
          const f32x2 inv2 = pair2(inv, inv);
#pragma unroll
          for (int j = 0; j < W; ++j) {
            x0[j] = mul2(x0[j], inv2);
            x1[j] = mul2(x1[j], inv2);
          }
        }
        // values that do not rotate take nothing from their neighbours, not even 0 * NaN
#pragma unroll
        for (int j = 0; j < W; ++j) {
          f32x2 z0, z1;
          if (!INTERLEAVED) {
            z0 = x1[j];
            z1 = x0[j];
          } else {
            float l, r;
            unpair2(x0[j], l, r);
            z0 = pair2(r, l);
            unpair2(x1[j], l, r);
            z1 = pair2(r, l);
          }
          if (NORM) {
            y0[j] = mul2(x0[j], a0[j]);
            y1[j] = mul2(x1[j], a1[j]);
            if (rot0) y0[j] = fma2(z0, b0[j], y0[j]);
            if (rot1) y1[j] = fma2(z1, b1[j], y1[j]);
          } else {
            y0[j] = fma2(x0[j], a0[j], mul2(z0, b0[j]));
            y1[j] = fma2(x1[j], a1[j], mul2(z1, b1[j]));
          }
        }
        if (live) {                           // a token of no sequence is copied
          out0 = pack_pairs<T>(y0);
          if (NORM || rot1) out1 = pack_pairs<T>(y1);
        }
      }
      if (on && has0) *reinterpret_cast<uint4*>(at + v0 * V) = out0;
      if (on && has1) *reinterpret_cast<uint4*>(at + v1 * V) = out1;
      at += step * a.D;
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// Any head size, alignment and stride: the lanes of a warp share a head's values out one by one.
template <typename T, bool NORM>
__global__ void __launch_bounds__(kRotWarps * 32) rotary_any_kernel(const __grid_constant__ RotaryArgs a, int interleaved) {
  __shared__ float table[kRotWarps][2][kRotMaxPairs];
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t ta = ((int64_t)blockIdx.x * kRotWarps + warp) * a.tokens;
  if (ta >= a.T) return;
  const int64_t tb = a.T - ta < a.tokens ? a.T : ta + a.tokens;
  const int h0 = blockIdx.y * a.chunk_heads, h1 = min(h0 + a.chunk_heads, a.Hq + a.Hkv);
  const float *c = table[warp][0], *s = table[warp][1];
  Positions where;
  where.start();
  for (int64_t t = ta; t < tb; ++t) {
    where.at(a, t);
    fill_table(a, where.pos, table[warp][0], table[warp][1]);
    for (int h = h0; h < h1; ++h) {
      const bool is_k = h >= a.Hq;
      const T* src = is_k ? reinterpret_cast<const T*>(a.k) + t * a.k_tok + (int64_t)(h - a.Hq) * a.k_head
                          : reinterpret_cast<const T*>(a.q) + t * a.q_tok + (int64_t)h * a.q_head;
      T* dst = is_k ? reinterpret_cast<T*>(a.ko) + (t * a.Hkv + (h - a.Hq)) * a.D
                    : reinterpret_cast<T*>(a.qo) + (t * a.Hq + h) * a.D;
      const T* w = reinterpret_cast<const T*>(is_k ? a.kw : a.qw);
      if (!where.live) {
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
        inv = rsqrtf(fmaf(ss, a.per_head, a.eps));
      }
      auto value = [&](int d) {
        const float x = Elem<T>::to_f(src[d]);
        return NORM ? x * inv * Elem<T>::to_f(w[d]) : x;
      };
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
}

template <typename T>
int launch_rotary_t(RotaryArgs& a, bool norm, bool interleaved, cudaStream_t s) {
  constexpr int V = kVec<T>;
  // vectors need whole pairs in a lane's two vectors, and 16-byte rows
  const bool vec = a.D % V == 0 && a.D <= 64 * V && (interleaved ? 2 * a.pairs : a.pairs) % V == 0 && a.q_tok % V == 0 &&
                   a.q_head % V == 0 && aligned16(a.q) && aligned16(a.qo) &&
                   (!a.k || (a.k_tok % V == 0 && a.k_head % V == 0 && aligned16(a.k) && aligned16(a.ko))) &&
                   (!norm || (aligned16(a.qw) && (!a.k || aligned16(a.kw))));
  a.lanes = 1;
  if (vec) {
    const int half = interleaved ? 0 : a.pairs / V, units = half + (a.D / V - 2 * half + 1) / 2;
    while (a.lanes < units) a.lanes *= 2;
  }
  // Few tokens: the heads of a token are cut into pieces of whole steps until there is a warp for every SM's slots.
  // Many: every warp takes an equal run of tokens, so that all warps of the GPU start and end together.
  const int64_t slots = (int64_t)sm_count() * kRotWarpsPerSm;
  const int heads = a.Hq + a.Hkv, step = vec ? 32 / a.lanes : 1;
  const int64_t want = slots / a.T < 1 ? 1 : slots / a.T, most = ceil_div(heads, step);
  a.chunks = (int)(want < most ? want : most);
  a.chunk_heads = (int)ceil_div(ceil_div(heads, a.chunks), step) * step;
  a.chunks = (int)ceil_div(heads, a.chunk_heads);
  a.per_head = 1.0f / (float)a.D;
  const int64_t run = ceil_div(a.T * a.chunks, slots), blocks = ceil_div(ceil_div(a.T, run), kRotWarps);
  if (run > 0x7FFFFFFFll || a.chunks > 65535) return fail(PMX_ERR_UNSUPPORTED, "rotary_embedding: too many tokens or heads");
  a.tokens = (int)run;
  const dim3 grid((unsigned)blocks, (unsigned)a.chunks), block(kRotWarps * 32);
  if (vec) {
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
