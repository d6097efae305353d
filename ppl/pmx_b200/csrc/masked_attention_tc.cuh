// The tensor-core kernel of masked_attention.cu (included there, inside its namespaces): 16-bit tensors, head
// sizes up to 128.
//
// A CTA computes one or two tiles of 128 rows against the keys of their sequence, 128 at a time.  A row is a
// (query token, query head) of ONE key head: the G query heads that share it are packed into the tile
// (128 / G tokens of them), so each key and value crosses to the SM once for the whole group.
//   warp 8   TMA: keys and values through a ring of 128-row buffers (128-byte swizzle)
//   warp 9   one thread issues the tcgen05 products: S_w = Q_w K^T into tensor memory columns [128 w, +128),
//            O_w += P_w V into columns [256 + 128 w, +128); P_w is read from tensor memory, V is the MN-major operand
//   warps 0-3 and 4-7  the softmax of S_0 and S_1, one thread per row (a thread owns a tensor memory lane, so the
//            row's maximum and sum need no exchange); P_w overwrites S_w in 16 bits
//   warps 10, 11  go over those value tiles of which some rows see a part only
// With more than 128 rows (PAIR) the two tiles share the keys; with fewer, both softmax halves work on the same
// rows, on the even and the odd key tiles, and meet at the end: either way one half's softmax runs
// beside the other's products.  The running maximum moves only when a row's new maximum lies more than 2^8
// above it, so that O in tensor memory is rescaled rarely; probabilities stay below 2^8, exact in the 16-bit types'
// range, and the sum divides the same scale out again.
// Few rows and many keys: the key tiles are dealt out over several CTAs, whose partial results (fp32, with maximum
// and sum) a second kernel merges.
//
// A masked score becomes -inf whatever the product holds.  A masked VALUE needs more: 0 * inf and 0 * NaN are NaN in
// the second product, so in the tiles that are not seen whole by every row, values that are not finite are replaced by
// zeros in shared memory, and if there were any among the sequence's own, the epilogue adds them back for the rows
// that see them.
constexpr int kTile = 128;                  // keys of a tile, rows of a tile
constexpr int kRing = 5;                    // ring buffers: two keys and two values in use, one on the way
constexpr int kAttnThreads = 384;
constexpr int kMaxSplits = 32;
constexpr float kLazy = 8.0f;               // log2 of how far a maximum may run ahead
constexpr unsigned long long kAttnWaitNs = 2000000000ull;

__device__ int g_attention_status[4];       // record of a bounded wait that ran out: code, role, tile, CTA

struct TileMaps {
  CUtensorMap q, k, v, ck, cv;              // ck, cv: the drafted tokens' (trees only)
};

struct TcArgs {
  AttnArgs a;
  float* part_o;                            // [splits][Tq * Hq][D]
  float2* part_ml;                          // [splits][Tq * Hq] maximum (log2), sum
  int group, tokens;                        // query heads per key head, tokens of a row tile
  int row_blocks, splits, pair, zero_ctas;
};

struct Ctl {
  uint64_t full[kRing], empty[kRing], raw[kRing];
  uint64_t q_full, s_full[2], p_ready[2], o_full[2];
  uint32_t tmem;
  volatile int abort;
  int any_bad;
};

__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, Ctl* c, int role, int tile) {
  if (mbar_try_wait(bar, parity)) return true;
  const unsigned long long t0 = global_ns();
  for (uint32_t it = 1;; ++it) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((it & 63u) == 0u) {
      if (c->abort) return false;
      if (global_ns() - t0 > kAttnWaitNs) {
        c->abort = 1;
        if (atomicExch(&g_attention_status[0], 1) != 1) {
          g_attention_status[1] = role;
          g_attention_status[2] = tile;
          g_attention_status[3] = (int)blockIdx.x;
        }
        return false;
      }
    }
  }
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem desc]
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Shared-memory descriptor of an MN-major operand: rows (K) of 64 values = 128 bytes with the 128-byte swizzle, 8-row
// groups 1024 bytes apart; the next 64 values of MN are a 128-row block further.
__device__ __forceinline__ uint64_t smem_desc_mn(uint32_t saddr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr >> 4) & 0x3FFF);
  d |= static_cast<uint64_t>((kTile * 128) >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}
// 32 lanes x 32 consecutive 32-bit columns
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void named_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ void named_arrive(int id, int threads) {
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ bool named_any(int id, int threads, bool v) {
  int r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.s32 p, %3, 0;\n\t"
      "bar.red.or.pred q, %1, %2, p;\n\t"
      "selp.s32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(id), "r"(threads), "r"((int)v)
      : "memory");
  return r != 0;
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// exponent bits all ones in either half of a word: the add carries into the sign bit, and no further
template <typename T>
__device__ __forceinline__ uint32_t not_finite2(uint32_t w) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return ((w & 0x7F807F80u) + 0x00800080u) & 0x80008000u;
  return ((w & 0x7C007C00u) + 0x04000400u) & 0x80008000u;
}

// the share of the key tiles that one CTA takes, and what its rows see
struct Work {
  int b, h, x, split;
  Sequence s;
  int tok0;            // first token of the CTA's rows, in the sequence
  int halves;          // row tiles in use (1 without PAIR)
  int t0, nt[2];       // first key tile; tiles of each row tile (without PAIR: nt[0] is the CTA's)
  int drafted;         // index of the drafted tokens' tile, -1: none
  int partial;         // first tile that some row does not see whole
};

__device__ __forceinline__ Work make_work(const TcArgs& p, int idx) {
  Work w;
  const AttnArgs& a = p.a;
  // row blocks that see the most keys first
  const int per = a.B * a.Hkv * p.splits;
  w.x = p.row_blocks - 1 - idx / per;
  idx %= per;
  w.split = idx % p.splits;
  idx /= p.splits;
  w.h = idx % a.Hkv;
  w.b = idx / a.Hkv;
  w.s = load_sequence(a, w.b);
  const int block_tokens = p.pair ? 2 * p.tokens : p.tokens;
  w.tok0 = w.x * block_tokens;
  w.halves = 0;
  w.drafted = -1;
  w.t0 = w.nt[0] = w.nt[1] = w.partial = 0;
  if (w.tok0 >= w.s.n) return w;
  w.halves = p.pair && w.tok0 + p.tokens < w.s.n ? 2 : 1;
  int total[2];
  const int64_t first = visible(a, w.s, w.tok0);
  w.partial = (int)(first / kTile);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int last = w.tok0 + (i + 1) * p.tokens - 1;
    const int64_t seen = visible(a, w.s, last < w.s.n ? last : w.s.n - 1);
    total[i] = (int)((seen + kTile - 1) / kTile);
    if (a.tree_mask) w.drafted = total[i]++;
  }
  if (w.halves == 1) total[1] = total[0];
  // contiguous shares of the longer row tile's key tiles
  const int share = (total[1] + p.splits - 1) / p.splits;
  w.t0 = w.split * share < total[1] ? w.split * share : total[1];
  const int t1 = w.t0 + share < total[1] ? w.t0 + share : total[1];
  w.nt[0] = (total[0] < t1 ? total[0] : t1) - w.t0;
  if (w.nt[0] < 0) w.nt[0] = 0;
  w.nt[1] = w.halves == 2 ? t1 - w.t0 : 0;
  return w;
}

// rows of a key tile that hold keys of the sequence
__device__ __forceinline__ int tile_rows(const Work& w, int t) {
  if (t == w.drafted) return w.s.n;
  const int64_t left = w.s.len - (int64_t)t * kTile;
  return (int)(left < kTile ? left : kTile);
}

template <typename T, int DP, bool SCORE>
__global__ void __launch_bounds__(kAttnThreads, 1)
masked_attention_kernel(const __grid_constant__ TileMaps maps, const __grid_constant__ TcArgs p) {
  constexpr int kTileBytes = kTile * DP * 2;
  constexpr int kBlockBytes = kTile * 128;          // 64 columns of a tile
  constexpr int kDBlocks = DP / 64;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Ctl* ctl = reinterpret_cast<Ctl*>(smem + (2 + kRing) * kTileBytes);
  const AttnArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_launch_dependents();
  pdl_wait();
  const int work_ctas = p.row_blocks * a.B * a.Hkv * p.splits;
  if ((int)blockIdx.x >= work_ctas) {
    // rows of no sequence: zeros, or partial results that count for nothing
    const int64_t lo = clamp64(__ldcg(a.seqstarts), 0, a.Tq), hi = clamp64(__ldcg(a.seqstarts + a.B), lo, a.Tq);
    const int64_t rows = (lo + a.Tq - hi) * a.Hq, step = (int64_t)p.zero_ctas * (kAttnThreads / 32);
    for (int64_t r = ((int64_t)blockIdx.x - work_ctas) * (kAttnThreads / 32) + warp; r < rows; r += step) {
      const int64_t row = r < lo * a.Hq ? r : r + (hi - lo) * a.Hq;
      if (p.splits == 1) {
        T* out = reinterpret_cast<T*>(a.out) + row * a.D;
        for (int d = lane; d < a.D; d += 32) out[d] = Elem<T>::from_f(0.f);
      } else if (lane < p.splits) {
        p.part_ml[(int64_t)lane * a.Tq * a.Hq + row] = make_float2(-INFINITY, 0.f);
      }
    }
    return;
  }
  const Work w = make_work(p, (int)blockIdx.x);
  if (w.halves == 0) return;
  // without PAIR the two softmax halves take turns on the CTA's tiles
  const int total = p.pair ? (w.nt[1] > w.nt[0] ? w.nt[1] : w.nt[0]) : w.nt[0];
  const int rows_tile = p.tokens * p.group;
  // the row of a softmax thread
  const int half = warp >> 2, r = threadIdx.x & 127;
  const int tok = w.tok0 + (p.pair ? half * p.tokens : 0) + r / p.group;
  const bool row_ok = warp < 8 && r < rows_tile && tok < w.s.n;
  const int head = w.h * p.group + r % p.group;
  const int64_t out_row = (w.s.q0 + tok) * a.Hq + head;
  if (a.tree_mask && w.x == 0 && w.split == 0) {
    // the sequence's new keys and values go into the cache, where this launch does not read them
    for (int i = threadIdx.x; i < w.s.n * (a.D / 8) * 2; i += kAttnThreads) {
      const int ch = i % (a.D / 8), kv = i / (a.D / 8) & 1, t = i / (a.D / 8) >> 1;
      const int64_t row = w.s.kv0 + w.s.len + t;
      if (row >= a.past.rows) continue;
      const T* src = kv ? reinterpret_cast<const T*>(a.cur.v) + (w.s.q0 + t) * a.cur.v_row + w.h * a.cur.v_head
                        : reinterpret_cast<const T*>(a.cur.k) + (w.s.q0 + t) * a.cur.k_row + w.h * a.cur.k_head;
      T* dst = kv ? reinterpret_cast<T*>(const_cast<void*>(a.past.v)) + row * a.past.v_row + w.h * a.past.v_head
                  : reinterpret_cast<T*>(const_cast<void*>(a.past.k)) + row * a.past.k_row + w.h * a.past.k_head;
      *reinterpret_cast<uint4*>(dst + ch * 8) = ld_stream16(src + ch * 8);
    }
  }
  if (total == 0) {
    if (row_ok && (p.pair || half == 0)) {
      if (p.splits == 1) {
        T* out = reinterpret_cast<T*>(a.out) + out_row * a.D;
        for (int d = 0; d < a.D; d += 8) *reinterpret_cast<uint4*>(out + d) = make_uint4(0, 0, 0, 0);
      } else {
        p.part_ml[(int64_t)w.split * a.Tq * a.Hq + out_row] = make_float2(-INFINITY, 0.f);
      }
    }
    return;
  }

  if (threadIdx.x == 0) {
    for (int i = 0; i < kRing; ++i) {
      mbar_init(&ctl->full[i], 1);
      mbar_init(&ctl->empty[i], 1);
      mbar_init(&ctl->raw[i], 1);
    }
    mbar_init(&ctl->q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ctl->s_full[i], 1);
      mbar_init(&ctl->p_ready[i], 4);
      mbar_init(&ctl->o_full[i], 1);
    }
    ctl->abort = 0;
    ctl->any_bad = 0;
    fence_barrier_init();
  }
  if (warp == 9) {
    tmem_alloc(&ctl->tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl->tmem;
  const uint32_t q_addr = smem_u32(smem), ring = q_addr + 2 * kTileBytes;
  // Order of the ring: the keys of the first `lag` tiles, then values and keys in turn.  Entry of the values of tile i:
  const int lag = p.pair ? 1 : 2;
  auto v_entry = [&](int i) { return 2 * i + lag < total + i ? 2 * i + lag : total + i; };

  // The softmax warpgroups hold a row of scores in registers; the third one needs few.  216 x 256 + 56 x 128 =
  // 62464 of the 168 x 384 = 64512 registers that the block starts with.
  if (warp >= 8) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
  if (warp == 8) {
    // ------------------------------------------------------------------ TMA
    if (lane == 0) {
      prefetch_tensormap(&maps.k);
      prefetch_tensormap(&maps.v);
      mbar_expect_tx(&ctl->q_full, (uint32_t)(w.halves * kDBlocks * 128 * rows_tile));
      for (int i = 0; i < w.halves; ++i)
        for (int d = 0; d < kDBlocks; ++d)
          tma_load_3d(q_addr + i * kTileBytes + d * kBlockBytes, &maps.q, &ctl->q_full, d * 64, w.h * p.group,
                      (int)w.s.q0 + w.tok0 + i * p.tokens);
      int slot = 0;
      uint32_t phase = 0;
      bool ok = true;
      auto load = [&](int i, bool values) {
        ok = wait_bar(&ctl->empty[slot], phase ^ 1u, ctl, 0, i);
        if (!ok) return;
        const int t = w.t0 + i;
        const bool draft = t == w.drafted;
        uint64_t* bar = values && t >= w.partial ? &ctl->raw[slot] : &ctl->full[slot];
        const CUtensorMap* map = draft ? (values ? &maps.cv : &maps.ck) : (values ? &maps.v : &maps.k);
        const int row = draft ? (int)w.s.q0 : (int)w.s.kv0 + t * kTile;
        mbar_expect_tx(bar, (uint32_t)(kDBlocks * 128 * (draft ? kTreeLimit : kTile)));
        for (int d = 0; d < kDBlocks; ++d)
          tma_load_3d(ring + slot * kTileBytes + d * kBlockBytes, map, bar, d * 64, w.h, row);
        if (++slot == kRing) { slot = 0; phase ^= 1u; }
      };
      for (int i = 0; i < lag && i < total && ok; ++i) load(i, false);
      for (int i = 0; i < total && ok; ++i) {
        load(i, true);
        if (ok && i + lag < total) load(i + lag, false);
      }
      if (!ok) {      // leave the copies in flight the time to land
        const unsigned long long t0 = global_ns();
        while (global_ns() - t0 < 1000000ull) __nanosleep(1000);
      }
    }
  } else if (warp == 9) {
    // ------------------------------------------------------------------ products
    if (lane == 0) {
      const uint32_t idesc_s = make_idesc<T>(128, 128), idesc_d = make_idesc<T>(128, kTreeLimit);
      const uint32_t idesc_o = make_idesc<T>(128, DP) | (1u << 16);      // B is MN-major
      int slot = 0;
      uint32_t phase = 0, p_phase[2] = {0, 0};
      bool ok = wait_bar(&ctl->q_full, 0, ctl, 1, 0);
      auto next = [&]() { if (++slot == kRing) { slot = 0; phase ^= 1u; } };
      auto scores = [&](int q, int i) {             // row tile q and half: S = Q K_i^T from the current slot
        const uint32_t ka = ring + slot * kTileBytes, qa = q_addr + (p.pair ? q : 0) * kTileBytes;
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
          const uint32_t off = (kk / 4) * kBlockBytes + (kk % 4) * 32;
          umma_f16(tmem + q * 128, smem_desc_sw128(qa + off), smem_desc_sw128(ka + off),
                   w.t0 + i == w.drafted ? idesc_d : idesc_s, kk > 0 ? 1u : 0u);
        }
        umma_commit(&ctl->s_full[q]);
      };
      auto output = [&](int q, int i, bool first) { // O += P V_i from the current slot
        const uint32_t va = ring + slot * kTileBytes;
        const int steps = (tile_rows(w, w.t0 + i) + 15) / 16;
        for (int kk = 0; kk < steps; ++kk)
          umma_f16_ts(tmem + 256 + q * 128, tmem + q * 128 + kk * 8, smem_desc_mn(va + kk * 2048), idesc_o,
                      !first || kk > 0 ? 1u : 0u);
      };
      auto wait_p = [&](int q, int i) {
        ok = wait_bar(&ctl->p_ready[q], p_phase[q], ctl, 3, i);
        p_phase[q] ^= 1u;
        tc_fence_after();
      };
      auto wait_full = [&](int i) {
        ok = wait_bar(&ctl->full[slot], phase, ctl, 2, i);
        tc_fence_after();
      };
      if (!p.pair) {
        for (int i = 0; i < 2 && i < total && ok; ++i) {
          wait_full(i);
          if (!ok) break;
          scores(i, i);
          umma_commit(&ctl->empty[slot]);
          next();
        }
        for (int i = 0; i < total && ok; ++i) {
          const int q = i & 1;
          wait_full(i);
          if (ok) wait_p(q, i);
          if (!ok) break;
          output(q, i, i < 2);
          umma_commit(&ctl->empty[slot]);
          next();
          if (i + 2 < total) {
            wait_full(i + 2);
            if (!ok) break;
            scores(q, i + 2);
            umma_commit(&ctl->empty[slot]);
            next();
          } else {
            umma_commit(&ctl->o_full[q]);
          }
        }
      } else {
        if (ok) wait_full(0);
        if (ok) {
          for (int q = 0; q < 2; ++q)
            if (w.nt[q] > 0) scores(q, 0);
          umma_commit(&ctl->empty[slot]);
          next();
        }
        for (int i = 0; i < total && ok; ++i) {
          // the current slot holds V_i, the one behind it K_i+1
          wait_full(i);
          if (!ok) break;
          const int v_slot = slot;
          const uint32_t v_phase = phase;
          next();
          const int k_slot = slot;
          const uint32_t k_phase = phase;
          for (int q = 0; q < 2 && ok; ++q) {
            if (i >= w.nt[q]) continue;
            wait_p(q, i);
            if (!ok) break;
            slot = v_slot; phase = v_phase;
            output(q, i, i == 0);
            slot = k_slot; phase = k_phase;
            if (i + 1 < w.nt[q]) {
              wait_full(i + 1);
              if (!ok) break;
              scores(q, i + 1);
            } else {
              umma_commit(&ctl->o_full[q]);
            }
          }
          if (!ok) break;
          umma_commit(&ctl->empty[v_slot]);
          if (i + 1 < total) {
            umma_commit(&ctl->empty[k_slot]);
            next();
          }
        }
      }
      if (!ok) {      // ... and the products in flight the time to finish
        const unsigned long long t0 = global_ns();
        while (global_ns() - t0 < 1000000ull) __nanosleep(1000);
      }
    }
  } else {
    // ------------------------------------------------------------------ value tiles that some row sees a part of
    const int tid = threadIdx.x - 320;
    uint32_t phases = 0;
    int first = w.partial - w.t0;
    if (first < 0) first = 0;
    bool ok = true;
    for (int i = first; i < total && ok; ++i) {
      const int slot = v_entry(i) % kRing;
      ok = __all_sync(0xFFFFFFFFu, wait_bar(&ctl->raw[slot], phases >> slot & 1u, ctl, 4, i));
      phases ^= 1u << slot;
      const int rows = tile_rows(w, w.t0 + i), rows16 = (rows + 15) & ~15;
      if (ok) {
#pragma unroll
        for (int d = 0; d < kDBlocks; ++d) {
          uint4* at = reinterpret_cast<uint4*>(smem + (2 * kTileBytes) + slot * kTileBytes + d * kBlockBytes);
          for (int c = tid; c < rows16 * 8; c += 64) {
            uint4 v = at[c];
            uint32_t* e = reinterpret_cast<uint32_t*>(&v);
            if (not_finite2<T>(v.x) | not_finite2<T>(v.y) | not_finite2<T>(v.z) | not_finite2<T>(v.w)) {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const uint32_t bad = not_finite2<T>(e[j]);
                e[j] &= ~((bad >> 15) * 0xFFFFu);
              }
              at[c] = v;
              if (c / 8 < rows) ctl->any_bad = 1;
            }
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      ok = !named_any(3, 64, !ok);                  // the two warps leave together
      if (ok && tid == 0) mbar_arrive(&ctl->full[slot]);
    }
    named_arrive(2, 320);
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // ------------------------------------------------------------------ softmax
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_tmem = tmem + lanes + half * 128, o_tmem = tmem + lanes + 256 + half * 128;
    const int mine = p.pair ? w.nt[half] : (total + 1 - half) / 2;
    // all rows of this half see the tiles below this one whole
    const int64_t first_tok = w.tok0 + (p.pair ? half * p.tokens : 0);
    const int whole = p.pair && half && w.halves == 2 ? (int)(visible(a, w.s, first_tok) / kTile) : w.partial;
    const int64_t limit = row_ok ? visible(a, w.s, tok) : 0;
    uint64_t bits = a.tree_mask && row_ok ? (uint64_t)__ldcg(a.tree_mask + w.s.q0 + tok) : 0ull;
    if (w.s.n < kTreeLimit) bits &= (1ull << w.s.n) - 1;            // bits behind the sequence's tokens mean nothing
    constexpr float kLog2e = 1.4426950408889634f;
    const float sl2 = SCORE ? 1.0f : a.scale * kLog2e;             // score to log2 domain, where it is not there yet
    const float cap2 = a.cap * kLog2e, to_cap = a.cap > 0.f ? 2.0f * kLog2e * a.scale / a.cap : 0.f;
    const float slope2 = SCORE && a.slopes && row_ok ? __ldcg(a.slopes + head) * kLog2e : 0.f;
    float m = -INFINITY, l = 0.f;                                   // m: in log2 domain
    bool ok = true;
    for (int i = 0; i < mine; ++i) {
      const int t = w.t0 + (p.pair ? i : 2 * i + half);
      ok = __all_sync(0xFFFFFFFFu, wait_bar(&ctl->s_full[half], i & 1, ctl, 5, t));
      if (!ok) break;
      tc_fence_after();
      uint32_t raw[128];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(s_tmem + c * 32, raw + c * 32);
      tmem_wait_ld();
      float* x = reinterpret_cast<float*>(raw);
      if (SCORE) {
        if (a.cap > 0.f) {
          // c tanh(s / c) = c - 2 c / (exp(2 s / c) + 1)
#pragma unroll
          for (int c = 0; c < 128; ++c) x[c] = fmaf(-2.0f * cap2, rcp(ex2(x[c] * to_cap) + 1.0f), cap2);
        } else {
#pragma unroll
          for (int c = 0; c < 128; ++c) x[c] *= a.scale * kLog2e;
        }
        if (a.slopes) {
          const float at = (float)(tok + w.s.shift - (int64_t)t * kTile);
#pragma unroll
          for (int c = 0; c < 128; ++c) x[c] = fmaf(-slope2, fabsf(at - (float)c), x[c]);
        }
      }
      if (t == w.drafted) {
#pragma unroll
        for (int c = 0; c < 128; ++c) x[c] = c < 64 && (bits >> (c & 63) & 1) ? x[c] : -INFINITY;
      } else if (t >= whole) {
        const int64_t left = limit - (int64_t)t * kTile;
        const int n = left < 0 ? 0 : (left > kTile ? kTile : (int)left);
#pragma unroll
        for (int c = 0; c < 128; ++c) x[c] = c < n ? x[c] : -INFINITY;
      }
      float mx = x[0];
#pragma unroll
      for (int c = 1; c < 128; ++c) mx = fmaxf(mx, x[c]);
      mx *= sl2;
      if (i == 0) {
        m = mx;
      } else if (__any_sync(0xFFFFFFFFu, mx > m + kLazy)) {
        // a row moves by its own maximum alone: its result does not depend on the rows beside it
        const float next = mx > m + kLazy ? mx : m;
        const float f = next == m ? 1.0f : ex2(m - next);
        m = next;
        l *= f;
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(o_tmem + c * 32, o);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
          tmem_st32(o_tmem + c * 32, o);
        }
      }
      const float base = m == -INFINITY ? 0.f : m;
      float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t pk[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          const float e0 = ex2(fmaf(x[64 * c + 2 * j], sl2, -base)), e1 = ex2(fmaf(x[64 * c + 2 * j + 1], sl2, -base));
          sum0 += e0;
          sum1 += e1;
          pk[j] = pack2<T>(e0, e1);
        }
        tmem_st32(s_tmem + c * 32, pk);
      }
      l += sum0 + sum1;
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl->p_ready[half]);
    }
    // ---- the end: both halves' products are done, the smem of the ring is free
    if (ok && mine > 0) ok = __all_sync(0xFFFFFFFFu, wait_bar(&ctl->o_full[half], 0, ctl, 6, 0));
    tc_fence_after();
    named_sync(2, 320);
    const bool bad = ctl->any_bad != 0;
    // values that are not finite, of the rows this row sees in the tiles that were cleaned
    auto add_bad = [&](float* v, int col) {
      for (int i = w.partial > w.t0 ? w.partial - w.t0 : 0; i < total; ++i) {
        const int t = w.t0 + i;
        const bool draft = t == w.drafted;
        const int rows = tile_rows(w, t);
        for (int j = 0; j < rows; ++j) {
          if (!(draft ? (bits >> j & 1) : (int64_t)t * kTile + j < limit)) continue;
          const T* src = draft ? reinterpret_cast<const T*>(a.cur.v) + (w.s.q0 + j) * a.cur.v_row + w.h * a.cur.v_head
                               : reinterpret_cast<const T*>(a.past.v) + (w.s.kv0 + (int64_t)t * kTile + j) * a.past.v_row + w.h * a.past.v_head;
          float f[8];
          unpack16<T>(ld_stream16(src + col), f);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (!isfinite(f[e])) v[e] += f[e];
        }
      }
    };
    auto store = [&](float* v, int col, float inv) {       // 8 columns of this row
      if (!row_ok || col >= a.D) return;
      if (bad) add_bad(v, col);
      if (p.splits == 1) {
        float s[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] = v[e] * inv;
        *reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.out) + out_row * a.D + col) = pack16<T>(s);
      } else {
        float4* dst = reinterpret_cast<float4*>(p.part_o + ((int64_t)w.split * a.Tq * a.Hq + out_row) * a.D + col);
        dst[0] = make_float4(v[0], v[1], v[2], v[3]);
        dst[1] = make_float4(v[4], v[5], v[6], v[7]);
      }
    };
    if (p.pair) {
      if (ok && half < w.halves) {
        const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) {
          uint32_t o[32];
          if (mine > 0) {
            tmem_ld32(o_tmem + c * 32, o);
            tmem_wait_ld();
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = 0u;
          }
#pragma unroll
          for (int j = 0; j < 32; j += 8) store(reinterpret_cast<float*>(o) + j, c * 32 + j, inv);
        }
        if (p.splits > 1 && row_ok) p.part_ml[(int64_t)w.split * a.Tq * a.Hq + out_row] = make_float2(m, l);
      }
    } else {
      // each half hands the other its share of the columns through shared memory, [column][row]
      float* swap = reinterpret_cast<float*>(smem + 2 * kTileBytes);
      float2* ml = reinterpret_cast<float2*>(swap + DP * 128);
      ml[half * 128 + r] = make_float2(m, l);
      uint32_t o[DP / 2];
#pragma unroll
      for (int c = 0; c < DP / 64; ++c) {
        uint32_t g[32];
        if (mine > 0 && ok) {
          tmem_ld32(o_tmem + (half ^ 1) * (DP / 2) + c * 32, g);
          tmem_ld32(o_tmem + half * (DP / 2) + c * 32, o + c * 32);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) g[j] = o[c * 32 + j] = 0u;
        }
#pragma unroll
        for (int j = 0; j < 32; ++j) swap[((half ^ 1) * (DP / 2) + c * 32 + j) * 128 + r] = __uint_as_float(g[j]);
      }
      named_sync(4, 256);
      const float2 other = ml[(half ^ 1) * 128 + r];
      const float top = fmaxf(m, other.x);
      const float f0 = m == -INFINITY ? 0.f : ex2(m - top), f1 = other.x == -INFINITY ? 0.f : ex2(other.x - top);
      const float sum = l * f0 + other.y * f1;
      const float inv = sum == 0.f ? 0.f : 1.0f / sum;
      if (ok) {
#pragma unroll
        for (int c = 0; c < DP / 2; c += 8) {
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e)
            v[e] = __uint_as_float(o[c + e]) * f0 + swap[(half * (DP / 2) + c + e) * 128 + r] * f1;
          store(v, half * (DP / 2) + c, inv);
        }
        if (p.splits > 1 && row_ok && half == 0)
          p.part_ml[(int64_t)w.split * a.Tq * a.Hq + out_row] = make_float2(top, sum);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// out = sum over the splits of o 2^(m - max) / sum of l 2^(m - max); one warp per row, 4 columns per lane
template <typename T>
__global__ void __launch_bounds__(256) masked_attention_merge_kernel(const float* part_o, const float2* part_ml, T* out,
                                                                      int64_t rows, int D, int splits) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= rows) return;
  const float2 mine = lane < splits ? __ldcg(part_ml + lane * rows + row) : make_float2(-INFINITY, 0.f);
  float top = mine.x;
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
  const float f = mine.x == -INFINITY ? 0.f : ex2(mine.x - top);
  float sum = mine.y * f;
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  const unsigned used = __ballot_sync(0xFFFFFFFFu, mine.x != -INFINITY);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s = 0; s < splits; ++s) {
    const float fs = __shfl_sync(0xFFFFFFFFu, f, s);
    if (!(used >> s & 1) || lane * 4 >= D) continue;
    const float4 v = __ldcg(reinterpret_cast<const float4*>(part_o + ((int64_t)s * rows + row) * D) + lane);
    acc.x = fmaf(v.x, fs, acc.x);
    acc.y = fmaf(v.y, fs, acc.y);
    acc.z = fmaf(v.z, fs, acc.z);
    acc.w = fmaf(v.w, fs, acc.w);
  }
  if (lane * 4 < D) {
    T* dst = out + row * D + lane * 4;
    dst[0] = Elem<T>::from_f(acc.x * inv);
    dst[1] = Elem<T>::from_f(acc.y * inv);
    dst[2] = Elem<T>::from_f(acc.z * inv);
    dst[3] = Elem<T>::from_f(acc.w * inv);
  }
}

// ------------------------------------------------------------------------------------------------- host side
struct TcPlan {
  bool use;
  int group, tokens, pair, row_blocks, splits;
};

// Everything that sizes the workspace and the grid follows from shapes and host lengths alone.
TcPlan plan_tc(int64_t Tq, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_seqlen, int64_t max_kvlen, int dtype) {
  TcPlan pl{};
  if ((dtype != PMX_DTYPE_F16 && dtype != PMX_DTYPE_BF16) || D % 8 || D > 128 || Hkv <= 0 ||
      Hq % Hkv || Hq / Hkv > kTile)
    return pl;
  if (Tq <= 0 || B <= 0 || Hq <= 0 || D <= 0 || max_seqlen <= 0 || max_kvlen <= 0 || Tq >= (1ll << 31)) return pl;
  if (max_seqlen > Tq) max_seqlen = Tq;
  pl.group = (int)(Hq / Hkv);
  pl.tokens = kTile / pl.group;
  pl.pair = max_seqlen > pl.tokens;
  const int64_t blocks = ceil_div(max_seqlen, pl.pair ? 2 * pl.tokens : pl.tokens);
  const int64_t ctas = blocks * B * Hkv, tiles = ceil_div(max_kvlen, kTile);
  if (ctas > (1 << 24) || B > (1 << 20)) return pl;
  pl.row_blocks = (int)blocks;
  // Split the keys while that fills SMs that would idle, with at least 4 key tiles a CTA: below that the start of a
  // CTA and the merge cost more than the shorter walk gains.
  int64_t s = sm_count() / (ctas < 1 ? 1 : ctas);
  if (s > ceil_div(tiles, 4)) s = ceil_div(tiles, 4);
  pl.splits = (int)(s < 1 ? 1 : (s > kMaxSplits ? kMaxSplits : s));
  pl.use = true;
  return pl;
}

size_t tc_workspace(const TcPlan& pl, int64_t Tq, int64_t Hq, int64_t D) {
  if (!pl.use || pl.splits == 1) return 0;
  return (size_t)pl.splits * Tq * Hq * ((size_t)D * sizeof(float) + sizeof(float2));
}

bool rows_ok_for_tma(const void* base, int64_t row, int64_t head, int64_t rows) {
  return aligned16(base) && row > 0 && head > 0 && row % 8 == 0 && head % 8 == 0 && row < (1ll << 38) && head < (1ll << 38) &&
         rows < (1ll << 31) - 256;
}

// [rows, heads, D] with strides in elements; boxes of 64 columns, `heads_box` heads and `rows_box` rows
int make_head_map(CUtensorMap* map, const void* base, int64_t rows, int heads, int D, int64_t row_stride,
                  int64_t head_stride, uint32_t heads_box, uint32_t rows_box, int dtype, const char* name) {
  PFN_cuTensorMapEncodeTiled_v12000 fn = encode_fn();
  if (!fn) return fail(PMX_ERR_CUDA, "%s: cuTensorMapEncodeTiled is not available from this driver", name);
  cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)rows};
  cuuint64_t strides[2] = {(cuuint64_t)head_stride * 2, (cuuint64_t)row_stride * 2};
  cuuint32_t box[3] = {64, heads_box, rows_box}, estr[3] = {1, 1, 1};
  const CUtensorMapDataType dt = dtype == PMX_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const CUresult r = fn(map, dt, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(PMX_ERR_CUDA, "%s: cuTensorMapEncodeTiled failed with code %d (rows=%lld heads=%d head_dim=%d)", name, (int)r, (long long)rows, heads, D);
  return PMX_OK;
}

template <typename T, int DP>
int launch_tc_t(const TileMaps& maps, const TcArgs& p, cudaStream_t s) {
  const bool score = p.a.cap > 0.f || p.a.slopes;
  const void* kern = score ? (const void*)masked_attention_kernel<T, DP, true> : (const void*)masked_attention_kernel<T, DP, false>;
  const size_t smem = (size_t)(2 + kRing) * kTile * DP * 2 + sizeof(Ctl) + 1024;
  PMX_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  const int64_t grid = (int64_t)p.row_blocks * p.a.B * p.a.Hkv * p.splits + p.zero_ctas;
  void* args[] = {(void*)&maps, (void*)&p};
  const int st = launch_pdl(kern, dim3((unsigned)grid), dim3(kAttnThreads), smem, s, args);
  if (st != PMX_OK || p.splits == 1) return st;
  const int64_t rows = p.a.Tq * p.a.Hq;
  return launch_pdl_k(masked_attention_merge_kernel<T>, dim3((unsigned)ceil_div(rows, 8)), dim3(256), 0, s,
                      (const float*)p.part_o, (const float2*)p.part_ml, (T*)p.a.out, rows, p.a.D, p.splits);
}

// Runs the call on the tensor cores if they cover it (*done), otherwise leaves it to the row kernel.
int launch_tc(const AttnArgs& a, const TcPlan& pl, int dtype, const char* name, void* ws, cudaStream_t s, bool* done) {
  *done = false;
  if (!pl.use || !aligned16(a.out) || !rows_ok_for_tma(a.q, a.q_tok, a.q_head, a.Tq) ||
      !rows_ok_for_tma(a.past.k, a.past.k_row, a.past.k_head, a.past.rows) ||
      !rows_ok_for_tma(a.past.v, a.past.v_row, a.past.v_head, a.past.rows))
    return PMX_OK;
  if (a.tree_mask && (!rows_ok_for_tma(a.cur.k, a.cur.k_row, a.cur.k_head, a.cur.rows) ||
                      !rows_ok_for_tma(a.cur.v, a.cur.v_row, a.cur.v_head, a.cur.rows)))
    return PMX_OK;
  *done = true;
  TcArgs p{};
  p.a = a;
  p.group = pl.group; p.tokens = pl.tokens; p.row_blocks = pl.row_blocks; p.splits = pl.splits; p.pair = pl.pair;
  p.zero_ctas = (int)(a.Tq / 512 < 1 ? 1 : (a.Tq / 512 > 32 ? 32 : a.Tq / 512));
  p.part_ml = reinterpret_cast<float2*>(ws);
  p.part_o = reinterpret_cast<float*>(p.part_ml + (size_t)pl.splits * a.Tq * a.Hq);
  TileMaps m{};
  int st = make_head_map(&m.q, a.q, a.Tq, a.Hq, a.D, a.q_tok, a.q_head, (uint32_t)pl.group, (uint32_t)pl.tokens, dtype, name);
  if (st == PMX_OK) st = make_head_map(&m.k, a.past.k, a.past.rows, a.Hkv, a.D, a.past.k_row, a.past.k_head, 1, kTile, dtype, name);
  if (st == PMX_OK) st = make_head_map(&m.v, a.past.v, a.past.rows, a.Hkv, a.D, a.past.v_row, a.past.v_head, 1, kTile, dtype, name);
  if (st == PMX_OK && a.tree_mask) st = make_head_map(&m.ck, a.cur.k, a.cur.rows, a.Hkv, a.D, a.cur.k_row, a.cur.k_head, 1, kTreeLimit, dtype, name);
  if (st == PMX_OK && a.tree_mask) st = make_head_map(&m.cv, a.cur.v, a.cur.rows, a.Hkv, a.D, a.cur.v_row, a.cur.v_head, 1, kTreeLimit, dtype, name);
  if (st != PMX_OK) return st;
  const bool bf = dtype == PMX_DTYPE_BF16;
  if (a.D <= 64) return bf ? launch_tc_t<__nv_bfloat16, 64>(m, p, s) : launch_tc_t<__half, 64>(m, p, s);
  return bf ? launch_tc_t<__nv_bfloat16, 128>(m, p, s) : launch_tc_t<__half, 128>(m, p, s);
}
