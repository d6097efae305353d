// The tensor-core kernel of masked_attention.cu (included there, inside its namespaces): 16-bit tensors, head
// sizes up to 128.
//
// A work item is one or two tiles of 128 rows against (a run of) the keys of their sequence, 128 at a time.  A row is a
// (query token, query head) of ONE key head: the G query heads that share it are packed into the tile
// (128 / G tokens of them), so each key and value crosses to the SM once for the whole group.  One CTA per SM
// walks its items; its warps each run through all of them, so that the loads and products of the next item
// begin under the last one's end:
//   warp 8   makes the items (a queue in shared memory) and issues the TMA loads: keys and values through a ring
//            of 128-row buffers (128-byte swizzle)
//   warp 9   its elected lane issues the tcgen05 products: S_w = Q_w K^T into tensor memory columns [128 w, +128),
//            O_w += P_w V into columns [256 + 128 w, +128); P_w is read from tensor memory, V is the MN-major operand
//   warps 0-3 and 4-7  the softmax of S_0 and S_1, one thread per row (a thread owns a tensor memory lane, so the
//            row's maximum and sum need no exchange); P_w overwrites S_w in 16 bits and is handed over in two halves
//   warps 10, 11  store drafted keys and values, then go over those value tiles of which some rows see a part only
// With more than 128 rows (`pair`) the two tiles share the keys; an item is one block of rows, the longest first.  With
// fewer, both softmax halves work on the same rows, on the even and the odd key tiles, and meet at the end; the
// key tiles of all (sequence, key head) pairs are then dealt out evenly over the CTAs as one long list, and what a cut
// leaves in pieces is merged by a second kernel (fp32 results with maximum and sum).  Pairs with so few CTAs that SMs
// would idle split their keys too.
//
// On B200, bf16, device time of back-to-back replays of one input: 8192 causal tokens of 32/8 heads of 128 in 460-467 us, 1.18
// PFLOP/s (72 % of the measured rate); without the mask 950 us, 1.16 PFLOP/s; 32 trees of 16 tokens over 400 MB of cache in
// 90 us.  Among changing inputs, host included, the first and the last take 550 us (at the power cap) and 97-102 us.
// The bound is the tensor pipe and, next to it, the exponentials: per 128 x 128 scores 1024 cycles of products (head
// size 128) against 1024 of the special function unit, and a tile's softmax lies between its own two products.  So a
// half's softmax runs beside the other half's products, and is kept short.  The running maximum moves only when a
// row's new maximum lies more than 2^8 above it (2^4 in f16), so that O in tensor memory is rescaled rarely; probabilities
// stay below 2^8 (2^15 in f16, scaled up by 2^11), and the sum divides the same scale out again.  A probability is rounded to the
// inputs' type for the second product, whose operands have one type; the sum takes it unrounded.  The error
// against 64 bits is up to 1.4 times that of one rounding of the result.
//
// A masked score becomes -inf whatever the product holds.  A masked VALUE needs more: 0 * inf and 0 * NaN are NaN in
// the second product, so in the tiles that are not seen whole by every row, values that are not finite are replaced by
// zeros in shared memory, and if there were any among the sequence's own, the end of the item adds them back for the
// rows that see them.
constexpr int kTile = 128;                  // keys of a tile, rows of a tile
constexpr int kRing = 5;                    // ring buffers: two keys and two values in use, one on the way
constexpr int kAttnThreads = 384;
constexpr int kMaxSplits = 32;
constexpr int kQueue = 4;                   // items under way
constexpr int kMinTiles = 4;                // key tiles that a split of a pair of row tiles should have at least,
constexpr int kFlatTiles = 2;               // and that a CTA should have of the list of all key tiles (2: one for each half;
                                            // two drafted trees over 700 rows: a tenth faster than with 4)
// How far (log2) a row's maximum may run ahead of the one in use, and the power of two that probabilities are scaled by, in
// product and sum alike.  In f16, which ends at 2^16 and below at 2^-24, a weak key's probability would be lost in the product and
// stay in the sum: scaled, it is exact to half a step down to 2^-25 of the strongest key's and lost below 2^-36.  bf16 has
// the range of 32 bits.
template <typename T> constexpr float kLazy = std::is_same<T, __half>::value ? 4.0f : 8.0f;
template <typename T> constexpr float kScaleUp = std::is_same<T, __half>::value ? 11.0f : 0.0f;
constexpr unsigned long long kAttnWaitNs = 2000000000ull;

__device__ int g_attention_status[4];       // record of a bounded wait that ran out: code, role, tile, CTA

struct TileMaps {
  CUtensorMap q, k, v, ck, cv;              // ck, cv: the drafted tokens' (trees only)
};

struct TcArgs {
  AttnArgs a;
  // pair: partial results [splits][Tq * Hq][D], maximum (log2) and sum [splits][Tq * Hq].  Otherwise [2 * CTAs][128][D] and
  // [2 * CTAs][128]: a CTA's first piece in slot 2c when it begins inside an item, its last in 2c + 1 when it ends inside;
  // pieces[b * Hkv + h] = the CTAs (first, last) that share the item.
  float* part_o;
  float2* part_ml;
  int2* pieces;
  int4* cuts;                               // of each CTA: the item it begins and others end: first token, rows, key head, last CTA
  int group, tokens;                        // query heads per key head, tokens of a row tile
  int row_blocks, splits, pair;
  int pieces_of_item;                       // about the most, from the host's lengths
  int ctas;                                 // CTAs that the workspace has room for; more may run, with nothing but stores to do
  int flat;                                 // not pair: cut the list of key tiles evenly (otherwise whole items)
};

struct Work {
  int b, h, slot;      // slot: of the partial result, -1: none; h < 0: the end
  Sequence s;
  int tok0;            // first token of the item's rows, in the sequence
  int halves;          // row tiles in use (1 without pair)
  int t0, nt[2];       // first key tile; tiles of each row tile (without pair: nt[0] is the item's)
  int drafted;         // index of the drafted tokens' tile, -1: none
  int partial;         // first tile that some row does not see whole
  int number;          // of the item in this CTA, from 1
};

struct Ctl {
  uint64_t full[kRing], empty[kRing], raw[kRing];
  uint64_t q_full, q_empty, s_full[2], p_ready[2][2], o_full[2];
  uint64_t work_full[kQueue], work_empty[kQueue];
  float2 ml[256];
  Work work[kQueue];
  volatile int bad[kQueue];                 // number of the last item in this queue place that had a bad value
  uint32_t tmem;
  volatile int abort;
};

// The clock is read only after many polls: reading %globaltimer takes long, and a wait that ends meanwhile would be
// noticed late.
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, Ctl* c, int role, int tile) {
  unsigned long long t0 = 0;
  for (uint32_t it = 1;; ++it) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((it & 127u) == 0u) {
      if (c->abort) return false;
      const unsigned long long now = global_ns();
      if (t0 == 0) t0 = now;
      if (now - t0 > kAttnWaitNs) {
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
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
}
// D[tmem] = A * B ("first") or D += A * B ("more"), A from shared memory (descriptor) or from tensor memory ("ts")
#define PMX_UMMA(name, a_type, a_con, a_brackets_l, a_brackets_r, accumulate)                                        \
  __device__ __forceinline__ void name(uint32_t d_tmem, a_type a, uint64_t b_desc, uint32_t idesc) {                   \
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, " accumulate                                                   \
                 ", 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], " a_brackets_l "%1" a_brackets_r ", %2, %3, p;\n\t}" \
                 ::"r"(d_tmem), a_con(a), "l"(b_desc), "r"(idesc)                                                      \
                 : "memory");                                                                                          \
  }
PMX_UMMA(umma_f16_first, uint64_t, "l", "", "", "0")
PMX_UMMA(umma_f16_more, uint64_t, "l", "", "", "1")
PMX_UMMA(umma_f16_ts_first, uint32_t, "r", "[", "]", "0")
PMX_UMMA(umma_f16_ts_more, uint32_t, "r", "[", "]", "1")
#undef PMX_UMMA
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
__device__ __forceinline__ void tmem_st16u(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// waits for the loads from tensor memory before; the registers of the last one pass through, so that no use of
// them can move in front
__device__ __forceinline__ void tmem_wait_ld32(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                 "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
                 "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                 "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {     // NaN wins
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max3_number(float a, float b, float c) {     // NaN loses
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// tanh(y) / y of two values in [-1, 1]: a polynomial of degree 6 in y^2 whose largest relative error is least (weighted
// least squares iterated to equal ripples: 5.0e-8, 1.7e-7 with the roundings)
__device__ __forceinline__ f32x2 tanh_over_y(f32x2 y) {
  const f32x2 z = mul2(y, y);
  f32x2 p = fma2(z, pair2(0x1.10e5d0p-10f, 0x1.10e5d0p-10f), pair2(-0x1.968b68p-8f, -0x1.968b68p-8f));
  p = fma2(p, z, pair2(0x1.4c6e56p-6f, 0x1.4c6e56p-6f));
  p = fma2(p, z, pair2(-0x1.b5eb84p-5f, -0x1.b5eb84p-5f));
  p = fma2(p, z, pair2(0x1.10e672p-3f, 0x1.10e672p-3f));
  p = fma2(p, z, pair2(-0x1.55540ap-2f, -0x1.55540ap-2f));
  return fma2(p, z, pair2(0x1.fffffep-1f, 0x1.fffffep-1f));
}
// the same in [-0.4, 0.4], degree 3: 9.8e-8, 1.5e-7 with the roundings
__device__ __forceinline__ f32x2 tanh_over_y_near(f32x2 y) {
  const f32x2 z = mul2(y, y);
  f32x2 p = fma2(z, pair2(-0x1.858f22p-5f, -0x1.858f22p-5f), pair2(0x1.0fca24p-3f, 0x1.0fca24p-3f));
  p = fma2(p, z, pair2(-0x1.55502ap-2f, -0x1.55502ap-2f));
  return fma2(p, z, pair2(0x1.fffffcp-1f, 0x1.fffffcp-1f));
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

// Key tiles that rows [tok0, tok0 + tokens) of the sequence need, the drafted tokens' tile included.
__device__ __forceinline__ int key_tiles(const AttnArgs& a, const Sequence& s, int tok0, int tokens) {
  const int last = tok0 + tokens - 1;
  const int64_t seen = visible(a, s, last < s.n ? last : s.n - 1);
  return (int)((seen + kTile - 1) / kTile) + (a.tree_mask ? 1 : 0);
}
// What is left of a Work once b, h, s and tok0 are known: the tiles of its rows, cut to [t0, t1).
__device__ __forceinline__ void finish_work(const TcArgs& p, Work& w, int t0, int t1) {
  const AttnArgs& a = p.a;
  w.halves = p.pair && w.tok0 + p.tokens < w.s.n ? 2 : 1;
  w.partial = (int)(visible(a, w.s, w.tok0) / kTile);
  const int n0 = key_tiles(a, w.s, w.tok0, p.tokens);
  const int n1 = w.halves == 2 ? key_tiles(a, w.s, w.tok0, 2 * p.tokens) : n0;
  w.drafted = a.tree_mask ? n1 - 1 : -1;
  if (t1 > n1) t1 = n1;
  w.t0 = t0 < t1 ? t0 : t1;
  w.nt[0] = (n0 < t1 ? n0 : t1) - w.t0;
  if (w.nt[0] < 0) w.nt[0] = 0;
  w.nt[1] = w.halves == 2 ? t1 - w.t0 : 0;
}

// The items of one CTA, in order.  Run by all lanes of a warp.
// Pair, or whole items: the list of all items that have rows, row blocks that see the most keys first, is dealt out like
// cards, to and fro: a CTA that had the longest item of one deal has the shortest of the next.  8192 causal tokens: the
// fullest CTA has 1.02 times the mean, and 1.14 times when every deal begins at the same CTA; eight ragged prompts of up
// to 1501 tokens: 1.06, and 1.6 when blocks without rows are dealt out too.
struct Items {
  int deal, level, i0, rows;      // the next deal; its place in the list: row block, 32 sequences, the lane's sequence's rows
  int b;                          // flat: the sequence that [base, base + Hkv * tiles) of the list of key tiles belongs to
  int64_t base, u, u1, total;     // base otherwise: items before the place
  int tiles, ctas;
  Sequence s;
  __device__ __forceinline__ int tiles_of(const TcArgs& p, int seq, Sequence& q) {
    q = load_sequence(p.a, seq);
    if (q.n == 0) return 0;
    const int t = key_tiles(p.a, q, 0, p.tokens);
    return t < 1 ? 1 : t;         // rows that see nothing still have a result
  }
  __device__ __forceinline__ void load_rows(const AttnArgs& a, int first) {
    const int i = first + (int)(threadIdx.x & 31);
    i0 = first;
    rows = i < a.B ? load_sequence(a, i).n : 0;
  }
  __device__ __forceinline__ void start(const TcArgs& p) {
    const AttnArgs& a = p.a;
    if (!p.flat) {
      deal = 0;
      base = 0;
      level = p.row_blocks - 1;
      load_rows(a, 0);
      return;
    }
    const int lane = threadIdx.x & 31;
    if (lane == 0 && (int)blockIdx.x < p.ctas) p.cuts[blockIdx.x] = make_int4(0, 0, 0, 0);
    int64_t sum = 0;
    Sequence q;
    for (int i = lane; i < a.B; i += 32) sum += tiles_of(p, i, q);
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    total = sum * a.Hkv;
    const int64_t most = total / kFlatTiles;
    ctas = (int)(most < 1 ? 1 : (most < p.ctas ? most : p.ctas));
    u = (int)blockIdx.x < ctas ? (int64_t)blockIdx.x * total / ctas : total;
    u1 = (int)blockIdx.x < ctas ? (int64_t)(blockIdx.x + 1) * total / ctas : total;
    if (u >= u1) return;
    // the sequence that u falls into
    base = 0;
    for (int i0 = 0; i0 < a.B; i0 += 32) {
      const int i = i0 + lane;
      int64_t end = i < a.B ? (int64_t)tiles_of(p, i, q) * a.Hkv : 0;
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xFFFFFFFFu, end, o);
        if (lane >= o) end += v;
      }
      const unsigned past = __ballot_sync(0xFFFFFFFFu, base + end > u);
      if (past) {
        const int l = __ffs(past) - 1;
        b = i0 + l;
        if (l) base += __shfl_sync(0xFFFFFFFFu, end, l - 1);
        break;
      }
      base += __shfl_sync(0xFFFFFFFFu, end, 31);
    }
    tiles = tiles_of(p, b, s);
  }
  __device__ __forceinline__ bool next(const TcArgs& p, Work& w) {
    const AttnArgs& a = p.a;
    if (!p.flat) {
      const int64_t at = (int64_t)deal * gridDim.x + (deal & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
      const int block = (p.pair ? 2 : 1) * p.tokens, per = a.Hkv * p.splits;
      while (level >= 0) {
        const unsigned some = __ballot_sync(0xFFFFFFFFu, rows > level * block);
        const int64_t items = (int64_t)__popc(some) * per;
        if (at < base + items) {
          const int in = (int)(at - base), nth = in / per, lane = threadIdx.x & 31;
          const bool it = (some >> lane & 1) && __popc(some & ((1u << lane) - 1)) == nth;
          w.b = i0 + __ffs(__ballot_sync(0xFFFFFFFFu, it)) - 1;
          w.h = in % per / p.splits;
          const int split = in % p.splits;
          w.slot = p.splits > 1 ? split : -1;
          w.tok0 = level * block;
          w.s = load_sequence(a, w.b);
          const int all = key_tiles(a, w.s, w.tok0, block);
          const int share = (all + p.splits - 1) / p.splits;
          finish_work(p, w, split * share, (split + 1) * share);
          ++deal;
          return true;
        }
        base += items;
        if (i0 + 32 < a.B) {
          load_rows(a, i0 + 32);
        } else {
          --level;
          if (i0) load_rows(a, 0);
        }
      }
      return false;
    }
    if (u >= u1) return false;
    while (u >= base + (int64_t)tiles * a.Hkv) {
      base += (int64_t)tiles * a.Hkv;
      tiles = tiles_of(p, ++b, s);
    }
    const int64_t in = u - base;
    const int t0 = (int)(in % tiles), left = tiles - t0, take = u1 - u < left ? (int)(u1 - u) : left;
    w.b = b;
    w.h = (int)(in / tiles);
    w.s = s;
    w.tok0 = 0;
    finish_work(p, w, t0, t0 + take);
    w.slot = t0 > 0 ? 2 * (int)blockIdx.x : (take < tiles ? 2 * (int)blockIdx.x + 1 : -1);
    if (t0 == 0 && (threadIdx.x & 31) == 0) {     // the CTA that holds the first tile says who shares the item
      const int last = (int)(((u + tiles) * ctas - 1) / total);
      p.pieces[(int64_t)b * a.Hkv + w.h] = make_int2((int)blockIdx.x, last);
      if (take < tiles) p.cuts[blockIdx.x] = make_int4((int)s.q0, s.n * p.group, w.h, last);
    }
    u += take;
    return true;
  }
};

// rows of a key tile that hold keys of the sequence
__device__ __forceinline__ int tile_rows(const Work& w, int t) {
  if (t == w.drafted) return w.s.n;
  const int64_t left = w.s.len - (int64_t)t * kTile;
  return (int)(left < kTile ? left : kTile);
}

// Adds to 8 columns of a row's result the values that are not finite, of the keys the row sees in the tiles that were
// cleaned.  Rare, and kept out of the way of the registers of those who call it.
struct Cols8 { float v[8]; };
template <typename T>
__device__ __noinline__ Cols8 add_bad(Cols8 x, const AttnArgs* ap, const Work* wp, int col, int64_t limit, uint64_t bits,
                                      int total) {
  const AttnArgs& a = *ap;
  const Work& w = *wp;
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
        if (!isfinite(f[e])) x.v[e] += f[e];
    }
  }
  return x;
}

// BIAS: calls with a distance bias.  Where all keys of a tile lie before all rows it is linear in the key, and is added as
// the scores are read.
template <typename T, int DP, bool BIAS>
__global__ void __launch_bounds__(kAttnThreads, 1)
masked_attention_kernel(const __grid_constant__ TileMaps maps, const __grid_constant__ TcArgs p) {
  constexpr int kTileBytes = kTile * DP * 2;
  constexpr int kBlockBytes = kTile * 128;          // 64 columns of a tile
  constexpr int kDBlocks = DP / 64;
  extern __shared__ __align__(1024) uint8_t smem[];
  Ctl* ctl = reinterpret_cast<Ctl*>(smem + (2 + kRing) * kTileBytes);
  const AttnArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int i = 0; i < kRing; ++i) {
      mbar_init(&ctl->full[i], 1);
      mbar_init(&ctl->empty[i], 1);
      mbar_init(&ctl->raw[i], 1);
    }
    mbar_init(&ctl->q_full, 1);
    mbar_init(&ctl->q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ctl->s_full[i], 1);
      mbar_init(&ctl->p_ready[i][0], 4);
      mbar_init(&ctl->p_ready[i][1], 4);
      mbar_init(&ctl->o_full[i], 1);
    }
    for (int i = 0; i < kQueue; ++i) {
      mbar_init(&ctl->work_full[i], 1);
      mbar_init(&ctl->work_empty[i], 11);             // 8 softmax warps, the products' thread, 2 cleaning warps
      ctl->bad[i] = 0;
    }
    // the swizzled tiles need 1024-byte boundaries: the dynamic shared memory of a kernel without static shared
    // memory begins on one; should it ever not, the kernel says so instead of computing nonsense
    ctl->abort = (smem_u32(smem) & 1023u) != 0;
    if (ctl->abort && atomicExch(&g_attention_status[0], 1) != 1) g_attention_status[1] = 99;
    fence_barrier_init();
    prefetch_tensormap(&maps.q);
    prefetch_tensormap(&maps.k);
    prefetch_tensormap(&maps.v);
  }
  if (warp == 9) {
    tmem_alloc(&ctl->tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  // All 512 columns are this block's, so they begin at column 0 and addresses are constants; checked all the same.
  constexpr uint32_t tmem = 0;
  if (ctl->tmem != 0 && threadIdx.x == 0) {
    ctl->abort = 1;
    if (atomicExch(&g_attention_status[0], 1) != 1) g_attention_status[1] = 98;
  }
  const uint32_t q_addr = smem_u32(smem), ring = q_addr + 2 * kTileBytes;
  const int rows_tile = p.tokens * p.group;
  // Order of the ring within an item: the keys of the first `lag` tiles, then values and keys in turn.
  const int lag = p.pair ? 1 : 2;
  auto tiles_of = [&](const Work& w) { return w.nt[0] > w.nt[1] ? w.nt[0] : w.nt[1]; };

  // The softmax warpgroups hold a row of scores in registers; the third one needs few.  208 x 256 + 80 x 128 =
  // 63488 of the 168 x 384 = 64512 registers that the block starts with.
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    if (warp == 8) {
      // ---------------------------------------------------------------- items and loads
      Items items;
      items.start(p);
      int slot = 0, place = 0, number = 0;
      uint32_t phase = 0, place_phase = 0, q_phase = 0;
      bool ok = !ctl->abort;
      while (ok) {
        Work w;
        const bool more = items.next(p, w);
        ok = __all_sync(0xFFFFFFFFu, wait_bar(&ctl->work_empty[place], place_phase ^ 1u, ctl, 7, number));
        if (!ok) break;
        w.number = ++number;
        if (!more) w.h = -1;
        if (lane == 0) {
          ctl->work[place] = w;
          mbar_arrive(&ctl->work_full[place]);
        }
        if (++place == kQueue) { place = 0; place_phase ^= 1u; }
        if (!more) break;
        const int total = tiles_of(w);
        if (total == 0) continue;
        if (lane == 0) {
          ok = wait_bar(&ctl->q_empty, q_phase ^ 1u, ctl, 8, number);
          q_phase ^= 1u;
          if (ok) {
            mbar_expect_tx(&ctl->q_full, (uint32_t)(w.halves * kDBlocks * 128 * rows_tile));
            for (int i = 0; i < w.halves; ++i)
              for (int d = 0; d < kDBlocks; ++d)
                tma_load_3d(q_addr + i * kTileBytes + d * kBlockBytes, &maps.q, &ctl->q_full, d * 64, w.h * p.group,
                            (int)w.s.q0 + w.tok0 + i * p.tokens);
          }
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
        }
        ok = __shfl_sync(0xFFFFFFFFu, (int)ok, 0) != 0;
      }
      if (!ok) {      // leave the copies in flight the time to land
        const unsigned long long t0 = global_ns();
        while (global_ns() - t0 < 1000000ull) __nanosleep(1000);
      }
    } else if (warp == 9) {
      // ---------------------------------------------------------------- products
      // The whole warp runs the loop and one elected lane issues: operands that are the same in all lanes stay in
      // uniform registers.  (One thread on its own needed 125 cycles per product, more than the product takes.)
      const uint32_t idesc_s = make_idesc<T>(128, 128), idesc_d = make_idesc<T>(128, kTreeLimit);
      const uint32_t idesc_o = make_idesc<T>(128, DP) | (1u << 16);      // B is MN-major
      const uint64_t q_desc = smem_desc_sw128(q_addr), k_desc = smem_desc_sw128(ring), v_desc = smem_desc_mn(ring);
      constexpr uint64_t kTile16 = kTileBytes / 16, kBlock16 = kBlockBytes / 16;
      int slot = 0, place = 0;
      uint32_t phase = 0, place_phase = 0, q_phase = 0, p_phase0 = 0, p_phase1 = 0;
      bool ok = true;
      auto next = [&]() { if (++slot == kRing) { slot = 0; phase ^= 1u; } };
      for (;;) {
        ok = __all_sync(0xFFFFFFFFu, wait_bar(&ctl->work_full[place], place_phase, ctl, 9, 0));
        if (!ok) break;
        const Work& w = ctl->work[place];
        if (w.h < 0) break;
        const int n0 = __shfl_sync(0xFFFFFFFFu, w.nt[0], 0), n1 = __shfl_sync(0xFFFFFFFFu, w.nt[1], 0);
        const int total = n0 > n1 ? n0 : n1;
        const int drafted = __shfl_sync(0xFFFFFFFFu, w.drafted - w.t0, 0);          // from the item's first tile
        const int last_rows = __shfl_sync(0xFFFFFFFFu, total > 0 ? tile_rows(w, w.t0 + total - 1) : 0, 0);
        // the past's last tile may be short too where a drafted tile follows
        const int prev_rows = __shfl_sync(0xFFFFFFFFu, total > 1 ? tile_rows(w, w.t0 + total - 2) : 0, 0);
        auto wait = [&](uint64_t* bar, uint32_t parity, int role, int i) {
          ok = __all_sync(0xFFFFFFFFu, wait_bar(bar, parity, ctl, role, i));
          tc_fence_after();
        };
        // What an elected lane issues, without a branch where the tile is full:
        // S_q = Q_q K_i^T with the keys in slot `from`
        auto issue_scores = [&](int q, int i, int from) {
          const uint64_t kd = k_desc + from * kTile16, qd = q_desc + (p.pair ? q : 0) * kTile16;
          const uint32_t idesc = i == drafted ? idesc_d : idesc_s;
          umma_f16_first(q * 128, qd, kd, idesc);
#pragma unroll
          for (int kk = 1; kk < DP / 16; ++kk) {
            const uint64_t off = (kk / 4) * kBlock16 + (kk % 4) * 2;
            umma_f16_more(q * 128, qd + off, kd + off, idesc);
          }
          umma_commit(&ctl->s_full[q]);
        };
        // O_q += P_q V for the 64 keys of one half of the tile in slot `from`, of which `rows` exist
        auto issue_output = [&](int q, int from, int upper, int rows, bool first) {
          const uint64_t vd = v_desc + from * kTile16 + upper * 512;
          const uint32_t pt = q * 128 + upper * 32, ot = 256 + q * 128;
          rows -= upper * 64;
          if (rows > 48) {
            if (first) umma_f16_ts_first(ot, pt, vd, idesc_o);
            else umma_f16_ts_more(ot, pt, vd, idesc_o);
            umma_f16_ts_more(ot, pt + 8, vd + 128, idesc_o);
            umma_f16_ts_more(ot, pt + 16, vd + 256, idesc_o);
            umma_f16_ts_more(ot, pt + 24, vd + 384, idesc_o);
          } else {
            for (int kk = 0; kk * 16 < rows; ++kk) {
              if (first && kk == 0) umma_f16_ts_first(ot, pt, vd, idesc_o);
              else umma_f16_ts_more(ot, pt + kk * 8, vd + kk * 128, idesc_o);
            }
          }
        };
        auto scores = [&](int q, int i) {
          if (elect_one()) issue_scores(q, i, slot);
          __syncwarp();
        };
        // One tile of one half: the products with its probabilities (the first 64 keys' are ready earlier), then the scores
        // of the half's next tile, if `next_i` >= 0, from slot `k_slot`; `frees`: slots that nothing needs after this.
        auto step = [&](int q, uint32_t& p_phase, int i, bool first, int v_slot, int next_i, int k_slot, bool frees,
                        bool last_scores) {
          const int rows = i == total - 1 ? last_rows : (i == total - 2 ? prev_rows : kTile);
          wait(&ctl->p_ready[q][0], p_phase, 3, i);
          if (!ok) return;
          if (elect_one()) issue_output(q, v_slot, 0, rows, first);
          __syncwarp();
          wait(&ctl->p_ready[q][1], p_phase, 3, i);
          p_phase ^= 1u;
          if (!ok) return;
          if (elect_one()) {
            issue_output(q, v_slot, 1, rows, false);
            if (next_i >= 0) issue_scores(q, next_i, k_slot);
            else umma_commit(&ctl->o_full[q]);
            if (frees) {
              umma_commit(&ctl->empty[v_slot]);
              if (k_slot != v_slot) umma_commit(&ctl->empty[k_slot]);
              if (last_scores) umma_commit(&ctl->q_empty);
            }
          }
          __syncwarp();
        };
        auto commit = [&](uint64_t* bar) {
          if (elect_one()) umma_commit(bar);
          __syncwarp();
        };
        if (total > 0) {
          wait(&ctl->q_full, q_phase, 1, 0);
          q_phase ^= 1u;
        }
        if (!p.pair) {
          for (int i = 0; i < 2 && i < total && ok; ++i) {
            wait(&ctl->full[slot], phase, 2, i);
            if (!ok) break;
            if (i == 0) scores(0, i); else scores(1, i);
            commit(&ctl->empty[slot]);
            if (i + 1 == total) commit(&ctl->q_empty);
            next();
          }
          auto turn = [&](int q, uint32_t& p_phase, int i) {
            wait(&ctl->full[slot], phase, 2, i);
            if (!ok) return;
            const int v_slot = slot;
            const bool more = i + 2 < total;
            if (more) {
              next();
              wait(&ctl->full[slot], phase, 2, i + 2);
              if (!ok) return;
            }
            step(q, p_phase, i, i < 2, v_slot, more ? i + 2 : -1, slot, true, i + 3 == total);
            next();
          };
          for (int i = 0; i < total && ok; i += 2) {
            turn(0, p_phase0, i);
            if (ok && i + 1 < total) turn(1, p_phase1, i + 1);
          }
        } else {
          if (total > 0 && ok) wait(&ctl->full[slot], phase, 2, 0);
          if (total > 0 && ok) {
            if (n0 > 0) scores(0, 0);
            if (n1 > 0) scores(1, 0);
            commit(&ctl->empty[slot]);
            if (total == 1) commit(&ctl->q_empty);
            next();
          }
          // V_i and, behind it, K_i+1 are waited for one step ahead, between the two halves: what follows a half's last
          // product delays the other half's first one
          int v_slot = slot, k_slot = slot;
          auto fetched = [&](int i) {
            wait(&ctl->full[slot], phase, 2, i);
            v_slot = k_slot = slot;
            next();
            if (ok && i + 1 < total) {
              wait(&ctl->full[slot], phase, 2, i + 1);
              k_slot = slot;
              next();
            }
          };
          if (total > 0 && ok) fetched(0);
          for (int i = 0; i < total && ok; ++i) {
            const int v = v_slot, k = k_slot;
            if (i < n0) step(0, p_phase0, i, i == 0, v, i + 1 < n0 ? i + 1 : -1, k, n1 == 0, i + 2 == total);
            if (ok && i + 1 < total) fetched(i + 1);
            if (ok && i < n1) step(1, p_phase1, i, i == 0, v, i + 1 < n1 ? i + 1 : -1, k, true, i + 2 == total);
          }
        }
        if (!ok) break;
        if (lane == 0) mbar_arrive(&ctl->work_empty[place]);
        if (++place == kQueue) { place = 0; place_phase ^= 1u; }
      }
      if (!ok) {      // leave the products in flight the time to finish
        const unsigned long long t0 = global_ns();
        while (global_ns() - t0 < 1000000ull) __nanosleep(1000);
      }
    } else {
      // ---------------------------------------------------------------- cleaning, and drafted keys and values
      const int tid = threadIdx.x - 320;
      {   // rows of no sequence, and those past max_seqlen: zeros, or partial results that count for nothing
        auto blank = [&](int64_t row) {
          if (!p.pair || p.splits == 1) {
            T* out = reinterpret_cast<T*>(a.out) + row * a.D;
            for (int d = lane * 8; d < a.D; d += 256) *reinterpret_cast<uint4*>(out + d) = make_uint4(0, 0, 0, 0);
          } else if (lane < p.splits) {
            p.part_ml[(int64_t)lane * a.Tq * a.Hq + row] = make_float2(-INFINITY, 0.f);
          }
        };
        const int64_t lo = clamp64(__ldcg(a.seqstarts), 0, a.Tq), hi = clamp64(__ldcg(a.seqstarts + a.B), lo, a.Tq);
        const int64_t rows = (lo + a.Tq - hi) * a.Hq, step = (int64_t)gridDim.x * 2;
        for (int64_t r = (int64_t)blockIdx.x * 2 + (tid >> 5); r < rows; r += step) blank(r < lo * a.Hq ? r : r + (hi - lo) * a.Hq);
        for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
          const int64_t first = clamp64(__ldcg(a.seqstarts + b), 0, a.Tq) + a.max_seqlen, end = clamp64(__ldcg(a.seqstarts + b + 1), 0, a.Tq);
          for (int64_t r = first * a.Hq + (tid >> 5); r < end * a.Hq; r += 2) blank(r);
        }
      }
      if (a.tree_mask) {
        // Drafted keys and values into the cache, where this launch does not read them: a run of tokens for each of these
        // warps of the whole grid.  (Stored by the CTAs that read them, the rows of one head by one CTA, a single tree of
        // 62 tokens took 25 us; so it takes 14.)
        const int64_t warps = (int64_t)gridDim.x * 2, run = (a.Tq + warps - 1) / warps;
        const int64_t ta = ((int64_t)blockIdx.x * 2 + (tid >> 5)) * run, tb = ta + run < a.Tq ? ta + run : a.Tq;
        const int chunks = a.D / 8, count = a.Hkv * 2 * chunks;
        int64_t end = ta;                             // the first token that needs a look-up
        Sequence s;
        s.n = 0;
        s.q0 = s.kv0 = s.len = s.store = 0;
        for (int64_t t = ta; t < tb; ++t) {
          if (t >= end) {
            int before = 0;
            for (int i = lane; i <= a.B; i += 32) before += __ldcg(a.seqstarts + i) <= t ? 1 : 0;
            const int b = __reduce_add_sync(0xFFFFFFFFu, before) - 1;
            end = t + 1;
            s.n = 0;
            if (b >= 0 && b < a.B) {
              s = load_sequence(a, b);
              if (t < s.q0 + s.n) end = s.q0 + s.n;
            }
          }
          const int64_t row = stored(a, s, t - s.q0);
          if (t - s.q0 < 0 || t - s.q0 >= s.n || row < 0) continue;
          for (int i0 = lane; i0 < count; i0 += 32 * 4) {
            uint4 held[4];
            T* dst[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int i = i0 + 32 * j, hk = i / chunks, ch = i - hk * chunks, h = hk >> 1;
              dst[j] = nullptr;
              if (i < count) {
                held[j] = ld_stream16(hk & 1 ? reinterpret_cast<const T*>(a.cur.v) + t * a.cur.v_row + h * a.cur.v_head + ch * 8
                                             : reinterpret_cast<const T*>(a.cur.k) + t * a.cur.k_row + h * a.cur.k_head + ch * 8);
                dst[j] = (hk & 1 ? reinterpret_cast<T*>(const_cast<void*>(a.past.v)) + row * a.past.v_row + h * a.past.v_head
                                 : reinterpret_cast<T*>(const_cast<void*>(a.past.k)) + row * a.past.k_row + h * a.past.k_head) + ch * 8;
              }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (dst[j]) *reinterpret_cast<uint4*>(dst[j]) = held[j];
          }
        }
      }
      uint32_t phases = 0, place_phase = 0;
      int place = 0, entry0 = 0;
      bool ok = true;
      for (;;) {
        ok = __all_sync(0xFFFFFFFFu, wait_bar(&ctl->work_full[place], place_phase, ctl, 10, 0));
        ok = !named_any(3, 64, !ok);                // the two warps leave together
        if (!ok) break;
        const Work& w = ctl->work[place];
        if (w.h < 0) break;
        const int total = tiles_of(w);
        for (int i = w.partial > w.t0 ? w.partial - w.t0 : 0; i < total && ok; ++i) {
          const int entry = 2 * i + lag < total + i ? 2 * i + lag : total + i;     // of the values of tile i
          const int slot = (entry0 + entry) % kRing;
          ok = __all_sync(0xFFFFFFFFu, wait_bar(&ctl->raw[slot], phases >> slot & 1u, ctl, 4, i));
          phases ^= 1u << slot;
          const int rows = tile_rows(w, w.t0 + i), rows16 = (rows + 15) & ~15;
          if (ok) {
#pragma unroll
            for (int d = 0; d < kDBlocks; ++d) {
              uint4* at = reinterpret_cast<uint4*>(smem + (2 + slot) * kTileBytes + d * kBlockBytes);
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
                  if (c / 8 < rows) ctl->bad[place] = w.number;
                }
              }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          }
          ok = !named_any(3, 64, !ok);
          if (ok && tid == 0) mbar_arrive(&ctl->full[slot]);
        }
        if (!ok) break;
        entry0 = (entry0 + 2 * total) % kRing;
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl->work_empty[place]);
        if (++place == kQueue) { place = 0; place_phase ^= 1u; }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // ------------------------------------------------------------------ softmax
    const int half = warp >> 2, r = threadIdx.x & 127;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_tmem = tmem + lanes + half * 128, o_tmem = tmem + lanes + 256 + half * 128;
    constexpr float kLog2e = 1.4426950408889634f;
    // cap in log2 domain; s / c of a product, finite so that a score of zero stays zero with a cap of next to nothing
    const float cap2 = a.cap * kLog2e, to_y = a.cap > 0.f ? fminf(a.scale / a.cap, 1e30f) : 0.f;
    const float sl2 = a.scale * kLog2e;
    const bool score = a.cap > 0.f || a.slopes;       // scores are rewritten, in log2 domain then
    const float sl = score ? 1.0f : sl2;
    int place = 0;
    uint32_t place_phase = 0, s_phase = 0, o_phase = 0;
    bool ok = true;
    // What a thread needs to know of its row.  Asked for anew wherever it is needed: the loop over the tiles has no register
    // to spare for it.
    struct Row {
      int tok, head;
      bool ok;
      int64_t limit;       // keys of the past that it sees
      uint64_t bits;       // drafted tokens that it sees
    };
    const int row_tok = r / p.group, row_head = r % p.group;
    auto row_of = [&](const Work& w) {
      asm volatile("" ::: "memory");
      Row x;
      x.tok = w.tok0 + (p.pair ? half * p.tokens : 0) + row_tok;
      x.ok = r < rows_tile && x.tok < w.s.n;
      x.head = w.h * p.group + row_head;
      x.limit = x.ok ? visible(a, w.s, x.tok) : 0;
      x.bits = a.tree_mask && x.ok ? (uint64_t)__ldcg(a.tree_mask + w.s.q0 + x.tok) : 0ull;
      if (w.s.n < kTreeLimit) x.bits &= (1ull << w.s.n) - 1;           // bits behind the sequence's tokens mean nothing
      return x;
    };
    // Cap, distance bias and mask: the scores of a tile as they have to be, written back to tensor memory.  A pass of its own
    // in a loop that is not unrolled, run only where there is something to do: the hot loop is as long as the instruction
    // caches can bear (8192 capped tokens, otherwise alike: 961 us so, 1184 us with the same arithmetic unrolled in it; code that
    // was merely skipped cost a fifth).
    auto adjust = [&](const Work& w, int t, int whole, float slope2, float place_of_row, float to_vote) {
      uint32_t seen[4] = {0xFFFFFFFFu, 0xFFFFFFFFu, 0xFFFFFFFFu, 0xFFFFFFFFu};
      if (t >= whole) {
        const Row row = row_of(w);
        const int64_t left = row.limit - (int64_t)t * kTile;
        const bool drafted = t == w.drafted;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int n = left < 32 * k ? 0 : (left >= 32 * k + 32 ? 32 : (int)left - 32 * k);
          seen[k] = n == 32 ? 0xFFFFFFFFu : (1u << n) - 1u;
          if (drafted) seen[k] = k == 0 ? (uint32_t)row.bits : (k == 1 ? (uint32_t)(row.bits >> 32) : 0u);
        }
      }
      const f32x2 sc = a.cap > 0.f || !score ? pair2(1.f, 1.f) : pair2(sl2, sl2);
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        uint32_t raw[32];
        float* x = reinterpret_cast<float*>(raw);
        tmem_ld32(s_tmem + c * 32, raw);
        tmem_wait_ld32(raw);
        const uint32_t bits = c < 2 ? (c == 0 ? seen[0] : seen[1]) : (c == 2 ? seen[2] : seen[3]);
        if (a.cap > 0.f) {
          auto largest = [&]() {             // NaN left out
            float big = 0.f;
#pragma unroll
            for (int j = 0; j < 32; j += 2) big = max3_number(big, fabsf(x[j]), fabsf(x[j + 1]));
            return big;
          };
          // The warp votes for a form by what its rows see.  The forms round differently, so what a row may not see must not
          // count, nor lanes without a row, which hold the next sequence's or what was in shared memory before (their to_vote
          // is 0).  And the last form's scores share a reciprocal, through which a hidden NaN would reach a visible one.
          // Both are seen to where the vote is not for the short form at once, out of the usual way (32 capped trees of 16
          // over 4096 rows: 110 us without it, 116 so, 119 with all hidden scores set to zero first; 8192 capped tokens: 726,
          // 734, 740).  Each row by itself would leave its neighbours out too, but takes a third longer near the cap.
          float big = largest();
          bool near = __all_sync(0xFFFFFFFFu, !(big * to_vote > 0.4f));
          if (!near) {
            if (bits != 0xFFFFFFFFu) {
#pragma unroll
              for (int j = 0; j < 32; ++j) x[j] = bits & (1u << j) ? x[j] : 0.f;
              big = largest();
            }
            near = __all_sync(0xFFFFFFFFu, !(big * to_vote > 0.4f));
          }
          if (near) {
            // |s| <= 0.4 c, as almost everywhere: the short polynomial (8192 capped tokens: 730 us, 80 us more without it)
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              const f32x2 xx = pair2(x[j], x[j + 1]);
              unpair2(mul2(mul2(xx, pair2(sl2, sl2)), tanh_over_y_near(mul2(xx, pair2(to_y, to_y)))), x[j], x[j + 1]);
            }
          } else if (__all_sync(0xFFFFFFFFu, !(big * to_vote > 1.0f))) {
            // tanh by its polynomial, off the special function unit
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              const f32x2 xx = pair2(x[j], x[j + 1]);
              unpair2(mul2(mul2(xx, pair2(sl2, sl2)), tanh_over_y(mul2(xx, pair2(to_y, to_y)))), x[j], x[j + 1]);
            }
          } else {
            // c - 2 c / (exp(2 s / c) + 1), two quotients by one reciprocal of the product; 2^60 is as good as
            // infinity here and leaves the product finite
            const float to_cap = 2.0f * kLog2e * to_y;
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              const float d0 = ex2(min_nan(x[j] * to_cap, 60.f)) + 1.0f, d1 = ex2(min_nan(x[j + 1] * to_cap, 60.f)) + 1.0f;
              const float q = rcp(d0 * d1) * (-2.0f * cap2);
              x[j] = fmaf(q, d1, cap2);
              x[j + 1] = fmaf(q, d0, cap2);
            }
          }
        }
        if (BIAS) {
          const float at = place_of_row - (float)((t - w.t0) * kTile + 32 * c);
          if (__all_sync(0xFFFFFFFFu, at >= 31.f)) {
            // all 32 keys lie before all rows: the bias climbs by the slope from key to key
            f32x2 b0 = pair2(-slope2 * at, -slope2 * (at - 1.f)), b1 = pair2(-slope2 * (at - 2.f), -slope2 * (at - 3.f));
            const f32x2 up = pair2(4.f * slope2, 4.f * slope2);
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
              unpair2(fma2(pair2(x[j], x[j + 1]), sc, b0), x[j], x[j + 1]);
              unpair2(fma2(pair2(x[j + 2], x[j + 3]), sc, b1), x[j + 2], x[j + 3]);
              b0 = add2(b0, up);
              b1 = add2(b1, up);
            }
          } else {
            const float one = a.cap > 0.f ? 1.0f : sl2;
#pragma unroll
            for (int j = 0; j < 32; ++j) x[j] = fmaf(-slope2, fabsf(at - (float)j), x[j] * one);
          }
        }
        if (bits != 0xFFFFFFFFu) {
#pragma unroll
          for (int j = 0; j < 32; ++j) x[j] = bits & (1u << j) ? x[j] : -INFINITY;
        }
        __syncwarp();
        tmem_st32(s_tmem + c * 32, raw);
      }
      tmem_wait_st();
    };
    for (;;) {
      ok = __all_sync(0xFFFFFFFFu, wait_bar(&ctl->work_full[place], place_phase, ctl, 11, 0));
      if (!p.pair) ok = !named_any(4, 256, !ok);     // the two halves leave together
      if (!ok) break;
      const Work& w = ctl->work[place];
      if (w.h < 0) break;
      const int mine = p.pair ? w.nt[half] : (tiles_of(w) + 1 - half) / 2;
      // all rows of this half see the tiles below this one whole
      const int whole = p.pair && half && w.halves == 2 ? (int)(visible(a, w.s, w.tok0 + p.tokens) / kTile) : w.partial;
      float slope2 = 0.f, place_of_row = 0.f;                         // of the row; its place among the item's keys
      if (BIAS) {
        const Row row = row_of(w);
        if (row.ok) slope2 = __ldcg(a.slopes + row.head) * kLog2e;
        place_of_row = (float)(row.tok + w.s.shift - (int64_t)w.t0 * kTile);
      }
      // s / c of a product, for the vote in adjust(): 0 in lanes without a row
      const float to_vote = r < rows_tile && w.tok0 + (p.pair ? half * p.tokens : 0) + row_tok < w.s.n ? to_y : 0.f;
      float m = -INFINITY, l = 0.f;                                   // m: in log2 domain
      const int t_step = p.pair ? 1 : 2;
      int t = w.t0 + (p.pair ? 0 : half);
      for (int i = 0; i < mine; ++i, t += t_step) {
        ok = __all_sync(0xFFFFFFFFu, wait_bar(&ctl->s_full[half], s_phase, ctl, 5, t));
        s_phase ^= 1u;
        if (!ok) break;
        tc_fence_after();
        const float at = place_of_row - (float)((t - w.t0) * kTile);      // the row, from the tile's first key
        const bool linear = BIAS && a.cap == 0.f && t < whole && __all_sync(0xFFFFFFFFu, at >= (float)(kTile - 1));
        if ((score && !linear) || t >= whole) adjust(w, t, whole, slope2, place_of_row, to_vote);
        uint32_t raw[128];
        float* x = reinterpret_cast<float*>(raw);
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(s_tmem + c * 32, raw + 32 * c);
        float mx = -INFINITY, mx1 = -INFINITY;
        const float slope_t = linear ? slope2 : 0.f, sl_t = BIAS && linear ? sl2 : sl;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          tmem_wait_ld32(raw + 32 * c);
          if (BIAS) {                          // as above, 32 keys at a time
            const float ac = at - 32.f * (float)c;
            f32x2 b0 = pair2(-slope_t * ac, -slope_t * (ac - 1.f)), b1 = pair2(-slope_t * (ac - 2.f), -slope_t * (ac - 3.f));
#pragma unroll
            for (int j = 32 * c; j < 32 * c + 32; j += 4) {
              unpair2(fma2(pair2(x[j], x[j + 1]), pair2(sl_t, sl_t), b0), x[j], x[j + 1]);
              unpair2(fma2(pair2(x[j + 2], x[j + 3]), pair2(sl_t, sl_t), b1), x[j + 2], x[j + 3]);
              b0 = add2(b0, pair2(4.f * slope_t, 4.f * slope_t));
              b1 = add2(b1, pair2(4.f * slope_t, 4.f * slope_t));
            }
          }
#pragma unroll
          for (int j = 32 * c; j < 32 * c + 32; j += 4) {
            mx = max3(mx, x[j], x[j + 1]);
            mx1 = max3(mx1, x[j + 2], x[j + 3]);
          }
        }
        mx = max_nan(mx, mx1);
        if (!BIAS) mx *= sl;
        if (i == 0) {
          m = mx;
        } else {
          const bool moves = !(mx <= m + kLazy<T>) && !(m == INFINITY);
          if (__any_sync(0xFFFFFFFFu, moves)) {
            const float f = moves && m != mx ? ex2(m - mx) : 1.0f;
            m = moves ? mx : m;
            l *= f;
#pragma unroll 1
            for (int c = 0; c < DP; c += 32) {
              uint32_t o[32];
              tmem_ld32(o_tmem + c, o);
              tmem_wait_ld32(o);
#pragma unroll
              for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
              tmem_st32(o_tmem + c, o);
            }
          }
        }
        // -inf: nothing seen so far; +inf: inf - inf, NaN for the whole row
        const float base = m == -INFINITY ? 0.f : (m == INFINITY ? __int_as_float(0x7FC00000) : m - kScaleUp<T>);
        f32x2 sum = pair2(0.f, 0.f), sum1 = sum;
        auto probabilities = [&](int c) {      // exponentials and sum of 32 scores, and their probabilities into tensor memory
          const f32x2 nb = pair2(-base, -base), sc = pair2(sl, sl);
          uint32_t pk[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const f32x2 xx = pair2(x[32 * c + 2 * j], x[32 * c + 2 * j + 1]);
            float e0, e1;
            unpair2(BIAS ? add2(xx, nb) : fma2(xx, sc, nb), e0, e1);
            e0 = ex2(e0);
            e1 = ex2(e1);
            if (j & 1) sum = add2(sum, pair2(e0, e1));
            else sum1 = add2(sum1, pair2(e0, e1));
            pk[j] = pack2<T>(e0, e1);
          }
          tmem_st16u(s_tmem + c * 16, pk);
        };
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          probabilities(c);
          if (c & 1) {
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ctl->p_ready[half][c >> 1]);
          }
        }
        sum = add2(sum, sum1);
        float s0, s1;
        unpair2(sum, s0, s1);
        l += s0 + s1;
      }
      // ---- the end of the item: the products of this half are done
      if (ok && mine > 0) {
        ok = __all_sync(0xFFFFFFFFu, wait_bar(&ctl->o_full[half], o_phase, ctl, 6, w.number));
        o_phase ^= 1u;
      }
      tc_fence_after();
      const Row row = row_of(w);
      const int total = tiles_of(w);
      const bool row_ok = row.ok;
      const int64_t out_row = (w.s.q0 + row.tok) * a.Hq + row.head;
      // Whether a value was replaced is known once the products of ALL of a row's tiles are done: here where a row's tiles
      // belong to one half, behind the meeting of the halves where they share them.
      bool bad = ctl->bad[place] == w.number;
      auto store = [&](Cols8& x, int col, float inv, float* part) {       // 8 columns of this row
        if (bad) x = add_bad<T>(x, &a, &w, col, row.limit, row.bits, total);
        if (!part) {
#pragma unroll
          for (int e = 0; e < 8; ++e) x.v[e] *= inv;
          *reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.out) + out_row * a.D + col) = pack16<T>(x.v);
        } else {
          reinterpret_cast<float4*>(part + col)[0] = make_float4(x.v[0], x.v[1], x.v[2], x.v[3]);
          reinterpret_cast<float4*>(part + col)[1] = make_float4(x.v[4], x.v[5], x.v[6], x.v[7]);
        }
      };
      if (p.pair) {
        if (!ok) break;
        if (half < w.halves) {
          const float inv = l == 0.f ? 0.f : 1.0f / l;
          float* part = nullptr;
          if (w.slot >= 0) {
            const int64_t at = (int64_t)w.slot * a.Tq * a.Hq + out_row;
            part = p.part_o + at * a.D;
            if (row_ok) p.part_ml[at] = make_float2(m, l);
          }
#pragma unroll 1
          for (int c = 0; c < DP; c += 32) {
            uint32_t o[32];
            tmem_ld32(o_tmem + c, o);
            tmem_wait_ld();
            if (mine == 0) {
#pragma unroll
              for (int j = 0; j < 32; ++j) o[j] = 0u;
            }
#pragma unroll
            for (int j = 0; j < 32; j += 8) {
              Cols8 x;
#pragma unroll
              for (int e = 0; e < 8; ++e) x.v[e] = __uint_as_float(o[j + e]);
              if (row_ok && c + j < a.D) store(x, c + j, inv, part);
            }
          }
        }
      } else {
        // each half finishes its share of the columns; a row's lane is the same in both
        ctl->ml[half * 128 + r] = make_float2(m, l);
        tc_fence_before();
        ok = !named_any(4, 256, !ok);
        if (!ok) break;
        tc_fence_after();
        bad = ctl->bad[place] == w.number;
        const float2 other = ctl->ml[(half ^ 1) * 128 + r];
        const float top = fmaxf(m, other.x);
        const float f0 = m == -INFINITY ? 0.f : ex2(m - top), f1 = other.x == -INFINITY ? 0.f : ex2(other.x - top);
        const float sum = l * f0 + other.y * f1;
        const float inv = sum == 0.f ? 0.f : 1.0f / sum;
        const bool other_has = half ? total > 0 : total > 1;
        float* part = nullptr;
        if (w.slot >= 0) {
          part = p.part_o + ((int64_t)w.slot * 128 + r) * a.D;
          if (half == 0) p.part_ml[(int64_t)w.slot * 128 + r] = make_float2(top, sum);
        }
#pragma unroll 1
        for (int c = half * (DP / 2); c < (half + 1) * (DP / 2); c += 32) {
          uint32_t o[32], g[32];
          // loaded whether there is a result or not: a conditional load would keep its 64 registers from the tile loop
          tmem_ld32(o_tmem + c, o);
          tmem_ld32(tmem + lanes + 256 + (half ^ 1) * 128 + c, g);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            Cols8 x;
#pragma unroll
            for (int e = 0; e < 8; ++e)
              x.v[e] = (mine > 0 ? __uint_as_float(o[j + e]) * f0 : 0.f) + (other_has ? __uint_as_float(g[j + e]) * f1 : 0.f);
            if (row_ok && c + j < a.D) store(x, c + j, inv, part);
          }
        }
        tc_fence_before();
        named_sync(4, 256);            // both have read before the next item's products overwrite
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl->work_empty[place]);
      if (++place == kQueue) { place = 0; place_phase ^= 1u; }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(ctl->tmem, 512);
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
    uint2 v;
    v.x = pack2<T>(acc.x * inv, acc.y * inv);
    v.y = pack2<T>(acc.z * inv, acc.w * inv);
    *reinterpret_cast<uint2*>(out + row * D + lane * 4) = v;
  }
}

// The same for items whose key tiles were dealt out: WARPS warps per row share the pieces of its item.  One warp up to
// four pieces, whose loads are all under way at once, for the rows of the at most one item that each CTA began and others
// ended (looking up what each row of the call needs took 4 us more of 92 with 32 sequences, 40 of 178 with 128).
// Beyond four pieces a block for every row, as a single warp would wait for memory once for every four (one row over 100 000
// keys, 148 pieces: 30 us, 48 us with one warp; eight drafted tokens over 12 000: 18 and 27).
template <typename T, int WARPS>
__global__ void __launch_bounds__(256) masked_attention_join_kernel(const __grid_constant__ TcArgs p) {
  __shared__ float4 shares[WARPS > 1 ? 8 : 1][32];
  __shared__ float sums[8];
  pdl_launch_dependents();
  pdl_wait();
  const AttnArgs& a = p.a;
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5, part = warp % WARPS;
  int2 who;
  int r;
  int64_t row;
  if (WARPS == 1) {                                // rows of the item that a CTA began and others ended
    const int4 cut = __ldcg(p.cuts + blockIdx.y);
    r = (int)blockIdx.x * 8 + warp;
    if (r >= cut.y) return;
    who = make_int2((int)blockIdx.y, cut.w);
    row = (int64_t)(cut.x + r / p.group) * a.Hq + cut.z * p.group + r % p.group;
  } else {                                         // all rows
    row = blockIdx.x;
    const int64_t t = row / a.Hq;
    // the row's sequence: the last that begins at or before it
    int before = 0, start = 0;
    for (int i = lane; i <= a.B; i += 32) {
      const int64_t v = __ldcg(a.seqstarts + i);
      if (v <= t) {
        ++before;
        start = v > start ? (int)v : start;
      }
    }
    const int b = __reduce_add_sync(0xFFFFFFFFu, before) - 1;
    const int head = (int)(row - t * a.Hq), h = head / p.group;
    const int64_t i = t - __reduce_max_sync(0xFFFFFFFFu, start);
    if (b < 0 || b >= a.B || i >= a.max_seqlen) return;
    who = __ldcg(p.pieces + (int64_t)b * a.Hkv + h);
    // In one piece: the result is there.  Starts that do not rise can lead to a sequence without an item, whose entry was
    // never written.
    if (who.x < 0 || who.x >= who.y || who.y >= p.ctas) return;
    r = (int)i * p.group + head % p.group;
  }
  const int n = who.y - who.x + 1;                 // pieces, of which this warp takes every WARPS-th
  auto place = [&](int c) { return (int64_t)(c == 0 ? 2 * who.x + 1 : 2 * (who.x + c)) * 128 + r; };
  auto stat = [&](int c) { return c < n ? __ldcg(p.part_ml + place(c)) : make_float2(-INFINITY, 0.f); };
  auto values = [&](int c) {
    return c < n && lane * 4 < a.D ? __ldcg(reinterpret_cast<const float4*>(p.part_o + place(c) * a.D) + lane) : make_float4(0.f, 0.f, 0.f, 0.f);
  };
  // a lane has the maximum and sum of one of the warp's pieces; results are loaded four pieces ahead of what their factors
  // wait for
  float2 ml = stat(part + lane * WARPS);
  float4 v[4] = {values(part), values(part + WARPS), values(part + 2 * WARPS), values(part + 3 * WARPS)};
  float top = ml.x;
  for (int c = WARPS > 1 ? lane : lane + 32; c < n; c += 32) top = fmaxf(top, stat(c).x);
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
  float sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int c0 = 0; part + c0 * WARPS < n; c0 += 4) {
    if (c0 && (c0 & 31) == 0) ml = stat(part + (c0 + lane) * WARPS);
    const float f_lane = ml.x == -INFINITY ? 0.f : ex2(ml.x - top);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int from = (c0 & 31) + k;
      const float f = __shfl_sync(0xFFFFFFFFu, f_lane, from), l = __shfl_sync(0xFFFFFFFFu, ml.y, from);
      const bool some = __shfl_sync(0xFFFFFFFFu, ml.x, from) != -INFINITY;
      const float4 x = v[k];
      v[k] = values(part + (c0 + 4 + k) * WARPS);
      if (some) {
        sum = fmaf(l, f, sum);
        acc.x = fmaf(x.x, f, acc.x);
        acc.y = fmaf(x.y, f, acc.y);
        acc.z = fmaf(x.z, f, acc.z);
        acc.w = fmaf(x.w, f, acc.w);
      }
    }
  }
  if (WARPS > 1) {
    shares[warp][lane] = acc;
    sums[warp] = sum;
    __syncthreads();                // all warps of the block have the same row, none has left
    if (part) return;
    for (int o = 1; o < WARPS; ++o) {
      const float4 x = shares[o][lane];
      acc.x += x.x;
      acc.y += x.y;
      acc.z += x.z;
      acc.w += x.w;
      sum += sums[o];
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  if (lane * 4 < a.D) {
    uint2 v;
    v.x = pack2<T>(acc.x * inv, acc.y * inv);
    v.y = pack2<T>(acc.z * inv, acc.w * inv);
    *reinterpret_cast<uint2*>(reinterpret_cast<T*>(a.out) + row * a.D + lane * 4) = v;
  }
}

// ------------------------------------------------------------------------------------------------- host side
struct TcPlan {
  bool use;
  int group, tokens, pair, row_blocks, splits, flat, grid, pieces;
};

// Everything that sizes the workspace and the grid follows from shapes and host lengths alone.
TcPlan plan_tc(int64_t Tq, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_seqlen, int64_t max_kvlen, int dtype) {
  TcPlan pl{};
  if ((dtype != PMX_DTYPE_F16 && dtype != PMX_DTYPE_BF16) || D % 8 || D > 128 || Hkv <= 0 ||
      Hq % Hkv || Hq / Hkv > kTile)
    return pl;
  if (Tq <= 0 || B <= 0 || Hq <= 0 || D <= 0 || max_seqlen <= 0 || max_kvlen <= 0 || Tq >= (1ll << 31)) return pl;
  if (max_seqlen > Tq) max_seqlen = Tq;
  if (max_kvlen > (1ll << 31)) max_kvlen = 1ll << 31;      // more rows than tensors have here; products below stay in range
  pl.group = (int)(Hq / Hkv);
  pl.tokens = kTile / pl.group;
  pl.pair = max_seqlen > pl.tokens;
  const int64_t blocks = ceil_div(max_seqlen, pl.pair ? 2 * pl.tokens : pl.tokens);
  const int64_t items = blocks * B * Hkv, tiles = ceil_div(max_kvlen, kTile) + 1;      // + 1: drafted tokens
  if (items > (1 << 24) || B > (1 << 20)) return pl;
  pl.row_blocks = (int)blocks;
  const int64_t sms = sm_count();
  int64_t grid;
  if (pl.pair) {
    // Split the keys while that fills SMs that would idle, with enough key tiles left for each: below that the start of an
    // item and the merge cost more than the shorter walk gains.
    int64_t s = sms / items;
    if (s > tiles / kMinTiles) s = tiles / kMinTiles;
    pl.splits = (int)(s < 1 ? 1 : (s > kMaxSplits ? kMaxSplits : s));
    grid = items * pl.splits;
  } else {
    pl.splits = 1;
    pl.flat = tiles > kMinTiles;
    grid = pl.flat ? ceil_div(items * tiles, kFlatTiles) : items;
  }
  pl.grid = (int)(grid < sms ? grid : sms);
  const int64_t each = ceil_div(items * tiles, pl.grid);           // key tiles of a CTA
  pl.pieces = (int)ceil_div(tiles, each < kFlatTiles ? kFlatTiles : each);
  pl.use = true;
  return pl;
}

// 16-byte aligned parts: maximum and sum, results, and who shares an item
size_t tc_workspace(const TcPlan& pl, int64_t Tq, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, size_t* o_at = nullptr,
                    size_t* pieces_at = nullptr, size_t* cuts_at = nullptr) {
  if (!pl.use || (pl.splits == 1 && !pl.flat)) return 0;
  const size_t rows = pl.flat ? (size_t)pl.grid * 2 * kTile : (size_t)pl.splits * Tq * Hq;
  const size_t o = (rows * sizeof(float2) + 15) & ~(size_t)15, pieces = o + rows * D * sizeof(float);
  if (o_at) *o_at = o;
  if (pieces_at) *pieces_at = pieces;
  const size_t cuts = (pieces + (size_t)B * Hkv * sizeof(int2) + 15) & ~(size_t)15;
  if (cuts_at) *cuts_at = cuts;
  return pl.flat ? cuts + (size_t)pl.grid * sizeof(int4) : pieces;
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
int launch_tc_t(const TileMaps& maps, const TcArgs& p, int grid, cudaStream_t s) {
  const void* kern = p.a.slopes ? (const void*)masked_attention_kernel<T, DP, true> : (const void*)masked_attention_kernel<T, DP, false>;
  const size_t smem = (size_t)(2 + kRing) * kTile * DP * 2 + sizeof(Ctl);
  static_assert((2 + kRing) * kTile * DP * 2 + sizeof(Ctl) <= 227 * 1024, "shared memory of an SM");
  PMX_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  void* args[] = {(void*)&maps, (void*)&p};
  const int st = launch_pdl(kern, dim3((unsigned)grid), dim3(kAttnThreads), smem, s, args);
  if (st != PMX_OK || (p.splits == 1 && !p.flat)) return st;
  const int64_t rows = p.a.Tq * p.a.Hq;
  const dim3 merge_grid((unsigned)ceil_div(rows, 8)), merge_block(256);
  if (p.flat && p.pieces_of_item > 4 && p.a.Tq * p.a.Hq < (1ll << 31))      // a block per row
    return launch_pdl_k(masked_attention_join_kernel<T, 8>, dim3((unsigned)(p.a.Tq * p.a.Hq)), merge_block, 0, s, p);
  const int64_t most = (int64_t)p.a.max_seqlen * p.group;          // rows of an item
  if (p.flat) return launch_pdl_k(masked_attention_join_kernel<T, 1>, dim3((unsigned)ceil_div(most < kTile ? most : kTile, 8), (unsigned)p.ctas), merge_block, 0, s, p);
  return launch_pdl_k(masked_attention_merge_kernel<T>, merge_grid, merge_block, 0, s, (const float*)p.part_o,
                      (const float2*)p.part_ml, (T*)p.a.out, rows, p.a.D, p.splits);
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
  p.flat = pl.flat;
  p.ctas = pl.grid;
  p.pieces_of_item = pl.pieces;
  int64_t grid = pl.grid;
  if (a.tree_mask && grid < ceil_div(a.Tq, 2)) grid = ceil_div(a.Tq, 2) < sm_count() ? ceil_div(a.Tq, 2) : sm_count();
  size_t o_at = 0, pieces_at = 0, cuts_at = 0;
  tc_workspace(pl, a.Tq, a.B, a.Hq, a.Hkv, a.D, &o_at, &pieces_at, &cuts_at);
  p.part_ml = reinterpret_cast<float2*>(ws);
  p.part_o = reinterpret_cast<float*>((char*)ws + o_at);
  p.pieces = reinterpret_cast<int2*>((char*)ws + pieces_at);
  p.cuts = reinterpret_cast<int4*>((char*)ws + cuts_at);
  TileMaps m{};
  int st = make_head_map(&m.q, a.q, a.Tq, a.Hq, a.D, a.q_tok, a.q_head, (uint32_t)pl.group, (uint32_t)pl.tokens, dtype, name);
  if (st == PMX_OK) st = make_head_map(&m.k, a.past.k, a.past.rows, a.Hkv, a.D, a.past.k_row, a.past.k_head, 1, kTile, dtype, name);
  if (st == PMX_OK) st = make_head_map(&m.v, a.past.v, a.past.rows, a.Hkv, a.D, a.past.v_row, a.past.v_head, 1, kTile, dtype, name);
  if (st == PMX_OK && a.tree_mask) st = make_head_map(&m.ck, a.cur.k, a.cur.rows, a.Hkv, a.D, a.cur.k_row, a.cur.k_head, 1, kTreeLimit, dtype, name);
  if (st == PMX_OK && a.tree_mask) st = make_head_map(&m.cv, a.cur.v, a.cur.rows, a.Hkv, a.D, a.cur.v_row, a.cur.v_head, 1, kTreeLimit, dtype, name);
  if (st != PMX_OK) return st;
  const bool bf = dtype == PMX_DTYPE_BF16;
  if (a.D <= 64) return bf ? launch_tc_t<__nv_bfloat16, 64>(m, p, (int)grid, s) : launch_tc_t<__half, 64>(m, p, (int)grid, s);
  return bf ? launch_tc_t<__nv_bfloat16, 128>(m, p, (int)grid, s) : launch_tc_t<__half, 128>(m, p, (int)grid, s);
}
