// Attention of chunks over a page pool on the tcgen05 tensor cores (bf16,
// fp16; head_dim 64 and 128).  The operator is avq_paged_attn.cu's; this
// kernel takes the sequences with more than kFewRows rows.
//
// The rows of one (sequence, key head) are its (token, head of the group)
// pairs, token by token, so that a key tile serves the whole group and short
// chunks of many heads fill the tensor core's 128 rows.  A CTA works on 256
// rows, two tiles of 128 that take turns: while the tensor cores multiply one
// tile's scores or values, the other tile's threads work on its softmax.
//
//   warps 0-3, 4-7  softmax of tile 0 / 1, a thread per row: S from TMEM, the
//                   running maximum, p = exp2(s - m), P to TMEM (the columns
//                   of S), the row's sum; O is rescaled in TMEM only when the
//                   maximum grew by more than 2^8 (the sums stay exact: P and
//                   l refer to the same, older maximum)
//   warp 8          issues S = Q K^T and O += P V
//   warps 9-11      load Q (by TMA where the heads of a group divide 128, else
//                   by cp.async) and the key and value tiles (128 keys each)
//                   into a ring, in the 128-byte swizzled layout that the
//                   tensor cores read: warps 9 and 10 by TMA where whole pages
//                   fill a tile or whole tiles a page (page sizes 8, 16, .. 128
//                   and multiples of 128), else all three by cp.async, where a
//                   page may begin and end anywhere in a tile
//
// Work: plan_kernel lists the (sequence, 256 rows) items and their key tiles,
// cuts the (key head, item) pairs into pieces that get smaller toward the end,
// and the persistent CTAs fetch pieces by an atomic counter (which CTA takes a
// piece has no influence on its result).  Pieces of one pair are joined by
// combine_tc_kernel in the order of the keys.
//
// Every wait is bounded (avq_tc.cuh).
#include <cuda.h>

#include <algorithm>
#include <cstring>
#include <type_traits>

#include "avq_mma.cuh"
#include "avq_paged.cuh"
#include "avq_tc.cuh"

namespace avq {

namespace {

// Bit 0: a CTA gave up on a bounded wait; bit 1: the batch's lists are not sound.
__device__ int g_fault_paged_tc;

constexpr int TM = 128, TK = 128;  // rows of a tile, keys of a tile
constexpr int kItemRows = 2 * TM;
constexpr int kTcThreads = 384, kLoaders = 3, W_MMA = 8, W_LOAD = 9;
constexpr int kMaxSlots = 8 * kSms;    // pieces of split pairs, each with a slot of partial sums
constexpr int kMaxPieces = kSms;       // of a pair
constexpr float kLazy = 8.f;           // log2 of the growth that rescales O

template <int D> constexpr int ring_slots() { return D == 128 ? 5 : 8; }
template <int D> constexpr int tile_bytes() { return TK * D * 2; }

// What a CTA needs to know of a piece.
struct __align__(16) PieceWork {
  int head, seq, row0, rows;      // key head, sequence; first row in it, rows from there on
  int key0, tiles, pieces, slot;  // first key, key tiles; pieces of its pair, its slot of partial sums
  int q0, pos0, len, end;         // the sequence's first token and its position; its keys, those that the rows see
  int pair, first;                // first key that any row sees, in the tile of the pair's first key
  int unused[2];
};

// The plan in the workspace: a header; the pieces; the items; the (key head, item) pairs, head by head.
struct Plan {
  int* head;         // [0] pieces, [1] the next piece to fetch, [2] items
  PieceWork* piece;  // [pieces]
  int* base;         // [B + 1] first item of each sequence
  int* seq;          // [items] sequence
  int* part;         // index of the 256-row part in it
  int* tiles;        // key tiles
  int* sum;          // key tiles of the items before
  int* split;        // [pairs] pieces
  int* slot;         // [pairs] first slot of partial sums, where there are several pieces
  unsigned* odd;     // [pairs][8] a bit for each row whose sums are not finite where keys that it does not see may be why
};

__host__ __device__ inline long long plan_ints(long long B, long long items, long long Hkv) {
  return 8 + (items * Hkv + kMaxSlots) * (long long)(sizeof(PieceWork) / 4) + (B + 1) + 4 * items + (2 + kItemRows / 32) * items * Hkv;
}
__host__ __device__ inline Plan plan_at(int* p, long long B, long long items, long long Hkv) {
  Plan q;
  q.head = p;
  q.piece = reinterpret_cast<PieceWork*>(p + 8);
  q.base = reinterpret_cast<int*>(q.piece + items * Hkv + kMaxSlots);
  q.seq = q.base + B + 1;
  q.part = q.seq + items;
  q.tiles = q.part + items;
  q.sum = q.tiles + items;
  q.split = q.sum + items;
  q.slot = q.split + items * Hkv;
  q.odd = reinterpret_cast<unsigned*>(q.slot + items * Hkv);
  return q;
}

// Keys of a 256-row item: [lo, hi), lo a multiple of TK.
__device__ __forceinline__ int2 item_keys(const PagedAttnArgs& a, const SeqRange& s, int part, int G) {
  const long long r0 = (long long)part * kItemRows, r1 = min((long long)s.n * G, r0 + kItemRows) - 1;
  const int lo = window_start(a, s.pos0 + (int)(r0 / G)) / TK * TK;
  const int hi = a.causal ? max(0, min(s.len, s.pos0 + (int)(r1 / G) + 1)) : s.len;
  return make_int2(lo, max(lo, hi));
}

// ---- the plan ---------------------------------------------------------------------------

constexpr int kPlanThreads = 256;  // (1024 take 1 us longer: their barriers)

// Exclusive prefix of v over the block; *total receives the sum.
__device__ int block_prefix(int v, int* total) {
  __shared__ int s_warp[kPlanThreads / 32];
  __shared__ int s_total;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) s_warp[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int w = lane < kPlanThreads / 32 ? s_warp[lane] : 0;
    const int own = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    if (lane < kPlanThreads / 32) s_warp[lane] = w - own;
    if (lane == 31) s_total = w;
  }
  __syncthreads();
  *total = s_total;
  return s_warp[warp] + x - v;
}

__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const PagedAttnArgs a, int row_min, int max_items,
                                                            int* __restrict__ ws) {
  Plan p = plan_at(ws, a.B, max_items, a.Hkv);
  // what the plan itself reads again stays in shared memory where it fits (a round trip to memory for each of the
  // plan's steps would be most of its time); the joining kernel reads `seq` and `part` from the workspace
  constexpr int kHeld = 1024;
  __shared__ int s_base[kHeld + 1], s_seq[kHeld], s_part[kHeld], s_tiles[kHeld], s_sum[kHeld];
  int *const out_seq = p.seq, *const out_part = p.part;
  if (a.B <= kHeld && max_items <= kHeld) {
    p.base = s_base;
    p.seq = s_seq;
    p.part = s_part;
    p.tiles = s_tiles;
    p.sum = s_sum;
  }
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, G = a.H / a.Hkv;
  const long long room = (long long)a.W * a.page_size;
  asm volatile("griddepcontrol.launch_dependents;");
  bool bad = false;
  int items = 0;
  long long beside = 0;  // what the kernel of few rows does, in key tiles that take the tensor cores as long
  for (int b0 = 0; b0 < a.B; b0 += kPlanThreads) {
    const int b = b0 + tid;
    int parts = 0, few = 0;
    if (b < a.B) {
      const SeqRange s = load_seq(a.q_start, a.kv_len, b, a.N, room, &bad);
      const long long rows = (long long)s.n * G;
      parts = rows > row_min ? (int)((rows + kItemRows - 1) / kItemRows) : 0;
      if (rows > 0 && parts == 0) {
        const int keys = s.len - min(s.len, window_start(a, s.pos0));
        few = (int)min((long long)keys * a.Hkv * a.D / (TK * 128), 1ll << 20);
      }
    }
    int total, total_few;
    const int at = items + block_prefix(parts, &total);
    block_prefix(few, &total_few);
    if (b < a.B) p.base[b] = min(at, max_items);
    items += total;
    beside += total_few;
  }
  // token ranges that overlap could name more items than the batch has rows for
  if (items > max_items) bad = true;
  items = min(items, max_items);
  if (tid == 0) {
    p.base[a.B] = items;
    p.head[2] = items;
  }
  if (bad) atomicOr(&g_fault_paged_tc, kFaultTables);
  __syncthreads();
  for (int b = warp; b < a.B; b += kPlanThreads / 32) {
    const int i0 = p.base[b], n = p.base[b + 1] - i0;
    if (n == 0) continue;
    const SeqRange s = load_seq(a.q_start, a.kv_len, b, a.N, room, &bad);
    for (int i = lane; i < n; i += 32) {
      const int part = n - 1 - i;  // the last rows see the most keys: longest first
      const int2 k = item_keys(a, s, part, G);
      p.seq[i0 + i] = out_seq[i0 + i] = b;
      p.part[i0 + i] = out_part[i0 + i] = part;
      p.tiles[i0 + i] = max(1, (k.y - k.x + TK - 1) / TK);
    }
  }
  __syncthreads();
  int head_tiles = 0;  // key tiles of one head
  for (int i0 = 0; i0 < items; i0 += kPlanThreads) {
    const int i = i0 + tid;
    int total;
    const int at = head_tiles + block_prefix(i < items ? p.tiles[i] : 0, &total);
    if (i < items) p.sum[i] = at;
    head_tiles += total;
  }
  __syncthreads();  // (the cuts below read the sums of other warps' items)
  // The pairs in order, each cut so that no piece is larger than an SM's share of the work that is left from its
  // sequence and head on, so that the SMs finish together, nor than a quarter of an SM's whole share: CTAs that read
  // the same keys then do so at about the same time (whole shares: 1095 us for 256 queries x 64 heads over 131072 keys,
  // quarters 1018, sixths 1062, where the pieces' own cost shows).  Pieces below an eighth of the share or kLeast tiles
  // are not made (a piece's partial sums are twice the bytes of a key and value tile; 4 prompts of 100 tokens over
  // 1000: 35 us at 16, 37 at 8, 44 at 4), nor more pieces of a pair than there are SMs, for which the joining kernel
  // has room.
  // Beside sequences of few rows the SMs that get no piece have their work: pieces are then as long as an SM's share of
  // all of it, if one round of the SMs takes them (a chunk of 256 tokens over 30000 beside 32 single ones over 4000, 32
  // heads over 8: 193 us, 245 cut as above; where it takes two, 512 over 8000 beside 8 over 500, 105 and 92).
  // Without them a few pairs are cut into as many equal pieces as half a round of the SMs takes, or a round where they
  // are cut anyway, down to half of kLeast (64 tokens over 8000, 32 heads over 8: 53 us as above, 42 so; over 20000 63
  // and 58; 3 prompts of 100 over 3000 48 and 43).
  constexpr int kLeast = 16;
  auto capped = [](long long x) { return (int)min(x, 1ll << 30); };
  const int work = capped((long long)head_tiles * a.Hkv), pairs = items * a.Hkv;
  int least = max(kLeast, work / (8 * kSms)), top = max(least, work / (4 * kSms));
  if (pairs <= kSms) {
    const int even = beside > 0 ? max(kLeast, capped(work + beside) / kSms) : max(kLeast / 2, work / kSms + 1);
    int n = 0, total;
    bool cut = beside > 0;
    for (int i = tid; i < items; i += kPlanThreads) {
      n += (p.tiles[i] - 1) / even + 1;
      cut = cut || p.tiles[i] > kLeast;
    }
    block_prefix(n, &total);
    if ((long long)total * a.Hkv <= (__syncthreads_or(cut) ? kSms : kSms / 2)) least = top = even;
  }
  int pieces = 0, slots = 0;
  for (int c0 = 0; c0 < pairs; c0 += kPlanThreads) {
    const int c = c0 + tid;
    int n = 0, head = 0, i = 0;
    if (c < pairs) {
      head = c / items;
      i = c - head * items;
      const int left = work - capped((long long)head * head_tiles) - p.sum[p.base[p.seq[i]]];
      const int most = min(top, max(least, (left + kSms - 1) / kSms));
      n = min((p.tiles[i] - 1) / most + 1, kMaxPieces);
    }
    int total, total_slots;
    const int slot = slots + block_prefix(n > 1 ? n : 0, &total_slots);
    if (n > 1 && slot + n > kMaxSlots) n = 1;  // no room for its partial sums
    const int at = pieces + block_prefix(n, &total);
    if (c < pairs) {
      PieceWork w;
      const SeqRange s = load_seq(a.q_start, a.kv_len, p.seq[i], a.N, room, &bad);
      const int2 k = item_keys(a, s, p.part[i], G);
      w.head = head;
      w.seq = p.seq[i];
      w.row0 = p.part[i] * kItemRows;
      w.rows = s.n * G - w.row0;
      w.pieces = n;
      w.q0 = s.q0;
      w.pos0 = s.pos0;
      w.len = s.len;
      w.end = k.y;
      w.first = window_start(a, s.pos0 + w.row0 / G);
      w.pair = c;
      const int all = p.tiles[i];
      for (int x = 0, t = 0; x < n; ++x) {  // equal shares of the pair's tiles
        const int next = (int)((long long)all * (x + 1) / n);
        w.key0 = k.x + t * TK;
        w.tiles = next - t;
        w.slot = slot + x;
        p.piece[at + x] = w;
        t = next;
      }
      p.split[c] = n;
      p.slot[c] = slot;
      for (int x = 0; x < kItemRows / 32; ++x) p.odd[(long long)c * (kItemRows / 32) + x] = 0;
    }
    pieces += total;
    slots += total_slots;
  }
  if (tid == 0) {
    p.head[0] = pieces;
    p.head[1] = 0;
  }
}

// ---- attention ------------------------------------------------------------------------------

template <int D>
struct TcShared {
  static constexpr int Q = 0;
  static constexpr int RING = 2 * tile_bytes<D>();
  static constexpr int BARS = RING + ring_slots<D>() * tile_bytes<D>();
  // queries; tiles full and empty; scores, probabilities (of the first 64 keys, of the others) and sums of each row
  // tile; the last value tile's rows; what is in flight when a wait was given up
  static constexpr int B_Q = 0, B_FULL = 1, B_EMPTY = B_FULL + ring_slots<D>(), B_S = B_EMPTY + ring_slots<D>(),
                       B_P = B_S + 2, B_O = B_P + 4, B_TAIL = B_O + 2,
                       B_DRAIN = B_TAIL + 1, NBARS = B_DRAIN + 1;
  static constexpr int MISC = (BARS + NBARS * 8 + 15) / 16 * 16;
  static constexpr int WORK = MISC + 16;  // two pieces
  static constexpr int TOTAL = WORK + 2 * (int)sizeof(PieceWork);
};

// max of three, a NaN wins.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ float max2(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmov.b64 rc, {%6, %7};\n\t"
      "fma.rn.f32x2 rd, ra, rb, rc;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}

// The two words of a 128-byte-swizzled matrix descriptor (avq_tc.cuh, sdesc_sw128).  Only the address, in the low word,
// changes from one multiplication to the next; kept apart, a step of it is one 32-bit addition (with the whole
// descriptor formed for each multiplication the issuing thread took 100 cycles for each, the tensor cores' 64).
constexpr uint32_t kDescHigh = 64u | (1u << 14) | (2u << 29);
constexpr uint32_t kDescRows = 1u << 16;                  // K-major rows
constexpr uint32_t kDescCols = (TK * 128 / 16) << 16;     // MN-major: the 64-column blocks lie TK * 128 bytes apart

// True in one lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(r));
  return r != 0;
}
__device__ __forceinline__ uint32_t desc_low(uint32_t addr, uint32_t kind) { return (addr >> 4) | kind; }
__device__ __forceinline__ void mma_ss_low(uint32_t d, uint32_t a_low, uint32_t b_low, uint32_t idesc, bool acc) {
  asm volatile(
      "{ .reg .pred p; .reg .b64 a, b; setp.ne.b32 p, %4, 0; mov.b64 a, {%1, %5}; mov.b64 b, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p; }" ::"r"(d),
      "r"(a_low), "r"(b_low), "r"(idesc), "r"((uint32_t)acc), "n"(kDescHigh)
      : "memory");
}
__device__ __forceinline__ void mma_ts_low(uint32_t d, uint32_t a, uint32_t b_low, uint32_t idesc, bool acc) {
  asm volatile(
      "{ .reg .pred p; .reg .b64 b; setp.ne.b32 p, %4, 0; mov.b64 b, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p; }" ::"r"(d),
      "r"(a), "r"(b_low), "r"(idesc), "r"((uint32_t)acc), "n"(kDescHigh)
      : "memory");
}

struct TensorMaps {
  CUtensorMap k, v;  // a pool: d, and slots, heads and pages in the coordinates x, y and z of its `pos`
  CUtensorMap q;     // d, heads, tokens
  int4 kpos, vpos;
  int has_q;
};

// The (token, head of the group) pairs of rows that a thread steps through, without a division for each.
struct RowStep {
  int tok, h, by_tok, by_h, G;
  __device__ RowStep(int row, int by, int g) : tok(row / g), h(row % g), by_tok(by / g), by_h(by % g), G(g) {}
  __device__ void next() {
    tok += by_tok;
    h += by_h;
    if (h >= G) {
      h -= G;
      ++tok;
    }
  }
};

// exp2 of a pair on the fused multiply-adds: x = n + f with |f| <= 1/2 (n in the low bits of x + 1.5 2^23), 2^f by a
// polynomial (least maximum relative error on the interval: 2^-13.7 of degree 3 for bf16, 2^-18.5 of degree 4 for
// fp16, far below the rounding of P), n added to the exponent.  From -126 down it stays at about 2^-126, so it
// serves tiles without hidden keys.
template <int DT>
__device__ __forceinline__ float2 ex2_poly(float2 x) {
  constexpr float kMagic = 12582912.f;
  x.x = fmaxf(x.x, -126.f);
  x.y = fmaxf(x.y, -126.f);
  const float2 magic = make_float2(kMagic, kMagic);
  const float2 r = add_f32x2(x, magic);
  const float2 n = add_f32x2(r, make_float2(-kMagic, -kMagic));
  const float2 f = fma2(n, make_float2(-1.f, -1.f), x);
  float2 p;
  auto both = [](float c) { return make_float2(c, c); };
  if (DT == DT_BF16) {
    p = fma2(f, both(0.0551716238f), both(0.2426111251f));
    p = fma2(p, f, both(0.6932609677f));
    p = fma2(p, f, both(0.9999280572f));
  } else {
    p = fma2(f, both(0.0095700966f), both(0.0559178591f));
    p = fma2(p, f, both(0.2402474433f));
    p = fma2(p, f, both(0.6931217909f));
    p = fma2(p, f, both(0.9999992847f));
  }
  return make_float2(__int_as_float(__float_as_int(p.x) + (__float_as_int(r.x) << 23)),
                     __int_as_float(__float_as_int(p.y) + (__float_as_int(r.y) << 23)));
}
// The pairs of eight that take the polynomial.  A quarter at head_dim 64, where a step has half the multiplications to
// the same exponentials (4 prompts of about 2048 tokens over 8192: 576 us with none, 559 a quarter, 590 three eighths);
// none at head_dim 128 (256 queries over 131072 keys: 1012 us with none, 1015 a quarter, 1080 three eighths).
template <int D> constexpr uint32_t poly_pairs() { return D == 64 ? 0x12u : 0u; }

template <int DT, int D, bool TMA>
__global__ void __launch_bounds__(kTcThreads, 1) paged_attn_tc_kernel(const __grid_constant__ TensorMaps maps,
                                                                      const PagedAttnArgs a, int max_items,
                                                                      int* __restrict__ plan_ws,
                                                                      float* __restrict__ partials, int out_wide) {
  using T = typename Storage<DT>::T;
  using L = TcShared<D>;
  constexpr int NR = ring_slots<D>(), TB = tile_bytes<D>();
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const uint32_t raw = tc::smem_addr(smem_raw);
  unsigned char* sm = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + L::BARS);
  uint32_t* tslot = reinterpret_cast<uint32_t*>(sm + L::MISC);
  volatile int* abort = reinterpret_cast<volatile int*>(sm + L::MISC + 4);
  PieceWork* works = reinterpret_cast<PieceWork*>(sm + L::WORK);  // this turn's piece and the next
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, G = a.H / a.Hkv;
  const Plan plan = plan_at(plan_ws, a.B, max_items, a.Hkv);

  if (tid == 0) {
    tc::mbar_init(&bars[L::B_Q], maps.has_q ? 1 : kLoaders * 32);
    for (int i = 0; i < NR; ++i) {
      tc::mbar_init(&bars[L::B_FULL + i], TMA ? 1 : kLoaders * 32);
      tc::mbar_init(&bars[L::B_EMPTY + i], 1);
    }
    for (int t = 0; t < 2; ++t) {
      tc::mbar_init(&bars[L::B_S + t], 1);
      tc::mbar_init(&bars[L::B_P + 2 * t], TM);
      tc::mbar_init(&bars[L::B_P + 2 * t + 1], TM);
      tc::mbar_init(&bars[L::B_O + t], 1);
    }
    tc::mbar_init(&bars[L::B_TAIL], 1);
    tc::mbar_init(&bars[L::B_DRAIN], 1);
    *abort = 0;
    tc::fence_mbar_init();
    if (TMA) {
      tc::tma_prefetch_desc(&maps.k);
      tc::tma_prefetch_desc(&maps.v);
    }
    if (maps.has_q) tc::tma_prefetch_desc(&maps.q);
  }
  if (warp == W_MMA) tc::tmem_alloc(tslot, 512);
  tc::tc_before_sync();
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the plan
  const int pieces = plan.head[0];
  // Fetches the piece of a turn: tiles 0 when none is left.
  auto fetch = [&](int turn) {
    const int piece = atomicAdd(&plan.head[1], 1);
    PieceWork none{};
    works[turn & 1] = piece < pieces ? plan.piece[piece] : none;
  };
  if (tid == kTcThreads - 1) fetch(0);
  __syncthreads();
  tc::tc_after_sync();
  const uint32_t tbase = *tslot;
  const uint32_t col_s = tbase, col_o = tbase + 2 * TK;  // S (and P) of tile t at 128 t, O at 256 + D t
  // The piece of a turn, or false when none is left.  Every role calls it once a turn, after the CTA's barrier.
  PieceWork w;
  auto take = [&](int turn) {
    w = works[turn & 1];
    return w.tiles > 0;
  };
  // The end of a turn: false in every thread when one gave up.
  auto turn_over = [&]() {
    const bool go_on = !__syncthreads_or(*abort != 0);
    tc::tc_after_sync();
    return go_on;
  };

  // the launch's 384 x 168 registers: 208 for each softmax thread, 88 for the others
  if (warp >= W_MMA) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp >= W_LOAD) {
      // ---- loaders ----
      const int lw = warp - W_LOAD;
      int ring = 0, tails = 0;  // ring tiles, tiles with a tail so far
      for (int turn = 0; take(turn); ++turn) {
        const int head = w.head, rows = w.rows, nt = rows > TM ? 2 : 1, row0 = w.row0, tiles = w.tiles, key0 = w.key0;
        const int end = w.end, first = w.first;
        bool bad = false;
        constexpr int CPR = D / 8, RPI = 32 / CPR;               // 16-byte chunks of a row, rows of a warp's copy
        constexpr int NI = (TK / RPI + kLoaders - 1) / kLoaders;  // copies of a tile by one warp
        const int sub = lane / CPR, chunk = lane % CPR;
        const uint32_t col = (uint32_t)((chunk >> 3) * TM * 128);
        if (!maps.has_q) {
          const T* q = static_cast<const T*>(a.q);
          RowStep at(row0 + lw * RPI + sub, kLoaders * RPI, G);
          for (int r = lw * RPI + sub; r < nt * TM; r += kLoaders * RPI, at.next()) {
            const bool ok = r < rows;
            const T* from = q + (long long)(w.q0 + at.tok) * a.qs.t + (long long)(head * G + at.h) * a.qs.h + chunk * 8;
            cp_async16(sm + L::Q + (r / TM) * TB + col + (r % TM) * 128 + (((chunk & 7) ^ (r & 7)) << 4), ok ? from : q,
                       ok);
          }
          tc::cp_async_arrive(&bars[L::B_Q]);
        } else if (lw == kLoaders - 1 && lane == 0) {
          // (rows behind the piece's last one hold other tokens, or zeros: nothing of theirs is written)
          tc::mbar_expect_tx(&bars[L::B_Q], nt * TB);
          for (int x = 0; x < nt * (D / 64); ++x) {
            const int t = x / (D / 64), half = x % (D / 64);
            tc::tma_load_3d(sm + L::Q + t * TB + half * TM * 128, &maps.q, half * 64, head * G,
                            w.q0 + (row0 + t * TM) / G, &bars[L::B_Q]);
          }
        }
        const int* row_table = a.table + (long long)w.seq * a.table_stride;
        bool ok = true;
        if constexpr (TMA) {
          // The first warp brings the keys, the second the values; lane x of it one box of a tile: 64 columns of the
          // rows of one page, or of the tile where the page is larger.  (The lanes' copies are issued one after the
          // other, about 130 cycles each: with 16-token pages one warp for both took 4500 cycles a step, the whole step
          // 3300 with two.)
          if (lw < 2) {
            const bool is_v = lw == 1;
            const CUtensorMap* map = is_v ? &maps.v : &maps.k;
            const int4 pos = is_v ? maps.vpos : maps.kpos;
            const int R = min(a.page_size, TK), boxes = TK / R * (D / 64);
            const int row = lane / (D / 64) * R, half = lane % (D / 64);
            // Whether any row sees a key of this lane's box.  (The first tile begins before a window does, perhaps on
            // pages that are not the sequence's any more: they are not looked up, and the box is zeros.)
            auto seen = [&](int key) { return lane < boxes && key < end && key + R > first; };
            // the table entry of this lane's box, read one tile ahead
            auto look_up = [&](int k0) {
              const int key = k0 + row;
              return seen(key) ? row_table[key / a.page_size] : -1;
            };
            int ahead = look_up(key0), j = 0;
            for (; ok && j < tiles; ++j) {
              const int i = ring + 2 * j + lw, slot = i % NR, use = i / NR, k0 = key0 + j * TK;
              const int key = k0 + row, in_page = key % a.page_size;
              int page = a.num_pages;  // outside the map: reads as zeros
              if (seen(key)) {
                if (ahead >= 0 && ahead < a.num_pages) page = ahead;
                else bad = true;
              }
              if (j + 1 < tiles) ahead = look_up(k0 + TK);
              if (use > 0) {
                ok = tc::mbar_wait(&bars[L::B_EMPTY + slot], (use - 1) & 1, abort);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
              }
              // the last keys' page goes on behind them: those value rows become zeros before the tensor cores see them
              const bool tail = is_v && end - k0 < TK && end % R != 0;
              uint64_t* full = &bars[L::B_FULL + slot];
              uint64_t* bar = tail ? &bars[L::B_TAIL] : full;
              unsigned char* dst = sm + L::RING + slot * TB;
              if (lane == 0) tc::mbar_expect_tx(bar, TB);
              __syncwarp();
              if (lane < boxes) {
                auto coordinate = [&](int d) { return d == pos.x ? in_page : (d == pos.y ? head : page); };
                tc::tma_load_4d(dst + half * TM * 128 + row * 128, map, half * 64, coordinate(1), coordinate(2),
                                coordinate(3), bar);
              }
              if (tail) {
                ok = tc::mbar_wait(bar, tails & 1, abort);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                ++tails;
                const int r0 = max(0, end - k0), r1 = min(TK, (r0 + R - 1) / R * R);
                for (int x = lane; x < (r1 - r0) * (D / 8); x += 32) {
                  const int r = r0 + x / (D / 8), c = x % (D / 8);
                  *reinterpret_cast<uint4*>(dst + (c >> 3) * TM * 128 + r * 128 + (c & 7) * 16) = uint4{};
                }
                tc::fence_async_smem();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(full);
              }
            }
            if (!ok)  // let the copies in flight land before the CTA leaves
              for (int u = max(0, j - NR); u < j; ++u) {
                const int i = ring + 2 * u + lw;
                const long long since = clock64();
                while (!tc::mbar_try(&bars[L::B_FULL + i % NR], (i / NR) & 1) &&
                       clock64() - since < tc::kWaitCycles / 8) {
                }
              }
          }
        } else {
          const T* kbase = static_cast<const T*>(a.kpool) + (long long)head * a.kps.h;
          const T* vbase = static_cast<const T*>(a.vpool) + (long long)head * a.vps.h;
          long long off[2][2];  // [key, value][the first 32 rows of the warp's list, the rest]
          for (int i = 0; ok && i < 2 * tiles; ++i) {
            const int is_v = i & 1, slot = (ring + i) % NR, use = (ring + i) / NR;
            if (!is_v) {
              // the warp's rows of this tile: row q of its list is row (lw + 3 (q / RPI)) RPI + q % RPI
#pragma unroll
              for (int hf = 0; hf < 2; ++hf) {
                const int q = hf * 32 + lane, r = (lw + kLoaders * (q / RPI)) * RPI + q % RPI;
                const int key = key0 + (i >> 1) * TK + r;
                off[0][hf] = off[1][hf] = -1;
                if (r < TK && key >= first && key < end) {
                  const int page = row_table[key / a.page_size], s = key % a.page_size;
                  if (page >= 0 && page < a.num_pages) {
                    off[0][hf] = (long long)page * a.kps.p + (long long)s * a.kps.s;
                    off[1][hf] = (long long)page * a.vps.p + (long long)s * a.vps.s;
                  } else {
                    bad = true;
                  }
                }
              }
            }
            if (use > 0) {
              ok = tc::mbar_wait(&bars[L::B_EMPTY + slot], (use - 1) & 1, abort);
              ok = __all_sync(0xffffffffu, ok);
              if (!ok) break;
            }
            unsigned char* dst = sm + L::RING + slot * TB + col;
            const T* base = is_v ? vbase : kbase;
#pragma unroll
            for (int x = 0; x < NI; ++x) {
              const int g = lw + kLoaders * x;  // copy g of the tile: rows g RPI ..
              const int q = x * RPI + sub;
              const int hf = (x * RPI) >> 5;
              const long long o = __shfl_sync(0xffffffffu, is_v ? off[1][hf] : off[0][hf], q & 31);
              const int r = g * RPI + sub;
              if (g < TK / RPI)
                cp_async16(dst + r * 128 + (((chunk & 7) ^ (r & 7)) << 4), base + (o >= 0 ? o + chunk * 8 : 0), o >= 0);
            }
            tc::cp_async_arrive(&bars[L::B_FULL + slot]);  // arrives when this thread's copies have landed
          }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        ring += 2 * tiles;
        if (tid == kTcThreads - 1) fetch(turn + 1);
        if (bad) atomicOr(&g_fault_paged_tc, kFaultTables);
        if (!turn_over()) break;
      }
    } else {
      // ---- MMA issuer: the whole warp runs the loop, so that the descriptors stay in uniform registers (formed by one
      // lane on its own each multiplication took longer to issue than to compute); one elected lane issues ----
      int slot = 0, q_phase = 0;
      uint32_t ring_phase = 0;         // of the ring's slots from `slot` on, until it wraps
      uint32_t p_phase[2] = {0, 0};    // of each row tile's P
      const int fmt = DT == DT_BF16 ? 1 : 0;
      const uint32_t id_s = tc::idesc_f16(fmt, TM, TK, false), id_o = tc::idesc_f16(fmt, TM, D, true);
      const uint32_t q_low = desc_low(tc::smem_addr(sm + L::Q), kDescRows);
      const uint32_t r_low = desc_low(tc::smem_addr(sm + L::RING), 0);
      for (int turn = 0; take(turn); ++turn) {
        const int nt = __shfl_sync(0xffffffffu, w.rows > TM ? 2 : 1, 0), tiles = __shfl_sync(0xffffffffu, w.tiles, 0);
        auto agree = [&](bool ok) { return (bool)__all_sync(0xffffffffu, ok); };
        auto step_on = [&](int& at, uint32_t& phase) {
          if (++at == NR) {
            at = 0;
            phase ^= 1;
          }
        };
        auto issue_s = [&](int t, int at) {
          const uint32_t k_low = r_low + kDescRows + at * (TB / 16), qt = q_low + t * (TB / 16);
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
              const uint32_t o = ((kk >> 2) * TM * 128 + (kk & 3) * 32) / 16;
              mma_ss_low(col_s + t * TK, qt + o, k_low + o, id_s, kk > 0);
            }
            tc::mma_commit(&bars[L::B_S + t]);
            if (t == nt - 1) tc::mma_commit(&bars[L::B_EMPTY + at]);
          }
          __syncwarp();
        };
        // cp.async writes through the generic proxy; the tensor cores read through the async proxy, which a fence after
        // each wait puts behind those writes
        bool ok = agree(tc::mbar_wait(&bars[L::B_Q], q_phase & 1, abort) &&
                        tc::mbar_wait(&bars[L::B_FULL + slot], ring_phase, abort));
        if (ok) {
          tc::fence_async_smem();
          tc::tc_after_sync();
          issue_s(0, slot);
          if (nt > 1) issue_s(1, slot);
          step_on(slot, ring_phase);
        }
        for (int j = 0; ok && j < tiles; ++j) {
          // the values of these keys and the next keys
          const int v_at = slot;
          const uint32_t v_phase = ring_phase;
          step_on(slot, ring_phase);
          const int k_at = slot;
          const uint32_t k_phase = ring_phase;
          const bool more = j + 1 < tiles;
          if (more) step_on(slot, ring_phase);
          ok = tc::mbar_wait(&bars[L::B_FULL + v_at], v_phase, abort) &&
               (!more || tc::mbar_wait(&bars[L::B_FULL + k_at], k_phase, abort));
          const uint32_t v_low = r_low + kDescCols + v_at * (TB / 16);
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (t >= nt) break;
            // P of this tile's first 64 keys is in TMEM, and every thread is done with S; then P of the others
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
              ok = agree(ok && tc::mbar_wait(&bars[L::B_P + 2 * t + hf], p_phase[t], abort));
              if (!ok) break;
              if constexpr (!TMA) tc::fence_async_smem();
              tc::tc_after_sync();
              if (elect_one()) {
#pragma unroll
                for (int kk = hf * (TK / 32); kk < (hf + 1) * (TK / 32); ++kk)
                  mma_ts_low(col_o + t * D, col_s + t * TK + kk * 8, v_low + kk * (16 * 128 / 16), id_o,
                             j > 0 || kk > 0);
                if (hf == 1 && t == nt - 1) tc::mma_commit(&bars[L::B_EMPTY + v_at]);
                if (hf == 1 && !more) tc::mma_commit(&bars[L::B_O + t]);
              }
              __syncwarp();
            }
            if (!ok) break;
            p_phase[t] ^= 1;
            // the scores of the next keys take the columns of P: the tensor cores work in the order of issue
            if (more) issue_s(t, k_at);
          }
        }
        if (!ok) {  // let what was issued finish before the CTA leaves
          if (elect_one()) tc::mma_commit(&bars[L::B_DRAIN]);
          const long long since = clock64();
          while (!tc::mbar_try(&bars[L::B_DRAIN], 0) && clock64() - since < tc::kWaitCycles / 8) {
          }
        }
        __syncwarp();
        ++q_phase;
        if (!turn_over()) break;
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // ---- softmax of tile t: this thread's row is lane (tid % 128) of the tile ----
    const int t = warp >> 2, r = t * TM + (tid & 127);
    int s_count = 0, o_phase = 0;  // S tiles and pieces of this row tile so far
    for (int turn = 0; works[turn & 1].tiles > 0; ++turn) {
      // (read again at the end: few registers are left beside a row of scores)
      const PieceWork& w = works[turn & 1];
      if (t * TM >= w.rows) {
        if (!turn_over()) break;
        continue;
      }
      const int tiles = w.tiles, key0 = w.key0;
      const uint32_t lanes = (uint32_t)(warp & 3) << 21;
      const uint32_t s_at = col_s + t * TK + lanes, o_at = col_o + t * D + lanes;
      int first = 0, last = INT_MAX;  // visible keys; rows behind the last one need no mask
      if (r < w.rows) {
        const int2 v = visible(a, w.pos0 + (w.row0 + r) / G, w.len);
        first = v.x;
        last = v.y;
      }
      float m = -INFINITY, l = 0.f;
      bool ok = true;
      for (int j = 0; j < tiles; ++j) {
        ok = tc::mbar_wait(&bars[L::B_S + t], (s_count + j) & 1, abort);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        tc::tc_after_sync();
        uint32_t s[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tc::tmem_ld32(s_at + c * 32, s[c]);
        tc::tmem_wait_ld();
        const int k0 = key0 + j * TK;
        const bool hidden = __any_sync(0xffffffffu, k0 < first || last - k0 < TK);
        if (hidden) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              const int key = k0 + c * 32 + e;
              if (key < first || key >= last) s[c][e] = 0xff800000u;  // -inf
            }
        }
        auto at = [&](int c, int e) { return __uint_as_float(s[c][e]); };
        float x[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) x[c] = max2(at(c, 0), at(c, 1));
#pragma unroll
        for (int e = 2; e < 32; e += 2)
#pragma unroll
          for (int c = 0; c < 4; ++c) x[c] = max3(x[c], at(c, e), at(c, e + 1));
        const float mx = max2(max3(x[0], x[1], x[2]), x[3]) * a.scale_log2;
        // (the maximum of a row whose keys are all hidden so far stays -inf, which is no growth; a NaN is)
        if (__any_sync(0xffffffffu, !(mx <= m + kLazy))) {
          float mn = max2(m, mx);
          if (mn == INFINITY) mn = NAN;  // a softmax over +inf
          const float f = mn == m ? 1.f : ex2(m - mn);
          m = mn;
          l *= f;
          if (j > 0) {
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
              uint32_t o[32];
              tc::tmem_ld32(o_at + c * 32, o);
              tc::tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tc::tmem_st32(o_at + c * 32, o);
            }
          }
        }
        const float sub = m == -INFINITY ? 0.f : -m;
        const float2 scale2 = make_float2(a.scale_log2, a.scale_log2), sub2 = make_float2(sub, sub);
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        // P to TMEM by 32 keys; the tensor cores may start on the first 64.  Hidden keys need zeros: no polynomial
        auto exps = [&](auto exact) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float2 y = fma2(make_float2(at(c, 2 * e), at(c, 2 * e + 1)), scale2, sub2);
              float2 p;
              if (!exact.value && ((poly_pairs<D>() >> (e & 7)) & 1)) p = ex2_poly<DT>(y);
              else p = make_float2(ex2(y.x), ex2(y.y));
              sum[e & 1] = add_f32x2(sum[e & 1], p);
              pk[e] = pack2<DT>(p.x, p.y);
            }
            tc::tmem_st16(s_at + c * 16, pk);
            if (c & 1) {
              tc::tmem_wait_st();
              tc::tc_before_sync();
              tc::mbar_arrive(&bars[L::B_P + 2 * t + (c >> 1)]);
            }
          }
        };
        if (hidden) exps(std::true_type{});
        else exps(std::false_type{});
        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
      }
      if (ok) {
        ok = tc::mbar_wait(&bars[L::B_O + t], o_phase & 1, abort);
        ok = __all_sync(0xffffffffu, ok);
      }
      if (ok) {
        tc::tc_after_sync();
        const bool whole = w.pieces == 1;
        const int rows = w.rows, head = w.head;
        float zero = 0.f;  // NaN once a sum is not finite
        // a row that sees no key is zero; one whose keys all score -inf is 0 / 0
        const float f = whole ? (last > first ? (m == -INFINITY ? NAN : 1.f / l) : 0.f) : 1.f;
        if (whole) {
          const int at_row = min(w.row0 + r, w.row0 + rows - 1), tok = w.q0 + at_row / G, h = head * G + at_row % G;
          T* dst = static_cast<T*>(a.out) + (long long)tok * a.os.t + (long long)h * a.os.h;
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tc::tmem_ld32(o_at + c * 32, o);
            tc::tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) zero = fmaf(__uint_as_float(o[e]), 0.f, zero);
            if (r >= rows) continue;
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
              uint32_t y[4];
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                const float y0 = __uint_as_float(o[e + 2 * x]) * f, y1 = __uint_as_float(o[e + 2 * x + 1]) * f;
                y[x] = last > first ? pack2<DT>(y0, y1) : 0u;
              }
              if (out_wide) {
                *reinterpret_cast<uint4*>(dst + c * 32 + e) = make_uint4(y[0], y[1], y[2], y[3]);
              } else {
                const T* one = reinterpret_cast<const T*>(y);
#pragma unroll
                for (int i = 0; i < 8; ++i) dst[c * 32 + e + i] = one[i];
              }
            }
          }
        } else {
          // four columns of 256 rows side by side: a warp's stores are contiguous
          float* pd = partials + (long long)w.slot * (kItemRows * (D + 2));
          if (r < rows) {
            pd[kItemRows * D + r] = m;
            pd[kItemRows * (D + 1) + r] = l;
          }
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tc::tmem_ld32(o_at + c * 32, o);
            tc::tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) zero = fmaf(__uint_as_float(o[e]), 0.f, zero);
            if (r < rows) {
#pragma unroll
              for (int e = 0; e < 32; e += 4)
                *reinterpret_cast<uint4*>(pd + ((c * 8 + e / 4) * kItemRows + r) * 4) =
                    make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
            }
          }
        }
        // (the joining kernel then looks at the row; scores that are not finite make NaN of all of it, which is right)
        if (zero != 0.f && l == l && r < rows && (first > key0 || last < min(w.end, key0 + tiles * TK)))
          atomicOr(&plan.odd[(long long)w.pair * (kItemRows / 32) + (r >> 5)], 1u << (r & 31));
        tc::tc_before_sync();
      }
      s_count += tiles;
      ++o_phase;
      if (!turn_over()) break;
    }
  }
  __syncthreads();
  if (warp == W_MMA) tc::tmem_free(tbase, 512);
  if (tid == 0 && *abort) atomicOr(&g_fault_paged_tc, 1);
}

// Joins a pair's pieces: a block per (pair, 32 rows), in the order of the keys.  Rows that hidden values have spoiled
// are formed again.
constexpr int kJoinRows = 32;  // (a word of Plan::odd)

template <int DT, int D>
__global__ void __launch_bounds__(256, 4) combine_tc_kernel(const PagedAttnArgs a, int max_items,
                                                         int* __restrict__ plan_ws,
                                                         const float* __restrict__ partials, int out_wide) {
  using T = typename Storage<DT>::T;
  const Plan plan = plan_at(plan_ws, a.B, max_items, a.Hkv);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int items = plan.head[2], pair = blockIdx.x, G = a.H / a.Hkv;
  if (pair >= items * a.Hkv) return;
  const int np = plan.split[pair], head = pair / items, item = pair - head * items;
  const unsigned odd = plan.odd[(long long)pair * (kItemRows / 32) + blockIdx.y];
  if (np <= 1 && !odd) return;
  bool bad = false;
  const SeqRange seq = load_seq(a.q_start, a.kv_len, plan.seq[item], a.N, (long long)a.W * a.page_size, &bad);
  const int row0 = plan.part[item] * kItemRows, rows = min(kItemRows, seq.n * G - row0);
  const long long stride = kItemRows * (D + 2);
  const float* base = partials + (long long)plan.slot[pair] * stride;
  // the pieces' weights, a warp for four rows
  __shared__ float weight[kMaxPieces][kJoinRows];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r0 = blockIdx.y * kJoinRows;
  if (r0 >= rows) return;
  __shared__ unsigned s_alone;  // rows that are formed alone
  if (odd) {
    if (threadIdx.x == 0) s_alone = 0;
    __syncthreads();
    const int* row_table = a.table + (long long)plan.seq[item] * a.table_stride;
    const int2 keys = item_keys(a, seq, plan.part[item], G);
    // (keys before the first one's page were not looked up)
    const int lo = max(keys.x, window_start(a, seq.pos0 + row0 / G) / a.page_size * a.page_size);
    for (int r = r0 + warp; r < min(rows, r0 + kJoinRows); r += 8) {
      if (!(odd >> (r - r0) & 1)) continue;
      const int tok = seq.q0 + (row0 + r) / G, h = head * G + (row0 + r) % G;
      const int2 v = visible(a, seq.pos0 + (row0 + r) / G, seq.len);
      if (!hidden_odd<DT, D>(a, row_table, head, lo, keys.y, v)) continue;
      float x[D / 32], m, l;
      const T* q_row = static_cast<const T*>(a.q) + (long long)tok * a.qs.t + (long long)h * a.qs.h;
      row_alone<DT, D>(a, row_table, head, q_row, v.x, v.y, x, &m, &l);
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
        static_cast<T*>(a.out)[(long long)tok * a.os.t + (long long)h * a.os.h + i * 32 + lane] =
            from_f<DT>(v.y > v.x ? x[i] / l : 0.f);
      if (lane == 0) atomicOr(&s_alone, 1u << (r - r0));
    }
    __syncthreads();
    if (np <= 1) return;
  }
#pragma unroll
  for (int x = 0; x < kJoinRows / 8; ++x) {
    const int row = warp * (kJoinRows / 8) + x, r = min(r0 + row, rows - 1);
    const float* bm = base + kItemRows * D + r;
    float M = -INFINITY;
    for (int s = lane; s < np; s += 32) M = fmaxf(M, bm[s * stride]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    float sum = 0.f;
    for (int s = lane; s < np; s += 32) {
      const float m = bm[s * stride], l = bm[s * stride + kItemRows];
      // a piece whose keys the row does not see (or that all score -inf) has no weight; a NaN stays one
      const float f = m == -INFINITY ? 0.f : ex2(m - M);
      weight[s][row] = f;
      if (f != 0.f) sum = fmaf(l, f, sum);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    for (int s = lane; s < np; s += 32) weight[s][row] *= 1.f / sum;  // (no weight at all: 0 / 0)
  }
  __syncthreads();
  const int r = r0 + lane;
  if (r >= rows || (odd && s_alone >> lane & 1)) return;
  const int2 seen = visible(a, seq.pos0 + (row0 + r) / G, seq.len);
  constexpr int NC = D / 4 / 8;  // a thread's groups of four columns
  float4 x[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) x[c] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = 0; s < np; ++s) {
    const float f = weight[s][lane];
    float4 o[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c)
      o[c] = *reinterpret_cast<const float4*>(base + s * stride + ((warp * NC + c) * kItemRows + r) * 4);
    if (f == 0.f) continue;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      x[c].x = fmaf(o[c].x, f, x[c].x);
      x[c].y = fmaf(o[c].y, f, x[c].y);
      x[c].z = fmaf(o[c].z, f, x[c].z);
      x[c].w = fmaf(o[c].w, f, x[c].w);
    }
  }
  const int tok = seq.q0 + (row0 + r) / G, h = head * G + (row0 + r) % G;
  T* dst = static_cast<T*>(a.out) + (long long)tok * a.os.t + (long long)h * a.os.h + warp * NC * 4;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const float y[4] = {x[c].x, x[c].y, x[c].z, x[c].w};
    T e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = from_f<DT>(seen.y > seen.x ? y[i] : 0.f);
    if (out_wide) {
      *reinterpret_cast<uint2*>(dst + c * 4) = *reinterpret_cast<const uint2*>(e);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) dst[c * 4 + i] = e[i];
    }
  }
}

// A pool as a tensor map with boxes of 64 columns and the rows of a page (of a tile, where the page is larger); false
// where pages and tiles do not fit each other, or the layout cannot be mapped.
bool pool_map(CUtensorMap* m, int dt, const void* pool, PoolStrides s, const PagedAttnArgs& a, int4* pos) {
  const int ps = a.page_size;
  if (!(ps >= 8 && TK % ps == 0) && ps % TK != 0) return false;
  struct Dim {
    long long stride, extent;
    int which;  // 1 slot, 2 head, 3 page
  } dd[3] = {{s.s, ps, 1}, {s.h, a.Hkv, 2}, {s.p, a.num_pages, 3}};
  std::sort(dd, dd + 3, [](const Dim& x, const Dim& y) { return x.stride < y.stride; });
  cuuint64_t dims[4] = {(cuuint64_t)a.D, 0, 0, 0}, str[3];
  cuuint32_t box[4] = {64, 1, 1, 1};
  int at[4] = {0, 0, 0, 0};
  for (int i = 0; i < 3; ++i) {
    if (dd[i].stride <= 0 || dd[i].extent <= 0) return false;
    dims[i + 1] = (cuuint64_t)dd[i].extent;
    str[i] = (cuuint64_t)dd[i].stride * 2;
    at[dd[i].which] = i + 1;
    if (dd[i].which == 1) box[i + 1] = (cuuint32_t)std::min(ps, TK);
  }
  *pos = make_int4(at[1], at[2], at[3], 0);
  return tc::encode16(m, dt, 4, pool, dims, str, box);
}

// The queries as a tensor map whose boxes are 128 rows, tokens by heads of a group; false where these do not fit.
bool query_map(CUtensorMap* m, int dt, const PagedAttnArgs& a) {
  const int G = a.H / a.Hkv;
  if (G > TM || TM % G || a.qs.h <= 0 || a.qs.t <= 0) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)a.D, (cuuint64_t)a.H, (cuuint64_t)a.N};
  const cuuint64_t str[2] = {(cuuint64_t)a.qs.h * 2, (cuuint64_t)a.qs.t * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)G, (cuuint32_t)(TM / G)};
  return tc::encode16(m, dt, 3, a.q, dims, str, box);
}

long long most_items(int B, int N, int G, int row_min) {
  const long long rows = (long long)N * G;
  return rows / kItemRows + std::min<long long>(B, rows / (row_min + 1)) + 1;
}
// Whether an output row takes 16-byte stores.
bool out_rows_wide(const PagedAttnArgs& a) {
  return reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && a.os.t % 8 == 0 && a.os.h % 8 == 0;
}
size_t plan_bytes(int B, long long items, int Hkv) {
  return align_up((size_t)plan_ints(B, items, Hkv) * sizeof(int));
}

}  // namespace

size_t paged_attn_tc_workspace_bytes(int B, int N, int H, int Hkv, int D, int row_min) {
  const long long items = most_items(B, N, H / Hkv, row_min);
  return plan_bytes(B, items, Hkv) + align_up((size_t)kMaxSlots * kItemRows * (D + 2) * sizeof(float));
}

template <int DT>
int launch_paged_attention_tc(const PagedAttnArgs& a, int row_min, void* workspace, cudaStream_t st) {
  const long long items = most_items(a.B, a.N, a.H / a.Hkv, row_min);
  int* ws = static_cast<int*>(workspace);
  float* partials = reinterpret_cast<float*>(static_cast<char*>(workspace) + plan_bytes(a.B, items, a.Hkv));
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  TensorMaps maps;
  std::memset(&maps, 0, sizeof(maps));
  const bool tma = pool_map(&maps.k, DT, a.kpool, a.kps, a, &maps.kpos) &&
                   pool_map(&maps.v, DT, a.vpool, a.vps, a, &maps.vpos);
  maps.has_q = query_map(&maps.q, DT, a);
  auto go = [&](auto kfn, int total) -> int {
    {
      AVQ_TIMED("paged_plan", st);
      plan_kernel<<<1, kPlanThreads, 0, st>>>(a, row_min, (int)items, ws);
      if (cudaPeekAtLastError() != cudaSuccess) return AVQ_ERR_CUDA;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    {
      AVQ_TIMED("paged_attn_tc", st);
      const int smem = total + 1024;
      static std::atomic<unsigned long long> allowed[4];
      if (!allow_smem((const void*)kfn, smem, allowed[(a.D == 64 ? 0 : 2) + tma])) return AVQ_ERR_CUDA;
      cfg.gridDim = dim3(kSms);
      cfg.blockDim = dim3(kTcThreads);
      cfg.dynamicSmemBytes = smem;
      if (cudaLaunchKernelEx(&cfg, kfn, maps, a, (int)items, ws, partials, (int)out_rows_wide(a)) != cudaSuccess)
        return AVQ_ERR_CUDA;
    }
    return AVQ_OK;
  };
  if (a.D == 64)
    return go(tma ? paged_attn_tc_kernel<DT, 64, true> : paged_attn_tc_kernel<DT, 64, false>, TcShared<64>::TOTAL);
  return go(tma ? paged_attn_tc_kernel<DT, 128, true> : paged_attn_tc_kernel<DT, 128, false>, TcShared<128>::TOTAL);
}

template <int DT>
int launch_paged_combine_tc(const PagedAttnArgs& a, int row_min, void* workspace, cudaStream_t st) {
  const long long items = most_items(a.B, a.N, a.H / a.Hkv, row_min);
  int* ws = static_cast<int*>(workspace);
  const float* partials =
      reinterpret_cast<const float*>(static_cast<char*>(workspace) + plan_bytes(a.B, items, a.Hkv));
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cfg.gridDim = dim3((unsigned)(items * a.Hkv), kItemRows / kJoinRows);
  cfg.blockDim = dim3(256);
  AVQ_TIMED("paged_combine_tc", st);
  return cudaLaunchKernelEx(&cfg, a.D == 64 ? combine_tc_kernel<DT, 64> : combine_tc_kernel<DT, 128>, a, (int)items, ws,
                            partials, (int)out_rows_wide(a)) == cudaSuccess
             ? AVQ_OK
             : AVQ_ERR_CUDA;
}

int read_fault_paged_tc(int* code, cudaStream_t st) {
  int zero = 0;
  if (cudaMemcpyFromSymbolAsync(code, g_fault_paged_tc, sizeof(int), 0, cudaMemcpyDeviceToHost, st) != cudaSuccess ||
      cudaMemcpyToSymbolAsync(g_fault_paged_tc, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, st) != cudaSuccess ||
      cudaStreamSynchronize(st) != cudaSuccess)
    return AVQ_ERR_CUDA;
  return AVQ_OK;
}

template int launch_paged_attention_tc<DT_BF16>(const PagedAttnArgs&, int, void*, cudaStream_t);
template int launch_paged_attention_tc<DT_F16>(const PagedAttnArgs&, int, void*, cudaStream_t);
template int launch_paged_combine_tc<DT_BF16>(const PagedAttnArgs&, int, void*, cudaStream_t);
template int launch_paged_combine_tc<DT_F16>(const PagedAttnArgs&, int, void*, cudaStream_t);

}  // namespace avq
