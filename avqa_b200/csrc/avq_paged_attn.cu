// Attention of a packed batch of new tokens over a page pool:
//
//   out[i, h] = sum_j p_ij v_j,  p_i = softmax_j(scale * q[i, h] . k_j)
//
// over the keys j that token i sees: every key of its sequence, or with
// `causal` those at its own position and before, or of these the last
// `window`.  Query head h reads key head h / (H / Hkv).  A token that sees no
// key gets zeros.
//
// paged_attn_mma_kernel: the kernel of few rows (single tokens, short drafts)
// and of every type and head width.  Its rows are the (token, head of the
// group) pairs of one sequence and key head, 8 or 16 to a CTA, so that one read
// of a key serves the whole group; the sequence's keys are cut into spans, a CTA
// each.  Memory bounds it: every key and value is read once, by cp.async into
// a ring of each warp's own (16 or 32 keys a stage), so that no barrier joins
// the warps until their sums meet at the end (32 sequences of up to 32768 keys,
// 8 key heads of 128, bf16: 454 us, 6.4 TB/s).  The span follows from the
// lengths, which only the device knows: every CTA (for many sequences a kernel
// before it) adds up the batch's work, takes the span that cuts it into about
// target_ctas pieces, and finds its own.
// Few short sequences go to clusters of CTAs instead, which join their sums
// through shared memory (one token of 4097 keys, 8 key heads: 12 us).
//
// The scores, the running maximum and sum, and the output are fp32.  bf16 and
// fp16 multiply on mma.sync with the probabilities rounded to the dtype
// (their error is of the size of the output's own rounding); fp32 operands
// are split in two tf32 parts, whose three products carry 22 bits.
//
// combine_kernel joins the pieces of a row by their maxima and sums, in the
// order of the keys.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "avq_mma.cuh"
#include "avq_paged.cuh"

namespace avq {

namespace {

__device__ int g_fault_tables_paged;

constexpr int kWarps = 4;
constexpr int kMaxGroup = 16;   // rows of a group, at most
// The pieces that a batch of `total` keys (over its row groups and key heads) is cut into.  Long batches: about three
// rounds of the CTAs that the SMs hold at once; less fills the last round badly, more pays a CTA's own cost too often
// (32 sequences of up to 32768 keys, 8 heads of 128: 503 us at 2 per SM, 454 at 8, 455 at 16).  Short ones: a single
// round, as a CTA's first loads and its merge are then most of its time (one sequence of 16384 keys, 8 heads of 128: 18
// us at 2 per SM, 30 at 8; of 32768 keys 34 and 44).  The two meet between 2^19 keys (55 and 63 us) and 2^20 (104, 97).
// Measured where two CTAs or more share an SM; where one does (wide rows, fp32), the single round becomes two.
constexpr int kTargetCtas = 8 * kSms, kFewestCtas = 2 * kSms, kMinSpan = 128;
constexpr long long kFewKeys = 1 << 19;
// A cluster of eight CTAs for each (row group, key head), without a second kernel, where two CTAs to an SM hold them
// all and the keys of a sequence are few (bf16, 8 key heads of 128: 1024 keys 7 us and in pieces 8.5, 4096 keys 11.2
// and 11.4, 8192 keys 16.6 and 13.5; 64 pairs of 512 keys, more than the SMs hold: 15 and 11).  fp32, whose keys cost
// four times as much: 1024 keys 9.6 and 11.5, 2048 keys 14 and 12.
constexpr int kCluster = 8;
constexpr long long kClusterItems = 2 * kSms / kCluster, kClusterKeys = 4096;
// Rows (new tokens x heads of a group) of a sequence up to which one pass of 16-row groups over its keys is
// taken, above which the tcgen05 kernel.
constexpr int kFewRows = 16;

__host__ __device__ constexpr int target_ctas(long long total) { return total > kFewKeys ? kTargetCtas : kFewestCtas; }

struct Piece {  // what one CTA works on
  int b, group, head, span_i;  // sequence, row group, key head, index of the span
  int nspan;                   // spans of the sequence
  SeqRange seq;
  int lo, hi;                  // keys of the span
  bool found;
};

// Rows of a sequence that this kernel owns, in groups of RB.
template <int RB>
__device__ __forceinline__ int row_groups(int G, int n, int row_max) {
  const long long rows = (long long)n * G;
  return rows > row_max ? 0 : (int)((rows + RB - 1) / RB);
}

// First key that any token of the sequence sees.
__device__ __forceinline__ int first_key(const PagedAttnArgs& a, const SeqRange& s) {
  return min(window_start(a, s.pos0), s.len);
}

// How a sequence is cut: its row groups, the first key that it sees, its spans.
struct Cut {
  int groups, first, spans;
};
template <int RB>
__device__ __forceinline__ Cut cut_of(const PagedAttnArgs& a, const SeqRange& s, int row_max, unsigned span) {
  const int f = first_key(a, s);
  return {row_groups<RB>(a.H / a.Hkv, s.n, row_max), f, max(1, (int)(((unsigned)(s.len - f) + span - 1) / span))};
}
// The keys of a sequence, over its row groups and key heads.
template <int RB>
__device__ __forceinline__ long long work_of(const PagedAttnArgs& a, const SeqRange& s, int row_max) {
  return (long long)row_groups<RB>(a.H / a.Hkv, s.n, row_max) * a.Hkv * (s.len - first_key(a, s));
}
// The span that cuts a batch of so much work into about target_ctas pieces, in multiples of UNIT keys (a CTA's step).
template <int UNIT>
__device__ __forceinline__ unsigned span_of(long long total) {
  const int target = target_ctas(total);
  return (unsigned)min((max((total + target - 1) / target, (long long)kMinSpan) + UNIT - 1) / UNIT * UNIT,
                       (long long)(1 << 30));
}

// The pieces of a long list of sequences, by lists_kernel: where each sequence's begin.  Adding up the whole list in
// every CTA, which costs the least for a short one, takes most of a long one's time (8 key heads of 128, bf16,
// sequences of up to 1000 keys: 64 of them 38.6 us so and 40.6 with the lists, 96 52.9 and 51.2, 256 152 and 111, 2048
// 3754 and 729, of which the keys need 702).
constexpr int kListed = 64;
struct Lists {
  unsigned* head;    // [0] the span, [1] pieces, [2] (row group, key head) pairs
  unsigned* pieces;  // [B] pieces of the sequences before
  unsigned* pairs;   // [B] pairs of the sequences before
  unsigned* slots;   // [B] slots of partial sums of the sequences before
};
__host__ __device__ inline Lists lists_at(unsigned* p, int B) { return {p, p + 8, p + 8 + B, p + 8 + 2ll * B}; }
size_t lists_bytes(int B) { return B > kListed ? align_up((8 + 3ull * B) * sizeof(unsigned)) : 0; }

constexpr int kListThreads = 1024;

template <int RB, int UNIT>
__global__ void __launch_bounds__(kListThreads) lists_kernel(const PagedAttnArgs a, int row_max, unsigned* ws) {
  __shared__ long long s_total[kListThreads / 32];
  __shared__ unsigned s_warp[3][kListThreads / 32];
  const Lists out = lists_at(ws, a.B);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long room = (long long)a.W * a.page_size;
  bool bad = false;
  long long total = 0;
  for (int b = tid; b < a.B; b += kListThreads)
    total += work_of<RB>(a, load_seq(a.q_start, a.kv_len, b, a.N, room, &bad), row_max);
  if (bad) atomicOr(&g_fault_tables_paged, kFaultTables);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (lane == 0) s_total[warp] = total;
  __syncthreads();
  total = 0;
  for (int w = 0; w < kListThreads / 32; ++w) total += s_total[w];
  const unsigned span = span_of<UNIT>(total);
  unsigned before[3] = {0, 0, 0};  // pieces, pairs, slots of the sequences before this turn's
  for (int b0 = 0; b0 < a.B; b0 += kListThreads) {
    const int b = b0 + tid;
    unsigned mine[3] = {0, 0, 0}, pre[3];
    if (b < a.B) {
      const Cut c = cut_of<RB>(a, load_seq(a.q_start, a.kv_len, b, a.N, room, &bad), row_max, span);
      mine[1] = (unsigned)c.groups * a.Hkv;
      mine[0] = mine[1] * c.spans;
      mine[2] = c.spans > 1 ? mine[0] : 0u;
    }
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      pre[i] = mine[i];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned x = __shfl_up_sync(0xffffffffu, pre[i], o);
        if (lane >= o) pre[i] += x;
      }
      if (lane == 31) s_warp[i][warp] = pre[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const unsigned w = s_warp[i][lane];  // (as many warps as lanes)
      unsigned x = lane < warp ? w : 0u, all = w;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        x += __shfl_xor_sync(0xffffffffu, x, o);
        all += __shfl_xor_sync(0xffffffffu, all, o);
      }
      pre[i] += before[i] + x - mine[i];
      before[i] += all;
    }
    __syncthreads();
    if (b < a.B) {
      out.pieces[b] = pre[0];
      out.pairs[b] = pre[1];
      out.slots[b] = pre[2];
    }
  }
  if (tid == 0) {
    out.head[0] = span;
    out.head[1] = before[0];
    out.head[2] = before[1];
  }
}

// Finds the piece of index `at`: a (sequence, key head, span, row group) when `spans`, else a (sequence, key head, row
// group) with every span of it.  Each warp does the same work, from the lists if there are any.  *slot receives the
// piece's slot of partial sums (without `spans` that of its first span, the others `stride` apart).
template <int RB, int UNIT>
__device__ Piece find_piece(const PagedAttnArgs& a, int row_max, unsigned at, bool spans, bool report, unsigned* lists,
                            int* slot, int* stride) {
  const int lane = threadIdx.x & 31;
  const long long room = (long long)a.W * a.page_size;
  Piece p;
  p.found = false;
  unsigned span, rel = 0, base = 0;  // the index in the sequence's pieces, its first slot
  Cut cut{0, 0, 0};
  bool bad = false;
  if (lists) {
    const Lists l = lists_at(lists, a.B);
    span = l.head[0];
    if (at >= l.head[spans ? 1 : 2]) return p;
    const unsigned* begin = spans ? l.pieces : l.pairs;
    int lo = 0;  // the last sequence that begins at or before the index
    for (int n = a.B; n > 1;) {
      const int step = (n + 31) / 32, i = lane * step;
      const int k = __popc(__ballot_sync(0xffffffffu, i < n && begin[lo + min(i, n - 1)] <= at)) - 1;
      lo += k * step;
      n = min(step, n - k * step);
    }
    p.b = lo;
    p.seq = load_seq(a.q_start, a.kv_len, lo, a.N, room, &bad);
    cut = cut_of<RB>(a, p.seq, row_max, span);
    rel = at - begin[lo];
    base = l.slots[lo];
    p.found = true;
  } else {
    long long total = 0;
    for (int b = lane; b < a.B; b += 32)
      total += work_of<RB>(a, load_seq(a.q_start, a.kv_len, b, a.N, room, &bad), row_max);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if (report && bad) atomicOr(&g_fault_tables_paged, kFaultTables);
    span = span_of<UNIT>(total);
    unsigned before = 0, slots = 0;  // pieces and partial slots of the sequences before
    for (int b0 = 0; b0 < a.B && !p.found; b0 += 32) {
      const int b = b0 + lane;
      SeqRange s{0, 0, 0, 0};
      Cut c{0, 0, 0};
      if (b < a.B) {
        s = load_seq(a.q_start, a.kv_len, b, a.N, room, &bad);
        c = cut_of<RB>(a, s, row_max, span);
      }
      // (only cut sequences need slots: at most twice the target, as ceil(x) < 2 x for x > 1)
      const unsigned mine = (unsigned)c.groups * a.Hkv * c.spans, count = spans ? mine : (unsigned)c.groups * a.Hkv;
      const unsigned slotted = c.spans > 1 ? mine : 0u;
      unsigned pre = count, pre_slots = slotted;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned x = __shfl_up_sync(0xffffffffu, pre, o), y = __shfl_up_sync(0xffffffffu, pre_slots, o);
        if (lane >= o) {
          pre += x;
          pre_slots += y;
        }
      }
      const unsigned hit = __ballot_sync(0xffffffffu, before + pre > at);
      if (hit) {
        const int src = __ffs(hit) - 1;
        rel = at - before - __shfl_sync(0xffffffffu, pre - count, src);
        base = slots + __shfl_sync(0xffffffffu, pre_slots - slotted, src);
        p.b = b0 + src;
        p.seq.q0 = __shfl_sync(0xffffffffu, s.q0, src);
        p.seq.n = __shfl_sync(0xffffffffu, s.n, src);
        p.seq.len = __shfl_sync(0xffffffffu, s.len, src);
        p.seq.pos0 = __shfl_sync(0xffffffffu, s.pos0, src);
        cut.groups = __shfl_sync(0xffffffffu, c.groups, src);
        cut.first = __shfl_sync(0xffffffffu, c.first, src);
        cut.spans = __shfl_sync(0xffffffffu, c.spans, src);
        p.found = true;
      }
      before += __shfl_sync(0xffffffffu, pre, 31);
      slots += __shfl_sync(0xffffffffu, pre_slots, 31);
    }
    if (!p.found) return p;
  }
  // row groups of one span lie side by side: they read the same keys
  const unsigned n_groups = cut.groups, rest = n_groups == 1 ? rel : rel / n_groups;
  p.nspan = cut.spans;
  p.group = (int)(rel - rest * n_groups);
  p.head = (int)(spans ? rest / (unsigned)p.nspan : rest);
  p.span_i = spans ? (int)(rest - (unsigned)p.head * p.nspan) : 0;
  p.lo = (int)min((unsigned)p.seq.len, cut.first + p.span_i * span);
  p.hi = (int)min((unsigned)p.seq.len, cut.first + (p.span_i + 1) * span);
  *slot = (int)(base + ((unsigned)p.head * p.nspan + p.span_i) * n_groups + p.group);
  *stride = (int)n_groups;
  return p;
}

// ---- operands -----------------------------------------------------------------------

template <int DT> struct Operand {
  using T = typename Storage<DT>::T;
  static constexpr int kPad = 8;    // a row of D + 8 elements keeps ldmatrix free of bank conflicts
};
template <> struct Operand<DT_F32> {
  using T = float;
  static constexpr int kPad = 4;    // rows 4 words apart: the key and value fragments' lanes hit 32 banks
};

__device__ __forceinline__ void mma_tf32(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = hi + lo + (less than 2^-22 of x), both tf32.  (An infinity leaves a NaN in the low part: rows whose sums are not
// finite are formed again on their own.)
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(x));
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(x - __uint_as_float(hi)));
}
// d += a * b.  The tensor cores' own sums truncate: one step's products are summed there, the steps by rounded fp32
// additions.
__device__ __forceinline__ void mma_split(float* d, const uint32_t* ah, const uint32_t* al, float b0, float b1) {
  uint32_t h0, l0, h1, l1;
  split_tf32(b0, h0, l0);
  split_tf32(b1, h1, l1);
  float x[4] = {0.f, 0.f, 0.f, 0.f};
  mma_tf32(x, al, h0, h1);
  mma_tf32(x, ah, l0, l1);
  mma_tf32(x, ah, h0, h1);
#pragma unroll
  for (int e = 0; e < 4; ++e) d[e] += x[e];
}

// Keys of a warp's step: 8 KB of keys and values, 16 keys at least (a step's shuffles, votes and address
// arithmetic are the same for 32 keys as for 16).
template <int DT, int DP>
constexpr int step_keys() { return DP * (int)sizeof(typename Storage<DT>::T) <= 128 ? 32 : 16; }
template <int DT, int DP>
constexpr int stage_elems() { return 2 * step_keys<DT, DP>() * (DP + Operand<DT>::kPad); }
// Stages of a warp's ring: two, so that one CTA's first loads overlap another's streams: three CTAs share an SM at 16
// bits up to 128 dimensions, two in fp32 up to 64.  Wider rows leave room for one (fp32 of 129 dimensions on: with one
// stage).  Three stages in a cluster, where fewer CTAs run.
template <int DT, int DP, bool CL>
constexpr int ring_stages() {
  return DP * (int)sizeof(typename Storage<DT>::T) > 512 ? 1 : (CL && DT != DT_F32 ? 3 : 2);
}
template <int DT, int DP, int RB, bool CL>
constexpr size_t mma_smem() {
  const size_t T = sizeof(typename Storage<DT>::T);
  const size_t ring = (size_t)kWarps * ring_stages<DT, DP, CL>() * stage_elems<DT, DP>() * T;
  const size_t merge = (size_t)kWarps * RB * (DP + 2) * sizeof(float);
  // the queries, in fp32 as their two parts
  return std::max(ring, merge) + (size_t)(DT == DT_F32 ? 2 : 1) * RB * (DP + Operand<DT>::kPad) * T;
}

// An 8 x 8 block of 16-bit values, two of a row to a lane, transposed.
__device__ __forceinline__ uint32_t transposed8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// WIDE: 16-byte copies.  SAME: the pools have the same strides, so that a key's place is its value's, and are below
// 2^32 chunks of 16 bytes.
// RB: the rows of a group.  16 are the rows of the products S = Q K^T and O = P V; eight are the columns of the
// transposed products (bf16, fp16), S^T = K Q^T and O^T = V^T P^T, whose 16 rows are keys and dimensions: half the
// products and half the scores of a row tile that would be half empty.  P^T needs the other layout, which movmatrix
// makes of each 8 x 8 block.
// CL: the spans of a (row group, key head) are the CTAs of a cluster, in equal shares of the sequence's keys, and join
// their sums through each other's shared memory, without a second kernel.
__device__ __forceinline__ float peer_float(const float* p, int rank) {
  uint32_t at;
  float x;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(at) : "memory");
  return x;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <int DT, int DP, bool WIDE, bool SAME, int RB, bool CL>
__global__ void __launch_bounds__(kWarps * 32) paged_attn_mma_kernel(const PagedAttnArgs a, int row_max,
                                                                     int q_wide, int beside, unsigned* lists,
                                                                     float* __restrict__ part) {
  using T = typename Storage<DT>::T;
  constexpr int KS = step_keys<DT, DP>(), NK = KS / 8;  // keys of a step, in columns of 8
  static_assert(RB == 16 || (RB == 8 && DT != DT_F32), "");
  constexpr int LDS = DP + Operand<DT>::kPad, NT = RB == 8 ? DP / 16 : DP / 8, STAGES = ring_stages<DT, DP, CL>();
  constexpr int EPC = 16 / (int)sizeof(T), CPR = DP / EPC;  // elements of a 16-byte chunk, chunks of a row
  extern __shared__ __align__(128) unsigned char smem_raw[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, G = a.H / a.Hkv;
  asm volatile("griddepcontrol.launch_dependents;");
  int slot = 0, slot_stride = 0;
  Piece p = find_piece<RB, kWarps * KS>(a, row_max, CL ? blockIdx.x / kCluster : blockIdx.x, !CL,
                                        blockIdx.x == 0 && warp == 0, lists, &slot, &slot_stride);
  // a grid that runs beside another ends after it, so that what waits for this one has waited for both
  auto leave = [&]() {
    if (beside && blockIdx.x == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
  };
  if (!p.found) {  // (all CTAs of a cluster look for the same)
    leave();
    return;
  }
  const int rank = blockIdx.x % kCluster;
  if constexpr (CL) {
    const int first = first_key(a, p.seq), each = (p.seq.len - first + kCluster - 1) / kCluster;
    const int share = (each + kWarps * KS - 1) / (kWarps * KS) * (kWarps * KS);
    p.lo = (int)min((long long)p.seq.len, first + (long long)rank * share);
    p.hi = (int)min((long long)p.seq.len, p.lo + (long long)share);
  }
  const bool direct = !CL && p.nspan == 1;
  T* sq = reinterpret_cast<T*>(smem_raw);                                  // [RB][LDS]
  T* sq_low = sq + RB * LDS;                                               // fp32: the queries' low parts
  T* shared = DT == DT_F32 ? sq_low + RB * LDS : sq_low;
  T* ring = shared + warp * STAGES * stage_elems<DT, DP>();                // this warp's stages
  const int row0 = p.group * RB, nrow = min(RB, p.seq.n * G - row0);

  if (q_wide) {
    for (int i = tid; i < RB * CPR; i += kWarps * 32) {
      const int r = i / CPR, c = (i - r * CPR) * EPC;
      const bool ok = r < nrow && c < a.D;
      const int tok = p.seq.q0 + (row0 + (ok ? r : 0)) / G, h = p.head * G + (row0 + (ok ? r : 0)) % G;
      cp_async16(sq + r * LDS + c,
                 static_cast<const T*>(a.q) + (long long)tok * a.qs.t + (long long)h * a.qs.h + (ok ? c : 0), ok);
    }
  } else {
    for (int i = tid; i < RB * DP; i += kWarps * 32) {
      const int r = i / DP, d = i - r * DP;
      T x = from_f<DT>(0.f);
      if (r < nrow && d < a.D) {
        const int tok = p.seq.q0 + (row0 + r) / G, h = p.head * G + (row0 + r) % G;
        x = static_cast<const T*>(a.q)[(long long)tok * a.qs.t + (long long)h * a.qs.h + d];
      }
      sq[r * LDS + d] = x;
    }
  }
  cp_async_commit();

  // the keys that any row of the group sees
  // this thread's two rows: lane / 4 and eight on, or two neighbours
  const int ra = RB == 8 ? (lane & 3) * 2 : lane >> 2, rb = RB == 8 ? ra + 1 : ra + 8;
  const int2 va = visible(a, p.seq.pos0 + (row0 + min(ra, nrow - 1)) / G, p.seq.len);
  const int2 vb = visible(a, p.seq.pos0 + (row0 + min(rb, nrow - 1)) / G, p.seq.len);
  const int2 vf = visible(a, p.seq.pos0 + row0 / G, p.seq.len);
  const int2 vl = visible(a, p.seq.pos0 + (row0 + nrow - 1) / G, p.seq.len);
  const int lo = max(p.lo, vf.x), hi = min(p.hi, vl.y);
  const int steps = hi > lo ? (hi - lo + kWarps * KS - 1) / (kWarps * KS) : 0;
  // keys in [every_lo, every_hi) are visible to every row
  const int every_lo = vl.x, every_hi = min(hi, vf.y);
  const T* kbase = static_cast<const T*>(a.kpool) + (long long)p.head * a.kps.h;
  const T* vbase = static_cast<const T*>(a.vpool) + (long long)p.head * a.vps.h;
  const int* row_table = a.table + (long long)p.b * a.table_stride;
  bool bad = false;

  // One stage: KS keys and their values.  Keys outside the span, and pages outside the pool, read as zeros.  Each lane
  // looks up one key, its table entry one stage ahead, and the chunks' lanes take the place from it; the stages come in
  // order, so the page and the slot only step on.
  const int step_pages = kWarps * KS / a.page_size, step_slots = kWarps * KS - step_pages * a.page_size;
  int key = lo + warp * KS + lane % KS, page_at = key / a.page_size, in_page = key - page_at * a.page_size;
  int ahead = key < hi ? row_table[page_at] : -1;
  auto load = [&](int step) {
    T* dst = ring + (step % STAGES) * stage_elems<DT, DP>();
    long long ko = -1, vo = -1;
    if (key < hi) {
      if (ahead >= 0 && ahead < a.num_pages) {
        ko = (long long)ahead * a.kps.p + (long long)in_page * a.kps.s;
        if (!SAME) vo = (long long)ahead * a.vps.p + (long long)in_page * a.vps.s;
      } else {
        bad = true;
      }
    }
    key += kWarps * KS;
    page_at += step_pages;
    in_page += step_slots;
    if (in_page >= a.page_size) {
      in_page -= a.page_size;
      ++page_at;
    }
    ahead = key < hi ? row_table[page_at] : -1;
    if constexpr (WIDE) {
      const int c = lane % CPR * EPC;
      const bool in_row = c < a.D;  // (rows of up to 32 chunks)
      T* d = dst + lane / CPR * LDS + c;
      const uint32_t chunk = SAME ? (uint32_t)(ko / EPC) : 0u;  // the place in 16-byte chunks; all ones: none
#pragma unroll
      for (int i = 0; i < KS * CPR / 32; ++i) {
        const int r = CPR <= 32 ? i * (32 / CPR) + lane / CPR : i / (CPR / 32);
        const int cc = CPR <= 32 ? c : (i % (CPR / 32) * 32 + lane) * EPC;
        T* to = CPR <= 32 ? d + i * (32 / CPR) * LDS : dst + r * LDS + cc;
        if constexpr (SAME) {
          const uint32_t at = __shfl_sync(0xffffffffu, ko < 0 ? 0xffffffffu : chunk, r);
          const bool ok = at != 0xffffffffu && (CPR <= 32 ? in_row : cc < a.D);
          const long long off = ok ? (long long)at * EPC + cc : 0;
          cp_async16(to, kbase + off, ok);
          cp_async16(to + KS * LDS, vbase + off, ok);
        } else {
          const long long k_at = __shfl_sync(0xffffffffu, ko, r), v_at = __shfl_sync(0xffffffffu, vo, r);
          const bool ok = k_at >= 0 && cc < a.D;
          cp_async16(to, kbase + (ok ? k_at + cc : 0), ok);
          cp_async16(to + KS * LDS, vbase + (ok ? v_at + cc : 0), ok);
        }
      }
    } else {
      for (int r = 0; r < KS; ++r) {
        const long long k_at = __shfl_sync(0xffffffffu, ko, r), v_at = __shfl_sync(0xffffffffu, vo, r);
        for (int c = lane; c < DP; c += 32) {
          const bool ok = k_at >= 0 && c < a.D;
          dst[r * LDS + c] = ok ? kbase[k_at + c] : from_f<DT>(0.f);
          dst[(KS + r) * LDS + c] = ok ? vbase[v_at + c] : from_f<DT>(0.f);
        }
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) load(i);

  cp_async_wait<STAGES - 1>();  // the queries
  __syncthreads();
  if constexpr (DT == DT_F32) {
    for (int i = tid; i < RB * DP; i += kWarps * 32) {
      const int at = i / DP * LDS + i % DP;
      uint32_t h, l;
      split_tf32(sq[at], h, l);
      sq[at] = __uint_as_float(h);
      sq_low[at] = __uint_as_float(l);
    }
    __syncthreads();
  }
  uint32_t qf[DT == DT_F32 ? 1 : DP / 16][RB == 8 ? 2 : 4];
  if constexpr (RB == 8) {
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        qf[kk][e] = *reinterpret_cast<const uint32_t*>(sq + (lane >> 2) * LDS + kk * 16 + e * 8 + (lane & 3) * 2);
  } else if constexpr (DT != DT_F32) {
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk)
      ldsm_x4(qf[kk][0], qf[kk][1], qf[kk][2], qf[kk][3], sq + (lane & 15) * LDS + kk * 16 + (lane >> 4) * 8);
  }
  float o[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
  float ma = -INFINITY, mb = -INFINITY, la = 0.f, lb = 0.f;
  const int ct = (lane & 3) * 2;
  constexpr int kFirst = RB == 8 ? 4 : 1, kBehind = RB == 8 ? 32 : 4;  // the lanes that share a row's scores

  for (int step = 0; step < steps; ++step) {
    load(step + STAGES - 1);
    cp_async_wait<STAGES - 1>();
    __syncwarp();
    const T* sk = ring + (step % STAGES) * stage_elems<DT, DP>();
    const T* sv = sk + KS * LDS;
    // the scores: of columns j of 8 keys, [0, 1] row a, [2, 3] row b; transposed, of 16 keys, [0, 2] and [1, 3]
    constexpr int NS = RB == 8 ? KS / 16 : NK;
    constexpr int A1 = RB == 8 ? 2 : 1, B0 = RB == 8 ? 1 : 2;
    float s[NS][4];
#pragma unroll
    for (int j = 0; j < NS; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
    if constexpr (RB == 8) {
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
        for (int j = 0; j < NS; ++j) {
          uint32_t ka[4];
          ldsm_x4(ka[0], ka[1], ka[2], ka[3], sk + (j * 16 + (lane & 15)) * LDS + kk * 16 + (lane >> 4) * 8);
          mma16816<DT>(s[j], ka, qf[kk][0], qf[kk][1]);
        }
    } else if constexpr (DT != DT_F32) {
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) {
        const int qd = lane >> 3;
#pragma unroll
        for (int j = 0; j < NK; j += 2) {
          uint32_t b0, b1, b2, b3;
          ldsm_x4(b0, b1, b2, b3, sk + (j * 8 + (qd >> 1) * 8 + (lane & 7)) * LDS + kk * 16 + (qd & 1) * 8);
          mma16816<DT>(s[j], qf[kk], b0, b1);
          mma16816<DT>(s[j + 1], qf[kk], b2, b3);
        }
      }
    } else {
#pragma unroll 4
      for (int kk = 0; kk < DP / 8; ++kk) {
        const int c = kk * 8 + (lane & 3), r = lane >> 2;
        uint32_t ah[4], al[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int at = (r + (e & 1) * 8) * LDS + c + (e >> 1) * 4;
          ah[e] = __float_as_uint(to_f(sq[at]));
          al[e] = __float_as_uint(to_f(sq_low[at]));
        }
#pragma unroll
        for (int j = 0; j < NK; ++j)
          mma_split(s[j], ah, al, to_f(sk[(j * 8 + r) * LDS + c]), to_f(sk[(j * 8 + r) * LDS + c + 4]));
      }
    }
#pragma unroll
    for (int j = 0; j < NS; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[j][e] *= a.scale_log2;
    const int k0 = lo + (step * kWarps + warp) * KS;
    if (k0 < every_lo || k0 + KS > every_hi) {
#pragma unroll
      for (int j = 0; j < NS; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = RB == 8 ? k0 + j * 16 + (lane >> 2) + (e >> 1) * 8 : k0 + j * 8 + ct + (e & 1);
          const int2 v = (RB == 8 ? e & 1 : e >> 1) ? vb : va;
          if (key < v.x || key >= min(v.y, hi)) s[j][e] = -INFINITY;
        }
    }
    // (fmaxf drops a NaN score; its probability is NaN and carries it into the sum)
    float ta = -INFINITY, tb = -INFINITY;
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      ta = fmaxf(ta, fmaxf(s[j][0], s[j][A1]));
      tb = fmaxf(tb, fmaxf(s[j][B0], s[j][3]));
    }
#pragma unroll
    for (int of = kFirst; of < kBehind; of <<= 1) {
      ta = fmaxf(ta, __shfl_xor_sync(0xffffffffu, ta, of));
      tb = fmaxf(tb, __shfl_xor_sync(0xffffffffu, tb, of));
    }
    const float na = fmaxf(ma, ta), nb = fmaxf(mb, tb);
    if (__any_sync(0xffffffffu, na > ma || nb > mb)) {
      const float ca = na > ma ? ex2(ma - na) : 1.f, cb = nb > mb ? ex2(mb - nb) : 1.f;
      la *= ca;
      lb *= cb;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        o[j][0] *= ca;
        o[j][A1] *= ca;
        o[j][B0] *= cb;
        o[j][3] *= cb;
      }
      ma = na;
      mb = nb;
    }
    // a row with no visible key so far keeps probabilities of zero
    const float xa = ma == -INFINITY ? 0.f : ma, xb = mb == -INFINITY ? 0.f : mb;
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      s[j][0] = ex2(s[j][0] - xa);
      s[j][A1] = ex2(s[j][A1] - xa);
      s[j][B0] = ex2(s[j][B0] - xb);
      s[j][3] = ex2(s[j][3] - xb);
      la += s[j][0] + s[j][A1];
      lb += s[j][B0] + s[j][3];
    }
    if constexpr (RB == 8) {
#pragma unroll
      for (int j = 0; j < NS; ++j) {
        const uint32_t p0 = transposed8(pack2<DT>(s[j][0], s[j][1])), p1 = transposed8(pack2<DT>(s[j][2], s[j][3]));
#pragma unroll
        for (int jj = 0; jj < NT; ++jj) {
          uint32_t va4[4];
          ldsm_x4_t(va4[0], va4[1], va4[2], va4[3],
                    sv + (j * 16 + (lane >> 4) * 8 + (lane & 7)) * LDS + jj * 16 + ((lane >> 3) & 1) * 8);
          mma16816<DT>(o[jj], va4, p0, p1);
        }
      }
    } else if constexpr (DT != DT_F32) {
#pragma unroll
      for (int j = 0; j < NK; j += 2) {
        const uint32_t pf[4] = {pack2<DT>(s[j][0], s[j][1]), pack2<DT>(s[j][2], s[j][3]),
                                pack2<DT>(s[j + 1][0], s[j + 1][1]), pack2<DT>(s[j + 1][2], s[j + 1][3])};
#pragma unroll
        for (int jj = 0; jj < NT / 2; ++jj) {
          uint32_t b0, b1, b2, b3;
          const int qd = lane >> 3;
          ldsm_x4_t(b0, b1, b2, b3, sv + (j * 8 + (qd & 1) * 8 + (lane & 7)) * LDS + jj * 16 + (qd >> 1) * 8);
          mma16816<DT>(o[2 * jj], pf, b0, b1);
          mma16816<DT>(o[2 * jj + 1], pf, b2, b3);
        }
      }
    } else {
      // the k index t of the fragment stands for key 2t, t + 4 for key 2t + 1: the accumulators' own layout
#pragma unroll
      for (int j = 0; j < NK; ++j) {
        uint32_t ph[4], pl[4];
        split_tf32(s[j][0], ph[0], pl[0]);
        split_tf32(s[j][2], ph[1], pl[1]);
        split_tf32(s[j][1], ph[2], pl[2]);
        split_tf32(s[j][3], ph[3], pl[3]);
#pragma unroll
        for (int jj = 0; jj < NT; ++jj) {
          const T* v0 = sv + (j * 8 + ct) * LDS + jj * 8 + (lane >> 2);
          mma_split(o[jj], ph, pl, to_f(v0[0]), to_f(v0[LDS]));
        }
      }
    }
    __syncwarp();
  }
  cp_async_wait<0>();
#pragma unroll
  for (int of = kFirst; of < kBehind; of <<= 1) {
    la += __shfl_xor_sync(0xffffffffu, la, of);
    lb += __shfl_xor_sync(0xffffffffu, lb, of);
  }
  if (bad) atomicOr(&g_fault_tables_paged, kFaultTables);
  __syncthreads();  // every warp is done with its ring

  // the warps' sums meet: one row's maximum, then the scaled sums
  float* sm = reinterpret_cast<float*>(shared);  // [kWarps][RB] maxima, then sums, then outputs
  float* sl = sm + kWarps * RB;
  float* so = sl + kWarps * RB;  // [kWarps][RB][DP]
  if (RB == 8 ? lane < 4 : (lane & 3) == 0) {
    sm[warp * RB + ra] = ma;
    sm[warp * RB + rb] = mb;
  }
  __syncthreads();
  float Ma = sm[ra], Mb = sm[rb];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) {
    Ma = fmaxf(Ma, sm[w * RB + ra]);
    Mb = fmaxf(Mb, sm[w * RB + rb]);
  }
  const float fa = ma == -INFINITY ? 0.f : ex2(ma - Ma), fb = mb == -INFINITY ? 0.f : ex2(mb - Mb);
  // (a maximum of +inf gives NaN here and in the probabilities, as a softmax over +inf does)
  if (RB == 8 ? lane < 4 : (lane & 3) == 0) {
    sl[warp * RB + ra] = la * fa;
    sl[warp * RB + rb] = lb * fb;
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    if constexpr (RB == 8) {  // dimensions lane / 4 and eight on
      float* w = so + (warp * RB + ra) * DP + j * 16 + (lane >> 2);
      w[0] = o[j][0] * fa;
      w[8] = o[j][2] * fa;
      w[DP] = o[j][1] * fb;
      w[DP + 8] = o[j][3] * fb;
      continue;
    }
    float* w = so + (warp * RB + ra) * DP + j * 8 + ct;
    *reinterpret_cast<float2*>(w) = make_float2(o[j][0] * fa, o[j][1] * fa);
    if (nrow > 8) *reinterpret_cast<float2*>(w + 8 * DP) = make_float2(o[j][2] * fb, o[j][3] * fb);
  }
  __syncthreads();
  // Where a piece's sums go: the output, its slot, or this CTA's shared memory (in place of the first warp's).
  auto slot_at = [&]() { return part + (long long)slot * (RB * (DP + 2)); };
  float* const x_at = CL ? so : slot_at();
  float* const m_at = CL ? sm : slot_at() + RB * DP;
  float* const l_at = CL ? sl : slot_at() + RB * DP + RB;
  bool odd = false;  // a sum that is not finite
  for (int i = tid; i < nrow * DP; i += kWarps * 32) {
    const int r = i / DP, d = i - r * DP;
    if (d >= a.D && direct) continue;
    float x = 0.f, l = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      x += so[(w * RB + r) * DP + d];
      if (direct || d == 0) l += sl[w * RB + r];
    }
    odd = odd || !isfinite(x);
    if (direct) {
      const int tok = p.seq.q0 + (row0 + r) / G, h = p.head * G + (row0 + r) % G;
      const int2 v = visible(a, p.seq.pos0 + (row0 + r) / G, p.seq.len);
      // a row that sees no key is zero; one whose keys all score -inf is 0 / 0
      static_cast<T*>(a.out)[(long long)tok * a.os.t + (long long)h * a.os.h + d] =
          from_f<DT>(v.y > v.x ? x / l : 0.f);
    } else {
      x_at[r * DP + d] = x;
      if (d == 0) {
        float M = sm[r];
        for (int k = 1; k < kWarps; ++k) M = fmaxf(M, sm[k * RB + r]);
        m_at[r] = M;
        l_at[r] = l;
      }
    }
  }
  // rows that do not all see the same keys, or fp32's parts, and a sum that is not finite: such a row on its own
  if ((DT == DT_F32 || every_lo > lo || every_hi < hi) && __syncthreads_or(odd)) {
    for (int r = warp; r < nrow; r += kWarps) {
      bool spoiled = false;
      for (int d = lane; d < DP; d += 32) {
        float x = so[r * DP + d];
        if (!CL)
          for (int w = 1; w < kWarps; ++w) x += so[(w * RB + r) * DP + d];
        spoiled = spoiled || !isfinite(x);
      }
      if (!__any_sync(0xffffffffu, spoiled)) continue;
      const int tok = p.seq.q0 + (row0 + r) / G, h = p.head * G + (row0 + r) % G;
      const int2 v = visible(a, p.seq.pos0 + (row0 + r) / G, p.seq.len);
      if (DT != DT_F32 && !hidden_odd<DT, DP>(a, row_table, p.head, lo, hi, v)) continue;
      float x[DP / 32], M, l;
      const T* q_row = static_cast<const T*>(a.q) + (long long)tok * a.qs.t + (long long)h * a.qs.h;
      row_alone<DT, DP>(a, row_table, p.head, q_row, max(v.x, p.lo), min(v.y, p.hi), x, &M, &l);
      T* out = static_cast<T*>(a.out) + (long long)tok * a.os.t + (long long)h * a.os.h;
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) {
        const int d = i * 32 + lane;
        if (!direct) x_at[r * DP + d] = x[i];
        else if (d < a.D) out[d] = from_f<DT>(v.y > v.x ? x[i] / l : 0.f);
      }
      if (!direct && lane == 0) {
        m_at[r] = M;
        l_at[r] = l;
      }
    }
  }
  if constexpr (CL) {
    cluster_sync();
    for (int i = rank * (kWarps * 32) + tid; i < nrow * DP; i += kCluster * kWarps * 32) {
      const int r = i / DP, d = i - r * DP;
      if (d >= a.D) continue;
      float m[kCluster], M = -INFINITY, x = 0.f, l = 0.f;
#pragma unroll
      for (int c = 0; c < kCluster; ++c) {
        m[c] = peer_float(sm + r, c);
        M = fmaxf(M, m[c]);
      }
#pragma unroll
      for (int c = 0; c < kCluster; ++c) {
        const float xc = peer_float(so + r * DP + d, c), lc = peer_float(sl + r, c);
        // a share whose keys the row does not see (or that all score -inf) adds nothing
        const float f = m[c] == -INFINITY ? 0.f : ex2(m[c] - M);
        if (m[c] == -INFINITY && lc == 0.f) continue;
        x = fmaf(xc, f, x);
        l = fmaf(lc, f, l);
      }
      const int tok = p.seq.q0 + (row0 + r) / G, h = p.head * G + (row0 + r) % G;
      const int2 v = visible(a, p.seq.pos0 + (row0 + r) / G, p.seq.len);
      static_cast<T*>(a.out)[(long long)tok * a.os.t + (long long)h * a.os.h + d] =
          from_f<DT>(v.y > v.x ? x / l : 0.f);
    }
    cluster_sync();  // until every peer has read
  }
  leave();
}

// Joins the spans of one (sequence, key head, row group), or every gridDim.y-th row of it: a warp per row, or several
// where the rows are few, each on every so-manieth span, with a row of partial sums in one load of the warp.
constexpr int kJoinWarps = 8;
// CTAs up to which the rows of a pair go to several (one sequence of 32768 keys, one key head: 66 us of a call with one
// CTA a pair, 20 with one a row).
constexpr int kJoinCtas = 4 * kSms;

template <int DT, int DP, int RB>
__global__ void __launch_bounds__(kJoinWarps * 32) combine_kernel(const PagedAttnArgs a, int row_max, unsigned* lists,
                                                                  const float* __restrict__ part) {
  using T = typename Storage<DT>::T;
  constexpr int VW = DP >= 128 ? 4 : 2, NV = DP / (32 * VW);  // floats of a lane's vector, vectors of a lane
  __shared__ float s_x[kJoinWarps][DP];
  __shared__ float s_l[kJoinWarps];
  const int G = a.H / a.Hkv, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // the lists are older than the attention kernel, which this launch may overtake
  int slot = 0, stride = 0;
  const Piece p =
      find_piece<RB, kWarps * step_keys<DT, DP>()>(a, row_max, blockIdx.x, false, false, lists, &slot, &stride);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (!p.found || p.nspan == 1) return;
  const int row0 = p.group * RB, nrow = min(RB, p.seq.n * G - row0);
  const long long step = (long long)stride * (RB * (DP + 2));
  const float* base = part + (long long)slot * (RB * (DP + 2));
  const int rows = (nrow - (int)blockIdx.y + (int)gridDim.y - 1) / (int)gridDim.y;  // of this CTA
  if (rows <= 0) return;
  const int per_row = rows >= kJoinWarps ? 1 : kJoinWarps / rows;  // warps of a row
  const int share = warp % per_row;
  for (int i_row = warp / per_row; i_row < rows || per_row > 1; i_row += kJoinWarps / per_row) {
    const bool mine = i_row < rows && warp < rows * per_row;
    const int r = i_row * gridDim.y + blockIdx.y;
    float x[NV][VW], l = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < VW; ++e) x[i][e] = 0.f;
    if (mine) {
      const float* bm = base + RB * DP + r;
      float M = -INFINITY;
      for (int s = lane; s < p.nspan; s += 32) M = fmaxf(M, bm[s * step]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
#pragma unroll 4
      for (int s = share; s < p.nspan; s += per_row) {
        const float m = bm[s * step], ls = bm[s * step + RB];
        const float* w = base + s * step + r * DP;
        float y[NV][VW];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          if constexpr (VW == 4) {
            const float4 v = *reinterpret_cast<const float4*>(w + (i * 32 + lane) * 4);
            y[i][0] = v.x;
            y[i][1] = v.y;
            y[i][2] = v.z;
            y[i][3] = v.w;
          } else {
            const float2 v = *reinterpret_cast<const float2*>(w + lane * 2);
            y[i][0] = v.x;
            y[i][1] = v.y;
          }
        }
        // a span whose keys the row does not see (or that all score -inf) adds nothing
        if (m == -INFINITY && ls == 0.f) continue;
        const float f = m == -INFINITY ? 0.f : ex2(m - M);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int e = 0; e < VW; ++e) x[i][e] = fmaf(y[i][e], f, x[i][e]);
        l = fmaf(ls, f, l);
      }
    }
    if (per_row > 1) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VW; ++e) s_x[warp][(i * 32 + lane) * VW + e] = x[i][e];
      if (lane == 0) s_l[warp] = l;
      __syncthreads();
      if (mine && share == 0)
        for (int w = 1; w < per_row; ++w) {
#pragma unroll
          for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < VW; ++e) x[i][e] += s_x[warp + w][(i * 32 + lane) * VW + e];
          l += s_l[warp + w];
        }
    }
    if (mine && share == 0) {
      const int tok = p.seq.q0 + (row0 + r) / G, h = p.head * G + (row0 + r) % G;
      const int2 v = visible(a, p.seq.pos0 + (row0 + r) / G, p.seq.len);
      T* dst = static_cast<T*>(a.out) + (long long)tok * a.os.t + (long long)h * a.os.h;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VW; ++e) {
          const int d = (i * 32 + lane) * VW + e;
          if (d < a.D) dst[d] = from_f<DT>(v.y > v.x ? x[i][e] / l : 0.f);
        }
    }
    if (per_row > 1) break;  // all rows have a warp
  }
}

// (row group, key head) pairs of the sequences with at most row_max rows, at most.
long long most_items(int B, int N, int H, int Hkv, int row_max, int group) {
  const long long G = H / Hkv, rows = (long long)N * G;
  return std::min(rows / group + std::min<long long>(B, rows),
                  std::min<long long>(B, N) * ((row_max + (long long)group - 1) / group)) * Hkv;
}
// Which kernels a call launches: this file's takes the sequences with at most row_max rows, the tcgen05 kernel, where
// it is launched too, the others.
struct Choice {
  bool many;
  int row_max;
  int group;  // rows of a group in this file's kernel
};

Choice choose(int dtype, int N, int H, int Hkv, int D, int max_q, bool operands) {
  const long long G = H / Hkv, most = (long long)(max_q > 0 ? std::min(max_q, N) : N) * G;
  const bool many = most > kFewRows && dtype != DT_F32 && (D == 64 || D == 128) && operands;
  // groups of eight where the sequences that come here have no more rows: beside the tcgen05 kernel, single tokens
  const int group = dtype != DT_F32 && operands && (many ? G : most) <= 8 ? 8 : 16;
  return {many, many ? kFewRows : 1 << 30, group};
}

int padded_dim(int D) { return D <= 64 ? 64 : (D <= 128 ? 128 : 256); }
size_t slots_bytes(int D) {
  return align_up((size_t)2 * kTargetCtas * kMaxGroup * (padded_dim(D) + 2) * sizeof(float));
}

bool wide_rows(const void* p, std::initializer_list<long long> strides, int elem) {
  if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  for (long long s : strides)
    if (s * elem % 16) return false;
  return true;
}

template <int DT, int DP, int RB>
int launch_mma(const PagedAttnArgs& a, const Choice& c, void* tc_workspace, float* part, unsigned* lists,
               cudaStream_t st) {
  using T = typename Storage<DT>::T;
  const int E = (int)sizeof(T), row_max = c.row_max;
  const bool beside = c.many;
  const bool wide = a.D * E % 16 == 0 && wide_rows(a.kpool, {a.kps.p, a.kps.h, a.kps.s}, E) &&
                    wide_rows(a.vpool, {a.vps.p, a.vps.h, a.vps.s}, E);
  const bool q_wide = a.D * E % 16 == 0 && wide_rows(a.q, {a.qs.t, a.qs.h}, E);
  const long long items = most_items(a.B, a.N, a.H, a.Hkv, row_max, RB);
  const long long extent = (long long)std::max(a.num_pages - 1, 0) * a.kps.p + (long long)(a.page_size - 1) * a.kps.s;
  const bool same = a.kps.p == a.vps.p && a.kps.s == a.vps.s && a.kps.p >= 0 && a.kps.s >= 0 &&
                    extent / (16 / E) < 0xffffffffll;
  const long long room = std::min((long long)a.W * a.page_size, 1ll << 31);  // keys of a sequence, at most
  // a cluster for each (row group, key head) where they are few and their keys are: one kernel and no partial sums in
  // memory; else spans enough to fill the SMs
  const bool clusters = !beside && items <= kClusterItems && room * (DT == DT_F32 ? 4 : 1) <= kClusterKeys;
  const int variant = !wide ? 0 : (!same ? 1 : (clusters ? 3 : 2));
  auto kfn = variant == 0   ? paged_attn_mma_kernel<DT, DP, false, false, RB, false>
             : variant == 1 ? paged_attn_mma_kernel<DT, DP, true, false, RB, false>
             : variant == 2 ? paged_attn_mma_kernel<DT, DP, true, true, RB, false>
                            : paged_attn_mma_kernel<DT, DP, true, true, RB, true>;
  const size_t smem = variant == 3 ? mma_smem<DT, DP, RB, true>() : mma_smem<DT, DP, RB, false>();
  static std::atomic<unsigned long long> allowed[4];
  if (!allow_smem((const void*)kfn, smem, allowed[variant])) return AVQ_ERR_CUDA;
  if (lists) {
    AVQ_TIMED("paged_lists", st);
    lists_kernel<RB, kWarps * step_keys<DT, DP>()><<<1, kListThreads, 0, st>>>(a, row_max, lists);
    if (cudaPeekAtLastError() != cudaSuccess) return AVQ_ERR_CUDA;
  }
  if constexpr (DT != DT_F32 && DP <= 128) {
    if (beside) {  // (its plan begins when the lists are there, and so does all that follows)
      const int rc = launch_paged_attention_tc<DT>(a, row_max, tc_workspace, st);
      if (rc != AVQ_OK) return rc;
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.stream = st;
  cudaLaunchAttribute attr;
  if (variant == 3) {
    AVQ_TIMED("paged_attn", st);
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = kCluster;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    cfg.gridDim = dim3((unsigned)(items * kCluster));
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = smem;
    return cudaLaunchKernelEx(&cfg, kfn, a, row_max, (int)q_wide, 0, lists, part) == cudaSuccess ? AVQ_OK
                                                                                                  : AVQ_ERR_CUDA;
  }
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  {
    AVQ_TIMED("paged_attn", st);
    // beside the tcgen05 kernel, whose SMs it takes over one by one (it needs nothing of its)
    // (every piece has its CTA: the target's, and one partly filled span for each pair)
    cfg.gridDim = dim3((unsigned)(items + std::min<long long>(target_ctas(items * room), items * (room / kMinSpan))));
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.numAttrs = beside ? 1 : 0;
    if (cudaLaunchKernelEx(&cfg, kfn, a, row_max, (int)q_wide, (int)beside, lists, part) != cudaSuccess)
      return AVQ_ERR_CUDA;
  }
  if constexpr (DT != DT_F32 && DP <= 128) {
    if (beside) {
      const int rc = launch_paged_combine_tc<DT>(a, row_max, tc_workspace, st);
      if (rc != AVQ_OK) return rc;
    }
  }
  AVQ_TIMED("paged_combine", st);
  // the launch overlaps the attention kernel's end; the kernel waits for its results itself
  long long split = 1;
  while (split < RB && items * split < kJoinCtas) split *= 2;
  cfg.gridDim = dim3((unsigned)items, (unsigned)split);
  cfg.blockDim = dim3(kJoinWarps * 32);
  cfg.dynamicSmemBytes = 0;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, combine_kernel<DT, DP, RB>, a, row_max, lists, (const float*)part) == cudaSuccess
             ? AVQ_OK
             : AVQ_ERR_CUDA;
}

}  // namespace

size_t paged_attn_workspace_bytes(int dtype, int B, int N, int H, int Hkv, int D, int max_q) {
  const size_t few = slots_bytes(D) + lists_bytes(B);
  const Choice with = choose(dtype, N, H, Hkv, D, max_q, true);  // (the operands' alignment may still rule it out)
  return with.many ? few + paged_attn_tc_workspace_bytes(B, N, H, Hkv, D, with.row_max) : few;
}

template <int DT>
int launch_paged_attention(const PagedAttnArgs& a, cudaStream_t st) {
  if (a.B == 0 || a.N == 0) return AVQ_OK;
  const int E = (int)sizeof(typename Storage<DT>::T);
  const bool operands = a.scale_log2 > 0.f && wide_rows(a.q, {a.qs.t, a.qs.h}, E) &&
                        wide_rows(a.kpool, {a.kps.p, a.kps.h, a.kps.s}, E) &&
                        wide_rows(a.vpool, {a.vps.p, a.vps.h, a.vps.s}, E);
  const Choice c = choose(DT, a.N, a.H, a.Hkv, a.D, a.max_q, operands);
  // the workspace: slots of partial sums, the lists, what the tcgen05 kernel needs
  char* ws = static_cast<char*>(a.workspace);
  float* part = reinterpret_cast<float*>(ws);
  ws += slots_bytes(a.D);
  unsigned* lists = a.B > kListed ? reinterpret_cast<unsigned*>(ws) : nullptr;
  ws += lists_bytes(a.B);
  auto go = [&](auto group) -> int {
    constexpr int RB = decltype(group)::value;
    if (a.D <= 64) return launch_mma<DT, 64, RB>(a, c, ws, part, lists, st);
    if (a.D <= 128) return launch_mma<DT, 128, RB>(a, c, ws, part, lists, st);
    return launch_mma<DT, 256, RB>(a, c, ws, part, lists, st);
  };
  if constexpr (DT != DT_F32) {
    if (c.group == 8) return go(std::integral_constant<int, 8>{});
  }
  return go(std::integral_constant<int, 16>{});
}

int read_fault_paged(int* code, cudaStream_t st) {
  int zero = 0;
  if (cudaMemcpyFromSymbolAsync(code, g_fault_tables_paged, sizeof(int), 0, cudaMemcpyDeviceToHost, st) !=
          cudaSuccess ||
      cudaMemcpyToSymbolAsync(g_fault_tables_paged, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, st) !=
          cudaSuccess ||
      cudaStreamSynchronize(st) != cudaSuccess)
    return AVQ_ERR_CUDA;
  return AVQ_OK;
}

template int launch_paged_attention<DT_F32>(const PagedAttnArgs&, cudaStream_t);
template int launch_paged_attention<DT_BF16>(const PagedAttnArgs&, cudaStream_t);
template int launch_paged_attention<DT_F16>(const PagedAttnArgs&, cudaStream_t);

}  // namespace avq
