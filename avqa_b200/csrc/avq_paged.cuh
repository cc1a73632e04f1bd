// Shared declarations of the packed-batch operators: rotary positions
// (avq_rotary.cu), the paged append (avq_rotary.cu) and attention over a page
// pool (avq_paged_attn.cu, avq_paged_attn_tc.cu).
//
// A packed batch holds the new tokens of all sequences one behind the other:
// tokens q_start[b] .. q_start[b+1]-1 belong to sequence b, which holds
// kv_len[b] tokens with them.  New token i of sequence b has the position
// kv_len[b] - (q_start[b+1] - i); position p lives in slot p % page_size of
// pool page block_table[b][p / page_size].
//
// The lists are device data that the host never reads, so the kernels check
// them: a sequence whose token range is not inside [0, N] counts as empty, a
// length beyond the table's row is cut to it, a page outside the pool is
// neither written nor read, and each of these raises kFaultTables in the
// device fault word that avq_device_fault reports.
#pragma once

#include <atomic>

#include "avq_kernels.cuh"

namespace avq {

// Allows a kernel its dynamic shared memory, once a device (`done`: the kernel's own record, a bit per device).
inline bool allow_smem(const void* kernel, size_t bytes, std::atomic<unsigned long long>& done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
  if (bit && (done.load(std::memory_order_relaxed) & bit)) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != cudaSuccess)
    return false;
  done.fetch_or(bit, std::memory_order_relaxed);
  return true;
}

constexpr int kFaultTables = 2;  // bit 1 of the device fault record (bit 0: an abandoned wait)
constexpr int kSms = 148;
// Tokens that a table's row may hold.  The kernels count keys in 32 bits and step past a sequence's last key by up to
// five steps of 128 keys (loads that are asked for ahead, the rest of a tile), which must not wrap.
constexpr long long kMaxRoom = 0x7fffffffll - 65536;

struct Strides2 {  // element strides of a packed [N, H, D] operand (token, head)
  long long t, h;
};
struct PoolStrides {  // element strides of a [pages, H, page_size, D] pool (page, head, slot)
  long long p, h, s;
};

// ---- rotary positions ---------------------------------------------------------------

constexpr int kMaxPairs = 128;  // head_dim <= 256

struct RotarySpec {
  int pairs;        // R/2 rotated pairs; dimensions >= 2 * pairs pass through
  int interleaved;  // pairs (2i, 2i+1) instead of (i, i + R/2)
  int reversed;     // rotate by the negative angle (the gradient)
  double half_turns[kMaxPairs];  // angle per position, in units of pi
  unsigned char axis[kMaxPairs];
};

struct RotaryRows {  // rows [b, h, t, 0..D) of one operand and where they go
  const void* src;
  void* dst;
  long long sb, sh, st, db, dh, dt;
  int heads;
};

struct RotaryArgs {
  RotaryRows q, k;   // heads 0: absent
  int B, T, D;
  const void* positions;  // int32 / int64 [axes, B, T] by strides, or nullptr: pos0 + t
  int pos_bytes;
  long long pa, pb, pt;
  long long pos0;
};

struct PagedAppendArgs {
  RotaryRows q;      // optional (heads 0); sb, db unused
  const void* k;
  Strides2 ks;
  const void* v;
  Strides2 vs;
  void* kpool;
  PoolStrides kps;
  void* vpool;
  PoolStrides vps;
  const int* table;
  long long table_stride;
  const int* kv_len;
  const int* q_start;
  int B, N, Hkv, D, num_pages, page_size, W;
  const void* positions;  // [axes, N] by strides, or nullptr: the cache position
  int pos_bytes;
  long long pa, pt;
};

template <int DT>
int launch_rotary(const RotarySpec& spec, const RotaryArgs& a, cudaStream_t st);
template <int DT>
int launch_paged_append(const RotarySpec& spec, const PagedAppendArgs& a, cudaStream_t st);
int read_fault_rotary(int* code, cudaStream_t st);

// ---- paged attention ------------------------------------------------------------------

struct PagedAttnArgs {
  const void* q;
  Strides2 qs;
  const void* kpool;
  PoolStrides kps;
  const void* vpool;
  PoolStrides vps;
  const int* table;
  long long table_stride;
  const int* kv_len;
  const int* q_start;
  int B, N, H, Hkv, D, num_pages, page_size, W;
  int causal, window;
  float scale_log2;  // softmax scale * log2(e): the kernels work with exp2
  void* out;
  Strides2 os;
  int max_q;         // host bound of the new tokens per sequence, 0: unknown
  void* workspace;
};

// The tcgen05 kernel (bf16, fp16; head_dim 64 and 128; 16-byte rows; scale > 0) for the sequences with more than
// row_min rows (new tokens x heads of a group).
size_t paged_attn_tc_workspace_bytes(int B, int N, int H, int Hkv, int D, int row_min);
template <int DT>
int launch_paged_attention_tc(const PagedAttnArgs& a, int row_min, void* workspace, cudaStream_t st);
template <int DT>
int launch_paged_combine_tc(const PagedAttnArgs& a, int row_min, void* workspace, cudaStream_t st);
int read_fault_paged_tc(int* code, cudaStream_t st);

size_t paged_attn_workspace_bytes(int dtype, int B, int N, int H, int Hkv, int D, int max_q);
template <int DT>
int launch_paged_attention(const PagedAttnArgs& a, cudaStream_t st);
int read_fault_paged(int* code, cudaStream_t st);

// ---- device helpers -------------------------------------------------------------------

struct SeqRange {
  int q0, n;   // first packed token, new tokens
  int len;     // tokens with the new ones, cut to the table's row
  int pos0;    // position of the first new token (negative when len < n)
};

// Sequence b's range, checked; *bad is raised where the lists are not sound.
__device__ __forceinline__ SeqRange load_seq(const int* q_start, const int* kv_len, int b, int N, long long room,
                                             bool* bad) {
  SeqRange s;
  const int a = q_start[b], e = q_start[b + 1], len = kv_len[b];
  const bool sound = a >= 0 && e >= a && e <= N;
  s.q0 = sound ? a : 0;
  s.n = sound ? e - a : 0;
  s.len = len < 0 ? 0 : (len > room ? (int)room : len);
  s.pos0 = (int)min((long long)max(len, 0), kMaxRoom) - s.n;
  *bad = *bad || !sound || len < 0 || len > room;
  return s;
}

// First key in the window of the token at position pos (which may be negative, the window any int).
__device__ __forceinline__ int window_start(const PagedAttnArgs& a, int pos) {
  return a.window > 0 ? (int)max(0ll, (long long)pos + 1 - a.window) : 0;
}

// Keys visible to the token at position pos: [first, last).
__device__ __forceinline__ int2 visible(const PagedAttnArgs& a, int pos, int len) {
  return make_int2(window_start(a, pos), !a.causal ? len : (pos < 0 ? 0 : min(len, pos + 1)));
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A product over a tile of rows takes every key of its tile or span for every row, those that a row does not see with
// a probability of zero; where such a key's value is not finite, that makes 0 * inf = NaN of the row.  A row whose sums
// are not finite, though its scores are, is looked at again: where one of the keys that it does not see holds such a
// value (hidden_odd) it is formed alone (row_alone); else the keys that it sees made it so, and it stays.
//
// What it costs (a NaN in one column of one value): in the history that all rows see, little (256 queries over 131072
// keys 0.95 ms without and 0.92 with, 4 prompts of about 2048 tokens over 8192 0.68 and 0.85); among the new tokens,
// where the rows before it are formed alone, much (187 ms and 13 ms).

// Whether a value that is not finite lies on a key of [lo, hi) outside v, by one warp.
template <int DT, int DP>
__device__ bool hidden_odd(const PagedAttnArgs& a, const int* row_table, int head, int lo, int hi, int2 v) {
  using T = typename Storage<DT>::T;
  const int lane = threadIdx.x & 31;
  for (int part = 0; part < 2; ++part) {
    const int to = part ? hi : min(hi, v.x);
    for (int key = part ? max(lo, v.y) : lo; key < to; ++key) {
      const int page = row_table[key / a.page_size], s = key % a.page_size;
      if (page < 0 || page >= a.num_pages) continue;  // (reads as zeros)
      const T* x = static_cast<const T*>(a.vpool) + page * a.vps.p + head * a.vps.h + s * a.vps.s;
      bool odd = false;
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) {
        const int d = i * 32 + lane;
        odd = odd || (d < a.D && !isfinite(to_f(x[d])));
      }
      if (__any_sync(0xffffffffu, odd)) return true;
    }
  }
  return false;
}

// The row again, key by key over its visible keys [lo, hi), by one warp: its sums before division (the lanes'
// dimensions lane, lane + 32, ..), its maximum (times log2 e) and its sum.
template <int DT, int DP>
__device__ void row_alone(const PagedAttnArgs& a, const int* row_table, int head, const typename Storage<DT>::T* q,
                          int lo, int hi, float (&x)[DP / 32], float* m_out, float* l_out) {
  using T = typename Storage<DT>::T;
  constexpr int U = 4, N = DP / 32;  // keys at a time, whose loads are in flight together
  const int lane = threadIdx.x & 31;
  float qd[N], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    x[i] = 0.f;
    qd[i] = i * 32 + lane < a.D ? to_f(q[i * 32 + lane]) : 0.f;
  }
  for (int key0 = lo; key0 < hi; key0 += U) {
    const int key = key0 + lane % U, s = key % a.page_size;
    const int mine = key < hi ? row_table[key / a.page_size] : -1;
    const bool held = mine >= 0 && mine < a.num_pages;  // a page outside the pool reads as zeros
    const long long ko = held ? mine * a.kps.p + s * a.kps.s : -1, vo = held ? mine * a.vps.p + s * a.vps.s : -1;
    T kd[U][N], vd[U][N];
    bool there[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long at = __shfl_sync(0xffffffffu, ko, u), v_at = __shfl_sync(0xffffffffu, vo, u);
      there[u] = at >= 0;
      const T* k = there[u] ? static_cast<const T*>(a.kpool) + head * a.kps.h + at : q;  // (any address that holds)
      const T* v = there[u] ? static_cast<const T*>(a.vpool) + head * a.vps.h + v_at : q;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int d = min(i * 32 + lane, a.D - 1);
        kd[u][i] = k[d];
        vd[u][i] = v[d];
      }
    }
    float score[U], mn = m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      score[u] = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i)
        score[u] = there[u] && i * 32 + lane < a.D ? fmaf(qd[i], to_f(kd[u][i]), score[u]) : score[u];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
      for (int u = 0; u < U; ++u) score[u] += __shfl_xor_sync(0xffffffffu, score[u], o);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      score[u] = key0 + u < hi ? score[u] * a.scale_log2 : -INFINITY;
      mn = fmaxf(mn, score[u]);
    }
    const float base = mn == -INFINITY ? 0.f : mn, f = mn > m ? ex2(m - base) : 1.f;
    l *= f;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] *= f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float p = ex2(score[u] - base);  // (zero behind the last key)
      l += p;
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = fmaf(there[u] ? to_f(vd[u][i]) : 0.f, p, x[i]);
    }
    m = mn;
  }
  *m_out = m;
  *l_out = l;
}

}  // namespace avq
