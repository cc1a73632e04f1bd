// Rotary positions and the paged append.
//
//   y_a = x_a cos t - x_b sin t,   y_b = x_a sin t + x_b cos t
//
// for the pairs (a, b) = (i, i + R/2) or (2i, 2i + 1), with the angle
// t_i = position[axis(i)] * frequency_i; dimensions from R on pass through.
// The gradient is the transposed rotation, by -t.  A packed batch's append is
// the same pass with other destinations: rotated keys and copied values go to
// the pool slots of their positions, rotated queries to a tensor.
//
// The angle is formed in half turns in fp64 (position * frequency / pi) and
// reduced to [-1, 1] exactly; sincospif then works on the fp32 value of the
// reduced angle.  The sine and cosine are within 2^-22 for positions up to
// 2^24 (the fp64 product's own rounding, 2^-52 of the angle, passes that at
// about 2^30).  The products are fp32 and each output is rounded
// once.
//
// What bounds it: memory.  Every row is read and written once; a block forms
// the sines and cosines of its few tokens once, in shared memory, and all
// heads of the tokens use them.  A task is one pair of vectors of a row (16
// bytes each where the layout allows it); a thread keeps its task and walks
// the rows, two in flight.  Small blocks, ten to an SM: one's prologue (the
// positions, the angles) overlaps the others' copies.
#include <algorithm>

#include "avq_paged.cuh"

namespace avq {

namespace {

__device__ int g_fault_tables_rotary;

constexpr int kThreads = 128, kMaxTokens = 16;

// n / d for n * d < 2^32: one multiplication by floor(2^32 / d) + 1 (d > 1).
struct Div {
  uint32_t m;
  int d;
  __device__ int operator()(int n) const { return d == 1 ? n : (int)__umulhi((uint32_t)n, m); }
};

// 48 registers a thread: at D = 128 (bf16, 64 heads, 8192 tokens) 47.6 us, 5.6 TB/s; three blocks of 256 threads took
// 50.9, six of them, which spill, 63.0.
constexpr int kMinBlocks = 10;

template <int BYTES> struct Raw;
template <> struct Raw<16> { using T = uint4; };
template <> struct Raw<8> { using T = uint2; };
template <> struct Raw<4> { using T = uint32_t; };
template <> struct Raw<2> { using T = unsigned short; };

struct Geometry {
  int tokens;            // B * T, or N
  int block_tokens;      // tokens of a block
  int head_step;         // heads of a block (grid.y slices)
  int rot_tasks, tasks;  // tasks of a row that rotate, all tasks of a row
};


template <int DT, int VEC, bool PAGED, int kUnroll>
__global__ void __launch_bounds__(kThreads, kMinBlocks) rotary_kernel(const __grid_constant__ RotarySpec spec,
                                                                      const RotaryArgs a, const PagedAppendArgs p,
                                                                      const Geometry g) {
  using T = typename Storage<DT>::T;
  using V = typename Raw<VEC * (int)sizeof(T)>::T;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  float2* cs = reinterpret_cast<float2*>(smem_raw);  // [block_tokens][pairs], see slot()
  __shared__ long long s_src_q[kMaxTokens], s_dst_q[kMaxTokens], s_src_k[kMaxTokens], s_dst_k[kMaxTokens];
  __shared__ long long s_src_v[kMaxTokens], s_dst_v[kMaxTokens], s_pos[kMaxTokens];
  __shared__ int s_state[kMaxTokens];  // 0: rows behind the last sequence, 1: no place in the pool, 2: a place
  const int tid = threadIdx.x, tok0 = blockIdx.x * g.block_tokens;
  const int nt = min(g.block_tokens, g.tokens - tok0);
  const int heads = PAGED ? a.q.heads + 2 * p.Hkv : a.q.heads + a.k.heads;
  const int h0 = blockIdx.y * g.head_step, h1 = min(heads, h0 + g.head_step);
  if (tid < nt) {
    const int tok = tok0 + tid;
    if constexpr (PAGED) {
      // the token's sequence: the last one that begins at or before it
      int lo = 0, hi = p.B;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (p.q_start[mid + 1] <= tok) lo = mid + 1;
        else hi = mid;
      }
      int state = 0;
      long long pos = 0;
      if (lo < p.B) {
        bool bad = false;
        const SeqRange s = load_seq(p.q_start, p.kv_len, lo, p.N, (long long)p.W * p.page_size, &bad);
        if (tok >= s.q0 && tok < s.q0 + s.n) {
          pos = (long long)s.pos0 + (tok - s.q0);
          state = 1;
          const long long page_i = pos / p.page_size;
          if (pos >= 0 && page_i < p.W) {
            const int page = p.table[(long long)lo * p.table_stride + page_i], slot = (int)(pos % p.page_size);
            if (page >= 0 && page < p.num_pages) {
              state = 2;
              s_dst_k[tid] = (long long)page * p.kps.p + (long long)slot * p.kps.s;
              s_dst_v[tid] = (long long)page * p.vps.p + (long long)slot * p.vps.s;
            }
          }
          bad = bad || (state == 1 && pos >= 0);
        }
        if (bad) atomicOr(&g_fault_tables_rotary, kFaultTables);
      }
      s_state[tid] = state;
      s_pos[tid] = pos;
      s_src_q[tid] = (long long)tok * a.q.st;
      s_dst_q[tid] = (long long)tok * a.q.dt;
      s_src_k[tid] = (long long)tok * p.ks.t;
      s_src_v[tid] = (long long)tok * p.vs.t;
    } else {
      const int b = tok / a.T, t = tok - b * a.T;
      s_state[tid] = 2;
      s_pos[tid] = a.pos0 + t;
      s_src_q[tid] = b * a.q.sb + t * a.q.st;
      s_dst_q[tid] = b * a.q.db + t * a.q.dt;
      s_src_k[tid] = b * a.k.sb + t * a.k.st;
      s_dst_k[tid] = b * a.k.db + t * a.k.dt;
    }
  }
  __syncthreads();

  // sines and cosines: pair f = v * VEC + i of a token in the order [i / 2][v][i % 2], so that the vectors that
  // neighbouring threads read lie side by side
  auto slot = [&](int t, int v, int i) {
    if constexpr (VEC == 1) return t * spec.pairs + v;
    else return t * spec.pairs + ((i >> 1) * g.rot_tasks + v) * 2 + (i & 1);
  };
  for (int x = tid; x < nt * spec.pairs; x += kThreads) {
    const int t = x / spec.pairs, f = x - t * spec.pairs;
    long long pos = s_pos[t];
    const void* given = PAGED ? p.positions : a.positions;
    if (given) {
      const int ax = spec.axis[f], tok = tok0 + t;
      long long at;
      if constexpr (PAGED) {
        at = ax * p.pa + tok * p.pt;
      } else {
        const int b = tok / a.T;
        at = ax * a.pa + b * a.pb + (tok - b * a.T) * a.pt;
      }
      pos = (PAGED ? p.pos_bytes : a.pos_bytes) == 8 ? static_cast<const long long*>(given)[at]
                                                     : (long long)static_cast<const int*>(given)[at];
    }
    const double turns = (double)pos * spec.half_turns[f];
    float s, c;
    sincospif((float)fma(-2.0, rint(0.5 * turns), turns), &s, &c);
    cs[slot(t, f / VEC, f % VEC)] = make_float2(c, spec.reversed ? -s : s);
  }
  __syncthreads();

  // A thread keeps its task v of a row and walks rows (token, head) of one operand after the other, kUnroll at a time.
  const int rows_at_once = kThreads / g.tasks, v = tid % g.tasks, first = tid / g.tasks;
  if (first >= rows_at_once) return;
  auto walk = [&](const T* src, T* dst, const long long* src_at, const long long* dst_at, long long src_h,
                  long long dst_h, int begin, int end, bool rotates, int state) {
    const int n = end - begin;  // heads
    if (n <= 0) return;
    const bool rot = rotates && v < g.rot_tasks;
    int off0, off1;
    if (rot) {
      off0 = spec.interleaved ? 2 * v * VEC : v * VEC;
      off1 = spec.interleaved ? off0 + VEC : spec.pairs + v * VEC;
    } else {
      off0 = rotates ? 2 * spec.pairs + 2 * (v - g.rot_tasks) * VEC : 2 * v * VEC;
      off1 = off0 + VEC;
    }
    if (off0 >= a.D) return;
    const bool two = off1 < a.D;
    const Div by_heads = {(uint32_t)(n == 1 ? 0u : 0xffffffffu / (uint32_t)n + 1u), n};
    for (int row = first; row < nt * n; row += kUnroll * rows_at_once) {
      V lo[kUnroll], hi[kUnroll];
      T* to[kUnroll];
      int tok[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int x = row + u * rows_at_once, t = by_heads(x), h = begin + x - t * n;
        to[u] = nullptr;
        if (x >= nt * n || (PAGED && s_state[t] < state)) continue;
        const T* from = src + src_at[t] + h * src_h;
        to[u] = dst + dst_at[t] + h * dst_h;
        tok[u] = t;
        lo[u] = *reinterpret_cast<const V*>(from + off0);
        if (two) hi[u] = *reinterpret_cast<const V*>(from + off1);
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        if (!to[u]) continue;
        if (rot) {
          T* x0 = reinterpret_cast<T*>(&lo[u]);
          T* x1 = reinterpret_cast<T*>(&hi[u]);
          const float2* r = cs + slot(tok[u], v, 0);
          float2 w[VEC];
          if constexpr (VEC == 1) {
            w[0] = r[0];
          } else {
#pragma unroll
            for (int i = 0; i < VEC; i += 2) {
              const float4 y = *reinterpret_cast<const float4*>(r + (i >> 1) * g.rot_tasks * 2);
              w[i] = make_float2(y.x, y.y);
              w[i + 1] = make_float2(y.z, y.w);
            }
          }
          if (!spec.interleaved) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              const float xa = to_f(x0[i]), xb = to_f(x1[i]);
              x0[i] = from_f<DT>(xa * w[i].x - xb * w[i].y);
              x1[i] = from_f<DT>(xa * w[i].y + xb * w[i].x);
            }
          } else {
            T e[2 * VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              e[i] = x0[i];
              e[VEC + i] = x1[i];
            }
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              const float xa = to_f(e[2 * i]), xb = to_f(e[2 * i + 1]);
              e[2 * i] = from_f<DT>(xa * w[i].x - xb * w[i].y);
              e[2 * i + 1] = from_f<DT>(xa * w[i].y + xb * w[i].x);
            }
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              x0[i] = e[i];
              x1[i] = e[VEC + i];
            }
          }
        }
        *reinterpret_cast<V*>(to[u] + off0) = lo[u];
        if (two) *reinterpret_cast<V*>(to[u] + off1) = hi[u];
      }
    }
  };
  const int hq = a.q.heads;
  walk(static_cast<const T*>(a.q.src), static_cast<T*>(a.q.dst), s_src_q, s_dst_q, a.q.sh, a.q.dh, min(h0, hq),
       min(h1, hq), true, 1);
  if constexpr (PAGED) {
    walk(static_cast<const T*>(p.k), static_cast<T*>(p.kpool), s_src_k, s_dst_k, p.ks.h, p.kps.h,
         min(max(h0 - hq, 0), p.Hkv), min(max(h1 - hq, 0), p.Hkv), true, 2);
    walk(static_cast<const T*>(p.v), static_cast<T*>(p.vpool), s_src_v, s_dst_v, p.vs.h, p.vps.h,
         max(h0 - hq - p.Hkv, 0), max(h1 - hq - p.Hkv, 0), false, 2);
  } else {
    walk(static_cast<const T*>(a.k.src), static_cast<T*>(a.k.dst), s_src_k, s_dst_k, a.k.sh, a.k.dh, max(h0 - hq, 0),
         max(h1 - hq, 0), true, 2);
  }
}

// The widest vector (elements) whose loads and stores are aligned in every row of the call.
struct Widest {
  int vec;
  explicit Widest(int elem_bytes) : vec(16 / elem_bytes), bytes(elem_bytes) {}
  void elements(long long n) {
    while (vec > 1 && n % vec) vec >>= 1;
  }
  void pointer(const void* p) {
    while (vec > 1 && reinterpret_cast<uintptr_t>(p) % (uintptr_t)(vec * bytes)) vec >>= 1;
  }
  int bytes;
};

Geometry geometry(const RotarySpec& spec, int D, int tokens, int heads, int vec) {
  Geometry g;
  g.tokens = tokens;
  g.rot_tasks = spec.pairs / vec;
  g.tasks = g.rot_tasks + (D - 2 * spec.pairs + 2 * vec - 1) / (2 * vec);
  // as many tokens as keep one sine and cosine to a thread; fewer tokens, and slices of the heads, where the call
  // would otherwise leave SMs without a block
  int bt = std::max(1, std::min(kMaxTokens, kThreads / std::max(spec.pairs, 16)));
  while (bt > 1 && (tokens + bt - 1) / bt < 2 * kSms) bt >>= 1;
  const int blocks = (tokens + bt - 1) / bt;
  const int most = std::max(1, heads * g.tasks * bt / 32);
  const int slices = std::max(1, std::min(most, 2 * kSms / std::max(blocks, 1)));
  g.block_tokens = bt;
  g.head_step = (heads + slices - 1) / slices;
  return g;
}

template <int DT, bool PAGED>
int go(const RotarySpec& spec, const RotaryArgs& a, const PagedAppendArgs& p, int tokens, int heads, int vec,
       cudaStream_t st) {
  const Geometry g = geometry(spec, a.D, tokens, heads, vec);
  const dim3 grid((tokens + g.block_tokens - 1) / g.block_tokens, (heads + g.head_step - 1) / g.head_step);
  const size_t smem = std::max<size_t>(16, (size_t)g.block_tokens * spec.pairs * sizeof(float2));
  constexpr int U = 2;
  auto run = [&](auto kfn) { kfn<<<grid, kThreads, smem, st>>>(spec, a, p, g); };
  if constexpr (DT == DT_F32) {
    if (vec == 4) run(rotary_kernel<DT, 4, PAGED, U>);
    else if (vec == 2) run(rotary_kernel<DT, 2, PAGED, U>);
    else run(rotary_kernel<DT, 1, PAGED, U>);
  } else {
    if (vec == 8) run(rotary_kernel<DT, 8, PAGED, U>);
    else if (vec == 4) run(rotary_kernel<DT, 4, PAGED, U>);
    else if (vec == 2) run(rotary_kernel<DT, 2, PAGED, U>);
    else run(rotary_kernel<DT, 1, PAGED, U>);
  }
  return cudaPeekAtLastError() == cudaSuccess ? AVQ_OK : AVQ_ERR_CUDA;
}

void rows_limit(Widest& w, const RotaryRows& r, bool batched) {
  if (!r.heads) return;
  w.pointer(r.src);
  w.pointer(r.dst);
  for (long long s : {r.sh, r.st, r.dh, r.dt}) w.elements(s);
  if (batched) {
    w.elements(r.sb);
    w.elements(r.db);
  }
}

}  // namespace

template <int DT>
int launch_rotary(const RotarySpec& spec, const RotaryArgs& a, cudaStream_t st) {
  const int heads = a.q.heads + a.k.heads;
  if (a.B == 0 || a.T == 0 || heads == 0) return AVQ_OK;
  Widest w((int)sizeof(typename Storage<DT>::T));
  w.elements(spec.pairs);
  w.elements(a.D - 2 * spec.pairs);
  rows_limit(w, a.q, true);
  rows_limit(w, a.k, true);
  AVQ_TIMED("rotary", st);
  return go<DT, false>(spec, a, PagedAppendArgs{}, a.B * a.T, heads, w.vec, st);
}

template <int DT>
int launch_paged_append(const RotarySpec& spec, const PagedAppendArgs& p, cudaStream_t st) {
  const int heads = p.q.heads + 2 * p.Hkv;
  if (p.B == 0 || p.N == 0) return AVQ_OK;
  RotaryArgs a{};
  a.q = p.q;
  a.B = 1;
  a.T = p.N;
  a.D = p.D;
  Widest w((int)sizeof(typename Storage<DT>::T));
  w.elements(spec.pairs);
  w.elements(p.D - 2 * spec.pairs);
  rows_limit(w, p.q, false);
  for (const void* x : {p.k, p.v, (const void*)p.kpool, (const void*)p.vpool}) w.pointer(x);
  for (long long s : {p.ks.t, p.ks.h, p.vs.t, p.vs.h, p.kps.p, p.kps.h, p.kps.s, p.vps.p, p.vps.h, p.vps.s})
    w.elements(s);
  AVQ_TIMED("paged_append", st);
  return go<DT, true>(spec, a, p, p.N, heads, w.vec, st);
}

int read_fault_rotary(int* code, cudaStream_t st) {
  int zero = 0;
  if (cudaMemcpyFromSymbolAsync(code, g_fault_tables_rotary, sizeof(int), 0, cudaMemcpyDeviceToHost, st) !=
          cudaSuccess ||
      cudaMemcpyToSymbolAsync(g_fault_tables_rotary, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, st) !=
          cudaSuccess ||
      cudaStreamSynchronize(st) != cudaSuccess)
    return AVQ_ERR_CUDA;
  return AVQ_OK;
}

#define AVQ_INSTANCE(DT)                                                                \
  template int launch_rotary<DT>(const RotarySpec&, const RotaryArgs&, cudaStream_t); \
  template int launch_paged_append<DT>(const RotarySpec&, const PagedAppendArgs&, cudaStream_t);
AVQ_INSTANCE(DT_F32)
AVQ_INSTANCE(DT_BF16)
AVQ_INSTANCE(DT_F16)
#undef AVQ_INSTANCE

}  // namespace avq
