// Log probabilities of given tokens, entropy and top alternatives of rows of logits, and their gradient.
//
// With z = x / temperature, m = max z, s = sum e^(z - m), u = sum (z - m) e^(z - m):
//   log p_j = (z_j - m) - log s,   H = log s - u / s,
//   dH / dz_j = -p_j (log p_j + H),   d log p_i / dz_j = [i = j] - p_j.
// z - m is (x - max x) / temperature wherever it is taken of single logits: differences of logits of the type's lowest value do
// not overflow, and no error grows with what all logits of a row share. The sums of the forward pass save the subtraction: they
// are taken relative to m rounded (`Sums`), and what the rounding put in is taken out of their logarithm at the end.
#include "common.cuh"
#include <type_traits>

namespace {
using namespace fsb;

constexpr float L2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int MAX_TOP = 32;

__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16(v); }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half(v); }
template <> __device__ __forceinline__ float from_f(float v) { return v; }

// Maximum that hands NaN on.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// Order of the alternatives: by value, minus zero equal to zero, NaN on top; the lower index first among equals. A larger key
// comes first; no key is 0.
__device__ __forceinline__ uint32_t value_key(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t b = __float_as_uint(v + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }
__device__ __forceinline__ unsigned long long order_key(float v, int index) {
  return static_cast<unsigned long long>(value_key(v)) << 32 | (0xffffffffu - static_cast<uint32_t>(index));
}

constexpr int MAX_CHUNKS = 8;       // chunk maxima a thread keeps
constexpr int GROUPS = 64;          // groups of threads whose maxima bound the alternatives
constexpr int CAP = 512;            // candidates a CTA keeps
constexpr int MAX_PARTS = 8;        // CTAs of a row (a portable cluster)
// A thread's chunk: 2^chunk_bits(n) of its n vectors, four or more, so that there are MAX_CHUNKS at most (n is 0 in a row too short
// for a whole vector).
constexpr int chunk_bits(int n) {
  int bits = 2;
  while ((MAX_CHUNKS << bits) < n) ++bits;
  return bits;
}

__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ uint4 load_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
template <typename T> struct Vec;     // 16 bytes: L elements
template <> struct Vec<__nv_bfloat16> {
  static constexpr int L = 8;
  static constexpr uint32_t NEG_INF = 0xff80ff80u;
  static __device__ __forceinline__ float largest(const uint4 (&v)[4]) {   // a NaN if there is one
    __nv_bfloat162 m[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v[q]);
      m[q] = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    }
    const float2 f = __bfloat1622float2(__hmax2_nan(__hmax2_nan(m[0], m[1]), __hmax2_nan(m[2], m[3])));
    return max_nan(f.x, f.y);
  }
  static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[2 * j] = __uint_as_float(w[j] << 16);
      f[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  }
};
template <> struct Vec<__half> {
  static constexpr int L = 8;
  static constexpr uint32_t NEG_INF = 0xfc00fc00u;
  static __device__ __forceinline__ float largest(const uint4 (&v)[4]) {
    __half2 m[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const __half2* h = reinterpret_cast<const __half2*>(&v[q]);
      m[q] = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    }
    const float2 f = __half22float2(__hmax2_nan(__hmax2_nan(m[0], m[1]), __hmax2_nan(m[2], m[3])));
    return max_nan(f.x, f.y);
  }
  static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[8]) {
    const __half2* h = reinterpret_cast<const __half2*>(&v);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 a = __half22float2(h[j]);
      f[2 * j] = a.x;
      f[2 * j + 1] = a.y;
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
    uint4 v;
    __half2* h = reinterpret_cast<__half2*>(&v);
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = __floats2half2_rn(f[2 * j], f[2 * j + 1]);
    return v;
  }
};
template <> struct Vec<float> {
  static constexpr int L = 4;
  static constexpr uint32_t NEG_INF = 0xff800000u;
  static __device__ __forceinline__ float largest(const uint4 (&v)[4]) {
    float m[4];
#pragma unroll
    for (int q = 0; q < 4; ++q)
      m[q] = max_nan(max_nan(__uint_as_float(v[q].x), __uint_as_float(v[q].y)), max_nan(__uint_as_float(v[q].z), __uint_as_float(v[q].w)));
    return max_nan(max_nan(m[0], m[1]), max_nan(m[2], m[3]));
  }
  static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};

// Rows of a tensor [batches, inner, V]: batches `ldb` elements apart, their rows `ld`.
struct Rows {
  long long inner, ldb, ld;
  template <typename T>
  __device__ __forceinline__ const T* at(const T* x, long long row) const {
    return inner == 0 ? x + row * ld : x + row / inner * ldb + row % inner * ld;
  }
};
// A row as whole 16-byte vectors between a head and a tail of single elements.
struct RowSpan {
  int head, nvec, tail;
};
template <typename T>
__device__ __forceinline__ RowSpan row_span(const T* r, int V) {
  RowSpan s;
  s.head = min(static_cast<int>((16 - (reinterpret_cast<uintptr_t>(r) & 15)) & 15) / static_cast<int>(sizeof(T)), V);
  s.nvec = (V - s.head) / Vec<T>::L;
  s.tail = V - s.head - s.nvec * Vec<T>::L;
  return s;
}

// Sum / maximum over the block, in every thread; the order of the additions is fixed.
template <int THREADS, typename F>
__device__ __forceinline__ float block_reduce(float v, float* red, F op) {
  constexpr int WARPS = THREADS / 32;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[threadIdx.x & (WARPS - 1)];
#pragma unroll
  for (int o = WARPS / 2; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Running sums in base 2 relative to the rounded product o = fl(-m c) of a maximum m, c = log2(e) / temperature:
// s = sum 2^(x c + o), u = sum (x c + o) 2^(x c + o). An fma takes x c exactly, so that the exponents' errors are relative to
// themselves; the maximum counts as 2^over, over = m c + o, and not as 1. |over| is half a step of m c at most: 2 up to FAR, beyond which
// the sums are not used.
constexpr float FAR = 0x1p26f;
__device__ __forceinline__ float offset_of(float m, float c) { return __fmul_rn(-m, c); }
struct Sums {
  float m, s, u;
  __device__ __forceinline__ void raise(float to, float c) {
    const float d = offset_of(to, c) - offset_of(m, c), f = ex2(d);
    u = (u + s * d) * f;
    s *= f;
    m = to;
  }
};

template <int THREADS>
struct SumsSmem {
  float red[32];
  float warp[THREADS / 32][3];                    // m, s, u of the warps
  float part[MAX_PARTS][3];                       // ... and of the row's parts (in the first CTA)
};
template <int THREADS>
struct TopSmem {
  unsigned long long lists[MAX_PARTS * MAX_TOP];  // alternatives of the row's parts (in the first CTA; 0: none)
  unsigned long long best[32];                    // ... of this part, then of the row
  unsigned long long cand[CAP];
  alignas(16) uint32_t groups[GROUPS];
  float cmax[MAX_CHUNKS][THREADS];
  uint16_t work[MAX_CHUNKS * THREADS];
  uint32_t bound;
  int count[4];
};

// Keys of `from`[0, n), all different but for zeros (none), put in order, largest first: rank by counting, the n keys read as
// broadcasts. `to` has 32 places, zeroed before.
template <int THREADS>
__device__ __forceinline__ void rank_keys(const unsigned long long* from, int n, unsigned long long* to) {
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const unsigned long long mine = from[i];
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) rank += from[j] > mine ? 1 : 0;
    if (rank < 32 && mine != 0) to[rank] = mine;
  }
}

// The alternatives of this CTA's part [lo, hi) in sm.best (largest first, 0: none). Elements that can be among the k largest are
// at least as large as the k-th largest of the maxima of 64 groups of threads; they are collected from the chunks whose maximum
// says that they have some, and ranked. Random logits leave k to 1.5 k of them. Where there are more than fit (masked or equal
// logits), those above the bound are collected and those equal to it counted off from the lowest index; where even the former
// do not fit, k maxima are taken one after the other.
template <typename T, int THREADS>
__device__ __forceinline__ void part_top(const T* r, int first_vec, int end_vec, int head, float edge, int edge_at, float tmax, int cl_bits,
                                      int k, int lo, int hi, TopSmem<THREADS>& sm) {
  constexpr int L = Vec<T>::L, WARPS = THREADS / 32, PER = THREADS / GROUPS;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t own = value_key(tmax);
  uint32_t v = own;
#pragma unroll
  for (int o = PER / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (tid % PER == 0) sm.groups[tid / PER] = v;
  if (tid < 32) sm.best[tid] = 0;
  if (tid < 4) sm.count[tid] = 0;
  __syncthreads();
  {   // rank of group tid / PER, each of its threads counting over a part of the groups
    constexpr int MANY = GROUPS / PER;
    const int group = tid / PER, from = tid % PER * MANY;
    const uint32_t mine = sm.groups[group];
    int rank = 0;
#pragma unroll
    for (int j = from; j < from + MANY; j += 4) {
      const uint4 o = *reinterpret_cast<const uint4*>(&sm.groups[j]);
      rank += (o.x > mine || (o.x == mine && j < group)) + (o.y > mine || (o.y == mine && j + 1 < group)) +
              (o.z > mine || (o.z == mine && j + 2 < group)) + (o.w > mine || (o.w == mine && j + 3 < group));
    }
#pragma unroll
    for (int o = PER / 2; o > 0; o >>= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
    if (rank == k - 1) sm.bound = mine;
  }
  __syncthreads();
  const uint32_t bound = sm.bound;
  // Two steps, so that a warp does not walk the chunks of its lanes one after the other: the chunks that hold something go on a
  // list, then every thread takes vectors of listed chunks.
  auto collect = [&](uint32_t least, int& chunks, int& count) {
    const float lf = key_value(least);
    auto offer = [&](float f, int at) {
      if (value_key(f) >= least) {
        const int slot = atomicAdd(&count, 1);
        if (slot < CAP) sm.cand[slot] = order_key(f, at);
      }
    };
    if (own >= least) {
      if (edge_at >= 0) offer(edge, edge_at);
      uint32_t some = 0;
#pragma unroll
      for (int ch = 0; ch < MAX_CHUNKS; ++ch) some |= (value_key(sm.cmax[ch][tid]) >= least ? 1u : 0u) << ch;
      for (; some != 0; some &= some - 1) sm.work[atomicAdd(&chunks, 1)] = static_cast<uint16_t>((__ffs(some) - 1) * THREADS + tid);
    }
    __syncthreads();
    const int units = chunks << cl_bits;
    for (int i = tid; i < units; i += THREADS) {
      if (*static_cast<volatile int*>(&count) > CAP) break;   // too many already: masked logits, for the most part
      const int w = sm.work[i >> cl_bits], j = (w / THREADS << cl_bits) + (i & ((1 << cl_bits) - 1));
      const int vec = first_vec + w % THREADS + j * THREADS;
      if (vec >= end_vec) continue;                   // the last chunk of a thread may be short, or there may be none
      const int at = head + vec * L;
      float f[L];
      Vec<T>::unpack(*reinterpret_cast<const uint4*>(r + at), f);
      uint32_t some = 0;
#pragma unroll
      for (int e = 0; e < L; ++e) some |= (f[e] < lf ? 0u : 1u) << e;     // NaN too
      for (; some != 0; some &= some - 1) offer(to_f(r[at + __ffs(some) - 1]), at + __ffs(some) - 1);
    }
    __syncthreads();
  };
  collect(bound, sm.count[0], sm.count[1]);
  const int n = sm.count[1];
  if (n <= CAP) {
    rank_keys<THREADS>(sm.cand, n, sm.best);
    __syncthreads();
    return;
  }
  if (bound != 0xffffffffu) collect(bound + 1, sm.count[2], sm.count[3]);
  const int above = sm.count[3];
  if (above <= CAP) {
    rank_keys<THREADS>(sm.cand, above, sm.best);
    int have = above;                                 // those equal to the bound follow in index order
    for (int base = lo; base < hi && have < k; base += THREADS) {
      const int i = base + tid;
      const bool eq = i < hi && value_key(to_f(r[i])) == bound;
      const uint32_t votes = __ballot_sync(0xffffffffu, eq);
      __syncthreads();
      if (lane == 0) sm.groups[warp] = __popc(votes);
      __syncthreads();
      int before = have, all = have;
      for (int w = 0; w < WARPS; ++w) {
        if (w < warp) before += sm.groups[w];
        all += sm.groups[w];
      }
      const int at = before + __popc(votes & ((1u << lane) - 1));
      if (eq && at < 32) sm.best[at] = order_key(to_f(r[i]), i);
      have = all;
    }
    __syncthreads();
    return;
  }
  unsigned long long last = ~0ull;
  for (int c = 0; c < k; ++c) {
    unsigned long long b = 0;
    for (int i = lo + tid; i < hi; i += THREADS) {
      const unsigned long long key = order_key(to_f(r[i]), i);
      if (key < last && key > b) b = key;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, b, o);
      b = other > b ? other : b;
    }
    __syncthreads();
    if (lane == 0) sm.cand[warp] = b;
    __syncthreads();
    for (int w = 0; w < WARPS; ++w) b = sm.cand[w] > b ? sm.cand[w] : b;
    last = b;
    if (tid == 0) sm.best[c] = b;
  }
  __syncthreads();
}

// One read of the logits: a row, or a part of it where there are few rows (the CTAs of a cluster then leave their sums and
// alternatives with the first one). Every thread keeps a running maximum and sums relative to it, and the maxima of its chunks
// for the alternatives. Bound by memory, closely followed by the issue of instructions (some ten an element at first): the
// maximum of four vectors at a time and loads without bounds checks but for the row's rest, 8192 x 128256 bf16 343 -> 317 us
// (6.6 TB/s) without alternatives, 432 -> 389 with 8 (347 to 390 from one GPU to another).
template <typename T, bool TOP, int THREADS>
__global__ void __launch_bounds__(THREADS, (sizeof(T) == 4 ? 1536 : 1280) / THREADS)
logprobs_kernel(const T* __restrict__ x, const long long* __restrict__ target, int V, const Rows rows, float inv_t, int k,
                long long ignore_index, int parts, float* __restrict__ logprob, float* __restrict__ entropy,
                float2* __restrict__ stats, float* __restrict__ top_lp, long long* __restrict__ top) {
  constexpr int L = Vec<T>::L, WARPS = THREADS / 32;
  __shared__ SumsSmem<THREADS> sm;
  __shared__ typename std::conditional<TOP, TopSmem<THREADS>, int>::type ts;
  const long long row = blockIdx.x / parts;
  const int part = static_cast<int>(blockIdx.x % parts);
  const T* r = rows.at(x, row);
  const long long tgt = target[row];
  const int tid = threadIdx.x, lane = tid & 31;
  if (tgt == ignore_index) {                         // the same for every CTA of the row: none of them meets a barrier
    if (part == 0) {
      if (tid == 0) {
        logprob[row] = entropy[row] = 0.f;
        if (stats) stats[row] = make_float2(0.f, 0.f);
      }
      if (tid < k) {
        top_lp[row * k + tid] = 0.f;
        top[row * k + tid] = -1;
      }
    }
    return;
  }
  if (parts > 1) cluster_arrive();                   // waited for before the exchange
  const bool inside = tgt >= 0 && tgt < V;
  const float xt = part == 0 && tid == 0 && inside ? to_f(r[tgt]) : 0.f;
  const float c = inv_t * L2E;
  // Sums start at a finite maximum, so that nothing below it (masked tokens, whatever their number) leaves a trace: a row whose
  // maximum is not above it, or as far on the other side, or whose sum is not a finite number, is done again at the end, with
  // differences taken before they are scaled.
  const float floor_ = -FAR / c;
  const RowSpan span = row_span(r, V);
  const int per = (span.nvec + parts - 1) / parts;
  const int first_vec = min(part * per, span.nvec), end_vec = min(first_vec + per, span.nvec);
  const int n = (end_vec - first_vec + THREADS - 1) / THREADS;      // vectors of a thread
  const int cl_bits = TOP ? chunk_bits(n) : 0;
  Sums a{floor_, 0.f, 0.f};
  float tmax = -INFINITY, cmax = -INFINITY;
  int chunk = 0, in_chunk = 0;
  auto take = [&](const uint4 (&v)[4]) {
    const float vm = Vec<T>::largest(v);
    if (vm > a.m) a.raise(vm, c);
    const float mo = offset_of(a.m, c);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float f[L];
      Vec<T>::unpack(v[q], f);
#pragma unroll
      for (int j = 0; j < L; ++j) {
        const float d = max_nan(fmaf(f[j], c, mo), -256.f), e = ex2(d);   // 2^-256 is 0: nothing from masked tokens
        a.s += e;
        a.u = fmaf(d, e, a.u);
      }
    }
    if constexpr (TOP) {
      cmax = max_nan(cmax, vm);
      in_chunk += 4;
      if (in_chunk == 1 << cl_bits) {
        ts.cmax[chunk++][tid] = cmax;
        tmax = max_nan(tmax, cmax);
        cmax = -INFINITY;
        in_chunk = 0;
      }
    }
  };
  const uint4* g = reinterpret_cast<const uint4*>(r + span.head) + tid;
  int i = first_vec;
  for (; i + 4 * THREADS <= end_vec; i += 4 * THREADS) {
    uint4 v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = load_stream(g + i + q * THREADS);
    take(v);
  }
  if (i + tid < end_vec) {                            // the rest of the row; absent vectors hold minus infinity
    uint4 v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q)
      v[q] = i + q * THREADS + tid < end_vec ? load_stream(g + i + q * THREADS)
                                             : make_uint4(Vec<T>::NEG_INF, Vec<T>::NEG_INF, Vec<T>::NEG_INF, Vec<T>::NEG_INF);
    take(v);
  }
  if constexpr (TOP) {
    tmax = max_nan(tmax, cmax);
    for (; chunk < MAX_CHUNKS; ++chunk) {
      ts.cmax[chunk][tid] = cmax;
      cmax = -INFINITY;
    }
  }
  // the elements before and after the vectors, one a thread
  const int edges = (part == 0 ? span.head : 0) + (part == parts - 1 ? span.tail : 0);
  float edge = -INFINITY;
  int edge_at = -1;
  if (tid < edges) {
    edge_at = part == 0 && tid < span.head ? tid : V - edges + tid;
    edge = to_f(r[edge_at]);
    tmax = max_nan(tmax, edge);
    if (edge > a.m) a.raise(edge, c);
    const float d = max_nan(fmaf(edge, c, offset_of(a.m, c)), -256.f), e = ex2(d);
    a.s += e;
    a.u = fmaf(d, e, a.u);
  }
  // the sums of the warp, then of the block: in the same order in every thread
  float wm = a.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) wm = fmaxf(wm, __shfl_xor_sync(0xffffffffu, wm, o));
  a.raise(wm, c);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
    a.u += __shfl_xor_sync(0xffffffffu, a.u, o);
  }
  if (lane == 0) {
    sm.warp[tid >> 5][0] = wm;
    sm.warp[tid >> 5][1] = a.s;
    sm.warp[tid >> 5][2] = a.u;
  }
  __syncthreads();
  auto combine = [&](const float (*of)[3], int n) {
    float top_m = of[0][0];
#pragma unroll 4
    for (int i = 1; i < n; ++i) top_m = fmaxf(top_m, of[i][0]);
    Sums t{top_m, 0.f, 0.f};
#pragma unroll 2
    for (int i = 0; i < n; ++i) {
      Sums o{of[i][0], of[i][1], of[i][2]};
      o.raise(top_m, c);
      t.s += o.s;
      t.u += o.u;
    }
    return t;
  };
  Sums all = combine(sm.warp, WARPS);
  if constexpr (TOP) {
    const int lo = part == 0 ? 0 : span.head + first_vec * L, hi = part == parts - 1 ? V : span.head + end_vec * L;
    part_top<T, THREADS>(r, first_vec, end_vec, span.head, edge, edge_at, tmax, cl_bits, k, lo, hi, ts);
  }
  if (parts > 1) {
    cluster_wait();                                  // every CTA of the cluster has started: the first one's memory is there
    if (tid < 32) {
      const uint32_t dst = map_to_cta(smem_u32(&sm.part[part][0]), 0);
      if (lane == 0) {
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst), "f"(all.m) : "memory");
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst + 4), "f"(all.s) : "memory");
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst + 8), "f"(all.u) : "memory");
      }
      if constexpr (TOP) {
        if (lane < k)
          asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(map_to_cta(smem_u32(&ts.lists[part * k + lane]), 0)), "l"(ts.best[lane]) : "memory");
      }
    }
    __syncwarp();
    cluster_sync_all();
    if (part != 0) return;
    all = combine(sm.part, parts);
    if constexpr (TOP) {
      if (tid < 32) ts.best[tid] = 0;
      __syncthreads();
      rank_keys<THREADS>(ts.lists, parts * k, ts.best);
      __syncthreads();
    }
  }
  float log_s = 0.f, H = 0.f;
  const bool again = !(all.m > floor_ && all.m * c < FAR && all.s < INFINITY);     // the same in all threads
  if (again) {
    auto add = [](float p, float q) { return p + q; };
    float mx = -INFINITY;
    for (int i = tid; i < V; i += THREADS) mx = max_nan(mx, to_f(r[i]));
    mx = block_reduce<THREADS>(mx, sm.red, [](float p, float q) { return max_nan(p, q); });
    float s = 0.f, u = 0.f;
    for (int i = tid; i < V; i += THREADS) {
      const float d = (to_f(r[i]) - mx) * inv_t;
      if (d != -INFINITY) {
        const float e = __expf(d);
        s += e;
        u += e == 0.f ? 0.f : d * e;
      }
    }
    s = block_reduce<THREADS>(s, sm.red, add);
    u = block_reduce<THREADS>(u, sm.red, add);
    all.m = mx;
    log_s = logf(s);
    H = log_s - u / s;
  }
  if (tid >= 32) return;
  if (!again) {
    // The maximum counts as 2^over. A row with one token left is exact: its sum is ex2(over) itself, and its mean differs from
    // `over` by the roundings of a product and a quotient, 2^-23 |over| together, below which a difference is none.
    const float over = fmaf(all.m, c, offset_of(all.m, c)), gap = all.u / all.s - over;
    log_s = logf(all.s / ex2(over));
    H = log_s - (fabsf(gap) <= 0x1p-22f * fabsf(over) ? 0.f : gap) * LN2;
  }
  log_s = max_nan(log_s, 0.f);                       // the sum has a term of 1, and no entropy is negative: roundings aside
  H = max_nan(H, 0.f);
  if (tid == 0) {
    logprob[row] = inside ? (xt - all.m) * inv_t - log_s : __uint_as_float(0x7fc00000u);
    entropy[row] = H;
    if (stats) stats[row] = make_float2(all.m, log_s);
  }
  if constexpr (TOP) {
    if (tid < k) {
      const unsigned long long best = ts.best[tid];
      const float v = key_value(static_cast<uint32_t>(best >> 32));
      top[row * k + tid] = static_cast<int>(0xffffffffu - static_cast<uint32_t>(best));
      top_lp[row * k + tid] = (v - all.m) * inv_t - log_s;
    }
  }
}

// dx_j = [ -p_j (G + gH (log p_j + H)) + g [j = target] + sum_i g_i [j = top_i] ] / temperature, G = g + sum_i g_i.
// Row blockIdx.x, part blockIdx.y. With l = log2 p_j the first term is p_j (l A + B); the chosen positions are written again.
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, 1280 / THREADS)
logprobs_bwd_kernel(const T* __restrict__ x, const long long* __restrict__ target, int V, const Rows rows, float inv_t, int k,
                    long long ignore_index, const long long* __restrict__ top, const float2* __restrict__ stats,
                    const float* __restrict__ entropy, const float* __restrict__ glp, const float* __restrict__ gh,
                    const float* __restrict__ gtop, T* __restrict__ dx, long long ldd) {
  constexpr int L = Vec<T>::L;
  const long long row = blockIdx.x;
  const T* r = rows.at(x, row);
  T* d = dx + row * ldd;
  const long long tgt = target[row];
  const int tid = threadIdx.x;
  const bool ignored = tgt == ignore_index;
  const float g = glp && !ignored ? glp[row] : 0.f, h = gh && !ignored ? gh[row] : 0.f;
  float G = g;
  bool any = g != 0.f || h != 0.f;
  if (gtop && !ignored)
    for (int i = 0; i < k; ++i) {
      G += gtop[row * k + i];
      any |= gtop[row * k + i] != 0.f;
    }
  if (tgt < 0 || tgt >= V) G += g * __uint_as_float(0x7fc00000u);      // a target outside the vocabulary: NaN
  const float2 st = stats[row];
  const float m = st.x, log_s = st.y, H = entropy[row], c = inv_t * L2E;
  const float A = -h * LN2 * inv_t, B = -(G + h * H) * inv_t, shift = -log_s * L2E;
  auto smooth = [&](float v) {
    const float l = max_nan(fmaf(v - m, c, shift), -256.f);
    return ex2(l) * fmaf(l, A, B);
  };
  const RowSpan span = row_span(r, V);
  const bool vec = ((reinterpret_cast<uintptr_t>(r) ^ reinterpret_cast<uintptr_t>(d)) & 15) == 0;
  const int parts = gridDim.y, part = blockIdx.y;
  int lo, hi;                                         // elements of this CTA
  if (vec) {
    const int per = (span.nvec + parts - 1) / parts;
    const int first = min(part * per, span.nvec), end = min(first + per, span.nvec);
    lo = part == 0 ? 0 : span.head + first * L;
    hi = part == parts - 1 ? V : span.head + end * L;
    const uint4* src = reinterpret_cast<const uint4*>(r + span.head);
    uint4* dst = reinterpret_cast<uint4*>(d + span.head);
    if (!any) {
      for (int i = first + tid; i < end; i += THREADS) dst[i] = make_uint4(0, 0, 0, 0);
    } else {
      for (int i = first + tid; i < end; i += 4 * THREADS) {
        uint4 v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (i + q * THREADS < end) v[q] = load_stream(src + i + q * THREADS);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if (i + q * THREADS >= end) continue;
          float f[L];
          Vec<T>::unpack(v[q], f);
#pragma unroll
          for (int j = 0; j < L; ++j) f[j] = smooth(f[j]);
          dst[i + q * THREADS] = Vec<T>::pack(f);
        }
      }
    }
    const int edges = (part == 0 ? span.head : 0) + (part == parts - 1 ? span.tail : 0);
    if (tid < edges) {
      const int at = part == 0 && tid < span.head ? tid : V - edges + tid;
      d[at] = from_f<T>(any ? smooth(to_f(r[at])) : 0.f);
    }
  } else {
    const int per = (V + parts - 1) / parts;
    lo = min(part * per, V);
    hi = min(lo + per, V);
    for (int i = lo + tid; i < hi; i += THREADS) d[i] = from_f<T>(any ? smooth(to_f(r[i])) : 0.f);
  }
  if (!any) return;
  __syncthreads();
  // the chosen positions again, with what they get besides: alternatives differ from one another, the target may be one
  if (gtop && tid < k) {
    const long long at = top[row * k + tid];
    if (at >= lo && at < hi)
      d[at] = from_f<T>(smooth(to_f(r[at])) + (gtop[row * k + tid] + (at == tgt ? g : 0.f)) * inv_t);
  }
  if (tid == MAX_TOP && tgt >= lo && tgt < hi) {
    bool taken = false;
    if (gtop)
      for (int i = 0; i < k; ++i) taken |= top[row * k + i] == tgt;
    if (!taken) d[tgt] = from_f<T>(smooth(to_f(r[tgt])) + g * inv_t);
  }
}

constexpr int SMALL = 128, LARGE = 256;     // threads of a CTA

// CTAs of a row: as many as `places` allow (two already where `first` does), with 4096 elements or more each.
int row_parts(long long T, int V, int first, int places) {
  int parts = 1;
  while (parts < MAX_PARTS && T * parts * 2 <= (parts == 1 ? first : places) && V / (parts * 2) >= 4096) parts *= 2;
  return parts;
}
// Small CTAs, of which an SM holds ten, hide the ends of short rows; a long row, or the only one an SM has, streams faster into a
// large one. Forward with 8 alternatives, 128 / 256 threads: 20000 x 2000 bf16 95 / 174 us, 6000 x 12000 47 / 72, 8192 x 32000
// 122 / 143, 4096 x 64000 104 / 113, 4096 x 128256 199 / 199, 1500 x 50021 fp32 63 / 59, 148 x 128256 30 / 19. CTAs of 512 threads,
// two to an SM: 8192 x 128256 466 / 389.
bool small_ctas(long long ctas, int V, int size) { return V <= 8192 || (static_cast<long long>(V) * size <= 128 * 1024 && ctas >= 592); }

inline int ok() { return cudaGetLastError() == cudaSuccess ? FSB_OK : FSB_ERR_LAUNCH; }
}  // namespace

// kind: 0 bf16, 1 fp16, 2 fp32. x: T rows of V elements, ld elements apart; with inner > 0 in batches of `inner` rows that start ldb
// elements apart. logprob, entropy [T]; stats [T, 2] (maximum
// and log s, for the backward pass; may be null); top_lp, top [T, k].
FSB_API int fsb_token_logprobs(const void* x, int kind, const long long* target, long long T, int V, long long inner, long long ldb,
                               long long ld, float inv_t, int k, long long ignore_index, float* logprob, float* entropy, void* stats, float* top_lp,
                               long long* top, cudaStream_t stream) {
  if (T < 0 || V <= 0 || k < 0 || k > MAX_TOP || k > V || kind < 0 || kind > 2 || inner < 0) return FSB_ERR_BAD_ARG;
  const Rows rows{inner, ldb, ld};
  if (T > 0x7fffffffll) return FSB_ERR_TOO_LARGE;
  if (T == 0) return FSB_OK;
  // Two CTAs of 256 threads for an SM's only row (148 x 128256: 10.1 / 13.4 us without and with 8 alternatives, one CTA 16.1 /
  // 18.5); more parts only towards one an SM, since their exchange costs more than it gains (74 x 128256 with alternatives, 2 / 4
  // / 8 parts: 10.3, 12.7, 19.8 us; without 7.3, 8.1, 8.3).
  const int parts = row_parts(T, V, 296, 148);
  if (T * parts > 0x7fffffffll) return FSB_ERR_TOO_LARGE;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(T * parts), 1, 1);
  const bool small = small_ctas(T * parts, V, kind == 2 ? 4 : 2);
  cfg.blockDim = dim3(small ? SMALL : LARGE, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = parts;
  at.val.clusterDim.y = 1;
  at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = parts > 1 ? 1 : 0;
  auto run = [&](auto* p) {
    using E = std::remove_const_t<std::remove_pointer_t<decltype(p)>>;
    auto kernel = k > 0 ? (small ? logprobs_kernel<E, true, SMALL> : logprobs_kernel<E, true, LARGE>)
                        : (small ? logprobs_kernel<E, false, SMALL> : logprobs_kernel<E, false, LARGE>);
    const cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, p, target, V, rows, inv_t, k, ignore_index, parts, logprob, entropy,
                                               static_cast<float2*>(stats), top_lp, top);
    const int rc = ok();   // also clears the error of a launch that failed
    return err == cudaSuccess ? rc : static_cast<int>(FSB_ERR_LAUNCH);
  };
  if (kind == 0) return run(static_cast<const __nv_bfloat16*>(x));
  if (kind == 1) return run(static_cast<const __half*>(x));
  return run(static_cast<const float*>(x));
}

// top, stats, entropy as the forward left them; glp, gh [T], gtop [T, k] (each may be null); dx [T, V] with row stride ldd.
FSB_API int fsb_token_logprobs_bwd(const void* x, int kind, const long long* target, long long T, int V, long long inner,
                                   long long ldb, long long ld, float inv_t, int k, long long ignore_index, const long long* top, const void* stats, const float* entropy,
                                   const float* glp, const float* gh, const float* gtop, void* dx, long long ldd,
                                   cudaStream_t stream) {
  if (T < 0 || V <= 0 || k < 0 || k > MAX_TOP || k > V || kind < 0 || kind > 2 || inner < 0) return FSB_ERR_BAD_ARG;
  const Rows rows{inner, ldb, ld};
  if (T > 0x7fffffffll) return FSB_ERR_TOO_LARGE;
  if (T == 0) return FSB_OK;
  // Parts have nothing to exchange here: up to 4096 CTAs, so that the last wave weighs little (1500 x 50021 fp32, 1 / 2 parts: 116 /
  // 108 us; 1000 x 50000 bf16, 1 / 4: 45 / 38), not more (4096 x 128256, 1 / 8: 339 / 368).
  auto run = [&](auto* p) {
    using E = std::remove_const_t<std::remove_pointer_t<decltype(p)>>;
    const dim3 grid(static_cast<unsigned>(T), row_parts(T, V, 4096, 4096));
    const bool small = V <= 8192;     // longer rows: even (8192 x 32000 187 / 189 us, 4096 x 128256 362 / 350)
    auto kernel = small ? logprobs_bwd_kernel<E, SMALL> : logprobs_bwd_kernel<E, LARGE>;
    kernel<<<grid, small ? SMALL : LARGE, 0, stream>>>(p, target, V, rows, inv_t, k, ignore_index, top,
                                                       static_cast<const float2*>(stats), entropy, glp, gh, gtop,
                                                       static_cast<E*>(dx), ldd);
    return ok();
  };
  if (kind == 0) return run(static_cast<const __nv_bfloat16*>(x));
  if (kind == 1) return run(static_cast<const __half*>(x));
  return run(static_cast<const float*>(x));
}
