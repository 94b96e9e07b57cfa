// Log probabilities of given tokens, entropy and top alternatives of rows of logits, and their gradient.
//
// With z = x / temperature, m = max z, s = sum e^(z - m), u = sum (z - m) e^(z - m):
//   log p_j = (z_j - m) - log s,   H = log s - u / s,
//   dH / dz_j = -p_j (log p_j + H),   d log p_i / dz_j = [i = j] - p_j.
// z - m is taken as (x - max x) / temperature: differences of logits of the type's lowest value do not overflow.
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
__device__ __forceinline__ unsigned long long order_key(float v, int index) {
  return static_cast<unsigned long long>(value_key(v)) << 32 | (0xffffffffu - static_cast<uint32_t>(index));
}

constexpr int THREADS = 512;

// Sum / maximum over the block, in every thread; the order of the additions is fixed.
template <typename F>
__device__ __forceinline__ float block_reduce(float v, float* red, F op) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[threadIdx.x & (THREADS / 32 - 1)];
#pragma unroll
  for (int o = THREADS / 64; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// One CTA per row: maximum, sums, then the alternatives one after the other.
template <typename T>
__global__ void __launch_bounds__(THREADS)
logprobs_kernel(const T* __restrict__ x, const long long* __restrict__ target, int V, long long ld, float inv_t, int k,
                long long ignore_index, float* __restrict__ logprob, float* __restrict__ entropy, float2* __restrict__ stats,
                float* __restrict__ top_lp, long long* __restrict__ top) {
  __shared__ float red[THREADS / 32];
  __shared__ unsigned long long best[THREADS / 32];
  const long long row = blockIdx.x;
  const T* r = x + row * ld;
  const long long tgt = target[row];
  const int tid = threadIdx.x;
  if (tgt == ignore_index) {
    if (tid == 0) {
      logprob[row] = entropy[row] = 0.f;
      stats[row] = make_float2(0.f, 0.f);
    }
    if (tid < k) {
      top_lp[row * k + tid] = 0.f;
      top[row * k + tid] = -1;
    }
    return;
  }
  float m = -INFINITY;
  for (int i = tid; i < V; i += THREADS) m = max_nan(m, to_f(r[i]));
  m = block_reduce(m, red, [](float a, float b) { return max_nan(a, b); });
  float s = 0.f, u = 0.f;
  for (int i = tid; i < V; i += THREADS) {
    const float d = (to_f(r[i]) - m) * inv_t;
    if (d != -INFINITY) {
      const float e = __expf(d);
      s += e;
      u += d * e;
    }
  }
  auto add = [](float a, float b) { return a + b; };
  s = block_reduce(s, red, add);
  u = block_reduce(u, red, add);
  const float log_s = logf(s);
  if (tid == 0) {
    logprob[row] = tgt >= 0 && tgt < V ? (to_f(r[tgt]) - m) * inv_t - log_s : __uint_as_float(0x7fc00000u);
    entropy[row] = log_s - u / s;
    stats[row] = make_float2(m, log_s);
  }
  unsigned long long last = ~0ull;
  for (int c = 0; c < k; ++c) {
    unsigned long long b = 0;
    for (int i = tid; i < V; i += THREADS) {
      const unsigned long long key = order_key(to_f(r[i]), i);
      if (key < last && key > b) b = key;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, b, o);
      b = other > b ? other : b;
    }
    __syncthreads();
    if ((tid & 31) == 0) best[tid >> 5] = b;
    __syncthreads();
    for (int w = 0; w < THREADS / 32; ++w) b = best[w] > b ? best[w] : b;
    last = b;
    if (tid == 0) {
      const int at = static_cast<int>(0xffffffffu - static_cast<uint32_t>(b));
      top[row * k + c] = at;
      top_lp[row * k + c] = (to_f(r[at]) - m) * inv_t - log_s;
    }
  }
}

// dx_j = [ -p_j (G + gH (log p_j + H)) + g [j = target] + sum_i g_i [j = top_i] ] / temperature, G = g + sum_i g_i.
template <typename T>
__global__ void __launch_bounds__(THREADS)
logprobs_bwd_kernel(const T* __restrict__ x, const long long* __restrict__ target, int V, long long ld, float inv_t, int k,
                    long long ignore_index, const long long* __restrict__ top, const float2* __restrict__ stats,
                    const float* __restrict__ entropy, const float* __restrict__ glp, const float* __restrict__ gh,
                    const float* __restrict__ gtop, T* __restrict__ dx, long long ldd) {
  const long long row = blockIdx.x;
  const T* r = x + row * ld;
  T* d = dx + row * ldd;
  const long long tgt = target[row];
  const int tid = threadIdx.x;
  const bool ignored = tgt == ignore_index;
  const float g = glp && !ignored ? glp[row] : 0.f, h = gh && !ignored ? gh[row] : 0.f;
  float G = g;
  bool any = g != 0.f || h != 0.f;
  if (gtop && !ignored)
    for (int c = 0; c < k; ++c) {
      G += gtop[row * k + c];
      any |= gtop[row * k + c] != 0.f;
    }
  if (!any) {
    for (int i = tid; i < V; i += THREADS) d[i] = from_f<T>(0.f);
    return;
  }
  if (tgt < 0 || tgt >= V) G += g * __uint_as_float(0x7fc00000u);      // a target outside the vocabulary: NaN
  const float m = stats[row].x, log_s = stats[row].y, H = entropy[row];
  auto smooth = [&](float v) {
    const float lp = (v - m) * inv_t - log_s, p = __expf(lp);
    return p == 0.f ? 0.f * G : -p * (G + h * (lp + H));
  };
  for (int i = tid; i < V; i += THREADS) d[i] = from_f<T>(smooth(to_f(r[i])) * inv_t);
  __syncthreads();
  // the chosen positions again, with what they get besides: alternatives differ from one another, the target may be one
  bool taken = false;
  if (gtop)
    for (int c = 0; c < k; ++c) taken |= top[row * k + c] == tgt;
  if (tid < k && gtop) {
    const long long at = top[row * k + tid];
    d[at] = from_f<T>((smooth(to_f(r[at])) + gtop[row * k + tid] + (at == tgt ? g : 0.f)) * inv_t);
  }
  if (tid == MAX_TOP && !taken && tgt >= 0 && tgt < V) d[tgt] = from_f<T>((smooth(to_f(r[tgt])) + g) * inv_t);
}

inline int ok() { return cudaGetLastError() == cudaSuccess ? FSB_OK : FSB_ERR_LAUNCH; }
}  // namespace

// kind: 0 bf16, 1 fp16, 2 fp32. x [T, V] with row stride ld elements; logprob, entropy [T]; stats [T, 2] (maximum
// and log s, for the backward pass); top_lp, top [T, k].
FSB_API int fsb_token_logprobs(const void* x, int kind, const long long* target, long long T, int V, long long ld, float inv_t,
                               int k, long long ignore_index, float* logprob, float* entropy, void* stats, float* top_lp,
                               long long* top, cudaStream_t stream) {
  if (T < 0 || V <= 0 || k < 0 || k > MAX_TOP || k > V || kind < 0 || kind > 2) return FSB_ERR_BAD_ARG;
  if (T > 0x7fffffffll) return FSB_ERR_TOO_LARGE;
  if (T == 0) return FSB_OK;
  auto run = [&](auto* p) {
    logprobs_kernel<<<static_cast<unsigned>(T), THREADS, 0, stream>>>(p, target, V, ld, inv_t, k, ignore_index, logprob, entropy,
                                                                      static_cast<float2*>(stats), top_lp, top);
    return ok();
  };
  if (kind == 0) return run(static_cast<const __nv_bfloat16*>(x));
  if (kind == 1) return run(static_cast<const __half*>(x));
  return run(static_cast<const float*>(x));
}

// top, stats, entropy as the forward left them; glp, gh [T], gtop [T, k] (each may be null); dx [T, V] with row stride ldd.
FSB_API int fsb_token_logprobs_bwd(const void* x, int kind, const long long* target, long long T, int V, long long ld, float inv_t,
                                   int k, long long ignore_index, const long long* top, const void* stats, const float* entropy,
                                   const float* glp, const float* gh, const float* gtop, void* dx, long long ldd,
                                   cudaStream_t stream) {
  if (T < 0 || V <= 0 || k < 0 || k > MAX_TOP || k > V || kind < 0 || kind > 2) return FSB_ERR_BAD_ARG;
  if (T > 0x7fffffffll) return FSB_ERR_TOO_LARGE;
  if (T == 0) return FSB_OK;
  auto run = [&](auto* p) {
    using E = std::remove_const_t<std::remove_pointer_t<decltype(p)>>;
    logprobs_bwd_kernel<<<static_cast<unsigned>(T), THREADS, 0, stream>>>(p, target, V, ld, inv_t, k, ignore_index, top,
                                                                          static_cast<const float2*>(stats), entropy, glp, gh, gtop, static_cast<E*>(dx), ldd);
    return ok();
  };
  if (kind == 0) return run(static_cast<const __nv_bfloat16*>(x));
  if (kind == 1) return run(static_cast<const __half*>(x));
  return run(static_cast<const float*>(x));
}
