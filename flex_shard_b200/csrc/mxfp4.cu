// MXFP4 (e2m1 data, two codes a byte, one power-of-two e8m0 scale per 32 elements) for sm_100a: quantisers, the expansion
// of codes into values and the block-scaled product (tcgen05.mma kind::mxf4.block_scale).
//
// Scale of a group with largest magnitude amax = f 2^k (1 <= f < 2): the smallest power of two s with amax / s <= 6, that is
// 2^(k-2) for f <= 1.5 and 2^(k-1) otherwise, stored as the byte log2(s) + 127, not below 0 (an all-zero group: 0). A group
// that holds a NaN or an infinity gets the byte 255, the format's NaN, so that the products it enters are NaN.
// q = e2m1(x / s), rounded to nearest with ties to even; the quotient is exact. The code of an even column is the low nibble.
//
// Scale tensors are in the tensor core's block layout (128 rows x 4 groups = 512 bytes, the byte of (row r, group g) at
// (r % 32) * 16 + (r / 32) * 4 + g), as for MXFP8; padding rows and groups hold 127.
#include "common.cuh"
#include <cuda_fp4.h>
#include <cuda_fp8.h>

// the MXFP8 quantisers and product (mxfp8.cu), on which the gradients run
FSB_API int fsb_mx_quant_act(const void* x, void* q, void* scales, long long T, int K, long long ldx, long long ldq,
                             cudaStream_t stream);
FSB_API int fsb_mx_quant_rows(const void* x, void* q, void* scales, long long T, int K, long long ldx, long long ldq,
                              cudaStream_t stream);
FSB_API int fsb_gemm_mxfp8(const void* aq, const void* sfa, const void* bq, const void* sfb, void* d, int M, int N, int K,
                           long long lda, long long ldb, long long ldd, int a_mn, int b_mn, int d_fp32, int* status,
                           cudaStream_t stream);

namespace {
using namespace fsb;

// Waits for the kernel that this one was launched behind, where it may start before that one ends; nothing otherwise.
__device__ __forceinline__ void wait_for_previous_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_kernel_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Biased exponent from the bits of amax (not negative). 0x7f800000 and above: an infinity or a NaN.
__device__ __forceinline__ uint32_t mx4_exponent(uint32_t bits) {
  if (bits >= 0x7f800000u) return 255u;
  const int e = static_cast<int>(bits >> 23) - 2 + ((bits & 0x7fffffu) > 0x400000u ? 1 : 0);
  return e < 0 ? 0u : static_cast<uint32_t>(e);
}
__device__ __forceinline__ float mx4_inv(uint32_t e) {   // 2^(127 - e) for e <= 253; 0 for the NaN byte (all codes 0)
  return e == 255u ? 0.f : __uint_as_float((254u - e) << 23);
}
__device__ __forceinline__ float mx4_scale(uint32_t e) {   // 2^(e - 127); the NaN byte gives a NaN
  return e == 0u ? __uint_as_float(0x00400000u) : e == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(e << 23);
}
__device__ __forceinline__ long long blocked_offset(long long r, int g, int n_gb) {
  return ((r >> 7) * n_gb + (g >> 2)) * 512 + (r & 31) * 16 + ((r >> 5) & 3) * 4 + (g & 3);
}
// The magnitudes' bits order like the magnitudes, with infinities and NaN on top, so the maximum is taken on integers.
__device__ __forceinline__ uint32_t amax8_bits(const uint4& raw, uint32_t m) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) m = max(m, max(w[j] << 16 & 0x7fff0000u, w[j] & 0x7fff0000u));
  return m;
}
// Eight bf16 as eight codes. x * inv is exact or rounds far below the smallest code's half step. With inv == 0 (the NaN
// byte) infinities and NaN would give NaN, for which the conversion has no code: the codes are 0.
__device__ __forceinline__ uint32_t quant8_fp4(const uint4& raw, float inv) {
  if (inv == 0.f) return 0u;
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw);
  uint32_t o = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = __bfloat1622float2(h[j]);
    o |= static_cast<uint32_t>(__nv_cvt_float2_to_fp4x2(make_float2(f.x * inv, f.y * inv), __NV_E2M1, cudaRoundNearest)) << (8 * j);
  }
  return o;
}
__device__ __forceinline__ uint4 load8_any(const __nv_bfloat16* p, bool vec) {
  if (vec) return *reinterpret_cast<const uint4*>(p);
  const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
  return make_uint4(h[0] | static_cast<uint32_t>(h[1]) << 16, h[2] | static_cast<uint32_t>(h[3]) << 16,
                    h[4] | static_cast<uint32_t>(h[5]) << 16, h[6] | static_cast<uint32_t>(h[7]) << 16);
}

// ------------------------------------------------------------------ activation quantiser (1x32 groups)
// Two threads per group, 16 columns each, UNITS such pieces a thread in flight: bound by memory, 2.53 bytes an element. The
// eight threads of a scale block's row gather its four bytes into one word. Rows past T and groups past K / 32 get the byte
// 127. I: the type that counts pieces (a 64-bit quotient per piece costs as much as the rest).
// 5765 x 14336: 40.9 us (5.1 TB/s); one piece a thread 43.9, four 42.6; with 64-bit counting and 8 columns a thread 67.9.
constexpr int UNITS = 2;
template <typename I>
__global__ void __launch_bounds__(256)
mx4_quant_act_kernel(const __nv_bfloat16* __restrict__ x, uint8_t* __restrict__ q, uint8_t* __restrict__ scales, long long T,
                     int K, long long ldx, int n_gb, int vec) {
  let_next_kernel_start();
  const I units = n_gb * 8;                               // pieces of a padded row
  const I total = static_cast<I>((T + 127) / 128 * 128) * units, share = total / UNITS;   // both multiples of 8
  const I i0 = static_cast<I>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i0 >= share) return;                                // the eight threads of a row's block leave together
  uint4 v[UNITS][2];
  long long row[UNITS];
  int u[UNITS];
  bool live[UNITS];
#pragma unroll
  for (int j = 0; j < UNITS; ++j) {
    const I i = i0 + j * share, r = i / units;
    row[j] = r;
    u[j] = static_cast<int>(i - r * units);
    live[j] = row[j] < T && u[j] * 16 < K;
    v[j][0] = v[j][1] = make_uint4(0, 0, 0, 0);
    if (live[j]) {
      const __nv_bfloat16* p = x + row[j] * ldx + u[j] * 16;
      v[j][0] = load8_any(p, vec);
      v[j][1] = load8_any(p + 8, vec);
    }
  }
  const unsigned octet = 0xffu << (threadIdx.x & 24);
#pragma unroll
  for (int j = 0; j < UNITS; ++j) {
    uint32_t m = amax8_bits(v[j][1], amax8_bits(v[j][0], 0u));
    m = max(m, __shfl_xor_sync(octet, m, 1));
    const uint32_t e = mx4_exponent(m);
    uint32_t word = (live[j] ? e : 127u) << (4 * (threadIdx.x & 6));
    word |= __shfl_xor_sync(octet, word, 2);
    word |= __shfl_xor_sync(octet, word, 4);
    if ((threadIdx.x & 7) == 0) *reinterpret_cast<uint32_t*>(scales + blocked_offset(row[j], u[j] >> 1, n_gb)) = word;
    if (live[j]) {
      const float inv = mx4_inv(e);
      *reinterpret_cast<uint2*>(q + row[j] * (K / 2) + u[j] * 8) = make_uint2(quant8_fp4(v[j][0], inv), quant8_fp4(v[j][1], inv));
    }
  }
}

// ------------------------------------------------------------------ weight quantiser (32x32 tiles)
// A block takes 128 rows x 32 TC columns, a warp 32 rows of them: TC tiles, 4 TC 16-byte reads a lane in flight, 64 TC bytes of a
// row side by side. One tile exponent serves the forward product (groups along the columns) and the input gradient (groups along
// the rows); the block writes its part of the scale block of either operand, padding included (a grid that covers whole scale
// blocks). Bound by memory, 2.53 bytes an element: 28660 x 4096 58.6 us (5.1 TB/s) with TC = 4, 60.2 with TC = 1, which gives a
// small weight four times the blocks: 500 x 2048 2.7 us against 4.5.
template <int TC>
__global__ void __launch_bounds__(128)
mx4_quant_weight_kernel(const __nv_bfloat16* __restrict__ w, uint8_t* __restrict__ q, uint8_t* __restrict__ tile_exp,
                        uint8_t* __restrict__ fwd, uint8_t* __restrict__ dgrad, int rows, int cols, long long ldw, int vec) {
  constexpr int LANES = 4 * TC, STEP = 32 / LANES;    // lanes of a row, rows of a pass
  __shared__ uint8_t exps[4][TC];                     // [tile row][tile column] of the block; 127 outside the matrix
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c0 = blockIdx.x * 32 * TC + lane % LANES * 8;
  const long long row0 = static_cast<long long>(blockIdx.y) * 128 + warp * 32, r0 = row0 + lane / LANES;
  const bool in_cols = c0 < cols;
  uint4 v[LANES];
#pragma unroll
  for (int i = 0; i < LANES; ++i)
    v[i] = in_cols && r0 + STEP * i < rows ? load8_any(w + (r0 + STEP * i) * ldw + c0, vec) : make_uint4(0, 0, 0, 0);
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < LANES; ++i) m = amax8_bits(v[i], m);
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
#pragma unroll
  for (int o = LANES; o < 32; o *= 2) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  const uint32_t e = mx4_exponent(m);
  const float inv = mx4_inv(e);
#pragma unroll
  for (int i = 0; i < LANES; ++i)
    if (in_cols && r0 + STEP * i < rows) *reinterpret_cast<uint32_t*>(q + (r0 + STEP * i) * (cols / 2) + c0 / 2) = quant8_fp4(v[i], inv);
  if (lane < LANES && (lane & 3) == 0) {
    const bool inside = in_cols && row0 < rows;
    exps[warp][lane >> 2] = inside ? static_cast<uint8_t>(e) : 127;
    if (inside) tile_exp[(row0 >> 5) * (cols / 32) + (c0 >> 5)] = static_cast<uint8_t>(e);
  }
  if (fwd == nullptr) return;
  __syncthreads();
  const int t = threadIdx.x, col_blocks = (cols + 127) / 128;
  const long long at = static_cast<long long>(blockIdx.y) * 128 + t;            // row of the forward operand
#pragma unroll
  for (int g = 0; g < TC; ++g) fwd[blocked_offset(at, blockIdx.x * TC + g, col_blocks)] = at < rows ? exps[t >> 5][g] : 127;
  if (t < 32 * TC) {                                                            // row of the transposed operand: four groups
    uint32_t d = 0;
#pragma unroll
    for (int g = 0; g < 4; ++g) d |= static_cast<uint32_t>(exps[g][t >> 5]) << (8 * g);
    *reinterpret_cast<uint32_t*>(dgrad + blocked_offset(static_cast<long long>(blockIdx.x) * 32 * TC + t, blockIdx.y * 4, gridDim.y)) = d;
  }
}

// ------------------------------------------------------------------ expansion
// Codes as the values they stand for: e4m3 without the scales (KIND 0, every e2m1 value is one of e4m3), bf16 (1) or fp32 (2)
// with them. e2m1 values times powers of two are exact in all three, but for what underflows. Pieces of 16 (e4m3) or 8 codes,
// EXPAND_UNITS a thread in flight: bound by memory. 28660 x 4096 to bf16 / e4m3: 50 / 29 us (5.9 / 6.1 TB/s), two pieces a thread
// 55 / 30, one 68 / 35.
constexpr int EXPAND_UNITS = 4;
__device__ __forceinline__ __half2 fp4x2_values(uint32_t byte) {
  return __half2(__nv_cvt_fp4x2_to_halfraw2(static_cast<__nv_fp4x2_storage_t>(byte), __NV_E2M1));
}
template <int KIND, typename I>
__global__ void __launch_bounds__(256)
mx4_expand_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ scales, void* __restrict__ out, long long T, int K,
                  long long ldq, int n_gb) {
  constexpr int C = KIND == 0 ? 16 : 8;
  const I units = K / C, total = static_cast<I>(T) * units, share = (total + EXPAND_UNITS - 1) / EXPAND_UNITS;
  const I i0 = static_cast<I>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i0 >= share) return;
  uint32_t c[EXPAND_UNITS][C / 8];
  uint32_t e[EXPAND_UNITS];
  long long at[EXPAND_UNITS];
#pragma unroll
  for (int j = 0; j < EXPAND_UNITS; ++j) {
    const I i = i0 + j * share, r = i / units;
    const int u = static_cast<int>(i - r * units);
    at[j] = i < total ? static_cast<long long>(r) * K + u * C : -1;
    if (at[j] < 0) continue;
    const uint32_t* p = reinterpret_cast<const uint32_t*>(q + static_cast<long long>(r) * ldq) + u * (C / 8);
#pragma unroll
    for (int w = 0; w < C / 8; ++w) c[j][w] = p[w];
    if (KIND != 0) e[j] = scales[blocked_offset(r, u >> 2, n_gb)];
  }
#pragma unroll
  for (int j = 0; j < EXPAND_UNITS; ++j) {
    if (at[j] < 0) continue;
    if constexpr (KIND == 0) {
      uint32_t o[4];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t two = c[j][w >> 1] >> (16 * (w & 1));
        const uint32_t lo = __nv_cvt_halfraw2_to_fp8x2(fp4x2_values(two & 0xffu), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_halfraw2_to_fp8x2(fp4x2_values(two >> 8 & 0xffu), __NV_SATFINITE, __NV_E4M3);
        o[w] = lo | hi << 16;
      }
      *reinterpret_cast<uint4*>(static_cast<uint8_t*>(out) + at[j]) = make_uint4(o[0], o[1], o[2], o[3]);
    } else {
      const float s = mx4_scale(e[j]);
      float2 f[4];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        f[w] = __half22float2(fp4x2_values(c[j][0] >> (8 * w) & 0xffu));
        f[w].x *= s;
        f[w].y *= s;
      }
      if constexpr (KIND == 2) {
        float4* d = reinterpret_cast<float4*>(static_cast<float*>(out) + at[j]);
        d[0] = make_float4(f[0].x, f[0].y, f[1].x, f[1].y);
        d[1] = make_float4(f[2].x, f[2].y, f[3].x, f[3].y);
      } else {
        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(out) + at[j]) =
            make_uint4(pack_bf16x2(f[0].x, f[0].y), pack_bf16x2(f[1].x, f[1].y), pack_bf16x2(f[2].x, f[2].y), pack_bf16x2(f[3].x, f[3].y));
      }
    }
  }
}

// ------------------------------------------------------------------ block-scaled product
// out[t, n] = sum_k a[t, k] b[n, k]. The weight b is the tensor core's M operand (128 rows a tile), the rows t its N operand,
// so that a tile of few rows costs few columns. A stage is 256 deep (128 bytes a row, the swizzle's width): four 64-deep MMAs,
// each with two scale bytes a row. The scales travel as whole blocks (two per 128 rows and stage) and are copied to TMEM right
// before the MMAs. Codes past K read as zeros; so do scale blocks past the last one.
constexpr int BM = 128, BK = 256, KB = BK / 2;      // KB: bytes of a row in a stage
constexpr int SF_BYTES = 1024;                      // two scale blocks
constexpr int NUM_THREADS = 192;                    // warp 0 TMA, warp 1 MMA, warps 2..5 epilogue

template <int BN>
struct Tile {
  static constexpr int A_STAGE = BM * KB, B_STAGE = BN * KB;
  static constexpr int STAGE_BYTES = A_STAGE + B_STAGE + 2 * SF_BYTES;   // a multiple of 1 KB for BN >= 16 in steps of 8
  static constexpr int STAGES = 4;                                       // two CTAs fit an SM (BN = 128: one)
  // steps of a CTA along K that are worth the joining of the parts (measured with 2, 4, 8 and without a split: 32 x 6144 x 4096
  // 12.9, 9.4, 9.7, 10.4 us; 64 x 4096 x 14336 13.7, 13.7, 13.1, 22.9; 128 x 6144 x 4096 20.9, 20.9, 14.1, 12.6)
  static constexpr int LEAST = BN == 128 ? 14 : BN == 64 ? 8 : 4;
  static constexpr int SMEM = STAGES * STAGE_BYTES + 1024 + 256;
  static constexpr int SF_COL0 = BN < 32 ? 32 : BN;                      // first scale column
  static constexpr int TMEM_COLS = BN <= 64 ? 128 : 256;                 // accumulator + two sets of 8 + 8 scale columns
};

constexpr int MAX_SPLIT = 8;                        // CTAs along K (a portable cluster)

struct Args {
  int M, N, K;
  int split, chunk;                                 // CTAs of a cluster along K, 256-deep steps of each
  void* d;
  long long ldd;
  int d_fp32;
  int* status;
};

__device__ __forceinline__ void tmem_cp_32x128b_x4(uint32_t taddr, uint64_t sdesc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sdesc) : "memory");
}
// Unswizzled K-major descriptor: 8-row groups of 16-byte rows are 128 bytes apart.
__device__ __forceinline__ uint64_t make_sf_desc(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr >> 4) & 0x3FFF);
  d |= static_cast<uint64_t>(128 >> 4) << 32;   // SBO
  d |= 1ull << 46;
  return d;
}
__device__ __forceinline__ void umma_mxf4(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t tsfa,
                                          uint32_t tsfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
      ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(tsfa), "r"(tsfb)
      : "memory");
}
// e2m1 x e2m1 (format 1 of this kind), e8m0 scales, both operands K-major; sf_id: first of the scale word's bytes used (0, 2)
__device__ __forceinline__ constexpr uint32_t make_idesc_mx4(uint32_t m, uint32_t n, uint32_t sf_id) {
  return (sf_id << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | (1u << 23) | ((m >> 7) << 27) | (sf_id << 29);
}

// Four neighbouring columns of row t.
__device__ __forceinline__ void store4(const Args& args, int t, int n, const float4& v) {
  const long long at = static_cast<long long>(t) * args.ldd + n;
  if (args.d_fp32) {
    float* d = static_cast<float*>(args.d) + at;
    if (n + 4 <= args.N && (reinterpret_cast<uintptr_t>(d) & 15) == 0) {
      *reinterpret_cast<float4*>(d) = v;
      return;
    }
    const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < args.N) d[i] = f[i];
  } else {
    __nv_bfloat16* d = static_cast<__nv_bfloat16*>(args.d) + at;
    if (n + 4 <= args.N && (reinterpret_cast<uintptr_t>(d) & 7) == 0) {
      *reinterpret_cast<uint2*>(d) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
      return;
    }
    const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < args.N) d[i] = __float2bfloat16(f[i]);
  }
}
// End of the one-SM kernels, for all threads of a CTA: its epilogue warps (2 to 5) have left its sums [rows][128] at `smem` (a
// thread there has one weight row, 2 bytes of each output row; here it stores 8 of one). With several CTAs along K the cluster's
// sums are added in CTA order and the CTAs divide the rows; all parts' 16 bytes are on their way before the first is added.
__device__ __forceinline__ void store_rows(const Args& args, const uint8_t* smem, int part, int t0, int rows, int n0) {
  const int thread = static_cast<int>(threadIdx.x) - 64, n = thread % 32 * 4;
  if (args.split == 1) {
    if (thread < 0) return;
    asm volatile("bar.sync 1, 128;" ::: "memory");
#pragma unroll 4
    for (int t = thread / 32; t < rows; t += 4) store4(args, t0 + t, n0 + n, *reinterpret_cast<const float4*>(smem + (t * BM + n) * 4));
    return;
  }
  __syncwarp();
  cluster_sync_all();
  if (thread >= 0) {
    const int per = (rows + args.split - 1) / args.split, end = min((part + 1) * per, rows);
#pragma unroll 2
    for (int t = part * per + thread / 32; t < end; t += 4) {
      const uint32_t own = smem_u32(smem) + (t * BM + n) * 4;
      float4 o[MAX_SPLIT], sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int p = 0; p < MAX_SPLIT; ++p) {
        o[p] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (p < args.split)
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(o[p].x), "=f"(o[p].y), "=f"(o[p].z), "=f"(o[p].w) : "r"(map_to_cta(own, p)));
      }
#pragma unroll
      for (int p = 0; p < MAX_SPLIT; ++p) {
        sum.x += o[p].x;
        sum.y += o[p].y;
        sum.z += o[p].z;
        sum.w += o[p].w;
      }
      store4(args, t0 + t, n0 + n, sum);
    }
  }
  __syncwarp();
  cluster_sync_all();                                          // the others' sums have been read
}

template <int BN>
__global__ void __launch_bounds__(NUM_THREADS)
gemm_mxfp4_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                  const __grid_constant__ CUtensorMap map_sfw, const __grid_constant__ CUtensorMap map_sfx, const Args args) {
  using S = Tile<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::STAGES * S::STAGE_BYTES);
  uint64_t* full_bar = bars;
  uint64_t* empty_bar = bars + S::STAGES;
  uint64_t* tmem_full = bars + 2 * S::STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * S::STAGES + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tw = blockIdx.x / args.split, part = blockIdx.x % args.split, tx = blockIdx.y, rows = min(BN, args.M - tx * BN);
  const int num_kb = (args.K + BK - 1) / BK;
  const int kb0 = min(part * args.chunk, num_kb), steps = min(kb0 + args.chunk, num_kb) - kb0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(tmem_full, 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, S::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      tma_prefetch_desc(&map_w);
      tma_prefetch_desc(&map_x);
      auto load_weight = [&](int i) {
        const int s = i % S::STAGES, kb = kb0 + i;
        uint8_t* sa = smem + s * S::STAGE_BYTES;
        mbar_expect_tx(&full_bar[s], S::STAGE_BYTES);
        tma_load_2d(sa, &map_w, &full_bar[s], kb * KB, tw * BM);
        tma_load_2d(sa + S::A_STAGE + S::B_STAGE, &map_sfw, &full_bar[s], kb * 256, tw);   // 256 words: two blocks
      };
      const int ahead = min(steps, S::STAGES);
      for (int i = 0; i < ahead; ++i) load_weight(i);          // does not wait for the rows' quantiser
      wait_for_previous_kernel();
      for (int i = 0; i < steps; ++i) {
        const int s = i % S::STAGES, kb = kb0 + i;
        if (i >= ahead) {
          if (!mbar_wait(&empty_bar[s], ((i / S::STAGES) & 1) ^ 1, abort_flag)) {
            atomicExch(args.status, FSB_ERR_WAIT_TIMEOUT_EMPTY);
            *abort_flag = 1;
            break;
          }
          load_weight(i);
        }
        uint8_t* sb = smem + s * S::STAGE_BYTES + S::A_STAGE;
        tma_load_2d(sb, &map_x, &full_bar[s], kb * KB, tx * BN);
        tma_load_2d(sb + S::B_STAGE + SF_BYTES, &map_sfx, &full_bar[s], kb * 256, tx * BN / 128);
      }
    }
  } else if (warp == 1) {
    // The whole warp walks the loop; one elected lane issues the tcgen05 instructions.
    bool ok = steps > 0;
    for (int i = 0; i < steps; ++i) {
      const int s = i % S::STAGES;
      if (!mbar_wait(&full_bar[s], (i / S::STAGES) & 1, abort_flag)) {
        if (lane == 0) {
          atomicExch(args.status, FSB_ERR_WAIT_TIMEOUT_FULL);
          *abort_flag = 1;
        }
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t sa = smem_u32(smem + s * S::STAGE_BYTES);
      const uint64_t da = make_smem_desc_sw128(sa, 16, 1024);
      const uint64_t db = make_smem_desc_sw128(sa + S::A_STAGE, 16, 1024);
      const uint32_t ssf = sa + S::A_STAGE + S::B_STAGE;
      const uint32_t tsf = tmem_base + S::SF_COL0 + (i & 1) * 16;   // 2 x 4 columns of weight scales, 2 x 4 of row scales
      if (elect_one()) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          tmem_cp_32x128b_x4(tsf + 4 * h, make_sf_desc(ssf + 512 * h));
          tmem_cp_32x128b_x4(tsf + 8 + 4 * h, make_sf_desc(ssf + SF_BYTES + 512 * h));
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_mxf4(tmem_base, da + 2 * k, db + 2 * k, make_idesc_mx4(BM, BN, (k & 1) * 2), tsf + 4 * (k >> 1),
                    tsf + 8 + 4 * (k >> 1), (i | k) != 0);
        umma_commit(&empty_bar[s]);
      }
      __syncwarp();
    }
    if (ok) {
      if (elect_one()) umma_commit(tmem_full);
      __syncwarp();
    }
  } else {
    const int quarter = warp & 3;
    const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    const bool done = steps > 0 && mbar_wait_warp(tmem_full, 0, abort_flag);
    if (steps > 0 && !done && lane == 0) {
      atomicExch(args.status, FSB_ERR_WAIT_TIMEOUT_TMEM_FULL);
      *abort_flag = 1;
    }
    tc_fence_after();
    uint32_t* sums = reinterpret_cast<uint32_t*>(smem) + quarter * 32 + lane;   // the stages are free by now
#pragma unroll
    for (int c0 = 0; c0 < BN; c0 += 16) {
      if (c0 >= rows) break;
      uint32_t v[16];
      if (done) {
        tmem_ld_32x16(t_row + c0, v);
        tmem_ld_wait();
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = 0;                 // nothing along K for this CTA
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) sums[(c0 + i) * BM] = v[i];
    }
    tc_fence_before();
  }
  store_rows(args, smem, part, tx * BN, rows, tw * BM);
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    if (*abort_flag) {
      const unsigned long long t0 = clock64();
      while (clock64() - t0 < 2000000ull) {
      }
    }
    tc_fence_after();
    tmem_dealloc(tmem_base, S::TMEM_COLS);
  }
}

// ------------------------------------------------------------------ few rows: quantised on the way, split along K
// Up to 16 rows of bf16 against a weight in one launch, as long as a CTA's share of them is FEW_GROUPS groups or less. The CTAs of a cluster share a tile of 128 weight rows and divide its
// K; each quantises its own columns of the rows straight into shared memory (the 128-byte swizzle's order: one group is one
// 16-byte chunk) while the weight streams in, and the partial sums meet in the cluster's shared memory, added in CTA order.
// Bound by the weight's bytes where there are enough of them, else by the latency of one load, one chain of MMAs and the exchange.
constexpr int F_BN = 16, F_STAGES = 3;
constexpr int F_STAGE_BYTES = BM * KB + SF_BYTES;            // weight codes and scales: 17 KB
constexpr int F_ROW_BYTES = F_BN * KB + SF_BYTES;            // the rows' codes and scales of 256 columns: 3 KB
constexpr int F_SF_COL0 = 32, F_TMEM_COLS = 64;
constexpr int FEW_GROUPS = 512;                                // most groups a CTA quantises, four a thread
constexpr int few_smem(int chunk) { return F_STAGES * F_STAGE_BYTES + chunk * F_ROW_BYTES + 1024 + 256; }

__global__ void __launch_bounds__(NUM_THREADS)
linear_mxfp4_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_sfw,
                        const __nv_bfloat16* __restrict__ x, long long ldx, int vec, const Args args) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* rows_q = smem + F_STAGES * F_STAGE_BYTES;          // [chunk][16 rows][128 bytes]
  uint8_t* rows_sf = rows_q + args.chunk * F_BN * KB;              // [chunk][two scale blocks]
  uint64_t* bars = reinterpret_cast<uint64_t*>(rows_sf + args.chunk * SF_BYTES);
  uint64_t* full_bar = bars;
  uint64_t* empty_bar = bars + F_STAGES;
  uint64_t* rows_ready = bars + 2 * F_STAGES;
  uint64_t* tmem_full = bars + 2 * F_STAGES + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * F_STAGES + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tw = blockIdx.x / args.split, part = blockIdx.x % args.split;
  const int num_kb = (args.K + BK - 1) / BK;
  const int kb0 = min(part * args.chunk, num_kb), steps = min(kb0 + args.chunk, num_kb) - kb0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < F_STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(rows_ready, 128);
    mbar_init(tmem_full, 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, F_TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  float acc[F_BN];                                            // the epilogue warps' sums: one weight row, 16 rows of x
#pragma unroll
  for (int i = 0; i < F_BN; ++i) acc[i] = 0.f;
  const int quarter = warp & 3, n_local = quarter * 32 + lane;

  if (warp == 0) {
    if (lane == 0) {
      tma_prefetch_desc(&map_w);
      for (int i = 0; i < steps; ++i) {
        const int s = i % F_STAGES;
        if (!mbar_wait(&empty_bar[s], ((i / F_STAGES) & 1) ^ 1, abort_flag)) {
          atomicExch(args.status, FSB_ERR_WAIT_TIMEOUT_EMPTY);
          *abort_flag = 1;
          break;
        }
        uint8_t* sa = smem + s * F_STAGE_BYTES;
        mbar_expect_tx(&full_bar[s], F_STAGE_BYTES);
        tma_load_2d(sa, &map_w, &full_bar[s], (kb0 + i) * KB, tw * BM);
        tma_load_2d(sa + BM * KB, &map_sfw, &full_bar[s], (kb0 + i) * 256, tw);
      }
    }
  } else if (warp == 1) {
    bool ok = steps > 0;
    if (ok && !mbar_wait(rows_ready, 0, abort_flag)) {
      if (lane == 0) {
        atomicExch(args.status, FSB_ERR_WAIT_TIMEOUT_FULL);
        *abort_flag = 1;
      }
      ok = false;
    }
    for (int i = 0; i < steps && ok; ++i) {
      const int s = i % F_STAGES;
      if (!mbar_wait(&full_bar[s], (i / F_STAGES) & 1, abort_flag)) {
        if (lane == 0) {
          atomicExch(args.status, FSB_ERR_WAIT_TIMEOUT_FULL);
          *abort_flag = 1;
        }
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t sa = smem_u32(smem + s * F_STAGE_BYTES);
      const uint64_t da = make_smem_desc_sw128(sa, 16, 1024);
      const uint64_t db = make_smem_desc_sw128(smem_u32(rows_q + i * F_BN * KB), 16, 1024);
      const uint32_t sfw = sa + BM * KB, sfx = smem_u32(rows_sf + i * SF_BYTES);
      const uint32_t tsf = tmem_base + F_SF_COL0 + (i & 1) * 16;
      if (elect_one()) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          tmem_cp_32x128b_x4(tsf + 4 * h, make_sf_desc(sfw + 512 * h));
          tmem_cp_32x128b_x4(tsf + 8 + 4 * h, make_sf_desc(sfx + 512 * h));
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_mxf4(tmem_base, da + 2 * k, db + 2 * k, make_idesc_mx4(BM, F_BN, (k & 1) * 2), tsf + 4 * (k >> 1),
                    tsf + 8 + 4 * (k >> 1), (i | k) != 0);
        umma_commit(&empty_bar[s]);
      }
      __syncwarp();
    }
    if (ok) {
      if (elect_one()) umma_commit(tmem_full);
      __syncwarp();
    }
  } else if (steps > 0) {
    // a thread per group of 32 columns of a row; groups past K hold zeros with scale 1 (rows past M are never read)
    const int groups = steps * 8;
    for (int i = threadIdx.x - 64; i < args.M * groups; i += 128) {
      const int r = i / groups, g = i - r * groups, kb = g >> 3, in = g & 7;
      const int col = (kb0 + kb) * BK + in * 32;
      uint4 v[4];
      uint32_t m = 0;
      const bool live = col < args.K;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = live ? load8_any(x + r * ldx + col + 8 * j, vec) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < 4; ++j) m = amax8_bits(v[j], m);
      const uint32_t e = mx4_exponent(m);
      const float inv = mx4_inv(e);
      *reinterpret_cast<uint4*>(rows_q + kb * F_BN * KB + r * KB + ((in ^ (r & 7)) << 4)) =
          make_uint4(quant8_fp4(v[0], inv), quant8_fp4(v[1], inv), quant8_fp4(v[2], inv), quant8_fp4(v[3], inv));
      rows_sf[kb * SF_BYTES + (in >> 2) * 512 + r * 16 + (in & 3)] = live ? static_cast<uint8_t>(e) : 127;
    }
    fence_proxy_async_smem();                                 // written by threads, read by the tensor core
    mbar_arrive(rows_ready);
    if (!mbar_wait_warp(tmem_full, 0, abort_flag)) {
      if (lane == 0) {
        atomicExch(args.status, FSB_ERR_WAIT_TIMEOUT_TMEM_FULL);
        *abort_flag = 1;
      }
    } else {
      tc_fence_after();
      uint32_t v[16];
      tmem_ld_32x16(tmem_base + (static_cast<uint32_t>(quarter * 32) << 16), v);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < F_BN; ++i) acc[i] = __uint_as_float(v[i]);
    }
    tc_fence_before();
  }
  if (warp >= 2) {
#pragma unroll
    for (int i = 0; i < F_BN; ++i) reinterpret_cast<float*>(smem)[i * BM + n_local] = acc[i];   // the first stage is free by now
  }
  store_rows(args, smem, part, 0, args.M, tw * BM);
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    if (*abort_flag) {
      const unsigned long long t0 = clock64();
      while (clock64() - t0 < 2000000ull) {
      }
    }
    tc_fence_after();
    tmem_dealloc(tmem_base, F_TMEM_COLS);
  }
}

// ------------------------------------------------------------------ block-scaled product on SM pairs
// 256 x 256 tiles of a CTA pair, rows t as the M operand. Per CTA and stage: 128 rows of each operand, the scale blocks of its
// own 128 rows of A (two: 1 KB) and of all 256 rows of B (four), which the tensor core of each SM wants in its own TMEM;
// tcgen05.cp on a pair copies them in both CTAs at once. An accumulator of 256 columns and the scales leave no room for a
// second one, so eight warps move a finished tile from TMEM into registers and hand the accumulator back before they store it:
// through shared memory, in boxes that the copy engine writes out (a thread has a row there; its own 16-byte stores, 32 rows an
// instruction, held the next tile up: 8192 x 28672 x 4096 382 us, 318 without any stores).
constexpr int P_BN = 256;
constexpr int P_A = BM * KB, P_B = BM * KB;
constexpr int P_STAGE_BYTES = P_A + P_B + 3 * SF_BYTES;   // 35 KB
constexpr int P_STAGES = 5;
constexpr int P_BOX = 32 * 128;                           // a warp's staging for stores: 32 rows of 128 bytes
constexpr int P_SMEM = P_STAGES * P_STAGE_BYTES + 8 * P_BOX + 1024 + 256;
constexpr int P_THREADS = 64 + 32 * 8;   // warp 0 TMA, warp 1 MMA, warps 2..9 epilogue (two per lane quarter, 128 columns each)
constexpr int P_SF_COL0 = 256, P_SF_SET = 32;   // a stage's scales: 2 x 4 columns of A, 2 x 8 of B

__device__ __forceinline__ void tmem_cp_32x128b_x4_pair(uint32_t taddr, uint64_t sdesc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sdesc) : "memory");
}
__device__ __forceinline__ void umma_mxf4_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t tsfa,
                                               uint32_t tsfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
      ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(tsfa), "r"(tsfb)
      : "memory");
}

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* smem_src, int32_t c0, int32_t c1) {
  uint64_t policy;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group.L2::cache_hint [%0, {%2, %3}], [%1], %4;"
               ::"l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(smem_src)), "r"(c0), "r"(c1), "l"(policy)
               : "memory");
}

// boxes: map_d describes the output (its rows start on 16-byte boundaries); otherwise threads store it.
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(P_THREADS, 1)
gemm_mxfp4_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                       const __grid_constant__ CUtensorMap map_sfa, const __grid_constant__ CUtensorMap map_sfb,
                       const __grid_constant__ CUtensorMap map_d, const int boxes, const Args args) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + P_STAGES * P_STAGE_BYTES + 8 * P_BOX);
  uint64_t* full_bar = bars;                        // [P_STAGES]  used in CTA 0
  uint64_t* empty_bar = bars + P_STAGES;            // [P_STAGES]  one per CTA
  uint64_t* tmem_full = bars + 2 * P_STAGES;        // one per CTA
  uint64_t* tmem_empty = bars + 2 * P_STAGES + 1;   // used in CTA 0: the epilogue warps of both CTAs
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * P_STAGES + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int tiles_m = (args.M + 2 * BM - 1) / (2 * BM), tiles_n = (args.N + P_BN - 1) / P_BN;
  const int num_tiles = tiles_m * tiles_n;
  const int num_kb = (args.K + BK - 1) / BK;
  const int tile0 = static_cast<int>(blockIdx.x >> 1), tile_step = static_cast<int>(gridDim.x >> 1);

  if (threadIdx.x == 0) {
    for (int s = 0; s < P_STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(tmem_full, 1);
    mbar_init(tmem_empty, 16);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) tmem_alloc_pair(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();   // the peer's barriers are initialised before anything is signalled across the pair
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      tma_prefetch_desc(&map_a);
      tma_prefetch_desc(&map_b);
      tma_prefetch_desc(&map_sfa);
      tma_prefetch_desc(&map_sfb);
      wait_for_previous_kernel();
      uint32_t it = 0;
      bool ok = true;
      for (int tile = tile0; tile < num_tiles && ok; tile += tile_step) {
        int tm, tn;
        grouped_tile_coords(tile, tiles_m, tiles_n, tm, tn);
        const int mb = tm * 2 + static_cast<int>(rank);   // 128-row block of A
        const int m0 = mb * BM, n0 = tn * P_BN + static_cast<int>(rank) * BM;
        for (int kb = 0; kb < num_kb; ++kb, ++it) {
          const int s = it % P_STAGES;
          if (!mbar_wait(&empty_bar[s], ((it / P_STAGES) & 1) ^ 1, abort_flag)) {
            atomicExch(args.status, FSB_ERR_WAIT_TIMEOUT_EMPTY);
            *abort_flag = 1;
            ok = false;
            break;
          }
          uint8_t* sa = smem + s * P_STAGE_BYTES;
          uint8_t* sb = sa + P_A;
          uint8_t* ssf = sb + P_B;
          const uint32_t full0 = map_to_cta(smem_u32(&full_bar[s]), 0);
          if (rank == 0) mbar_expect_tx(&full_bar[s], 2 * P_STAGE_BYTES);   // the bytes of both CTAs
          tma_load_2d_pair(sa, &map_a, full0, kb * KB, m0);
          tma_load_2d_pair(sb, &map_b, full0, kb * KB, n0);
          // blocks past the last one read as zeros, like the codes they belong to
          tma_load_2d_pair(ssf, &map_sfa, full0, kb * 256, mb);
          tma_load_2d_pair(ssf + SF_BYTES, &map_sfb, full0, kb * 256, tn * 2);   // two rows of blocks
        }
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {   // one CTA issues for the pair; the whole warp walks the loop
      uint32_t it = 0, local_tile = 0;
      bool ok = true;
      for (int tile = tile0; tile < num_tiles && ok; tile += tile_step, ++local_tile) {
        if (!mbar_wait(tmem_empty, (local_tile & 1) ^ 1, abort_flag)) {
          if (lane == 0) {
            atomicExch(args.status, FSB_ERR_WAIT_TIMEOUT_TMEM_EMPTY);
            *abort_flag = 1;
          }
          break;
        }
        tc_fence_after();
        for (int kb = 0; kb < num_kb; ++kb, ++it) {
          const int s = it % P_STAGES;
          if (!mbar_wait(&full_bar[s], (it / P_STAGES) & 1, abort_flag)) {
            if (lane == 0) {
              atomicExch(args.status, FSB_ERR_WAIT_TIMEOUT_FULL);
              *abort_flag = 1;
            }
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + s * P_STAGE_BYTES);
          const uint64_t da = make_smem_desc_sw128(sa, 16, 1024);
          const uint64_t db = make_smem_desc_sw128(sa + P_A, 16, 1024);
          const uint32_t ssf = sa + P_A + P_B;
          const uint32_t tsfa = tmem_base + P_SF_COL0 + (it & 1) * P_SF_SET, tsfb = tsfa + 8;
          const uint32_t e_own = smem_u32(&empty_bar[s]);
          if (elect_one()) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {   // the two 128-deep halves of the stage
              tmem_cp_32x128b_x4_pair(tsfa + 4 * h, make_sf_desc(ssf + 512 * h));
              tmem_cp_32x128b_x4_pair(tsfb + 8 * h, make_sf_desc(ssf + SF_BYTES + 512 * h));
              tmem_cp_32x128b_x4_pair(tsfb + 8 * h + 4, make_sf_desc(ssf + 2 * SF_BYTES + 512 * h));
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_mxf4_pair(tmem_base, da + 2 * k, db + 2 * k, make_idesc_mx4(2 * BM, P_BN, (k & 1) * 2), tsfa + 4 * (k >> 1),
                             tsfb + 8 * (k >> 1), (kb | k) != 0);
            umma_commit_pair(e_own);
            umma_commit_pair(map_to_cta(e_own, 1));
          }
          __syncwarp();
        }
        if (ok) {
          const uint32_t f_own = smem_u32(tmem_full);
          if (elect_one()) {
            umma_commit_pair(f_own);
            umma_commit_pair(map_to_cta(f_own, 1));
          }
          __syncwarp();
        }
      }
    }
  } else {
    const int quarter = warp & 3;
    const int part = (warp - 2) >> 2;
    const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + part * 128;
    uint8_t* box = smem + P_STAGES * P_STAGE_BYTES + (warp - 2) * P_BOX;
    const uint32_t box_row = smem_u32(box) + lane * 128;
    uint32_t local_tile = 0;
    for (int tile = tile0; tile < num_tiles; tile += tile_step, ++local_tile) {
      int tm, tn;
      grouped_tile_coords(tile, tiles_m, tiles_n, tm, tn);
      const int row = (tm * 2 + static_cast<int>(rank)) * BM + quarter * 32 + lane;
      if (!mbar_wait_warp(tmem_full, local_tile & 1, abort_flag)) {
        if (lane == 0) {
          atomicExch(args.status, FSB_ERR_WAIT_TIMEOUT_TMEM_FULL);
          *abort_flag = 1;
        }
        break;
      }
      tc_fence_after();
      uint32_t v[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld_32x32(t_row + 32 * c, v[c]);
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(map_to_cta(smem_u32(tmem_empty), 0));   // the next tile may start
      if (boxes) {
        // 128 bytes of a row at a time, 16-byte chunk i of row r at chunk i ^ (r % 8): the store's swizzle, and no bank conflicts
        auto put = [&](int i, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(box_row + ((i ^ (lane & 7)) << 4)), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
        };
        auto send = [&](int col) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (row < args.M && col < args.N) tma_store_2d(&map_d, box, col, row);   // lane 0 has the box's first row
            tma_store_commit();
            tma_store_wait_read0();                            // the box may be filled again
          }
          __syncwarp();
        };
        const int col0 = tn * P_BN + part * 128;
        if (args.d_fp32) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
#pragma unroll
            for (int i = 0; i < 8; ++i) put(i, v[c][4 * i], v[c][4 * i + 1], v[c][4 * i + 2], v[c][4 * i + 3]);
            send(col0 + 32 * c);
          }
        } else {
#pragma unroll
          for (int c = 0; c < 4; c += 2) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              uint32_t o[4];
#pragma unroll
              for (int j = 0; j < 4; ++j)
                o[j] = pack_bf16x2(__uint_as_float(v[c + i / 4][i % 4 * 8 + 2 * j]), __uint_as_float(v[c + i / 4][i % 4 * 8 + 2 * j + 1]));
              put(i, o[0], o[1], o[2], o[3]);
            }
            send(col0 + 32 * c);
          }
        }
        continue;
      }
      if (row >= args.M) continue;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int col = tn * P_BN + part * 128 + c * 32;
        const int ncols = min(32, args.N - col);
        if (args.d_fp32) {
          float* dp = static_cast<float*>(args.d) + static_cast<long long>(row) * args.ldd + col;
          if (ncols == 32 && (reinterpret_cast<uintptr_t>(dp) & 15) == 0) {
#pragma unroll
            for (int i = 0; i < 32; i += 4) *reinterpret_cast<uint4*>(dp + i) = make_uint4(v[c][i], v[c][i + 1], v[c][i + 2], v[c][i + 3]);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i < ncols) dp[i] = __uint_as_float(v[c][i]);
          }
        } else {
          __nv_bfloat16* dp = static_cast<__nv_bfloat16*>(args.d) + static_cast<long long>(row) * args.ldd + col;
          if (ncols == 32 && (reinterpret_cast<uintptr_t>(dp) & 15) == 0) {
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
              uint4 o;
              o.x = pack_bf16x2(__uint_as_float(v[c][i]), __uint_as_float(v[c][i + 1]));
              o.y = pack_bf16x2(__uint_as_float(v[c][i + 2]), __uint_as_float(v[c][i + 3]));
              o.z = pack_bf16x2(__uint_as_float(v[c][i + 4]), __uint_as_float(v[c][i + 5]));
              o.w = pack_bf16x2(__uint_as_float(v[c][i + 6]), __uint_as_float(v[c][i + 7]));
              *reinterpret_cast<uint4*>(dp + i) = o;
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i < ncols) dp[i] = __float2bfloat16(__uint_as_float(v[c][i]));
          }
        }
      }
    }
  }

  if (warp >= 2 && lane == 0) tma_store_wait_all();
  __syncwarp();
  // Every loop above is bounded, so all warps of both CTAs arrive here; neither CTA may leave before both are done.
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  if (warp == 1) {
    if (*abort_flag) {
      const unsigned long long t0 = clock64();
      while (clock64() - t0 < 2000000ull) {
      }
    }
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

inline int ok() { return cudaGetLastError() == cudaSuccess ? FSB_OK : FSB_ERR_LAUNCH; }

// codes [rows, K] as bytes, boxes of box_rows rows x 128 bytes
int codes_map(CUtensorMap* map, const void* q, long long rows, int K, long long ld, int box_rows) {
  return fsb_make_tmap_2d(map, q, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, rows, K / 2, ld, box_rows, KB);
}
// blocked scales: one row of n_gb * 128 words per 128 operand rows, boxes of box_rows rows x two blocks
int scales_map(CUtensorMap* map, const void* sf, long long rows, int K, int box_rows) {
  const uint64_t words = static_cast<uint64_t>((K + 127) / 128) * 128;
  return fsb_make_tmap_2d_plain(map, sf, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, (rows + 127) / 128, words, words, box_rows, 256);
}

// Bytes of the blocked scales of an operand [rows, cols]; whether scratch memory can be used and holds what is needed.
long long scale_bytes(long long rows, int cols) { return (rows + 127) / 128 * 128 * ((cols + 127) / 128 * 4); }
bool fits(const void* scratch, long long bytes, long long need) {
  return scratch != nullptr && (reinterpret_cast<uintptr_t>(scratch) & 15) == 0 && bytes >= need;
}

// CTAs along K for `tiles` tiles: as many as there are places for, each with `least` 256-deep steps or more.
int k_split(long long tiles, int num_kb, int least, int places) {
  const int most = min(MAX_SPLIT, max(1, num_kb / least)), split = static_cast<int>(max(1ll, min(static_cast<long long>(most), places / tiles)));
  const int chunk = (num_kb + split - 1) / split;
  return (num_kb + chunk - 1) / chunk;
}

// Launch of a kernel whose clusters are `split` CTAs along x. PDL: it may start while the kernel before it in the stream still
// runs, and waits for that kernel's results itself.
template <typename... P, typename... A>
int launch_split(void (*kernel)(P...), dim3 grid, int smem, int split, bool pdl, cudaStream_t stream, const A&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(NUM_THREADS, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[2] = {};
  cfg.attrs = at;
  if (split > 1) {
    cudaLaunchAttribute& c = at[cfg.numAttrs++];
    c.id = cudaLaunchAttributeClusterDimension;
    c.val.clusterDim.x = split;
    c.val.clusterDim.y = 1;
    c.val.clusterDim.z = 1;
  }
  if (pdl) {
    cudaLaunchAttribute& c = at[cfg.numAttrs++];
    c.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    c.val.programmaticStreamSerializationAllowed = 1;
  }
  const cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, args...);
  const int rc = ok();   // also clears the error of a launch that failed
  return err == cudaSuccess ? rc : static_cast<int>(FSB_ERR_LAUNCH);
}
// The kernel's shared-memory limit raised once per device.
template <typename Kernel>
bool raise_smem(Kernel kernel, bool (&raised)[64], int bytes) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return false;
  if (!raised[dev]) raised[dev] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess;
  return raised[dev];
}

// How the rows are divided where they are few: by their quantisation inside the product, unless a CTA's share of them is more than
// its threads quantise while the weight arrives, or than fits.
constexpr int MOST_SMEM = 227 * 1024;
bool few_rows(Args& a) {
  if (a.M > F_BN) return false;
  const int tiles = (a.N + BM - 1) / BM, num_kb = (a.K + BK - 1) / BK;
  a.split = k_split(tiles, num_kb, 2, 296);
  a.chunk = (num_kb + a.split - 1) / a.split;
  return few_smem(a.chunk) <= MOST_SMEM && a.M * a.chunk * 8 <= FEW_GROUPS;
}
int launch_few(const void* x, const void* bq, const void* sfb, const Args& a, long long ldx, long long ldb, cudaStream_t stream) {
  static bool raised[64] = {false};
  if (!raise_smem(linear_mxfp4_few_kernel, raised, MOST_SMEM)) return FSB_ERR_LAUNCH;
  const int tiles = (a.N + BM - 1) / BM;
  CUtensorMap map_w, map_sfw;
  int rc = codes_map(&map_w, bq, a.N, a.K, ldb, BM);
  if (rc == FSB_OK) rc = scales_map(&map_sfw, sfb, a.N, a.K, 1);
  if (rc != FSB_OK) return rc;
  const int vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && ldx % 8 == 0;
  return launch_split(linear_mxfp4_few_kernel, dim3(tiles * a.split), few_smem(a.chunk), a.split, false, stream, map_w, map_sfw,
                      static_cast<const __nv_bfloat16*>(x), ldx, vec, a);
}

template <int BN>
int launch(const void* aq, const void* sfa, const void* bq, const void* sfb, Args a, long long lda, long long ldb, bool pdl,
           cudaStream_t stream) {
  static bool raised[64] = {false};
  if (!raise_smem(gemm_mxfp4_kernel<BN>, raised, Tile<BN>::SMEM)) return FSB_ERR_LAUNCH;
  CUtensorMap map_w, map_x, map_sfw, map_sfx;
  int rc = codes_map(&map_w, bq, a.N, a.K, ldb, BM);
  if (rc == FSB_OK) rc = codes_map(&map_x, aq, a.M, a.K, lda, BN);
  if (rc == FSB_OK) rc = scales_map(&map_sfw, sfb, a.N, a.K, 1);
  if (rc == FSB_OK) rc = scales_map(&map_sfx, sfa, a.M, a.K, 1);
  if (rc != FSB_OK) return rc;
  const int tiles_w = (a.N + BM - 1) / BM, tiles_x = (a.M + BN - 1) / BN, num_kb = (a.K + BK - 1) / BK;
  if (tiles_x > 65535) return FSB_ERR_TOO_LARGE;
  a.split = k_split(static_cast<long long>(tiles_w) * tiles_x, num_kb, Tile<BN>::LEAST, BN == 128 ? 148 : 296);
  a.chunk = (num_kb + a.split - 1) / a.split;
  return launch_split(gemm_mxfp4_kernel<BN>, dim3(tiles_w * a.split, tiles_x), Tile<BN>::SMEM, a.split, pdl, stream, map_w, map_x,
                      map_sfw, map_sfx, a);
}

// Clusters of the pair kernel that fit the current device at once (-1: unusable).
int resident_pairs() {
  static int pairs[64] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return -1;
  if (pairs[dev] == 0) pairs[dev] = fsb_resident_pairs(gemm_mxfp4_pair_kernel, P_THREADS, P_SMEM);
  return pairs[dev];
}
int launch_pairs(const void* aq, const void* sfa, const void* bq, const void* sfb, const Args& a, long long lda, long long ldb,
                 int pairs, bool pdl, cudaStream_t stream) {
  CUtensorMap map_a, map_b, map_sfa, map_sfb, map_d = {};
  int rc = codes_map(&map_a, aq, a.M, a.K, lda, BM);
  if (rc == FSB_OK) rc = codes_map(&map_b, bq, a.N, a.K, ldb, BM);
  if (rc == FSB_OK) rc = scales_map(&map_sfa, sfa, a.M, a.K, 1);
  if (rc == FSB_OK) rc = scales_map(&map_sfb, sfb, a.N, a.K, 2);
  if (rc != FSB_OK) return rc;
  const int size = a.d_fp32 ? 4 : 2;
  const int boxes = (reinterpret_cast<uintptr_t>(a.d) & 15) == 0 && a.ldd * size % 16 == 0;
  if (boxes) rc = fsb_make_tmap_2d(&map_d, a.d, a.d_fp32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, size,
                                   a.M, a.N, a.ldd, 32, 128 / size);
  if (rc != FSB_OK) return rc;
  const int tiles = ((a.M + 2 * BM - 1) / (2 * BM)) * ((a.N + P_BN - 1) / P_BN);
  cudaLaunchConfig_t cfg{};                                  // the cluster's size is the kernel's own
  cfg.gridDim = dim3(2 * (tiles < pairs ? tiles : pairs));
  cfg.blockDim = dim3(P_THREADS, 1, 1);
  cfg.dynamicSmemBytes = P_SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = pdl ? 1 : 0;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, gemm_mxfp4_pair_kernel, map_a, map_b, map_sfa, map_sfb, map_d, boxes, a);
  rc = ok();
  return err == cudaSuccess ? rc : static_cast<int>(FSB_ERR_LAUNCH);
}
// pdl: the kernel before this one in the stream is the quantiser of a.
int product(const void* aq, const void* sfa, const void* bq, const void* sfb, const Args& a, long long lda, long long ldb, bool pdl,
            cudaStream_t stream) {
  if (a.M <= 16) return launch<16>(aq, sfa, bq, sfb, a, lda, ldb, pdl, stream);
  if (a.M <= 32) return launch<32>(aq, sfa, bq, sfb, a, lda, ldb, pdl, stream);
  if (a.M <= 64) return launch<64>(aq, sfa, bq, sfb, a, lda, ldb, pdl, stream);
  // More 128 x 128 tiles than SMs: pairs of them, on SM pairs. One SM a tile against pairs, with the quantiser: 256 x 6144 x 4096
  // (96 tiles) 12.8 / 15.3 us, 512 x 4096 x 4096 (128) 12.8 / 14.2, 512 x 6144 x 4096 (192) 22.2 / 15.9, 128 x 28672 x 4096 (224)
  // 25.2 / 23.0, 777 x 5000 x 2080 (280) 20.6 / 18.0, 1024 x 4096 x 4096 (256) 23.1 / 15.4.
  const long long tiles = static_cast<long long>((a.M + BM - 1) / BM) * ((a.N + BM - 1) / BM);
  if (tiles > 148) {
    const int pairs = resident_pairs();
    if (pairs > 0) return launch_pairs(aq, sfa, bq, sfb, a, lda, ldb, pairs, pdl, stream);
  }
  return launch<128>(aq, sfa, bq, sfb, a, lda, ldb, pdl, stream);
}
}  // namespace

// x: bf16 [T, K], K % 32 == 0, row stride ldx; q: [T, K / 2] bytes; scales: pad128(T) * pad4(K / 32) bytes, all written.
FSB_API int fsb_mx4_quant_act(const void* x, void* q, void* scales, long long T, int K, long long ldx, cudaStream_t stream) {
  if (K <= 0 || K % 32 != 0 || T < 0 || (reinterpret_cast<uintptr_t>(q) & 7) != 0 || (reinterpret_cast<uintptr_t>(scales) & 3) != 0)
    return FSB_ERR_BAD_ARG;
  if (T == 0) return FSB_OK;
  const int n_gb = (K + 127) / 128;
  const long long share = (T + 127) / 128 * 128 * (n_gb * 8) / UNITS, blocks = (share + 255) / 256;
  if (blocks > 0x7fffffffll) return FSB_ERR_TOO_LARGE;
  const int vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && ldx % 8 == 0;
  auto kernel = share * UNITS < (1ll << 31) ? mx4_quant_act_kernel<unsigned> : mx4_quant_act_kernel<long long>;
  kernel<<<static_cast<unsigned>(blocks), 256, 0, stream>>>(static_cast<const __nv_bfloat16*>(x), static_cast<uint8_t*>(q),
                                                            static_cast<uint8_t*>(scales), T, K, ldx, n_gb, vec);
  return ok();
}

// w: bf16 [rows, cols], cols % 32 == 0; q: [rows, cols / 2] bytes; tile_exp: [ceil(rows / 32), cols / 32] bytes. fwd / dgrad:
// blocked scales of the operands [rows, cols] and [cols, rows], padding included (both or neither).
FSB_API int fsb_mx4_quant_weight(const void* w, void* q, void* tile_exp, void* fwd, void* dgrad, int rows, int cols, long long ldw,
                                 cudaStream_t stream) {
  if (rows < 0 || cols <= 0 || cols % 32 != 0 || (fwd == nullptr) != (dgrad == nullptr) ||
      ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(fwd) | reinterpret_cast<uintptr_t>(dgrad)) & 3) != 0)
    return FSB_ERR_BAD_ARG;
  if (rows == 0) return FSB_OK;
  const int col_blocks = (cols + 127) / 128;
  const long long row_blocks = (static_cast<long long>(rows) + 127) / 128;
  if (row_blocks > 65535) return FSB_ERR_TOO_LARGE;
  const int vec = (reinterpret_cast<uintptr_t>(w) & 15) == 0 && ldw % 8 == 0;
  const bool wide = col_blocks * row_blocks >= 148 * 4;      // the blocks of four tiles a warp fill the SMs
  auto kernel = wide ? mx4_quant_weight_kernel<4> : mx4_quant_weight_kernel<1>;
  kernel<<<dim3(wide ? col_blocks : 4 * col_blocks, static_cast<unsigned>(row_blocks)), 128, 0, stream>>>(
      static_cast<const __nv_bfloat16*>(w), static_cast<uint8_t*>(q), static_cast<uint8_t*>(tile_exp), static_cast<uint8_t*>(fwd),
      static_cast<uint8_t*>(dgrad), rows, cols, ldw, vec);
  return ok();
}

// q: [T, K / 2] codes with row stride ldq bytes; scales: blocked (not read for kind 0); out: [T, K] contiguous, e4m3 without
// scales (kind 0), bf16 (1) or fp32 (2).
FSB_API int fsb_mx4_expand(const void* q, const void* scales, void* out, long long T, int K, long long ldq, int kind,
                           cudaStream_t stream) {
  if (K <= 0 || K % 32 != 0 || T < 0 || ldq % 4 != 0 || (reinterpret_cast<uintptr_t>(q) & 3) != 0 || kind < 0 || kind > 2)
    return FSB_ERR_BAD_ARG;
  if (T == 0) return FSB_OK;
  const long long units = T * (K / (kind == 0 ? 16 : 8)), blocks = ((units + EXPAND_UNITS - 1) / EXPAND_UNITS + 255) / 256;
  if (blocks > 0x7fffffffll) return FSB_ERR_TOO_LARGE;
  auto run = [&](auto kernel) {
    kernel<<<static_cast<unsigned>(blocks), 256, 0, stream>>>(static_cast<const uint8_t*>(q), static_cast<const uint8_t*>(scales),
                                                              out, T, K, ldq, (K + 127) / 128);
    return ok();
  };
  const bool small = units < (1ll << 31);
  if (kind == 0) return small ? run(mx4_expand_kernel<0, unsigned>) : run(mx4_expand_kernel<0, long long>);
  if (kind == 1) return small ? run(mx4_expand_kernel<1, unsigned>) : run(mx4_expand_kernel<1, long long>);
  return small ? run(mx4_expand_kernel<2, unsigned>) : run(mx4_expand_kernel<2, long long>);
}

// d[M, N] = A B^T for codes aq [M, K / 2] and bq [N, K / 2] (row strides lda, ldb bytes, multiples of 16) with blocked scales
// sfa, sfb; K % 32 == 0.
FSB_API int fsb_gemm_mxfp4(const void* aq, const void* sfa, const void* bq, const void* sfb, void* d, int M, int N, int K,
                           long long lda, long long ldb, long long ldd, int d_fp32, int* status, cudaStream_t stream) {
  if (M <= 0 || N <= 0 || K <= 0 || K % 32 != 0 || lda % 16 != 0 || ldb % 16 != 0) return FSB_ERR_BAD_ARG;
  if ((reinterpret_cast<uintptr_t>(sfa) | reinterpret_cast<uintptr_t>(sfb) | reinterpret_cast<uintptr_t>(aq) |
       reinterpret_cast<uintptr_t>(bq)) & 15)
    return FSB_ERR_BAD_ARG;
  const Args a{M, N, K, 1, 0, d, ldd, d_fp32, status};
  return product(aq, sfa, bq, sfb, a, lda, ldb, false, stream);
}

// d[M, N] = Q(x) B^T for bf16 x [M, K] with row stride ldx: the quantiser and the product, in one launch for up to 16 rows of which
// a CTA has up to FEW_GROUPS groups (16 x 6144 x 4096, not 16 x 28672 x 4096, whose tiles leave no CTAs to divide K).
// scratch: M * (K / 2) + pad128(M) * pad4(K / 32) bytes or more, on a 16-byte boundary; not used where fsb_mxfp4_linear_few says 1, which is
// where the call is one launch.
FSB_API int fsb_mxfp4_linear_few(int M, int N, int K) {
  Args a{M, N, K};
  return M > 0 && N > 0 && K > 0 && few_rows(a);
}
FSB_API int fsb_mxfp4_linear(const void* x, long long ldx, const void* bq, long long ldb, const void* sfb, void* d, long long ldd,
                             void* scratch, long long scratch_bytes, int M, int N, int K, int* status, cudaStream_t stream) {
  if (M <= 0 || N <= 0 || K <= 0 || K % 32 != 0 || ldb % 16 != 0) return FSB_ERR_BAD_ARG;
  if ((reinterpret_cast<uintptr_t>(sfb) | reinterpret_cast<uintptr_t>(bq)) & 15) return FSB_ERR_BAD_ARG;
  Args a{M, N, K, 1, 0, d, ldd, 0, status};
  if (few_rows(a)) return launch_few(x, bq, sfb, a, ldx, ldb, stream);
  a.split = 1;
  const long long codes = static_cast<long long>(M) * (K / 2);      // K / 2 is a multiple of 16
  if (!fits(scratch, scratch_bytes, codes + scale_bytes(M, K))) return FSB_ERR_BAD_ARG;
  uint8_t* q = static_cast<uint8_t*>(scratch);
  uint8_t* sf = q + codes;
  const int rc = fsb_mx4_quant_act(x, q, sf, M, K, ldx, stream);
  return rc == FSB_OK ? product(q, sf, bq, sfb, a, K / 2, ldb, true, stream) : rc;
}

// dx[T, K] = Q8(dy) W for dy [T, N] bf16 (row stride lddy) and the codes wq [N, K / 2] with the scales of the
// operand [K, N]; N and K multiples of 128. dy in MXFP8 groups along N, the codes as e4m3 with their own scales.
// scratch: T * N + N * K + pad128(T) * (N / 32) bytes or more, on a 16-byte boundary. One entry for the three launches: the time of a
// small backward pass is the host's (T = 500, N = K = 2048: forward and both gradients 167.5 us with an entry each, 145.9 so).
FSB_API int fsb_mxfp4_linear_dx(const void* dy, long long lddy, const void* wq, long long ldw, const void* dgrad_scale, void* dx,
                                void* scratch, long long scratch_bytes, int T, int N, int K, int* status, cudaStream_t stream) {
  if (T <= 0 || N <= 0 || K <= 0 || N % 128 != 0 || K % 128 != 0) return FSB_ERR_BAD_ARG;
  if (!fits(scratch, scratch_bytes, (static_cast<long long>(T) + K) * N + scale_bytes(T, N))) return FSB_ERR_BAD_ARG;
  uint8_t* q = static_cast<uint8_t*>(scratch);
  uint8_t* w = q + static_cast<long long>(T) * N;
  uint8_t* sf = w + static_cast<long long>(N) * K;             // rows past T stay unset: they scale outputs that are not stored
  int rc = fsb_mx_quant_act(dy, q, sf, T, N, lddy, N, stream);
  if (rc == FSB_OK) rc = fsb_mx4_expand(wq, nullptr, w, N, K, ldw, 0, stream);
  if (rc == FSB_OK) rc = fsb_gemm_mxfp8(q, sf, w, dgrad_scale, dx, T, K, N, N, K, K, 0, 1, 0, status, stream);
  return rc;
}

// dw[N, K] = dy^T x in MXFP8 groups of 32 rows, for dy [T, N] and x [T, K] bf16; T, N and K multiples of 128; bf16 or fp32 dw.
// scratch: T * (N + K) + (T / 32) * (N + K) bytes or more, on a 16-byte boundary.
FSB_API int fsb_mxfp4_linear_dw(const void* dy, long long lddy, const void* x, long long ldx, void* dw, int dw_fp32, void* scratch,
                                long long scratch_bytes, int T, int N, int K, int* status, cudaStream_t stream) {
  if (T <= 0 || N <= 0 || K <= 0 || T % 128 != 0 || N % 128 != 0 || K % 128 != 0) return FSB_ERR_BAD_ARG;
  if (!fits(scratch, scratch_bytes, (static_cast<long long>(T) + T / 32) * (static_cast<long long>(N) + K))) return FSB_ERR_BAD_ARG;
  uint8_t* a = static_cast<uint8_t*>(scratch);
  uint8_t* b = a + static_cast<long long>(T) * N;
  uint8_t* sa = b + static_cast<long long>(T) * K;
  uint8_t* sb = sa + static_cast<long long>(T / 32) * N;
  int rc = fsb_mx_quant_rows(dy, a, sa, T, N, lddy, N, stream);
  if (rc == FSB_OK) rc = fsb_mx_quant_rows(x, b, sb, T, K, ldx, K, stream);
  if (rc == FSB_OK) rc = fsb_gemm_mxfp8(a, sa, b, sb, dw, N, K, T, N, K, K, 1, 1, dw_fp32, status, stream);
  return rc;
}
