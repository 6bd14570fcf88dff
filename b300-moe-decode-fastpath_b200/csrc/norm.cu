// Residual addition and root-mean-square norm of token rows, the step in front of the layer:
//   s = x + r,   r' = round(s),   y = s * w / sqrt(mean(s^2) + eps)
// with y rounded to BF16, or to E4M3 with one FP32 scale per row by the rule of
// fp8_quantize_rows_kernel (scale = max|y| / 448, 1 for a row of zeros).  s is held in FP32 and
// is what is normalised: r' is a rounded copy of it.  No counterpart in the reference.
//
// A row is read once and stays in registers between the sum of its squares, the largest |y|
// and the stores (of the longest rows up to 28 bytes a thread do not), so the kernel moves the
// bytes of its operands: x, r, r', y.  Many rows are bound by HBM: 8192 x 4096 in 40.5 us
// (6.63 TB/s, 1.01 of the measured copy rate), 4096 x 7168 with FP32 residual and weight 53.4 us
// (1.00); with E4M3 result 38.3 us (0.93: each element is rounded to a code twice) and 55.2 us
// (0.89); 4099 x 2880 E4M3 in 16.6 us (0.76: the same, and the start and end of a short kernel).
// One row is bound by the latency of one load, one barrier and one store: 1.8 us for 4096 columns.
#include <cuda_fp8.h>

#include <type_traits>

#include "common.cuh"

namespace b200moe {

namespace {

constexpr float kNormE4m3Max = 448.0f;
constexpr float kNormBracket = 1.0f / (1 << 21);
constexpr float kNormLeastScale = 1.17549435e-38f;  // 2^-126, the smallest normal number
// Threads of a row: one for each vector up to 256, then two or four vectors each, whatever the
// number of rows, so that a row's result depends on that row alone.  More threads keep fewer rows
// of an SM apart in time (512: 8192 x 4096 E4M3 47.3 us against 38.3 us, 4099 x 2880 19.2 against
// 16.6 us, though 4096 x 7168 with FP32 operands 52.6 against 55.1 us), and bring nothing where
// rows are few (one for each vector up to 1024: 296 x 7168 4.2 us against 3.5 us, 1 x 16384 4.0
// against 3.4 us, 64 x 2880 E4M3 2.5 against 2.65 us).
constexpr int kNormThreads = 256;

// eight consecutive elements, as they lie in memory; 16-byte accesses
template <typename T>
struct Raw8 {
  uint4 q[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i) q[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 4) {
      const uint4& v = q[i / 4];
      return __uint_as_float(i % 4 == 0 ? v.x : i % 4 == 1 ? v.y : i % 4 == 2 ? v.z : v.w);
    } else {
      const uint32_t w = i / 2 == 0 ? q[0].x : i / 2 == 1 ? q[0].y : i / 2 == 2 ? q[0].z : q[0].w;
      return __uint_as_float(i % 2 ? w & 0xFFFF0000u : w << 16);
    }
  }
};
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
  uint32_t words[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    words[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(words[0], words[1], words[2], words[3]);
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

struct NormNone { uint16_t unused; };  // no residual

// Sum and, with MAX, maximum over the threads of one row: blockDim.x threads, whole warps, rows in
// threadIdx.y.  `slots` has one pair per warp of the block.
template <bool MAX>
__device__ __forceinline__ void row_reduce(float& sum, float& most, float2* slots) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (MAX) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
  }
  const int warps = blockDim.x >> 5;
  if (warps == 1) return;
  float2* mine = slots + threadIdx.y * warps;
  if ((threadIdx.x & 31) == 0) mine[threadIdx.x >> 5] = make_float2(sum, most);
  __syncthreads();
  sum = mine[0].x;
  most = mine[0].y;
  for (int i = 1; i < warps; ++i) {
    sum += mine[i].x;
    if (MAX) most = fmaxf(most, mine[i].y);
  }
}

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
// (Not inlined: inside the unrolled loops its registers cost the blocks an SM holds, 36.7 us
// instead of 34.2 us for 4096 x 7168.)
__device__ __noinline__ uint32_t divided_codes(float a, float b, float c, float d, float scale) {
  return e4m3x4(__fdiv_rn(a, scale), __fdiv_rn(b, scale), __fdiv_rn(c, scale), __fdiv_rn(d, scale));
}
// The codes of y / scale as fp8_quantize_rows_kernel defines them, by IEEE division.  A product
// with the reciprocal differs from the quotient by at most 3 * 2^-24 of it, so the quotient lies
// between products with a reciprocal that is 2^-21 smaller and one that is 2^-21 larger; where
// both round to the same codes, those are the quotient's, as rounding keeps the order.  Only the
// others, one group of four in some 20,000, are divided (8192 x 4096: 38.3 us, every element
// divided 42.7 us, products alone 36.4 us with a code beside a border off by one now and then).
__device__ __forceinline__ uint32_t quotient_codes(const float (&y)[4], float scale, float below,
                                                   float above) {
  const uint32_t lo = e4m3x4(y[0] * below, y[1] * below, y[2] * below, y[3] * below);
  const uint32_t hi = e4m3x4(y[0] * above, y[1] * above, y[2] * above, y[3] * above);
  return lo == hi ? lo : divided_codes(y[0], y[1], y[2], y[3], scale);
}

// THREADS: most threads of a block, which limits the registers of a thread to 65536 / THREADS.
// No operand is __restrict__: that would promise that it is read-only from the kernel's start, and a
// dependent launch starts while the kernel in front may still be storing it (a weight too: an
// earlier norm's row, a copy of new parameters).
template <typename R, typename W, bool FP8, int VECS, int THREADS = 1024>
__global__ void __launch_bounds__(THREADS)
add_rms_norm_kernel(const __nv_bfloat16* x, const R* residual, const W* weight,
                    long long rows, int hidden, float eps, __nv_bfloat16* out, uint8_t* codes,
                    float* scale_out, R* residual_out) {
  __shared__ float2 slots[32];
  // Four vectors of a thread with a residual and an FP32 operand do not fit 64 registers when the
  // weight waits in them as well: it is loaded vector by vector (FP32 residual and weight,
  // 2048 x 32768: 139.6 us against 191 us with what was spilled; E4M3 with BF16 residual and FP32
  // weight, 4096 x 7168: 36.0 against 38.2 us).
  constexpr bool kLateWeight = VECS == 4 && THREADS == 1024 && !std::is_same<R, NormNone>::value &&
                               (sizeof(R) == 4 || sizeof(W) == 4);
  const long long row = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  const bool live = row < rows;  // the last block's surplus rows only keep the barrier
  const size_t base = live ? (size_t)row * hidden : 0;

  pdl_launch_dependents();
  pdl_wait();
  // everything that a row needs is on its way before anything is waited for
  Raw8<__nv_bfloat16> rx[VECS];
  Raw8<R> rr[VECS];
  Raw8<W> rw[VECS];
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int c = (threadIdx.x + i * blockDim.x) * 8;
    if (live && c < hidden) {
      rx[i].load(x + base + c);
      if constexpr (!std::is_same<R, NormNone>::value) rr[i].load(residual + base + c);
      if (!kLateWeight) rw[i].load(weight + c);
    }
  }
  // y = factor * t with t = s w and one factor per row, so that the largest |y| is known as soon
  // as the largest |t|: both reductions share a barrier
  float t[VECS][8];
  float sum = 0.0f, most = 0.0f;
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int c = (threadIdx.x + i * blockDim.x) * 8;
    if (!(live && c < hidden)) continue;
    if (kLateWeight) rw[i].load(weight + c);
    float s[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      s[j] = rx[i].get(j);
      if constexpr (!std::is_same<R, NormNone>::value) s[j] += rr[i].get(j);
      sum = fmaf(s[j], s[j], sum);
      t[i][j] = s[j] * rw[i].get(j);
      if (FP8) most = fmaxf(most, fabsf(t[i][j]));
    }
    if constexpr (!std::is_same<R, NormNone>::value) store8(residual_out + base + c, s);
  }
  row_reduce<FP8>(sum, most, slots);
  const float factor = rsqrtf(sum / (float)hidden + eps);

  if constexpr (FP8) {
    const float largest = most * factor;
    const float scale = largest > 0.0f ? __fdiv_rn(largest, kNormE4m3Max) : 1.0f;
    if (live && threadIdx.x == 0) scale_out[row] = scale;
    // Below 2^-126 the reciprocal may be infinite: with 0 as the lower bound only groups of four
    // that round to zero whatever the quotients are go undivided.
    const float inverse = __frcp_rn(scale);
    const float below = scale >= kNormLeastScale ? inverse * (1.0f - kNormBracket) : 0.0f;
    const float above = inverse * (1.0f + kNormBracket);
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int c = (threadIdx.x + i * blockDim.x) * 8;
      if (!(live && c < hidden)) continue;
      uint32_t packed[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float y[4] = {t[i][4 * j] * factor, t[i][4 * j + 1] * factor,
                            t[i][4 * j + 2] * factor, t[i][4 * j + 3] * factor};
        packed[j] = quotient_codes(y, scale, below, above);
      }
      *reinterpret_cast<uint2*>(codes + base + c) = make_uint2(packed[0], packed[1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int c = (threadIdx.x + i * blockDim.x) * 8;
      if (!(live && c < hidden)) continue;
#pragma unroll
      for (int j = 0; j < 8; ++j) t[i][j] *= factor;
      store8(out + base + c, t[i]);
    }
  }
}

template <typename R, typename W, bool FP8>
cudaError_t launch_norm(const void* x, const void* residual, const void* weight, long long rows,
                        int hidden, float eps, void* out, uint8_t* codes, float* scale,
                        void* residual_out, cudaStream_t stream) {
  const int vecs = hidden / 8;
  int per = 1;  // vectors of a thread
  while (per < 4 && (vecs + per - 1) / per > kNormThreads) per *= 2;
  int threads = ((vecs + per - 1) / per + 31) / 32 * 32;
  int together = 1;  // rows of a block
  while (threads * together * 2 <= 256 && together < rows) together *= 2;
  const dim3 block(threads, together);
  const dim3 grid((unsigned)((rows + together - 1) / together));
  auto run = [&](auto kernel) {
    // The launch overlaps the end of the kernel in front, for which the kernel waits before it
    // reads anything (1 x 4096: 2.05 -> 1.8 us, 4099 x 2880 16.4 -> 15.8 us, 8192 x 4096 E4M3 38.9
    // -> 38.3 us back to back; 296 x 4096 2.9 -> 3.1 us).
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = grid;
    config.blockDim = block;
    config.stream = stream;
    config.attrs = &attr;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, static_cast<const __nv_bfloat16*>(x),
                              static_cast<const R*>(residual), static_cast<const W*>(weight), rows,
                              hidden, eps, static_cast<__nv_bfloat16*>(out), codes, scale,
                              static_cast<R*>(residual_out));
  };
  if (per == 1) return run(add_rms_norm_kernel<R, W, FP8, 1>);
  if (per == 2) return run(add_rms_norm_kernel<R, W, FP8, 2>);
  // Four vectors with an FP32 residual: blocks of up to 512 threads (H <= 16384) may have 73 to
  // 102 registers a thread, with everything on its way at once (4096 x 7168, FP32 weight: 53.4 us
  // against 57.5 us with the weight loaded late and 74.4 us with spills).
  if constexpr (sizeof(R) == 4)
    if (threads <= 512) return run(add_rms_norm_kernel<R, W, FP8, 4, 512>);
  return run(add_rms_norm_kernel<R, W, FP8, 4>);
}

template <typename R, typename W>
cudaError_t launch_norm_out(const void* x, const void* residual, const void* weight,
                            long long rows, int hidden, float eps, void* out, uint8_t* codes,
                            float* scale, void* residual_out, cudaStream_t stream) {
  return codes ? launch_norm<R, W, true>(x, residual, weight, rows, hidden, eps, out, codes,
                                         scale, residual_out, stream)
               : launch_norm<R, W, false>(x, residual, weight, rows, hidden, eps, out, codes,
                                          scale, residual_out, stream);
}

template <typename R>
cudaError_t launch_norm_weight(const void* x, const void* residual, const void* weight,
                               bool weight_f32, long long rows, int hidden, float eps, void* out,
                               uint8_t* codes, float* scale, void* residual_out,
                               cudaStream_t stream) {
  return weight_f32 ? launch_norm_out<R, float>(x, residual, weight, rows, hidden, eps, out,
                                                codes, scale, residual_out, stream)
                    : launch_norm_out<R, __nv_bfloat16>(x, residual, weight, rows, hidden, eps,
                                                        out, codes, scale, residual_out, stream);
}

}  // namespace

cudaError_t launch_add_rms_norm(const void* x, const void* residual, bool residual_f32,
                                const void* weight, bool weight_f32, long long rows, int hidden,
                                float eps, void* out, uint8_t* codes, float* scale,
                                void* residual_out, cudaStream_t stream) {
  if (!residual)
    return launch_norm_weight<NormNone>(x, nullptr, weight, weight_f32, rows, hidden, eps, out,
                                        codes, scale, nullptr, stream);
  if (residual_f32)
    return launch_norm_weight<float>(x, residual, weight, weight_f32, rows, hidden, eps, out,
                                     codes, scale, residual_out, stream);
  return launch_norm_weight<__nv_bfloat16>(x, residual, weight, weight_f32, rows, hidden, eps,
                                           out, codes, scale, residual_out, stream);
}

}  // namespace b200moe
