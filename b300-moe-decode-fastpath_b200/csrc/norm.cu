// Residual addition and root-mean-square norm of token rows, the step in front of the layer:
//   s = x + r,   r' = round(s),   y = s * w / sqrt(mean(s^2) + eps)
// with y rounded to BF16, or to E4M3 with one FP32 scale per row by the rule of
// fp8_quantize_rows_kernel (scale = max|y| / 448, 1 for a row of zeros).  s is held in FP32 and
// is what is normalised: r' is a rounded copy of it.  No counterpart in the reference.
//
// A row is read once and stays in registers between the sum of its squares, the largest |y|
// and the stores, so the kernel moves exactly the bytes of its operands: x, r, r', y.
#include <cuda_fp8.h>

#include <type_traits>

#include "common.cuh"

namespace b200moe {

namespace {

constexpr float kNormE4m3Max = 448.0f;

// eight consecutive elements as FP32; 16-byte accesses
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]);
template <>
__device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 q = *reinterpret_cast<const uint4*>(p);
  const uint32_t words[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(words[i] << 16);
    v[2 * i + 1] = __uint_as_float(words[i] & 0xFFFF0000u);
  }
}
template <>
__device__ __forceinline__ void load8<float>(const float* p, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0];
  const float4 b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
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

struct NormNone {};  // no residual

// Sum (or maximum) over the threads of one row: blockDim.x threads, whole warps, rows in
// threadIdx.y.  `slots` has one float per warp of the block.
template <bool MAX>
__device__ __forceinline__ float row_reduce(float v, float* slots) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    const float o = __shfl_xor_sync(0xffffffffu, v, d);
    v = MAX ? fmaxf(v, o) : v + o;
  }
  const int warps = blockDim.x >> 5;
  if (warps == 1) return v;
  float* mine = slots + threadIdx.y * warps;
  if ((threadIdx.x & 31) == 0) mine[threadIdx.x >> 5] = v;
  __syncthreads();
  v = mine[0];
  for (int i = 1; i < warps; ++i) v = MAX ? fmaxf(v, mine[i]) : v + mine[i];
  return v;
}

template <typename R, typename W, bool FP8, int VECS>
__global__ void __launch_bounds__(1024)
add_rms_norm_kernel(const __nv_bfloat16* x, const R* residual, const W* __restrict__ weight,
                    long long rows, int hidden, float eps, __nv_bfloat16* out, uint8_t* codes,
                    float* scale_out, R* residual_out) {
  __shared__ float s_sum[32], s_max[32];
  const long long row = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  const bool live = row < rows;  // the last block's surplus rows only keep the barriers
  const size_t base = live ? (size_t)row * hidden : 0;

  float s[VECS][8];
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int c = (threadIdx.x + i * blockDim.x) * 8;
    if (live && c < hidden) {
      load8<__nv_bfloat16>(x + base + c, s[i]);
      if constexpr (!std::is_same<R, NormNone>::value) {
        float r[8];
        load8<R>(residual + base + c, r);
#pragma unroll
        for (int j = 0; j < 8; ++j) s[i][j] += r[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) s[i][j] = 0.0f;
    }
  }
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    if constexpr (!std::is_same<R, NormNone>::value) {
      const int c = (threadIdx.x + i * blockDim.x) * 8;
      if (live && c < hidden) store8(residual_out + base + c, s[i]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) sum = fmaf(s[i][j], s[i][j], sum);
  }
  sum = row_reduce<false>(sum, s_sum);
  const float factor = rsqrtf(sum / (float)hidden + eps);

  float largest = 0.0f;
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int c = (threadIdx.x + i * blockDim.x) * 8;
    if (live && c < hidden) {
      float w[8];
      load8<W>(weight + c, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        s[i][j] = s[i][j] * factor * w[j];
        if (FP8) largest = fmaxf(largest, fabsf(s[i][j]));
      }
      if (!FP8) store8(out + base + c, s[i]);
    }
  }
  if constexpr (FP8) {
    largest = row_reduce<true>(largest, s_max);
    const float scale = largest > 0.0f ? __fdiv_rn(largest, kNormE4m3Max) : 1.0f;
    if (live && threadIdx.x == 0) scale_out[row] = scale;
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int c = (threadIdx.x + i * blockDim.x) * 8;
      if (live && c < hidden) {
        uint32_t packed[2] = {0u, 0u};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t b = __nv_cvt_float_to_fp8(__fdiv_rn(s[i][j], scale), __NV_SATFINITE,
                                                   __NV_E4M3);
          packed[j / 4] |= b << (8 * (j % 4));
        }
        *reinterpret_cast<uint2*>(codes + base + c) = make_uint2(packed[0], packed[1]);
      }
    }
  }
}

template <typename R, typename W, bool FP8>
cudaError_t launch_norm(const void* x, const void* residual, const void* weight, long long rows,
                        int hidden, float eps, void* out, uint8_t* codes, float* scale,
                        void* residual_out, cudaStream_t stream) {
  const int vecs = hidden / 8;
  int per = 1;  // vectors of a thread
  while (per < 4 && (vecs + per - 1) / per > 256) per *= 2;
  int threads = ((vecs + per - 1) / per + 31) / 32 * 32;
  int together = 1;  // rows of a block
  while (threads * together * 2 <= 256 && together < rows) together *= 2;
  const dim3 block(threads, together);
  const dim3 grid((unsigned)((rows + together - 1) / together));
  auto run = [&](auto kernel) {
    kernel<<<grid, block, 0, stream>>>(
        static_cast<const __nv_bfloat16*>(x), static_cast<const R*>(residual),
        static_cast<const W*>(weight), rows, hidden, eps, static_cast<__nv_bfloat16*>(out), codes,
        scale, static_cast<R*>(residual_out));
    return cudaGetLastError();
  };
  if (per == 1) return run(add_rms_norm_kernel<R, W, FP8, 1>);
  if (per == 2) return run(add_rms_norm_kernel<R, W, FP8, 2>);
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
