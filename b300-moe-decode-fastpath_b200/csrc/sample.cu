// Sampling of one token per row of logits, from given random numbers.  No counterpart in the
// reference.  With m the largest logit of the row and w_i = exp((x_i - m) / temperature):
//   order    tokens by descending logit, equal ones by ascending index
//   min-p    drops tokens with w_i < min_p
//   top-k    keeps the first k of the order
//   top-p    keeps of those the shortest run of the order whose w add up to top_p of their sum
//   draw     the first token i, in index order, with (sum of kept w up to i) > u * (sum of kept w)
// A temperature that is not above zero takes the first token of the order.  NaN logits count as
// -inf, tokens at -inf are never drawn; a row of nothing else gives -1.
//
// No sorting.  What is kept is a prefix of the order, so it is described by its last element: a
// threshold on the logit and the index of the last token kept among those equal to it.  The
// threshold is found by selection: a histogram over 2048 bins linear in m - x (for top-k of
// counts, for top-p of weights) finds the bin where the wanted sum is crossed, then three
// histograms over the digits (11, 11 and 10 bits) of the logit's ordered bit pattern find the
// value inside that bin.  A row is read from memory once and stays in the shared memory of a
// cluster of up to eight blocks, which exchange histograms and sums as distributed shared
// memory.
//
// Exact sums.  With a large vocabulary the borders between tokens lie closer together than FP32
// sums resolve, and sums in another order would move them.  The weights are therefore integers,
// w_i * 2^45 rounded to nearest: their sums are exact in 64 bits for up to 2^18 tokens, do not
// depend on the order in which threads add them, and an atomic of integers leaves no trace of
// who came first.  The exponential behind them is computed in FP64 to about 2^-52: reduction to
// 2^(k/64) * 2^r with a table of 64 powers (Tang's table-driven scheme) and the Taylor
// polynomial of degree 5 on |r| <= 2^-7.
#include <cooperative_groups.h>

#include "common.cuh"

namespace b200moe {

namespace {

namespace cg = cooperative_groups;
typedef unsigned long long u64;

constexpr int kSampleThreads = 512;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kBins = 2048;
constexpr int kWeightBits = 45;
constexpr int kMaxCluster = 8;
constexpr uint32_t kMinusInfKey = 0xFF800000u;  // descending_key(-inf)

struct SampleParams {
  const void* logits;
  long long row_stride;
  int vocab, slice;             // slice: tokens of one block
  const float* uniforms;
  const float* temperature;     // per row, or nullptr: the value
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_v, top_p_v, min_p_v;
  int top_k_v;
  int64_t* ids;
  float* logprobs;
};

// ascending order of this key = descending order of the logit (no NaN)
__device__ __forceinline__ uint32_t descending_key(float x) {
  // -0 and 0 are equal logits: adding 0 makes one of them
  const uint32_t bits = __float_as_uint(x + 0.0f);
  return (bits & 0x80000000u) ? bits : ~(bits | 0x80000000u);
}

struct Published {       // what a block shows the others of its cluster
  u64 sum;
  u64 found[4];          // a selection's result: {bin, sum before, sum in bin, count in bin}
  float best;
  int first;
};

struct SampleShared {
  u64 mass[kBins];
  unsigned count[kBins];
  u64 bin_mass[kBins];       // cluster totals of the bins this block owns
  unsigned bin_count[kBins];
  double power[64];
  u64 warp_sum[kSampleWarps];
  Published pub;
  float warp_best[kSampleWarps];
  int warp_first[kSampleWarps];
  u64 total;
};

// FP32 -> FP64 by moving bits (zero and subnormal numbers come out within 2^-126, which is
// nothing against the differences they enter); the conversion unit is four times slower
__device__ __forceinline__ double widen(float x) {
  const uint32_t u = __float_as_uint(x);
  const uint32_t hi = (u & 0x80000000u) | (((u & 0x7FFFFFFFu) >> 3) + 0x38000000u);
  return __hiloint2double((int)hi, (int)(u << 29));
}

// exp of (x - best) / temperature as an integer multiple of 2^-45; `rate` is log2(e) / temperature
struct Weigher {
  const double* power;
  double best, rate;
  float best_f;
  double least;  // min-p: smaller weights are dropped

  __device__ __forceinline__ double exponent(float x) const {
    return x == best_f ? 0.0 : (widen(x) - best) * rate;
  }
  __device__ __forceinline__ u64 operator()(float x) const {
    const double y = exponent(x);
    if (!(y > -46.5)) return 0ull;  // rounds to zero; also -inf
    // y = k / 64 + r: adding 1.5 * 2^46 leaves k in the low bits of the sum
    const double magic = 105553116266496.0;
    const double shifted = y + magic;
    const int k = __double2loint(shifted);
    const double z = (y - (shifted - magic)) * 0.69314718055994530942;
    double e = fma(z, 1.0 / 120.0, 1.0 / 24.0);
    e = fma(z, e, 1.0 / 6.0);
    e = fma(z, e, 0.5);
    e = fma(z, e, 1.0);
    const double t = power[k & 63];
    const double v = fma(t * z, e, t);          // 2^(k mod 64 / 64 + r)
    // times 2^(floor(k / 64) + 45) through the exponent field
    const double w =
        __hiloint2double(__double2hiint(v) + ((k >> 6) + kWeightBits) * (1 << 20), __double2loint(v));
    if (w < least) return 0ull;
    // round to an integer in the low bits: w <= 2^45
    const double rounded = w + 4503599627370496.0;
    return (u64)__double_as_longlong(rounded) & ((1ull << 52) - 1ull);
  }
};

// The tokens kept so far: those that come before (key, index) in the order, or are it.
struct Kept {
  uint32_t key;
  int last;
  __device__ __forceinline__ bool holds(uint32_t k, int index) const {
    return k < key || (k == key && index <= last);
  }
};

struct Row {
  const float* x;      // this block's tokens in shared memory
  int n, base;         // how many, and the index of the first
  int chunk;           // tokens of a warp, consecutive
  float best, scale;   // linear bins: (best - x) * scale
  __device__ __forceinline__ int bin(float v) const {
    return v == best ? 0 : min(kBins - 1, (int)((best - v) * scale));
  }
};

__device__ __forceinline__ u64 warp_total(u64 v) {
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}

// Sum over the cluster of one value per warp (already in sh.warp_sum); sh.pub.sum keeps the
// block's own share.
__device__ u64 cluster_total(SampleShared& sh, cg::cluster_group& cluster) {
  __syncthreads();
  if (threadIdx.x == 0) {
    u64 s = 0ull;
    for (int i = 0; i < kSampleWarps; ++i) s += sh.warp_sum[i];
    sh.pub.sum = s;
  }
  cluster.sync();
  u64 s = 0ull;
  for (unsigned r = 0; r < cluster.num_blocks(); ++r) s += cluster.map_shared_rank(&sh.pub, r)->sum;
  return s;
}

// The bin of the cluster's histogram in which the running sum reaches `need` (1 <= need <= the
// histogram's sum): {bin, sum before it, its sum, its count}.  BY_MASS: sums of weights, else of
// counts.  Each block adds up its share of the bins over the cluster, the one whose share holds
// the crossing finds it.
template <bool BY_MASS>
__device__ void find_bin(SampleShared& sh, cg::cluster_group& cluster, u64 need, u64 (&found)[4]) {
  const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int share = kBins / blocks;
  cluster.sync();  // every block's histogram is complete
  u64 mine = 0ull;
  for (int b = threadIdx.x; b < share; b += kSampleThreads) {
    u64 m = 0ull;
    unsigned c = 0u;
    for (int r = 0; r < blocks; ++r) {
      if (BY_MASS) m += cluster.map_shared_rank(sh.mass, r)[rank * share + b];
      c += cluster.map_shared_rank(sh.count, r)[rank * share + b];
    }
    sh.bin_mass[b] = BY_MASS ? m : (u64)c;
    sh.bin_count[b] = c;
    mine += BY_MASS ? m : (u64)c;
  }
  mine = warp_total(mine);
  if ((threadIdx.x & 31) == 0) sh.warp_sum[threadIdx.x >> 5] = mine;
  cluster_total(sh, cluster);
  u64 before = 0ull;
  int owner = 0;
  for (; owner < blocks - 1; ++owner) {
    const u64 s = cluster.map_shared_rank(&sh.pub, owner)->sum;
    if (before + s >= need) break;
    before += s;
  }
  if (owner == rank && threadIdx.x < 32) {
    // 32 lanes, consecutive bins each
    const int lane = threadIdx.x, per = share / 32;
    u64 s = 0ull;
    for (int i = 0; i < per; ++i) s += sh.bin_mass[lane * per + i];
    u64 upto = s;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const u64 o = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += o;
    }
    u64 run = before + upto - s;
    if (run < need && before + upto >= need) {
      for (int i = 0; i < per; ++i) {
        const u64 m = sh.bin_mass[lane * per + i];
        if (run + m >= need) {
          sh.pub.found[0] = (u64)(rank * share + lane * per + i);
          sh.pub.found[1] = run;
          sh.pub.found[2] = m;
          sh.pub.found[3] = sh.bin_count[lane * per + i];
          break;
        }
        run += m;
      }
    }
  }
  cluster.sync();
  for (int i = 0; i < 4; ++i) found[i] = cluster.map_shared_rank(&sh.pub, owner)->found[i];
}

template <bool BY_MASS>
__device__ __forceinline__ void clear_bins(SampleShared& sh) {
  for (int b = threadIdx.x; b < kBins; b += kSampleThreads) {
    if (BY_MASS) sh.mass[b] = 0ull;
    sh.count[b] = 0u;
  }
}

// The shortest prefix of the kept tokens whose sum (of counts, or of weights) reaches `need`;
// the histogram over the linear bins is in sh.mass / sh.count.
template <bool BY_MASS>
__device__ Kept select(SampleShared& sh, cg::cluster_group& cluster, const Row& row,
                       const Weigher& weigh, const Kept kept, u64 need) {
  u64 found[4];
  find_bin<BY_MASS>(sh, cluster, need, found);
  const int bin = (int)found[0];
  u64 rest = need - found[1];
  uint32_t prefix = 0u, mask = 0u;
  const int shifts[3] = {21, 10, 0}, widths[3] = {11, 11, 10};
#pragma unroll 1
  for (int level = 0; level < 3; ++level) {
    const int shift = shifts[level];
    const uint32_t digits = (1u << widths[level]) - 1u;
    __syncthreads();
    clear_bins<BY_MASS>(sh);
    __syncthreads();
    for (int i = threadIdx.x; i < row.n; i += kSampleThreads) {
      const float v = row.x[i];
      const uint32_t key = descending_key(v);
      if (row.bin(v) != bin || (key & mask) != prefix || !kept.holds(key, row.base + i)) continue;
      u64 w = 0ull;
      if (BY_MASS) {
        w = weigh(v);
        if (w == 0ull) continue;
        atomicAdd(&sh.mass[(key >> shift) & digits], w);
      }
      atomicAdd(&sh.count[(key >> shift) & digits], 1u);
    }
    find_bin<BY_MASS>(sh, cluster, rest, found);
    rest -= found[1];
    prefix |= (uint32_t)found[0] << shift;
    mask |= digits << shift;
  }
  // all tokens of the last bin have the same logit: how many of them are needed
  const u64 equal = found[3];
  const u64 each = BY_MASS ? found[2] / equal : 1ull;
  const u64 ties = (rest + each - 1ull) / each;
  Kept next;
  next.key = prefix;
  next.last = 0x7FFFFFFF;
  if (ties >= equal) {
    if (prefix == kept.key) next.last = kept.last;
    return next;
  }
  // the index of the ties-th of them
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int from = warp * row.chunk, to = min(row.n, from + row.chunk);
  unsigned n = 0u;
  for (int i = from + lane; i < to; i += 32)
    n += descending_key(row.x[i]) == prefix && kept.holds(prefix, row.base + i);
  n = __reduce_add_sync(0xffffffffu, n);
  if (lane == 0) sh.warp_sum[warp] = n;
  cluster_total(sh, cluster);
  u64 before = 0ull;
  for (unsigned r = 0; r < cluster.block_rank(); ++r)
    before += cluster.map_shared_rank(&sh.pub, r)->sum;
  for (int i = 0; i < warp; ++i) before += sh.warp_sum[i];
  if (threadIdx.x == 0) sh.pub.first = -1;
  __syncthreads();
  if (before < ties && before + n >= ties) {  // in this warp's tokens
    for (int i = from; i < to; i += 32) {
      const bool hit = i + lane < to && descending_key(row.x[i + lane]) == prefix &&
                       kept.holds(prefix, row.base + i + lane);
      const unsigned votes = __ballot_sync(0xffffffffu, hit);
      const unsigned want = (unsigned)(ties - before);  // >= 1
      if ((unsigned)__popc(votes) >= want) {
        if (hit && (unsigned)__popc(votes & ((2u << lane) - 1u)) == want)
          sh.pub.first = row.base + i + lane;
        break;
      }
      before += __popc(votes);
    }
  }
  cluster.sync();
  for (unsigned r = 0; r < cluster.num_blocks(); ++r) {
    const int f = cluster.map_shared_rank(&sh.pub, r)->first;
    if (f >= 0) next.last = f;
  }
  cluster.sync();
  return next;
}

template <typename T>
__device__ __forceinline__ float logit_at(const T* p, int i);
template <>
__device__ __forceinline__ float logit_at<float>(const float* p, int i) { return __ldg(p + i); }
template <>
__device__ __forceinline__ float logit_at<__nv_bfloat16>(const __nv_bfloat16* p, int i) {
  return __bfloat162float(p[i]);
}

template <typename T>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(const SampleParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  SampleShared& sh = *reinterpret_cast<SampleShared*>(smem);
  float* x = reinterpret_cast<float*>(smem + sizeof(SampleShared));
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), blocks = (int)cluster.num_blocks();
  const int row_id = blockIdx.x / blocks;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;

  Row row;
  row.x = x;
  row.base = min(p.vocab, rank * p.slice);
  row.n = min(p.vocab - row.base, p.slice);
  row.chunk = (row.n + 32 * kSampleWarps - 1) / (32 * kSampleWarps) * 32;

  const float temperature = p.temperature ? __ldg(p.temperature + row_id) : p.temperature_v;
  const int top_k = p.top_k ? __ldg(p.top_k + row_id) : p.top_k_v;
  const float top_p = p.top_p ? __ldg(p.top_p + row_id) : p.top_p_v;
  const float min_p = p.min_p ? __ldg(p.min_p + row_id) : p.min_p_v;
  const float u = __ldg(p.uniforms + row_id);

  // the row's tokens into shared memory, and the largest
  const T* src = static_cast<const T*>(p.logits) + (size_t)row_id * p.row_stride + row.base;
  float best = -INFINITY;
#pragma unroll 4
  for (int i = threadIdx.x; i < row.n; i += kSampleThreads) {
    float v = logit_at<T>(src, i);
    if (v != v) v = -INFINITY;
    x[i] = v;
    best = fmaxf(best, v);
  }
  if (threadIdx.x < 64) sh.power[threadIdx.x] = exp2((double)threadIdx.x / 64.0);
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, m));
  if (lane == 0) sh.warp_best[warp] = best;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < kSampleWarps; ++i) best = fmaxf(best, sh.warp_best[i]);
    sh.pub.best = best;
  }
  cluster.sync();
  best = -INFINITY;
  for (int r = 0; r < blocks; ++r) best = fmaxf(best, cluster.map_shared_rank(&sh.pub, r)->best);
  row.best = best;

  if (best == -INFINITY || !(temperature > 0.0f)) {  // nothing to draw, or nothing to draw by
    int first = 0x7FFFFFFF;
    for (int i = threadIdx.x; i < row.n; i += kSampleThreads)
      if (x[i] == best) {
        first = row.base + i;
        break;
      }
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0) sh.warp_first[warp] = first;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int i = 1; i < kSampleWarps; ++i) first = min(first, sh.warp_first[i]);
      sh.pub.first = first;
    }
    cluster.sync();
    if (rank == 0 && threadIdx.x == 0) {
      for (int r = 1; r < blocks; ++r) first = min(first, cluster.map_shared_rank(&sh.pub, r)->first);
      const bool none = best == -INFINITY;
      p.ids[row_id] = none ? -1 : first;
      if (p.logprobs) p.logprobs[row_id] = none ? -INFINITY : 0.0f;
    }
    cluster.sync();  // no block leaves while another reads its shared memory
    return;
  }

  Weigher weigh;
  weigh.power = sh.power;
  weigh.best = widen(best);
  weigh.best_f = best;
  weigh.rate = 1.4426950408889634074 / (double)temperature;
  // min-p in units of 2^-45; not above the largest weight, NaN: off
  weigh.least = min_p > 0.0f ? ldexp((double)fminf(min_p, 1.0f), kWeightBits) : 0.0;
  // 2047 linear bins over the range of logits whose weight is not zero, one for the rest
  row.scale = fminf((float)(2047.0 / 32.3) / temperature, 3.0e38f);

  Kept kept;
  kept.key = kMinusInfKey - 1u;  // every logit above -inf
  kept.last = 0x7FFFFFFF;

  // ---- top-k ------------------------------------------------------------------------------
  if (top_k > 0 && top_k < p.vocab) {
    __syncthreads();
    clear_bins<false>(sh);
    __syncthreads();
    unsigned live = 0u;
    for (int i = threadIdx.x; i < row.n; i += kSampleThreads) {
      const float v = x[i];
      if (v == -INFINITY) continue;
      ++live;
      atomicAdd(&sh.count[row.bin(v)], 1u);
    }
    live = __reduce_add_sync(0xffffffffu, live);
    if (lane == 0) sh.warp_sum[warp] = live;
    if (cluster_total(sh, cluster) > (u64)top_k)
      kept = select<false>(sh, cluster, row, weigh, kept, (u64)top_k);
    else
      cluster.sync();  // the counts above are read before the next sums replace them
  }

  // ---- weights; top-p ---------------------------------------------------------------------
  const bool nucleus = top_p < 1.0f;
  const int from = warp * row.chunk, to = min(row.n, from + row.chunk);
  u64 sum = 0ull;
  if (nucleus) {
    __syncthreads();
    clear_bins<true>(sh);
    __syncthreads();
  }
  for (int i = from + lane; i < to; i += 32) {
    const float v = x[i];
    if (!kept.holds(descending_key(v), row.base + i)) continue;
    const u64 w = weigh(v);
    if (w == 0ull) continue;
    sum += w;
    if (nucleus) {
      const int b = row.bin(v);
      atomicAdd(&sh.mass[b], w);
      atomicAdd(&sh.count[b], 1u);
    }
  }
  __syncthreads();
  sum = warp_total(sum);
  if (lane == 0) sh.warp_sum[warp] = sum;
  u64 total = cluster_total(sh, cluster);
  if (nucleus) {
    double need_d = ceil((double)fmaxf(top_p, 0.0f) * (double)total);
    u64 need = need_d < 1.0 ? 1ull : (u64)need_d;
    if (need < total) {
      kept = select<true>(sh, cluster, row, weigh, kept, need);
      sum = 0ull;
      for (int i = from + lane; i < to; i += 32) {
        const float v = x[i];
        if (kept.holds(descending_key(v), row.base + i)) sum += weigh(v);
      }
      __syncthreads();
      sum = warp_total(sum);
      if (lane == 0) sh.warp_sum[warp] = sum;
      total = cluster_total(sh, cluster);
    }
  }

  // ---- draw -------------------------------------------------------------------------------
  u64 target = u > 0.0f ? (u64)((double)fminf(u, 1.0f) * (double)total) : 0ull;
  if (target >= total) target = total - 1ull;
  u64 before = 0ull;
  for (int r = 0; r < rank; ++r) before += cluster.map_shared_rank(&sh.pub, r)->sum;
  for (int i = 0; i < warp; ++i) before += sh.warp_sum[i];
  if (before <= target && target < before + sum) {  // one warp of the cluster
    for (int i = from; i < to; i += 32) {
      const float v = i + lane < to ? x[i + lane] : -INFINITY;
      const u64 w = kept.holds(descending_key(v), row.base + i + lane) ? weigh(v) : 0ull;
      u64 upto = w;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const u64 o = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += o;
      }
      const unsigned past = __ballot_sync(0xffffffffu, before + upto > target);
      if (past) {
        if (lane == __ffs(past) - 1) {
          p.ids[row_id] = row.base + i + lane;
          if (p.logprobs)
            p.logprobs[row_id] =
                (float)(weigh.exponent(v) * 0.69314718055994530942 -
                        (log((double)total) - kWeightBits * 0.69314718055994530942));
        }
        break;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
  }
  cluster.sync();  // no block leaves while another reads its shared memory
}

}  // namespace

cudaError_t launch_sample(const void* logits, bool logits_f32, long long row_stride, int rows,
                          int vocab, const float* uniforms, const float* temperature,
                          float temperature_v, const int32_t* top_k, int top_k_v,
                          const float* top_p, float top_p_v, const float* min_p, float min_p_v,
                          int64_t* ids, float* logprobs, int sm_count, cudaStream_t stream) {
  SampleParams p;
  p.logits = logits;
  p.row_stride = row_stride;
  p.vocab = vocab;
  p.uniforms = uniforms;
  p.temperature = temperature;
  p.top_k = top_k;
  p.top_p = top_p;
  p.min_p = min_p;
  p.temperature_v = temperature_v;
  p.top_k_v = top_k_v;
  p.top_p_v = top_p_v;
  p.min_p_v = min_p_v;
  p.ids = ids;
  p.logprobs = logprobs;
  int blocks = 1;
  while (blocks < kMaxCluster && ((vocab + blocks - 1) / blocks > 16384 ||
                                  (rows * blocks * 2 <= sm_count && vocab / blocks > 4096)))
    blocks *= 2;
  p.slice = (vocab + blocks - 1) / blocks;
  const size_t bytes = sizeof(SampleShared) + (size_t)p.slice * sizeof(float);
  const void* kernel = logits_f32 ? (const void*)sample_kernel<float>
                                  : (const void*)sample_kernel<__nv_bfloat16>;
  cudaError_t err =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (err != cudaSuccess) return err;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)rows * blocks);
  config.blockDim = dim3(kSampleThreads);
  config.dynamicSmemBytes = bytes;
  config.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)blocks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  config.attrs = attr;
  config.numAttrs = 1;
  void* args[] = {&p};
  return cudaLaunchKernelExC(&config, kernel, args);
}

}  // namespace b200moe
