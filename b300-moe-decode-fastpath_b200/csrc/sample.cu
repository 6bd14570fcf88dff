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
// No sorting of the row.  What is kept is a prefix of the order, so it is described by its last
// element: a threshold on the logit and the index of the last token kept among those equal to it.
// A histogram over 2048 bins linear in the logit (for top-k of counts, for top-p of weights) finds
// the bin in which the wanted sum is crossed; the few hundred tokens of that bin are collected in
// a list, narrowed down by a second histogram over 256 pieces of the bin and compared with one
// another.  Where top-k leaves few tokens altogether they are collected instead, and one block
// does the rest.  A bin with more than 1024 tokens (equal logits, a range far from that of the
// weights) is taken apart by three histograms over the digits (11, 11 and 10 bits) of the logit's
// ordered bit pattern.  A row is read from memory once and stays in the shared memory of a cluster
// of up to eight blocks, which exchange histograms, lists and sums as distributed shared memory.
//
// What bounds it.  Few rows: the chain of load, four to five cluster barriers (0.23 us each, a
// remote read 0.37 us) and two passes over shared memory: 14.4 us for top-p over 32000 tokens,
// 13.3 us for 17 rows of 32003 with top-k and top-p, 11.1 us for plain draws from 8 rows of
// 129280.  Many rows: the same chain twice, since two blocks to an SM make 1.7 waves of 64 rows
// of 129280, with passes between its barriers that are chains of dependent operations (twelve in
// FP64 a token) and atomics: 34.6 us plain, 75.7 us with top-p 0.9, 37.8 us with top-k, 48.5 us
// mixed (5.0 us for the bytes alone).  Neither arithmetic nor memory is near its limit: with top-p
// an instruction is issued in 40 % of the cycles, the FP64 pipe is busy in 8 %, DRAM in 5 %, and
// warps wait for results, for barriers and for shared memory.  Shared-memory atomics
// of 64 bits are loops of compare-and-swap (9,000 to 16,000 cycles for 16,384 tokens, 240,000
// where they meet in four bins), those of 32 bits are not (1,300 and 4,300), so a weight is added
// as three parts of 15 bits.
//
// Exact sums.  With a large vocabulary the borders between tokens lie closer together than FP32
// sums resolve, and sums in another order would move them.  The weights are therefore integers,
// w_i * 2^45 rounded to nearest: their sums are exact in 64 bits for up to 2^18 tokens, do not
// depend on the order in which threads add them, and an atomic of integers leaves no trace of
// who came first.  The exponential behind them is computed in FP64 to about 2^-49: reduction to
// 2^(k/128) * 2^r with a table of 128 powers (Tang's table-driven scheme) and the Taylor
// polynomial of degree 4 on |r| <= 2^-8.  A thread weighs four tokens at a time and without
// branches, so that their chains of dependent FP64 operations overlap (a pass over a block's
// 16,160 tokens: 4.7 us against 6.4 us).
#include <cooperative_groups.h>
#include <float.h>

#include "common.cuh"

namespace b200moe {

namespace {

namespace cg = cooperative_groups;
typedef unsigned long long u64;

constexpr int kSampleThreads = 512;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kBins = 2048;
constexpr int kWeightBits = 45;
constexpr int kPowers = 128;
constexpr int kMaxCluster = 8;
constexpr int kWide = 4;      // tokens that a thread weighs at a time
constexpr int kPad = kSampleThreads * kWide;

// Weights are added up in the histogram as three parts of 15 bits (the highest may be 2^15):
// with at most 2^15 tokens in a block their sums stay within 32 bits.
constexpr int kPartBits = 15;
constexpr int kGroups = 64;            // groups of 32 bins
constexpr int kList = 1024;            // tokens of a list
// Lists of up to so many tokens are compared pair by pair, longer ones sorted: two sorts of 64 to
// 128 tokens take 4 us, two comparisons 1 us, but the work of a comparison grows with the square.
constexpr int kPairs = 256;
constexpr int kPieces = 256;           // of a bin

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

// ascending order of this key = descending order of the logit (no NaN); and back
__device__ __forceinline__ uint32_t descending_key(float x) {
  // -0 and 0 are equal logits: adding 0 makes one of them
  const uint32_t bits = __float_as_uint(x + 0.0f);
  return (bits & 0x80000000u) ? bits : ~(bits | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? key : ~key & 0x7FFFFFFFu);
}

struct Found {
  int bin;      // -1: the whole histogram stays below what was asked for
  u64 before;   // sum of the bins before it
  u64 amount;   // its own
};

struct alignas(16) SampleShared {
  uint32_t part[3][kBins];     // counts: the first one only
  u64 list[kList];             // of this block: {key, index}
  u64 group[kGroups];          // of this block
  u64 group_total[kGroups];    // of the cluster
  u64 bins[kMaxCluster][32];   // a group of bins of every block
  double power[kPowers];
  u64 warp_sum[kSampleWarps];
  u64 sum;                     // what a block shows the others: sum, largest logit, an index
  float best;
  int first;
  unsigned list_n[2];          // of the count stage and of the weight stage
  Found found;
  float warp_best[kSampleWarps];
  int warp_first[kSampleWarps];
  unsigned piece_n;
  float kept_x;
  int kept_last;
};

// exp of (x - best) / temperature as an integer multiple of 2^-45; `rate` is log2(e) / temperature
struct Weigher {
  const double* power;   // 2^(i/128 + 45)
  double best, rate;
  float best_f;
  float lowest;          // a logit whose weight rounds to zero (then also that of all below it)
  bool bounded;          // there is such a logit, and the largest one is finite
  bool has_least;
  double least;          // min-p: smaller weights are dropped

  __device__ __forceinline__ void set(const double* power_, float best_, float temperature,
                                      float min_p) {
    power = power_;
    best_f = best_;
    best = (double)best_;
    rate = 1.4426950408889634074 / (double)temperature;
    lowest = best_ - 40.0f * temperature;  // 2^-57.7
    bounded = isfinite(best_) && isfinite(lowest) && ((double)lowest - best) * rate < -48.0;
    // min-p in units of 2^-45, not above the largest weight; NaN: off
    has_least = min_p > 0.0f;
    least = has_least ? ldexp((double)fminf(min_p, 1.0f), kWeightBits) : 0.0;
  }
  // y > -1000; k: y in units of 2^-7, rounded
  __device__ __forceinline__ u64 power_of(double y, int& k) const {
    // y = k / 128 + r: adding 1.5 * 2^45 leaves k in the low bits of the sum
    const double magic = 52776558133248.0;
    const double shifted = y + magic;
    k = __double2loint(shifted);
    const double r = y - (shifted - magic);
    // 2^r = 1 + r (c1 + r (c2 + r (c3 + r c4))), cn = ln(2)^n / n!
    constexpr double c1 = 0.69314718055994530942;
    constexpr double c2 = c1 * c1 / 2, c3 = c2 * c1 / 3, c4 = c3 * c1 / 4;
    double e = fma(r, c4, c3);
    e = fma(r, e, c2);
    e = fma(r, e, c1);
    const double t = power[k & (kPowers - 1)];
    const double v = fma(t * r, e, t);          // 2^(k mod 128 / 128 + r + 45)
    // times 2^floor(k / 128) through the exponent field
    const double w = __hiloint2double(
        __double2hiint(v) + (int)(((unsigned)k & ~(unsigned)(kPowers - 1)) << 13), __double2loint(v));
    // round to an integer in the low bits: w <= 2^45
    const u64 n = (u64)__double_as_longlong(w + 4503599627370496.0) & ((1ull << 52) - 1ull);
    return has_least && w < least ? 0ull : n;
  }
  __device__ __forceinline__ double exponent(float x) const {
    return x == best_f ? 0.0 : ((double)x - best) * rate;
  }
  // any logit but NaN; -inf: 0.  bin: of the weight histogram, four units of 2^-7 octaves each
  __device__ __forceinline__ u64 operator()(float x, int& bin) const {
    int k;
    u64 w;
    if (bounded) {
      w = power_of(((double)fmaxf(x, lowest) - best) * rate, k);
    } else {
      const double y = exponent(x);
      const bool counts = x != -INFINITY && y > -48.0;
      w = power_of(counts ? y : 0.0, k);
      if (!counts) w = 0ull;
    }
    bin = -k >> 2;  // below 2048: y is above -58
    return w;
  }
  __device__ __forceinline__ u64 operator()(float x) const {
    int bin;
    return (*this)(x, bin);
  }
  // A range of logits that holds all of a bin's (and a few of its neighbours').
  __device__ __forceinline__ void range_of(int bin, float& low, float& high) const {
    low = -INFINITY;
    high = INFINITY;
    if (!bounded) return;
    const double a = best - (4 * bin + 3.5) / (128.0 * rate), b = best - (4 * bin - 0.5) / (128.0 * rate);
    low = (float)(a - 1e-6 * fabs(a) - 1e-37);
    high = (float)(b + 1e-6 * fabs(b) + 1e-37);
  }
  // the part of the bin that x lies in, of kPieces
  __device__ __forceinline__ int piece(float x, int bin) const {
    const double t = (-128.0 * exponent(x) - (4 * bin - 0.5)) * (kPieces / 4);
    return (int)fmin(fmax(t, 0.0), (double)(kPieces - 1));
  }
};

// The tokens kept so far: those with a larger logit, and up to index `last` those with this one.
struct Kept {
  float x;
  int last;
  __device__ __forceinline__ bool holds(float v, int index) const {
    return v > x || (v == x && index <= last);
  }
};

struct Row {
  const float* x;      // this block's tokens in shared memory, -inf behind them
  int n, base;         // how many, and the index of the first
  int chunk;           // tokens of a warp, consecutive; a multiple of 32 kWide
  float best, scale;   // bins of the count histogram: linear, (best - x) * scale
  __device__ __forceinline__ int bin(float v) const {
    return v == best ? 0 : min(kBins - 1, (int)((best - v) * scale));
  }
  // whether bin(v) == b, for a bin's borders as numbers
  __device__ __forceinline__ bool in_bin(float v, int b) const {
    const float t = v == best ? 0.0f : (best - v) * scale;
    return t >= (float)b && (t < (float)(b + 1) || b == kBins - 1);
  }
  // and up to bin b
  __device__ __forceinline__ bool upto_bin(float v, int b) const {
    return v == best || (best - v) * scale < (float)(b + 1) || b == kBins - 1;
  }
  // the part of bin b that v lies in, of kPieces
  __device__ __forceinline__ int piece(float v, int b) const {
    const float t = v == best ? 0.0f : (best - v) * scale;
    return max(0, min(kPieces - 1, (int)((t - (float)b) * (float)kPieces)));
  }
};

__device__ __forceinline__ u64 warp_total(u64 v) {
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}

__device__ __forceinline__ u64 inclusive_scan(u64 v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const u64 o = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v += o;
  }
  return v;
}

// Sum over the block of one value per warp (already in sh.warp_sum).
__device__ __forceinline__ u64 block_total(SampleShared& sh) {
  __syncthreads();
  u64 s = 0ull;
#pragma unroll
  for (int i = 0; i < kSampleWarps; ++i) s += sh.warp_sum[i];
  return s;
}
// The value that every block of the cluster holds at `p`, one block per lane (0 in other lanes).
template <typename V>
__device__ __forceinline__ V cluster_read(cg::cluster_group& cluster, V* p) {
  const unsigned lane = threadIdx.x & 31;
  return lane < cluster.num_blocks() ? *cluster.map_shared_rank(p, lane) : V(0);
}
// The same over the cluster; sh.sum keeps the block's own share, before: that of the blocks in
// front of it.
__device__ __forceinline__ u64 cluster_total(SampleShared& sh, cg::cluster_group& cluster,
                                             u64& before) {
  const u64 mine = block_total(sh);
  if (threadIdx.x == 0) sh.sum = mine;
  cluster.sync();
  const u64 upto = inclusive_scan(cluster_read(cluster, &sh.sum));
  before = __shfl_sync(0xffffffffu, upto, (int)cluster.block_rank()) - mine;
  return __shfl_sync(0xffffffffu, upto, 31);
}

template <bool BY_MASS>
__device__ __forceinline__ void clear_bins(SampleShared& sh) {
  for (int b = threadIdx.x; b < kBins; b += kSampleThreads) {
    sh.part[0][b] = 0u;
    if (BY_MASS) sh.part[1][b] = sh.part[2][b] = 0u;
  }
}
// `part`: three arrays of BINS counters, one behind the other
template <int BINS>
__device__ __forceinline__ void add_mass(uint32_t* part, int bin, u64 w) {
  constexpr uint32_t mask = (1u << kPartBits) - 1u;
  atomicAdd(part + bin, (uint32_t)w & mask);
  atomicAdd(part + BINS + bin, (uint32_t)(w >> kPartBits) & mask);
  atomicAdd(part + 2 * BINS + bin, (uint32_t)(w >> (2 * kPartBits)));
}
template <bool BY_MASS, int BINS = kBins>
__device__ __forceinline__ u64 bin_amount(const uint32_t* part, int bin) {
  u64 v = part[bin];
  if (BY_MASS)
    v += ((u64)part[BINS + bin] << kPartBits) + ((u64)part[2 * BINS + bin] << (2 * kPartBits));
  return v;
}
// The bin of the cluster's histogram in which the running sum reaches need(total), and the
// histogram's total.  Every block finds it for itself: from the sums of 64 groups of 32 bins of
// all blocks, then from the bins of one group.
template <bool BY_MASS, typename Need>
__device__ Found find_bin(SampleShared& sh, cg::cluster_group& cluster, Need need_of, u64& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int blocks = (int)cluster.num_blocks();
  __syncthreads();
  {  // four bins per thread, eight threads per group
    static_assert(kBins == 4 * kSampleThreads && kBins == 32 * kGroups, "bins per thread");
    u64 v = 0ull;
#pragma unroll
    for (int i = 0; i < 4; ++i) v += bin_amount<BY_MASS>(sh.part[0], 4 * threadIdx.x + i);
#pragma unroll
    for (int m = 4; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    if ((threadIdx.x & 7) == 0) sh.group[threadIdx.x / 8] = v;
  }
  cluster.sync();
  {  // as many neighbouring lanes as there are blocks share a group
    static_assert(kGroups * kMaxCluster <= kSampleThreads, "one group of one block per thread");
    const int group = threadIdx.x / blocks, r = threadIdx.x % blocks;
    u64 v = group < kGroups ? cluster.map_shared_rank(sh.group, r)[group] : 0ull;
    for (int m = blocks >> 1; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    if (group < kGroups && r == 0) sh.group_total[group] = v;
  }
  __syncthreads();
  const u64 a = sh.group_total[2 * lane], b = sh.group_total[2 * lane + 1];
  const u64 upto = inclusive_scan(a + b);
  total = __shfl_sync(0xffffffffu, upto, 31);
  const u64 need = need_of(total);
  Found found;
  found.bin = -1;
  found.before = found.amount = 0ull;
  if (need > total) return found;  // in every block alike
  const int at = __ffs(__ballot_sync(0xffffffffu, upto >= need)) - 1;
  u64 before = __shfl_sync(0xffffffffu, upto - a - b, at);
  const u64 first = __shfl_sync(0xffffffffu, a, at);
  int group = 2 * at;
  if (before + first < need) {
    before += first;
    ++group;
  }
  const int bin = group * 32 + lane;
  if (warp < blocks)  // one warp per block of the cluster: a single trip
    sh.bins[warp][lane] = bin_amount<BY_MASS>(cluster.map_shared_rank(sh.part[0], warp), bin);
  __syncthreads();
  if (warp == 0) {
    u64 v = 0ull;
    for (int r = 0; r < blocks; ++r) v += sh.bins[r][lane];
    const u64 run = before + inclusive_scan(v);
    if (lane == __ffs(__ballot_sync(0xffffffffu, run >= need)) - 1) {
      sh.found.bin = bin;
      sh.found.before = run - v;
      sh.found.amount = v;
    }
  }
  __syncthreads();
  return sh.found;
}

// (logit, index) as one integer, in the order of the tokens
__device__ __forceinline__ u64 place(uint32_t key, int index) { return ((u64)key << 32) | (unsigned)index; }
__device__ __forceinline__ float logit_at(u64 place) { return logit_of((uint32_t)(place >> 32)); }

// Appends the warp's chosen tokens to the block's list; `count` goes on counting where that is
// full.
__device__ __forceinline__ void append(bool chosen, u64 entry, u64* list, unsigned* count) {
  const unsigned votes = __ballot_sync(0xffffffffu, chosen);
  if (votes == 0u) return;
  const int lane = threadIdx.x & 31, leader = __ffs(votes) - 1;
  unsigned base = 0u;
  if (lane == leader) base = atomicAdd(count, (unsigned)__popc(votes));
  base = __shfl_sync(0xffffffffu, base, leader);
  const unsigned at = base + __popc(votes & ((1u << lane) - 1u));
  if (chosen && at < (unsigned)kList) list[at] = entry;
}
// The number of tokens in all lists of the cluster, and, where they fit, a copy of them in
// `merged`.  The lists have to stay until every block has come past a further cluster barrier.
__device__ __forceinline__ unsigned merge_lists(SampleShared& sh, cg::cluster_group& cluster,
                                                unsigned* count, u64* merged) {
  const unsigned blocks = cluster.num_blocks();
  unsigned n[kMaxCluster], total = 0u;
  const unsigned held = cluster_read(cluster, count);
#pragma unroll
  for (int r = 0; r < kMaxCluster; ++r) {
    n[r] = __shfl_sync(0xffffffffu, held, r);
    total += n[r];
  }
  if (merged && total <= (unsigned)kList) {
    unsigned at = 0u;
#pragma unroll
    for (unsigned r = 0; r < kMaxCluster; ++r) {
      if (r < blocks)
        for (unsigned i = threadIdx.x; i < n[r]; i += kSampleThreads)
          merged[at + i] = cluster.map_shared_rank(sh.list, r)[i];
      at += n[r];
    }
  }
  return total;
}

// For n <= kPairs entries in shared memory: of the entry that this thread shares with its
// neighbours (`lanes` of them), how many come before it, and the sum of their weights.
struct Before {
  int entry;     // -1: none
  bool first;    // of the threads that share it
  int rank;
  u64 sum;
};
__device__ __forceinline__ Before compare_all(const u64* entry, const u64* weight, int n) {
  const int padded = n <= 1 ? 1 : 1 << (32 - __clz(n - 1));
  const int lanes = min(32, kSampleThreads / padded), part = threadIdx.x & (lanes - 1);
  Before b;
  b.entry = threadIdx.x / lanes;
  b.first = part == 0;
  b.rank = 0;
  b.sum = 0ull;
  const bool in = b.entry < n;
  const u64 mine = in ? entry[b.entry] : 0ull;
#pragma unroll 2
  for (int j = part; j < n; j += lanes)
    if (entry[j] < mine) {
      ++b.rank;
      b.sum += weight[j];
    }
  for (int m = lanes >> 1; m > 0; m >>= 1) {
    b.rank += __shfl_xor_sync(0xffffffffu, b.rank, m);
    b.sum += __shfl_xor_sync(0xffffffffu, b.sum, m);
  }
  if (!in) b.entry = -1;
  return b;
}

// Sorts `count` integers, two per thread (2 t and 2 t + 1), ascending; what is behind them must be
// ~0.  A bitonic network: partners within a warp exchange by shuffles, others through `scratch`
// (two integers per thread).  Threads without a share only keep the barriers.
__device__ __forceinline__ void sort_block(u64 (&v)[2], int count, ulonglong2* scratch) {
  const int t = threadIdx.x;
  const int padded = max(2, count <= 1 ? 1 : 1 << (32 - __clz(count - 1)));
  const bool in = 2 * (t & ~31) < padded;  // whole warps
  for (int size = 2; size <= padded; size <<= 1) {
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      const bool up = (2 * t & size) == 0;
      if (stride >= 64) {
        __syncthreads();
        if (in) scratch[t] = make_ulonglong2(v[0], v[1]);
        __syncthreads();
      }
      if (!in) continue;
      if (stride == 1) {
        const bool ascending = size == 2 ? (t & 1) == 0 : up;
        if ((v[0] > v[1]) == ascending) {
          const u64 x = v[0];
          v[0] = v[1];
          v[1] = x;
        }
        continue;
      }
      const bool low = (2 * t & stride) == 0;  // keeps the smaller of the two where ascending
      u64 other[2];
      if (stride >= 64) {
        const ulonglong2 o = scratch[t ^ (stride >> 1)];
        other[0] = o.x;
        other[1] = o.y;
      } else {
        other[0] = __shfl_xor_sync(0xffffffffu, v[0], stride >> 1);
        other[1] = __shfl_xor_sync(0xffffffffu, v[1], stride >> 1);
      }
#pragma unroll
      for (int q = 0; q < 2; ++q)
        if ((other[q] < v[q]) == (low == up)) v[q] = other[q];
    }
  }
}
// Sum of v over the threads before this one, and over all.
__device__ __forceinline__ u64 block_scan(SampleShared& sh, u64 v, u64& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 upto = inclusive_scan(v);
  __syncthreads();  // the sums before have been read
  if (lane == 31) sh.warp_sum[warp] = upto;
  __syncthreads();
  u64 before = 0ull;
  total = 0ull;
#pragma unroll
  for (int i = 0; i < kSampleWarps; ++i) {
    const u64 w = sh.warp_sum[i];
    if (i < warp) before += w;
    total += w;
  }
  return before + upto - v;
}
// The shortest prefix of the kept tokens whose sum (of counts, or of weights) ends in bin
// `found.bin` of the linear histogram, `rest` (at least 1) into it.
template <bool BY_MASS>
__device__ Kept select(SampleShared& sh, cg::cluster_group& cluster, const Row& row,
                       const Weigher& weigh, const Kept kept, const int bin, u64 rest) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int from = warp * row.chunk, to = min(row.n, from + row.chunk);
  // the bin's tokens
  unsigned* count = &sh.list_n[BY_MASS];
  float low, high;
  if (BY_MASS) weigh.range_of(bin, low, high);
  for (int i = from + lane; i < from + row.chunk; i += 32 * kWide) {
    float v[kWide];
    bool chosen[kWide], any = false;
#pragma unroll
    for (int j = 0; j < kWide; ++j) {
      v[j] = row.x[i + 32 * j];
      chosen[j] = v[j] != -INFINITY && (BY_MASS ? v[j] >= low && v[j] <= high : row.in_bin(v[j], bin));
      any |= chosen[j];
    }
    if (!__any_sync(0xffffffffu, any)) continue;
#pragma unroll
    for (int j = 0; j < kWide; ++j) {
      const int index = row.base + i + 32 * j;
      if (BY_MASS && chosen[j]) {  // a neighbour of the bin, or dropped by min-p?
        int b;
        chosen[j] = weigh(v[j], b) != 0ull && b == bin;
      }
      append(chosen[j] && kept.holds(v[j], index), place(descending_key(v[j]), index), sh.list, count);
    }
  }
  cluster.sync();  // the lists are complete, and the histogram has been read
  u64* merged = reinterpret_cast<u64*>(&sh.part[2][0]);  // the pieces are in part[0] and part[1]
  const unsigned n = merge_lists(sh, cluster, count, merged);
  Kept next;
  if (n <= (unsigned)kList) {
    // A histogram of the list over 256 pieces of the bin narrows it down to the tokens of one
    // piece, mostly one or two; those are sorted.  Every block does this for itself.
    static_assert(kList <= 2 * kSampleThreads, "two tokens per thread");
    static_assert(3 * kPieces <= kBins, "the three parts of the pieces fit part[0]");
    uint32_t* pieces = sh.part[0];
    for (int i = threadIdx.x; i < 3 * kPieces; i += kSampleThreads) pieces[i] = 0u;
    if (threadIdx.x == 0) sh.piece_n = 0u;
    __syncthreads();
    u64 e[2], w[2];
    int piece[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const unsigned i = threadIdx.x + q * kSampleThreads;
      w[q] = 0ull;
      piece[q] = -1;
      if (i >= n) continue;
      e[q] = merged[i];
      const float v = logit_at(e[q]);
      w[q] = BY_MASS ? weigh(v) : 1ull;
      piece[q] = BY_MASS ? weigh.piece(v, bin) : row.piece(v, bin);
      if (w[q]) add_mass<kPieces>(pieces, piece[q], w[q]);
    }
    __syncthreads();
    // every warp: eight pieces per lane
    u64 amount[kPieces / 32], sum = 0ull;
#pragma unroll
    for (int i = 0; i < kPieces / 32; ++i) {
      amount[i] = bin_amount<true, kPieces>(pieces, lane * (kPieces / 32) + i);
      sum += amount[i];
    }
    u64 run = inclusive_scan(sum) - sum;
    int mine = -1;
    if (run < rest && run + sum >= rest) {
#pragma unroll
      for (int i = 0; i < kPieces / 32; ++i) {
        if (mine >= 0) break;
        if (run + amount[i] >= rest) mine = lane * (kPieces / 32) + i;
        else run += amount[i];
      }
    }
    const int at = __ffs(__ballot_sync(0xffffffffu, mine >= 0)) - 1;
    mine = __shfl_sync(0xffffffffu, mine, at);
    rest -= __shfl_sync(0xffffffffu, run, at);
    u64* some = reinterpret_cast<u64*>(&sh.part[1][0]);
#pragma unroll
    for (int q = 0; q < 2; ++q)
      if (piece[q] == mine) some[atomicAdd(&sh.piece_n, 1u)] = e[q];
    __syncthreads();
    const int m = (int)sh.piece_n;
    if (m <= kPairs) {
      u64* weight = some + kPairs;
      if (threadIdx.x < m) weight[threadIdx.x] = BY_MASS ? weigh(logit_at(some[threadIdx.x])) : 1ull;
      __syncthreads();
      const Before b = compare_all(some, weight, m);
      if (b.entry >= 0 && b.first && b.sum < rest && b.sum + weight[b.entry] >= rest) {
        sh.kept_x = logit_at(some[b.entry]);
        sh.kept_last = (int)(uint32_t)some[b.entry];
      }
    } else {
      u64 v[2], total;
#pragma unroll
      for (int q = 0; q < 2; ++q) v[q] = 2 * threadIdx.x + q < m ? some[2 * threadIdx.x + q] : ~0ull;
      sort_block(v, m, reinterpret_cast<ulonglong2*>(&sh.part[1][0]));
#pragma unroll
      for (int q = 0; q < 2; ++q) w[q] = v[q] == ~0ull ? 0ull : BY_MASS ? weigh(logit_at(v[q])) : 1ull;
      const u64 before = block_scan(sh, w[0] + w[1], total);
      if (before < rest && before + w[0] + w[1] >= rest) {
        const u64 last = before + w[0] >= rest ? v[0] : v[1];
        sh.kept_x = logit_at(last);
        sh.kept_last = (int)(uint32_t)last;
      }
    }
    __syncthreads();
    next.x = sh.kept_x;
    next.last = sh.kept_last;
    cluster.sync();  // the lists have been read
    return next;
  }

  uint32_t prefix = 0u, mask = 0u;
  const int shifts[3] = {21, 10, 0}, widths[3] = {11, 11, 10};
  Found found;
#pragma unroll 1
  for (int level = 0; level < 3; ++level) {
    const int shift = shifts[level];
    const uint32_t digits = (1u << widths[level]) - 1u;
    cluster.sync();  // the histogram before has been read
    clear_bins<BY_MASS>(sh);
    __syncthreads();
    for (int i = threadIdx.x; i < row.n; i += kSampleThreads) {
      const float v = row.x[i];
      const uint32_t key = descending_key(v);
      if ((key & mask) != prefix || !kept.holds(v, row.base + i)) continue;
      const int digit = (key >> shift) & digits;
      if (BY_MASS) {
        int b;
        const u64 w = weigh(v, b);
        if (w && b == bin) add_mass<kBins>(sh.part[0], digit, w);
      } else if (row.bin(v) == bin) {
        atomicAdd(&sh.part[0][digit], 1u);
      }
    }
    u64 total;
    found = find_bin<BY_MASS>(sh, cluster, [&](u64) { return rest; }, total);
    rest -= found.before;
    prefix |= (uint32_t)found.bin << shift;
    mask |= digits << shift;
  }
  // all tokens of the last bin have the same logit: how many of them are needed
  const u64 each = BY_MASS ? weigh(logit_of(prefix)) : 1ull;
  const u64 equal = found.amount / each;
  const u64 ties = (rest + each - 1ull) / each;
  next.x = logit_of(prefix);
  next.last = 0x7FFFFFFF;
  if (ties >= equal) {
    if (next.x == kept.x) next.last = kept.last;
    cluster.sync();  // the histogram has been read
    return next;
  }
  // the index of the ties-th of them
  unsigned hits = 0u;
  for (int i = from + lane; i < to; i += 32)
    hits += row.x[i] == next.x && kept.holds(next.x, row.base + i);
  hits = __reduce_add_sync(0xffffffffu, hits);
  if (lane == 0) sh.warp_sum[warp] = hits;
  if (threadIdx.x == 0) sh.first = -1;
  u64 before;
  cluster_total(sh, cluster, before);
  for (int i = 0; i < warp; ++i) before += sh.warp_sum[i];
  if (before < ties && before + hits >= ties) {  // in this warp's tokens
    for (int i = from; i < to; i += 32) {
      const bool hit = i + lane < to && row.x[i + lane] == next.x &&
                       kept.holds(next.x, row.base + i + lane);
      const unsigned votes = __ballot_sync(0xffffffffu, hit);
      const unsigned want = (unsigned)(ties - before);  // >= 1
      if ((unsigned)__popc(votes) >= want) {
        if (hit && (unsigned)__popc(votes & ((2u << lane) - 1u)) == want)
          sh.first = row.base + i + lane;
        break;
      }
      before += __popc(votes);
    }
  }
  cluster.sync();
  for (unsigned r = 0; r < cluster.num_blocks(); ++r) {
    const int f = *cluster.map_shared_rank(&sh.first, r);
    if (f >= 0) next.last = f;
  }
  cluster.sync();
  return next;
}

// The weights of the kept tokens among the warp's, summed over its lanes' shares.  The kept ones
// are packed, so that a warp weighs 32 of them at a time however few there are (top-p 0.9 of
// 129280 tokens keeps about one in ten: 5.8 us of a block when every token is weighed).
__device__ __forceinline__ u64 sum_kept(SampleShared& sh, const Row& row, const Weigher& weigh,
                                        const Kept kept) {
  constexpr int kRoom = 32 * (kWide + 1);
  static_assert(kSampleWarps * kRoom <= 3 * kBins, "the packed logits lie where the histogram was");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, from = warp * row.chunk;
  float* packed = reinterpret_cast<float*>(&sh.part[0][0]) + warp * kRoom;
  int held = 0;
  u64 sum = 0ull;
  for (int i = from + lane; i < from + row.chunk; i += 32 * kWide) {
#pragma unroll
    for (int j = 0; j < kWide; ++j) {
      const float v = row.x[i + 32 * j];
      const bool wanted = kept.holds(v, row.base + i + 32 * j);
      const unsigned votes = __ballot_sync(0xffffffffu, wanted);
      if (wanted) packed[held + __popc(votes & ((1u << lane) - 1u))] = v;
      held += __popc(votes);
    }
    __syncwarp();
    while (held >= 32) {
      held -= 32;
      sum += weigh(packed[held + lane]);
    }
    __syncwarp();
  }
  if (lane < held) sum += weigh(packed[lane]);
  return sum;
}

// Top-p's share of a sum of weights, at least 1.
__device__ __forceinline__ u64 mass_needed(float top_p, u64 total) {
  const double need = ceil((double)fmaxf(top_p, 0.0f) * (double)total);
  return need < 1.0 ? 1ull : (u64)need;
}
// The weight at which the draw falls.
__device__ __forceinline__ u64 draw_target(float u, u64 total) {
  const u64 target = u > 0.0f ? (u64)((double)fminf(u, 1.0f) * (double)total) : 0ull;
  return target >= total ? total - 1ull : target;
}
__device__ __forceinline__ void store_result(const SampleParams& p, int row_id,
                                             const Weigher& weigh, int index, float x, u64 total) {
  p.ids[row_id] = index;
  if (p.logprobs)
    p.logprobs[row_id] = (float)(weigh.exponent(x) * 0.69314718055994530942 -
                                 (log((double)total) - kWeightBits * 0.69314718055994530942));
}

// All that is left after top-k fits a list (in part[2]): one block cuts it to k tokens, weighs
// them, cuts to top-p and draws.  A short list is compared entry by entry, a long one sorted by
// the order and, for the draw, by index.
__device__ void finish_list(SampleShared& sh, const SampleParams& p, int row_id,
                            const Weigher& weigh, u64* entry, int n, int top_k, float top_p,
                            float u) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 total;
  __syncthreads();
  if (n <= kPairs) {
    u64* weight = reinterpret_cast<u64*>(&sh.part[0][0]);
    if (threadIdx.x < n) weight[threadIdx.x] = weigh(logit_at(entry[threadIdx.x]));
    __syncthreads();
    const Before b = compare_all(entry, weight, n);
    const bool mine = b.entry >= 0 && b.first;
    u64 w = mine && b.rank < top_k ? weight[b.entry] : 0ull;
    u64 sum = warp_total(w);
    if (lane == 0) sh.warp_sum[warp] = sum;
    total = block_total(sh);  // and all weights have been read
    if (top_p < 1.0f) {
      if (b.sum >= mass_needed(top_p, total)) w = 0ull;
      sum = warp_total(w);
      __syncthreads();
      if (lane == 0) sh.warp_sum[warp] = sum;
      total = block_total(sh);
    }
    // again by index; {index, key}
    u64* by_index = reinterpret_cast<u64*>(&sh.part[1][0]);
    if (mine) {
      weight[b.entry] = w;
      by_index[b.entry] = (entry[b.entry] << 32) | (entry[b.entry] >> 32);
    }
    __syncthreads();
    const Before d = compare_all(by_index, weight, n);
    const u64 target = draw_target(u, total);
    if (d.entry >= 0 && d.first && d.sum <= target && target < d.sum + weight[d.entry])
      store_result(p, row_id, weigh, (int)(uint32_t)entry[d.entry], logit_at(entry[d.entry]), total);
    return;
  }
  const int at = 2 * threadIdx.x;
  ulonglong2* scratch = reinterpret_cast<ulonglong2*>(&sh.part[0][0]);
  u64 v[2], w[2];
#pragma unroll
  for (int q = 0; q < 2; ++q) v[q] = at + q < n ? entry[at + q] : ~0ull;
  __syncthreads();
  sort_block(v, n, scratch);
#pragma unroll
  for (int q = 0; q < 2; ++q)
    w[q] = at + q < n && at + q < top_k ? weigh(logit_at(v[q])) : 0ull;
  u64 before = block_scan(sh, w[0] + w[1], total);
  if (top_p < 1.0f) {
    const u64 need = mass_needed(top_p, total);
    if (before + w[0] >= need) w[1] = 0ull;
    if (before >= need) w[0] = 0ull;
  }
  // {index, place in the order}; what is not kept goes to the end
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    entry[at + q] = v[q];
    v[q] = w[q] ? (v[q] << 32) | (unsigned)(at + q) : ~0ull;
  }
  __syncthreads();
  sort_block(v, n, scratch);
  float x[2];
  int index[2];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const u64 e = v[q] != ~0ull ? entry[(unsigned)v[q]] : 0ull;
    x[q] = logit_at(e);
    index[q] = (int)(uint32_t)e;
    w[q] = v[q] != ~0ull ? weigh(x[q]) : 0ull;
  }
  before = block_scan(sh, w[0] + w[1], total);
  const u64 target = draw_target(u, total);
  if (before <= target && target < before + w[0] + w[1]) {
    const int q = target < before + w[0] ? 0 : 1;
    store_result(p, row_id, weigh, index[q], x[q], total);
  }
}

// The block's logits into shared memory at x[0..n), NaN as -inf; returns the thread's largest.
// 16-byte loads where the row's address allows, all of a thread's in flight at once.
__device__ __forceinline__ float keep(float v, float& best) {
  if (v != v) v = -INFINITY;
  best = fmaxf(best, v);
  return v;
}
// elements in front of the first 16-byte boundary
template <typename T>
__device__ __forceinline__ int head_of(const T* src) {
  return (int)((16u - (unsigned)(reinterpret_cast<uintptr_t>(src) & 15u)) % 16u / sizeof(T));
}
// x + head_of(src) is on a 16-byte boundary too
template <typename T>
__device__ __forceinline__ float load_row(const T* __restrict__ src, int n, float* x) {
  constexpr int kVec = 16 / sizeof(T), kAhead = 8;
  float best = -INFINITY;
  const int head = min(n, head_of(src));
  const int vecs = (n - head) / kVec;
  for (int start = threadIdx.x; start < vecs; start += kAhead * kSampleThreads) {
    uint4 q[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (start + i * kSampleThreads < vecs)
        q[i] = __ldg(reinterpret_cast<const uint4*>(src + head) + start + i * kSampleThreads);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (start + i * kSampleThreads >= vecs) break;
      float4* dst = reinterpret_cast<float4*>(x + head + (start + i * kSampleThreads) * kVec);
      const uint32_t words[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
      float v[kVec];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 4) {
          v[j] = keep(__uint_as_float(words[j]), best);
        } else {
          v[2 * j] = keep(__uint_as_float(words[j] << 16), best);
          v[2 * j + 1] = keep(__uint_as_float(words[j] & 0xFFFF0000u), best);
        }
      }
#pragma unroll
      for (int j = 0; j < kVec / 4; ++j)
        dst[j] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
    }
  }
  const int rest = n - vecs * kVec;  // before and behind the vectors
  if (threadIdx.x < rest) {
    const int i = threadIdx.x < head ? threadIdx.x : threadIdx.x + vecs * kVec;
    x[i] = keep((float)src[i], best);
  }
  return best;
}

template <typename T>
__global__ void __launch_bounds__(kSampleThreads, 2) sample_kernel(const SampleParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  SampleShared& sh = *reinterpret_cast<SampleShared*>(smem);
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), blocks = (int)cluster.num_blocks();
  const int row_id = blockIdx.x / blocks;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;

  Row row;
  row.base = min(p.vocab, rank * p.slice);
  row.n = min(p.vocab - row.base, p.slice);
  row.chunk = (row.n + kPad - 1) / kPad * (kPad / kSampleWarps);

  const float temperature = p.temperature ? __ldg(p.temperature + row_id) : p.temperature_v;
  const int top_k = p.top_k ? __ldg(p.top_k + row_id) : p.top_k_v;
  const float top_p = p.top_p ? __ldg(p.top_p + row_id) : p.top_p_v;
  const float min_p = p.min_p ? __ldg(p.min_p + row_id) : p.min_p_v;
  const float u = __ldg(p.uniforms + row_id);

  // the row's tokens into shared memory, and the largest
  const T* src = static_cast<const T*>(p.logits) + (size_t)row_id * p.row_stride + row.base;
  float* x = reinterpret_cast<float*>(smem + sizeof(SampleShared)) + ((4 - head_of(src)) & 3);
  row.x = x;
  clear_bins<true>(sh);
  if (threadIdx.x < kPowers) sh.power[threadIdx.x] = exp2((double)threadIdx.x / kPowers + kWeightBits);
  if (threadIdx.x < 2) sh.list_n[threadIdx.x] = 0u;
  float best = load_row<T>(src, row.n, x);
  for (int i = row.n + threadIdx.x; i < row.chunk * kSampleWarps; i += kSampleThreads) x[i] = -INFINITY;
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, m));
  if (lane == 0) sh.warp_best[warp] = best;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < kSampleWarps; ++i) best = fmaxf(best, sh.warp_best[i]);
    sh.best = best;
  }
  cluster.sync();
  best = lane < blocks ? *cluster.map_shared_rank(&sh.best, lane) : -INFINITY;
#pragma unroll
  for (int m = 4; m > 0; m >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, m));
  best = __shfl_sync(0xffffffffu, best, 0);
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
      sh.first = first;
    }
    cluster.sync();
    if (rank == 0 && threadIdx.x == 0) {
      for (int r = 1; r < blocks; ++r) first = min(first, *cluster.map_shared_rank(&sh.first, r));
      const bool none = best == -INFINITY;
      p.ids[row_id] = none ? -1 : first;
      if (p.logprobs) p.logprobs[row_id] = none ? -INFINITY : 0.0f;
    }
    cluster.sync();  // no block leaves while another reads its shared memory
    return;
  }

  Weigher weigh;
  weigh.set(sh.power, best, temperature, min_p);
  // 2047 linear bins over the range of logits whose weight is not zero, one for the rest.  Above
  // zero also at an infinite temperature: logits that lie infinitely far apart (FP32's range, or
  // one of them infinite) then fall into the last bin, where zero would make their bin NaN.
  row.scale = fminf(fmaxf((float)(2047.0 / 32.3) / temperature, FLT_MIN), 3.0e38f);

  Kept kept;
  kept.x = -FLT_MAX;  // every logit above -inf
  kept.last = 0x7FFFFFFF;
  bool all = true;               // as long as that is so, the weights alone tell

  // ---- top-k ------------------------------------------------------------------------------
  const int from = warp * row.chunk;
  if (top_k > 0 && top_k < p.vocab) {
    unsigned beyond = 0u;  // in the last bin, where most tokens are: counted apart
    for (int i = from + lane; i < from + row.chunk; i += 32 * kWide) {
      float v[kWide];
#pragma unroll
      for (int j = 0; j < kWide; ++j) v[j] = x[i + 32 * j];
#pragma unroll
      for (int j = 0; j < kWide; ++j) {
        const int b = row.bin(v[j]);
        if (v[j] == -INFINITY) continue;
        if (b == kBins - 1) ++beyond;
        else atomicAdd(&sh.part[0][b], 1u);
      }
    }
    beyond = __reduce_add_sync(0xffffffffu, beyond);
    if (lane == 0 && beyond) atomicAdd(&sh.part[0][kBins - 1], beyond);
    u64 live;
    const Found found = find_bin<false>(sh, cluster, [&](u64) { return (u64)top_k; }, live);
    if (found.bin >= 0 && live > (u64)top_k) {
      if (found.before + found.amount <= (u64)kList) {
        // all tokens up to the end of this bin: the first block of the cluster goes on alone
        for (int i = from + lane; i < from + row.chunk; i += 32 * kWide) {
          float v[kWide];
          bool chosen[kWide], any = false;
#pragma unroll
          for (int j = 0; j < kWide; ++j) {
            v[j] = x[i + 32 * j];
            chosen[j] = v[j] != -INFINITY && row.upto_bin(v[j], found.bin);
            any |= chosen[j];
          }
          if (!__any_sync(0xffffffffu, any)) continue;
#pragma unroll
          for (int j = 0; j < kWide; ++j)
            append(chosen[j], place(descending_key(v[j]), row.base + i + 32 * j), sh.list,
                   &sh.list_n[0]);
        }
        cluster.sync();  // the lists are complete, and the histogram has been read
        u64* merged = reinterpret_cast<u64*>(&sh.part[2][0]);
        if (rank == 0) {
          const int n = (int)merge_lists(sh, cluster, &sh.list_n[0], merged);
          cluster.sync();
          finish_list(sh, p, row_id, weigh, merged, n, top_k, top_p, u);
        } else {
          cluster.sync();  // no block leaves while another reads its shared memory
        }
        return;
      }
      kept = select<false>(sh, cluster, row, weigh, kept, found.bin, (u64)top_k - found.before);
      all = false;
    } else {
      cluster.sync();  // the histogram has been read
    }
    clear_bins<true>(sh);
    __syncthreads();
  }

  // ---- weights; top-p ---------------------------------------------------------------------
  const bool nucleus = top_p < 1.0f;
  u64 sum = 0ull;
  for (int i = from + lane; i < from + row.chunk; i += 32 * kWide) {
    float v[kWide];
    u64 w[kWide];
    int bin[kWide];
#pragma unroll
    for (int j = 0; j < kWide; ++j) {
      v[j] = x[i + 32 * j];
      w[j] = weigh(v[j], bin[j]);
    }
    if (!all) {
#pragma unroll
      for (int j = 0; j < kWide; ++j)
        if (!kept.holds(v[j], row.base + i + 32 * j)) w[j] = 0ull;
    }
#pragma unroll
    for (int j = 0; j < kWide; ++j) sum += w[j];
    if (nucleus) {
#pragma unroll
      for (int j = 0; j < kWide; ++j)
        if (w[j]) add_mass<kBins>(sh.part[0], bin[j], w[j]);
    }
  }
  u64 total = 0ull;
  if (nucleus) {
    const Found found =
        find_bin<true>(sh, cluster, [&](u64 all) { return mass_needed(top_p, all); }, total);
    const u64 need = mass_needed(top_p, total);
    if (found.bin >= 0 && need < total) {
      kept = select<true>(sh, cluster, row, weigh, kept, found.bin, need - found.before);
      all = false;
      sum = sum_kept(sh, row, weigh, kept);
    }
  }
  sum = warp_total(sum);
  if (lane == 0) sh.warp_sum[warp] = sum;
  u64 before;
  total = cluster_total(sh, cluster, before);

  // ---- draw -------------------------------------------------------------------------------
  const u64 target = draw_target(u, total);
  cluster.sync();  // no block leaves while another reads its shared memory
  if (before <= target && target < before + sh.sum) {  // one block of the cluster
    // the warp whose tokens hold the target; its tokens, one per thread
    int owner = 0;
    for (; owner < kSampleWarps - 1; ++owner) {
      const u64 w = sh.warp_sum[owner];
      if (target < before + w) break;
      before += w;
    }
    const int first = owner * row.chunk, end = min(row.n, first + row.chunk);
    for (int start = first; start < end; start += kSampleThreads) {
      const int i = start + threadIdx.x;
      const float v = i < end ? x[i] : -INFINITY;
      u64 w = weigh(v);
      if (!all && !kept.holds(v, row.base + i)) w = 0ull;
      u64 upto = inclusive_scan(w);
      __syncthreads();  // the sums before have been read
      if (lane == 31) sh.warp_sum[warp] = upto;
      __syncthreads();
      upto += before;
      for (int k = 0; k < warp; ++k) upto += sh.warp_sum[k];
      if (w && upto - w <= target && target < upto)
        store_result(p, row_id, weigh, row.base + i, v, total);
      for (int k = 0; k < kSampleWarps; ++k) before += sh.warp_sum[k];
    }
  }
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
  // Blocks of a row: as many as keep a block's tokens at 16384 or fewer, so that two blocks share
  // an SM (64 rows of 129280 mixed: 48.5 us against 55.6 us with 32768); and while SMs are left
  // and a block has more than 1536 tokens, more (one row of 32000, top-p: 14.4 us with eight
  // against 22.4 us with two; of 8000: 13.1 us with eight against 14.2 us with two).
  int blocks = 1;
  while (blocks < kMaxCluster && ((vocab + blocks - 1) / blocks > 16384 ||
                                  ((long long)rows * blocks * 2 <= sm_count && vocab / blocks > 1536)))
    blocks *= 2;
  p.slice = (vocab + blocks - 1) / blocks;
  const size_t bytes = sizeof(SampleShared) + (size_t)((p.slice + kPad - 1) / kPad * kPad + 3) * sizeof(float);
  const void* kernel = logits_f32 ? (const void*)sample_kernel<float>
                                  : (const void*)sample_kernel<__nv_bfloat16>;
  static std::atomic<uint64_t> allowed[2];
  cudaError_t err = allow_shared_memory(kernel, allowed[logits_f32]);
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
