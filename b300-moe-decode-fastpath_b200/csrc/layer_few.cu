// The whole expert layer for at most eight tokens in ONE kernel:
//   z = x Wr^T,  top-k of z,  p = softmax of the chosen z,
//   a[t,k] = p * silu(gate_e x_t) * (up_e x_t),   out[t] = sum_k down_e a[t,k]
// The regular path (b200moe_forward) needs the router's product and top-k in front and is four
// to five kernels; with a few tokens the launches between them cost more than the arithmetic.
// No counterpart in the reference.
//
// What bounds it.  Every weight row of an expert in use is read once and multiplied with at most
// eight columns: 1 to 8 multiply-adds a byte, so HBM bounds the large layers and fixed costs the
// small ones.  One block of 16 warps per SM stays for the whole call (cooperative launch) and the
// three phases -- logits, gate+up, down -- are separated by two grid barriers.
//
// Split.  Rows of the weight matrices are dealt out evenly to the blocks: block b takes
// gate/up column pairs [b P / G, (b+1) P / G) of the P = (experts in use) * I pairs, and output
// rows [b H / G, (b+1) H / G) of the down projection, for which it adds up all experts itself --
// no partial sums in memory, no atomics on them, and sums in an order that only the shape and
// the routing decide.  Inside the block the reduction dimension is cut into units of 128 bytes a
// row, dealt to the warps in turn; the warps' partial tiles are added in shared memory.
//
// The tile.  A warp multiplies 16 or 32 rows by 8 columns with mma.m16n8k16.  The column index
// is the token, for gate/up and down alike, so the token operand needs no gathering: for gate+up
// all tokens are multiplied and only those routed to the expert are kept; for down the columns
// of the other tokens (zero, with E4M3 weights a copy) are masked when a unit's tile is added: a
// weight of NaN or infinity reaches only the tokens routed to it.  mma.sync and not tcgen05: 8
// columns of useful work leave the tensor pipe idle either way, and operands that arrive in
// registers need no descriptor, no tensor memory and no block-wide handshake per tile.
//   Measured (weights from HBM, in a graph; copy rate 6.56 TB/s): H = 2048, I = 768, 128 experts,
// top-8: 25.3 us for one token (floor 11.6: 7 us go by before the first weight, 3 us at the second
// barrier), 98 to 106 us for eight (73.9; SMs end gate+up up to 9 us apart); H = 4096, I = 14336,
// 8 experts, top-2: 118 us (107) and 422 us (412); E4M3 74.5 us (37) and 246 us (206) at the two
// shapes for eight tokens, 106 us (68) for three with H = I = 2880, 32 experts, top-8, where the
// 20 output rows of a block fill 32 rows of MMAs (without the MMAs 16 us less, without loading
// activations 9 us less).  The router's product, top-k and the regular path, in a graph: 45, 99,
// 127 and 421 us; E4M3 230 us for eight tokens, 104 us for three, 34 us against 23 us for one token
// at the first shape, 82 us against 72 us at the second.
//
// Loads.  Each lane copies with cp.async the very 16 bytes that it will use as fragments (rows
// g and g+8, four lanes side by side in a row), into a ring of its warp in shared memory, and
// reads them back itself: no barrier between producer and consumer.  Any permutation of the
// reduction dimension is allowed as long as both operands share it, which is why a lane's 16
// consecutive bytes can serve as its part of the fragment.
// The ring does not stop at the grid barrier: while a block waits for the activations, its
// warps' first down tiles are already on their way.
//
// Precision.  Logits are summed with the rounding errors of all additions kept (two-sum), so
// that they are good to about 2^-48: experts that lie next to one another at the border are
// told apart as in 64 bits.  Products and sums are FP32.  With BF16 weights the activations are
// held as the sum of two BF16 numbers (16 significant bits), as the regular path holds them.
// With E4M3 weights both operands of the MMAs are FP16: one conversion instruction turns two
// codes into two FP16 numbers exactly (to BF16 it takes five), token rows are multiplied by a
// power of two that brings their largest element to [2^13, 2^14) and fit exactly, and
// activations, scaled the same way, keep 11 significant bits (the regular path: twelve), which
// is eight times finer than the BF16 rounding of the result.
#include <cuda_fp16.h>

#include "common.cuh"

namespace b200moe {

namespace {

constexpr int kFewWarps = 16;
constexpr int kFewThreads = kFewWarps * 32;
constexpr int kFewSlots = kFewMaxTokens * 8;  // experts in use, at most; also assignments
// Stages of a warp's ring.  Two, 64 KB (32 rows a stage: 128 KB) of an SM in flight, cover the
// latency of HBM; with a third the copies of all warps queue longer in front of the loads of
// activations (BF16, 8 tokens, H = 4096, I = 14336, 8 experts: 422 us against 434 us with three or
// four; H = 2048, I = 768, 128 experts: 97.6 against 98.8 us; but one token, H = I = 2880:
// 84.5 against 79.5 us).
constexpr int kFewStages = 2;

struct FewParams {
  const __nv_bfloat16* x;
  const void* router;
  const uint8_t* gate_up;   // bytes; BF16 or E4M3
  const uint8_t* down;
  const float* gate_up_scale;
  const float* down_scale;
  int tokens, hidden, inter, experts, top_k;
  int x_pitch;              // bytes of a token row in shared memory
  unsigned long long inter_inverse;  // ceil(2^40 / inter)
  double* logits;           // [tokens, experts]
  uint32_t* act_max;        // [tokens * top_k]  E4M3 only: bit pattern of max |activation|
  uint16_t* act_hi;         // [tokens * top_k, inter]  BF16 high parts; E4M3: FP32, in the
  int act_pitch;            //   order of act_place, `act_pitch` elements a row
  uint16_t* act_lo;         // BF16 low parts
  __nv_bfloat16* out;
  int64_t* ids_out;
  float* weights_out;
  unsigned int* sync;       // three counters, zero between calls
  uint32_t* status;
};

template <int SUBS>
struct alignas(128) FewShared {
  float red[kFewWarps][SUBS * 128];
  double logit[kFewWarps];
  float weight[kFewSlots];              // by assignment
  int expert[kFewSlots];                // by slot (experts in use, ascending)
  int chosen[kFewSlots];                // expert by assignment
  uint32_t act_max[kFewSlots];          // by assignment, of this block's activations
  uint32_t used[B200MOE_MAX_EXPERTS / 32];  // experts in use, one bit each
  signed char assign[kFewSlots][kFewMaxTokens];  // assignment of (slot, token), or below zero
  uint32_t members[kFewSlots];          // tokens of a slot, one bit each
  float x_unscale[kFewMaxTokens];       // E4M3: 2^-s of the token rows
  float a_scale[kFewSlots], a_unscale[kFewSlots];  // E4M3: 2^s and 2^-s of the activation rows
  uint32_t x_max[kFewMaxTokens];
  int abort;
};

// 16 bytes, or with bytes == 0 a piece of zeros, for which nothing is read and `src` (which may
// lie behind the end of its matrix) is replaced by an address inside
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes,
                                           const void* inside) {
  src = bytes ? src : inside;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
template <bool F16>
__device__ __forceinline__ void mma_16x8x16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                            uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (F16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// four E4M3 codes -> two FP16 pairs, exactly
__device__ __forceinline__ void e4m3x4_to_f16x4(uint32_t w, uint32_t& p01, uint32_t& p23) {
  asm("{\n\t.reg .b16 lo, hi;\n\t"
      "mov.b32 {lo, hi}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, lo;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, hi;\n\t}"
      : "=r"(p01), "=r"(p23)
      : "r"(w));
}

// One 16-byte piece of rows g and g+8 times the token operand of the same elements: 8 BF16
// elements (two MMAs, `b` 4 words) or 16 E4M3 elements (four MMAs, `b` 8 words).
template <bool FP8>
__device__ __forceinline__ void multiply_piece(float (&c)[4], const uint4& top, const uint4& bottom,
                                               const uint32_t* b) {
  const uint32_t t[4] = {top.x, top.y, top.z, top.w};
  const uint32_t u[4] = {bottom.x, bottom.y, bottom.z, bottom.w};
  if constexpr (FP8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t t01, t23, u01, u23;
      e4m3x4_to_f16x4(t[i], t01, t23);
      e4m3x4_to_f16x4(u[i], u01, u23);
      mma_16x8x16<true>(c, t01, u01, t23, u23, b[2 * i], b[2 * i + 1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      mma_16x8x16<false>(c, t[2 * i], u[2 * i], t[2 * i + 1], u[2 * i + 1], b[2 * i], b[2 * i + 1]);
  }
}

// Where element `col` of an FP32 activation row lies.  The down projection's lane t of four takes
// elements 16 t .. 16 t + 15 of each run of 64, four at a time: with the fours of the four lanes
// side by side one load reads whole sectors; in plain order it reads half of each, and every
// sector is fetched twice (8 tokens, H = 4096, I = 14336, 8 experts: 284 -> 263 us; H = 2048,
// I = 768, 128 experts: 99 -> 81 us).
__device__ __forceinline__ int act_place(int col) {
  return (col & ~63) | ((col & 12) << 2) | ((col >> 2) & 12) | (col & 3);
}

// Grid barrier in two halves: arrive (one thread, for the stores that come before it), then wait
// (the block; bounded, after that it goes on to its end without further work).  The counters are
// compared as signed numbers: with one that starts below zero (a scratch that was not cleared)
// no block passes, all give up, and the last one leaves the counters at zero for the next call.
__device__ __forceinline__ void grid_arrive(unsigned int* counter) {
  asm volatile("fence.acq_rel.gpu;" ::: "memory");
  asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(counter) : "memory");
}
__device__ __forceinline__ bool grid_wait(unsigned int* counter, uint32_t* status, int* abort) {
  if (threadIdx.x == 0) {
    const uint64_t t0 = global_timer_ns();
    uint32_t spins = 0;
    while (true) {
      unsigned int seen;
      asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(seen) : "l"(counter) : "memory");
      if ((int)seen >= (int)gridDim.x) break;
      if ((++spins & 255u) == 0u && global_timer_ns() - t0 > 5ull * kPipeWaitLimitNs) {
        atomicOr(status, B200MOE_STATUS_PIPE_TIMEOUT);
        *abort = 1;
        break;
      }
    }
    __threadfence();
  }
  __syncthreads();
  return *abort == 0;
}

// s + p with the rounding error of the addition collected in e
__device__ __forceinline__ void two_sum(float& s, float& e, float p) {
  const float t = __fadd_rn(s, p);
  const float z = __fsub_rn(t, s);
  e = __fadd_rn(e, __fadd_rn(__fsub_rn(s, __fsub_rn(t, z)), __fsub_rn(p, z)));
  s = t;
}

// Order as integers: larger values larger, NaN above every number, 0 and -0 equal, nothing at 0
__device__ __forceinline__ unsigned long long order_of(double v) {
  const unsigned long long bits = (unsigned long long)__double_as_longlong(v + 0.0);
  if (v != v) return ~0ull;
  return (bits >> 63) ? ~bits : (bits | 0x8000000000000000ull);
}
__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t bits = __float_as_uint(v + 0.0f);
  if (v != v) return ~0u;
  return (bits >> 31) ? ~bits : (bits | 0x80000000u);
}

// The power of two that brings a row with the largest magnitude `bits` (an FP32 pattern) to
// [2^13, 2^14): no finite element overflows FP16, and elements down to 2^-27 of the largest keep
// the eight bits of BF16.  A row of zeros: 1.  A row with infinities or NaN: 2^-114, under which
// its finite elements stay finite.
__device__ __forceinline__ float row_scale(uint32_t bits) {
  if (bits == 0u) return 1.0f;
  const int e = (int)(bits >> 23);            // biased exponent, 255 for inf and NaN
  int s = e == 255 ? -114 : 13 + 127 - e;
  s = s > 126 ? 126 : s;                      // subnormal rows
  return __uint_as_float((uint32_t)(s + 127) << 23);
}

template <bool ROUTER_F32>
struct RouterVec {  // eight router weights in flight
  uint4 raw[ROUTER_F32 ? 2 : 1];
  __device__ __forceinline__ void load(const void* router, size_t at) {
    if constexpr (ROUTER_F32) {
      const uint4* src = reinterpret_cast<const uint4*>(static_cast<const float*>(router) + at);
      raw[0] = __ldg(src);
      raw[1] = __ldg(src + 1);
    } else {
      raw[0] = __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(router) + at));
    }
  }
  __device__ __forceinline__ void get(float (&w)[8]) const {
    if constexpr (ROUTER_F32) {
      const uint32_t r[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w,
                             raw[1].x, raw[1].y, raw[1].z, raw[1].w};
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = __uint_as_float(r[i]);
    } else {
      const uint32_t r[4] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[2 * i] = __uint_as_float(r[i] << 16);
        w[2 * i + 1] = __uint_as_float(r[i] & 0xFFFF0000u);
      }
    }
  }
};

// Logits of the experts b, b + G, ...  Warps are dealt to (token, slice of the row): with T
// tokens rounded up to a power of two P, warp w takes token w mod P and slice w / P of 16 / P.
// x arrives in shared memory by copies that the caller has under way; each lane's first router
// vector is loaded meanwhile.
template <bool ROUTER_F32, typename Shared>
__device__ __forceinline__ void router_logits(const FewParams& p, Shared& sh,
                                              const uint8_t* x_rows) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int shift = p.tokens > 4 ? 3 : p.tokens > 2 ? 2 : p.tokens > 1 ? 1 : 0;
  const int token = warp & ((1 << shift) - 1), slices = kFewWarps >> shift;
  const int vecs = p.hidden / 8, from = (warp >> shift) * 32 + lane;
  const bool busy = token < p.tokens;
  const uint8_t* x = x_rows + token * p.x_pitch;
  RouterVec<ROUTER_F32> vec;
  if (busy && blockIdx.x < p.experts && from < vecs)
    vec.load(p.router, (size_t)blockIdx.x * p.hidden + 8 * from);
  cp_async_wait<0>();
  __syncthreads();
#pragma unroll 1
  for (int e = blockIdx.x; e < p.experts; e += gridDim.x) {
    float s = 0.0f, err = 0.0f;
    if (busy) {
#pragma unroll 1
      for (int v = from; v < vecs; v += 32 * slices) {
        float w[8];
        vec.get(w);
        int ahead = v + 32 * slices, ahead_e = e;
        if (ahead >= vecs) {
          ahead = from;
          ahead_e += gridDim.x;
        }
        if (ahead_e < p.experts) vec.load(p.router, (size_t)ahead_e * p.hidden + 8 * ahead);
        const uint4 q = *reinterpret_cast<const uint4*>(x + 16 * v);
        const uint32_t words[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float xv = (i & 1) ? __uint_as_float(words[i / 2] & 0xFFFF0000u)
                                   : __uint_as_float(words[i / 2] << 16);
          const float prod = __fmul_rn(w[i], xv);  // exact for BF16 x BF16
          if constexpr (ROUTER_F32) err += __fmaf_rn(w[i], xv, -prod);
          two_sum(s, err, prod);
        }
      }
    }
    // an error term of an overflowed or NaN sum is NaN itself: the sum alone tells
    double d = (double)s;
    if (isfinite(s)) d += (double)err;
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) d += __shfl_xor_sync(0xffffffffu, d, m);
    if (lane == 0) sh.logit[warp] = d;
    __syncthreads();
    if (threadIdx.x < p.tokens) {  // all in warp 0, which arrives at the barrier
      d = 0.0;
      for (int i = 0; i < slices; ++i) d += sh.logit[(i << shift) + threadIdx.x];
      __stcg(p.logits + (size_t)threadIdx.x * p.experts + e, d);
    }
    if (e + gridDim.x < p.experts) __syncthreads();
  }
}

// Top-k of every token, one warp each, then the list of experts in use.  Every block does this
// for itself from the logits.  The candidates are compared as FP32, which rounds the 64-bit logits
// monotonically; only where two are equal as FP32 do the 64 bits decide, and then the lower id.
template <typename Shared>
__device__ __forceinline__ void choose_experts(const FewParams& p, Shared& sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (warp < p.tokens) {
    double v[8];
    uint32_t key[8];  // 0: taken or absent
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = lane + 32 * i;
      v[i] = e < p.experts ? __ldcg(p.logits + (size_t)warp * p.experts + e) : 0.0;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) key[i] = lane + 32 * i < p.experts ? order_of((float)v[i]) : 0u;
#pragma unroll 1
    for (int k = 0; k < p.top_k; ++k) {
      uint32_t best = key[0];
#pragma unroll
      for (int i = 1; i < 8; ++i) best = max(best, key[i]);
      best = __reduce_max_sync(0xffffffffu, best);
      // how many keys are the best one (upper half), and the sum of their ids: of one, its id
      unsigned id = 0u;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (key[i] == best) id += 0x10000u + (unsigned)(lane + 32 * i);
      const bool held = id != 0u;
      id = __reduce_add_sync(0xffffffffu, id);
      if (id >> 16 == 1u) {
        id &= 0xffffu;
      } else {
        int at = 0;
        unsigned long long most = 0ull;  // among the equal ones, by all 64 bits
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (key[i] == best && order_of(v[i]) > most) {
            most = order_of(v[i]);
            at = i;
          }
        const unsigned hi = __reduce_max_sync(0xffffffffu, (unsigned)(most >> 32));
        const bool in_hi = (unsigned)(most >> 32) == hi;
        const unsigned lo = __reduce_max_sync(0xffffffffu, in_hi ? (unsigned)most : 0u);
        const bool in_both = held && in_hi && (unsigned)most == lo;
        id = __reduce_min_sync(0xffffffffu, in_both ? (unsigned)(lane + 32 * at) : 0xffffffffu);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if ((unsigned)(lane + 32 * i) == id) key[i] = 0u;
      if (lane == k) sh.chosen[warp * p.top_k + k] = (int)id;
    }
    __syncwarp();
    if (lane < p.top_k) {
      const int id = sh.chosen[warp * p.top_k + lane];
      atomicOr(&sh.used[id >> 5], 1u << (id & 31));
    }
  }
  __syncthreads();
  if (threadIdx.x < p.tokens * p.top_k) {  // number the experts in use in ascending order
    const int a = threadIdx.x, e = sh.chosen[a], t = a / p.top_k;
    int slot = __popc(sh.used[e >> 5] & ((1u << (e & 31)) - 1u));
#pragma unroll
    for (int i = 0; i < B200MOE_MAX_EXPERTS / 32; ++i)
      if (i < e >> 5) slot += __popc(sh.used[i]);
    sh.expert[slot] = e;
    sh.assign[slot][t] = (signed char)a;
    atomicOr(&sh.members[slot], 1u << t);
    if (blockIdx.x == 0 && p.ids_out) p.ids_out[a] = e;
  }
  __syncthreads();
}

// Softmax over a token's chosen logits, in its warp.
template <typename Shared>
__device__ __forceinline__ void softmax_weights(const FewParams& p, Shared& sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (warp >= p.tokens) return;
  const int a = warp * p.top_k + lane;
  double mine = 0.0;
  if (lane < p.top_k) mine = __ldcg(p.logits + (size_t)warp * p.experts + sh.chosen[a]);
  const double top = __shfl_sync(0xffffffffu, mine, 0);
  float w = lane < p.top_k ? expf((float)(mine - top)) : 0.0f;
  float sum = w;
#pragma unroll
  for (int m = 4; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
  if (lane < p.top_k) {
    w /= sum;
    sh.weight[a] = w;
    if (blockIdx.x == 0 && p.weights_out) p.weights_out[a] = w;
  }
}

// What one block does, and the order in which a warp's ring is filled: first the gate/up tiles,
// then the down tiles.  Both sides of the ring -- the copies and the products -- walk it.
// TILES: down tiles that share one load of the activations.
template <bool FP8, int SUBS, int TILES>
struct FewWork {
  static constexpr int kUnit = FP8 ? 128 : 64;   // elements of a row in one stage (128 bytes)
  static constexpr int kPiece = FP8 ? 16 : 8;    // elements in 16 bytes
  static constexpr int kElem = FP8 ? 1 : 2;      // bytes of an element
  static constexpr int kStageBytes = SUBS * 2048;

  int row0, rows, down_tiles, down_height;       // down: this block's output rows
  int units_h, units_i;                          // stages along H; along I
  bool wide;                                     // down: a stage is 16 rows by two units
  int pair0, pairs, tiles, height;               // gate/up: this block's pairs, in equal tiles
  int slots;                                     // experts in use

  // what the dimensions alone say
  __device__ explicit FewWork(const FewParams& p) {
    row0 = (int)((unsigned)p.hidden * blockIdx.x / gridDim.x);
    rows = (int)((unsigned)p.hidden * (blockIdx.x + 1u) / gridDim.x) - row0;
    down_tiles = (rows + 16 * SUBS - 1) / (16 * SUBS);
    down_height = down_tiles ? (rows + down_tiles - 1) / down_tiles : 0;
    // a block with few output rows fills the stage with a second unit of them (E4M3, 4 tokens,
    // H = 2048, I = 2880: 75 us, with half the stage empty 86 us)
    wide = SUBS == 2 && down_height <= 16;
    const int unit = wide ? 2 * kUnit : kUnit;
    units_h = (p.hidden + kUnit - 1) / kUnit;
    units_i = (p.inter + unit - 1) / unit;
  }
  // and what the routing adds; used: one bit per expert in use
  __device__ void deal_pairs(const FewParams& p, const uint32_t* used) {
    slots = 0;
#pragma unroll
    for (int i = 0; i < B200MOE_MAX_EXPERTS / 32; ++i) slots += __popc(used[i]);
    const unsigned total = (unsigned)slots * p.inter;   // at most 2^22, times the grid < 2^32
    pair0 = (int)(total * blockIdx.x / gridDim.x);
    pairs = (int)(total * (blockIdx.x + 1u) / gridDim.x) - pair0;
    tiles = (pairs + 8 * SUBS - 1) / (8 * SUBS);
    height = tiles ? (pairs + tiles - 1) / tiles : 0;
  }
  // the expert (by slot) of a gate/up pair: pair / inter, exact for pairs below 2^24
  static __device__ __forceinline__ int slot_of(const FewParams& p, int pair) {
    return (int)(((unsigned long long)(unsigned)pair * p.inter_inverse) >> 40);
  }
};

// Fills the ring: one stage per call, in order.
template <bool FP8, int SUBS, int TILES, typename Shared>
struct FewProducer {
  using Work = FewWork<FP8, SUBS, TILES>;
  const FewParams& p;
  const Shared& sh;
  const Work& w;
  uint32_t dst, ring_end;
  const uint8_t* top[SUBS];    // gate/up: this lane's gate rows, first piece
  const uint8_t* base;         // down: this lane's row g of the group's first tile, first piece
  size_t up_bytes;             // gate row -> up row of the same column
  int ok[SUBS];                // gate/up: 16 where the row exists, else 0
  unsigned tail;               // pieces that exist in the last unit of a row, one bit each
  int warp, lane;
  int tile = 0;                // gate/up: tile; down: first tile of the group
  int unit;                    // gate/up: unit of the tile; down: unit of the expert
  int slot = 0, sub = 0;       // down: expert, tile within the group
  bool down = false, done = false;

  __device__ FewProducer(const FewParams& p_, const Shared& sh_, const Work& w_, uint32_t ring,
                         int warp_, int lane_)
      : p(p_), sh(sh_), w(w_), dst(ring), ring_end(ring + kFewStages * Work::kStageBytes), warp(warp_),
        lane(lane_), unit(warp_) {
    up_bytes = (size_t)p.inter * p.hidden * Work::kElem;
    set_tail(p.hidden, w.units_h, 1);
    enter_gate();
  }
  // pieces 2 s and 2 s + 1 of a stage are those of sub-tile s, or, where a stage holds `units` =
  // 2 units, of the unit s
  __device__ __forceinline__ void set_tail(int length, int count, int units) {
    tail = 0u;
#pragma unroll
    for (int i = 0; i < 2 * SUBS; ++i) {
      const int k = (count - 1) * units * Work::kUnit + (lane & 3) * Work::kPiece +
                    (i & 1) * (Work::kUnit / 2) + (units == 2 ? (i >> 1) * Work::kUnit : 0);
      if (k < length) tail |= 1u << i;
    }
  }
  // moves on to the next gate/up tile that has a unit for this warp
  __device__ __forceinline__ void enter_gate() {
    while (unit >= w.units_h && tile < w.tiles) {
      unit -= w.units_h;
      ++tile;
    }
    if (tile >= w.tiles) {
      down = true;
      tile = 0;
      unit = warp;
      set_tail(p.inter, w.units_i, w.wide ? 2 : 1);
      done = w.down_tiles == 0;
      enter_down();
      return;
    }
#pragma unroll
    for (int s = 0; s < SUBS; ++s) {
      const int i = s * 8 + (lane >> 2), local = tile * w.height + i;
      const bool live = i < w.height && local < w.pairs;
      ok[s] = live ? 16 : 0;
      const int pair = w.pair0 + (live ? local : 0);
      const int sl = Work::slot_of(p, pair);
      const size_t row = (size_t)sh.expert[sl] * 2 * p.inter + (pair - sl * p.inter);
      top[s] = p.gate_up + row * p.hidden * Work::kElem + (lane & 3) * 16;
    }
  }
  // moves on to the expert that holds this warp's next unit
  __device__ __forceinline__ void enter_down() {
    while (!done && unit >= w.units_i) {
      unit -= w.units_i;
      if (++slot == w.slots) {
        slot = 0;
        unit = warp;
        tile += TILES;
        done = tile >= w.down_tiles;
      }
    }
    if (done) return;
    const size_t row = (size_t)sh.expert[slot] * p.hidden + w.row0 + tile * w.down_height + (lane >> 2);
    base = p.down + row * p.inter * Work::kElem + (lane & 3) * 16;
  }
  __device__ __forceinline__ void copy(uint32_t to, const uint8_t* from, bool piece0, bool piece1,
                                       const uint8_t* inside) {
    cp_async16(to, from, piece0 ? 16 : 0, inside);
    cp_async16(to + 512, from + 64, piece1 ? 16 : 0, inside);
  }
  __device__ __forceinline__ void next() {
    if (!down) {
      const unsigned m = unit == w.units_h - 1 ? tail : 3u;
#pragma unroll
      for (int s = 0; s < SUBS; ++s) {
        if (s * 8 >= w.height) break;
        const uint8_t* a = top[s] + unit * 128;
        copy(dst + s * 2048, a, ok[s] && (m & 1u), ok[s] && (m & 2u), p.gate_up);
        copy(dst + s * 2048 + 1024, a + up_bytes, ok[s] && (m & 1u), ok[s] && (m & 2u), p.gate_up);
      }
      unit += kFewWarps;
      if (unit >= w.units_h) enter_gate();
    } else if (!done) {
      const unsigned m = unit == w.units_i - 1 ? tail : 15u;
      const size_t stride8 = (size_t)p.inter * (8 * Work::kElem);
      const int row = (tile + sub) * w.down_height + (lane >> 2);
      const uint8_t* a = base + (size_t)(sub * w.down_height) * p.inter * Work::kElem +
                         unit * (w.wide ? 256 : 128);
#pragma unroll
      for (int s = 0; s < SUBS; ++s) {
        const int i = (w.wide ? 0 : s * 16) + (lane >> 2), r = row + (w.wide ? 0 : s * 16);
        const bool live = i < w.down_height && r < w.rows;
        const bool live8 = i + 8 < w.down_height && r + 8 < w.rows;
        const bool m0 = m & (1u << (2 * s)), m1 = m & (2u << (2 * s));
        copy(dst + s * 2048, a, live && m0, live && m1, p.down);
        copy(dst + s * 2048 + 1024, a + stride8, live8 && m0, live8 && m1, p.down);
        a += w.wide ? (size_t)128 : 2 * stride8;
      }
      if (++sub == TILES || tile + sub == w.down_tiles) {
        sub = 0;
        unit += kFewWarps;
        if (unit >= w.units_i) enter_down();
      }
    }
    cp_async_commit();  // an empty group when there is nothing left
    dst += Work::kStageBytes;
    if (dst == ring_end) dst -= kFewStages * Work::kStageBytes;
  }
};

template <bool FP8, bool ROUTER_F32, int SUBS, int TILES>
__global__ void __launch_bounds__(kFewThreads, 1) layer_few_kernel(const FewParams p) {
  using Work = FewWork<FP8, SUBS, TILES>;
  using Shared = FewShared<SUBS>;
  constexpr int kWords = FP8 ? 16 : 8;  // 32-bit words of the token operand in one unit
  extern __shared__ __align__(128) uint8_t smem[];
  Shared& sh = *reinterpret_cast<Shared*>(smem);
  uint8_t* x_rows = smem + sizeof(Shared);
  const uint32_t rings = smem_u32(x_rows) + (uint32_t)align_up((size_t)p.tokens * p.x_pitch, 128);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t4 = lane & 3;

  // token rows, zero up to the end of the last unit
  const int row_vecs = (p.hidden + Work::kUnit - 1) / Work::kUnit * Work::kUnit / 8;
  for (int t = 0; t < p.tokens; ++t)
    for (int v = threadIdx.x; v < row_vecs; v += kFewThreads)
      cp_async16(smem_u32(x_rows) + t * p.x_pitch + 16 * v, p.x + (size_t)t * p.hidden + 8 * v,
                 8 * v < p.hidden ? 16 : 0, p.x);
  cp_async_commit();
  if (blockIdx.x == 0) {
    if (threadIdx.x == 0) *p.status = 0u;
    if (FP8 && threadIdx.x < kFewSlots) p.act_max[threadIdx.x] = 0u;
  }
  if (threadIdx.x == 0) sh.abort = 0;
  if (threadIdx.x < kFewSlots) {
    sh.act_max[threadIdx.x] = 0u;
    sh.members[threadIdx.x] = 0;
  }
  if (threadIdx.x < kFewMaxTokens) {
    sh.x_max[threadIdx.x] = 0u;
    sh.used[threadIdx.x] = 0u;
  }
  static_assert(kFewMaxTokens == B200MOE_MAX_EXPERTS / 32, "one word per thread");
  (&sh.assign[0][0])[threadIdx.x] = -1;
  static_assert(kFewThreads == kFewSlots * kFewMaxTokens, "one entry per thread");
  router_logits<ROUTER_F32>(p, sh, x_rows);
  if (warp == 0) {  // the block's logits were stored by this warp
    __syncwarp();
    if (lane == 0) grid_arrive(p.sync);
  }
  Work w(p);

  if constexpr (FP8) {  // token rows to scaled FP16, in place, while the other blocks arrive
    const int vecs = row_vecs;
    __syncthreads();
    for (int t = 0; t < p.tokens; ++t) {
      uint32_t most = 0u;
      for (int v = threadIdx.x; v < vecs; v += kFewThreads) {
        const uint4 q = *reinterpret_cast<const uint4*>(x_rows + t * p.x_pitch + 16 * v);
        const uint32_t words[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) most = max(most, max(words[i] & 0x7FFFu, (words[i] >> 16) & 0x7FFFu));
      }
      most = __reduce_max_sync(0xffffffffu, most);
      if (lane == 0) atomicMax(&sh.x_max[t], most);
    }
    __syncthreads();
    for (int t = 0; t < p.tokens; ++t) {
      const float scale = row_scale(sh.x_max[t] << 16);
      if (threadIdx.x == 0) sh.x_unscale[t] = 1.0f / scale;
      for (int v = threadIdx.x; v < vecs; v += kFewThreads) {
        uint4* at = reinterpret_cast<uint4*>(x_rows + t * p.x_pitch + 16 * v);
        const uint4 q = *at;
        uint32_t words[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const __half2 h = __floats2half2_rn(__uint_as_float(words[i] << 16) * scale,
                                              __uint_as_float(words[i] & 0xFFFF0000u) * scale);
          words[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        *at = make_uint4(words[0], words[1], words[2], words[3]);
      }
    }
  }
  bool ok = grid_wait(p.sync, p.status, &sh.abort);

  if (ok) {
    choose_experts(p, sh);
    if constexpr (FP8) {  // a token that is not the expert's: ~(assignment of one that is)
      const int slot = threadIdx.x / kFewMaxTokens, t = threadIdx.x % kFewMaxTokens;
      const uint32_t members = sh.members[slot];
      if (members && !(members >> t & 1u))
        sh.assign[slot][t] = (signed char)~sh.assign[slot][__ffs(members) - 1];
    }
    w.deal_pairs(p, sh.used);
    uint32_t src = rings + warp * kFewStages * Work::kStageBytes + lane * 16;
    const uint32_t ring_end = src + kFewStages * Work::kStageBytes;
    FewProducer<FP8, SUBS, TILES, Shared> producer(p, sh, w, src, warp, lane);
#pragma unroll 1
    for (int i = 0; i < kFewStages; ++i) producer.next();
    softmax_weights(p, sh);

    // ---- gate + up -----------------------------------------------------------------
    const uint32_t x_lane = smem_u32(x_rows) + g * p.x_pitch + t4 * Work::kPiece * 2;
    int unit = warp;
#pragma unroll 1
    for (int tile = 0; tile < w.tiles; ++tile) {
      float c[SUBS][4];
#pragma unroll
      for (int s = 0; s < SUBS; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) c[s][i] = 0.0f;
#pragma unroll 1
      for (; unit < w.units_h; unit += kFewWarps) {
        uint32_t b[kWords];  // token operand: elements of both halves of the unit
#pragma unroll
        for (int i = 0; i < kWords / 4; ++i) {
          uint4 q = make_uint4(0u, 0u, 0u, 0u);
          if (g < p.tokens)
            q = lds128(x_lane + unit * Work::kUnit * 2 +
                       (FP8 ? (i / 2) * Work::kUnit + (i % 2) * 16 : i * Work::kUnit));
          b[4 * i] = q.x; b[4 * i + 1] = q.y; b[4 * i + 2] = q.z; b[4 * i + 3] = q.w;
        }
        cp_async_wait<kFewStages - 1>();
        uint4 a[SUBS][4];
#pragma unroll
        for (int s = 0; s < SUBS; ++s)
#pragma unroll
          for (int i = 0; i < 4; ++i) a[s][i] = lds128(src + s * 2048 + i * 512);
        producer.next();
        src += Work::kStageBytes;
        if (src == ring_end) src -= kFewStages * Work::kStageBytes;
#pragma unroll
        for (int s = 0; s < SUBS; ++s) {
          multiply_piece<FP8>(c[s], a[s][0], a[s][2], b);
          multiply_piece<FP8>(c[s], a[s][1], a[s][3], b + kWords / 2);
        }
      }
      unit -= w.units_h;
      __syncthreads();  // the sums of the tile before are read
      if (2 * t4 < p.tokens) {
#pragma unroll
        for (int s = 0; s < SUBS; ++s) {
          float* red = sh.red[warp] + s * 128 + 2 * t4;
          *reinterpret_cast<float2*>(red + g * 8) = make_float2(c[s][0], c[s][1]);
          *reinterpret_cast<float2*>(red + (g + 8) * 8) = make_float2(c[s][2], c[s][3]);
        }
      }
      __syncthreads();
      if (threadIdx.x < 64 * SUBS) {  // one column pair of one token each
        const int i = threadIdx.x >> 3, tok = threadIdx.x & 7;
        const int local = tile * w.height + i;
        if (i < w.height && local < w.pairs && tok < p.tokens) {
          const int pair = w.pair0 + local;
          const int slot = Work::slot_of(p, pair), col = pair - slot * p.inter;
          const int a = sh.assign[slot][tok];
          if (a >= 0) {
            const int at = (i >> 3) * 128 + (i & 7) * 8 + tok;
            float gate = 0.0f, up = 0.0f;
#pragma unroll
            for (int i2 = 0; i2 < kFewWarps; ++i2) {
              gate += sh.red[i2][at];
              up += sh.red[i2][at + 64];
            }
            if constexpr (FP8) {
              const float* s = p.gate_up_scale + (size_t)sh.expert[slot] * 2 * p.inter + col;
              gate *= __ldg(s) * sh.x_unscale[tok];
              up *= __ldg(s + p.inter) * sh.x_unscale[tok];
            }
            const float act = gate / (1.0f + expf(-gate)) * up * sh.weight[a];
            if constexpr (FP8) {
              reinterpret_cast<float*>(p.act_hi)[(size_t)a * p.act_pitch + act_place(col)] = act;
              atomicMax(&sh.act_max[a], __float_as_uint(act) & 0x7FFFFFFFu);
            } else {
              const __nv_bfloat16 high = __float2bfloat16_rn(act);
              const float rest = act - __bfloat162float(high);
              p.act_hi[(size_t)a * p.inter + col] = __bfloat16_as_ushort(high);
              p.act_lo[(size_t)a * p.inter + col] =
                  __bfloat16_as_ushort(__float2bfloat16_rn(isfinite(rest) ? rest : 0.0f));
            }
          }
        }
      }
    }
    if constexpr (FP8) {
      __syncthreads();
      if (threadIdx.x < p.tokens * p.top_k && sh.act_max[threadIdx.x])
        atomicMax(p.act_max + threadIdx.x, sh.act_max[threadIdx.x]);
    }
    __syncthreads();
    if (threadIdx.x == 0) grid_arrive(p.sync + 1);
    // the scales of this block's output rows, experts one after another, where the token rows were
    float* scales = reinterpret_cast<float*>(x_rows);
    if constexpr (FP8)
      for (int i = threadIdx.x; i < w.slots * w.rows; i += kFewThreads) {
        const int sl = i / w.rows;
        scales[i] = __ldg(p.down_scale + (size_t)sh.expert[sl] * p.hidden + w.row0 + (i - sl * w.rows));
      }
    ok = grid_wait(p.sync + 1, p.status, &sh.abort);
    if constexpr (FP8) {
      if (threadIdx.x < p.tokens * p.top_k) {
        const float scale = row_scale(__ldcg(p.act_max + threadIdx.x));
        sh.a_scale[threadIdx.x] = scale;
        sh.a_unscale[threadIdx.x] = 1.0f / scale;
      }
      __syncthreads();
    }

    // ---- down ----------------------------------------------------------------------
    const bool ragged = p.inter % (w.wide ? 2 * Work::kUnit : Work::kUnit) != 0;
#pragma unroll 1
    for (int first = 0; ok && first < w.down_tiles; first += TILES) {
      float total[TILES][SUBS][4];
#pragma unroll
      for (int r = 0; r < TILES; ++r)
#pragma unroll
        for (int s = 0; s < SUBS; ++s)
#pragma unroll
          for (int i = 0; i < 4; ++i) total[r][s][i] = 0.0f;
      int slot = 0, unit = warp;
#pragma unroll 1
      while (true) {
        while (unit >= w.units_i && slot < w.slots) {
          unit -= w.units_i;
          ++slot;
        }
        if (slot >= w.slots) break;
        const int a = sh.assign[slot][g];
        // the tokens of this lane's two columns
        const unsigned members = sh.members[slot] >> (2 * t4);
        float row_scales[TILES][SUBS][2];
        float u0 = 1.0f, u1 = 1.0f, scale = 1.0f;
        if constexpr (FP8) {
          const float* sc = scales + slot * w.rows + first * w.down_height + g;
#pragma unroll
          for (int r = 0; r < TILES; ++r)
#pragma unroll
            for (int s = 0; s < SUBS; ++s) {
              const int i = (w.wide ? 0 : s * 16) + g, row = (first + r) * w.down_height + i;
              const float* at = sc + r * w.down_height + (w.wide ? 0 : s * 16);
              row_scales[r][s][0] = i < w.down_height && row < w.rows ? at[0] : 0.0f;
              row_scales[r][s][1] = i + 8 < w.down_height && row + 8 < w.rows ? at[8] : 0.0f;
            }
          const int a0 = sh.assign[slot][2 * t4], a1 = sh.assign[slot][2 * t4 + 1];
          if (a0 >= 0) u0 = sh.a_unscale[a0];
          if (a1 >= 0) u1 = sh.a_unscale[a1];
          if (a >= 0) scale = sh.a_scale[a];
        }
        // The activations of the unit (wide: of both) for the lane's token.  With E4M3 weights a
        // token that is not routed to this expert reads the row of one that is, and its column is
        // masked below: without a condition the eight loads of a lane go out together (with one
        // 145 us instead of 117 us at 3 tokens, H = I = 2880), and the bytes are in the same load
        // anyway (with a row of another expert 255 us instead of 246 us at 8 tokens, H = 4096,
        // I = 14336; 81 us instead of 74.5 us at H = 2048, I = 768, 128 experts).
        uint32_t hi[SUBS][kWords], lo[SUBS][kWords];
        const bool whole = !(ragged && unit == w.units_i - 1);
        const size_t act_row = (size_t)(a < 0 ? ~a : a) * p.act_pitch;
#pragma unroll
        for (int s = 0; s < SUBS; ++s) {
          if (s && !w.wide) {  // both sub-tiles are of the same unit
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
              hi[s][i] = hi[0][i];
              if (!FP8) lo[s][i] = lo[0][i];
            }
            break;
          }
          const int start = (w.wide ? 2 * unit + s : unit) * Work::kUnit;
          const int k = start + t4 * Work::kPiece;
          if constexpr (FP8) {
            const float4* from = reinterpret_cast<const float4*>(
                                     reinterpret_cast<const float*>(p.act_hi) + act_row + start) + t4;
#pragma unroll
            for (int i = 0; i < 8; ++i) {  // elements k + (0..15) and k + 64 + (0..15)
              float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
              if (whole || k + (i / 4) * 64 + i % 4 * 4 < p.inter) v = __ldcg(from + i * 4);
              const __half2 h0 = __floats2half2_rn(v.x * scale, v.y * scale);
              const __half2 h1 = __floats2half2_rn(v.z * scale, v.w * scale);
              hi[s][2 * i] = *reinterpret_cast<const uint32_t*>(&h0);
              hi[s][2 * i + 1] = *reinterpret_cast<const uint32_t*>(&h1);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int at = k + i * (Work::kUnit / 2);
              uint4 q = make_uint4(0u, 0u, 0u, 0u), q2 = q;
              if (a >= 0 && at < p.inter) {
                q = __ldcg(reinterpret_cast<const uint4*>(p.act_hi + (size_t)a * p.inter + at));
                q2 = __ldcg(reinterpret_cast<const uint4*>(p.act_lo + (size_t)a * p.inter + at));
              }
              hi[s][4 * i] = q.x; hi[s][4 * i + 1] = q.y; hi[s][4 * i + 2] = q.z; hi[s][4 * i + 3] = q.w;
              lo[s][4 * i] = q2.x; lo[s][4 * i + 1] = q2.y; lo[s][4 * i + 2] = q2.z; lo[s][4 * i + 3] = q2.w;
            }
          }
        }
#pragma unroll
        for (int r = 0; r < TILES; ++r) {
          if (first + r >= w.down_tiles) break;
          cp_async_wait<kFewStages - 1>();
          uint4 q[SUBS][4];
#pragma unroll
          for (int s = 0; s < SUBS; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) q[s][i] = lds128(src + s * 2048 + i * 512);
          producer.next();
          src += Work::kStageBytes;
          if (src == ring_end) src -= kFewStages * Work::kStageBytes;
#pragma unroll
          for (int s = 0; s < SUBS; ++s) {
            float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            multiply_piece<FP8>(c, q[s][0], q[s][2], hi[s]);
            multiply_piece<FP8>(c, q[s][1], q[s][3], hi[s] + kWords / 2);
            if constexpr (FP8) {
              c[0] *= row_scales[r][s][0] * u0;
              c[1] *= row_scales[r][s][0] * u1;
              c[2] *= row_scales[r][s][1] * u0;
              c[3] *= row_scales[r][s][1] * u1;
            } else {
              multiply_piece<FP8>(c, q[s][0], q[s][2], lo[s]);
              multiply_piece<FP8>(c, q[s][1], q[s][3], lo[s] + kWords / 2);
            }
            if (members & 1u) {
              total[r][s][0] += c[0];
              total[r][s][2] += c[2];
            }
            if (members & 2u) {
              total[r][s][1] += c[1];
              total[r][s][3] += c[3];
            }
          }
        }
        unit += kFewWarps;
      }
      if (w.wide) {  // two units of the same 16 rows
#pragma unroll
        for (int i = 0; i < 4; ++i) total[0][0][i] += total[0][SUBS - 1][i];
      }
#pragma unroll
      for (int r = 0; r < TILES; ++r) {
        if (first + r >= w.down_tiles) break;
        __syncthreads();  // the sums of the tile before are read
        if (2 * t4 < p.tokens) {
#pragma unroll
          for (int s = 0; s < SUBS; ++s) {
            float* red = sh.red[warp] + s * 128 + 2 * t4;
            *reinterpret_cast<float2*>(red + g * 8) = make_float2(total[r][s][0], total[r][s][1]);
            *reinterpret_cast<float2*>(red + (g + 8) * 8) =
                make_float2(total[r][s][2], total[r][s][3]);
          }
        }
        __syncthreads();
        if (threadIdx.x < SUBS * 128) {
          const int i = threadIdx.x % (SUBS * 16), tok = threadIdx.x / (SUBS * 16);
          const int row = (first + r) * w.down_height + i;
          if (i < w.down_height && row < w.rows && tok < p.tokens) {
            float v = 0.0f;
#pragma unroll
            for (int i2 = 0; i2 < kFewWarps; ++i2) v += sh.red[i2][i * 8 + tok];
            p.out[(size_t)tok * p.hidden + w.row0 + row] = __float2bfloat16_rn(v);
          }
        }
      }
    }
    cp_async_wait<0>();
  }
  // the last block to come here leaves the counters at zero for the next call
  if (threadIdx.x == 0 && atomicAdd(p.sync + 2, 1u) == gridDim.x - 1) {
    p.sync[0] = p.sync[1] = p.sync[2] = 0u;
    __threadfence();
  }
}

// Rows of a stage, tiles of a group, and the shared memory of a block for a call whose token rows
// take `x_bytes` of it and whose blocks have up to `rows` output rows.
//   Stages of 16 rows, groups of four tiles of the down projection.  BF16 with stages of 32 rows,
// two tiles and a ring of three: 455 us instead of 422 us at 8 tokens, H = 4096, I = 14336,
// 8 experts; 102.5 instead of 97.6 us at H = 2048, I = 768, 128 experts.  Two tiles of 16 rows:
// the same where a block has no more, 431 instead of 418 us at H = 7168, I = 2048, 32 experts.
//   E4M3, where a block has no more than 32 output rows (the token rows then leave the room on 148
// SMs): stages of 32 rows, one tile.  That halves the loads and conversions of activations per
// byte of weights (80 us against 90 us at H = 2048, I = 768, 128 experts; 106 against 124 us with
// 3 tokens, H = I = 2880, 32 experts; 253 against 267 us at H = 4096, I = 14336, 8 experts); with
// more rows a group of two such tiles does not fit in the registers (H = 7168, 8 tokens: 268
// against 250 us).
struct FewShape {
  bool large;
  size_t bytes;
};
FewShape few_shape(bool fp8, size_t x_bytes, int rows) {
  constexpr size_t kRing = (size_t)kFewStages * kFewWarps * 2048;
  const size_t large = sizeof(FewShared<2>) + x_bytes + 2 * kRing;
  if (fp8 && rows <= 32 && large <= kMostSharedMemory) return {true, large};
  return {false, sizeof(FewShared<1>) + x_bytes + kRing};
}
// the longest token rows fit
static_assert(sizeof(FewShared<1>) + kFewMaxTokens * (B200MOE_LAYER_MAX_HIDDEN * 2 + 64) +
                  kFewStages * kFewWarps * 2048 <= kMostSharedMemory, "shared memory");

template <bool FP8, bool ROUTER_F32>
const void* few_kernel(bool large) {
  if constexpr (FP8)
    if (large) return (const void*)layer_few_kernel<true, ROUTER_F32, 2, 1>;
  return (const void*)layer_few_kernel<FP8, ROUTER_F32, 1, 4>;
}

}  // namespace

cudaError_t launch_layer_few(const void* x, const void* router, bool router_f32,
                             const void* gate_up, const void* down, const float* gate_up_scale,
                             const float* down_scale, int tokens, int hidden, int inter,
                             int experts, int top_k, double* logits, uint32_t* act_max,
                             void* acts, void* out, int64_t* ids_out, float* weights_out,
                             unsigned int* sync, uint32_t* status, int sm_count,
                             cudaStream_t stream) {
  const bool fp8 = gate_up_scale != nullptr;
  FewParams p;
  p.x = static_cast<const __nv_bfloat16*>(x);
  p.router = router;
  p.gate_up = static_cast<const uint8_t*>(gate_up);
  p.down = static_cast<const uint8_t*>(down);
  p.gate_up_scale = gate_up_scale;
  p.down_scale = down_scale;
  p.tokens = tokens;
  p.hidden = hidden;
  p.inter = inter;
  p.experts = experts;
  p.top_k = top_k;
  // row pitch of the token operand: 64 (BF16) or 16 (E4M3) bytes over a multiple of 128, which
  // keeps the eight lanes of a 128-byte shared-memory read on different banks
  const int unit = fp8 ? 128 : 64;
  p.inter_inverse = ((1ull << 40) + inter - 1) / inter;
  p.x_pitch = (hidden + unit - 1) / unit * unit * 2 + (fp8 ? 16 : 64);
  p.logits = logits;
  p.act_max = act_max;
  p.act_hi = static_cast<uint16_t*>(acts);
  p.act_lo = p.act_hi + (size_t)tokens * top_k * inter;
  p.act_pitch = (int)align_up((size_t)inter, 64);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.ids_out = ids_out;
  p.weights_out = weights_out;
  p.sync = sync;
  p.status = status;
  // the down scales of a block lie where its token rows were, which are longer on any GPU with
  // more than 16 SMs
  if (fp8 && (size_t)tokens * top_k * ((hidden + sm_count - 1) / sm_count) * sizeof(float) >
                 (size_t)tokens * p.x_pitch)
    return cudaErrorInvalidConfiguration;
  const FewShape shape = few_shape(fp8, align_up((size_t)tokens * p.x_pitch, 128),
                                   (hidden + sm_count - 1) / sm_count);
  const void* kernel = fp8 ? (router_f32 ? few_kernel<true, true>(shape.large)
                                         : few_kernel<true, false>(shape.large))
                           : (router_f32 ? few_kernel<false, true>(shape.large)
                                         : few_kernel<false, false>(shape.large));
  static std::atomic<uint64_t> allowed[2][2][2];
  cudaError_t err = allow_shared_memory(kernel, allowed[fp8][router_f32][shape.large]);
  if (err != cudaSuccess) return err;
  void* args[] = {&p};
  return cudaLaunchCooperativeKernel(kernel, dim3(sm_count), dim3(kFewThreads), args, shape.bytes,
                                     stream);
}

}  // namespace b200moe
