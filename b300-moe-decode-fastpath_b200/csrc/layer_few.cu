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
// no partial sums in memory, no atomics, and sums in an order that only the shape and the
// routing decide.  Inside the block the reduction dimension is cut into units of 128 bytes a
// row, dealt to the warps in turn; the warps' partial tiles are added in shared memory.
//
// The tile.  A warp multiplies 16 rows by 8 columns with mma.m16n8k16.  The column index is the
// token, for gate/up and down alike, so the token operand needs no gathering: for gate+up all
// tokens are multiplied and only those routed to the expert are kept; for down the other tokens'
// columns are zero and are masked once more when an expert's tile is added (a weight of NaN or
// infinity reaches only the tokens routed to it).  mma.sync and not tcgen05: 8 columns of useful
// work leave the tensor pipe idle either way, and operands that arrive in registers need no
// descriptor, no tensor memory and no block-wide handshake per tile.
//
// Loads.  Each lane copies with cp.async the very 16 bytes that it will use as fragments (rows
// g and g+8, four lanes side by side in a row), into a ring of its warp in shared memory, and
// reads them back itself: no barrier between producer and consumer, and up to 200 KB in flight
// on an SM.  Any permutation of the reduction dimension is allowed as long as both operands
// share it, which is why a lane's 16 consecutive bytes can serve as its part of the fragment.
// The ring does not stop at the grid barrier: while a block waits for the activations, its
// warps' first down tiles are already on their way.
//
// Precision.  Logits are summed with the rounding errors of all additions kept (two-sum), so
// that they are good to about 2^-48: experts that lie next to one another at the border are
// told apart as in 64 bits.  Products and sums are FP32; the activations are held as the sum of
// two BF16 numbers (16 significant bits), as the regular path holds them.
#include "common.cuh"

namespace b200moe {

namespace {

constexpr int kFewWarps = 16;
constexpr int kFewThreads = kFewWarps * 32;
constexpr int kFewStageBytes = 2048;            // 16 rows x 128 bytes: one stage of one warp
constexpr int kFewSlots = kFewMaxTokens * 8;    // experts in use, at most
constexpr int kFewMaxTiles = 4;                 // 16-row tiles of the down projection taken together

struct FewParams {
  const __nv_bfloat16* x;
  const void* router;
  const uint8_t* gate_up;   // bytes; BF16 or E4M3
  const uint8_t* down;
  const float* gate_up_scale;
  const float* down_scale;
  int tokens, hidden, inter, experts, top_k;
  int x_pitch;              // bytes of a token row in shared memory
  int stages;               // ring stages of a warp
  double* logits;           // [tokens, experts]
  __nv_bfloat16* act_hi;    // [tokens * top_k, inter]
  __nv_bfloat16* act_lo;
  __nv_bfloat16* out;
  int64_t* ids_out;
  float* weights_out;
  unsigned int* sync;       // three counters, zero between calls
  uint32_t* status;
};

struct alignas(128) FewShared {
  double logit[kFewWarps][kFewMaxTokens];
  float red[2][kFewWarps][128];
  float weight[kFewSlots];              // by assignment
  int expert[kFewSlots];                // by slot (experts in use, ascending)
  int chosen[kFewSlots];                // expert by assignment
  int slot_of[B200MOE_MAX_EXPERTS];
  signed char assign[kFewSlots][kFewMaxTokens];  // assignment of (slot, token), or -1
  int num_slots;
  int abort;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  const int bytes = valid ? 16 : 0;  // 0: the 16 bytes are zeroed, nothing is read
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
// all but the newest `pending` groups have arrived
__device__ __forceinline__ void cp_async_wait_for(int pending) {
  switch (pending) {
    case 0: cp_async_wait<0>(); break;
    case 1: cp_async_wait<1>(); break;
    case 2: cp_async_wait<2>(); break;
    case 3: cp_async_wait<3>(); break;
    case 4: cp_async_wait<4>(); break;
    case 5: cp_async_wait<5>(); break;
    default: cp_async_wait<6>(); break;
  }
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ void mma_16x8x16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                            uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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
      e4m3x4_to_bf16x4(t[i], t01, t23);
      e4m3x4_to_bf16x4(u[i], u01, u23);
      mma_16x8x16(c, t01, u01, t23, u23, b[2 * i], b[2 * i + 1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      mma_16x8x16(c, t[2 * i], u[2 * i], t[2 * i + 1], u[2 * i + 1], b[2 * i], b[2 * i + 1]);
  }
}

// Grid barrier: bounded, after which the block goes on to its end without further work.
__device__ __forceinline__ bool grid_barrier(unsigned int* counter, uint32_t* status, int* abort) {
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    atomicAdd(counter, 1u);
    const uint64_t t0 = global_timer_ns();
    uint32_t spins = 0;
    while (true) {
      unsigned int seen;
      asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(seen) : "l"(counter) : "memory");
      if (seen >= gridDim.x) break;
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

// 64-bit order of a double: larger values larger, NaN above every number
__device__ __forceinline__ unsigned long long order_of(double v) {
  const unsigned long long bits = (unsigned long long)__double_as_longlong(v);
  if (v != v) return ~0ull;
  const unsigned long long k = (bits >> 63) ? ~bits : (bits | 0x8000000000000000ull);
  return k;
}

// Logits of the experts b, b + G, ...; x is in shared memory.
template <bool ROUTER_F32>
__device__ __forceinline__ void router_logits(const FewParams& p, FewShared& sh,
                                              const uint8_t* x_rows) {
  const int vecs = p.hidden / 8;
  for (int e = blockIdx.x; e < p.experts; e += gridDim.x) {
    float s[kFewMaxTokens], err[kFewMaxTokens];
#pragma unroll
    for (int t = 0; t < kFewMaxTokens; ++t) s[t] = err[t] = 0.0f;
    for (int v = threadIdx.x; v < vecs; v += kFewThreads) {
      float w[8];
      if constexpr (ROUTER_F32) {
        const float4* src = reinterpret_cast<const float4*>(
            static_cast<const float*>(p.router) + (size_t)e * p.hidden + 8 * v);
        const float4 a = __ldg(src), b = __ldg(src + 1);
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
        w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
      } else {
        const uint4 q = __ldg(reinterpret_cast<const uint4*>(
            static_cast<const __nv_bfloat16*>(p.router) + (size_t)e * p.hidden + 8 * v));
        const uint32_t words[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[2 * i] = __uint_as_float(words[i] << 16);
          w[2 * i + 1] = __uint_as_float(words[i] & 0xFFFF0000u);
        }
      }
#pragma unroll
      for (int t = 0; t < kFewMaxTokens; ++t) {
        if (t >= p.tokens) break;
        const uint4 q = *reinterpret_cast<const uint4*>(x_rows + t * p.x_pitch + 16 * v);
        const uint32_t words[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float xv = (i & 1) ? __uint_as_float(words[i / 2] & 0xFFFF0000u)
                                   : __uint_as_float(words[i / 2] << 16);
          const float prod = __fmul_rn(w[i], xv);  // exact for BF16 x BF16
          if constexpr (ROUTER_F32) err[t] += __fmaf_rn(w[i], xv, -prod);
          two_sum(s[t], err[t], prod);
        }
      }
    }
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int t = 0; t < kFewMaxTokens; ++t) {
      if (t >= p.tokens) break;
      // an error term of an overflowed or NaN sum is NaN itself: the sum alone tells
      double d = (double)s[t];
      if (isfinite(s[t])) d += (double)err[t];
#pragma unroll
      for (int m = 16; m > 0; m >>= 1) d += __shfl_xor_sync(0xffffffffu, d, m);
      if (lane == 0) sh.logit[warp][t] = d;
    }
    __syncthreads();
    if (threadIdx.x < p.tokens) {
      double d = 0.0;
      for (int i = 0; i < kFewWarps; ++i) d += sh.logit[i][threadIdx.x];
      __stcg(p.logits + (size_t)threadIdx.x * p.experts + e, d);
    }
    __syncthreads();
  }
}

// Top-k and softmax of every token, one warp each, then the list of experts in use.  Every
// block does this for itself from the logits.
__device__ __forceinline__ void choose_experts(const FewParams& p, FewShared& sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < B200MOE_MAX_EXPERTS; i += kFewThreads) sh.slot_of[i] = -1;
  for (int i = threadIdx.x; i < kFewSlots * kFewMaxTokens; i += kFewThreads)
    (&sh.assign[0][0])[i] = -1;
  __syncthreads();
  if (warp < p.tokens) {
    double v[8];
    unsigned long long key[8];  // 0: taken or absent
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = lane + 32 * i;
      v[i] = e < p.experts ? __ldcg(p.logits + (size_t)warp * p.experts + e) : 0.0;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) key[i] = lane + 32 * i < p.experts ? order_of(v[i]) : 0ull;
    double top = 0.0;
    float mine = 0.0f, denom = 0.0f;
    int my_id = 0;
    for (int k = 0; k < p.top_k; ++k) {
      unsigned long long best = 0ull;
      int best_i = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (key[i] > best) {
          best = key[i];
          best_i = i;
        }
      const unsigned hi = __reduce_max_sync(0xffffffffu, (unsigned)(best >> 32));
      const bool in_hi = (unsigned)(best >> 32) == hi;
      const unsigned lo = __reduce_max_sync(0xffffffffu, in_hi ? (unsigned)best : 0u);
      const bool in_both = in_hi && (unsigned)best == lo;
      const unsigned id =
          __reduce_min_sync(0xffffffffu, in_both ? (unsigned)(lane + 32 * best_i) : 0xffffffffu);
      double value = 0.0;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if ((unsigned)(lane + 32 * i) == id) {
          value = v[i];
          key[i] = 0ull;
        }
      value = __shfl_sync(0xffffffffu, value, id & 31);
      if (k == 0) top = value;
      const float w = expf((float)(value - top));
      denom += w;
      if (lane == k) {
        mine = w;
        my_id = (int)id;
      }
    }
    if (lane < p.top_k) {
      const int a = warp * p.top_k + lane;
      const float w = mine / denom;
      sh.weight[a] = w;
      sh.chosen[a] = my_id;
      sh.slot_of[my_id] = 0;  // in use; numbered below
      if (blockIdx.x == 0) {
        if (p.ids_out) p.ids_out[a] = my_id;
        if (p.weights_out) p.weights_out[a] = w;
      }
    }
  }
  __syncthreads();
  if (warp == 0) {
    int count = 0;
    for (int base = 0; base < p.experts; base += 32) {
      const int e = base + lane;
      const bool used = e < p.experts && sh.slot_of[e] == 0;
      const unsigned votes = __ballot_sync(0xffffffffu, used);
      if (used) {
        const int slot = count + __popc(votes & ((1u << lane) - 1u));
        sh.slot_of[e] = slot;
        sh.expert[slot] = e;
      }
      count += __popc(votes);
    }
    if (lane == 0) sh.num_slots = count;
  }
  __syncthreads();
  if (threadIdx.x < p.tokens * p.top_k)
    sh.assign[sh.slot_of[sh.chosen[threadIdx.x]]][threadIdx.x / p.top_k] = (signed char)threadIdx.x;
  __syncthreads();
}

// The order in which a warp's ring is filled: first the gate/up tiles of its block, then the
// down tiles.  Both sides of the ring -- the copies and the products -- walk it.
template <bool FP8>
struct FewWork {
  static constexpr int kUnit = FP8 ? 128 : 64;   // elements of a row in one stage
  static constexpr int kPiece = FP8 ? 16 : 8;    // elements in 16 bytes
  static constexpr int kElem = FP8 ? 1 : 2;      // bytes of an element

  int pair0, pairs, tiles, height;               // gate/up: this block's pairs and tiles
  int row0, rows, down_tiles, down_height;       // down: its output rows
  int units_h, units_i, down_units;              // stages along H; along I; along all experts

  __device__ FewWork(const FewParams& p, int slots) {
    const long long total = (long long)slots * p.inter;
    pair0 = (int)(total * blockIdx.x / gridDim.x);
    pairs = (int)(total * (blockIdx.x + 1) / gridDim.x) - pair0;
    tiles = (pairs + 7) / 8;
    height = tiles ? (pairs + tiles - 1) / tiles : 0;
    row0 = (int)((long long)p.hidden * blockIdx.x / gridDim.x);
    rows = (int)((long long)p.hidden * (blockIdx.x + 1) / gridDim.x) - row0;
    down_tiles = (rows + 15) / 16;
    down_height = down_tiles ? (rows + down_tiles - 1) / down_tiles : 0;
    units_h = (p.hidden + kUnit - 1) / kUnit;
    units_i = (p.inter + kUnit - 1) / kUnit;
    down_units = slots * units_i;
  }
};

// Fills the ring: one stage per call, in order.
template <bool FP8>
struct FewProducer {
  using Work = FewWork<FP8>;
  const FewParams& p;
  const FewShared& sh;
  const Work& w;
  uint32_t ring;       // this lane's place in the warp's first stage
  int warp, lane;
  int stage = 0;       // next stage to fill
  bool down = false;
  int tile = 0;        // gate/up: tile; down: first tile of the group
  int unit;            // unit within the tile (gate/up) or along all experts (down)
  int sub = 0;         // down: tile within the group
  const uint8_t* top = nullptr;     // gate/up: this lane's gate row and up row
  const uint8_t* bottom = nullptr;
  bool live = false;

  __device__ FewProducer(const FewParams& p_, const FewShared& sh_, const Work& w_, uint32_t ring_,
                         int warp_, int lane_)
      : p(p_), sh(sh_), w(w_), ring(ring_), warp(warp_), lane(lane_), unit(warp_) {
    enter_tile();
  }

  // moves on to the next tile that has a unit for this warp
  __device__ void enter_tile() {
    while (!down && unit >= w.units_h) {
      unit -= w.units_h;
      ++tile;
      if (tile >= w.tiles) break;
    }
    if (!down && tile >= w.tiles) {
      down = true;
      tile = 0;
      sub = 0;
      unit = warp;
      return;
    }
    const int i = tile * w.height + (lane >> 2);
    live = (lane >> 2) < w.height && i < w.pairs;
    const int pair = w.pair0 + (live ? i : 0);
    const int slot = pair / p.inter;
    const size_t col = (size_t)(pair - slot * p.inter);
    const size_t row_bytes = (size_t)p.hidden * Work::kElem;
    top = p.gate_up + ((size_t)sh.expert[slot] * 2 * p.inter + col) * row_bytes;
    bottom = top + (size_t)p.inter * row_bytes;
  }

  __device__ void next() {
    const uint32_t dst = ring + stage * kFewStageBytes;
    const int piece = (lane & 3) * Work::kPiece;
    if (!down) {
      const int k = unit * Work::kUnit + piece, k2 = k + Work::kUnit / 2;
      const bool a = live && k < p.hidden, b = live && k2 < p.hidden;
      cp_async16(dst, a ? top + (size_t)k * Work::kElem : p.gate_up, a);
      cp_async16(dst + 512, b ? top + (size_t)k2 * Work::kElem : p.gate_up, b);
      cp_async16(dst + 1024, a ? bottom + (size_t)k * Work::kElem : p.gate_up, a);
      cp_async16(dst + 1536, b ? bottom + (size_t)k2 * Work::kElem : p.gate_up, b);
      unit += kFewWarps;
      if (unit >= w.units_h) enter_tile();
    } else if (tile < w.down_tiles && unit < w.down_units) {
      const int slot = unit / w.units_i;
      const int k = (unit - slot * w.units_i) * Work::kUnit + piece, k2 = k + Work::kUnit / 2;
      const int i = lane >> 2, r = (tile + sub) * w.down_height + i;
      const bool t = i < w.down_height && r < w.rows;
      const bool u = i + 8 < w.down_height && r + 8 < w.rows;
      const uint8_t* base =
          p.down + (((size_t)sh.expert[slot] * p.hidden + w.row0 + r) * p.inter + k) * Work::kElem;
      const uint8_t* base8 = base + (size_t)8 * p.inter * Work::kElem;
      const bool a = k < p.inter, b = k2 < p.inter;
      const int half = Work::kUnit / 2 * Work::kElem;
      cp_async16(dst, t && a ? base : p.down, t && a);
      cp_async16(dst + 512, t && b ? base + half : p.down, t && b);
      cp_async16(dst + 1024, u && a ? base8 : p.down, u && a);
      cp_async16(dst + 1536, u && b ? base8 + half : p.down, u && b);
      const int group = min(kFewMaxTiles, w.down_tiles - tile);
      if (++sub == group) {
        sub = 0;
        unit += kFewWarps;
        if (unit >= w.down_units) {
          unit = warp;
          tile += group;
        }
      }
    }
    cp_async_commit();  // an empty group when there is nothing left
    if (++stage == p.stages) stage = 0;
  }
};

template <bool FP8, bool ROUTER_F32>
__global__ void __launch_bounds__(kFewThreads, 1) layer_few_kernel(const FewParams p) {
  using Work = FewWork<FP8>;
  extern __shared__ __align__(128) uint8_t smem[];
  FewShared& sh = *reinterpret_cast<FewShared*>(smem);
  uint8_t* x_rows = smem + sizeof(FewShared);
  uint8_t* rings = x_rows + align_up((size_t)p.tokens * p.x_pitch, 128);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t4 = lane & 3;

  if (threadIdx.x == 0) {
    sh.abort = 0;
    if (blockIdx.x == 0) *p.status = 0u;
  }
  // token rows, zero up to the end of the last unit
  const int row_vecs = (p.hidden + Work::kUnit - 1) / Work::kUnit * Work::kUnit / 8;
  for (int t = 0; t < p.tokens; ++t)
    for (int v = threadIdx.x; v < row_vecs; v += kFewThreads) {
      uint4 q = make_uint4(0u, 0u, 0u, 0u);
      if (8 * v < p.hidden)
        q = *reinterpret_cast<const uint4*>(p.x + (size_t)t * p.hidden + 8 * v);
      *reinterpret_cast<uint4*>(x_rows + t * p.x_pitch + 16 * v) = q;
    }
  __syncthreads();
  router_logits<ROUTER_F32>(p, sh, x_rows);
  bool ok = grid_barrier(p.sync, p.status, &sh.abort);

  if (ok) {
    choose_experts(p, sh);
    const Work w(p, sh.num_slots);
    const uint32_t ring = smem_u32(rings) + warp * p.stages * kFewStageBytes + lane * 16;
    FewProducer<FP8> producer(p, sh, w, ring, warp, lane);
    for (int i = 0; i < p.stages; ++i) producer.next();
    int stage = 0;
    const uint32_t x_lane = smem_u32(x_rows) + g * p.x_pitch + t4 * Work::kPiece * 2;
    int buffer = 0;

    // ---- gate + up -----------------------------------------------------------------
    int unit = warp;
    for (int tile = 0; tile < w.tiles; ++tile) {
      float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      for (; unit < w.units_h; unit += kFewWarps) {
        // token operand: elements of both halves of the unit
        uint32_t b[FP8 ? 16 : 8];
#pragma unroll
        for (int i = 0; i < (FP8 ? 4 : 2); ++i) {
          uint4 q = make_uint4(0u, 0u, 0u, 0u);
          if (g < p.tokens)
            q = lds128(x_lane + unit * Work::kUnit * 2 +
                       (FP8 ? (i / 2) * Work::kUnit + (i % 2) * 16 : i * Work::kUnit));
          b[4 * i] = q.x; b[4 * i + 1] = q.y; b[4 * i + 2] = q.z; b[4 * i + 3] = q.w;
        }
        cp_async_wait_for(p.stages - 1);
        const uint32_t src = ring + stage * kFewStageBytes;
        const uint4 a0 = lds128(src), a1 = lds128(src + 512);
        const uint4 b0 = lds128(src + 1024), b1 = lds128(src + 1536);
        producer.next();
        if (++stage == p.stages) stage = 0;
        multiply_piece<FP8>(c, a0, b0, b);
        multiply_piece<FP8>(c, a1, b1, b + (FP8 ? 8 : 4));
      }
      unit -= w.units_h;
      float* red = sh.red[buffer][warp];
      *reinterpret_cast<float2*>(red + g * 8 + 2 * t4) = make_float2(c[0], c[1]);
      *reinterpret_cast<float2*>(red + (g + 8) * 8 + 2 * t4) = make_float2(c[2], c[3]);
      __syncthreads();
      if (warp == tile % kFewWarps) {  // this warp finishes the tile, the others go on
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int o = lane + 32 * half, i = o >> 3, tok = o & 7;
          const int local = tile * w.height + i;
          if (i < w.height && local < w.pairs && tok < p.tokens) {
            const int pair = w.pair0 + local;
            const int slot = pair / p.inter, col = pair - slot * p.inter;
            const int a = sh.assign[slot][tok];
            if (a >= 0) {
              float gate = 0.0f, up = 0.0f;
#pragma unroll
              for (int i2 = 0; i2 < kFewWarps; ++i2) {
                gate += sh.red[buffer][i2][o];
                up += sh.red[buffer][i2][o + 64];
              }
              if constexpr (FP8) {
                const float* s = p.gate_up_scale + (size_t)sh.expert[slot] * 2 * p.inter + col;
                gate *= __ldg(s);
                up *= __ldg(s + p.inter);
              }
              const float act = gate / (1.0f + expf(-gate)) * up * sh.weight[a];
              const __nv_bfloat16 hi = __float2bfloat16_rn(act);
              const float rest = act - __bfloat162float(hi);
              p.act_hi[(size_t)a * p.inter + col] = hi;
              p.act_lo[(size_t)a * p.inter + col] =
                  __float2bfloat16_rn(isfinite(rest) ? rest : 0.0f);
            }
          }
        }
      }
      buffer ^= 1;
    }
    ok = grid_barrier(p.sync + 1, p.status, &sh.abort);

    // ---- down ----------------------------------------------------------------------
    for (int first = 0; ok && first < w.down_tiles; first += kFewMaxTiles) {
      const int group = min(kFewMaxTiles, w.down_tiles - first);
      float total[kFewMaxTiles][4];
#pragma unroll
      for (int r = 0; r < kFewMaxTiles; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) total[r][i] = 0.0f;
      for (int unit = warp; unit < w.down_units; unit += kFewWarps) {
        const int slot = unit / w.units_i;
        const int k = (unit - slot * w.units_i) * Work::kUnit + t4 * Work::kPiece;
        const int a = sh.assign[slot][g];
        uint32_t hi[FP8 ? 16 : 8], lo[FP8 ? 16 : 8];
#pragma unroll
        for (int i = 0; i < (FP8 ? 4 : 2); ++i) {
          const int at = k + (FP8 ? (i / 2) * (Work::kUnit / 2) + (i % 2) * 8 : i * (Work::kUnit / 2));
          uint4 q = make_uint4(0u, 0u, 0u, 0u), q2 = q;
          if (a >= 0 && at < p.inter) {
            q = __ldcg(reinterpret_cast<const uint4*>(p.act_hi + (size_t)a * p.inter + at));
            q2 = __ldcg(reinterpret_cast<const uint4*>(p.act_lo + (size_t)a * p.inter + at));
          }
          hi[4 * i] = q.x; hi[4 * i + 1] = q.y; hi[4 * i + 2] = q.z; hi[4 * i + 3] = q.w;
          lo[4 * i] = q2.x; lo[4 * i + 1] = q2.y; lo[4 * i + 2] = q2.z; lo[4 * i + 3] = q2.w;
        }
        // the tokens of this lane's two columns
        const bool has0 = sh.assign[slot][2 * t4] >= 0, has1 = sh.assign[slot][2 * t4 + 1] >= 0;
#pragma unroll
        for (int r = 0; r < kFewMaxTiles; ++r) {
          if (r >= group) break;
          float s0 = 1.0f, s1 = 1.0f;
          if constexpr (FP8) {
            const int row = (first + r) * w.down_height + g;
            const float* s = p.down_scale + (size_t)sh.expert[slot] * p.hidden + w.row0 + row;
            s0 = g < w.down_height && row < w.rows ? __ldg(s) : 0.0f;
            s1 = g + 8 < w.down_height && row + 8 < w.rows ? __ldg(s + 8) : 0.0f;
          }
          cp_async_wait_for(p.stages - 1);
          const uint32_t src = ring + stage * kFewStageBytes;
          const uint4 a0 = lds128(src), a1 = lds128(src + 512);
          const uint4 b0 = lds128(src + 1024), b1 = lds128(src + 1536);
          producer.next();
          if (++stage == p.stages) stage = 0;
          float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          multiply_piece<FP8>(c, a0, b0, hi);
          multiply_piece<FP8>(c, a1, b1, hi + (FP8 ? 8 : 4));
          multiply_piece<FP8>(c, a0, b0, lo);
          multiply_piece<FP8>(c, a1, b1, lo + (FP8 ? 8 : 4));
          if (has0) {
            total[r][0] = fmaf(c[0], s0, total[r][0]);
            total[r][2] = fmaf(c[2], s1, total[r][2]);
          }
          if (has1) {
            total[r][1] = fmaf(c[1], s0, total[r][1]);
            total[r][3] = fmaf(c[3], s1, total[r][3]);
          }
        }
      }
#pragma unroll
      for (int r = 0; r < kFewMaxTiles; ++r) {
        if (r >= group) break;
        float* red = sh.red[buffer][warp];
        *reinterpret_cast<float2*>(red + g * 8 + 2 * t4) = make_float2(total[r][0], total[r][1]);
        *reinterpret_cast<float2*>(red + (g + 8) * 8 + 2 * t4) =
            make_float2(total[r][2], total[r][3]);
        __syncthreads();
        if (threadIdx.x < 128) {
          const int i = threadIdx.x & 15, tok = threadIdx.x >> 4;
          const int row = (first + r) * w.down_height + i;
          if (i < w.down_height && row < w.rows && tok < p.tokens) {
            float v = 0.0f;
#pragma unroll
            for (int i2 = 0; i2 < kFewWarps; ++i2) v += sh.red[buffer][i2][i * 8 + tok];
            p.out[(size_t)tok * p.hidden + w.row0 + row] = __float2bfloat16_rn(v);
          }
        }
        buffer ^= 1;
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

int few_pitch(int hidden, bool fp8) {
  // row pitch of the token operand: 64 (BF16) or 16 (FP8) bytes over a multiple of 128, which
  // keeps the eight lanes of a 128-byte shared-memory read on different banks
  const int unit = fp8 ? 128 : 64;
  return (hidden + unit - 1) / unit * unit * 2 + (fp8 ? 16 : 64);
}

}  // namespace

cudaError_t launch_layer_few(const void* x, const void* router, bool router_f32,
                             const void* gate_up, const void* down, const float* gate_up_scale,
                             const float* down_scale, int tokens, int hidden, int inter,
                             int experts, int top_k, double* logits, void* act_hi, void* act_lo,
                             void* out, int64_t* ids_out, float* weights_out, unsigned int* sync,
                             uint32_t* status, int sm_count, cudaStream_t stream) {
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
  p.x_pitch = few_pitch(hidden, fp8);
  p.logits = logits;
  p.act_hi = static_cast<__nv_bfloat16*>(act_hi);
  p.act_lo = static_cast<__nv_bfloat16*>(act_lo);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.ids_out = ids_out;
  p.weights_out = weights_out;
  p.sync = sync;
  p.status = status;
  constexpr size_t kMost = 227 * 1024;
  const size_t fixed = sizeof(FewShared) + align_up((size_t)tokens * p.x_pitch, 128);
  int stages = (int)((kMost - fixed) / (kFewWarps * kFewStageBytes));
  if (kMost < fixed || stages < 1) return cudaErrorInvalidValue;
  p.stages = stages > 6 ? 6 : stages;
  const size_t bytes = fixed + (size_t)p.stages * kFewWarps * kFewStageBytes;
  const void* kernel =
      fp8 ? (router_f32 ? (const void*)layer_few_kernel<true, true>
                        : (const void*)layer_few_kernel<true, false>)
          : (router_f32 ? (const void*)layer_few_kernel<false, true>
                        : (const void*)layer_few_kernel<false, false>);
  cudaError_t err =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (err != cudaSuccess) return err;
  void* args[] = {&p};
  return cudaLaunchCooperativeKernel(kernel, dim3(sm_count), dim3(kFewThreads), args, bytes,
                                     stream);
}

}  // namespace b200moe
