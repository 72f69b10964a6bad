// A whole mixture-of-experts layer for 1 to 32 tokens in two kernels.
//
//   out[m] = s * sum_k w[m, k] * W2[e] . Q2(act(W1[e] . Q1(x[m]))),  e = ids[m, k]
//
// k_few_up: routing (and, from logits, the router's top-k), Q1, the gate and up projections and the
// activation; k_few_down: routing again, Q2, the down projection and the weighted sum over a token's
// experts.  Nothing is sorted or copied: with so few tokens the routing is a bit mask of tokens per
// touched expert, which every block builds for itself in shared memory.  (8-bit rows or activations whose
// codes do not fit beside a block's rings are quantised by k_few_codes in between; 4-bit rows whose codes do not
// fit in shared memory go part by part, each by its own pair of kernels.)
//
// What bounds it: the weights of the touched experts, read from HBM once each (once a part).  Split: k_few_up's unit
// is up to 16 (MX: 32) intermediate columns of one expert, gate and up rows together over the whole hidden
// size, so that activation and (4-bit experts) the block quantiser run on finished sums; k_few_down's
// unit is up to 32 output columns over ALL touched experts, so that the sum over a token's experts stays in
// registers.  Units go to the blocks in contiguous runs of equal length (their size is chosen for that), the
// 128-byte boxes of a unit to the warps (token_mma.cuh).  The second kernel is launched with programmatic
// serialisation: its blocks start as soon as there is room, build the routing and fill their rings with
// weights while the first kernel finishes, and wait for it before they read its activations.  No block
// waits for another, nothing is counted in memory, and results do not depend on timing.
//
// Measured (graph replays, weights apart from call to call): Mixtral bf16, one token 114 us, 6.2 TB/s of
// weights; DeepSeek-V3 fp8, one token 85 us, 4.1 TB/s, eight 468 us, 5.4 TB/s (the row tiles of bolt_moe_layer
// take 410); nvfp4, one token 64 us, eight 372 us, 3.8 TB/s.  Beside HBM they wait for: two prologues of 3 us each (instructions that are not in the
// cache yet, routing, the first loads), and with 4-bit codes the ALU: widening a code and scaling it costs
// about 2.3 instructions a weight pair, as long as HBM takes to bring it.
//
// Rounding: 16-bit experts round the activation to the weights' type (the tensor cores' operand);
// quantised experts keep fp32 up to their quantiser.  All sums are fp32, rounded once at the end.
#include <cuda.h>

#include <algorithm>
#include <atomic>

#include "act_pair.cuh"
#include "routing_row.cuh"
#include "tensor_map.cuh"
#include "token_mma.cuh"

namespace bolt {
namespace few {
namespace {

struct Params {
  const void* x;            // [tokens, hidden], 16-bit
  int x_dtype, out_dtype;
  int tokens, topk, hidden, inter, model_dim, experts, global_experts;
  const void* s1;           // 8-bit: fp32; 4-bit: scale bytes [experts, 2 inter, hidden / block]
  const void* s2;
  const float *g1, *g2, *a1, *a2;   // scales of whole tensors (4-bit), null: 1
  const float* wts;         // [tokens, topk]
  const int32_t* ids;
  const void* gating;       // router logits [tokens, global_experts]: ids and wts are made here
  int gating_dtype, renormalize, softmax;
  const int32_t* emap;
  ActParams act;
  float out_scale;
  void* out;
  // workspace: activations of every (expert, token) slot
  uint8_t* act_rows;        // 16-bit values, fp32 values (8-bit kinds) or codes (4-bit kinds)
  uint8_t* act_sf;          // scale bytes (4-bit kinds)
  float* act_amax;          // [slots][units of an expert] (per-channel kinds)
  int32_t* status;
  int slots_per_warp;
  int amax_cols;            // units of an expert in the first kernel
  int unit;                 // columns (first kernel) or rows (second) of a unit
  int group_warps;          // warps that share a unit (first kernel)
  // 8-bit codes of the rows, of the activations: made by every block in its shared memory, or read from
  // k_few_codes' output: codes [rows][columns], scales [rows][groups] (block-scaled) or [rows]
  int keep_x, keep_act;
  uint8_t *xq, *aq;
  float *xs, *as;
};

// ---------------------------------------------------------------------------
// routing
// ---------------------------------------------------------------------------
// The touched experts in ascending order, a slot for every (expert, token) in that order.
struct Routes {
  int* list;        // [touched] expert
  uint32_t* mask;   // [touched] its tokens
  int* off;         // [touched] slot of its first token
  float* coef;      // [slots] router weight (of all routes of a token to the expert)
  int* token;       // [slots]
  int touched, slots;
};
// shared memory of it: per touched expert (at most one a route) 3 words, per slot 2, per route 2, and the
// masks of all experts where the routes are more than a warp has lanes
__host__ __device__ inline int route_bytes(int experts, int routes) {
  return 4 * (7 * routes + (routes > 32 ? experts : 0)) + 64;
}

template <int NPL>
__device__ __noinline__ void route_token(const void* row, int dt, int experts, int topk, int renormalize,
                                         int softmax, int lane, float& w, int& id) {
  float v[NPL];
#pragma unroll
  for (int j = 0; j < NPL; ++j) {
    const int e = lane + 32 * j;
    v[j] = 0.f;
    if (e < experts)
      v[j] = dt == BOLT_F32    ? static_cast<const float*>(row)[e]
             : dt == BOLT_BF16 ? to_f32(static_cast<const __nv_bfloat16*>(row)[e])
                               : to_f32(static_cast<const __half*>(row)[e]);
  }
  topk_of_row<NPL>(v, experts, topk, renormalize, softmax, lane, w, id);
}

__device__ __forceinline__ int local_expert(const Params& p, int id) {
  if (id < 0 || id >= p.global_experts) return -1;
  const int e = p.emap != nullptr ? p.emap[id] : id;
  return e >= 0 && e < p.experts ? e : -1;
}

// `work(warp, warps)`: what else has to be done in front, by warps that routing does not need.
template <int kWarps, typename Work>
__device__ __forceinline__ void build_routes(const Params& p, Routes& r, uint8_t* mem, Work work) {
  constexpr int kThreads = 32 * kWarps;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int routes = p.tokens * p.topk, experts = p.experts;
  r.list = reinterpret_cast<int*>(mem);
  r.mask = reinterpret_cast<uint32_t*>(r.list + routes);
  r.off = reinterpret_cast<int*>(r.mask + routes);
  r.coef = reinterpret_cast<float*>(r.off + routes);
  r.token = reinterpret_cast<int*>(r.coef + routes);
  int* ids = r.token + routes;                               // [routes] local expert or -1
  float* wts = reinterpret_cast<float*>(ids + routes);       // [routes]
  int* totals = reinterpret_cast<int*>(wts + routes);        // [16]
  uint32_t* mask = reinterpret_cast<uint32_t*>(totals + 16); // [experts]
  const bool small = routes <= 32, one_warp = small && (p.gating == nullptr || p.tokens == 1);
  if (!one_warp) work(warp, kWarps);
  else if (warp > 0) work(warp - 1, kWarps - 1);
  if (!small)
    for (int e = tid; e < experts; e += kThreads) mask[e] = 0;
  if (p.gating != nullptr && (!one_warp || warp == 0)) {
    const int size = p.gating_dtype == BOLT_F32 ? 4 : 2;
    const int npl = (p.global_experts + 31) / 32;
    for (int m = one_warp ? 0 : warp; m < p.tokens; m += kWarps) {
      const void* row = static_cast<const uint8_t*>(p.gating) + (int64_t)m * p.global_experts * size;
      float w;
      int id;
      if (npl <= 1) route_token<1>(row, p.gating_dtype, p.global_experts, p.topk, p.renormalize, p.softmax, lane, w, id);
      else if (npl <= 4) route_token<4>(row, p.gating_dtype, p.global_experts, p.topk, p.renormalize, p.softmax, lane, w, id);
      else if (npl <= 8) route_token<8>(row, p.gating_dtype, p.global_experts, p.topk, p.renormalize, p.softmax, lane, w, id);
      else route_token<32>(row, p.gating_dtype, p.global_experts, p.topk, p.renormalize, p.softmax, lane, w, id);
      if (lane < p.topk) {
        ids[m * p.topk + lane] = local_expert(p, id);
        wts[m * p.topk + lane] = w;
      }
    }
    if (one_warp) __syncwarp();
    else __syncthreads();
  }
  if (small) {
    // one warp, a route a lane
    if (warp == 0) {
      int e = -1;
      float w = 0.f;
      if (lane < routes) {
        e = p.gating != nullptr ? ids[lane] : local_expert(p, p.ids[lane]);
        w = p.gating != nullptr ? wts[lane] : p.wts[lane];
      }
      const int m = lane / p.topk;
      // routes of the same token to the same expert are one slot, the first of them its owner
      const unsigned same = __match_any_sync(0xffffffffu, e);
      const unsigned row = p.topk == 32 ? ~0u : ((1u << p.topk) - 1u) << (m * p.topk);
      const unsigned twins = e >= 0 ? same & row : 0u;
      const bool owner = e >= 0 && lane == __ffs(twins) - 1;
      const bool leads = e >= 0 && lane == __ffs(same) - 1;          // of its expert
      float sum = 0.f;
      int before = 0, lower = 0;      // slots in front of this one, touched experts below this one
      uint32_t tokens = 0;
#pragma unroll 4
      for (int j = 0; j < routes; ++j) {
        const int ej = __shfl_sync(0xffffffffu, e, j);
        const float wj = __shfl_sync(0xffffffffu, w, j);
        const bool own = __shfl_sync(0xffffffffu, (int)owner, j) != 0, lead = __shfl_sync(0xffffffffu, (int)leads, j) != 0;
        if ((twins >> j) & 1u) sum += wj;
        if (own && (ej < e || (ej == e && j < lane))) ++before;
        if (lead && ej < e) ++lower;
        if (ej == e) tokens |= 1u << (j / p.topk);
      }
      if (owner) {
        r.coef[before] = sum;
        r.token[before] = m;
      }
      if (leads) {
        r.list[lower] = e;
        r.mask[lower] = tokens;
        r.off[lower] = before;
      }
      const unsigned leaders = __ballot_sync(0xffffffffu, leads), owners = __ballot_sync(0xffffffffu, owner);
      if (lane == 0) {
        totals[0] = __popc(leaders);
        totals[1] = __popc(owners);
      }
    }
    __syncthreads();
    r.touched = totals[0];
    r.slots = totals[1];
    return;
  }
  if (p.gating == nullptr)
    for (int i = tid; i < routes; i += kThreads) {
      ids[i] = local_expert(p, p.ids[i]);
      wts[i] = p.wts[i];
    }
  __syncthreads();
  for (int i = tid; i < routes; i += kThreads)
    if (ids[i] >= 0) atomicOr(&mask[ids[i]], 1u << (i / p.topk));
  __syncthreads();
  // exclusive sums over the experts: tokens (low half), touched experts (high half)
  int base = 0;
  for (int e0 = 0; e0 < experts; e0 += kThreads) {
    const int e = e0 + tid;
    const uint32_t tokens = e < experts ? mask[e] : 0u;
    const int c = __popc(tokens);
    const int mine = c | (c > 0 ? 0x10000 : 0);
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    if (lane == 31) totals[warp] = sum;
    __syncthreads();
    int before = base, all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += totals[w];
      all += totals[w];
    }
    before += sum - mine;
    if (c > 0) {
      const int at = before >> 16;
      r.list[at] = e;
      r.mask[at] = tokens;
      r.off[at] = before & 0xFFFF;
      mask[e] = at;               // from here on: the expert's place in the list
    }
    base += all;
    __syncthreads();
  }
  r.touched = base >> 16;
  r.slots = base & 0xFFFF;
  for (int i = tid; i < routes; i += kThreads) {
    const int e = ids[i];
    if (e < 0) continue;
    const int m = i / p.topk, first = m * p.topk, last = first + p.topk;
    bool again = false;
    float w = 0.f;
    for (int j = first; j < last; ++j) {
      const bool same = ids[j] == e;
      again |= same && j < i;
      if (same) w += wts[j];
    }
    if (again) continue;       // the same expert twice for a token: one slot, the weights' sum
    const int at = mask[e], slot = r.off[at] + __popc(r.mask[at] & ((1u << m) - 1u));
    r.coef[slot] = w;
    r.token[slot] = m;
  }
  __syncthreads();
}

__device__ __forceinline__ int slot_of(uint32_t mask, int off, int token) {
  return (mask >> token) & 1u ? off + __popc(mask & ((1u << token) - 1u)) : -1;
}

// ---------------------------------------------------------------------------
// a warp's ring of weight boxes
// ---------------------------------------------------------------------------
struct Ring {
  uint32_t base, bars;
  int slots, bytes, bytes_in;      // a slot's size, and what a copy brings
  int s_in = 0, s_out = 0;
  uint32_t ph = 0;
  __device__ void init(uint32_t smem, uint32_t bar, int n, int box_bytes, int copy_bytes) {
    bytes_in = copy_bytes;
    base = smem;
    bars = bar;
    slots = n;
    bytes = box_bytes;
  }
  // lane 0 only: the barrier and the address of the next box to bring
  __device__ __forceinline__ uint32_t next_in(uint32_t& dst) const {
    const uint32_t bar = bars + 8 * s_in;
    dst = base + s_in * bytes;
    mbar_expect_tx(bar, bytes_in);
    return bar;
  }
  __device__ __forceinline__ void advance_in() {
    if (++s_in == slots) s_in = 0;
  }
  __device__ __forceinline__ uint32_t wait(volatile int* abort_flag, int32_t* status) {
    mbar_wait(bars + 8 * s_out, ph, abort_flag, status, 30);
    return base + s_out * bytes;
  }
  __device__ __forceinline__ void release() {
    __syncwarp();
    if (++s_out == slots) {
      s_out = 0;
      ph ^= 1;
    }
  }
};

constexpr int kCtrlBytes = 1024;   // barriers and the abort flag
constexpr int kMaxBarriers = 126;  // 8 bytes each

__device__ __forceinline__ uint8_t* carve(uint8_t* raw) {
  return reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
}

// This block's run of `units`: the first units % blocks blocks have one more.
__device__ __forceinline__ void share_of(int units, int& first, int& end) {
  const int each = units / (int)gridDim.x, more = units - each * (int)gridDim.x, b = (int)blockIdx.x;
  first = b * each + min(b, more);
  end = first + each + (b < more ? 1 : 0);
}

// What both kernels begin with: barriers, the ring.
template <int kWarps>
__device__ __forceinline__ volatile int* start(Ring& ring, uint8_t* smem, int slots, int box_bytes,
                                               int bytes_in) {
  const int warp = threadIdx.x >> 5;
  uint8_t* ctrl = smem + kWarps * slots * box_bytes;
  const uint32_t bars = smem_u32(ctrl);
  if (threadIdx.x < kWarps * slots) mbar_init(bars + 8 * threadIdx.x, 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(ctrl + kCtrlBytes - 8);
  if (threadIdx.x == 0) *abort_flag = 0;
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  __syncthreads();
  ring.init(smem_u32(smem) + warp * slots * box_bytes, bars + 8 * warp * slots, slots, box_bytes, bytes_in);
  return abort_flag;
}
// A wait that ran out leaves copies in flight: give them time to land before the block's memory
// goes to another.
__device__ __forceinline__ void finish(volatile int* abort_flag) {
  __syncthreads();
  if (*abort_flag)
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
}

template <int MT, int NT, int TG>
__device__ __forceinline__ void put_sums(float* red, const float (&acc)[NT / TG][MT][TG][4], int warp, int lane,
                                         unsigned live) {
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (!((live >> nt) & 1u)) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i) red[(((warp * MT + mt) * NT + nt) * 4 + i) * 32 + lane] = acc[nt / TG][mt][nt % TG][i];
    }
}
template <int MT, int TG>
__device__ __forceinline__ void zero_sums(float (&v)[MT][TG][4]) {
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int nt = 0; nt < TG; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) v[mt][nt][i] = 0.f;
}
// Sum over the warps of element (row half r, row g of tile mt, token n).
template <int MT, int NT>
__device__ __forceinline__ float get_sum(const float* red, int warps, int mt, int r, int g, int n) {
  const int at = ((mt * NT + (n >> 3)) * 4 + 2 * r + (n & 1)) * 32 + 4 * g + ((n & 7) >> 1);
  float v = 0.f;
#pragma unroll 4
  for (int w = 0; w < warps; ++w) v += red[w * MT * NT * 128 + at];
  return v;
}

// Boxes hold up to 32 weight rows (64 for MX's gate and up rows: a block of 32 columns is quantised
// at once).  Sixteen warps an SM hide the latencies of a box that eight do not, with 128 registers a thread:
// MX above eight tokens, with its scales apart, needs more and takes eight warps.  Of the forms for more than 16
// tokens NV spills 312 bytes a thread in the first kernel, the block-scaled ones 116 and 124, the others up to 40.
constexpr int kMaxRows = 32;
constexpr int up_tiles(int k) { return k == K_MX4 ? 4 : 2; }
constexpr int up_box_bytes(int k) { return up_tiles(k) * 2048; }
constexpr int kDownTiles = kMaxRows / 16;
constexpr int kDownBoxBytes = kMaxRows * 128;
constexpr int up_scale_bytes(int k) {      // of a slot
  return k == K_NV4 ? 512 : k == K_MX4 ? 512 : is_block(k) ? 64 : 0;
}
constexpr int warps_of(int k, int nt) { return k == K_MX4 && nt > 1 ? 8 : 16; }
// Token tiles computed together; the four tiles of more than 16 tokens go one by one (few of them are live,
// and eight warps with the registers for four at once took 411 us where sixteen take 278:
// Qwen3-30B bf16, 32 tokens).
constexpr int tiles_at_once(int k, int nt) { return nt == 4 && k != K_MX4 ? 1 : nt; }
// blocks an SM holds as far as registers go: the second kernel's beside the first's
constexpr int blocks_of(int nt, int warps) { return nt == 1 && warps == 8 ? 2 : 1; }
// boxes that a warp's ring brings ahead, at most: six slots for one of eight warps with an SM's shared memory to
// themselves, three for the others
constexpr int most_pending(int warps, bool half_sm) { return warps == 8 && !half_sm ? 5 : 2; }
constexpr int red_bytes(int warps, int mt, int nt) { return warps * mt * nt * 128 * 4; }
// bytes of a kept row of codes: 16 more than it has, so that eight rows lie in different banks
__host__ __device__ constexpr int code_pitch(int k, int n) { return (int)row_bytes(k, n) + 16; }

// Rows of `cols` values to 8-bit codes in shared memory, a group of 128 values a warp and four groups at
// once: their loads travel together.
template <int K, typename RowOf, typename InvOf, typename Scale>
__device__ __forceinline__ void keep_codes(int w0, int wn, int lane, int rows, int cols, uint8_t* codes, int pitch,
                                           RowOf row_of, int dt, InvOf inv_of, Scale put_scale) {
  const int per_row = (cols + 127) / 128, all = rows * per_row;
  for (int i0 = w0; i0 < all; i0 += 4 * wn) {
    float4 v[4];
    int m[4], kb[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = i0 + j * wn;
      m[j] = i / per_row;
      kb[j] = i - m[j] * per_row;
      v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i < all && kb[j] * 128 + 4 * lane < cols) v[j] = load_values4(row_of(m[j]), dt, kb[j] * 128 + 4 * lane);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (i0 + j * wn >= all) break;
      float scale, inv;
      if constexpr (is_block(K)) {
        const float top = fmaxf(fmaxf(fabsf(v[j].x), fabsf(v[j].y)), fmaxf(fabsf(v[j].z), fabsf(v[j].w)));
        scale8<K>(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top))), scale, inv);
        if (lane == 0) put_scale(m[j], kb[j], scale);
      } else {
        inv = inv_of(m[j]);
      }
      const int c = kb[j] * 128 + 4 * lane;
      if (c < cols) *reinterpret_cast<uint32_t*>(codes + m[j] * pitch + c) = codes4<K>(v[j], inv);
    }
  }
}

// Rows to 8-bit codes in memory, a block a row: where the codes of all rows, or of all activations, do not fit
// beside a block's rings.
template <int K>
__global__ void __launch_bounds__(256) k_few_codes(const void* src, int dt, int cols, uint8_t* codes, float* scales) {
  __shared__ float top[8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  let_next_start();
  wait_for_previous();
  const int64_t row = blockIdx.x;
  const uint8_t* from = static_cast<const uint8_t*>(src) + row * cols * (dt == BOLT_F32 ? 4 : 2);
  float scale = 1.f, inv = 1.f;
  if constexpr (is_channel(K)) {
    float amax = 0.f;
    for (int c = 4 * threadIdx.x; c < cols; c += 1024) {
      const float4 v = load_values4(from, dt, c);
      amax = fmaxf(amax, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
    }
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (lane == 0) top[warp] = amax;
    __syncthreads();
    amax = top[0];
#pragma unroll
    for (int w = 1; w < 8; ++w) amax = fmaxf(amax, top[w]);
    scale8<K>(amax, scale, inv);
    if (threadIdx.x == 0) scales[row] = scale;
  }
  const int groups = (cols + 127) / 128;
  for (int kb = warp; kb < groups; kb += 8) {
    const int c = kb * 128 + 4 * lane;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (c < cols) v = load_values4(from, dt, c);
    if constexpr (is_block(K)) {
      const float most = fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w)));
      scale8<K>(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most))), scale, inv);
      if (lane == 0) scales[row * groups + kb] = scale;
    }
    if (c < cols) *reinterpret_cast<uint32_t*>(codes + row * cols + c) = codes4<K>(v, inv);
  }
}

// ---------------------------------------------------------------------------
// gate and up projections, activation
// ---------------------------------------------------------------------------
template <int K, int NT, int W>
__global__ void __launch_bounds__(32 * W, blocks_of(NT, W))
k_few_up(const __grid_constant__ CUtensorMap map, const Params p) {
  constexpr int MT = up_tiles(K), kBox = up_box_bytes(K), kWarps = W, TG = tiles_at_once(K, NT);
  constexpr int kCols = 8 * MT;       // columns a unit may have
  // rows of scales: of every gate and up row of a thread (4-bit), of the unit's gate and up block
  using Scales = ScaleRing<is_channel(K) ? (int)K_BF16 : K, is4(K) ? 2 * MT : 2>;
  static_assert(Scales::kBytes == up_scale_bytes(K), "the host reckons with a slot of this size");
  const int UC = is4(K) ? kCols : p.unit;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = carve(raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  if (tid == 0) asm volatile("prefetch.tensormap [%0];" ::"l"(&map) : "memory");
  Ring ring;
  volatile int* abort_flag = start<kWarps>(ring, smem, p.slots_per_warp, kBox, 2 * UC * 128);
  uint8_t* rest = smem + kWarps * p.slots_per_warp * kBox + kCtrlBytes;
  float* red = reinterpret_cast<float*>(rest);
  rest += red_bytes(kWarps, MT, NT);
  let_next_start();

  uint8_t* const route_mem = rest;
  rest += (route_bytes(p.experts, p.tokens * p.topk) + 15) & ~15;
  const uint32_t scale_mem = smem_u32(rest);
  rest += kWarps * p.slots_per_warp * Scales::kBytes;
  float* row_scale = reinterpret_cast<float*>(rest);       // [tokens][2]: scale, reciprocal
  if (is_channel(K)) rest += (8 * p.tokens + 15) & ~15;
  uint8_t* x_codes = rest;                                 // [tokens][pitch], scales behind them
  const int pitch = code_pitch(K, p.hidden);
  uint8_t* x_sf = x_codes + p.tokens * pitch;              // 4-bit: bytes
  float* x_scale = reinterpret_cast<float*>(x_sf);         // block-scaled: [tokens][hidden / 128]
  constexpr int kBlk = K == K_NV4 ? 16 : 32;
  const int sf_row = p.hidden / kBlk;

  // Q1 that needs whole rows, once per block.  In front of the first weights' copies: behind them a load
  // waits until they have all come.
  auto quantise = [&](int w0, int wn) {
    if (is_channel(K) && p.keep_x) {
      for (int m = w0; m < p.tokens; m += wn) {
        const uint16_t* row = static_cast<const uint16_t*>(p.x) + (int64_t)m * p.hidden;
        float amax = 0.f;
#pragma unroll 4
        for (int c = lane * 8; c < p.hidden; c += 256) {
          const uint4 u = *reinterpret_cast<const uint4*>(row + c);
          const uint32_t q[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (p.x_dtype == BOLT_BF16) {
              amax = fmaxf(amax, fabsf(__uint_as_float(q[j] << 16)));
              amax = fmaxf(amax, fabsf(__uint_as_float(q[j] & 0xFFFF0000u)));
            } else {
              const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&q[j]));
              amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
            }
          }
        }
        for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        if (lane == 0) scale8<K>(amax, row_scale[2 * m], row_scale[2 * m + 1]);
      }
      asm volatile("bar.sync 15, %0;" ::"r"(32 * wn) : "memory");
    }
    if (is8(K) && p.keep_x) {
      keep_codes<K>(w0, wn, lane, p.tokens, p.hidden, x_codes, pitch, [&](int m) {
        return static_cast<const void*>(static_cast<const uint16_t*>(p.x) + (int64_t)m * p.hidden); }, p.x_dtype,
        [&](int m) { return row_scale[2 * m + 1]; }, [&](int m, int kb, float scale) { x_scale[m * (p.hidden / 128) + kb] = scale; });
    }
    if constexpr (is4(K)) {
      const bool nv = K == K_NV4;
      const float inv_g = p.a1 != nullptr ? __frcp_rn(*p.a1) : 1.f;
      const int per_row = p.hidden / 32;
      for (int i = w0 * 32 + lane; i < p.tokens * per_row; i += wn * 32) {
        const int m = i / per_row, c = (i - m * per_row) * 32;
        float v[32];
        load_values32(v, static_cast<const uint16_t*>(p.x) + (int64_t)m * p.hidden, p.x_dtype, c);
        if (nv && p.a1 != nullptr) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] *= inv_g;
        }
        uint32_t w[4];
#pragma unroll
        for (int b = 0; b < 32 / kBlk; ++b) {
          float amax = 0.f;
#pragma unroll
          for (int j = 0; j < kBlk; ++j) amax = fp4::amax_nan(amax, v[b * kBlk + j]);
          const uint32_t byte = fp4::scale_byte<K == K_NV4>(amax);
          const fp4::Scaler sc = fp4::scaler_of<K == K_NV4>(byte);
#pragma unroll
          for (int j = 0; j < kBlk / 8; ++j)
            w[b * (kBlk / 8) + j] = fp4::codes8<K == K_NV4>(v + b * kBlk + 8 * j, sc);
          x_sf[(int64_t)m * sf_row + c / kBlk + b] = (uint8_t)byte;
        }
        *reinterpret_cast<uint4*>(x_codes + m * pitch + c / 2) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  };
  Routes r;
  build_routes<kWarps>(p, r, route_mem, quantise);

  const int per_expert = (p.inter + UC - 1) / UC;
  int u0, u1;
  share_of(r.touched * per_expert, u0, u1);
  const int nb = (int)((row_bytes(K, p.hidden) + 127) / 128);

  // The block's units go to its groups of warps in turn, the boxes of a group's units to its warps.
  const int per_group = p.group_warps, groups = kWarps / per_group;
  const int group = warp / per_group, in_group = warp - group * per_group;
  struct Place {
    int u, a, c, kb;      // unit: list[a], columns from c * UC; box of the reduction
  };
  auto settle = [&](Place& q) {
    while (q.kb >= nb) {
      q.kb -= nb;
      q.u += groups;
      q.c += groups;
      while (q.c >= per_expert) {
        q.c -= per_expert;
        ++q.a;
      }
    }
  };
  const int mine = u0 + group < u1 ? (u1 - u0 - group + groups - 1) / groups : 0;     // units of the group
  const int n_it = mine * nb > in_group ? (mine * nb - in_group + per_group - 1) / per_group : 0;
  const int first_u = u0 + group;
  Place in = {first_u, first_u / per_expert, first_u % per_expert, in_group}, cur = in;
  if (n_it > 0) {
    settle(in);
    cur = in;
  }
  int in_it = 0;
  const Scales scales = {scale_mem + (uint32_t)(warp * p.slots_per_warp) * Scales::kBytes};
  // the next box and its scales; past the last an empty group, so that groups stay one a box.  What
  // depends on the unit alone is kept from box to box.
  int in_e = 0;
  const uint8_t* in_scale = nullptr;
  auto enter = [&]() {
    in_e = r.list[in.a];
    if constexpr (is4(K)) {
      in_scale = static_cast<const uint8_t*>(p.s1) + ((int64_t)in_e * 2 * p.inter + in.c * UC + g) * sf_row;
    } else if constexpr (is_block(K)) {
      // (a unit of 8 or 16 columns lies in one block of 128)
      in_scale = static_cast<const uint8_t*>(p.s1) +
                 ((int64_t)in_e * (2 * p.inter / 128) + in.c * UC / 128) * (p.hidden / 128) * 4;
    }
  };
  if (n_it > 0) enter();
  const int half_rows = is4(K) ? p.inter * sf_row : p.inter / 128 * (p.hidden / 128) * 4;
  auto bring = [&]() {
    if (in_it < n_it) {
      if (in.kb >= nb) {
        settle(in);
        enter();
      }
      if (lane == 0) {
        uint32_t dst;
        const uint32_t bar = ring.next_in(dst);
        tma_load_4d(dst, &map, bar, in.kb * 128, in.c * UC, 0, in_e);
      }
      if constexpr (is4(K))
        scales.bring(ring.s_in, lane, in.kb, sf_row,
                     [&](int i) { return in_scale + (i & 1) * half_rows + 8 * (i >> 1) * sf_row; });
      else if constexpr (is_block(K))
        scales.bring(ring.s_in, lane, in.kb, 0, [&](int i) { return in_scale + i * half_rows + in.kb * 4; });
      ring.advance_in();
      in.kb += per_group;
      ++in_it;
    }
    cp_async_commit();
  };
  for (int i = 0; i < p.slots_per_warp; ++i) bring();

  if (is8(K) && !p.keep_x) wait_for_previous();      // k_few_codes
  const uint8_t* xq = p.keep_x ? x_codes : p.xq;
  const int xq_pitch = p.keep_x ? pitch : p.hidden;
  const float* xs = p.keep_x ? x_scale : p.xs;
  int it = 0;
  Place unit = {first_u, first_u / per_expert, first_u % per_expert, 0};
  // (the group's own barrier, named 1 to 8; a warp by itself needs none)
  auto group_sync = [&]() {
    if (per_group == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(32 * per_group) : "memory");
  };

  for (; unit.u < u1; unit.kb = nb, settle(unit)) {
    const int e = r.list[unit.a], c0 = unit.c * UC;
    const int off = r.off[unit.a], cnt = __popc(r.mask[unit.a]);
    const unsigned live = (1u << ((cnt + 7) / 8)) - 1u;
    float acc[NT / TG][MT][TG][4];
#pragma unroll
    for (int n = 0; n < NT / TG; ++n) zero_sums(acc[n]);
    int tok[NT];     // token of column g of every tile
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) tok[nt] = 8 * nt + g < cnt ? r.token[off + 8 * nt + g] : -1;

    int tok_of[NT][2];     // tokens of columns 2 t and 2 t + 1 (of a column without one: any)
    if constexpr (is_block(K)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) tok_of[nt][i] = r.token[off + min(8 * nt + 2 * t + i, cnt - 1)];
    }

    while (it < n_it && cur.u == unit.u) {
      const int kb = cur.kb;

      // what the columns of token tile nt are multiplied with
      auto load_x = [&](TokenBox<K>& x, int nt, int m) {
        if constexpr (is8(K)) {
          load_token<K>(x, m < 0 ? nullptr : xq + (int64_t)m * xq_pitch, p.hidden, kb, t);
        } else if constexpr (is16(K)) {
          load_token<K>(x, m < 0 ? nullptr : static_cast<const uint8_t*>(p.x) + (int64_t)m * p.hidden * 2,
                        p.hidden * 2, kb, t);
        } else {
          load_token<K>(x, m < 0 ? nullptr : x_codes + m * pitch, p.hidden / 2, kb, t);
          if constexpr (K == K_NV4) {
            load_block_scales<K>(x.sf, m < 0 ? nullptr : x_sf + (int64_t)m * sf_row, sf_row, kb, t);
          } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int col = 8 * nt + 2 * t + i;
              load_block_scales<K>(x.sf + 2 * i,
                                   col < cnt ? x_sf + (int64_t)r.token[off + col] * sf_row : nullptr, sf_row, kb, t);
            }
          }
        }
      };
      TokenBox<K> x[TG];
#pragma unroll
      for (int j = 0; j < TG; ++j)
        if ((live >> j) & 1u) load_x(x[j], j, tok[j]);
      RowScales<K> ws[MT];
      if constexpr (is4(K) || is_block(K)) {
        cp_async_wait<most_pending(kWarps, NT == 1)>(p.slots_per_warp - 1);
        if (K != K_NV4) __syncwarp();
        scales.read(ws, ring.s_out, lane);
      }
      const uint32_t box = ring.wait(abort_flag, p.status);
#pragma unroll
      for (int n = 0; n < NT / TG; ++n) {
        const unsigned here = live >> (n * TG);
        if (here == 0) break;
        if (n > 0) {
#pragma unroll
          for (int j = 0; j < TG; ++j) load_x(x[j], n * TG + j, tok[n * TG + j]);
        }
        if constexpr (is_block(K)) {
          float part[MT][TG][4];
          zero_sums(part);
          box_mma<K, MT, TG, true>(box, UC, lane, x, ws, here, part);
#pragma unroll
          for (int j = 0; j < TG; ++j) {
            if (!((here >> j) & 1u)) continue;
            const float x0 = xs[tok_of[n * TG + j][0] * nb + kb], x1 = xs[tok_of[n * TG + j][1] * nb + kb];
            const float sg = __uint_as_float(ws[0].sf[0][0]), su = __uint_as_float(ws[0].sf[1][0]);
            const float s0g = x0 * sg, s1g = x1 * sg, s0u = x0 * su, s1u = x1 * su;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              float(&sum)[4] = acc[n][mt][j];
              sum[0] = fmaf(part[mt][j][0], s0g, sum[0]);
              sum[1] = fmaf(part[mt][j][1], s1g, sum[1]);
              sum[2] = fmaf(part[mt][j][2], s0u, sum[2]);
              sum[3] = fmaf(part[mt][j][3], s1u, sum[3]);
            }
          }
        } else {
          box_mma<K, MT, TG, true>(box, UC, lane, x, ws, here, acc[n]);
        }
      }
      ring.release();
      bring();
      cur.kb += per_group;
      if (++it < n_it) settle(cur);
    }

    // ---- sums over the warps, activation, Q2 of the 4-bit kinds ----
    put_sums<MT, NT, TG>(red, acc, warp, lane, live);
    group_sync();
    const float* mine_red = red + group * per_group * MT * NT * 128;
    const int all = ((cnt * kCols + 31) / 32) * 32;      // whole warps take part in the exchanges
    for (int i = in_group * 32 + lane; i < all; i += 32 * per_group) {
      const int n = i / kCols, c = i % kCols, col = c0 + c;
      const bool have = n < cnt && c < UC && col < p.inter;
      const int slot = off + n;
      float a = 0.f;
      if (have) {
        float gate = get_sum<MT, NT>(mine_red, per_group, c >> 3, 0, c & 7, n);
        float up = get_sum<MT, NT>(mine_red, per_group, c >> 3, 1, c & 7, n);
        if constexpr (is_channel(K)) {
          const float* s1 = static_cast<const float*>(p.s1) + (int64_t)e * 2 * p.inter;
          const float xsc = p.keep_x ? row_scale[2 * r.token[slot]] : p.xs[r.token[slot]];
          gate *= xsc * s1[col];
          up *= xsc * s1[p.inter + col];
        } else if constexpr (is4(K)) {
          const float f = (p.g1 != nullptr ? p.g1[e] : 1.f) * (p.a1 != nullptr ? *p.a1 : 1.f);
          gate *= f;
          up *= f;
        }
        a = act_pair(p.act, gate, up);
      }
      if constexpr (is16(K)) {
        if (have) {
          const int64_t at = (int64_t)slot * p.inter + col;
          if (K == K_BF16) reinterpret_cast<__nv_bfloat16*>(p.act_rows)[at] = __float2bfloat16_rn(a);
          else reinterpret_cast<__half*>(p.act_rows)[at] = __float2half_rn(a);
        }
      } else if constexpr (is8(K)) {
        if (have) reinterpret_cast<float*>(p.act_rows)[(int64_t)slot * p.inter + col] = a;
        if constexpr (is_channel(K)) {
          float amax = fabsf(a);
#pragma unroll
          for (int o = kCols / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
          if (c == 0 && n < cnt) p.act_amax[(int64_t)slot * per_expert + unit.c] = amax;
        }
      } else {
        // a unit's columns of one slot are one block
        if (K == K_NV4 && p.a2 != nullptr) a *= __frcp_rn(*p.a2);
        float amax = fabsf(a);
#pragma unroll
        for (int o = kCols / 2; o > 0; o >>= 1) amax = fp4::amax_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        const uint32_t byte = fp4::scale_byte<K == K_NV4>(amax);
        const fp4::Scaler sc = fp4::scaler_of<K == K_NV4>(byte);
        const float q = sc.r == 0.f ? 0.f : fp4::quotient<K == K_NV4>(a, sc);
        const float other = __shfl_down_sync(0xffffffffu, q, 1);
        if (have && (c & 1) == 0)
          p.act_rows[(int64_t)slot * (p.inter / 2) + col / 2] = (uint8_t)fp4::pack2(q, other);
        if (have && c == 0) p.act_sf[(int64_t)slot * (p.inter / kBlk) + col / kBlk] = (uint8_t)byte;
      }
    }
    group_sync();
  }
  finish(abort_flag);
}

// ---------------------------------------------------------------------------
// down projection, sum over a token's experts
// ---------------------------------------------------------------------------
template <int K, int NT, int W>
__global__ void __launch_bounds__(32 * W, blocks_of(NT, W))
k_few_down(const __grid_constant__ CUtensorMap map, const Params p) {
  constexpr int MT = kDownTiles, kBox = kDownBoxBytes, kWarps = W, kThreads = 32 * kWarps,
                TG = tiles_at_once(K, NT);
  const int UR = p.unit;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = carve(raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  if (tid == 0) asm volatile("prefetch.tensormap [%0];" ::"l"(&map) : "memory");
  Ring ring;
  volatile int* abort_flag = start<kWarps>(ring, smem, p.slots_per_warp, kBox, UR * 128);
  uint8_t* rest = smem + kWarps * p.slots_per_warp * kBox + kCtrlBytes;
  float* red = reinterpret_cast<float*>(rest);
  rest += red_bytes(kWarps, MT, NT);
  Routes r;
  build_routes<kWarps>(p, r, rest, [](int, int) {});
  rest += (route_bytes(p.experts, p.tokens * p.topk) + 15) & ~15;
  using Scales = ScaleRing<K, 2 * MT>;
  const Scales scales = {smem_u32(rest) + (uint32_t)(warp * p.slots_per_warp) * Scales::kBytes};
  rest += kWarps * p.slots_per_warp * Scales::kBytes;

  const int units = (p.model_dim + UR - 1) / UR;
  int u0, u1;
  share_of(units, u0, u1);
  const int nb = (int)((row_bytes(K, p.inter) + 127) / 128);
  const int64_t boxes = (int64_t)(u1 - u0) * r.touched * nb;
  const int n_it = boxes > warp ? (int)((boxes - warp + kWarps - 1) / kWarps) : 0;

  // boxes in the order (unit, expert, place in the reduction), to the warps in turn
  struct Place {
    int u, a, kb;
  };
  auto settle = [&](Place& q) {
    while (q.kb >= nb) {
      q.kb -= nb;
      if (++q.a == r.touched) {
        q.a = 0;
        ++q.u;
      }
    }
  };
  Place in = {u0, 0, warp};
  int in_it = 0;
  constexpr int kBlk = K == K_NV4 ? 16 : 32;
  const int sf_row = p.inter / kBlk;
  // what depends on expert and unit alone is kept from box to box
  int in_e = 0;
  const uint8_t* in_scale = nullptr;
  int in_row[2 * MT];          // offsets of a thread's rows (those past the unit's: of any)
  auto enter = [&]() {
    in_e = r.list[in.a];
    const int row0 = in.u * UR + g, last = p.model_dim - 1;
    const int64_t rows_before = (int64_t)in_e * (is_block(K) ? p.model_dim / 128 : p.model_dim);
    const int row_len = is4(K) ? sf_row : is_block(K) ? p.inter / 128 * 4 : 4;
    in_scale = static_cast<const uint8_t*>(p.s2) + rows_before * row_len;
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) {
      const int row = min(row0 + 8 * i, last);
      in_row[i] = (is_block(K) ? row >> 7 : row) * row_len;
    }
  };
  if (n_it > 0) {
    settle(in);
    enter();
  }
  auto bring = [&]() {
    if (in_it < n_it) {
      if (in.kb >= nb) {
        settle(in);
        if (!is16(K)) enter();
        else in_e = r.list[in.a];
      }
      if (lane == 0) {
        uint32_t dst;
        const uint32_t bar = ring.next_in(dst);
        tma_load_3d(dst, &map, bar, in.kb * 128, in.u * UR, in_e);
      }
      if constexpr (is4(K))
        scales.bring(ring.s_in, lane, in.kb, sf_row, [&](int i) { return in_scale + in_row[i]; });
      else if constexpr (is8(K)) {
        // (each lane of four brings one of the four rows)
        static_assert(MT == 2, "four rows a thread");
        const int mine = t < 2 ? (t == 0 ? in_row[0] : in_row[1]) : (t == 2 ? in_row[2] : in_row[3]);
        scales.bring(ring.s_in, lane, in.kb, 0, [&](int) { return in_scale + mine + (is_block(K) ? in.kb * 4 : 0); });
      }
      ring.advance_in();
      in.kb += kWarps;
      ++in_it;
    }
    cp_async_commit();
  };
  for (int i = 0; i < p.slots_per_warp; ++i) bring();

  Place cur = {u0, 0, warp};
  if (n_it > 0) settle(cur);
  int it = 0;

  wait_for_previous();     // the activations
  float* row_scale = reinterpret_cast<float*>(rest);       // [slots][2]
  uint8_t* a_codes = rest + ((8 * p.tokens * p.topk + 15) & ~15);
  const int a_pitch = code_pitch(K, p.inter);
  float* a_scale = reinterpret_cast<float*>(a_codes + p.tokens * p.topk * a_pitch);     // [slots][boxes]
  if (is8(K) && p.keep_act) {
    if constexpr (is_channel(K)) {
      for (int s = warp; s < r.slots; s += kWarps) {
        float amax = 0.f;
        for (int i = lane; i < p.amax_cols; i += 32) amax = fmaxf(amax, p.act_amax[(int64_t)s * p.amax_cols + i]);
        for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        if (lane == 0) scale8<K>(amax, row_scale[2 * s], row_scale[2 * s + 1]);
      }
      __syncthreads();
    }
    keep_codes<K>(warp, kWarps, lane, r.slots, p.inter, a_codes, a_pitch, [&](int m) {
      return static_cast<const void*>(reinterpret_cast<const float*>(p.act_rows) + (int64_t)m * p.inter); }, BOLT_F32,
      [&](int m) { return row_scale[2 * m + 1]; }, [&](int m, int kb, float scale) { a_scale[m * nb + kb] = scale; });
    __syncthreads();
  }
  const uint8_t* aq = p.keep_act ? a_codes : p.aq;
  const int aq_pitch = p.keep_act ? a_pitch : p.inter;
  const float* as = p.keep_act ? a_scale : p.as;

  for (int u = u0; u < u1; ++u) {
    float acc[NT / TG][MT][TG][4];
#pragma unroll
    for (int n = 0; n < NT / TG; ++n) zero_sums(acc[n]);

    while (it < n_it && cur.u == u) {
      const int e = r.list[cur.a], kb = cur.kb;
      const uint32_t mask = r.mask[cur.a];
      const int off = r.off[cur.a];
      unsigned live = 0;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) live |= ((mask >> (8 * nt)) & 0xFFu) != 0u ? 1u << nt : 0u;

      auto load_x = [&](TokenBox<K>& x, int nt) {
        const int slot = slot_of(mask, off, 8 * nt + g);
        if constexpr (is8(K)) {
          load_token<K>(x, slot < 0 ? nullptr : aq + (int64_t)slot * aq_pitch, p.inter, kb, t);
        } else if constexpr (is16(K)) {
          load_token<K>(x, slot < 0 ? nullptr : p.act_rows + (int64_t)slot * p.inter * 2, p.inter * 2, kb, t);
        } else {
          load_token<K>(x, slot < 0 ? nullptr : p.act_rows + (int64_t)slot * (p.inter / 2), p.inter / 2, kb, t);
          if constexpr (K == K_NV4) {
            load_block_scales<K>(x.sf, slot < 0 ? nullptr : p.act_sf + (int64_t)slot * sf_row, sf_row, kb, t);
          } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int s = slot_of(mask, off, 8 * nt + 2 * t + i);
              load_block_scales<K>(x.sf + 2 * i, s < 0 ? nullptr : p.act_sf + (int64_t)s * sf_row, sf_row, kb, t);
            }
          }
        }
      };
      TokenBox<K> x[TG];
      if constexpr (TG == NT) {
#pragma unroll
        for (int j = 0; j < TG; ++j)
          if ((live >> j) & 1u) load_x(x[j], j);
      }
      const float whole = is4(K) ? (p.g2 != nullptr ? p.g2[e] : 1.f) * (p.a2 != nullptr ? *p.a2 : 1.f) : 1.f;
      RowScales<K> ws[MT];
      cp_async_wait<most_pending(kWarps, NT == 1)>(p.slots_per_warp - 1);
      if (K != K_NV4) __syncwarp();
      scales.read(ws, ring.s_out, lane);
      const uint32_t box = ring.wait(abort_flag, p.status);
#pragma unroll
      for (int n = 0; n < NT / TG; ++n) {
        const unsigned here = (live >> (n * TG)) & ((1u << TG) - 1u);
        if (here == 0) continue;
        if constexpr (TG != NT) load_x(x[0], n);
        float part[MT][TG][4];
        zero_sums(part);
        box_mma<K, MT, TG, false>(box, 0, lane, x, ws, here, part);
#pragma unroll
        for (int j = 0; j < TG; ++j) {
          if (!((here >> j) & 1u)) continue;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            // tokens that did not choose the expert get nothing (not even a NaN of its weights)
            const int slot = slot_of(mask, off, 8 * (n * TG + j) + 2 * t + i);
            if (slot < 0) continue;
            float f = r.coef[slot] * whole;
            if constexpr (is_block(K)) f *= as[slot * nb + kb];
            if constexpr (is_channel(K)) f *= p.keep_act ? row_scale[2 * slot] : p.as[slot];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              const float f0 = is8(K) ? f * __uint_as_float(ws[mt].sf[0][0]) : f;
              const float f1 = is8(K) ? f * __uint_as_float(ws[mt].sf[1][0]) : f;
              acc[n][mt][j][i] = fmaf(part[mt][j][i], f0, acc[n][mt][j][i]);
              acc[n][mt][j][2 + i] = fmaf(part[mt][j][2 + i], f1, acc[n][mt][j][2 + i]);
            }
          }
        }
      }
      ring.release();
      bring();
      cur.kb += kWarps;
      if (++it < n_it) settle(cur);
    }

    put_sums<MT, NT, TG>(red, acc, warp, lane, ~0u);
    __syncthreads();
    for (int i = tid; i < p.tokens * kMaxRows; i += kThreads) {
      const int n = i / kMaxRows, c = i % kMaxRows, col = u * UR + c;
      if (c >= UR || col >= p.model_dim) continue;
      const float v = get_sum<MT, NT>(red, kWarps, c >> 4, (c >> 3) & 1, c & 7, n) * p.out_scale;
      const int64_t at = (int64_t)n * p.model_dim + col;
      if (p.out_dtype == BOLT_BF16) static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(v);
      else if (p.out_dtype == BOLT_F16) static_cast<__half*>(p.out)[at] = __float2half_rn(v);
      else static_cast<float*>(p.out)[at] = v;
    }
    __syncthreads();
  }
  finish(abort_flag);
}

// ---------------------------------------------------------------------------
// dense 4-bit product with a few rows
// ---------------------------------------------------------------------------
// The second kernel's work without routing: units of weight rows, every row of x a column.
struct DenseParams {
  const uint8_t *x, *x_sf, *w_sf;     // codes [rows, k / 2], scale bytes [rows or n, k / block]
  const float* alpha;
  void* out;
  int out_dtype, rows, n, k, unit, slots_per_warp;
  int64_t out_ld;
  int32_t* status;
};

constexpr int dense_warps(int k, int nt) { return nt == 4 || k == K_MX4 ? 8 : 16; }
template <int K, int NT>
__global__ void __launch_bounds__(32 * dense_warps(K, NT), 1)
k_few_dense(const __grid_constant__ CUtensorMap map, const DenseParams p) {
  constexpr int MT = kDownTiles, kBox = kDownBoxBytes, kWarps = dense_warps(K, NT), kThreads = 32 * kWarps;
  const int UR = p.unit;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = carve(raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  if (tid == 0) asm volatile("prefetch.tensormap [%0];" ::"l"(&map) : "memory");
  Ring ring;
  volatile int* abort_flag = start<kWarps>(ring, smem, p.slots_per_warp, kBox, UR * 128);
  uint8_t* rest = smem + kWarps * p.slots_per_warp * kBox + kCtrlBytes;
  float* red = reinterpret_cast<float*>(rest);
  rest += red_bytes(kWarps, MT, NT);
  using Scales = ScaleRing<K, 2 * MT>;
  const Scales scales = {smem_u32(rest) + (uint32_t)(warp * p.slots_per_warp) * Scales::kBytes};

  const int units = (p.n + UR - 1) / UR;
  int u0, u1;
  share_of(units, u0, u1);
  const int nb = (p.k / 2 + 127) / 128;
  const int64_t boxes = (int64_t)(u1 - u0) * nb;
  const int n_it = boxes > warp ? (int)((boxes - warp + kWarps - 1) / kWarps) : 0;
  struct Place {
    int u, kb;
  };
  auto settle = [&](Place& q) {
    while (q.kb >= nb) {
      q.kb -= nb;
      ++q.u;
    }
  };
  Place in = {u0, warp};
  int in_it = 0;
  constexpr int kBlk = K == K_NV4 ? 16 : 32;
  const int sf_row = p.k / kBlk, row_len = p.k / 2;
  int64_t in_row[2 * MT];      // a thread's rows of scales (those past the unit's: any)
  auto enter = [&]() {
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) in_row[i] = (int64_t)min(in.u * UR + g + 8 * i, p.n - 1) * sf_row;
  };
  settle(in);
  enter();
  auto bring = [&]() {
    if (in_it < n_it) {
      if (in.kb >= nb) {
        settle(in);
        enter();
      }
      if (lane == 0) {
        uint32_t dst;
        const uint32_t bar = ring.next_in(dst);
        tma_load_3d(dst, &map, bar, in.kb * 128, in.u * UR, 0);
      }
      scales.bring(ring.s_in, lane, in.kb, sf_row, [&](int i) { return p.w_sf + in_row[i]; });
      ring.advance_in();
      in.kb += kWarps;
      ++in_it;
    }
    cp_async_commit();
  };
  for (int i = 0; i < p.slots_per_warp; ++i) bring();

  Place cur = {u0, warp};
  settle(cur);
  int it = 0;
  const unsigned live = (1u << ((p.rows + 7) / 8)) - 1u;
  const float alpha = p.alpha != nullptr ? *p.alpha : 1.f;

  for (int u = u0; u < u1; ++u) {
    float acc[1][MT][NT][4];
    zero_sums(acc[0]);
    while (it < n_it && cur.u == u) {
      auto load_x = [&](TokenBox<K>& x, int nt) {
        const int m = 8 * nt + g;
        load_token<K>(x, m < p.rows ? p.x + (int64_t)m * row_len : nullptr, row_len, cur.kb, t);
        if constexpr (K == K_NV4) {
          load_block_scales<K>(x.sf, m < p.rows ? p.x_sf + (int64_t)m * sf_row : nullptr, sf_row, cur.kb, t);
        } else {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int c = 8 * nt + 2 * t + i;
            load_block_scales<K>(x.sf + 2 * i, c < p.rows ? p.x_sf + (int64_t)c * sf_row : nullptr, sf_row, cur.kb, t);
          }
        }
      };
      RowScales<K> ws[MT];
      cp_async_wait<most_pending(kWarps, false)>(p.slots_per_warp - 1);
      if (K != K_NV4) __syncwarp();
      scales.read(ws, ring.s_out, lane);
      TokenBox<K> x[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) load_x(x[j], j);
      const uint32_t box = ring.wait(abort_flag, p.status);
      box_mma<K, MT, NT, false>(box, 0, lane, x, ws, live, acc[0]);
      ring.release();
      bring();
      cur.kb += kWarps;
      if (++it < n_it) settle(cur);
    }
    put_sums<MT, NT, NT>(red, acc, warp, lane, live);
    __syncthreads();
    for (int i = tid; i < p.rows * kMaxRows; i += kThreads) {
      const int n = i / kMaxRows, c = i % kMaxRows, col = u * UR + c;
      if (c >= UR || col >= p.n) continue;
      const float v = get_sum<MT, NT>(red, kWarps, c >> 4, (c >> 3) & 1, c & 7, n) * alpha;
      const int64_t at = (int64_t)n * p.out_ld + col;
      if (p.out_dtype == BOLT_BF16) static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(v);
      else if (p.out_dtype == BOLT_F16) static_cast<__half*>(p.out)[at] = __float2half_rn(v);
      else static_cast<float*>(p.out)[at] = v;
    }
    __syncthreads();
  }
  finish(abort_flag);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
int encode(CUtensorMap* map, const void* base, int dims, const cuuint64_t* size, const cuuint64_t* strides,
           const cuuint32_t* box) {
  const EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) {
    set_error("moe_decode: cuTensorMapEncodeTiled is not available");
    return BOLT_ERR_CUDA;
  }
  const cuuint32_t one[5] = {1, 1, 1, 1, 1};
  const CUresult rc = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, dims, const_cast<void*>(base), size, strides, box,
                         one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (rc != CUDA_SUCCESS) {
    set_error("moe_decode: cuTensorMapEncodeTiled failed (%d)", (int)rc);
    return BOLT_ERR_CUDA;
  }
  return BOLT_OK;
}

inline size_t a256(size_t n) { return (n + 255) & ~size_t(255); }
inline int a16(int n) { return (n + 15) & ~15; }

constexpr int kMinUnit = 8;
// Size of a unit, of 8 to `most`: every block gets the same number of units but for one, so the one that
// makes the largest share smallest (of two alike the larger; a unit costs about a row's time by itself).
int unit_size(int total, int most, int64_t copies, int blocks, int step = 1) {
  int best = most;
  int64_t least = INT64_MAX;
  for (int u = most; u >= kMinUnit; u -= step) {
    const int64_t units = copies * ((total + u - 1) / u);
    const int64_t share = (units + blocks - 1) / blocks * (u + 1);
    if (share < least) {
      least = share;
      best = u;
    }
  }
  return best;
}

// Warps that share a unit: as many as have four boxes of its reduction each.  With fewer boxes a warp, the
// end of a unit (sums over the warps, activation) is not covered by other groups' boxes.
int group_warps(int warps, int boxes) {
  while (warps > 1 && boxes < 4 * warps) warps /= 2;
  return warps;
}

// Bytes of the workspace's parts: activations, their 4-bit scales, their largest magnitudes, 8-bit codes and
// scales of the rows, of the activations.
constexpr int kParts = 7;
void workspace_parts(const bolt_decode_args* a, size_t (&part)[kParts]) {
  const size_t slots = (size_t)a->num_tokens * a->topk;
  const int k = a->kind;
  part[0] = a256(slots * (is8(k) ? 4 * (size_t)a->inter : (size_t)row_bytes(k, a->inter)));
  part[1] = is4(k) ? a256(slots * (a->inter / (k == K_NV4 ? 16 : 32))) : 0;
  part[2] = is_channel(k) ? a256(slots * ((a->inter + kMinUnit - 1) / kMinUnit) * 4) : 0;
  part[3] = is8(k) ? a256((size_t)a->num_tokens * a->hidden) : 0;
  part[4] = is8(k) ? a256((size_t)a->num_tokens * ((a->hidden + 127) / 128) * 4) : 0;
  part[5] = is8(k) ? a256(slots * a->inter) : 0;
  part[6] = is8(k) ? a256(slots * ((a->inter + 127) / 128) * 4) : 0;
}
size_t workspace_bytes(const bolt_decode_args* a) {
  size_t part[kParts], all = 0;
  workspace_parts(a, part);
  for (size_t n : part) all += n;
  return all;
}

// A kernel that may start while the one in front of it on the stream finishes (`early` false: it waits for that one,
// as a caller who leaves SMs to other kernels wants: blocks that start early would take those SMs and wait there).
template <typename... Params, typename... Args>
int launch_early(bool early, void (*kernel)(Params...), int blocks, int threads, int smem, cudaStream_t st,
                 const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = early ? 1 : 0;
  BOLT_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
  return BOLT_OK;
}

constexpr int kSmem = 226 * 1024, kHalfSmem = 113 * 1024;   // of a block, of one of two on an SM
int ring_slots(int smem, int fixed, int slot_bytes, int warps) {
  int slots = (smem - fixed) / (warps * slot_bytes);
  return slots * warps > kMaxBarriers ? kMaxBarriers / warps : slots;
}
// `kernels` not null: it becomes the number of kernels, and none is launched.
template <int K, int NT, int kWarps>
int launch(const bolt_decode_args* a, Params p, int blocks, cudaStream_t st, int* kernels) {
  constexpr int kSmem = blocks_of(NT, kWarps) == 2 ? kHalfSmem : bolt::few::kSmem;
  constexpr int kUpSlot = up_box_bytes(K) + up_scale_bytes(K), kDownSlot = kDownBoxBytes + ScaleRing<K, 2 * kDownTiles>::kBytes;
  const int routes = p.tokens * p.topk;
  int up = 1024 + kCtrlBytes + red_bytes(kWarps, up_tiles(K), NT) + a16(route_bytes(p.experts, routes));
  int down = 1024 + kCtrlBytes + red_bytes(kWarps, kDownTiles, NT) + a16(route_bytes(p.experts, routes));
  if (is_channel(K)) up += a16(8 * p.tokens);
  down += a16(8 * routes);
  if (is4(K)) up += p.tokens * (code_pitch(K, p.hidden) + p.hidden / (K == K_NV4 ? 16 : 32));
  if (is8(K)) {
    // codes are kept by every block for up to eight tokens, where they leave the rings two boxes a warp (a
    // launch less); making more of them 148 times over takes longer than a kernel that makes them once
    // (Qwen3-30B int8, 32 tokens: 30 us of the first kernel alone)
    const auto kept = [&](int rows, int cols) {
      return (int64_t)rows * (code_pitch(K, cols) + (is_block(K) ? cols / 128 * 4 : 0)) + 16;
    };
    const int64_t x_kept = kept(p.tokens, p.hidden), act_kept = kept(routes, p.inter);
    p.keep_x = NT == 1 && up + x_kept + 2 * kWarps * kUpSlot <= kSmem;
    if (p.keep_x) up += (int)x_kept;
    p.keep_act = NT == 1 && down + act_kept + 2 * kWarps * kDownSlot <= kSmem;
    if (p.keep_act) down += (int)act_kept;
  }
  const int up_slots = ring_slots(kSmem, up, kUpSlot, kWarps),
            down_slots = ring_slots(kSmem, down, kDownSlot, kWarps);
  if (up_slots < 1 || down_slots < 1) {
    set_error("moe_decode: %d tokens of hidden size %d do not fit in shared memory", p.tokens, p.hidden);
    return BOLT_ERR_UNSUPPORTED;
  }
  if (kernels != nullptr) {
    *kernels = 2 + (is8(K) ? !p.keep_x + !p.keep_act : 0);
    return BOLT_OK;
  }
  static std::atomic<bool> ready[2][kMaxDevices];
  int rc = configure_kernel(k_few_up<K, NT, kWarps>, kSmem, ready[0], 0, 0, 0, 0);
  if (rc == BOLT_OK) rc = configure_kernel(k_few_down<K, NT, kWarps>, kSmem, ready[1], 0, 0, 0, 0);
  if (rc != BOLT_OK) return rc;

  const int columns = is4(K) ? 8 * up_tiles(K)
                             : unit_size(p.inter, 8 * up_tiles(K), routes < p.experts ? routes : p.experts, blocks,
                                         is_block(K) ? 8 : 1);
  const int rows = unit_size(p.model_dim, kMaxRows, 1, blocks);
  const bool early = a->sm_count <= 0;
  CUtensorMap m1, m2;
  {
    const cuuint64_t kb = (cuuint64_t)row_bytes(K, p.hidden), i = p.inter;
    const cuuint64_t size[4] = {kb, i, 2, (cuuint64_t)p.experts};
    const cuuint64_t strides[3] = {kb, kb * i, 2 * kb * i};
    const cuuint32_t box[4] = {128, (cuuint32_t)columns, 2, 1};
    if ((rc = encode(&m1, a->w1, 4, size, strides, box)) != BOLT_OK) return rc;
  }
  {
    const cuuint64_t kb = (cuuint64_t)row_bytes(K, p.inter), n = p.model_dim;
    const cuuint64_t size[3] = {kb, n, (cuuint64_t)p.experts};
    const cuuint64_t strides[2] = {kb, kb * n};
    const cuuint32_t box[3] = {128, (cuuint32_t)rows, 1};
    if ((rc = encode(&m2, a->w2, 3, size, strides, box)) != BOLT_OK) return rc;
  }
  p.amax_cols = (p.inter + columns - 1) / columns;
  p.slots_per_warp = up_slots;
  p.unit = columns;
  p.group_warps = group_warps(kWarps, (int)((row_bytes(K, p.hidden) + 127) / 128));
  const int up_bytes = up + up_slots * kWarps * kUpSlot, down_bytes = down + down_slots * kWarps * kDownSlot;
  if constexpr (is8(K)) {
    if (!p.keep_x) {
      k_few_codes<K><<<p.tokens, 256, 0, st>>>(p.x, p.x_dtype, p.hidden, p.xq, p.xs);
      BOLT_LAUNCH_CHECK();
      if ((rc = launch_early(early, k_few_up<K, NT, kWarps>, blocks, 32 * kWarps, up_bytes, st, m1, p)) != BOLT_OK) return rc;
    }
  }
  if (!is8(K) || p.keep_x) {
    k_few_up<K, NT, kWarps><<<blocks, 32 * kWarps, up_bytes, st>>>(m1, p);
    BOLT_LAUNCH_CHECK();
  }
  p.slots_per_warp = down_slots;
  p.unit = rows;
  if constexpr (is8(K)) {
    if (!p.keep_act) {
      const void* act = p.act_rows;
      const int f32 = BOLT_F32;
      if ((rc = launch_early(early, k_few_codes<K>, routes, 256, 0, st, act, f32, p.inter, p.aq, p.as)) != BOLT_OK) return rc;
    }
  }
  return launch_early(early, k_few_down<K, NT, kWarps>, blocks, 32 * kWarps, down_bytes, st, m2, p);
}

// Blocks of eight warps and half an SM's shared memory where a block's share of the weights is small: the
// second kernel then starts beside the first, and its routing and first copies cost nothing.  Larger shares
// want the sixteen warps (us, these / those): 8 experts of 1024 x 512, bf16, two tokens 12.3 / 14.1; Qwen3-30B,
// nvfp4, one token (140 KB) 18.6 / 19.5, bf16, one token (510 KB) 28.3 / 26.0, two 48 / 41.
constexpr int64_t kSmallShare = 256 << 10;
template <int K>
int launch_kind(const bolt_decode_args* a, const Params& p, cudaStream_t st, int* kernels) {
  const int sms = a->sm_count > 0 ? a->sm_count : sm_count_of_current_device();
  const int64_t touched = std::min<int64_t>((int64_t)p.tokens * p.topk, p.experts);
  const int64_t share = touched * (2 * p.inter * row_bytes(K, p.hidden) + p.model_dim * row_bytes(K, p.inter)) / sms;
  if (p.tokens <= 8) {
    if (share <= kSmallShare) {
      const int rc = launch<K, 1, 8>(a, p, sms, st, kernels);
      if (rc != BOLT_ERR_UNSUPPORTED) return rc;      // (too many or too long rows for half an SM)
    }
    return launch<K, 1, warps_of(K, 1)>(a, p, sms, st, kernels);
  }
  if (p.tokens <= 16) return launch<K, 2, warps_of(K, 2)>(a, p, sms, st, kernels);
  return launch<K, 4, warps_of(K, 4)>(a, p, sms, st, kernels);
}

template <int K, int NT>
int launch_dense(const bolt_fp4_few_args* a, DenseParams p, int sms, cudaStream_t st) {
  constexpr int kWarps = dense_warps(K, NT);
  static std::atomic<bool> ready[kMaxDevices];
  int rc = configure_kernel(k_few_dense<K, NT>, kSmem, ready, 0, 0, 0, 0);
  if (rc != BOLT_OK) return rc;
  const int fixed = 1024 + kCtrlBytes + red_bytes(kWarps, kDownTiles, NT);
  constexpr int kSlot = kDownBoxBytes + ScaleRing<K, 2 * kDownTiles>::kBytes;
  p.slots_per_warp = ring_slots(kSmem, fixed, kSlot, kWarps);
  p.unit = unit_size(p.n, kMaxRows, 1, sms);
  const cuuint64_t kb = (cuuint64_t)p.k / 2;
  const cuuint64_t size[3] = {kb, (cuuint64_t)p.n, 1}, strides[2] = {kb, kb * p.n};
  const cuuint32_t box[3] = {128, (cuuint32_t)p.unit, 1};
  CUtensorMap map;
  if ((rc = encode(&map, a->w, 3, size, strides, box)) != BOLT_OK) return rc;
  const int units = (p.n + p.unit - 1) / p.unit;
  k_few_dense<K, NT><<<units < sms ? units : sms, 32 * kWarps, fixed + p.slots_per_warp * kWarps * kSlot, st>>>(
      map, p);
  BOLT_LAUNCH_CHECK();
  return BOLT_OK;
}
template <int K>
int launch_dense_kind(const bolt_fp4_few_args* a, const DenseParams& p, int sms, cudaStream_t st) {
  if (p.rows <= 8) return launch_dense<K, 1>(a, p, sms, st);
  if (p.rows <= 16) return launch_dense<K, 2>(a, p, sms, st);
  return launch_dense<K, 4>(a, p, sms, st);
}

int check_args(const bolt_decode_args* a) {
  BOLT_REQUIRE(a != nullptr, "moe_decode: null args");
  BOLT_REQUIRE(a->kind >= K_BF16 && a->kind <= K_MX4, "moe_decode: unknown kind %d", a->kind);
  BOLT_REQUIRE(a->num_tokens >= 0 && a->num_tokens <= kMaxTokens, "moe_decode: %d tokens, at most %d",
               a->num_tokens, kMaxTokens);
  BOLT_REQUIRE(a->topk > 0 && a->topk <= 32, "moe_decode: topk %d out of range", a->topk);
  BOLT_REQUIRE(a->num_experts > 0 && a->num_experts <= 1024 && a->global_num_experts > 0,
               "moe_decode: at most 1024 local experts");
  BOLT_REQUIRE(a->hidden > 0 && a->inter > 0 && a->model_dim > 0, "moe_decode: bad shape");
  const int k = a->kind;
  const int step = k == K_NV4 ? 64 : (k == K_MX4 || is_block(k)) ? 128 : is8(k) ? 16 : 8;
  BOLT_REQUIRE(a->hidden % step == 0 && a->inter % step == 0,
               "moe_decode: hidden size %d and intermediate size %d must be multiples of %d", a->hidden,
               a->inter, step);
  BOLT_REQUIRE(!is_block(k) || a->model_dim % 128 == 0, "moe_decode: output size %d must be a multiple of 128",
               a->model_dim);
  return BOLT_OK;
}

}  // namespace
}  // namespace few
}  // namespace bolt

extern "C" size_t bolt_moe_decode_workspace_bytes(const bolt_decode_args* a) {
  using namespace bolt::few;
  if (check_args(a) != BOLT_OK) return 0;
  return workspace_bytes(a) + 256;
}

namespace bolt {
namespace few {
namespace {
int check_operands(const bolt_decode_args* a) {
  const int k = a->kind;
  BOLT_REQUIRE(a->hidden_states && a->w1 && a->w2 && a->out && a->workspace, "moe_decode: null pointer");
  BOLT_REQUIRE(is16(k) || (a->w1_scale && a->w2_scale), "moe_decode: scales required");
  BOLT_REQUIRE(a->gating != nullptr || (a->topk_weights && a->topk_ids), "moe_decode: no routing");
  BOLT_REQUIRE(a->gating == nullptr || (a->global_num_experts <= 32 * kMaxPerLane && a->topk <= a->global_num_experts),
               "moe_decode: top-%d of %d experts", a->topk, a->global_num_experts);
  BOLT_REQUIRE(a->gating == nullptr || a->gating_dtype == BOLT_F32 || a->gating_dtype == BOLT_BF16 ||
                   a->gating_dtype == BOLT_F16,
               "moe_decode: bad gating dtype %d", a->gating_dtype);
  BOLT_REQUIRE(a->x_dtype == BOLT_BF16 || a->x_dtype == BOLT_F16, "moe_decode: rows must be 16-bit");
  BOLT_REQUIRE(!is16(k) || a->x_dtype == (k == K_BF16 ? BOLT_BF16 : BOLT_F16),
               "moe_decode: rows and weights of different types");
  BOLT_REQUIRE(a->out_dtype == BOLT_BF16 || a->out_dtype == BOLT_F16 || a->out_dtype == BOLT_F32,
               "moe_decode: bad output dtype %d", a->out_dtype);
  BOLT_REQUIRE(((reinterpret_cast<uintptr_t>(a->hidden_states) | reinterpret_cast<uintptr_t>(a->w1) |
                 reinterpret_cast<uintptr_t>(a->w2) | reinterpret_cast<uintptr_t>(a->workspace)) & 15) == 0,
               "moe_decode: operands must be 16-byte aligned");
  BOLT_REQUIRE(!is4(k) || ((reinterpret_cast<uintptr_t>(a->w1_scale) | reinterpret_cast<uintptr_t>(a->w2_scale)) & 3) == 0,
               "moe_decode: scale bytes must be 4-byte aligned");
  BOLT_REQUIRE(a->workspace_bytes >= workspace_bytes(a), "moe_decode: workspace too small");
  return BOLT_OK;
}

int decode_once(const bolt_decode_args* a, cudaStream_t st, int* kernels) {
  int rc = check_args(a);
  if (rc != BOLT_OK) return rc;
  if (kernels != nullptr) *kernels = 0;
  if (a->num_tokens == 0) return BOLT_OK;
  if (kernels == nullptr && (rc = check_operands(a)) != BOLT_OK) return rc;
  size_t part[kParts];
  workspace_parts(a, part);

  Params p = {};
  p.x = a->hidden_states;
  p.x_dtype = a->x_dtype;
  p.out_dtype = a->out_dtype;
  p.tokens = a->num_tokens;
  p.topk = a->topk;
  p.hidden = a->hidden;
  p.inter = a->inter;
  p.model_dim = a->model_dim;
  p.experts = a->num_experts;
  p.global_experts = a->global_num_experts;
  p.s1 = a->w1_scale;
  p.s2 = a->w2_scale;
  p.g1 = a->w1_global_scale;
  p.g2 = a->w2_global_scale;
  p.a1 = a->a1_global_scale;
  p.a2 = a->a2_global_scale;
  p.wts = a->topk_weights;
  p.ids = a->topk_ids;
  p.gating = a->gating;
  p.gating_dtype = a->gating_dtype;
  p.renormalize = a->renormalize;
  p.softmax = a->is_softmax;
  p.emap = a->expert_map;
  p.act = {a->activation, 1, a->act_alpha, a->act_limit};
  p.out_scale = a->routed_scaling_factor;
  p.out = a->out;
  p.act_rows = static_cast<uint8_t*>(a->workspace);
  p.act_sf = p.act_rows + part[0];
  p.act_amax = reinterpret_cast<float*>(p.act_sf + part[1]);
  p.xq = p.act_sf + part[1] + part[2];
  p.xs = reinterpret_cast<float*>(p.xq + part[3]);
  p.aq = p.xq + part[3] + part[4];
  p.as = reinterpret_cast<float*>(p.aq + part[5]);
  p.status = a->status;

  switch (a->kind) {
    case K_BF16: return launch_kind<K_BF16>(a, p, st, kernels);
    case K_F16: return launch_kind<K_F16>(a, p, st, kernels);
    case K_F8_BLOCK: return launch_kind<K_F8_BLOCK>(a, p, st, kernels);
    case K_I8_CHANNEL: return launch_kind<K_I8_CHANNEL>(a, p, st, kernels);
    case K_F8_CHANNEL: return launch_kind<K_F8_CHANNEL>(a, p, st, kernels);
    case K_I8_BLOCK: return launch_kind<K_I8_BLOCK>(a, p, st, kernels);
    case K_NV4: return launch_kind<K_NV4>(a, p, st, kernels);
    default: return launch_kind<K_MX4>(a, p, st, kernels);
  }
}
// (`kernels` as in launch)
int decode(const bolt_decode_args* a, cudaStream_t st, int* kernels) {
  const int rc = decode_once(a, st, kernels);
  if (rc != BOLT_ERR_UNSUPPORTED || a->num_tokens < 2) return rc;
  // the 4-bit codes of all rows do not fit in shared memory: half of the tokens after the other (they read
  // the experts that both touch twice)
  bolt_decode_args part = *a;
  part.num_tokens = a->num_tokens / 2;
  const int first = decode(&part, st, kernels);
  if (first != BOLT_OK) return first;
  const int64_t done = part.num_tokens;
  part.num_tokens = a->num_tokens - part.num_tokens;
  part.hidden_states = static_cast<const uint8_t*>(a->hidden_states) + done * a->hidden * 2;
  if (a->gating != nullptr) {
    part.gating = static_cast<const uint8_t*>(a->gating) + done * a->global_num_experts * dtype_bytes(a->gating_dtype);
  } else {
    part.topk_ids = a->topk_ids + done * a->topk;
    part.topk_weights = a->topk_weights + done * a->topk;
  }
  part.out = static_cast<uint8_t*>(a->out) + done * a->model_dim * dtype_bytes(a->out_dtype);
  int more = 0;
  const int second = decode(&part, st, kernels != nullptr ? &more : nullptr);
  if (kernels != nullptr) *kernels += more;
  return second;
}
}  // namespace
}  // namespace few
}  // namespace bolt

extern "C" int bolt_moe_decode(const bolt_decode_args* a, void* stream) {
  return bolt::few::decode(a, static_cast<cudaStream_t>(stream), nullptr);
}

extern "C" int bolt_moe_decode_kernel_count(const bolt_decode_args* a) {
  int kernels = 0;
  return bolt::few::decode(a, nullptr, &kernels) == BOLT_OK ? kernels : -1;
}

extern "C" int bolt_fp4_gemm_few(const bolt_fp4_few_args* a, void* stream) {
  using namespace bolt;
  using namespace bolt::few;
  BOLT_REQUIRE(a != nullptr, "fp4_gemm_few: null args");
  BOLT_REQUIRE(a->format == BOLT_FP4_NV || a->format == BOLT_FP4_MX, "fp4_gemm_few: unknown format %d", a->format);
  const bool nv = a->format == BOLT_FP4_NV;
  BOLT_REQUIRE(a->rows >= 0 && a->rows <= kMaxTokens && a->n >= 0 && a->k > 0 && a->k % (nv ? 64 : 128) == 0,
               "fp4_gemm_few: %d rows (at most %d) of %d columns (multiples of %d)", a->rows, kMaxTokens, a->k,
               nv ? 64 : 128);
  if (a->rows == 0 || a->n == 0) return BOLT_OK;
  BOLT_REQUIRE(a->x && a->x_scale && a->w && a->w_scale && a->out, "fp4_gemm_few: null pointer");
  BOLT_REQUIRE(((reinterpret_cast<uintptr_t>(a->x) | reinterpret_cast<uintptr_t>(a->w) |
                 reinterpret_cast<uintptr_t>(a->x_scale) | reinterpret_cast<uintptr_t>(a->w_scale)) & 15) == 0,
               "fp4_gemm_few: operands must be 16-byte aligned");
  BOLT_REQUIRE((a->out_dtype == BOLT_BF16 || a->out_dtype == BOLT_F16 || a->out_dtype == BOLT_F32) &&
                   a->out_ld >= a->n && reinterpret_cast<uintptr_t>(a->out) % dtype_bytes(a->out_dtype) == 0,
               "fp4_gemm_few: bad output");
  DenseParams p = {};
  p.x = static_cast<const uint8_t*>(a->x);
  p.x_sf = static_cast<const uint8_t*>(a->x_scale);
  p.w_sf = static_cast<const uint8_t*>(a->w_scale);
  p.alpha = a->alpha;
  p.out = a->out;
  p.out_dtype = a->out_dtype;
  p.rows = a->rows;
  p.n = a->n;
  p.k = a->k;
  p.out_ld = a->out_ld;
  p.status = a->status;
  const int sms = a->sm_count > 0 ? a->sm_count : sm_count_of_current_device();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return nv ? launch_dense_kind<K_NV4>(a, p, sms, st) : launch_dense_kind<K_MX4>(a, p, sms, st);
}
