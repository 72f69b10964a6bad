// 4-bit rows x 4-bit weights on the tensor cores' block-scaled 4-bit kind.
//
// tcgen05.mma with kind::mxf4nvf4 (E4M3 scales per 16 values) or kind::mxf4 (E8M0 per 32) multiplies
// packed e2m1 codes with both operands' block scales inside the instruction; the fp32 accumulator stays
// in TMEM over the whole reduction.  A tile is 128 rows x BN weight rows, a K block 256 values: 128
// bytes of a row, one 128-byte-swizzled box.
//
// The instruction reads scales from TMEM, which takes them from shared memory in 512-byte tiles of 128
// rows x 4 scales (byte (r % 32) * 16 + (r / 32) * 4 + i).  A small kernel in front, k_tile_scales, lays
// the scales of rows and weights out like that (an eighth of the codes' bytes); the product then brings
// them with the operands by bulk copies.  Doing it inside the product, through registers of spare warps,
// was measured first: the writes have to be made visible to the tensor core's proxy once per K block,
// and the product ran at 2700 TFLOP/s where it runs at 4000 without any scales (8192 x 7168 x 4096).
//
// Warp 0 brings boxes and scales, warp 1 issues the instructions, warp 3 the scales' copies to TMEM, warps
// 4 to 11 drain the accumulator.  Rows are read in sorted order: bringing them by token inside the
// product, four an instruction (tile::gather4, 68 cycles each) or by 16-byte copies of a spare warp, cost
// more than a sorted copy of the codes (DeepSeek-V3, 64 experts, 1500 tokens: GEMM 1 905 us by gather4).
#include <cuda.h>

#include <atomic>

#include "act_pair.cuh"
#include "fp4.cuh"
#include "row_store.cuh"
#include "tc_ptx.cuh"
#include "tensor_map.cuh"

namespace bolt {
namespace fp4gemm {
namespace {
using namespace tc;

constexpr int kThreads = 384;
constexpr int kBM = 128;
constexpr int kTmemCols = 512;
constexpr int kABytes = kBM * 128;
constexpr int kSets = 4;                 // of scale columns: 4 x 48 and 256 sums fit TMEM
constexpr int kOutBytes = 1024;          // per epilogue warp: 32 rows x 32 bytes

template <bool NV, int BN>
struct Shape {
  static constexpr int kTiles = NV ? 4 : 2;                 // 512-byte scale tiles of a K block
  static constexpr int kBlocks = 1 + BN / 128;              // of 128 rows: A, then B
  static constexpr int kSfBytes = kBlocks * kTiles * 512;
  static constexpr int kSfCols = kBlocks * kTiles * 4;      // of TMEM
  static constexpr int kBBytes = BN * 128;
  static constexpr int kStageBytes = kABytes + kBBytes + kSfBytes;
  static constexpr int kStages = (226 * 1024 - 2048 - 8 * kOutBytes) / ((kStageBytes + 1023) / 1024 * 1024);
  // operands first (1024-byte aligned), then the scales of all stages
  static constexpr int kOperandBytes = kABytes + kBBytes;
  static constexpr int kSmemBytes = 1024 + kStages * kStageBytes + 1024 + 8 * kOutBytes;
};

struct Params {
  const uint8_t *sfa, *sfb;              // tiles: [row block][K / 64 or K / 128][512], B per expert
  const float *alpha, *a_global, *b_global, *c_global;
  void* c;
  uint8_t* c_scale;
  int c_dtype;
  int64_t c_ld;
  int c_vec_ok;
  int rows, n, n_half, k, num_experts, capacity;
  int num_kb, k_tiles;                   // K blocks; scale tiles along K
  int n_blocks;                          // 128-row blocks of an expert's weights
  int tiles_n, group_m;
  int num_tokens;
  const int32_t *sorted_ids, *expert_ids, *num_valid;
  const float* sorted_weights;
  ActParams act;
  int32_t* status;
  uint32_t idesc;
};

template <bool NV>
__device__ __forceinline__ void mma_fp4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa,
                                        uint32_t sfb, uint32_t accumulate) {
  if (NV)
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %6, 0;\n"
        "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], "
        "p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %6, 0;\n"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], "
        "p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}

struct Tile {
  int m, n, expert;      // row tile, column tile; expert -1: nothing to do
};
// Tiles go row tile first within groups of group_m row tiles, so that the blocks of a wave share weight
// tiles through L2.
__device__ __forceinline__ Tile tile_of(const Params& p, int i, int num_m) {
  const int per_group = p.group_m * p.tiles_n;
  const int group = i / per_group, m0 = group * p.group_m;
  const int gm = min(num_m - m0, p.group_m), in = i - group * per_group;
  Tile t;
  t.n = in / gm;
  t.m = m0 + in - t.n * gm;
  t.expert = p.expert_ids != nullptr ? p.expert_ids[t.m] : 0;
  if (t.expert >= p.num_experts) t.expert = -1;
  return t;
}
// SiLU(gate) * up, with the hardware's reciprocal (within one step of the rounded one, 2^-23 of the value, where a
// 4-bit code resolves 2^-2: a true division would be longer for nothing); the other activations as a call, since an epilogue written out for every sum of a
// thread is bound by instruction fetch (with all of them inline the gated product took 418 us where
// its instructions take 100: 128 experts x 2 x 1536 x 4096).
__device__ __noinline__ float other_activation(ActParams p, float g, float u) { return act_pair(p, g, u); }
__device__ __forceinline__ float silu_mul(float g, float u) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + expf(-g)));
  return g * r * u;
}

template <bool NV, int BN, bool GATED>
__global__ void __launch_bounds__(kThreads, 1)
k_fp4_gemm(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_b, const Params p) {
  using S = Shape<NV, BN>;
  constexpr int kStages = S::kStages, kTiles = S::kTiles, kNB = BN / 128;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sf_mem = smem + kStages * S::kOperandBytes;
  uint8_t* ctrl = sf_mem + kStages * S::kSfBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(ctrl);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(ctrl + 512);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(ctrl + 516);
  const uint32_t smem_base = smem_u32(smem), sf_base = smem_u32(sf_mem);
  const uint32_t bar_full = smem_u32(bars), bar_empty = bar_full + 8 * kStages;
  const uint32_t bar_tfull = bar_empty + 8 * kStages, bar_tempty = bar_tfull + 8;
  const uint32_t bar_sf = bar_tempty + 8, bar_sf_free = bar_sf + 8 * kSets;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    mbar_init(bar_tfull, 1);
    mbar_init(bar_tempty, 8);
    for (int s = 0; s < kSets; ++s) {
      mbar_init(bar_sf + 8 * s, 1);
      mbar_init(bar_sf_free + 8 * s, 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"((uint32_t)kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  const int num_m = p.num_valid != nullptr ? min(*p.num_valid, p.capacity) / kBM : (p.rows + kBM - 1) / kBM;
  const int total = num_m * p.tiles_n;

  if (warp == 0) {
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int i = blockIdx.x; ok && i < total; i += gridDim.x) {
        const Tile t = tile_of(p, i, num_m);
        if (t.expert < 0) continue;
        const uint8_t* sfa = p.sfa + (int64_t)t.m * p.k_tiles * 512;
        const uint8_t* sfb[kNB];       // (a block that does not exist: any, its columns go nowhere)
#pragma unroll
        for (int b = 0; b < kNB; ++b)
          sfb[b] = p.sfb + ((int64_t)t.expert * p.n_blocks + min(t.n * kNB + b, p.n_blocks - 1)) * p.k_tiles * 512;
        for (int kb = 0; kb < p.num_kb; ++kb) {
          ok = mbar_wait(bar_empty + 8 * s, ph ^ 1, abort_flag, p.status, 40);
          if (!ok) break;
          const uint32_t full = bar_full + 8 * s, sa = smem_base + s * S::kOperandBytes;
          const uint32_t sf = sf_base + s * S::kSfBytes;
          const uint32_t sf_bytes = min(kTiles, p.k_tiles - kb * kTiles) * 512;
          mbar_expect_tx(full, kABytes + S::kBBytes + S::kBlocks * sf_bytes);
          bulk_load(sf, sfa + (int64_t)kb * kTiles * 512, sf_bytes, full);
#pragma unroll
          for (int b = 0; b < kNB; ++b)
            bulk_load(sf + (1 + b) * kTiles * 512, sfb[b] + (int64_t)kb * kTiles * 512, sf_bytes, full);
          tma_load_2d(sa, &tma_a, full, kb * 128, t.m * kBM);
          if (GATED) {
#pragma unroll
            for (int j = 0; j < BN / 64; ++j)
              tma_load_3d(sa + kABytes + j * 8192, &tma_b, full, kb * 128,
                          (j & 1) * p.n_half + t.n * (BN / 2) + (j >> 1) * 64, t.expert);
          } else {
            tma_load_3d(sa + kABytes, &tma_b, full, kb * 128, t.n * BN, t.expert);
          }
          if (++s == kStages) { s = 0; ph ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0, tph = 0, set = 0, sph = 0;
      bool ok = true;
      for (int i = blockIdx.x; ok && i < total; i += gridDim.x) {
        const Tile t = tile_of(p, i, num_m);
        if (t.expert < 0) continue;
        ok = mbar_wait(bar_tempty, tph ^ 1, abort_flag, p.status, 41);
        if (!ok) break;
        tc_fence_after();
        for (int kb = 0; kb < p.num_kb; ++kb) {
          ok = mbar_wait(bar_full + 8 * s, ph, abort_flag, p.status, 42) &&
               mbar_wait(bar_sf + 8 * set, sph, abort_flag, p.status, 43);
          if (!ok) break;
          tc_fence_after();
          const uint32_t sa = smem_base + s * S::kOperandBytes;
          const uint64_t adesc = make_smem_desc(sa), bdesc = make_smem_desc(sa + kABytes);
          const uint32_t sfa_t = tmem_base + BN + set * S::kSfCols, sfb_t = sfa_t + 4 * kTiles;
          const int steps = min(4, (p.k - kb * 256) / 64);    // 64 values an instruction
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (j >= steps) break;
            // NV: a step's four scales are one tile; MX: two steps share one, each has two bytes of four
            const int tile = NV ? j : j >> 1;
            const uint32_t id = NV ? 0u : (uint32_t)(j & 1) * 2u;
            mma_fp4<NV>(tmem_base, adesc + 2 * j, bdesc + 2 * j, p.idesc | (id << 4) | (id << 29),
                        sfa_t + 4 * tile, sfb_t + 4 * kNB * tile, (kb > 0 || j > 0) ? 1u : 0u);
          }
          tc_commit(bar_empty + 8 * s);
          tc_commit(bar_sf_free + 8 * set);
          if (++s == kStages) { s = 0; ph ^= 1; }
          if (++set == kSets) { set = 0; sph ^= 1; }
        }
        if (ok) tc_commit(bar_tfull);
        tph ^= 1;
      }
    }
  } else if (warp == 3) {
    // ------------------------------ scales to TMEM ------------------------------
    // A thread of its own issues the copies, into kSets sets of columns by turns: behind the instructions
    // of the thread that issues those they would wait for them, and they for the copies.
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0, set = 0, sph = 0;
      bool ok = true;
      for (int i = blockIdx.x; ok && i < total; i += gridDim.x) {
        const Tile t = tile_of(p, i, num_m);
        if (t.expert < 0) continue;
        for (int kb = 0; kb < p.num_kb; ++kb) {
          ok = mbar_wait(bar_full + 8 * s, ph, abort_flag, p.status, 42) &&
               mbar_wait(bar_sf_free + 8 * set, sph ^ 1, abort_flag, p.status, 43);
          if (!ok) break;
          tc_fence_after();
          const uint32_t sf = sf_base + s * S::kSfBytes;
          const uint32_t sfa_t = tmem_base + BN + set * S::kSfCols, sfb_t = sfa_t + 4 * kTiles;
          const int tiles = min(kTiles, p.k_tiles - kb * kTiles);
#pragma unroll
          for (int j = 0; j < kTiles; ++j) {
            if (j >= tiles) break;
            tc_cp_sf(sfa_t + 4 * j, make_sf_desc(sf + j * 512));
#pragma unroll
            for (int b = 0; b < kNB; ++b)
              tc_cp_sf(sfb_t + 4 * (kNB * j + b), make_sf_desc(sf + ((1 + b) * kTiles + j) * 512));
          }
          tc_commit(bar_sf + 8 * set);
          if (++s == kStages) { s = 0; ph ^= 1; }
          if (++set == kSets) { set = 0; sph ^= 1; }
        }
      }
    }
  } else if (warp >= 4) {
    // ------------------------------ epilogue ------------------------------
    constexpr int kCols = BN / 2;                  // columns of this warp's half
    const int q = warp & 3, h = (warp - 4) >> 2, row_in_tile = 32 * q + lane;
    const uint32_t acc = tmem_base + ((uint32_t)(32 * q) << 16) + h * kCols;
    uint8_t* stage = ctrl + 1024 + (warp - 4) * kOutBytes;
    float whole = (p.alpha != nullptr ? *p.alpha : 1.f) * (p.a_global != nullptr ? *p.a_global : 1.f);
    float inv_c = 1.f;
    if (GATED && p.c_global != nullptr) inv_c = __frcp_rn(*p.c_global);
    uint32_t tph = 0;
    for (int i = blockIdx.x; i < total; i += gridDim.x) {
      const Tile t = tile_of(p, i, num_m);
      if (t.expert < 0) continue;
      const int row = t.m * kBM + row_in_tile;
      const bool live = p.sorted_ids != nullptr ? (p.sorted_ids[row] & 0xFFFFFF) < p.num_tokens : row < p.rows;
      float f = whole;
      if (p.b_global != nullptr) f *= p.b_global[t.expert];
      if (p.sorted_weights != nullptr && live) f *= p.sorted_weights[row];
      if (!mbar_wait(bar_tfull, tph, abort_flag, p.status, 41)) break;
      tph ^= 1;
      tc_fence_after();
      // the accumulator is handed back before anything is converted: the next tile's instructions
      // wait for it
      uint32_t raw[kCols / 32][32];
#pragma unroll
      for (int j = 0; j < kCols / 32; ++j) tmem_ld32(acc + 32 * j, raw[j]);
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_tempty);
      if constexpr (!GATED) {
        const int col0 = t.n * BN + h * kCols;
        const int64_t row_off = (int64_t)row * p.c_ld;
#pragma unroll
        for (int j = 0; j < kCols / 32; ++j) {
          float v[32];
#pragma unroll
          for (int x = 0; x < 32; ++x) v[x] = __uint_as_float(raw[j][x]) * f;
          const int col = col0 + 32 * j;
          if (p.c_vec_ok && p.c_dtype != BOLT_F32 && col + 32 <= p.n) {
            // 32 rows x 32 bytes at a time through shared memory: a store instruction then writes
            // whole sectors of sixteen rows
            uint4 u[4];
            pack32_16bit(v, p.c_dtype, u);
            const unsigned live_mask = __ballot_sync(0xffffffffu, live);
            uint8_t* c8 = static_cast<uint8_t*>(p.c) + ((int64_t)(row - lane) * p.c_ld + col) * 2;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const int sw = (lane >> 2) & 1;
              *reinterpret_cast<uint4*>(stage + lane * 32 + (sw << 4)) = u[2 * half];
              *reinterpret_cast<uint4*>(stage + lane * 32 + ((sw ^ 1) << 4)) = u[2 * half + 1];
              __syncwarp();
#pragma unroll
              for (int pass = 0; pass < 2; ++pass) {
                const int r = 16 * pass + (lane >> 1), piece = lane & 1;
                const uint4 o = *reinterpret_cast<const uint4*>(stage + r * 32 + ((piece ^ ((r >> 2) & 1)) << 4));
                if ((live_mask >> r) & 1u)
                  *reinterpret_cast<uint4*>(c8 + (int64_t)r * p.c_ld * 2 + 32 * half + 16 * piece) = o;
              }
              __syncwarp();
            }
          } else if (live) {
            store_row32(p.c, p.c_dtype, row_off, col, p.n, v);
          }
        }
      } else {
        // half h: 64 gate columns, then the 64 up columns of the output columns from col0 on
        static_assert(!GATED || kCols == 128, "a thread holds 64 gate columns and their up columns");
        constexpr int kBlk = NV ? 16 : 32;
        const int col0 = t.n * (BN / 2) + 64 * h;
        if (col0 < p.n_half) {
          uint8_t* codes = static_cast<uint8_t*>(p.c) + ((int64_t)row * p.n_half + col0) / 2;
          // the next product's A scales, in its tiles already: one word (NV) or half of one (MX)
          constexpr int kSpan = 4 * kBlk;        // columns of a tile
          uint8_t* scales = p.c_scale + ((int64_t)t.m * (p.n_half / kSpan) + col0 / kSpan) * 512 +
                            (row_in_tile & 31) * 16 + (row_in_tile >> 5) * 4 + (NV ? 0 : (col0 / kBlk) & 3);
          uint32_t words[8], bytes = 0;
#pragma unroll
          for (int b = 0; b < 64 / kBlk; ++b) {
            float v[kBlk], amax = 0.f;
#pragma unroll
            for (int x = 0; x < kBlk; ++x) {
              const int c = b * kBlk + x;
              const float gate = __uint_as_float(raw[c >> 5][c & 31]) * f;
              const float up = __uint_as_float(raw[2 + (c >> 5)][c & 31]) * f;
              v[x] = (p.act.kind == BOLT_ACT_SILU ? silu_mul(gate, up) : other_activation(p.act, gate, up)) * inv_c;
              amax = fp4::amax_nan(amax, v[x]);
            }
            if (!live) amax = 0.f;
            const uint32_t byte = fp4::scale_byte<NV>(amax);
            fp4::Scaler sc = fp4::scaler_of<NV>(byte);
            if (!live) sc.r = 0.f;
#pragma unroll
            for (int x = 0; x < kBlk / 8; ++x) words[b * (kBlk / 8) + x] = fp4::codes8<NV>(v + 8 * x, sc);
            bytes |= byte << (8 * b);
          }
          *reinterpret_cast<uint4*>(codes) = make_uint4(words[0], words[1], words[2], words[3]);
          *reinterpret_cast<uint4*>(codes + 16) = make_uint4(words[4], words[5], words[6], words[7]);
          if (NV) *reinterpret_cast<uint32_t*>(scales) = bytes;
          else *reinterpret_cast<uint16_t*>(scales) = (uint16_t)bytes;
        }
      }
    }
  }

  // ------------------------------ teardown ------------------------------
  __syncwarp();
  if (*abort_flag) {
    for (int i = 0; i < 200; ++i) __nanosleep(1000);   // copies in flight land before the block's memory goes
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)kTmemCols)
                 : "memory");
}

// ---------------------------------------------------------------------------
// scales into the instruction's tiles
// ---------------------------------------------------------------------------
// A warp takes 128 rows and 16 bytes of each (four tiles): lane l reads the pieces of rows l, l + 32,
// l + 64 and l + 96 and writes lane l's 16 bytes of every tile, 512 consecutive bytes a warp.
struct TileParams {
  bolt_fp4_tile_job job[BOLT_FP4_TILE_JOBS];
  int blocks[BOLT_FP4_TILE_JOBS];       // 128-row blocks of an expert
  int64_t warps[BOLT_FP4_TILE_JOBS];    // blocks * experts * 16-byte pieces of a row
  int jobs, experts;
  const int32_t *sorted_ids, *expert_ids, *num_valid;
  int num_tokens, capacity;
};

__global__ void __launch_bounds__(256) k_tile_scales(const TileParams p) {
  const int lane = threadIdx.x & 31;
  // experts that no tile names are left alone
  extern __shared__ uint32_t named[];
  const int num_m = p.num_valid != nullptr ? min(*p.num_valid, p.capacity) / kBM : 0;
  const int experts = p.experts;
  if (p.expert_ids != nullptr) {
    for (int i = threadIdx.x; i < (experts + 31) / 32; i += blockDim.x) named[i] = 0u;
    __syncthreads();
    for (int i = threadIdx.x; i < num_m; i += blockDim.x) {
      const int e = p.expert_ids[i];
      if (e >= 0 && e < experts) atomicOr(&named[e >> 5], 1u << (e & 31));
    }
    __syncthreads();
  }
  const int64_t first = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int64_t step = ((int64_t)gridDim.x * blockDim.x) >> 5;
  for (int j = 0; j < p.jobs; ++j) {
    const bolt_fp4_tile_job& job = p.job[j];
    const bool vec_ok = job.row_bytes % 16 == 0;
    const int pieces = (job.row_bytes + 15) / 16;
    for (int64_t i = first; i < p.warps[j]; i += step) {
      const int64_t eb = i / pieces;
      const int piece = (int)(i - eb * pieces), e = (int)(eb / p.blocks[j]);
      const int b = (int)(eb - (int64_t)e * p.blocks[j]);
      if (job.by_sorted_id ? b >= num_m : (p.expert_ids != nullptr && !((named[e >> 5] >> (e & 31)) & 1u))) continue;
      uint4 v[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int r = lane + 32 * q;
        int row;
        if (job.by_sorted_id) {
          row = p.sorted_ids[b * 128 + r] & 0xFFFFFF;
          if (row >= p.num_tokens) row = -1;
        } else if (job.gated_half > 0) {
          const int col = b * 64 + (r & 63);
          row = col < job.gated_half ? (r >> 6) * job.gated_half + col : -1;
        } else {
          row = b * 128 + r < job.rows ? b * 128 + r : -1;
        }
        v[q] = make_uint4(0u, 0u, 0u, 0u);
        if (row < 0) continue;
        const uint8_t* src = static_cast<const uint8_t*>(job.src) + ((int64_t)e * job.rows + row) * job.row_bytes + piece * 16;
        if (vec_ok) {
          v[q] = *reinterpret_cast<const uint4*>(src);
        } else {
          uint32_t w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            w[k] = piece * 16 + 4 * k < job.row_bytes ? *reinterpret_cast<const uint32_t*>(src + 4 * k) : 0u;
          v[q] = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
      uint8_t* dst = static_cast<uint8_t*>(job.dst) + (eb * (job.row_bytes / 4) + piece * 4) * 512 + lane * 16;
      const uint4 out[4] = {make_uint4(v[0].x, v[1].x, v[2].x, v[3].x), make_uint4(v[0].y, v[1].y, v[2].y, v[3].y),
                            make_uint4(v[0].z, v[1].z, v[2].z, v[3].z), make_uint4(v[0].w, v[1].w, v[2].w, v[3].w)};
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (piece * 16 + 4 * k < job.row_bytes) *reinterpret_cast<uint4*>(dst + 512 * k) = out[k];
    }
  }
}

template <bool NV, int BN, bool GATED>
int launch(const CUtensorMap& ma, const CUtensorMap& mb, const Params& p, int grid, cudaStream_t st) {
  static std::atomic<bool> ready[kMaxDevices];
  const int rc = configure_kernel(k_fp4_gemm<NV, BN, GATED>, Shape<NV, BN>::kSmemBytes, ready, 0, 0, 0, 0);
  if (rc != BOLT_OK) return rc;
  k_fp4_gemm<NV, BN, GATED><<<grid, kThreads, Shape<NV, BN>::kSmemBytes, st>>>(ma, mb, p);
  BOLT_LAUNCH_CHECK();
  return BOLT_OK;
}

template <bool NV>
int launch_format(bool gated, int bn, const CUtensorMap& ma, const CUtensorMap& mb, const Params& p, int grid,
                  cudaStream_t st) {
  if (gated) return launch<NV, 256, true>(ma, mb, p, grid, st);
  if (bn == 128) return launch<NV, 128, false>(ma, mb, p, grid, st);
  return launch<NV, 256, false>(ma, mb, p, grid, st);
}

int blocks_of(int rows, int gated_half) { return gated_half > 0 ? (gated_half + 63) / 64 : (rows + kBM - 1) / kBM; }

}  // namespace
}  // namespace fp4gemm
}  // namespace bolt

extern "C" int bolt_fp4_tile_scales(const bolt_fp4_tile_args* a, void* stream) {
  using namespace bolt;
  using namespace bolt::fp4gemm;
  BOLT_REQUIRE(a != nullptr && a->jobs >= 0 && a->jobs <= BOLT_FP4_TILE_JOBS, "fp4_tile_scales: bad arguments");
  BOLT_REQUIRE(a->expert_ids == nullptr || (a->num_valid_ids && a->sorted_ids && a->capacity % kBM == 0),
               "fp4_tile_scales: the sort's arrays go together");
  TileParams p = {};
  int64_t warps = 0;
  for (int j = 0; j < a->jobs; ++j) {
    const bolt_fp4_tile_job& job = a->job[j];
    BOLT_REQUIRE(job.rows >= 0 && job.experts > 0 && job.row_bytes >= 0 && job.row_bytes % 4 == 0,
                 "fp4_tile_scales: bad shape");
    BOLT_REQUIRE(!job.by_sorted_id || (a->expert_ids && job.experts == 1 && job.gated_half == 0),
                 "fp4_tile_scales: rows through sorted ids need the sort's arrays");
    BOLT_REQUIRE(job.gated_half >= 0 && (job.gated_half == 0 || job.rows == 2 * job.gated_half),
                 "fp4_tile_scales: gated rows are two halves");
    const int blocks = job.by_sorted_id ? a->capacity / kBM : blocks_of(job.rows, job.gated_half);
    const int64_t n = (int64_t)blocks * job.experts * ((job.row_bytes + 15) / 16);
    if (n == 0) continue;
    BOLT_REQUIRE(job.src && job.dst && reinterpret_cast<uintptr_t>(job.src) % (job.row_bytes % 16 == 0 ? 16 : 4) == 0 &&
                     reinterpret_cast<uintptr_t>(job.dst) % 16 == 0,
                 "fp4_tile_scales: scales must be aligned to 16 bytes (rows of whole 16 bytes) or 4");
    p.job[p.jobs] = job;
    p.blocks[p.jobs] = blocks;
    p.warps[p.jobs++] = n;
    warps += n;
    if (!job.by_sorted_id && job.experts > p.experts) p.experts = job.experts;
  }
  if (p.jobs == 0) return BOLT_OK;
  p.sorted_ids = a->sorted_ids;
  p.expert_ids = a->expert_ids;
  p.num_valid = a->num_valid_ids;
  p.num_tokens = a->num_tokens;
  p.capacity = a->capacity;
  const int64_t want = (warps + 7) / 8, most = (int64_t)sm_count_of_current_device() * 8;
  const int smem = p.expert_ids != nullptr ? (p.experts + 31) / 32 * 4 : 0;
  BOLT_REQUIRE(smem <= 48 * 1024, "fp4_tile_scales: too many experts");
  k_tile_scales<<<(unsigned)(want < most ? want : most), 256, smem, static_cast<cudaStream_t>(stream)>>>(p);
  BOLT_LAUNCH_CHECK();
  return BOLT_OK;
}

extern "C" int bolt_fp4_gemm(const bolt_fp4_gemm_args* a, void* stream) {
  using namespace bolt;
  using namespace bolt::fp4gemm;
  BOLT_REQUIRE(a != nullptr, "fp4_gemm: null args");
  BOLT_REQUIRE(a->format == BOLT_FP4_NV || a->format == BOLT_FP4_MX, "fp4_gemm: unknown format %d", a->format);
  const bool nv = a->format == BOLT_FP4_NV, grouped = a->sorted_expert_ids != nullptr;
  const bool gated = a->epilogue == BOLT_EPI_SILU_MUL_QUANT;
  const int step = nv ? 64 : 128, block = nv ? 16 : 32;
  BOLT_REQUIRE(gated || a->epilogue == BOLT_EPI_STORE, "fp4_gemm: unknown epilogue %d", a->epilogue);
  BOLT_REQUIRE(a->rows >= 0 && a->n >= 0 && a->k > 0 && a->num_experts > 0, "fp4_gemm: bad shape");
  BOLT_REQUIRE(a->k % step == 0, "fp4_gemm: k %d must be a multiple of %d", a->k, step);
  BOLT_REQUIRE(!gated || (grouped && a->n % 2 == 0 && (a->n / 2) % step == 0),
               "fp4_gemm: the quantising epilogue is grouped and needs n / 2 in multiples of %d", step);
  BOLT_REQUIRE(grouped || (a->num_experts == 1 && a->sorted_ids == nullptr && a->sorted_weights == nullptr && a->num_valid_ids == nullptr),
               "fp4_gemm: dense operands have no sorted order");
  BOLT_REQUIRE(!grouped || (a->num_valid_ids && a->sorted_ids && a->capacity >= 0 && a->capacity % kBM == 0 &&
                            a->num_tokens >= 0 && a->rows >= a->capacity),
               "fp4_gemm: grouped operands need the sort's arrays and a capacity in whole tiles");
  const int all_rows = grouped ? a->capacity : a->rows;
  if (all_rows == 0 || a->n == 0 || (grouped && a->num_tokens == 0)) return BOLT_OK;
  BOLT_REQUIRE(a->a && a->a_tiles && a->b && a->b_tiles && a->c && (!gated || a->c_scale), "fp4_gemm: null pointer");
  BOLT_REQUIRE(((reinterpret_cast<uintptr_t>(a->a) | reinterpret_cast<uintptr_t>(a->a_tiles) |
                 reinterpret_cast<uintptr_t>(a->b) | reinterpret_cast<uintptr_t>(a->b_tiles)) & 15) == 0,
               "fp4_gemm: operands must be 16-byte aligned");
  if (gated)
    BOLT_REQUIRE(reinterpret_cast<uintptr_t>(a->c) % 16 == 0 && reinterpret_cast<uintptr_t>(a->c_scale) % 4 == 0,
                 "fp4_gemm: quantised output must be 16-byte aligned");
  else
    BOLT_REQUIRE((a->c_dtype == BOLT_BF16 || a->c_dtype == BOLT_F16 || a->c_dtype == BOLT_F32) && a->c_ld >= a->n &&
                     reinterpret_cast<uintptr_t>(a->c) % dtype_bytes(a->c_dtype) == 0,
                 "fp4_gemm: bad output");

  Params p = {};
  p.alpha = a->alpha;
  p.a_global = a->a_global;
  p.b_global = a->b_global;
  p.c_global = a->c_global;
  p.c = a->c;
  p.c_scale = static_cast<uint8_t*>(a->c_scale);
  p.c_dtype = a->c_dtype;
  p.c_ld = a->c_ld;
  p.c_vec_ok = !gated && reinterpret_cast<uintptr_t>(a->c) % 16 == 0 &&
               a->c_ld * dtype_bytes(a->c_dtype) % 16 == 0;
  p.rows = a->rows;
  p.n = a->n;
  p.n_half = a->n / 2;
  p.k = a->k;
  p.num_experts = a->num_experts;
  p.capacity = a->capacity;
  p.num_kb = (a->k + 255) / 256;
  p.k_tiles = a->k / (4 * block);
  p.n_blocks = blocks_of(a->n, gated ? a->n / 2 : 0);
  p.sfa = static_cast<const uint8_t*>(a->a_tiles);
  p.sfb = static_cast<const uint8_t*>(a->b_tiles);
  p.num_tokens = a->num_tokens;
  p.sorted_ids = a->sorted_ids;
  p.expert_ids = a->sorted_expert_ids;
  p.num_valid = a->num_valid_ids;
  p.sorted_weights = a->sorted_weights;
  p.act = {a->activation, 1, a->act_alpha, a->act_limit};
  p.status = a->status;

  const int sms = a->sm_count > 0 ? a->sm_count : sm_count_of_current_device();
  const int64_t tiles_m = (all_rows + kBM - 1) / kBM;
  // Column tiles of 128 where they save a wave: a K block of one takes about 0.6 of the time of one of
  // 256 (8192 x 7168 x 4096, NV: 256 columns 148 us; 777 x 4096 x 7168, MX: 128 columns 33 us, 256 22).
  auto waves = [&](int cols) { return (tiles_m * ((a->n + cols - 1) / cols) + sms - 1) / sms; };
  const int bn = !gated && 6 * waves(128) < 10 * waves(256) ? 128 : 256;
  p.tiles_n = gated ? (p.n_half + 127) / 128 : (a->n + bn - 1) / bn;
  p.group_m = grouped ? 4 : 16;
  // e2m1 x e2m1 (format 1), E4M3 or (bit 23) E8M0 scales, N >> 3 at bit 17, M >> 4 at bit 24
  p.idesc = (1u << 7) | (1u << 10) | ((uint32_t)(bn >> 3) << 17) | (nv ? 0u : 1u << 23) | ((uint32_t)(kBM >> 4) << 24);

  const EncodeTiledFn encode = encode_fn();
  if (encode == nullptr) {
    set_error("fp4_gemm: cuTensorMapEncodeTiled is unavailable");
    return BOLT_ERR_CUDA;
  }
  CUtensorMap ma, mb;
  const cuuint32_t ones[3] = {1, 1, 1};
  const cuuint64_t kb = (cuuint64_t)a->k / 2;
  {
    const cuuint64_t size[2] = {kb, (cuuint64_t)a->rows}, strides[1] = {kb};
    const cuuint32_t box[2] = {128, kBM};
    const CUresult rc = encode(&ma, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(a->a), size, strides, box, ones,
                               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) {
      set_error("fp4_gemm: tensor map for the rows failed (%d)", (int)rc);
      return BOLT_ERR_CUDA;
    }
  }
  {
    const cuuint64_t size[3] = {kb, (cuuint64_t)a->n, (cuuint64_t)a->num_experts}, strides[2] = {kb, kb * a->n};
    const cuuint32_t box[3] = {128, (cuuint32_t)(gated ? 64 : bn), 1};
    const CUresult rc = encode(&mb, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(a->b), size, strides, box, ones,
                               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) {
      set_error("fp4_gemm: tensor map for the weights failed (%d)", (int)rc);
      return BOLT_ERR_CUDA;
    }
  }
  const int64_t tiles = tiles_m * p.tiles_n;
  BOLT_REQUIRE(tiles < (1ll << 31), "fp4_gemm: too many tiles");
  const int grid = (int)(tiles < sms ? tiles : sms);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return nv ? launch_format<true>(gated, bn, ma, mb, p, grid, st) : launch_format<false>(gated, bn, ma, mb, p, grid, st);
}
