// Products grouped by expert with ragged sizes (a mixture of experts' Linear layers):
//   out[s, :] = epilogue( a[rows ? rows[s] : s, :] * w[e]^T + bias[e] ),   offsets[e] <= s < offsets[e + 1].
// The offsets live on the device (the router wrote them), so the host launches one wave of persistent CTAs and every
// CTA works the tile list out for itself: the prefix over the experts of their row tiles, times the column tiles.
//
// Three kernels.  On CTA pairs (256 x 256 tiles, cta_group::2, each CTA loads its 128 rows of A and half of W) for large
// products of some 500 rows an expert and more; on single CTAs (128 rows, 64 to 256 columns) below, where the weights' bytes count and the
// number of tiles is what spreads their stream over the SMs; and for a handful of rows in all (serving a token or two) dot
// products by warps, which have neither tensor maps to build nor a pipeline to fill.
//
// Operands: 128-byte K slabs in a ring of 128B-swizzled stages, W by TMA, and A too.  With `rows` the single-CTA kernel
// gathers A four rows a copy (tile::gather4, four warps: within 2 to 8 % of rows in order; 16-byte cp.async into the same
// places takes 1.5 times as long, its writes compete with the tensor core for shared memory).  The pair kernel would
// gather every row again for each of its column tiles; there a pass at copy bandwidth that puts the rows in order first,
// in caller scratch, is the better one (16384 x 5120 x 1280: 162 us against 160 us, but 127 against 135 us in int8, and 752
// against 764 us at 65536 rows under the power cap).
//
// Measured, one B200: 65536 x 5120 x 1280 bf16 with 16 experts, gathered, bias and GELU: 640 us = 1.34 PFLOP/s (one dense
// product of that size: 578 us here, 587 us by the vendor library); 16384 x 5120 x 1280 int8: 111 us = 1.9 POP/s (rows in order 102, even
// experts 96, one dense product 91); 2062 x 1280 x 5120 f16: 48 us, 4.9 TB/s; one token with two experts of 5120 x 1280, weights in
// HBM: 10.2 us, 2.6 TB/s (13.2 us gathered with bias and GELU).
//
// A tile computes all its rows whatever its expert has left (the rows behind them in shared memory may be anything: a
// row of the product depends on its own row of A alone), but stores only its own: whole tiles leave by TMA, the last
// ones of an expert row by row.
#include <atomic>

#include "elem16.cuh"
#include "overlap.h"

namespace samb {
namespace {

constexpr int BM = 128;
constexpr int BN = 256;
constexpr int SLAB_BYTES = 128;
constexpr int A_STAGE_BYTES = BM * SLAB_BYTES;
constexpr int NUM_ACC = 2;
constexpr int TMEM_COLS = NUM_ACC * BN;
constexpr int OUT_STAGE_BYTES = BM * 128;
constexpr int kMaxExperts = 512;

enum { kTypeBf16 = 0, kTypeF16 = 1, kTypeI8 = 2 };

struct GroupedParams {
  void* out;
  const uint8_t* a;
  const float* bias;               // [E, N] or null
  const float* a_scale;            // int8: per row of A
  const float* w_scale;            // int8: [E, N]
  const int* rows;                 // gather indexes, or null
  const int* offsets;              // [E + 1]
  int* status;
  long long ldo, a_rows, S;
  long long a_pitch;               // bytes between rows of A
  int E, N, K;
  int k_bytes, k_slabs, last_ksteps;
};

// mbar_wait by a warp in step; each lane has its own answer.  A wait that runs out may run out for some lanes only (a
// phase can complete between two lanes' last looks), and a lane that left its role alone would never come to the
// elect.sync and __syncwarp that the others go on to.  So the lanes keep their answers for themselves: one that has given up
// waits and issues no more (`ok` stays false), goes through the rest of the tile with its warp, and the warp
// votes at the tile's end and leaves its role together.  (A vote after every wait of the MMA warp cost 4 to 7 % of a large
// product: 145 against 139 us at 16384 x 5120 x 1280, and 163 us when one lane alone walks the loop.)
__device__ __noinline__ bool warp_wait_long(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status, uint32_t site) {
  return mbar_wait(bar, parity, abort_flag, status, site);
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status, uint32_t site) {
  if (mbar_try_wait(bar, parity)) return true;
  return warp_wait_long(bar, parity, abort_flag, status, site);
}

// The tile list, by one warp: first[e] = row tiles (of tile_rows) before expert e, start[e] = its first slot.  Offsets
// are clamped to [0, S] and made to rise, so that no list can point outside the buffers.  Returns the row tiles.
__device__ __forceinline__ int tile_list(const GroupedParams& p, int tile_rows, int* first, int* start) {
  const int lane = threadIdx.x & 31;
  int tiles = 0, at = 0;
  for (int e0 = 0; e0 < p.E; e0 += 32) {
    const int e = e0 + lane;
    int lo = 0, hi = 0;
    if (e < p.E) {
      lo = min(max(__ldg(p.offsets + e), 0), int(p.S));
      hi = min(max(__ldg(p.offsets + e + 1), 0), int(p.S));
    }
    int top = max(lo, hi);                               // largest offset up to this expert
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, top, o);
      if (lane >= o) top = max(top, up);
    }
    top = max(top, at);
    int below = __shfl_up_sync(0xffffffffu, top, 1);
    if (lane == 0) below = e0 == 0 ? lo : at;
    const int begin = max(lo, below), n = max(0, hi - begin);
    const int mine = (n + tile_rows - 1) / tile_rows;
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    if (e < p.E) {
      first[e] = tiles + sum - mine;
      start[e] = begin;
      if (e == p.E - 1) start[p.E] = begin + n;
    }
    tiles += __shfl_sync(0xffffffffu, sum, 31);
    at = __shfl_sync(0xffffffffu, top, 31);
  }
  if (lane == 0) first[p.E] = tiles;
  return tiles;
}

// Where a tile lies.  Tiles are numbered expert by expert, row tile by row tile, column tile by column tile; a role
// walks its tiles in rising order, so the expert only ever moves forward.
struct TileWalk {
  const int* first;
  const int* start;
  int tiles_n, tile_rows, e, m0, rows, ntile;
  __device__ __forceinline__ TileWalk(const int* f, const int* s, int tn, int tr)
      : first(f), start(s), tiles_n(tn), tile_rows(tr), e(0), m0(0), rows(0), ntile(0) {}
  __device__ __forceinline__ void at(int tile) {
    const int mt = tile / tiles_n;
    ntile = tile - mt * tiles_n;
    while (first[e + 1] <= mt) ++e;
    m0 = start[e] + (mt - first[e]) * tile_rows;
    rows = min(tile_rows, start[e + 1] - m0);
  }
};

// Four rows of a 2-D tensor, 128 bytes each, into 512 consecutive (swizzled) bytes; `m` has boxes one row high.
__device__ __forceinline__ void tma_gather4(void* smem_dst, const CUtensorMap* m, uint64_t* bar, int x, const int (&r)[4]) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
      ::"r"(smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(x), "r"(r[0]), "r"(r[1]),
      "r"(r[2]), "r"(r[3])
      : "memory");
}

// A wait gave up somewhere: the producer sees its copies in flight home before the CTA ends.  Those whose barrier will
// not complete any more (a partner stopped in between), and products that were issued before their warp's vote, get a tenth of
// a millisecond, many times what either takes; only then does the tensor memory go back.
template <int STAGES>
__device__ __forceinline__ void drain_copies(uint64_t* full_bar, uint32_t issued) {
  for (uint32_t i = issued > STAGES ? issued - STAGES : 0u; i < issued; ++i)
    for (uint32_t n = 0; n < 4096u && !mbar_try_wait(&full_bar[i % STAGES], (i / STAGES) & 1u); ++n) __nanosleep(64);
  for (int n = 0; n < 100; ++n) __nanosleep(1000);
}

__device__ __forceinline__ bool epi_all(bool pred) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\t"
      "bar.red.and.pred p, 1, 256, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r)
      : "r"(uint32_t(pred))
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void epi_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// ---------------------------------------------------------------------------------------------- single CTAs
constexpr int ONE_STAGES = 4;
constexpr int ONE_STAGE_BYTES = A_STAGE_BYTES + BN * SLAB_BYTES;
constexpr int A_BOX_ROWS = 32;                           // up to 64 rows of A: only the boxes that hold some are loaded
constexpr int A_BOX_BYTES = A_BOX_ROWS * SLAB_BYTES;
constexpr int ONE_THREADS = 64 + 256;                    // producer, MMA, eight epilogue warps
constexpr int GATHER_WARPS = 4, GATHER_GROUPS = BM / 4 / GATHER_WARPS;
constexpr int ONE_SMEM_BYTES = ONE_STAGES * ONE_STAGE_BYTES + OUT_STAGE_BYTES + 2 * BN * 4 + 2 * (kMaxExperts + 1) * 4 + 1024 + 256;

template <int kType, bool kGelu, bool kGather>
__global__ void __launch_bounds__(ONE_THREADS + (kGather ? 32 * GATHER_WARPS : 0), 1)
grouped_one_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmA32,
                   const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmOut, const GroupedParams p) {
  constexpr bool kInt8 = kType == kTypeI8;
  constexpr int STAGES = ONE_STAGES, STAGE_BYTES = ONE_STAGE_BYTES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* stage_out = smem + STAGES * STAGE_BYTES;
  float* s_bias = reinterpret_cast<float*>(stage_out + OUT_STAGE_BYTES);
  float* s_wscale = s_bias + BN;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(s_wscale + BN);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* acc_full = empty_bar + STAGES;
  uint64_t* acc_empty = acc_full + NUM_ACC;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + NUM_ACC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* s_bn = reinterpret_cast<int*>(tmem_slot + 2);
  int* s_first = reinterpret_cast<int*>(tmem_slot + 4);
  int* s_start = s_first + kMaxExperts + 1;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1 + (kGather ? GATHER_WARPS : 0));
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < NUM_ACC; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], 8);
    }
    fence_mbar_init();
    tma_prefetch_desc(&tmA);
    if (!kGather) tma_prefetch_desc(&tmA32);
    tma_prefetch_desc(&tmB);
    tma_prefetch_desc(&tmOut);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  if (warp == 2) {
    const int tiles = tile_list(p, BM, s_first, s_start);
    if (lane == 0) {
      // Column tile: waves x what a tile takes, in columns a K step: its own, as much as 64 more for its rows, and some 1000
      // in all for its start and epilogue.  A last wave that is mostly empty makes narrower tiles the better ones (2560
      // rows of 16 experts, 1280 x 5120: 192 columns 65 us, 256 columns 73 us).
      long long best = 0;
      int bn = BN;
      for (int w = BN; w >= 64; w -= 64) {
        const long long t = (long long)tiles * ((p.N + w - 1) / w);
        const long long cost = ((t + gridDim.x - 1) / gridDim.x) * ((long long)p.k_slabs * (w + 64) + 1000);
        if (w == BN || cost < best) { best = cost; bn = w; }
      }
      *s_bn = bn;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int bn = *s_bn;
  const int tiles_n = (p.N + bn - 1) / bn;
  const int num_tiles = s_first[p.E] * tiles_n;
  constexpr int slab_elems = kInt8 ? SLAB_BYTES : SLAB_BYTES / 2;
  TileWalk w(s_first, s_start, tiles_n, BM);
  uint32_t issued = 0;                                   // slabs that the producer has sent for

  if (warp == 0) {
    // ------------------------------------------------------------------ producer
    uint32_t stage = 0, phase = 0;
    bool ok = true;
    for (int tile = blockIdx.x; ok && tile < num_tiles; tile += gridDim.x) {
      w.at(tile);
      const int n0 = w.ntile * bn;
      const int a_boxes = w.rows > 2 * A_BOX_ROWS ? BM / A_BOX_ROWS : (w.rows + A_BOX_ROWS - 1) / A_BOX_ROWS;
      for (int ks = 0; ks < p.k_slabs; ++ks) {
        ok = ok && warp_wait(&empty_bar[stage], phase ^ 1u, abort_flag, p.status, 1);
        uint8_t* sa = smem + stage * STAGE_BYTES;
        uint64_t* bar = &full_bar[stage];
        if (elect_one() && ok) {
          mbar_expect_tx(bar, (kGather ? (w.rows + 3) / 4 * 512 : a_boxes * A_BOX_BYTES) + bn * SLAB_BYTES);
          if (!kGather) {
            if (a_boxes == BM / A_BOX_ROWS) {
              tma_load_2d(sa, &tmA, bar, ks * slab_elems, w.m0);
            } else {
              tma_load_2d(sa, &tmA32, bar, ks * slab_elems, w.m0);
              if (a_boxes == 2) tma_load_2d(sa + A_BOX_BYTES, &tmA32, bar, ks * slab_elems, w.m0 + A_BOX_ROWS);
            }
          }
#pragma unroll
          for (int b = 0; b < BN / 64; ++b)
            if (b * 64 < bn)
              tma_load_3d(sa + A_STAGE_BYTES + b * (64 * SLAB_BYTES), &tmB, bar, ks * slab_elems, n0 + b * 64, w.e);
        }
        __syncwarp();
        if (ok) ++issued;
        if (++stage == STAGES) { stage = 0; phase ^= 1u; }
      }
      ok = __all_sync(0xffffffffu, ok);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issue
    const uint32_t idesc = kInt8 ? make_idesc(kAccS32, kFmtS8, kFmtS8, BM, bn)
                                 : make_idesc(kAccF32, kType == kTypeF16 ? kFmtF16 : kFmtBF16,
                                              kType == kTypeF16 ? kFmtF16 : kFmtBF16, BM, bn);
    const uint64_t desc0 = make_smem_desc(smem_u32(smem), 16, 1024, kSwizzle128B);
    uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
    bool ok = true;
    for (int tile = blockIdx.x; ok && tile < num_tiles; tile += gridDim.x) {
      ok = warp_wait(&acc_empty[acc], acc_phase ^ 1u, abort_flag, p.status, 2);
      tc_fence_after();
      const uint32_t d_tmem = tmem_base + acc * BN;
      for (int ks = 0; ks < p.k_slabs; ++ks) {
        ok = ok && warp_wait(&full_bar[stage], phase, abort_flag, p.status, 3);
        tc_fence_after();
        if (elect_one() && ok) {
          const uint64_t adesc = desc0 + stage * (STAGE_BYTES / 16);
          const uint64_t bdesc = adesc + A_STAGE_BYTES / 16;
          const int nsteps = ks == p.k_slabs - 1 ? p.last_ksteps : 4;
#pragma unroll
          for (int k4 = 0; k4 < 4; ++k4) {
            if (k4 >= nsteps) break;
            const uint32_t accumulate = (ks | k4) != 0 ? 1u : 0u;
            if (kInt8) umma_i8_ss(d_tmem, adesc + k4 * 2, bdesc + k4 * 2, idesc, accumulate);
            else umma_f16_ss(d_tmem, adesc + k4 * 2, bdesc + k4 * 2, idesc, accumulate);
          }
          tc_commit(&empty_bar[stage]);
        }
        __syncwarp();
        if (++stage == STAGES) { stage = 0; phase ^= 1u; }
      }
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      if (elect_one()) tc_commit(&acc_full[acc]);
      __syncwarp();
      if (++acc == NUM_ACC) { acc = 0; acc_phase ^= 1u; }
    }
  } else if (kGather && warp >= ONE_THREADS / 32) {
    // ------------------------------------------------------------------ gathering warps
    // Warp g fetches the rows 4 (4 j + g) .. + 3 of the tile for every slab.  Their indexes are spread over the warp's
    // registers once a tile: the copy takes them from uniform registers, and shuffling them there for every slab, or
    // one lane a copy, made a copy cost 60 to 85 cycles of issue.
    const int g = warp - ONE_THREADS / 32;
    uint32_t stage = 0, phase = 0;
    bool ok = true;
    for (int tile = blockIdx.x; ok && tile < num_tiles; tile += gridDim.x) {
      w.at(tile);
      int mine[4], r[GATHER_GROUPS][4];                  // lane j: the rows of group j
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int m = ((lane & (GATHER_GROUPS - 1)) * GATHER_WARPS + g) * 4 + q;
        const int i = m < w.rows ? __ldg(p.rows + w.m0 + m) : 0;
        mine[q] = i >= 0 && i < p.a_rows ? i : 0;        // outside A: any row, the epilogue drops its product
      }
#pragma unroll
      for (int j = 0; j < GATHER_GROUPS; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) r[j][q] = __shfl_sync(0xffffffffu, mine[q], j);
      for (int ks = 0; ks < p.k_slabs; ++ks) {
        ok = ok && warp_wait(&empty_bar[stage], phase ^ 1u, abort_flag, p.status, 8);
        uint8_t* sa = smem + stage * STAGE_BYTES + g * 512;
        if (elect_one() && ok) {
#pragma unroll
          for (int j = 0; j < GATHER_GROUPS; ++j)
            if ((j * GATHER_WARPS + g) * 4 < w.rows)
              tma_gather4(sa + j * (GATHER_WARPS * 512), &tmA, &full_bar[stage], ks * slab_elems, r[j]);
          mbar_arrive(&full_bar[stage]);                 // a warp without rows must not fall behind either
        }
        __syncwarp();
        if (++stage == STAGES) { stage = 0; phase ^= 1u; }
      }
      ok = __all_sync(0xffffffffu, ok);
    }
  } else {
    // ------------------------------------------------------------------ epilogue
    const uint32_t lane_base = uint32_t(warp & 3) * 32u;
    const int half = (warp - 2) >> 2;
    const int erow = int(lane_base) + lane;
    const int et = int(threadIdx.x) - 64;
    uint32_t acc = 0, acc_phase = 0;
    for (int tile = blockIdx.x; tile < num_tiles; tile += gridDim.x) {
      w.at(tile);
      const int n0 = w.ntile * bn;
      {
        const int n = n0 + et;
        const bool inside = et < bn && n < p.N;
        s_bias[et] = inside && p.bias != nullptr ? __ldg(p.bias + (long long)w.e * p.N + n) : 0.f;
        if (kInt8) s_wscale[et] = inside ? __ldg(p.w_scale + (long long)w.e * p.N + n) : 0.f;
      }
      float a_scale = 1.f;
      bool there = true;                                 // this row's index points into A (else: a row of zeros)
      if ((kGather || kInt8) && erow < w.rows) {
        const int i = p.rows != nullptr ? __ldg(p.rows + w.m0 + erow) : w.m0 + erow;
        there = i >= 0 && i < p.a_rows;
        if (kInt8 && there) a_scale = __ldg(p.a_scale + i);
      }
      const bool got = mbar_wait(&acc_full[acc], acc_phase, abort_flag, p.status, 4);
      __syncwarp();                                      // the barrier takes warps in step
      if (!epi_all(got)) break;                          // also publishes the column vectors
      tc_fence_after();
      const uint32_t t_addr = tmem_base + (lane_base << 16) + acc * BN + half * 32;
      const bool whole = w.rows == BM;
#pragma unroll 1
      for (int c = 0; c < bn / 64; ++c) {
        const int col0 = n0 + c * 64;
        if (col0 >= p.N) break;                          // the same for every warp
        uint32_t r[32];
        tmem_ld_32x32b_x32(t_addr + c * 64, r);
        tmem_ld_wait();
        if (kGather && !there) {
#pragma unroll
          for (int j = 0; j < 32; ++j) r[j] = 0u;
        }
        uint4 packed[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          float v[8];
          const int ct0 = c * 64 + half * 32 + u * 8;
          epilogue8<kInt8, kInt8, true, kGelu>(r + u * 8, a_scale, s_wscale + ct0, s_bias + ct0, v);
          packed[u] = kType == kTypeF16 ? F16::pack(v) : Bf16::pack(v);
        }
        if (et == 0) tma_store_wait_read<0>();           // the staging tile's last store has read it
        epi_sync();
        uint8_t* srow = stage_out + erow * 128;
#pragma unroll
        for (int u = 0; u < 4; ++u)
          *reinterpret_cast<uint4*>(srow + (((half * 4 + u) ^ (erow & 7)) << 4)) = packed[u];
        if (whole) fence_proxy_async_smem();
        epi_sync();
        if (whole) {
          if (et == 0) {
            tma_store_2d(&tmOut, stage_out, col0, w.m0);  // clipped at the row end
            tma_store_commit();
          }
        } else {
          // eight threads a row: the rows behind the tile's own belong to the next expert, or to nobody
          const int unit = et & 7;
          for (int m = et >> 3; m < w.rows; m += 32)
            if (col0 + unit * 8 < p.N)
              *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + (w.m0 + (long long)m) * p.ldo + col0 + unit * 8) =
                  *reinterpret_cast<const uint4*>(stage_out + m * 128 + ((unit ^ (m & 7)) << 4));
        }
      }
      tc_fence_before();
      mbar_arrive_warp(&acc_empty[acc]);
      if (++acc == NUM_ACC) { acc = 0; acc_phase ^= 1u; }
    }
    if (et == 0) tma_store_wait_all<0>();
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {                                     // the same for every thread: all roles have ended
    if (warp == 0) drain_copies<STAGES>(full_bar, issued);
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// ---------------------------------------------------------------------------------------------- CTA pairs
// One MMA (M 256, N 256) issued by the pair's leader reads A and half of W from each CTA's shared memory.  Roles per
// CTA: warp 0 W (and A) by TMA, warp 1 MMA issue (leader), kEpiWarps epilogue warps for the CTA's own 128 rows, an output
// warp that sends each staged 64-column chunk and hands its staging tile back.  `full` lives in the leader, where both
// CTAs' copies are counted.
__host__ __device__ constexpr int pair_stages(bool int8) { return int8 ? 5 : 6; }
__host__ __device__ constexpr int pair_out_bufs(bool int8) { return int8 ? 3 : 1; }
constexpr int PAIR_STAGE_BYTES = A_STAGE_BYTES + (BN / 2) * SLAB_BYTES;
__host__ __device__ constexpr int pair_epi_warps(bool int8) { return int8 ? 16 : 8; }
__host__ __device__ constexpr int pair_smem_bytes(bool int8) {
  return pair_stages(int8) * PAIR_STAGE_BYTES + pair_out_bufs(int8) * OUT_STAGE_BYTES + 2 * (kMaxExperts + 1) * 4 + 1024 + 256;
}
__host__ __device__ constexpr int pair_threads(bool int8) { return 96 + 32 * pair_epi_warps(int8); }

template <int kType, bool kBias, bool kGelu>
__global__ void __launch_bounds__(pair_threads(kType == kTypeI8), 1)
grouped_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                    const __grid_constant__ CUtensorMap tmOut, const GroupedParams p) {
  constexpr bool kInt8 = kType == kTypeI8;
  constexpr int STAGES = pair_stages(kInt8), OUT_BUFS = pair_out_bufs(kInt8), STAGE_BYTES = PAIR_STAGE_BYTES;
  constexpr int kEpiWarps = pair_epi_warps(kInt8);
  constexpr int CW = 64 / (kEpiWarps / 4);               // columns of a 64-column chunk per warp
  constexpr int NV = CW / 8;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* stage_out0 = smem + STAGES * STAGE_BYTES;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(stage_out0 + OUT_BUFS * OUT_STAGE_BYTES);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* acc_full = empty_bar + STAGES;
  uint64_t* acc_empty = acc_full + NUM_ACC;
  uint64_t* stage_full = acc_empty + NUM_ACC;            // chunk staged by every epilogue warp, per staging tile
  uint64_t* stage_free = stage_full + 3;                 // the chunk's store has read the staging tile
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(stage_free + 3);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* s_first = reinterpret_cast<int*>(tmem_slot + 2);
  int* s_start = s_first + kMaxExperts + 1;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair = int(blockIdx.x >> 1), num_pairs = int(gridDim.x >> 1);

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < NUM_ACC; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], 2 * kEpiWarps);
    }
    for (int b = 0; b < 3; ++b) {
      mbar_init(&stage_full[b], kEpiWarps);
      mbar_init(&stage_free[b], 1);
    }
    fence_mbar_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    tma_prefetch_desc(&tmOut);
  }
  if (warp == 2) tile_list(p, 2 * BM, s_first, s_start);
  __syncthreads();
  cluster_sync_all();
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, TMEM_COLS);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  constexpr int slab_elems = kInt8 ? SLAB_BYTES : SLAB_BYTES / 2;
  const int tiles_n = (p.N + BN - 1) / BN;
  const int num_tiles = s_first[p.E] * tiles_n;
  const int skip = int(rank) * BM;                       // this CTA's first row of a tile
  TileWalk w(s_first, s_start, tiles_n, 2 * BM);
  uint32_t issued = 0;

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    if (lane == 0) {
      const uint32_t full0 = map_to_cta(&full_bar[0], 0);
      uint32_t stage = 0, phase = 0;
      bool ok = true;
      for (int tile = pair; ok && tile < num_tiles; tile += num_pairs) {
        w.at(tile);
        const int n0 = w.ntile * BN + int(rank) * (BN / 2);
        for (int ks = 0; ks < p.k_slabs; ++ks) {
          if (!(ok = mbar_wait(&empty_bar[stage], phase ^ 1u, abort_flag, p.status, 1))) break;
          uint8_t* sa = smem + stage * STAGE_BYTES;
          if (rank == 0) mbar_expect_tx(&full_bar[stage], 2 * STAGE_BYTES);
          tma_load_2d_pair(sa, &tmA, full0 + stage * 8, ks * slab_elems, w.m0 + skip);
          tma_load_3d_pair(sa + A_STAGE_BYTES, &tmB, full0 + stage * 8, ks * slab_elems, n0, w.e);
          ++issued;
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issue (leader)
    if (rank == 0) {
      const uint32_t fmt = kType == kTypeF16 ? kFmtF16 : kFmtBF16;
      const uint32_t idesc = kInt8 ? make_idesc(kAccS32, kFmtS8, kFmtS8, 2 * BM, BN) : make_idesc(kAccF32, fmt, fmt, 2 * BM, BN);
      const uint64_t desc0 = make_smem_desc(smem_u32(smem), 16, 1024, kSwizzle128B);
      const uint32_t empty_own = map_to_cta(&empty_bar[0], 0), empty_peer = map_to_cta(&empty_bar[0], 1);
      const uint32_t accf_own = map_to_cta(&acc_full[0], 0), accf_peer = map_to_cta(&acc_full[0], 1);
      uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
      bool ok = true;
      for (int tile = pair; ok && tile < num_tiles; tile += num_pairs) {
        ok = warp_wait(&acc_empty[acc], acc_phase ^ 1u, abort_flag, p.status, 2);
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * BN;
        for (int ks = 0; ks < p.k_slabs; ++ks) {
          ok = ok && warp_wait(&full_bar[stage], phase, abort_flag, p.status, 3);
          tc_fence_after();
          if (elect_one() && ok) {
            const uint64_t adesc = desc0 + stage * (STAGE_BYTES / 16);
            const uint64_t bdesc = adesc + A_STAGE_BYTES / 16;
            const int nsteps = ks == p.k_slabs - 1 ? p.last_ksteps : 4;
#pragma unroll
            for (int k4 = 0; k4 < 4; ++k4) {
              if (k4 >= nsteps) break;
              const uint32_t accumulate = (ks | k4) != 0 ? 1u : 0u;
              if (kInt8) umma_i8_ss_pair(d_tmem, adesc + k4 * 2, bdesc + k4 * 2, idesc, accumulate);
              else umma_f16_ss_pair(d_tmem, adesc + k4 * 2, bdesc + k4 * 2, idesc, accumulate);
            }
            tc_commit_pair(empty_own + stage * 8);
            tc_commit_pair(empty_peer + stage * 8);
          }
          __syncwarp();
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
        if (!(ok = __all_sync(0xffffffffu, ok))) break;
        if (elect_one()) {
          tc_commit_pair(accf_own + acc * 8);
          tc_commit_pair(accf_peer + acc * 8);
        }
        __syncwarp();
        if (++acc == NUM_ACC) { acc = 0; acc_phase ^= 1u; }
      }
    }
  } else if (warp == 2 + kEpiWarps) {
    // ------------------------------------------------------------------ output warp
    // Staged chunk n of this CTA lives in staging tile n % OUT_BUFS.  Only whole tiles are staged.
    if (lane == 0) {
      uint32_t n = 0;
      bool ok = true;
      for (int tile = pair; ok && tile < num_tiles; tile += num_pairs) {
        w.at(tile);
        const int n0 = w.ntile * BN;
        if (w.rows < skip + BM || n0 + BN > p.N) continue;
        for (int c = 0; c < BN / 64; ++c, ++n) {
          const uint32_t b = n % OUT_BUFS;
          if (!(ok = mbar_wait(&stage_full[b], (n / OUT_BUFS) & 1u, abort_flag, p.status, 6))) break;
          tma_store_2d(&tmOut, stage_out0 + b * OUT_STAGE_BYTES, n0 + c * 64, w.m0 + skip);
          tma_store_commit();
          // with several staging tiles, let this store run and hand back the tile of the one before it
          tma_store_wait_read<(OUT_BUFS > 1 ? 1 : 0)>();
          if (OUT_BUFS == 1) mbar_arrive(&stage_free[0]);
          else if (n > 0) mbar_arrive(&stage_free[(n - 1) % OUT_BUFS]);
        }
      }
      tma_store_wait_all<0>();
    }
  } else {
    // ------------------------------------------------------------------ epilogue warps, own 128 rows
    const uint32_t lane_base = uint32_t(warp & 3) * 32u;
    const int qc = (warp - 2) >> 2;
    const int erow = int(lane_base) + lane;
    const uint32_t acc_empty0 = map_to_cta(&acc_empty[0], 0);
    uint32_t acc = 0, acc_phase = 0, chunk_no = 0;
    for (int tile = pair; tile < num_tiles; tile += num_pairs) {
      w.at(tile);
      const int n0 = w.ntile * BN;
      const int mine = w.rows - skip;                    // rows of this CTA's half that exist (may be none)
      const float* g_bias = kBias ? p.bias + (long long)w.e * p.N + n0 : nullptr;
      const float* g_wscale = kInt8 ? p.w_scale + (long long)w.e * p.N + n0 : nullptr;
      float a_scale = 1.f;
      if (kInt8 && erow < mine) {
        const int i = p.rows != nullptr ? __ldg(p.rows + w.m0 + skip + erow) : w.m0 + skip + erow;
        if (i >= 0 && i < p.a_rows) a_scale = __ldg(p.a_scale + i);
      }
      if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[acc], acc_phase, abort_flag, p.status, 4))) break;
      tc_fence_after();
      const uint32_t t_addr = tmem_base + (lane_base << 16) + acc * BN + qc * CW;
      if (mine >= BM && n0 + BN <= p.N) {
        // A whole tile, without a branch in its arithmetic.  The tensor-memory load of chunk c + 1 is in flight while
        // chunk c is worked on, and the accumulator is handed back as soon as its last chunk is in registers.
        uint32_t rbuf[2][CW];
        if constexpr (CW == 32) tmem_ld_32x32b_x32(t_addr, rbuf[0]);
        else tmem_ld_32x32b_x16(t_addr, rbuf[0]);
#pragma unroll
        for (int c = 0; c < BN / 64; ++c) {
          tmem_ld_wait();
          if (c + 1 < BN / 64) {
            if constexpr (CW == 32) tmem_ld_32x32b_x32(t_addr + (c + 1) * 64, rbuf[(c + 1) & 1]);
            else tmem_ld_32x32b_x16(t_addr + (c + 1) * 64, rbuf[(c + 1) & 1]);
          } else {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster_relaxed(acc_empty0 + acc * 8);
          }
          const uint32_t(&r)[CW] = rbuf[c & 1];
          const uint32_t sbuf = chunk_no % OUT_BUFS, suse = chunk_no / OUT_BUFS;
          uint8_t* stage_out = stage_out0 + sbuf * OUT_STAGE_BYTES;
          bool ready = true;
          if (suse > 0) ready = mbar_test_wait(&stage_free[sbuf], (suse - 1u) & 1u);
          uint4 packed[NV];
#pragma unroll
          for (int u = 0; u < NV; ++u) {
            const int ct0 = c * 64 + qc * CW + u * 8;
            float v[8];
            epilogue8<kInt8, kInt8, kBias, kGelu>(r + u * 8, a_scale, g_wscale + ct0, g_bias + ct0, v);
            packed[u] = kType == kTypeF16 ? F16::pack(v) : Bf16::pack(v);
          }
          if (!ready) mbar_wait(&stage_free[sbuf], (suse - 1u) & 1u, abort_flag, p.status, 7);
          uint8_t* srow = stage_out + erow * 128;
#pragma unroll
          for (int u = 0; u < NV; ++u)
            *reinterpret_cast<uint4*>(srow + (((qc * NV + u) ^ (erow & 7)) << 4)) = packed[u];
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&stage_full[sbuf]);
          ++chunk_no;
        }
      } else {
        // The last rows of an expert or the last columns: straight from registers (N is a multiple of 8).
#pragma unroll 1
        for (int c = 0; c < BN / 64 && n0 + c * 64 < p.N && mine > 0; ++c) {
          uint32_t r[CW];
          if constexpr (CW == 32) tmem_ld_32x32b_x32(t_addr + c * 64, r);
          else tmem_ld_32x32b_x16(t_addr + c * 64, r);
          tmem_ld_wait();
          uint16_t* o = static_cast<uint16_t*>(p.out) + (w.m0 + skip + (long long)erow) * p.ldo + n0;
#pragma unroll
          for (int u = 0; u < NV; ++u) {
            const int ct0 = c * 64 + qc * CW + u * 8;
            if (n0 + ct0 < p.N && erow < mine) {
              float v[8];
              epilogue8<kInt8, kInt8, kBias, kGelu>(r + u * 8, a_scale, g_wscale + ct0, g_bias + ct0, v);
              *reinterpret_cast<uint4*>(o + ct0) = kType == kTypeF16 ? F16::pack(v) : Bf16::pack(v);
            }
          }
          __syncwarp();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_relaxed(acc_empty0 + acc * 8);
      }
      if (++acc == NUM_ACC) { acc = 0; acc_phase ^= 1u; }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 0 && lane == 0 && *abort_flag) drain_copies<STAGES>(full_bar, rank == 0 ? issued : 0u);
  cluster_sync_all();                                    // no CTA leaves while its peer may still signal it
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, TMEM_COLS);
  }
}

// ---------------------------------------------------------------------------------------------- a handful of rows
// A warp owns RN neighbouring rows of one expert's W and multiplies them with up to four rows of A at a time: lanes split
// K in 16-byte pieces, partial sums meet in shuffles.  Bound by the stream of weights (26 MB for one token with two
// experts of 5120 x 1280): eight 16-byte loads a lane in flight, RN = 4, 2 or 1 so that some sixteen warps an SM share it.
constexpr int FEW_WARPS = 8;

template <int kType>
struct Dot {                       // 16 bytes of both operands
  using Acc = f32x2;
  static __device__ __forceinline__ Acc zero() { return pack2(0.f, 0.f); }
  static __device__ __forceinline__ Acc add(const uint4& a, const uint4& b, Acc c) {
    const uint32_t u[4] = {a.x, a.y, a.z, a.w}, v[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (kType == kTypeF16) {
        const float2 s = F16::unpack2f(u[j]), t = F16::unpack2f(v[j]);
        c = ffma2(pack2(s.x, s.y), pack2(t.x, t.y), c);
      } else {
        c = ffma2(bf16x2_to_f32x2(u[j]), bf16x2_to_f32x2(v[j]), c);
      }
    }
    return c;
  }
  static __device__ __forceinline__ float sum(Acc c) {
    float lo, hi;
    unpack2(c, lo, hi);
    return lo + hi;
  }
};
template <>
struct Dot<kTypeI8> {
  using Acc = int;
  static __device__ __forceinline__ int zero() { return 0; }
  static __device__ __forceinline__ int add(const uint4& a, const uint4& b, int c) {
    c = __dp4a(int(a.x), int(b.x), c);
    c = __dp4a(int(a.y), int(b.y), c);
    c = __dp4a(int(a.z), int(b.z), c);
    return __dp4a(int(a.w), int(b.w), c);
  }
  static __device__ __forceinline__ int sum(int c) { return c; }
};

// The nth expert that has rows (by one warp): its number or -1, its first slot and its rows, by the rules of tile_list.
__device__ __forceinline__ int nth_expert(const GroupedParams& p, int nth, int& first, int& rows) {
  const int lane = threadIdx.x & 31;
  int at = 0;
  for (int e0 = 0; e0 < p.E; e0 += 32) {
    const int e = e0 + lane;
    int lo = 0, hi = 0;
    if (e < p.E) {
      lo = min(max(__ldg(p.offsets + e), 0), int(p.S));
      hi = min(max(__ldg(p.offsets + e + 1), 0), int(p.S));
    }
    int top = max(lo, hi);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, top, o);
      if (lane >= o) top = max(top, up);
    }
    top = max(top, at);
    int below = __shfl_up_sync(0xffffffffu, top, 1);
    if (lane == 0) below = e0 == 0 ? lo : at;
    const int begin = max(lo, below), n = max(0, hi - begin);
    const unsigned have = __ballot_sync(0xffffffffu, n > 0);
    if (__popc(have) > nth) {
      const int src = __ffs(__ballot_sync(0xffffffffu, n > 0 && __popc(have & ((1u << lane) - 1u)) == nth)) - 1;
      first = __shfl_sync(0xffffffffu, begin, src);
      rows = __shfl_sync(0xffffffffu, n, src);
      return e0 + src;
    }
    nth -= __popc(have);
    at = __shfl_sync(0xffffffffu, top, 31);
  }
  return -1;
}

template <int kType, int RN>
__global__ void __launch_bounds__(32 * FEW_WARPS)
grouped_few_kernel(const uint8_t* __restrict__ W, const long long w_pitch, const long long w_stride, const GroupedParams p,
                   const int gelu) {
  constexpr bool kInt8 = kType == kTypeI8;
  constexpr int TK = 4, UK = 8 / RN;                     // rows of A at a time; 16-byte steps of K in flight
  using D = Dot<kType>;
  const int lane = threadIdx.x & 31;
  const int n0 = (int(blockIdx.x) * FEW_WARPS + int(threadIdx.x >> 5)) * RN;
  if (n0 >= p.N) return;                                 // N is a multiple of 8: all RN rows exist
  int first = 0, rows = 0;
  const int e = nth_expert(p, int(blockIdx.y), first, rows);
  if (e < 0) return;
  const int steps = p.k_bytes >> 4;                      // 16-byte pieces of K
  const uint8_t* w = W + e * w_stride + n0 * w_pitch;
  for (int t0 = 0; t0 < rows; t0 += TK) {
    const uint8_t* a[TK];
    float scale[TK];
#pragma unroll
    for (int t = 0; t < TK; ++t) {
      int i = -1;
      if (t0 + t < rows) i = p.rows != nullptr ? __ldg(p.rows + first + t0 + t) : first + t0 + t;
      const bool there = i >= 0 && i < p.a_rows;
      a[t] = there ? p.a + i * p.a_pitch : nullptr;
      scale[t] = kInt8 && there ? __ldg(p.a_scale + i) : 1.f;
    }
    typename D::Acc acc[TK][RN];
#pragma unroll
    for (int t = 0; t < TK; ++t)
#pragma unroll
      for (int r = 0; r < RN; ++r) acc[t][r] = D::zero();
    for (int k0 = lane; k0 < steps; k0 += 32 * UK) {
      uint4 wv[UK][RN];
#pragma unroll
      for (int u = 0; u < UK; ++u)
#pragma unroll
        for (int r = 0; r < RN; ++r)
          wv[u][r] = k0 + u * 32 < steps ? __ldg(reinterpret_cast<const uint4*>(w + r * w_pitch) + k0 + u * 32)
                                         : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int t = 0; t < TK; ++t) {
        if (a[t] == nullptr) continue;                   // the same for the whole warp
#pragma unroll
        for (int u = 0; u < UK; ++u) {
          if (k0 + u * 32 >= steps) break;
          const uint4 av = __ldg(reinterpret_cast<const uint4*>(a[t]) + k0 + u * 32);
#pragma unroll
          for (int r = 0; r < RN; ++r) acc[t][r] = D::add(av, wv[u][r], acc[t][r]);
        }
      }
    }
    // lane t * RN + r finishes output (t, r)
    float mine = 0.f;
    float mine_scale = 1.f;
#pragma unroll
    for (int t = 0; t < TK; ++t)
#pragma unroll
      for (int r = 0; r < RN; ++r) {
        auto v = D::sum(acc[t][r]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (lane == t * RN + r) {
          mine = float(v);
          mine_scale = scale[t];
        }
      }
    const int t = lane / RN, n = n0 + lane % RN;
    if (t < TK && t0 + t < rows) {
      if (kInt8) mine = mine * mine_scale * __ldg(p.w_scale + (long long)e * p.N + n);
      if (p.bias != nullptr) mine += __ldg(p.bias + (long long)e * p.N + n);
      if (gelu) mine = gelu_erf(mine);
      static_cast<uint16_t*>(p.out)[(first + t0 + t) * p.ldo + n] = kType == kTypeF16 ? F16::from_float(mine) : Bf16::from_float(mine);
    }
  }
}

template <int kType>
void launch_few(const uint8_t* W, long long w_pitch, long long w_stride, const GroupedParams& p, bool gelu, cudaStream_t st) {
  const unsigned groups = unsigned(p.S < p.E ? p.S : p.E);
  const long long warps = (long long)p.N * groups, full = (long long)sm_count() * 16;
  const int rn = warps >= 4 * full ? 4 : warps >= 2 * full ? 2 : 1;
  const dim3 grid(unsigned((p.N + FEW_WARPS * rn - 1) / (FEW_WARPS * rn)), groups);
  if (rn == 4) grouped_few_kernel<kType, 4><<<grid, 32 * FEW_WARPS, 0, st>>>(W, w_pitch, w_stride, p, gelu);
  else if (rn == 2) grouped_few_kernel<kType, 2><<<grid, 32 * FEW_WARPS, 0, st>>>(W, w_pitch, w_stride, p, gelu);
  else grouped_few_kernel<kType, 1><<<grid, 32 * FEW_WARPS, 0, st>>>(W, w_pitch, w_stride, p, gelu);
}

// Rows in all up to which a call goes to the dot products.  us on the device with the weights in HBM, dot products / tile kernel,
// rows spread over the experts | all with one.  16 experts, 5120 x 1280 bf16: 1 row 6.9 / 11.2; 2 rows 10.2 / 12.3 | 9.2 / 11.3;
// 4 rows 18.5 / 16.1 | 11.8 / 11.2; 8 rows 24.9 / 19.3 | 18.4 / 11.5.  1280 x 5120 bf16: 2 rows 9.9 / 23.8 | 13.8 / 23.6; 4 rows
// 14.3 / 29.5 | 22.3 / 23.4; 8 rows 30.6 / 30.4 | 49.8 / 23.6; 12 rows 41.9 / 34.2 | 72 / 23.5.  int8 5120 x 1280: 4 rows 10.7 / 11.8 |
// 7.1 / 7.7; 8 rows 15.8 / 14.7 | 10.8 / 8.0; 12 rows 20.5 / 17.1 | 14.2 / 7.6.  32 experts, 512 x 512 bf16: 8 rows 4.1 / 8.0 |
// 6.2 / 6.6; 12 rows 4.5 / 8.1 | 9.0 / 6.6.  The host does not know how the rows are spread: at eight the two sides are even over
// these, above it the tile kernel is ahead but for small experts.
constexpr int64_t kFewSlots = 8;

// Rows of A in the order of the slots, packed: 16-byte vectors, several loads a thread in flight.  A row that does not
// exist is zeros.
constexpr int kOrderVecs = 4;
__global__ void __launch_bounds__(256)
order_rows_kernel(const GroupedParams p, uint4* __restrict__ to) {
  const unsigned nv = unsigned(p.k_bytes >> 4);
  const long long last = p.S * nv;
  const long long i0 = (long long)blockIdx.x * (256 * kOrderVecs) + threadIdx.x;
  uint4 v[kOrderVecs];
#pragma unroll
  for (int u = 0; u < kOrderVecs; ++u) {
    const long long i = i0 + u * 256;
    v[u] = make_uint4(0u, 0u, 0u, 0u);
    if (i < last) {
      const long long s = i / nv;
      const int r = __ldg(p.rows + s);
      if (r >= 0 && r < p.a_rows) v[u] = __ldg(reinterpret_cast<const uint4*>(p.a + r * p.a_pitch) + (i - s * nv));
    }
  }
#pragma unroll
  for (int u = 0; u < kOrderVecs; ++u)
    if (i0 + u * 256 < last) to[i0 + u * 256] = v[u];
}

using PairFn = void (*)(const CUtensorMap, const CUtensorMap, const CUtensorMap, const GroupedParams);
using OneFn = void (*)(const CUtensorMap, const CUtensorMap, const CUtensorMap, const CUtensorMap, const GroupedParams);

template <int kType>
OneFn one_of(bool gelu, bool gather) {
  if (gelu) return gather ? grouped_one_kernel<kType, true, true> : grouped_one_kernel<kType, true, false>;
  return gather ? grouped_one_kernel<kType, false, true> : grouped_one_kernel<kType, false, false>;
}
OneFn one_kernel(int type, bool gelu, bool gather) {
  return type == kTypeBf16 ? one_of<kTypeBf16>(gelu, gather) : type == kTypeF16 ? one_of<kTypeF16>(gelu, gather) : one_of<kTypeI8>(gelu, gather);
}
template <int kType>
PairFn pair_of(bool bias, bool gelu) {
  if (bias) return gelu ? grouped_pair_kernel<kType, true, true> : grouped_pair_kernel<kType, true, false>;
  return gelu ? grouped_pair_kernel<kType, false, true> : grouped_pair_kernel<kType, false, false>;
}
PairFn pair_kernel(int type, bool bias, bool gelu) {
  return type == kTypeBf16 ? pair_of<kTypeBf16>(bias, gelu) : type == kTypeF16 ? pair_of<kTypeF16>(bias, gelu) : pair_of<kTypeI8>(bias, gelu);
}

// When CTA pairs are the faster kernel for rows in order: from 512 rows an expert (int8: 1024; the last tile of an expert is
// half empty on average), two waves of tiles, and for 16-bit operands 1 KB of K (eight slabs; a short product is bound by
// its epilogue, where the int8 pair kernel's sixteen warps win all the same).  us, single CTAs / pairs.  bf16, K 1280: 16 experts
// 5120 wide at 256 rows an expert 70 / 73, at 384 91 / 92, at 512 112 / 103; 8 experts 1280 wide at 512 (80 tiles) 20.2 / 20.2, at
// 1024 (160 tiles) 29.6 / 27.2, at 4096 86 / 78; 32 experts 512 wide at 512 (128 tiles) 26.2 / 29.9, at 1024 44.5 / 40.1.  bf16, 8
// experts 1280 wide at 4096: K 512 41.6 / 39.7, K 256 34.8 / 34.2, K 128 30.0 / 32.0.  int8, there: K 128 36.3 / 28.6, K 1280 47.3 / 43.7;
// 5120 wide, K 1280 at 512 32.5 / 35.3, at 1024 51.5 / 47.3.
bool want_pairs(int64_t S, int E, int N, int64_t row_bytes, bool int8) {
  const int64_t tiles = (S / (2 * BM)) * ((N + BN - 1) / BN);
  return S >= (int8 ? 1024 : 512) * int64_t(E) && tiles >= 148 && (int8 || row_bytes >= 1024);
}

// The same for gathered rows, which pairs want in order first: the pass is worth it from some 2000 columns and eight waves.
// us, gathered on single CTAs / in order first for pairs.  8 experts, K 1280, bf16: 1280 wide at 4096 rows an expert 96 / 101; 5120
// wide at 512 (320 tiles) 58 / 54, at 1024 101 / 91, at 4096 371 / 318; int8: 1280 wide 57 / 59; 5120 wide 35 / 40, 62 / 53, 194 / 154.
bool want_order(int64_t S, int E, int N, int64_t row_bytes, bool int8) {
  const int64_t tiles = (S / (2 * BM)) * ((N + BN - 1) / BN);
  return want_pairs(S, E, N, row_bytes, int8) && N >= 2048 && tiles >= 592;
}

int launch_pairs(int type, bool gelu, const CUtensorMap& tmA, const CUtensorMap& tmB, const CUtensorMap& tmOut,
                 const GroupedParams& p, cudaStream_t st) {
  const bool int8 = type == kTypeI8;
  const bool bias = p.bias != nullptr;
  const PairFn kern = pair_kernel(type, bias, gelu);
  const int smem_bytes = pair_smem_bytes(int8);
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes) != cudaSuccess) return SAMB_E_LAUNCH;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.blockDim = dim3(unsigned(pair_threads(int8)));
  cfg.dynamicSmemBytes = size_t(smem_bytes);
  cfg.stream = st;
  cfg.gridDim = dim3(unsigned(sm_count() & ~1));
  // co-resident pairs per kernel variant (0 = not asked yet); host threads may ask at once, and give the same answer
  static std::atomic<int> cached_clusters[3][4] = {};
  std::atomic<int>& cached = cached_clusters[type][(bias ? 2 : 0) + (gelu ? 1 : 0)];
  int max_clusters = cached.load(std::memory_order_relaxed);
  if (max_clusters == 0) {
    if (cudaOccupancyMaxActiveClusters(&max_clusters, kern, &cfg) != cudaSuccess || max_clusters < 1) {
      cudaGetLastError();
      max_clusters = -1;
    }
    cached.store(max_clusters, std::memory_order_relaxed);
  }
  if (max_clusters < 1) return SAMB_E_SHAPE;
  long long pairs = max_clusters < sm_count() / 2 ? max_clusters : sm_count() / 2;
  const long long most = ((p.S + 2 * BM - 1) / (2 * BM) + p.E) * ((p.N + BN - 1) / BN);
  if (most < pairs) pairs = most;
  cfg.gridDim = dim3(unsigned(2 * pairs));
  if (cudaLaunchKernelEx(&cfg, kern, tmA, tmB, tmOut, p) != cudaSuccess) {
    cudaGetLastError();
    return SAMB_E_LAUNCH;
  }
  return launch_status();
}

int launch_grouped(int type, const void* A, int64_t lda, int64_t a_rows, const float* a_scale, const int32_t* rows,
                   const void* W, int64_t ldw, int64_t w_stride, const float* w_scale, const float* bias,
                   const int32_t* offsets, void* out, int64_t ldo, int64_t S, int E, int N, int K, int epilogue,
                   void* scratch, int32_t* status, void* stream) {
  if (S < 0 || a_rows < 0 || E <= 0 || N <= 0 || K <= 0 || status == nullptr) return SAMB_E_BADARG;
  if (epilogue & ~(SAMB_EPI_BIAS | SAMB_EPI_GELU)) return SAMB_E_BADARG;
  if (((epilogue & SAMB_EPI_BIAS) != 0) != (bias != nullptr)) return SAMB_E_BADARG;
  if (S > 0 && (A == nullptr || W == nullptr || out == nullptr || offsets == nullptr || a_rows == 0)) return SAMB_E_BADARG;
  if (type == kTypeI8 && S > 0 && (a_scale == nullptr || w_scale == nullptr)) return SAMB_E_BADARG;
  if (out != nullptr && (out == A || out == W)) return SAMB_E_BADARG;
  const int esz = type == kTypeI8 ? 1 : 2, kmul = 16 / esz;
  if (E > kMaxExperts || N % 8 || K % kmul || lda % kmul || ldw % kmul || w_stride % kmul || ldo % 8) return SAMB_E_SHAPE;
  if (lda < K || ldw < K || ldo < N || (E > 1 && w_stride < ldw * (N - 1) + K)) return SAMB_E_SHAPE;
  if (rows == nullptr && a_rows < S) return SAMB_E_SHAPE;
  if (a_rows >= (int64_t(1) << 31) - BM || S >= (int64_t(1) << 31) - BM) return SAMB_E_SHAPE;
  // tile numbers are 32-bit, at the narrowest column tile
  if (((S + BM - 1) / BM + E) * ((N + 63) / 64) >= (int64_t(1) << 31)) return SAMB_E_SHAPE;
  if ((reinterpret_cast<uintptr_t>(A) | reinterpret_cast<uintptr_t>(W) | reinterpret_cast<uintptr_t>(out) |
       reinterpret_cast<uintptr_t>(scratch)) & 15u)
    return SAMB_E_ALIGN;
  if ((reinterpret_cast<uintptr_t>(rows) | reinterpret_cast<uintptr_t>(offsets) | reinterpret_cast<uintptr_t>(bias) |
       reinterpret_cast<uintptr_t>(a_scale) | reinterpret_cast<uintptr_t>(w_scale)) & 3u)
    return SAMB_E_ALIGN;
  if (S > 0) {
    const int64_t room = rows != nullptr && want_order(S, E, N, int64_t(K) * esz, type == kTypeI8) ? S * K * esz : 0;
    const Runs written[2] = {rows_of(out, 2 * ldo, S, 2 * int64_t(N)), bytes_of(scratch, room)};
    const Runs read[7] = {rows_of(A, lda * esz, a_rows, int64_t(K) * esz), runs3(W, w_stride * esz, E, ldw * esz, N, int64_t(K) * esz),
                          bytes_of(bias, 4 * int64_t(E) * N), bytes_of(offsets, 4 * (int64_t(E) + 1)), bytes_of(rows, 4 * S),
                          bytes_of(a_scale, 4 * a_rows), bytes_of(w_scale, 4 * int64_t(E) * N)};
    if (share_memory(written[0], written[1])) return SAMB_E_BADARG;
    for (const Runs& w : written)
      for (const Runs& r : read)
        if (share_memory(w, r)) return SAMB_E_BADARG;
  }
  if (int e = check_device_arch()) return e;
  if (S == 0) return SAMB_OK;

  const CUtensorMapDataType dt = type == kTypeI8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                 : type == kTypeF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const uint32_t slab_elems = uint32_t(SLAB_BYTES / esz);
  CUtensorMap tmA, tmA32, tmB, tmOut;
  auto map_a = [&](CUtensorMap* to, const void* base, int64_t ld, int64_t n, int box_rows) {
    const uint64_t dims[2] = {uint64_t(K), uint64_t(n)};
    const uint64_t strides[2] = {uint64_t(esz), uint64_t(ld) * esz};
    const uint32_t box[2] = {slab_elems, uint32_t(box_rows)};
    return make_tensor_map(to, dt, 2, const_cast<void*>(base), dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  };
  auto map_w = [&](int box_rows) {
    const uint64_t dims[3] = {uint64_t(K), uint64_t(N), uint64_t(E)};
    const uint64_t strides[3] = {uint64_t(esz), uint64_t(ldw) * esz, uint64_t(E > 1 ? w_stride : ldw * N) * esz};
    const uint32_t box[3] = {slab_elems, uint32_t(box_rows), 1};
    return make_tensor_map(&tmB, dt, 3, const_cast<void*>(W), dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  };
  GroupedParams p;
  p.out = out; p.a = static_cast<const uint8_t*>(A); p.bias = bias; p.a_scale = a_scale; p.w_scale = w_scale; p.rows = rows;
  p.offsets = offsets; p.status = status;
  p.ldo = ldo; p.a_rows = a_rows; p.S = S; p.a_pitch = lda * esz; p.E = E; p.N = N; p.K = K;
  p.k_bytes = K * esz;
  p.k_slabs = (p.k_bytes + SLAB_BYTES - 1) / SLAB_BYTES;
  p.last_ksteps = (p.k_bytes - (p.k_slabs - 1) * SLAB_BYTES + 31) / 32;
  const bool gelu = (epilogue & SAMB_EPI_GELU) != 0, gather = rows != nullptr;
  auto st = static_cast<cudaStream_t>(stream);
  if (S <= kFewSlots) {
    const uint8_t* w = static_cast<const uint8_t*>(W);
    const long long pitch = ldw * esz, stride = w_stride * esz;
    if (type == kTypeBf16) launch_few<kTypeBf16>(w, pitch, stride, p, gelu, st);
    else if (type == kTypeF16) launch_few<kTypeF16>(w, pitch, stride, p, gelu, st);
    else launch_few<kTypeI8>(w, pitch, stride, p, gelu, st);
    return launch_status();
  }
  {
    const uint64_t dims[2] = {uint64_t(N), uint64_t(S)};
    const uint64_t strides[2] = {2, uint64_t(ldo) * 2};
    const uint32_t box[2] = {64, uint32_t(BM)};
    if (int e = make_tensor_map(&tmOut, type == kTypeF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                                2, out, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B))
      return e;
  }
  // what the products read: A itself, or its rows in order in the caller's scratch
  const bool int8 = type == kTypeI8;
  const bool order = gather && scratch != nullptr && want_order(S, E, N, p.k_bytes, int8);
  const void* from = order ? scratch : A;
  const int64_t from_ld = order ? K : lda, from_rows = order ? S : a_rows;
  if (order) {
    const long long vecs = S * (p.k_bytes / 16), blocks = (vecs + 256 * kOrderVecs - 1) / (256 * kOrderVecs);
    if (blocks > 0x7fffffff) return SAMB_E_SHAPE;
    order_rows_kernel<<<unsigned(blocks), 256, 0, st>>>(p, static_cast<uint4*>(scratch));
    if (int e = launch_status()) return e;
  }
  if (int e = map_a(&tmA, from, from_ld, from_rows, gather && !order ? 1 : BM)) return e;
  // the pair kernel's epilogue reads the column vectors in 16-byte pieces; it wants its rows in order
  if (want_pairs(S, E, N, p.k_bytes, int8) && (!gather || order) &&
      !((reinterpret_cast<uintptr_t>(bias) | reinterpret_cast<uintptr_t>(w_scale)) & 15u)) {
    if (int e = map_w(BN / 2)) return e;
    const int e = launch_pairs(type, gelu, tmA, tmB, tmOut, p, st);
    if (e != SAMB_E_SHAPE) return e;                     // pairs cannot be placed on this GPU: single CTAs
  }
  if (int e = map_a(&tmA32, from, from_ld, from_rows, A_BOX_ROWS)) return e;
  if (int e = map_w(64)) return e;
  const bool in_kernel = gather && !order;
  const OneFn kern = one_kernel(type, gelu, in_kernel);
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, ONE_SMEM_BYTES) != cudaSuccess)
    return SAMB_E_LAUNCH;
  const long long most = ((S + BM - 1) / BM + E) * ((N + 63) / 64);
  const unsigned grid = unsigned(most < sm_count() ? most : sm_count());
  kern<<<grid, ONE_THREADS + (in_kernel ? 32 * GATHER_WARPS : 0), ONE_SMEM_BYTES, st>>>(tmA, tmA32, tmB, tmOut, p);
  return launch_status();
}

}  // namespace
}  // namespace samb

extern "C" {

int64_t samb_gemm_grouped_scratch_bytes(int64_t S, int E, int N, int K, int is_i8) {
  if (S <= 0 || E <= 0 || N <= 0 || K <= 0) return 0;
  const int64_t row = int64_t(K) * (is_i8 ? 1 : 2);
  return samb::want_order(S, E, N, row, is_i8 != 0) ? S * row : 0;
}

int samb_gemm_grouped(const void* A, int64_t lda, int64_t a_rows, const int32_t* rows, const void* W, int64_t ldw,
                      int64_t w_stride, const float* bias, const int32_t* offsets, void* out, int64_t ldo, int64_t S,
                      int E, int N, int K, int is_f16, int epilogue, void* scratch, int32_t* status, void* stream) {
  return samb::launch_grouped(is_f16 ? samb::kTypeF16 : samb::kTypeBf16, A, lda, a_rows, nullptr, rows, W, ldw, w_stride,
                              nullptr, bias, offsets, out, ldo, S, E, N, K, epilogue, scratch, status, stream);
}

int samb_gemm_i8_grouped(const int8_t* Aq, int64_t lda, int64_t a_rows, const float* a_scale, const int32_t* rows,
                         const int8_t* Wq, int64_t ldw, int64_t w_stride, const float* w_scale, const float* bias,
                         const int32_t* offsets, void* out, int64_t ldo, int64_t S, int E, int N, int K, int epilogue,
                         void* scratch, int32_t* status, void* stream) {
  return samb::launch_grouped(samb::kTypeI8, Aq, lda, a_rows, a_scale, rows, Wq, ldw, w_stride, w_scale, bias, offsets,
                              out, ldo, S, E, N, K, epilogue, scratch, status, stream);
}

}  // extern "C"
