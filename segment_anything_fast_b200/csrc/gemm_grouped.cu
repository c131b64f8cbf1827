// Products grouped by expert with ragged sizes (a mixture of experts' Linear layers):
//   out[s, :] = epilogue( a[rows ? rows[s] : s, :] * w[e]^T + bias[e] ),   offsets[e] <= s < offsets[e + 1].
// The offsets live on the device (the router wrote them), so the host launches one wave of persistent CTAs and every
// CTA works the tile list out for itself: the prefix over the experts of their 128-row tiles, times the column tiles.
//
// Tile loop: warp 0 streams 128-byte K slabs of A and W into a ring of 128B-swizzled stages (TMA; with `rows` the A
// rows are gathered four at a time by tile::gather4, so no permuted copy of the activations exists), warp 1 issues
// tcgen05.mma into one of two accumulators in tensor memory, warps 2..9 drain the other one.  A tile reads 128 rows
// of A whatever its expert has left (rows of the next expert, discarded), but stores only its own: whole tiles
// leave by TMA, the last tile of an expert row by row from the staging tile.
//
// Column tile: 256, 128 or 64 wide, picked by the CTAs themselves so that the last wave is not mostly empty (a handful
// of tokens touches each expert's weights once, and the number of tiles is what spreads that stream over the SMs).
#include "elem16.cuh"

namespace samb {
namespace {

constexpr int BM = 128;
constexpr int BN = 256;
constexpr int SLAB_BYTES = 128;
constexpr int STAGES = 4;
constexpr int A_STAGE_BYTES = BM * SLAB_BYTES;
constexpr int B_BOX_ROWS = 64;
constexpr int B_BOX_BYTES = B_BOX_ROWS * SLAB_BYTES;
constexpr int B_STAGE_BYTES = BN * SLAB_BYTES;
constexpr int STAGE_BYTES = A_STAGE_BYTES + B_STAGE_BYTES;
constexpr int NUM_ACC = 2;
constexpr int TMEM_COLS = NUM_ACC * BN;
constexpr int EPI_WARPS = 8;
constexpr int NUM_THREADS = 64 + 32 * EPI_WARPS;
constexpr int OUT_STAGE_BYTES = BM * 128;
constexpr int kMaxExperts = 512;
constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + OUT_STAGE_BYTES + 2 * BN * 4 + 2 * (kMaxExperts + 1) * 4 + 1024 + 256;

enum { kTypeBf16 = 0, kTypeF16 = 1, kTypeI8 = 2 };

struct GroupedParams {
  void* out;
  const float* bias;               // [E, N] or null
  const float* a_scale;            // int8: per row of A
  const float* w_scale;            // int8: [E, N]
  const int* rows;                 // gather indexes, or null
  const int* offsets;              // [E + 1]
  int* status;
  long long ldo, a_rows, S;
  int E, N, K;
  int k_slabs, last_ksteps;
  int gelu;
};

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

// Four rows of a 2-D tensor into 4 x 128 consecutive bytes.
__device__ __forceinline__ void tma_gather4(void* smem_dst, const CUtensorMap* m, uint64_t* bar, int x, const int4& r) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
      ::"r"(smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(x), "r"(r.x), "r"(r.y),
      "r"(r.z), "r"(r.w)
      : "memory");
}

// Where a tile lies.  Tiles are numbered expert by expert, row tile by row tile, column tile by column tile; a role
// walks its tiles in rising order, so the expert only ever moves forward.
struct TileWalk {
  const int* first;                // [E + 1] row tiles before each expert
  const int* start;                // [E + 1] first slot of each expert, clamped
  int tiles_n, e, m0, rows, ntile;
  __device__ __forceinline__ TileWalk(const int* f, const int* s, int tn) : first(f), start(s), tiles_n(tn), e(0), m0(0), rows(0), ntile(0) {}
  __device__ __forceinline__ void at(int tile) {
    const int mt = tile / tiles_n;
    ntile = tile - mt * tiles_n;
    while (first[e + 1] <= mt) ++e;
    m0 = start[e] + (mt - first[e]) * BM;
    rows = min(BM, start[e + 1] - m0);
  }
};

template <int kType, bool kGelu>
__global__ void __launch_bounds__(NUM_THREADS, 1)
gemm_grouped_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                    const __grid_constant__ CUtensorMap tmOut, const GroupedParams p) {
  constexpr bool kInt8 = kType == kTypeI8;
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
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < NUM_ACC; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], EPI_WARPS);
    }
    fence_mbar_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    tma_prefetch_desc(&tmOut);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  if (warp == 2) {
    // the tile list.  Offsets are clamped to [0, S] and made to rise, so that no list can point outside the buffers.
    int tiles = 0, at = 0;
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const int e = e0 + lane;
      int lo = 0, hi = 0;
      if (e < p.E) {
        lo = min(max(__ldg(p.offsets + e), 0), int(p.S));
        hi = min(max(__ldg(p.offsets + e + 1), 0), int(p.S));
      }
      int top = max(lo, hi);                             // running maximum over the experts up to this one
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, top, o);
        if (lane >= o) top = max(top, up);
      }
      top = max(top, at);
      int below = __shfl_up_sync(0xffffffffu, top, 1);
      if (lane == 0) below = at;
      if (e0 == 0 && lane == 0) below = lo;
      const int begin = max(lo, below), n = max(0, hi - begin);
      const int mine = (n + BM - 1) / BM;
      int sum = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += up;
      }
      if (e < p.E) {
        s_first[e] = tiles + sum - mine;
        s_start[e] = begin;
        if (e == p.E - 1) s_start[p.E] = begin + n;
      }
      tiles += __shfl_sync(0xffffffffu, sum, 31);
      at = __shfl_sync(0xffffffffu, top, 31);
    }
    if (lane == 0) {
      s_first[p.E] = tiles;
      // waves x (columns + what a tile costs beside its columns)
      int best = 0, bn = BN;
      for (int w = BN; w >= 64; w >>= 1) {
        const long long t = (long long)tiles * ((p.N + w - 1) / w);
        const int cost = int((t + gridDim.x - 1) / gridDim.x) * (w + 64);
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
  TileWalk w(s_first, s_start, tiles_n);
  uint32_t issued = 0;                                   // slabs that the producer has sent for

  if (warp == 0) {
    // ------------------------------------------------------------------ producer
    uint32_t stage = 0, phase = 0;
    bool ok = true;
    for (int tile = blockIdx.x; ok && tile < num_tiles; tile += gridDim.x) {
      w.at(tile);
      const int n0 = w.ntile * bn;
      int4 src = make_int4(0, 0, 0, 0);                  // the four rows of A that this lane gathers
      if (p.rows != nullptr) {
        int r[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int m = lane * 4 + j;
          const int i = m < w.rows ? __ldg(p.rows + w.m0 + m) : 0;
          r[j] = i >= 0 && i < p.a_rows ? i : 0;         // outside A: any row, the epilogue drops its product
        }
        src = make_int4(r[0], r[1], r[2], r[3]);
      }
      for (int ks = 0; ks < p.k_slabs; ++ks) {
        if (!(ok = __all_sync(0xffffffffu, mbar_wait(&empty_bar[stage], phase ^ 1u, abort_flag, p.status, 1)))) break;
        uint8_t* sa = smem + stage * STAGE_BYTES;
        if (lane == 0) mbar_expect_tx(&full_bar[stage], A_STAGE_BYTES + bn * SLAB_BYTES);
        __syncwarp();
        if (p.rows != nullptr) tma_gather4(sa + lane * 512, &tmA, &full_bar[stage], ks * slab_elems, src);
        else if (lane == 0) tma_load_2d(sa, &tmA, &full_bar[stage], ks * slab_elems, w.m0);
        if (lane < bn / B_BOX_ROWS)
          tma_load_3d(sa + A_STAGE_BYTES + lane * B_BOX_BYTES, &tmB, &full_bar[stage], ks * slab_elems,
                      n0 + lane * B_BOX_ROWS, w.e);
        ++issued;
        if (++stage == STAGES) { stage = 0; phase ^= 1u; }
      }
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
      if (!(ok = __all_sync(0xffffffffu, mbar_wait(&acc_empty[acc], acc_phase ^ 1u, abort_flag, p.status, 2)))) break;
      tc_fence_after();
      const uint32_t d_tmem = tmem_base + acc * BN;
      for (int ks = 0; ks < p.k_slabs; ++ks) {
        if (!(ok = __all_sync(0xffffffffu, mbar_wait(&full_bar[stage], phase, abort_flag, p.status, 3)))) break;
        tc_fence_after();
        if (elect_one()) {
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
      if (!ok) break;
      if (elect_one()) tc_commit(&acc_full[acc]);
      __syncwarp();
      if (++acc == NUM_ACC) { acc = 0; acc_phase ^= 1u; }
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
      if (erow < w.rows) {
        const int i = p.rows != nullptr ? __ldg(p.rows + w.m0 + erow) : w.m0 + erow;
        there = i >= 0 && i < p.a_rows;
        if (kInt8 && there) a_scale = __ldg(p.a_scale + i);
      }
      const bool got = mbar_wait(&acc_full[acc], acc_phase, abort_flag, p.status, 4);
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
        if (!there) {
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
  if (warp == 0 && *abort_flag) {                        // a wait gave up: see the copies in flight home first
    for (uint32_t i = issued > STAGES ? issued - STAGES : 0u; i < issued; ++i)
      for (uint32_t n = 0; n < 65536u && !mbar_try_wait(&full_bar[i % STAGES], (i / STAGES) & 1u); ++n) __nanosleep(64);
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

using GroupedFn = void (*)(const CUtensorMap, const CUtensorMap, const CUtensorMap, const GroupedParams);

int launch_grouped(int type, const void* A, int64_t lda, int64_t a_rows, const float* a_scale, const int32_t* rows,
                   const void* W, int64_t ldw, int64_t w_stride, const float* w_scale, const float* bias,
                   const int32_t* offsets, void* out, int64_t ldo, int64_t S, int E, int N, int K, int epilogue,
                   int32_t* status, void* stream) {
  if (S < 0 || a_rows < 0 || E <= 0 || N <= 0 || K <= 0 || status == nullptr) return SAMB_E_BADARG;
  if (epilogue & ~(SAMB_EPI_BIAS | SAMB_EPI_GELU)) return SAMB_E_BADARG;
  if (((epilogue & SAMB_EPI_BIAS) != 0) != (bias != nullptr)) return SAMB_E_BADARG;
  if (S > 0 && (A == nullptr || W == nullptr || out == nullptr || offsets == nullptr || a_rows == 0)) return SAMB_E_BADARG;
  if (type == kTypeI8 && S > 0 && (a_scale == nullptr || w_scale == nullptr)) return SAMB_E_BADARG;
  const int esz = type == kTypeI8 ? 1 : 2, kmul = 16 / esz;
  if (E > kMaxExperts || N % 8 || K % kmul || lda % kmul || ldw % kmul || w_stride % kmul || ldo % 8) return SAMB_E_SHAPE;
  if (lda < K || ldw < K || ldo < N || (E > 1 && w_stride < ldw * (N - 1) + K)) return SAMB_E_SHAPE;
  if (rows == nullptr && a_rows < S) return SAMB_E_SHAPE;
  if (a_rows >= (int64_t(1) << 31) - BM || S >= (int64_t(1) << 31) - BM) return SAMB_E_SHAPE;
  // tile numbers are 32-bit, at the narrowest column tile
  if (((S + BM - 1) / BM + E) * ((N + 63) / 64) >= (int64_t(1) << 31)) return SAMB_E_SHAPE;
  if ((reinterpret_cast<uintptr_t>(A) | reinterpret_cast<uintptr_t>(W) | reinterpret_cast<uintptr_t>(out)) & 15u)
    return SAMB_E_ALIGN;
  if ((reinterpret_cast<uintptr_t>(rows) | reinterpret_cast<uintptr_t>(offsets) | reinterpret_cast<uintptr_t>(bias) |
       reinterpret_cast<uintptr_t>(a_scale) | reinterpret_cast<uintptr_t>(w_scale)) & 3u)
    return SAMB_E_ALIGN;
  if (int e = check_device_arch()) return e;
  if (S == 0) return SAMB_OK;

  const CUtensorMapDataType dt = type == kTypeI8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                 : type == kTypeF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const uint32_t slab_elems = uint32_t(SLAB_BYTES / esz);
  CUtensorMap tmA, tmB, tmOut;
  {
    const uint64_t dims[2] = {uint64_t(K), uint64_t(a_rows)};
    const uint64_t strides[2] = {uint64_t(esz), uint64_t(lda) * esz};
    const uint32_t box[2] = {slab_elems, uint32_t(rows != nullptr ? 1 : BM)};
    if (int e = make_tensor_map(&tmA, dt, 2, const_cast<void*>(A), dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return e;
  }
  {
    const uint64_t dims[3] = {uint64_t(K), uint64_t(N), uint64_t(E)};
    const uint64_t strides[3] = {uint64_t(esz), uint64_t(ldw) * esz, uint64_t(E > 1 ? w_stride : ldw * N) * esz};
    const uint32_t box[3] = {slab_elems, uint32_t(B_BOX_ROWS), 1};
    if (int e = make_tensor_map(&tmB, dt, 3, const_cast<void*>(W), dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return e;
  }
  {
    const uint64_t dims[2] = {uint64_t(N), uint64_t(S)};
    const uint64_t strides[2] = {2, uint64_t(ldo) * 2};
    const uint32_t box[2] = {64, uint32_t(BM)};
    if (int e = make_tensor_map(&tmOut, type == kTypeF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                                2, out, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B))
      return e;
  }
  GroupedParams p;
  p.out = out; p.bias = bias; p.a_scale = a_scale; p.w_scale = w_scale; p.rows = rows; p.offsets = offsets;
  p.status = status;
  p.ldo = ldo; p.a_rows = a_rows; p.S = S; p.E = E; p.N = N; p.K = K;
  p.k_slabs = (K * esz + SLAB_BYTES - 1) / SLAB_BYTES;
  p.last_ksteps = (K * esz - (p.k_slabs - 1) * SLAB_BYTES + 31) / 32;
  p.gelu = (epilogue & SAMB_EPI_GELU) != 0;
  static const GroupedFn kernels[3][2] = {{gemm_grouped_kernel<kTypeBf16, false>, gemm_grouped_kernel<kTypeBf16, true>},
                                          {gemm_grouped_kernel<kTypeF16, false>, gemm_grouped_kernel<kTypeF16, true>},
                                          {gemm_grouped_kernel<kTypeI8, false>, gemm_grouped_kernel<kTypeI8, true>}};
  const GroupedFn kern = kernels[type][p.gelu];
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES) != cudaSuccess)
    return SAMB_E_LAUNCH;
  const long long most = ((S + BM - 1) / BM + E) * ((N + 63) / 64);
  const unsigned grid = unsigned(most < sm_count() ? most : sm_count());
  kern<<<grid, NUM_THREADS, SMEM_BYTES, static_cast<cudaStream_t>(stream)>>>(tmA, tmB, tmOut, p);
  return launch_status();
}

}  // namespace
}  // namespace samb

extern "C" {

int samb_gemm_grouped(const void* A, int64_t lda, int64_t a_rows, const int32_t* rows, const void* W, int64_t ldw,
                      int64_t w_stride, const float* bias, const int32_t* offsets, void* out, int64_t ldo, int64_t S,
                      int E, int N, int K, int is_f16, int epilogue, int32_t* status, void* stream) {
  return samb::launch_grouped(is_f16 ? samb::kTypeF16 : samb::kTypeBf16, A, lda, a_rows, nullptr, rows, W, ldw, w_stride,
                              nullptr, bias, offsets, out, ldo, S, E, N, K, epilogue, status, stream);
}

int samb_gemm_i8_grouped(const int8_t* Aq, int64_t lda, int64_t a_rows, const float* a_scale, const int32_t* rows,
                         const int8_t* Wq, int64_t ldw, int64_t w_stride, const float* w_scale, const float* bias,
                         const int32_t* offsets, void* out, int64_t ldo, int64_t S, int E, int N, int K, int epilogue,
                         int32_t* status, void* stream) {
  return samb::launch_grouped(samb::kTypeI8, Aq, lda, a_rows, a_scale, rows, Wq, ldw, w_stride, w_scale, bias, offsets,
                              out, ldo, S, E, N, K, epilogue, status, stream);
}

}  // extern "C"
