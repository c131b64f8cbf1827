// The norms on either side of a residual addition in one pass over the rows:
//   x' = res_scale * r + gate * post(h),   y = pre(x'),
// post and pre being LayerNorm or root-mean-square norms (or absent), gate one vector for all rows or one for each
// of G equal blocks of rows (images).  y is computed from the fp32 x', not from its rounded copy: x' and y are each
// rounded once.
//
// A thread owns eight fixed columns and walks down the rows, four at a time, so the affine parameters and the gate (20
// bytes a column against the 8 bytes a column that a row moves) stay in its registers.  A block is as many warps as
// the width needs; the next four rows are on their way into shared memory (16-byte cp.async, each thread reads back
// what it copied) while four are worked on.
// Statistics: a warp reduces its own 256 columns in two passes (mean, then squared distances from it), and the
// warps' pairs (mean, M2) are joined by the parallel-variance formula
//   M2 = sum_w M2_w + n_w (mean_w - mean)^2,
// so a norm costs one block barrier for four rows and no difference of large squares is ever taken.  The four rows'
// sums share their shuffles: halves of the warp trade rows first, 6 shuffles instead of 20.
// Bound by HBM: 232 us for 131072 x 1280 bf16 with both norms and a gate an image (1.34 GB, 5.8 TB/s), 311 us for 1536 columns; a row at
// a time through registers took 635 us, held up by its barriers and shuffles.  Above 2048 columns that is still the way: 298 us for
// 16384 x 4096 (1.8 TB/s), 831 us for 16384 x 8192.  The quantised form is bound by instruction issue and the latency
// behind it (63 % of the issue slots with 4.6 warps a scheduler, DRAM 29 %): 389 us for 131072 x 1280, where the 16-bit form and a
// pass of samb_quant_rows_i8 take 346 us; 339 against 348 us for 16384 x 4096.
#include <atomic>

#include "elem16.cuh"
#include "overlap.h"

namespace samb {
namespace {

struct NormParams {
  const void* h;
  const void* r;
  const float* post_g;
  const float* post_b;
  const float* pre_g;
  const float* pre_b;
  const float* gate;
  void* x;
  void* y;               // 16-bit rows, or int8 rows when quantising
  float* y_scale;
  long long ldh, ldr, ldx;
  int rows, C, rows_per_gate, rows_per_block;
  float res_scale, eps;
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

__device__ __forceinline__ void load8(const float* p, int c, float (&v)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p + c)), b = __ldg(reinterpret_cast<const float4*>(p + c) + 1);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void fill8(float (&v)[8], float x) {
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = x;
}

// Statistics of a row whose columns are spread over the block: on return sub is what to subtract and mul what to
// multiply by.  `stat` is shared scratch for a pair a warp; a caller alternates between two of them, so that a buffer's
// next writes are a barrier away from its last reads.
template <bool kRms>
__device__ __forceinline__ void row_stats(const float (&v)[8], bool live, int C, float eps, float2* stat, float& sub,
                                          float& mul) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  float mean = 0.f, m2 = 0.f;
  if (!kRms) {
    float s = 0.f;
    if (live) {
#pragma unroll
      for (int j = 0; j < 8; ++j) s += v[j];
    }
    mean = warp_sum(s) * (1.0f / float(min(256, C - warp * 256)));      // over the columns of this warp
  }
  if (live) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float d = v[j] - mean;
      m2 = fmaf(d, d, m2);
    }
  }
  m2 = warp_sum(m2);
  const float inv_c = 1.0f / float(C);
  if (warps > 1) {
    if (lane == 0) stat[warp] = make_float2(mean, m2);
    __syncthreads();
    mean = m2 = 0.f;
    if (!kRms) {                                         // around the first warp's: a constant row stays exact
      const float first = stat[0].x;
      for (int w = 1; w < warps; ++w) mean = fmaf(stat[w].x - first, float(min(256, C - w * 256)), mean);
      mean = fmaf(mean, inv_c, first);
    }
    for (int w = 0; w < warps; ++w) {
      const float2 s = stat[w];
      const float d = s.x - mean;
      m2 += s.y;
      if (!kRms) m2 = fmaf(d * d, float(min(256, C - w * 256)), m2);
    }
  }
  sub = mean;
  mul = rsqrtf(fmaf(m2, inv_c, eps));
}

// The sum over the warp of four values: afterwards the lanes of group l >> 3 all hold the sum of value l >> 3.
__device__ __forceinline__ float warp_sum4(const float (&v)[4]) {
  const int lane = threadIdx.x & 31;
  const bool upper = (lane & 16) != 0, odd = (lane & 8) != 0;
  const float a = (upper ? v[2] : v[0]) + __shfl_xor_sync(0xffffffffu, upper ? v[0] : v[2], 16);
  const float b = (upper ? v[3] : v[1]) + __shfl_xor_sync(0xffffffffu, upper ? v[1] : v[3], 16);
  float c = (odd ? b : a) + __shfl_xor_sync(0xffffffffu, odd ? a : b, 8);
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
  return c;
}

// row_stats for four rows held as packed pairs and at most eight warps: lane l works on row l >> 3, and on warp l & 7
// when the warps' results are joined.
template <bool kRms>
__device__ __forceinline__ void row_stats4(const f32x2 (&v)[4][4], bool live, int C, float eps, float2* stat,
                                           float (&sub)[4], float (&mul)[4]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  float part[4], mean = 0.f;
  if (!kRms) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float lo, hi;
      unpack2(fadd2(fadd2(v[i][0], v[i][1]), fadd2(v[i][2], v[i][3])), lo, hi);
      part[i] = live ? lo + hi : 0.f;
    }
    mean = warp_sum4(part) * (1.0f / float(min(256, C - warp * 256)));
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float m = kRms ? 0.f : __shfl_sync(0xffffffffu, mean, i * 8);
    const f32x2 m2 = pack2(m, m);
    f32x2 q = pack2(0.f, 0.f);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x2 d = kRms ? v[i][j] : fsub2(v[i][j], m2);
      q = ffma2(d, d, q);
    }
    float lo, hi;
    unpack2(q, lo, hi);
    part[i] = live ? lo + hi : 0.f;
  }
  float m2 = warp_sum4(part);
  if (warps > 1) {
    if ((lane & 7) == 0) stat[warp * 4 + (lane >> 3)] = make_float2(mean, m2);
    __syncthreads();
    const int w = lane & 7;
    const float2 s = w < warps ? stat[w * 4 + (lane >> 3)] : make_float2(0.f, 0.f);
    const float n = w < warps ? float(min(256, C - w * 256)) : 0.f;
    if (!kRms) {                                         // around the first warp's: a constant row stays exact
      const float first = __shfl_sync(0xffffffffu, s.x, lane & 24);
      float t = w < warps ? (s.x - first) * n : 0.f;
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
      mean = fmaf(t, 1.0f / float(C), first);
    }
    const float d = s.x - mean;
    m2 = kRms ? s.y : fmaf(d * d, n, s.y);
    if (w >= warps) m2 = 0.f;                            // also where the mean is not a number
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) m2 += __shfl_xor_sync(0xffffffffu, m2, o);
  }
  const float r = rsqrtf(fmaf(m2, 1.0f / float(C), eps));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    sub[i] = kRms ? 0.f : __shfl_sync(0xffffffffu, mean, i * 8);
    mul[i] = __shfl_sync(0xffffffffu, r, i * 8);
  }
}

__device__ __forceinline__ void cp_async_16(uint32_t smem_dst, const void* gsrc) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_dst), "l"(gsrc) : "memory");
}

template <typename T>
__device__ __forceinline__ void unpack_pairs(const uint4& u, f32x2 (&v)[4]) {
  float f[8];
  T::unpack(u, f);
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = pack2(f[2 * j], f[2 * j + 1]);
}
template <typename T>
__device__ __forceinline__ uint4 pack_pairs(const f32x2 (&v)[4]) {
  float f[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) unpack2(v[j], f[2 * j], f[2 * j + 1]);
  return T::pack(f);
}

// Four rows at a time, at most eight warps (C up to 2048), the next four rows in flight.  Up to five warps (C up to 1280)
// four blocks fit an SM: 235 against 240 us for three at 131072 x 1280.
template <typename T, bool kRms, bool kQuant, int kWarps>
__global__ void __launch_bounds__(kWarps * 32, kWarps <= 5 ? 4 : 2)
block_norm_rows_kernel(const NormParams p) {
  extern __shared__ uint4 ring[];                        // [2 turns][h, r][4 rows][thread]
  __shared__ float2 s_post[2][32], s_pre[2][32];
  __shared__ float s_max[32];
  const int threads = blockDim.x, c = int(threadIdx.x) * 8;
  const bool live = c < p.C;
  const int begin = int(blockIdx.x) * p.rows_per_block;
  const int end = begin + min(p.rows_per_block, p.rows - begin);       // begin + rows_per_block may pass 2^31
  const bool has_post = p.post_g != nullptr, has_pre = p.pre_g != nullptr, has_res = p.r != nullptr;
  uint4* mine = ring + threadIdx.x;
  const uint16_t* h = static_cast<const uint16_t*>(p.h) + c;
  const uint16_t* r = static_cast<const uint16_t*>(p.r) + c;
  auto fetch = [&](int row0, int turn) {
    if (live) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (row0 + i >= end) break;
        cp_async_16(smem_u32(mine + ((turn * 2 + 0) * 4 + i) * threads), h + (row0 + i) * p.ldh);
        if (has_res) cp_async_16(smem_u32(mine + ((turn * 2 + 1) * 4 + i) * threads), r + (row0 + i) * p.ldr);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  fetch(begin, 0);

  f32x2 pg[4], pb[4], qg[4], qb[4];          // post's gain and offset (times the gate), pre's gain and offset
  auto load4 = [&](const float* v, float other, f32x2 (&to)[4]) {
    float f[8];
    fill8(f, other);
    if (live && v != nullptr) load8(v, c, f);
#pragma unroll
    for (int j = 0; j < 4; ++j) to[j] = pack2(f[2 * j], f[2 * j + 1]);
  };
  load4(p.pre_g, 1.f, qg);
  load4(p.pre_b, 0.f, qb);
  const f32x2 scale2 = pack2(p.res_scale, p.res_scale);
  int next_gate = begin, turn = 0;           // next_gate: first row that needs another gate vector than the one held

  for (int row0 = begin; row0 < end; row0 += 4, turn ^= 1) {
    fetch(row0 + 4, turn ^ 1);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    f32x2 v[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool there = live && row0 + i < end;
      unpack_pairs<T>(there ? mine[((turn * 2 + 0) * 4 + i) * threads] : make_uint4(0u, 0u, 0u, 0u), v[i]);
    }
    float sub[4], mul[4];
    if (has_post) {
      row_stats4<kRms>(v, live, p.C, p.eps, s_post[turn], sub, mul);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) v[i][j] = fmul2(kRms ? v[i][j] : fsub2(v[i][j], pack2(sub[i], sub[i])), pack2(mul[i], mul[i]));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = row0 + i;
      if (row < end && row >= next_gate) {               // the same for every thread
        load4(p.post_g, 1.f, pg);
        load4(p.post_b, 0.f, pb);
        if (p.gate != nullptr) {
          f32x2 g[4];
          load4(p.gate + (long long)(row / p.rows_per_gate) * p.C, 1.f, g);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            pg[j] = fmul2(pg[j], g[j]);
            pb[j] = fmul2(pb[j], g[j]);
          }
        }
        next_gate = (row / p.rows_per_gate + 1) * p.rows_per_gate;   // <= rows: whole blocks of rows
      }
      const bool there = live && row < end;
      f32x2 res[4];
      unpack_pairs<T>(there && has_res ? mine[((turn * 2 + 1) * 4 + i) * threads] : make_uint4(0u, 0u, 0u, 0u), res);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i][j] = ffma2(v[i][j], pg[j], ffma2(scale2, res[j], pb[j]));
      if (there) *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.x) + row * p.ldx + c) = pack_pairs<T>(v[i]);
    }
    if (!has_pre) continue;
    row_stats4<kRms>(v, live, p.C, p.eps, s_pre[turn], sub, mul);
    uint4 out[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f32x2 f[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        f[j] = ffma2(fmul2(kRms ? v[i][j] : fsub2(v[i][j], pack2(sub[i], sub[i])), pack2(mul[i], mul[i])), qg[j], qb[j]);
      out[i] = pack_pairs<T>(f);
      if (!kQuant && live && row0 + i < end)
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.y) + (long long)(row0 + i) * p.C + c) = out[i];
    }
    if (kQuant) {
      // the rounded row, as a quantised Linear fed with 16-bit rows would see it
      const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = threads >> 5;
      float amax[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        amax[i] = warp_max(live ? absmax_fold(absmax8(__floats2bfloat162_rn(0.f, 0.f), out[i])) : 0.f);
        if (warps > 1 && lane == 0) s_max[warp * 4 + i] = amax[i];
      }
      if (warps > 1) __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        for (int w = 0; warps > 1 && w < warps; ++w) amax[i] = fmaxf(amax[i], s_max[w * 4 + i]);
        float sc, inv_sc;
        row_scale(amax[i], sc, inv_sc);
        if (row0 + i < end) {
          if (threadIdx.x == 0) p.y_scale[row0 + i] = sc;
          if (live)
            *reinterpret_cast<uint2*>(static_cast<int8_t*>(p.y) + (long long)(row0 + i) * p.C + c) = quant8(out[i], sc, inv_sc);
        }
      }
    }
  }
}

// One row at a time: few rows, where latency counts, and wide ones.  kWide: up to 32 warps a block (C up to 8192), which
// leaves 64 registers a thread: the parameters are then read where they are used.
template <typename T, bool kRms, bool kQuant, bool kWide>
__global__ void __launch_bounds__(kWide ? 1024 : 256)
block_norm_kernel(const NormParams p) {
  constexpr int kMaxWarps = kWide ? 32 : 8;
  __shared__ float2 s_post[2][kMaxWarps], s_pre[2][kMaxWarps];
  __shared__ float s_max[kMaxWarps];         // used between the barriers of two norms
  const int c = int(threadIdx.x) * 8;
  const bool live = c < p.C;
  const int begin = int(blockIdx.x) * p.rows_per_block;
  const int end = begin + min(p.rows_per_block, p.rows - begin);       // begin + rows_per_block may pass 2^31
  const bool has_post = p.post_g != nullptr, has_pre = p.pre_g != nullptr;

  float pg[8], pb[8], qg[8], qb[8];          // post's gain and offset (times the gate), pre's gain and offset
  auto load_post = [&](int row) {
    fill8(pg, 1.f);
    fill8(pb, 0.f);
    if (!live) return;
    if (has_post) load8(p.post_g, c, pg);
    if (p.post_b != nullptr) load8(p.post_b, c, pb);
    if (p.gate != nullptr) {
      float g[8];
      load8(p.gate + (long long)(row / p.rows_per_gate) * p.C, c, g);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        pg[j] *= g[j];
        pb[j] *= g[j];
      }
    }
  };
  auto load_pre = [&]() {
    fill8(qg, 1.f);
    fill8(qb, 0.f);
    if (!live) return;
    if (has_pre) load8(p.pre_g, c, qg);
    if (p.pre_b != nullptr) load8(p.pre_b, c, qb);
  };
  int next_gate = begin, turn = 0;           // next_gate: first row that needs another gate vector than the one held
  if (!kWide) load_pre();

  for (int row = begin; row < end; ++row, turn ^= 1) {
    uint4 hr = make_uint4(0u, 0u, 0u, 0u), rr = hr;
    if (live) {
      hr = *(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.h) + row * p.ldh + c));
      if (p.r != nullptr) rr = *(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.r) + row * p.ldr + c));
    }
    if (kWide || row >= next_gate) {         // the same for every thread
      load_post(row);
      next_gate = (row / p.rows_per_gate + 1) * p.rows_per_gate;     // <= rows: whole blocks of rows
    }
    float v[8], r[8], sub = 0.f, mul = 1.f;
    T::unpack(hr, v);
    T::unpack(rr, r);
    if (has_post) row_stats<kRms>(v, live, p.C, p.eps, s_post[turn], sub, mul);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = fmaf((v[j] - sub) * mul, pg[j], fmaf(p.res_scale, r[j], pb[j]));
    if (live) *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.x) + row * p.ldx + c) = T::pack(v);
    if (!has_pre) continue;
    row_stats<kRms>(v, live, p.C, p.eps, s_pre[turn], sub, mul);
    if (kWide) load_pre();
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = fmaf((v[j] - sub) * mul, qg[j], qb[j]);
    const uint4 out = T::pack(v);
    if (!kQuant) {
      if (live) *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.y) + (long long)row * p.C + c) = out;
      continue;
    }
    // the rounded row, as a quantised Linear fed with 16-bit rows would see it
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    float amax = warp_max(live ? absmax_fold(absmax8(__floats2bfloat162_rn(0.f, 0.f), out)) : 0.f);
    if (warps > 1) {
      if (lane == 0) s_max[warp] = amax;
      __syncthreads();
      for (int w = 0; w < warps; ++w) amax = fmaxf(amax, s_max[w]);
    }
    float sc, inv_sc;
    row_scale(amax, sc, inv_sc);
    if (threadIdx.x == 0) p.y_scale[row] = sc;
    if (live) *reinterpret_cast<uint2*>(static_cast<int8_t*>(p.y) + (long long)row * p.C + c) = quant8(out, sc, inv_sc);
  }
}

// Dynamic shared memory of block_norm_rows_kernel: two turns of four rows of h and r.
constexpr int ring_bytes(int warps) { return 2 * 2 * 4 * warps * 32 * int(sizeof(uint4)); }
constexpr int kStaticBytes = 2 * 2 * 32 * int(sizeof(float2)) + 32 * int(sizeof(float));
static_assert(ring_bytes(5) + kStaticBytes <= 48 * 1024, "up to five warps need no opt-in");

template <typename T, bool kRms, bool kQuant>
int launch_typed(NormParams& p, cudaStream_t st) {
  const int warps = (p.C + 255) / 256, threads = warps * 32;
  const bool wide = warps > 8;
  const int smem = ring_bytes(warps);
  auto rows4 = warps <= 5 ? block_norm_rows_kernel<T, kRms, kQuant, 5> : block_norm_rows_kernel<T, kRms, kQuant, 8>;
  // resident blocks per SM by warps (a device fact, asked once; host threads may ask at once, and give the same answer)
  static std::atomic<int> cached_blocks[9] = {};
  int blocks_sm = 0;
  if (!wide) {
    // Above the 48 KB that a kernel may use unasked, counting its static arrays too (six warps: 48 KB of ring alone).  Always
    // the kernel's largest ring: the limit belongs to the kernel, and another host thread may be about to launch it.
    if (warps > 5 &&
        cudaFuncSetAttribute(rows4, cudaFuncAttributeMaxDynamicSharedMemorySize, ring_bytes(8)) != cudaSuccess)
      return SAMB_E_LAUNCH;
    blocks_sm = cached_blocks[warps].load(std::memory_order_relaxed);
    if (blocks_sm == 0) {
      if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&blocks_sm, rows4, threads, size_t(smem)) != cudaSuccess || blocks_sm < 1)
        return SAMB_E_LAUNCH;
      cached_blocks[warps].store(blocks_sm, std::memory_order_relaxed);
    }
  }
  const long long slots = (long long)sm_count() * blocks_sm;
  if (!wide && p.rows >= 4 * slots) {                    // four rows for every resident block: one resident wave
    p.rows_per_block = int(((p.rows + slots - 1) / slots + 3) / 4 * 4);
    rows4<<<unsigned((p.rows - 1) / p.rows_per_block + 1), threads, smem, st>>>(p);
    return launch_status();
  }
  const long long most = (long long)sm_count() * (wide ? 2 : 8);
  p.rows_per_block = int((p.rows + most - 1) / most);
  const unsigned blocks = unsigned((p.rows - 1) / p.rows_per_block + 1);
  if (wide) block_norm_kernel<T, kRms, kQuant, true><<<blocks, threads, 0, st>>>(p);
  else block_norm_kernel<T, kRms, kQuant, false><<<blocks, threads, 0, st>>>(p);
  return launch_status();
}

int launch_block_norm(const void* h, int64_t ldh, const void* r, int64_t ldr, const float* post_g, const float* post_b,
                      const float* pre_g, const float* pre_b, const float* gate, int64_t gate_rows, float res_scale,
                      float eps, int is_f16, int rms, void* x, int64_t ldx, void* y, float* y_scale, bool quant,
                      int64_t rows, int C, void* stream) {
  if (rows < 0 || C <= 0 || (rows > 0 && (h == nullptr || x == nullptr))) return SAMB_E_BADARG;
  if ((post_g == nullptr && post_b != nullptr) || (pre_g == nullptr && pre_b != nullptr)) return SAMB_E_BADARG;
  if (rows > 0 && ((pre_g == nullptr) != (y == nullptr) || (quant && (y == nullptr || y_scale == nullptr)))) return SAMB_E_BADARG;
  // outputs over inputs: row by row in place, so the rows have to lie alike
  if ((x != nullptr && (x == y || (x == h && ldx != ldh) || (x == r && ldx != ldr))) ||
      (y != nullptr && ((y == h && (quant || ldh != C)) || (y == r && (quant || ldr != C)))))
    return SAMB_E_BADARG;
  if (gate != nullptr && (gate_rows <= 0 || rows % gate_rows)) return SAMB_E_SHAPE;
  if (C % 8 || C > 8192 || rows > 0x7fffff00) return SAMB_E_SHAPE;          // row numbers stay in 32 bits
  if (ldh % 8 || ldx % 8 || ldh < C || ldx < C || (r != nullptr && (ldr % 8 || ldr < C))) return SAMB_E_SHAPE;
  const uintptr_t mis = reinterpret_cast<uintptr_t>(h) | reinterpret_cast<uintptr_t>(r) | reinterpret_cast<uintptr_t>(x) |
                        reinterpret_cast<uintptr_t>(post_g) | reinterpret_cast<uintptr_t>(post_b) |
                        reinterpret_cast<uintptr_t>(pre_g) | reinterpret_cast<uintptr_t>(pre_b) |
                        reinterpret_cast<uintptr_t>(gate) | reinterpret_cast<uintptr_t>(y);
  if ((mis & 15u) || (reinterpret_cast<uintptr_t>(y_scale) & 3u)) return SAMB_E_ALIGN;
  {
    // what is written is memory of its own, or lies exactly over rows that the call may replace (checked above)
    const Runs rh = rows_of(h, 2 * ldh, rows, 2 * C), rr = rows_of(r, 2 * ldr, rows, 2 * C), rx = rows_of(x, 2 * ldx, rows, 2 * C);
    const Runs ry = bytes_of(y, rows * C * (quant ? 1 : 2)), rs = bytes_of(quant ? y_scale : nullptr, rows * 4);
    const Runs vec[5] = {bytes_of(post_g, 4 * C), bytes_of(post_b, 4 * C), bytes_of(pre_g, 4 * C), bytes_of(pre_b, 4 * C),
                         bytes_of(gate, 4 * gate_rows * C)};
    if ((x != h && share_memory(rx, rh)) || (x != r && share_memory(rx, rr)) || (y != h && share_memory(ry, rh)) ||
        (y != r && share_memory(ry, rr)) || share_memory(rx, ry) || share_memory(rs, rh) || share_memory(rs, rr) ||
        share_memory(rs, rx) || share_memory(rs, ry))
      return SAMB_E_BADARG;
    for (const Runs& v : vec)
      if (share_memory(v, rx) || share_memory(v, ry) || share_memory(v, rs)) return SAMB_E_BADARG;
  }
  if (int e = check_device_arch()) return e;
  if (rows == 0) return SAMB_OK;
  NormParams p;
  p.h = h; p.r = r; p.post_g = post_g; p.post_b = post_b; p.pre_g = pre_g; p.pre_b = pre_b; p.gate = gate;
  p.x = x; p.y = y; p.y_scale = y_scale;
  p.ldh = ldh; p.ldr = ldr; p.ldx = ldx;
  p.rows = int(rows); p.C = C;
  p.rows_per_gate = int(gate != nullptr ? rows / gate_rows : rows);
  p.res_scale = res_scale; p.eps = eps;
  auto st = static_cast<cudaStream_t>(stream);
  if (quant) return rms ? launch_typed<Bf16, true, true>(p, st) : launch_typed<Bf16, false, true>(p, st);
  if (is_f16) return rms ? launch_typed<F16, true, false>(p, st) : launch_typed<F16, false, false>(p, st);
  return rms ? launch_typed<Bf16, true, false>(p, st) : launch_typed<Bf16, false, false>(p, st);
}

}  // namespace
}  // namespace samb

extern "C" {

int samb_block_norm(const void* h, int64_t ldh, const void* residual, int64_t ldr, const float* post_gamma,
                    const float* post_beta, const float* pre_gamma, const float* pre_beta, const float* gate,
                    int64_t gate_rows, float res_scale, float eps, int is_f16, int rms, void* x_new, int64_t ldx, void* y,
                    int64_t rows, int C, void* stream) {
  return samb::launch_block_norm(h, ldh, residual, ldr, post_gamma, post_beta, pre_gamma, pre_beta, gate, gate_rows,
                                 res_scale, eps, is_f16, rms, x_new, ldx, y, nullptr, false, rows, C, stream);
}

int samb_block_norm_quant_i8(const void* h, int64_t ldh, const void* residual, int64_t ldr, const float* post_gamma,
                             const float* post_beta, const float* pre_gamma, const float* pre_beta, const float* gate,
                             int64_t gate_rows, float res_scale, float eps, int rms, void* x_new, int64_t ldx, int8_t* yq,
                             float* y_scale, int64_t rows, int C, void* stream) {
  return samb::launch_block_norm(h, ldh, residual, ldr, post_gamma, post_beta, pre_gamma, pre_beta, gate, gate_rows,
                                 res_scale, eps, 0, rms, x_new, ldx, yq, y_scale, true, rows, C, stream);
}

}  // extern "C"
