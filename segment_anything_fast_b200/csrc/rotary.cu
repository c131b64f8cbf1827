// Rotary positions on planes of rows (head-major q and k, or any strided [planes, rows, d] view): pair p of a row,
// (a, b), becomes
//   (a cos t - b sin t,  b cos t + a sin t) * mscale,   t = position[axis(p)] * freqs[p],
// where the pairs are neighbours (interleaved) or lie rot / 2 apart (half layout), the first rot elements of a row
// are rotated and the rest are copied.  With two axes the first half of the pairs turns with the first coordinate,
// the second half with the second (rasters).
//
// Angles: a float angle of position 10^6 is off by 0.06 rad, and reducing a double angle costs more than the
// rotation.  A frequency is instead held as a 64-bit fixed-point fraction of a turn, F = frac(freq / 2 pi) * 2^64, and
// position * F modulo 2^64 is the exact fraction of the turn that this F reaches: one integer product, no reduction.
// Its top 32 bits, rounded to fp32, are the argument of sincospi: the angle is off by at most 2^-32 turns (bits dropped), 2^-26
// turns (fp32 holds 24 bits of up to half a turn; less for smaller angles) and position * 2^-63 turns (F: its own last
// place, and the second part of the product that makes it).
//
// A thread owns V pairs of a position and walks over the copies that share it (planes x repetitions of the
// positions), so the angles are worked out once and the copies stream, four of them in flight a thread.  Bound by HBM:
// 60 us for 32 planes x 32768 rows x 80 bf16 (335 MB, 5.6 TB/s; neighbours 61 us; 5 us more with one copy in flight).
#include "elem16.cuh"
#include "overlap.h"

namespace samb {
namespace {

struct RotaryParams {
  const uint16_t* x;
  uint16_t* out;
  const void* pos;
  const double* freqs;
  long long xp, xr, op, orow;      // strides in elements: plane, row
  unsigned period;                 // positions
  unsigned repeats;                // rows = repeats * period
  unsigned planes;
  unsigned step_plane, step_rep;   // gridDim.y copies on: so many planes and repetitions
  int pos64, axes, rot, half, d;
  int units, tails, tail_len;      // V-pair units of a row, then units of tail_len copied elements
  float mscale;
};

// V 16-bit elements in one access
template <int V>
__device__ __forceinline__ void load_vec(const uint16_t* p, uint16_t (&e)[V]) {
  if constexpr (V == 8) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    *reinterpret_cast<uint4*>(e) = u;
  } else if constexpr (V == 4) {
    *reinterpret_cast<uint2*>(e) = *reinterpret_cast<const uint2*>(p);
  } else if constexpr (V == 2) {
    *reinterpret_cast<uint32_t*>(e) = *reinterpret_cast<const uint32_t*>(p);
  } else {
    e[0] = *p;
  }
}
template <int V>
__device__ __forceinline__ void store_vec(uint16_t* p, const uint16_t (&e)[V]) {
  if constexpr (V == 8) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(e);
  else if constexpr (V == 4) *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(e);
  else if constexpr (V == 2) *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(e);
  else *p = e[0];
}

template <typename T, bool kInter, int V>
__global__ void __launch_bounds__(256)
rotary_kernel(const RotaryParams p) {
  const unsigned per_row = unsigned(p.units + p.tails);
  const unsigned long long t = (unsigned long long)blockIdx.x * blockDim.x + threadIdx.x;
  const unsigned row = unsigned(t / per_row);
  const int u = int(t - (unsigned long long)row * per_row);
  if (row >= p.period) return;
  // the copies of this thread: blockIdx.y, blockIdx.y + gridDim.y, ..., as (plane, repetition)
  unsigned left = (p.planes * p.repeats - blockIdx.y + gridDim.y - 1) / gridDim.y;
  unsigned plane = blockIdx.y / p.repeats, rep = blockIdx.y - plane * p.repeats;
  auto next = [&]() {
    plane += p.step_plane;
    rep += p.step_rep;
    if (rep >= p.repeats) {
      rep -= p.repeats;
      ++plane;
    }
  };

  if (u >= p.units) {                                    // elements behind the rotated ones
    const int c = p.rot + (u - p.units) * p.tail_len;
    for (; left > 0; --left, next()) {
      const long long r = (long long)rep * p.period + row;
      const uint16_t* src = p.x + plane * p.xp + r * p.xr + c;
      uint16_t* dst = p.out + plane * p.op + r * p.orow + c;
      if (p.tail_len == 8) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src);
      else *dst = *src;
    }
    return;
  }

  float cs[V], sn[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int pair = u * V + j;
    const int axis = p.axes == 2 && pair >= p.half / 2 ? 1 : 0;
    const long long at = (long long)row * p.axes + axis;
    const long long pos = p.pos64 ? static_cast<const long long*>(p.pos)[at] : (long long)static_cast<const int*>(p.pos)[at];
    // freq / 2 pi as an unevaluated sum of two doubles; the fraction of the first is a multiple of its last place
    constexpr double kInv = 0.15915494309189535, kInvLow = -9.839338337591243e-18, kOne = 18446744073709551616.0;
    const double f = p.freqs[pair], hi = f * kInv, lo = fma(f, kInv, -hi) + f * kInvLow;
    const unsigned long long step = (unsigned long long)((hi - floor(hi)) * kOne) + (unsigned long long)(long long)(lo * kOne);
    const int turn = int((unsigned)(((unsigned long long)pos * step) >> 32));           // [-1/2, 1/2) turns
    sincospif(float(turn) * 4.656612873077392578125e-10f, &sn[j], &cs[j]);              // * 2^-31: half turns
    cs[j] *= p.mscale;
    sn[j] *= p.mscale;
  }

  // the two parts of the unit: neighbours are one run of 2 V elements, halves are two runs of V
  constexpr int kRun = kInter ? 2 * V : V, kRuns = kInter ? 1 : 2;
  const int c = u * kRun;
  while (left > 0) {
    alignas(16) uint16_t e[4][kRuns][kRun];
    uint16_t* dst[4];
    const unsigned n = min(left, 4u);
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      if (b >= n) break;
      const long long r = (long long)rep * p.period + row;
      const uint16_t* src = p.x + plane * p.xp + r * p.xr + c;
      dst[b] = p.out + plane * p.op + r * p.orow + c;
      load_vec<kRun>(src, e[b][0]);
      if (!kInter) load_vec<kRun>(src + p.half, e[b][kRuns - 1]);
      next();
    }
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      if (b >= n) break;
      alignas(16) uint16_t o[kRuns][kRun];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int r1 = kRuns - 1, j0 = kInter ? 2 * j : j, j1 = kInter ? 2 * j + 1 : j;
        const float a = T::to_float(e[b][0][j0]), d = T::to_float(e[b][r1][j1]);
        o[0][j0] = T::from_float(fmaf(a, cs[j], -d * sn[j]));
        o[r1][j1] = T::from_float(fmaf(d, cs[j], a * sn[j]));
      }
      store_vec<kRun>(dst[b], o[0]);
      if (!kInter) store_vec<kRun>(dst[b] + p.half, o[kRuns - 1]);
    }
    left -= n;
  }
}

template <typename T, bool kInter, int V>
int launch_rotary(RotaryParams p, cudaStream_t st) {
  p.units = p.half / V;
  const unsigned long long threads = (unsigned long long)p.period * unsigned(p.units + p.tails);
  const unsigned long long bx = (threads + 255) / 256;
  if (bx > 0x7fffffffull) return SAMB_E_SHAPE;
  const unsigned copies = p.planes * p.repeats;
  // enough threads to fill the GPU, otherwise as many copies a thread as possible
  unsigned long long by = ((unsigned long long)sm_count() * 8 + bx - 1) / bx;
  if (by > copies) by = copies;
  if (by > 65535) by = 65535;
  p.step_plane = unsigned(by) / p.repeats;
  p.step_rep = unsigned(by) % p.repeats;
  rotary_kernel<T, kInter, V><<<dim3(unsigned(bx), unsigned(by)), 256, 0, st>>>(p);
  return launch_status();
}

template <typename T>
int pick_rotary(const RotaryParams& p, bool inter, cudaStream_t st) {
  // widest access that the layout allows: rows start at 16-byte boundaries, the second half of a pair at `half`
  if (inter) {
    if (p.half % 4 == 0) return launch_rotary<T, true, 4>(p, st);
    return launch_rotary<T, true, 1>(p, st);
  }
  if (p.half % 8 == 0) return launch_rotary<T, false, 8>(p, st);
  if (p.half % 4 == 0) return launch_rotary<T, false, 4>(p, st);
  if (p.half % 2 == 0) return launch_rotary<T, false, 2>(p, st);
  return launch_rotary<T, false, 1>(p, st);
}

}  // namespace
}  // namespace samb

extern "C" {

int samb_rotary(const void* x, int64_t plane_stride, int64_t row_stride, const void* positions, int positions_i64,
                int64_t period, int axes, const double* freqs, int rot, int interleaved, float mscale, void* out,
                int64_t out_plane_stride, int64_t out_row_stride, int64_t planes, int64_t rows, int d, int is_f16,
                void* stream) {
  using namespace samb;
  if (rows > 0 && planes > 0 && (x == nullptr || out == nullptr || positions == nullptr || freqs == nullptr))
    return SAMB_E_BADARG;
  if (planes < 0 || rows < 0 || d <= 0 || rot <= 0 || (axes != 1 && axes != 2)) return SAMB_E_BADARG;
  if (rot > d || rot % (2 * axes)) return SAMB_E_SHAPE;
  if (rows >= (int64_t(1) << 31) || planes >= (int64_t(1) << 31)) return SAMB_E_SHAPE;
  if (rows > 0 && (period <= 0 || rows % period)) return SAMB_E_SHAPE;
  if (plane_stride < 0 || row_stride < 0 || out_plane_stride < 0 || out_row_stride < 0) return SAMB_E_SHAPE;
  if ((plane_stride | row_stride | out_plane_stride | out_row_stride) & 7) return SAMB_E_ALIGN;
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)) & 15u) return SAMB_E_ALIGN;
  if ((reinterpret_cast<uintptr_t>(freqs) & 7u) || (reinterpret_cast<uintptr_t>(positions) & (positions_i64 ? 7u : 3u)))
    return SAMB_E_ALIGN;
  // in place means the same rows at the same strides
  if (x == out && (plane_stride != out_plane_stride || row_stride != out_row_stride)) return SAMB_E_BADARG;
  // no two rows of out may share memory
  {
    const bool by_row = rows > 1 && (planes <= 1 || out_row_stride >= out_plane_stride);     // rows are the outer axis
    const int64_t outer = by_row ? out_row_stride : out_plane_stride, inner = by_row ? out_plane_stride : out_row_stride;
    const int64_t n_outer = by_row ? rows : planes, n_inner = by_row ? planes : rows;
    if ((n_inner > 1 && inner < d) || (n_outer > 1 && outer < (n_inner > 1 ? (n_inner - 1) * inner : 0) + d))
      return SAMB_E_SHAPE;
  }
  {
    const Runs ro = runs3(out, 2 * out_plane_stride, planes, 2 * out_row_stride, rows, 2 * d);
    if ((x != out && share_memory(ro, runs3(x, 2 * plane_stride, planes, 2 * row_stride, rows, 2 * d))) ||
        share_memory(ro, bytes_of(positions, rows > 0 ? period * axes * (positions_i64 ? 8 : 4) : 0)) ||
        share_memory(ro, bytes_of(freqs, 4 * int64_t(rot))))
      return SAMB_E_BADARG;
  }
  if (int e = check_device_arch()) return e;
  if (rows == 0 || planes == 0) return SAMB_OK;
  if (planes * (rows / period) >= (int64_t(1) << 31)) return SAMB_E_SHAPE;
  RotaryParams p;
  p.x = static_cast<const uint16_t*>(x);
  p.out = static_cast<uint16_t*>(out);
  p.pos = positions;
  p.freqs = freqs;
  p.xp = plane_stride; p.xr = row_stride; p.op = out_plane_stride; p.orow = out_row_stride;
  p.period = unsigned(period);
  p.repeats = unsigned(rows / period);
  p.planes = unsigned(planes);
  p.pos64 = positions_i64 != 0;
  p.axes = axes; p.rot = rot; p.half = rot / 2; p.d = d;
  p.units = 0;
  p.tail_len = rot % 8 == 0 && d % 8 == 0 ? 8 : 1;
  p.tails = x == out ? 0 : (d - rot) / p.tail_len;
  p.mscale = mscale;
  auto st = static_cast<cudaStream_t>(stream);
  return is_f16 ? pick_rotary<F16>(p, interleaved != 0, st) : pick_rotary<Bf16>(p, interleaved != 0, st);
}

}  // extern "C"
