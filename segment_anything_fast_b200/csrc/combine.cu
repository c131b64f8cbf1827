// Combination of the experts' rows: y[t] = residual[t] + sum_j weights[t, j] * x[slots[t, j]], summed in fp32 in the
// order of j and rounded once.  A slot outside x (the router gives -1 to a choice that a token did not make) adds
// nothing.  Bound by HBM: every row of x is read once; a thread owns eight columns of a token and has the loads of
// all its choices in flight together.  52 us for 32768 tokens x 2 choices x 1280 bf16 with the residual (335 MB, 6.4 TB/s).
#include "elem16.cuh"
#include "overlap.h"

namespace samb {
namespace {

constexpr int kChoices = 8;

struct CombineParams {
  const uint16_t* x;
  const int* slots;
  const float* weights;
  const uint16_t* residual;
  uint16_t* out;
  long long ldx, ldr, ldo, x_rows;
  unsigned T, nvec;
};

template <typename T, int K>
__global__ void __launch_bounds__(256)
combine_kernel(const CombineParams p) {
  const unsigned long long i = (unsigned long long)blockIdx.x * 256 + threadIdx.x;
  const unsigned t = unsigned(i / p.nvec);
  const unsigned v = unsigned(i - (unsigned long long)t * p.nvec);
  if (t >= p.T) return;
  uint4 raw[K];
  float w[K];
#pragma unroll
  for (int j = 0; j < K; ++j) {
    const int s = __ldg(p.slots + (long long)t * K + j);
    const bool there = s >= 0 && s < p.x_rows;
    w[j] = there ? __ldg(p.weights + (long long)t * K + j) : 0.f;
    raw[j] = there ? __ldcs(reinterpret_cast<const uint4*>(p.x + s * p.ldx) + v) : make_uint4(0u, 0u, 0u, 0u);
  }
  float sum[8];
  if (p.residual != nullptr) {
    T::unpack(*(reinterpret_cast<const uint4*>(p.residual + t * p.ldr) + v), sum);
  } else {
#pragma unroll
    for (int c = 0; c < 8; ++c) sum[c] = 0.f;
  }
#pragma unroll
  for (int j = 0; j < K; ++j) {
    float f[8];
    T::unpack(raw[j], f);
#pragma unroll
    for (int c = 0; c < 8; ++c) sum[c] = fmaf(w[j], f[c], sum[c]);
  }
  *(reinterpret_cast<uint4*>(p.out + t * p.ldo) + v) = T::pack(sum);
}

template <typename T>
int launch_combine(const CombineParams& p, int k, cudaStream_t st) {
  const unsigned long long blocks = ((unsigned long long)p.T * p.nvec + 255) / 256;
  if (blocks > 0x7fffffffull) return SAMB_E_SHAPE;
  const unsigned b = unsigned(blocks);
  switch (k) {
    case 1: combine_kernel<T, 1><<<b, 256, 0, st>>>(p); break;
    case 2: combine_kernel<T, 2><<<b, 256, 0, st>>>(p); break;
    case 3: combine_kernel<T, 3><<<b, 256, 0, st>>>(p); break;
    case 4: combine_kernel<T, 4><<<b, 256, 0, st>>>(p); break;
    case 5: combine_kernel<T, 5><<<b, 256, 0, st>>>(p); break;
    case 6: combine_kernel<T, 6><<<b, 256, 0, st>>>(p); break;
    case 7: combine_kernel<T, 7><<<b, 256, 0, st>>>(p); break;
    default: combine_kernel<T, 8><<<b, 256, 0, st>>>(p); break;
  }
  return launch_status();
}

}  // namespace
}  // namespace samb

extern "C" {

int samb_combine_topk(const void* x, int64_t ldx, int64_t x_rows, const int32_t* slots, const float* weights,
                      const void* residual, int64_t ldr, void* out, int64_t ldo, int64_t T, int k, int C, int is_f16,
                      void* stream) {
  using namespace samb;
  if (T < 0 || k <= 0 || C <= 0 || x_rows < 0) return SAMB_E_BADARG;
  if (T > 0 && (slots == nullptr || weights == nullptr || out == nullptr || (x == nullptr && x_rows > 0))) return SAMB_E_BADARG;
  if (out != nullptr && (out == x || (out == residual && ldo != ldr))) return SAMB_E_BADARG;
  if (k > kChoices || C % 8 || T >= (int64_t(1) << 31)) return SAMB_E_SHAPE;
  if (ldx % 8 || ldo % 8 || ldx < C || ldo < C || (residual != nullptr && (ldr % 8 || ldr < C))) return SAMB_E_SHAPE;
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) | reinterpret_cast<uintptr_t>(out)) & 15u)
    return SAMB_E_ALIGN;
  if ((reinterpret_cast<uintptr_t>(slots) | reinterpret_cast<uintptr_t>(weights)) & 3u) return SAMB_E_ALIGN;
  {
    const Runs ro = rows_of(out, 2 * ldo, T, 2 * C);
    if (share_memory(ro, rows_of(x, 2 * ldx, x_rows, 2 * C)) || share_memory(ro, bytes_of(slots, 4 * T * k)) ||
        share_memory(ro, bytes_of(weights, 4 * T * k)) ||
        (out != residual && share_memory(ro, rows_of(residual, 2 * ldr, T, 2 * C))))
      return SAMB_E_BADARG;
  }
  if (int e = check_device_arch()) return e;
  if (T == 0) return SAMB_OK;
  CombineParams p;
  p.x = static_cast<const uint16_t*>(x);
  p.slots = slots; p.weights = weights;
  p.residual = static_cast<const uint16_t*>(residual);
  p.out = static_cast<uint16_t*>(out);
  p.ldx = ldx; p.ldr = ldr; p.ldo = ldo; p.x_rows = x_rows;
  p.T = unsigned(T); p.nvec = unsigned(C / 8);
  auto st = static_cast<cudaStream_t>(stream);
  return is_f16 ? launch_combine<F16>(p, k, st) : launch_combine<Bf16>(p, k, st);
}

}  // extern "C"
