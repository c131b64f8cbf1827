// The router of a mixture of experts: every token's k largest logits, their weights, and the order of the chosen
// (token, choice) pairs by expert in which the grouped products take them.
//
// Choice: eight lanes (up to 64 experts: four tokens a warp) or a warp (up to 512) hold a token's logits as order-preserving
// integers, the next tokens' on their way; each of the k rounds is a maximum over the lanes, the lowest index among
// equals.  Order: a stable counting sort.  Each block counts the experts of its own run of tokens; then (second launch, or
// after a barrier when one block is enough) it adds up the counts of the blocks before it and places its pairs in
// order: a warp owns a run of pairs, ranks equal experts among its lanes with match_any and keeps a running count per
// expert in shared memory.  Nothing depends on the order in which atomics arrive.  Bound by latency: 19 us for 32768 tokens x
// 64 experts, k = 4 (34 us with a warp a token, 20 us with four a warp by warp-wide maxima and ballots), 3.8 us for one token.
#include "common.cuh"

namespace samb {
namespace {

constexpr int kRouteWarps = 16;
constexpr int kRouteThreads = kRouteWarps * 32;
constexpr int kMaxExperts = 512;
constexpr int kMaxChoices = 8;

struct RouteParams {
  const float* logits;
  const float* bias;
  int* ids;
  float* weights;
  int* slots;
  int* rows;
  int* offsets;
  int* counts;                     // [blocks][E] scratch
  long long ld;
  int T, E, k;
  int tokens_per_block;
  int sigmoid, renorm;
  float scale;
};

// Larger float <=> larger integer; 0 stands below every key of a number that may be chosen.
__device__ __forceinline__ unsigned order_key(float v) {
  if (!(v > -INFINITY)) return 0u;                       // -inf and NaN are never chosen
  v = fminf(v, 3.402823466e38f) + 0.0f;                  // +inf counts as the largest number, -0 as +0
  const unsigned b = __float_as_uint(v);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// L lanes a token (8 or 32); lane `sub` of them holds the experts i * L + sub.
template <int L, int NE>
__device__ __forceinline__ void load_logits(const RouteParams& p, int token, bool live, float (&x)[NE]) {
  const int sub = threadIdx.x & (L - 1);
  const float* lr = p.logits + token * p.ld;
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    const int e = i * L + sub;
    x[i] = live && e < p.E ? __ldg(lr + e) : -INFINITY;
  }
}

template <int L>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <int L, int NE>
__device__ __forceinline__ void choose_token(const RouteParams& p, int token, bool live, const float (&bias)[NE],
                                             const float (&x)[NE]) {
  const int lane = threadIdx.x & 31, sub = lane & (L - 1);
  float v[NE];
  unsigned key[NE];
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    const bool on = x[i] > -INFINITY;                    // neither switched off (whatever the bias says) nor NaN
    v[i] = on ? fminf(x[i], 3.402823466e38f) : -INFINITY;
    key[i] = on ? order_key(p.bias != nullptr ? x[i] + bias[i] : x[i]) : 0u;
  }
  float top = 0.f, denom = 1.f;
  if (!p.sigmoid && !p.renorm) {                         // the sum over all experts cancels when renormalising
    top = -INFINITY;
#pragma unroll
    for (int i = 0; i < NE; ++i) top = fmaxf(top, v[i]);
    top = lanes_max<L>(top);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NE; ++i)
      if (v[i] > -INFINITY) s += expf(v[i] - top);
    denom = lanes_sum<L>(s);
  }
  int my_id = -1;                                        // lane j keeps choice j
  float my_x = -INFINITY;
  for (int j = 0; j < p.k; ++j) {
    unsigned best = 0u;
    int at = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < NE; ++i)
      if (key[i] > best) {                               // the lane's lowest index among equals
        best = key[i];
        at = i * L + sub;
      }
    if constexpr (L == 32) {
      const unsigned all = __reduce_max_sync(0xffffffffu, best);
      at = int(__reduce_min_sync(0xffffffffu, best == all ? unsigned(at) : 0x7fffffffu));
      if (all == 0u) break;                              // nobody is left
    } else {
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) {
        const unsigned ob = __shfl_xor_sync(0xffffffffu, best, o);
        const int oa = __shfl_xor_sync(0xffffffffu, at, o);
        if (ob > best || (ob == best && oa < at)) {
          best = ob;
          at = oa;
        }
      }
    }
    float xv = -INFINITY;
#pragma unroll
    for (int i = 0; i < NE; ++i)
      if (i * L + sub == at) {
        xv = v[i];
        key[i] = 0u;
      }
    xv = __shfl_sync(0xffffffffu, xv, (lane & ~(L - 1)) | (at & (L - 1)));
    if (sub == j && at != 0x7fffffff) {
      my_id = at;
      my_x = xv;
    }
  }
  float my_w;
  if (p.renorm) {
    // relative to the chosen ones' largest, so that they never all vanish; a sigmoid below e^-20 is an exponential
    const float m = lanes_max<8>(my_x);                  // lanes of no choice hold -inf; choices sit in the first eight
    my_w = p.sigmoid && m > -20.f ? 1.f / (1.f + expf(-my_x)) : expf(my_x - m);
    if (my_id < 0) my_w = 0.f;
    const float s = lanes_sum<8>(my_w);
    my_w = s > 0.f ? my_w / s : 0.f;
  } else {
    my_w = my_id < 0 ? 0.f : p.sigmoid ? 1.f / (1.f + expf(-my_x)) : expf(my_x - top) / denom;
  }
  if (live && sub < p.k) {
    const long long to = (long long)token * p.k + sub;
    p.ids[to] = my_id;
    p.weights[to] = my_w * p.scale;
  }
}

template <int L, int NE>
__device__ __forceinline__ void choose_block(const RouteParams& p, int t0, int t1) {
  constexpr int kStep = kRouteWarps * (32 / L);          // tokens a round of the block
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int mine = warp * (32 / L) + lane / L;
  float bias[NE], x[NE], next[NE];
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    const int e = i * L + (lane & (L - 1));
    bias[i] = p.bias != nullptr && e < p.E ? __ldg(p.bias + e) : 0.f;
  }
  load_logits<L, NE>(p, t0 + mine, t0 + mine < t1, next);
  for (int r0 = t0; r0 < t1; r0 += kStep) {              // the same number of rounds for every lane
    const int t = r0 + mine;
#pragma unroll
    for (int i = 0; i < NE; ++i) x[i] = next[i];
    load_logits<L, NE>(p, t + kStep, t + kStep < t1, next);
    choose_token<L, NE>(p, t, t < t1, bias, x);
  }
}

// counts of the block's pairs, into cnt[0 .. E)
__device__ __forceinline__ void count_block(const RouteParams& p, int t0, int t1, int* cnt) {
  for (int e = threadIdx.x; e < p.E; e += kRouteThreads) cnt[e] = 0;
  __syncthreads();                                       // also: the block's ids are written
  const long long lo = (long long)t0 * p.k, hi = (long long)t1 * p.k;
  for (long long i = lo + threadIdx.x; i < hi; i += kRouteThreads) {
    const int e = p.ids[i];
    if (e >= 0) atomicAdd(cnt + e, 1);                   // a count: the order does not matter
  }
  __syncthreads();
}

// Places the block's pairs.  base[e]: pairs of expert e in earlier blocks plus all pairs of earlier experts; run:
// [kRouteWarps][E] shared scratch; total: pairs placed over all blocks.
__device__ __forceinline__ void place_block(const RouteParams& p, int t0, int t1, const int* base, int* run, int total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long lo = (long long)t0 * p.k, n = (long long)(t1 - t0) * p.k;
  const long long part = (n + kRouteThreads - 1) / kRouteThreads * 32;      // pairs a warp, whole rounds of 32
  const long long w0 = lo + warp * part, w1 = min(lo + n, w0 + part);
  int* mine = run + warp * p.E;
  for (int e = lane; e < p.E; e += 32) mine[e] = 0;
  __syncwarp();
  for (long long i0 = w0; i0 < w1; i0 += 32) {
    const int e = i0 + lane < w1 ? p.ids[i0 + lane] : -1;
    const unsigned same = __match_any_sync(0xffffffffu, e);
    if (e >= 0 && (same & ((1u << lane) - 1u)) == 0u) mine[e] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.E; e += kRouteThreads) {   // counts -> first slot of each warp
    int at = base[e];
    for (int w = 0; w < kRouteWarps; ++w) {
      const int c = run[w * p.E + e];
      run[w * p.E + e] = at;
      at += c;
    }
  }
  __syncthreads();
  for (long long i0 = w0; i0 < w1; i0 += 32) {
    const long long i = i0 + lane;
    const int e = i < w1 ? p.ids[i] : -1;
    const unsigned same = __match_any_sync(0xffffffffu, e);
    const unsigned before = same & ((1u << lane) - 1u);
    int slot = -1;
    if (e >= 0) slot = mine[e] + __popc(before);
    __syncwarp();
    if (e >= 0 && before == 0u) mine[e] += __popc(same);
    __syncwarp();
    if (i < w1) {
      p.slots[i] = slot;
      if (slot >= 0) p.rows[slot] = int(i / p.k);
    }
  }
  // the slots that nobody takes
  const long long all = (long long)p.T * p.k;
  for (long long s = total + (long long)blockIdx.x * kRouteThreads + threadIdx.x; s < all; s += (long long)gridDim.x * kRouteThreads)
    p.rows[s] = -1;
}

// exclusive scan of tot[0 .. E) into off[0 .. E], by one warp
__device__ __forceinline__ void scan_experts(const int* tot, int* off, int E) {
  const int lane = threadIdx.x & 31;
  int carry = 0;
  for (int e0 = 0; e0 < E; e0 += 32) {
    const int c = e0 + lane < E ? tot[e0 + lane] : 0;
    int s = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += up;
    }
    if (e0 + lane < E) off[e0 + lane] = carry + s - c;
    carry += __shfl_sync(0xffffffffu, s, 31);
  }
  if (lane == 0) off[E] = carry;
}

// kOne: the only block does everything.  Otherwise this launch chooses and counts.
template <int L, int NE, bool kOne>
__global__ void __launch_bounds__(kRouteThreads)
route_choose_kernel(const RouteParams p) {
  extern __shared__ int sm[];
  const int t0 = min(p.T, int(blockIdx.x) * p.tokens_per_block), t1 = min(p.T, t0 + p.tokens_per_block);
  choose_block<L, NE>(p, t0, t1);
  count_block(p, t0, t1, sm);
  if (!kOne) {
    for (int e = threadIdx.x; e < p.E; e += kRouteThreads) p.counts[(long long)blockIdx.x * p.E + e] = sm[e];
    return;
  }
  int* off = sm + p.E;                                   // [E + 1]
  if (threadIdx.x < 32) scan_experts(sm, off, p.E);
  __syncthreads();
  for (int e = threadIdx.x; e <= p.E; e += kRouteThreads) p.offsets[e] = off[e];
  place_block(p, t0, t1, off, off + p.E + 1, off[p.E]);
}

__global__ void __launch_bounds__(kRouteThreads)
route_place_kernel(const RouteParams p) {
  extern __shared__ int sm[];
  int* tot = sm;                                         // [E]: pairs of the expert in all blocks
  int* off = tot + p.E;                                  // [E + 1]
  int* base = off + p.E + 1;                             // [E]
  int* run = base + p.E;                                 // [kRouteWarps][E]
  const int t0 = min(p.T, int(blockIdx.x) * p.tokens_per_block), t1 = min(p.T, t0 + p.tokens_per_block);
  for (int e = threadIdx.x; e < p.E; e += kRouteThreads) tot[e] = base[e] = 0;
  __syncthreads();
  // all counts: a thread adds up one expert over every few blocks; whole numbers, in any order
  int width = 32;
  while (width < p.E) width *= 2;                        // divides kRouteThreads (E <= 512)
  {
    const int e = int(threadIdx.x) & (width - 1), step = kRouteThreads / width;
    if (e < p.E) {
      int all = 0, before = 0;
#pragma unroll 8
      for (int b = int(threadIdx.x) / width; b < int(gridDim.x); b += step) {
        const int c = p.counts[(long long)b * p.E + e];
        all += c;
        if (b < int(blockIdx.x)) before += c;
      }
      if (all != 0) atomicAdd(tot + e, all);
      if (before != 0) atomicAdd(base + e, before);
    }
  }
  __syncthreads();
  if (threadIdx.x < 32) scan_experts(tot, off, p.E);
  __syncthreads();
  for (int e = threadIdx.x; e < p.E; e += kRouteThreads) base[e] += off[e];
  if (blockIdx.x == 0)
    for (int e = threadIdx.x; e <= p.E; e += kRouteThreads) p.offsets[e] = off[e];
  __syncthreads();
  place_block(p, t0, t1, base, run, off[p.E]);
}

constexpr int kSmallExperts = 64;                          // eight lanes a token

// One block for up to two rounds of its warps (64 experts: 128 tokens take 8.7 us in one block and in two launches alike, 256
// tokens 14.0 and 8.5), otherwise one a round of tokens, at most one an SM (their counts are read by every block).
int route_blocks(int64_t T, int E) {
  const int step = kRouteWarps * (E <= kSmallExperts ? 4 : 1);
  if (T <= 2 * step) return 1;
  const int64_t want = (T + step - 1) / step, most = 148;
  return int(want < most ? want : most);
}

template <int L, int NE>
int launch_route(RouteParams p, cudaStream_t st) {
  const int blocks = route_blocks(p.T, p.E);
  p.tokens_per_block = (p.T + blocks - 1) / blocks;
  const size_t one = sizeof(int) * size_t(p.E + p.E + 1 + kRouteWarps * p.E);
  if (blocks == 1) {
    route_choose_kernel<L, NE, true><<<1, kRouteThreads, one, st>>>(p);
    return launch_status();
  }
  route_choose_kernel<L, NE, false><<<blocks, kRouteThreads, sizeof(int) * p.E, st>>>(p);
  if (int e = launch_status()) return e;
  route_place_kernel<<<blocks, kRouteThreads, one + sizeof(int) * p.E, st>>>(p);
  return launch_status();
}

}  // namespace
}  // namespace samb

extern "C" {

int64_t samb_route_scratch_bytes(int64_t T, int E) {
  if (T < 0 || E <= 0 || E > samb::kMaxExperts) return 0;
  const int blocks = samb::route_blocks(T, E);
  return blocks == 1 ? 0 : int64_t(blocks) * E * int64_t(sizeof(int));
}

int samb_route_topk(const float* logits, int64_t ld, const float* bias, int64_t T, int E, int k, int sigmoid, int renorm,
                    float scale, int32_t* ids, float* weights, int32_t* slots, int32_t* rows, int32_t* offsets,
                    void* scratch, void* stream) {
  using namespace samb;
  if (T < 0 || E <= 0 || k <= 0 || offsets == nullptr) return SAMB_E_BADARG;
  if (T > 0 && (logits == nullptr || ids == nullptr || weights == nullptr || slots == nullptr || rows == nullptr))
    return SAMB_E_BADARG;
  if (E > kMaxExperts || k > kMaxChoices || k > E || ld < E || T > 0x7fff0000 / k) return SAMB_E_SHAPE;    // pairs in 32 bits
  const uintptr_t mis = reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(bias) |
                        reinterpret_cast<uintptr_t>(ids) | reinterpret_cast<uintptr_t>(weights) |
                        reinterpret_cast<uintptr_t>(slots) | reinterpret_cast<uintptr_t>(rows) |
                        reinterpret_cast<uintptr_t>(offsets) | reinterpret_cast<uintptr_t>(scratch);
  if (mis & 3u) return SAMB_E_ALIGN;
  if (route_blocks(T, E) > 1 && scratch == nullptr) return SAMB_E_BADARG;
  if (int e = check_device_arch()) return e;
  RouteParams p;
  p.logits = logits; p.bias = bias; p.ids = ids; p.weights = weights; p.slots = slots; p.rows = rows; p.offsets = offsets;
  p.counts = static_cast<int*>(scratch);
  p.ld = ld; p.T = int(T); p.E = E; p.k = k;
  p.sigmoid = sigmoid != 0; p.renorm = renorm != 0; p.scale = scale;
  auto st = static_cast<cudaStream_t>(stream);
  if (E <= 16) return launch_route<8, 2>(p, st);
  if (E <= 32) return launch_route<8, 4>(p, st);
  if (E <= kSmallExperts) return launch_route<8, 8>(p, st);
  if (E <= 128) return launch_route<32, 4>(p, st);
  if (E <= 256) return launch_route<32, 8>(p, st);
  return launch_route<32, 16>(p, st);
}

}  // extern "C"
