// The router of a mixture of experts: every token's k largest logits, their weights, and the order of the chosen
// (token, choice) pairs by expert in which the grouped products take them.
//
// Choice, up to 64 experts: four lanes a token, each with an ordered list of its k best (a value enters by k comparisons
// that do not wait for one another), joined by two bitonic merges.  Above: a warp a token, k rounds of a maximum over its
// lanes.  Among equals the lowest index.  Order: a stable counting sort.  Each block ranks the pairs of its own run of
// tokens among those of their expert (a warp owns a run of pairs, ranks equal experts among its lanes with match_any and
// keeps a running count per expert in shared memory); then (second launch, or after a barrier when one block is enough)
// it adds up the counts of the blocks before it and places its pairs.  Nothing depends on the order in which atomics
// arrive.  Bound by latency: 14.5 us for 32768 tokens x 64 experts, k = 4, in a captured run (with k rounds of maxima over eight
// lanes a token 5 us more, with a warp a token 20; with two lanes a token 0.7; a second launch that starts early 0.3 to 0.5 us
// less, which is not worth its own kind of dependency), 3.8 us for one token of 16 experts.
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
  int vec;                         // logits and bias can be read four at a time
  float scale;
};

constexpr float kLargest = 3.402823466e38f;

// The K best of a lane's values, best first; equal values stand in the order of their experts.
template <int K>
struct Best {
  float key[K];
  int id[K];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < K; ++j) {
      key[j] = -INFINITY;
      id[j] = -1;
    }
  }
  // experts arrive in rising order; -inf never gets in
  __device__ __forceinline__ void insert(float v, int e) {
    bool above[K];
#pragma unroll
    for (int j = 0; j < K; ++j) above[j] = v > key[j];
#pragma unroll
    for (int j = K - 1; j > 0; --j) {
      key[j] = fmaxf(fminf(v, key[j - 1]), key[j]);
      id[j] = above[j - 1] ? id[j - 1] : above[j] ? e : id[j];
    }
    key[0] = fmaxf(v, key[0]);
    id[0] = above[0] ? e : id[0];
  }
  // with the list of lane ^ o: the better of opposite ends are the K best of both, bitonic, and put in order
  __device__ __forceinline__ void merge(int o) {
    float ok[K];
    int oi[K];
#pragma unroll
    for (int j = 0; j < K; ++j) {
      ok[j] = __shfl_xor_sync(0xffffffffu, key[K - 1 - j], o);
      oi[j] = __shfl_xor_sync(0xffffffffu, id[K - 1 - j], o);
    }
#pragma unroll
    for (int j = 0; j < K; ++j)
      if (ok[j] > key[j] || (ok[j] == key[j] && oi[j] < id[j])) {
        key[j] = ok[j];
        id[j] = oi[j];
      }
#pragma unroll
    for (int s = K / 2; s > 0; s /= 2)
#pragma unroll
      for (int j = 0; j < K; ++j)
        if ((j & s) == 0 && (key[j + s] > key[j] || (key[j + s] == key[j] && id[j + s] < id[j]))) {
          const float t = key[j];
          const int i = id[j];
          key[j] = key[j + s];
          id[j] = id[j + s];
          key[j + s] = t;
          id[j + s] = i;
        }
  }
};

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

// Four experts' numbers from e on, `other` behind the last.
__device__ __forceinline__ float4 load4(const float* at, int e, int E, bool vec, float other) {
  if (vec) return e < E ? __ldg(reinterpret_cast<const float4*>(at + e)) : make_float4(other, other, other, other);
  return make_float4(e < E ? __ldg(at + e) : other, e + 1 < E ? __ldg(at + e + 1) : other,
                     e + 2 < E ? __ldg(at + e + 2) : other, e + 3 < E ? __ldg(at + e + 3) : other);
}

// L lanes a token; lane `sub` of them holds NV / 4 groups of four experts, group i being the (i * L + sub)th.
template <int L, int NV, int K>
__device__ __forceinline__ void choose_token(const RouteParams& p, int token, bool live) {
  const int sub = threadIdx.x & (L - 1);
  const float* lr = p.logits + (long long)(live ? token : 0) * p.ld;
  float4 x[NV / 4];
#pragma unroll
  for (int i = 0; i < NV / 4; ++i) x[i] = load4(lr, live ? (i * L + sub) * 4 : p.E, p.E, p.vec, -INFINITY);
  Best<K> best;
  best.clear();
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < NV / 4; ++i) {
    const int e = (i * L + sub) * 4;
    const float v[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
    float b[4] = {0.f, 0.f, 0.f, 0.f};
    if (p.bias != nullptr) {
      const float4 t = load4(p.bias, e, p.E, p.vec, 0.f);
      b[0] = t.x; b[1] = t.y; b[2] = t.z; b[3] = t.w;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float s = v[j] + b[j];
      // a logit switched off (whatever the bias says) or NaN is never chosen; +inf counts as the largest number
      best.insert(v[j] > -INFINITY && s > -INFINITY ? fminf(s, kLargest) : -INFINITY, e + j);
      top = fmaxf(top, v[j]);                            // drops NaN
    }
  }
#pragma unroll
  for (int o = 1; o < L; o *= 2) best.merge(o);
  float denom = 1.f;
  if (!p.sigmoid && !p.renorm) {                         // the sum over all experts cancels when renormalising
    top = fminf(lanes_max<L>(top), kLargest);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV / 4; ++i) {
      const float v[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (v[j] > -INFINITY) s += expf(fminf(v[j], kLargest) - top);
    }
    denom = lanes_sum<L>(s);
  }
  // lane `sub` finishes the choices sub, sub + L, ...
  constexpr int kMine = (K + L - 1) / L;
  int id[kMine];
  float xv[kMine], w[kMine], m = -INFINITY, sum = 0.f;
#pragma unroll
  for (int c = 0; c < kMine; ++c) {
    id[c] = -1;
#pragma unroll
    for (int l = 0; l < L; ++l)
      if (c * L + l < K && sub == l && c * L + l < p.k) id[c] = best.id[c * L + l];
    xv[c] = id[c] >= 0 ? fminf(__ldg(lr + id[c]), kLargest) : -INFINITY;
    m = fmaxf(m, xv[c]);
  }
  if (p.renorm) m = lanes_max<L>(m);
#pragma unroll
  for (int c = 0; c < kMine; ++c) {
    // renormalised: relative to the chosen ones' largest, so that they never all vanish; a sigmoid below e^-20 is an exponential
    if (p.sigmoid && (!p.renorm || m > -20.f)) w[c] = 1.f / (1.f + expf(-xv[c]));
    else w[c] = p.renorm ? expf(xv[c] - m) : expf(xv[c] - top) / denom;
    if (id[c] < 0) w[c] = 0.f;
    sum += w[c];
  }
  if (p.renorm) {
    sum = lanes_sum<L>(sum);
#pragma unroll
    for (int c = 0; c < kMine; ++c) w[c] = sum > 0.f ? w[c] / sum : 0.f;
  }
#pragma unroll
  for (int c = 0; c < kMine; ++c)
    if (live && c * L + sub < p.k) {
      const long long to = (long long)token * p.k + c * L + sub;
      p.ids[to] = id[c];
      p.weights[to] = w[c] * p.scale;
    }
}

// Larger float <=> larger integer; 0 stands below every key of a number that may be chosen.
__device__ __forceinline__ unsigned order_key(float v) {
  if (!(v > -INFINITY)) return 0u;                       // -inf and NaN are never chosen
  v = fminf(v, 3.402823466e38f) + 0.0f;                  // +inf counts as the largest number, -0 as +0
  const unsigned b = __float_as_uint(v);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// The weight of a choice held by one of L neighbouring lanes each (id -1: none).
template <int L>
__device__ __forceinline__ float weight_of(const RouteParams& p, int id, float x, float top, float denom) {
  float w;
  if (p.renorm) {
    // relative to the chosen ones' largest, so that they never all vanish; a sigmoid below e^-20 is an exponential
    const float m = lanes_max<L>(x);                     // lanes of no choice hold -inf
    w = p.sigmoid && m > -20.f ? 1.f / (1.f + expf(-x)) : expf(x - m);
    if (id < 0) w = 0.f;
    const float s = lanes_sum<L>(w);
    return s > 0.f ? w / s : 0.f;
  }
  if (id < 0) return 0.f;
  return p.sigmoid ? 1.f / (1.f + expf(-x)) : expf(x - top) / denom;
}

// A warp's values of a row of E numbers, lane l the i * 32 + l.
template <int NE>
__device__ __forceinline__ void load_warp(const float* at, int E, bool live, float other, float (&x)[NE]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < NE; ++i) x[i] = live && i * 32 + lane < E ? __ldg(at + i * 32 + lane) : other;
}

// Above 64 experts a warp a token, its lanes holding order-preserving integers (lane l the experts i * 32 + l): each of the k
// rounds is a maximum over the lanes, the lowest index among equals.  Lists in 4, 8 and 16 lanes a token take longer there but
// for the longest batches (k = 8, 1024 tokens of 128, 256 and 512 experts: 13, 18 and 28 us against 8.4, 11 and 16 us).
template <int NE>
__device__ __forceinline__ void choose_token_warp(const RouteParams& p, int token, const float (&bias)[NE], const float (&x)[NE]) {
  const int lane = threadIdx.x & 31;
  float v[NE];
  unsigned key[NE];
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    const bool on = x[i] > -INFINITY;                    // neither switched off (whatever the bias says) nor NaN
    v[i] = on ? fminf(x[i], kLargest) : -INFINITY;
    key[i] = on ? order_key(p.bias != nullptr ? x[i] + bias[i] : x[i]) : 0u;
  }
  float top = 0.f, denom = 1.f;
  if (!p.sigmoid && !p.renorm) {                         // the sum over all experts cancels when renormalising
    top = -INFINITY;
#pragma unroll
    for (int i = 0; i < NE; ++i) top = fmaxf(top, v[i]);
    top = lanes_max<32>(top);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NE; ++i)
      if (v[i] > -INFINITY) s += expf(v[i] - top);
    denom = lanes_sum<32>(s);
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
        at = i * 32 + lane;
      }
    const unsigned all = __reduce_max_sync(0xffffffffu, best);
    if (all == 0u) break;                                // nobody is left
    at = int(__reduce_min_sync(0xffffffffu, best == all ? unsigned(at) : 0x7fffffffu));
    float xv = -INFINITY;
#pragma unroll
    for (int i = 0; i < NE; ++i)
      if (i * 32 + lane == at) {
        xv = v[i];
        key[i] = 0u;
      }
    xv = __shfl_sync(0xffffffffu, xv, at & 31);
    if (lane == j) {
      my_id = at;
      my_x = xv;
    }
  }
  const float w = weight_of<8>(p, my_id, my_x, top, denom);      // choices sit in the first eight lanes
  if (lane < p.k) {
    const long long to = (long long)token * p.k + lane;
    p.ids[to] = my_id;
    p.weights[to] = w * p.scale;
  }
}

// Counts the block's pairs by expert, cnt[0 .. E), and ranks every pair among those of its expert in its warp's run
// (p.slots); run[warp][E] then holds the pairs of earlier warps.
__device__ __forceinline__ void rank_block(const RouteParams& p, long long lo, long long hi, long long& w0, long long& w1,
                                           int* cnt, int* run) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long part = (hi - lo + kRouteThreads - 1) / kRouteThreads * 32;      // pairs a warp, whole rounds of 32
  w0 = min(hi, lo + warp * part);
  w1 = min(hi, w0 + part);
  int* mine = run + warp * p.E;
  for (int e = lane; e < p.E; e += 32) mine[e] = 0;
  __syncthreads();                                       // also: the block's ids are written
  for (long long i0 = w0; i0 < w1; i0 += 32) {
    const long long i = i0 + lane;
    const int e = i < w1 ? p.ids[i] : -1;
    const unsigned same = __match_any_sync(0xffffffffu, e), before = same & ((1u << lane) - 1u);
    const int first = e >= 0 ? mine[e] : -1;
    __syncwarp();
    if (e >= 0 && before == 0u) mine[e] = first + __popc(same);
    __syncwarp();
    if (i < w1) p.slots[i] = e >= 0 ? first + __popc(before) : -1;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.E; e += kRouteThreads) {
    int at = 0;
#pragma unroll
    for (int w = 0; w < kRouteWarps; ++w) {
      const int c = run[w * p.E + e];
      run[w * p.E + e] = at;
      at += c;
    }
    cnt[e] = at;
  }
  __syncthreads();
}

// the places that nobody takes
__device__ __forceinline__ void clear_rows(const RouteParams& p, int total) {
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

// A single block does everything; several choose, count and rank among their own, and route_place_kernel puts them together.
template <int L, int NV, int K>
__global__ void __launch_bounds__(kRouteThreads)
route_choose_kernel(const RouteParams p) {
  extern __shared__ int sm[];
  int* cnt = sm;                                         // [E]
  int* off = cnt + p.E;                                  // [E + 1]
  int* run = off + p.E + 1;                              // [kRouteWarps][E]
  const int t0 = min(p.T, int(blockIdx.x) * p.tokens_per_block), t1 = min(p.T, t0 + p.tokens_per_block);
  const int warp = threadIdx.x >> 5;
  if constexpr (L == 32) {
    float bias[NV], x[NV], next[NV];
    load_warp<NV>(p.bias, p.E, p.bias != nullptr, 0.f, bias);
    load_warp<NV>(p.logits + (t0 + warp) * p.ld, p.E, t0 + warp < t1, -INFINITY, next);
    for (int t = t0 + warp; t < t1; t += kRouteWarps) {
#pragma unroll
      for (int i = 0; i < NV; ++i) x[i] = next[i];
      load_warp<NV>(p.logits + (t + kRouteWarps) * p.ld, p.E, t + kRouteWarps < t1, -INFINITY, next);
      choose_token_warp<NV>(p, t, bias, x);
    }
  } else {
    const int first = int(threadIdx.x) / L, warp_first = warp * (32 / L);
    for (int r = t0; r + warp_first < t1; r += kRouteThreads / L) choose_token<L, NV, K>(p, r + first, r + first < t1);
  }
  long long w0, w1;
  rank_block(p, (long long)t0 * p.k, (long long)t1 * p.k, w0, w1, cnt, run);
  const int lane = threadIdx.x & 31;
  int* mine = run + warp * p.E;
  if (gridDim.x > 1) {
    for (int e = threadIdx.x; e < p.E; e += kRouteThreads) p.counts[(long long)blockIdx.x * p.E + e] = cnt[e];
    for (long long i = w0 + lane; i < w1; i += 32) {
      const int e = p.ids[i];
      if (e >= 0) p.slots[i] += mine[e];
    }
    return;
  }
  if (warp == 0) scan_experts(cnt, off, p.E);
  __syncthreads();
  for (int e = threadIdx.x; e <= p.E; e += kRouteThreads) p.offsets[e] = off[e];
  for (long long i = w0 + lane; i < w1; i += 32) {
    const int e = p.ids[i];
    if (e >= 0) {
      const int slot = p.slots[i] + mine[e] + off[e];
      p.slots[i] = slot;
      p.rows[slot] = int(i / p.k);
    }
  }
  clear_rows(p, off[p.E]);
}

constexpr int kCountLoads = 20;                          // in flight a thread: all of 148 blocks' up to 64 experts

__global__ void __launch_bounds__(kRouteThreads)
route_place_kernel(const RouteParams p) {
  extern __shared__ int sm[];
  int* tot = sm;                                         // [E]: pairs of the expert in all blocks
  int* off = tot + p.E;                                  // [E + 1]
  int* base = off + p.E + 1;                             // [E]: pairs of the expert in earlier blocks
  const int t0 = min(p.T, int(blockIdx.x) * p.tokens_per_block), t1 = min(p.T, t0 + p.tokens_per_block);
  const long long lo = (long long)t0 * p.k, hi = (long long)t1 * p.k;
  long long i = lo + threadIdx.x;
  int e = -1, rank = 0;                                  // the thread's first pair, on its way during the sums
  if (i < hi) {
    e = p.ids[i];
    rank = p.slots[i];
  }
  for (int x = threadIdx.x; x < p.E; x += kRouteThreads) tot[x] = base[x] = 0;
  __syncthreads();
  // all counts: a thread adds up one expert over every few blocks; whole numbers, in any order
  int width = 32;
  while (width < p.E) width *= 2;                        // divides kRouteThreads (E <= 512)
  {
    const int x = int(threadIdx.x) & (width - 1), step = kRouteThreads / width;
    if (x < p.E) {
      int all = 0, before = 0;
      for (int b0 = int(threadIdx.x) / width; b0 < int(gridDim.x); b0 += kCountLoads * step) {
        int c[kCountLoads];
#pragma unroll
        for (int u = 0; u < kCountLoads; ++u) {
          const int b = b0 + u * step;
          c[u] = b < int(gridDim.x) ? p.counts[(long long)b * p.E + x] : 0;
        }
#pragma unroll
        for (int u = 0; u < kCountLoads; ++u) {
          all += c[u];
          if (b0 + u * step < int(blockIdx.x)) before += c[u];
        }
      }
      if (all != 0) atomicAdd(tot + x, all);
      if (before != 0) atomicAdd(base + x, before);
    }
  }
  __syncthreads();
  if (threadIdx.x < 32) scan_experts(tot, off, p.E);
  __syncthreads();
  if (blockIdx.x == 0)
    for (int x = threadIdx.x; x <= p.E; x += kRouteThreads) p.offsets[x] = off[x];
  while (i < hi) {
    if (e >= 0) {
      const int slot = rank + base[e] + off[e];
      p.slots[i] = slot;
      p.rows[slot] = int(i / p.k);
    }
    i += kRouteThreads;
    if (i < hi) {
      e = p.ids[i];
      rank = p.slots[i];
    }
  }
  clear_rows(p, off[p.E]);
}

constexpr int kListExperts = 64;                           // up to here lists in four lanes a token

// Blocks: one while it is the faster way (64 experts, k = 4: 128 tokens 6.5 us in one block, 7.6 us in several; 256 tokens 10.0
// and 7.5 us; 256 experts, k = 8: 16 tokens 6.8 us, 64 tokens 9.3 us in one and 8.3 us in several), then one for every 32
// tokens or every round of warps, at most one an SM (their counts are read by every block).
int route_blocks(int64_t T, int E) {
  const int64_t one = E <= kListExperts ? 128 : 16, a_block = E <= kListExperts ? 32 : 16, most = 148;
  if (T <= one) return 1;
  const int64_t want = (T + a_block - 1) / a_block;
  return int(want < most ? want : most);
}

template <int L, int NV>
int launch_route(RouteParams p, cudaStream_t st) {
  const int blocks = route_blocks(p.T, p.E);
  p.tokens_per_block = (p.T + blocks - 1) / blocks;
  const size_t smem = sizeof(int) * size_t(2 * p.E + 1 + kRouteWarps * p.E);
  auto choose = route_choose_kernel<L, NV, 8>;
  if constexpr (L < 32) {
    if (p.k <= 2) choose = route_choose_kernel<L, NV, 2>;
    else if (p.k <= 4) choose = route_choose_kernel<L, NV, 4>;
  }
  choose<<<blocks, kRouteThreads, smem, st>>>(p);
  if (int e = launch_status()) return e;
  if (blocks == 1) return SAMB_OK;
  route_place_kernel<<<blocks, kRouteThreads, sizeof(int) * size_t(3 * p.E + 1), st>>>(p);
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
  p.vec = E % 4 == 0 && ld % 4 == 0 && !((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(bias)) & 15u);
  if (E <= 16) return launch_route<4, 4>(p, st);
  if (E <= 32) return launch_route<4, 8>(p, st);
  if (E <= 64) return launch_route<4, 16>(p, st);
  if (E <= 128) return launch_route<32, 4>(p, st);
  if (E <= 256) return launch_route<32, 8>(p, st);
  return launch_route<32, 16>(p, st);
}

}  // extern "C"
