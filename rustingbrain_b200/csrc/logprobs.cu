// Token log probabilities, entropy and the most likely tokens of rows of logits, and their gradient (the ABI of
// include/logprobs_b200.h).
//
// Forward is one pass over the logits, bound by HBM: every thread keeps a running maximum m, s = sum 2^y and
// t = sum y 2^y with y = (x - m) log2(e), rescaled when the maximum moves.  The entropy is then log s - t / s: both
// terms are >= 0, so nothing cancels.  The alternatives cost no second pass: a thread keeps the maximum of each of four
// sets of its vectors and the vector that first reached it, the top_n-th best of 32 such (value, vector) pairs is a lower bound for the top_n-th best
// logit, and only the buckets that reach the bound (a twentieth of the row for 20 alternatives) are read again, by the whole CTA and out of L2.  What
// passes the bound is a few dozen values, each put in its place by counting the larger ones.
//
// One CTA takes a row.  When there are fewer rows than would fill the machine, a cluster of 2, 4 or 8 CTAs takes one and
// joins its sums and candidate lists through distributed shared memory: still one launch and no workspace.
//
// Measured in a graph: 8192 x 32000 bf16 94 us, 0.86 of the copy bandwidth (without half of the exponentials 93 us; CTAs that stay for
// several rows and load the next one early 105 us); 64 x 131071 f32 with 5 alternatives
// 13 us; one row of 32000 with 20 alternatives 9.2 us.  Gradient of 4096 x 32000 bf16 85 us, 0.95 of the copy bandwidth.

#include <cooperative_groups.h>
#include <cfloat>
#include <cstdio>
#include <cstring>

#include "../../include/logprobs_b200.h"
#include "../../include/moe_b200.h"
#include "common.cuh"
#include "warp_ops.cuh"

namespace cg = cooperative_groups;

namespace moe {
namespace {

constexpr int LP_THREADS = 128;              // 8192 x 32000 bf16 take 94 us; with 256 or 512 threads a CTA 105 and 131 (measured)
constexpr int LP_CTAS = 7;                   // CTAs an SM: 72 registers; 8 of them (64 registers, some spilled) take 96 us
constexpr int LP_WARPS = LP_THREADS / 32;
constexpr int LP_UNROLL = 4;                  // 16-byte loads in flight per thread
constexpr int LP_BUCKETS = LP_THREADS * LP_UNROLL;
constexpr int LP_CAND = 768;                  // candidates kept; more of them take the slow way
constexpr int LP_MAX_CLUSTER = 8;
constexpr float LP_LOG2E = 1.4426950408889634f;
constexpr float LP_LN2 = 0.6931471805599453f;
constexpr float LP_BIG = 1024.f;              // |m| above this: x - m is taken first, see LpSums
constexpr float LP_LOW = -1e30f;              // a logit below this has probability 0 when |m| <= LP_BIG
constexpr float LP_FLOOR = -1000.f;           // 2^-1000 is 0 in f32; keeps y finite, so that 0 * y is 0

template <typename T> struct LpVec;
template <> struct LpVec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void widen(const uint4& a, float* o) {
    o[0] = __uint_as_float(a.x); o[1] = __uint_as_float(a.y); o[2] = __uint_as_float(a.z); o[3] = __uint_as_float(a.w);
  }
  static __device__ __forceinline__ uint4 narrow(const float* o) {
    return make_uint4(__float_as_uint(o[0]), __float_as_uint(o[1]), __float_as_uint(o[2]), __float_as_uint(o[3]));
  }
};
template <> struct LpVec<bf16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void widen(const uint4& a, float* o) {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {   // a bf16 is the upper half of its f32
      o[2 * i] = __uint_as_float(w[i] << 16);
      o[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 narrow(const float* o) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 v = __floats2bfloat162_rn(o[2 * i], o[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// maximum that lets a NaN through (fmaxf drops it)
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}



// Largest value of a 16-byte vector (a NaN is passed over), and a vector with what lies below LP_LOW raised to it: its
// exponential is 0 either way, and a finite y keeps 0 * y at 0.  Both work on the packed values.
__device__ __forceinline__ uint4 vec_none(float) { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }   // -inf
__device__ __forceinline__ uint4 vec_none(bf16) { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
__device__ __forceinline__ float vec_max(const uint4& a, float) {
  return fmaxf(fmaxf(__uint_as_float(a.x), __uint_as_float(a.y)), fmaxf(__uint_as_float(a.z), __uint_as_float(a.w)));
}
__device__ __forceinline__ float vec_max(const uint4& a, bf16) {
  const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(&a);
  const __nv_bfloat162 m = __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]));
  return fmaxf(__low2float(m), __high2float(m));
}
__device__ __forceinline__ uint4 vec_raise(const uint4& a, float) {
  return make_uint4(__float_as_uint(max_nan(__uint_as_float(a.x), LP_LOW)), __float_as_uint(max_nan(__uint_as_float(a.y), LP_LOW)),
                    __float_as_uint(max_nan(__uint_as_float(a.z), LP_LOW)), __float_as_uint(max_nan(__uint_as_float(a.w), LP_LOW)));
}
__device__ __forceinline__ uint4 vec_raise(uint4 a, bf16) {
  const __nv_bfloat162 low = __float2bfloat162_rn(LP_LOW);
  __nv_bfloat162* p = reinterpret_cast<__nv_bfloat162*>(&a);
#pragma unroll
  for (int i = 0; i < 4; ++i) p[i] = __hmax2_nan(p[i], low);
  return a;
}

// Sums of a set of logits relative to its maximum m (never below -FLT_MAX, so that m itself stays finite in an empty set).
// The reference of the exponent is m2 = round(m log2 e), not m log2 e itself: the rounding shifts every y alike, and log s and
// t / s take the same shift back out, as long as it is small.  It is 2^-24 of m2, so above |m| = 1024 (where the f32 logits
// themselves are 2^-14 apart) the difference x - m is taken first, which is exact near the maximum and cannot overflow in the product.
struct LpSums {
  float m, s, t;
};
__device__ __forceinline__ float lp_shift(float from, float to) {   // y of `from` relative to `to`
  const float d = fabsf(to) > LP_BIG ? (from - to) * LP_LOG2E : __fmul_rn(from, LP_LOG2E) - __fmul_rn(to, LP_LOG2E);
  return max_nan(d, LP_FLOOR);
}
__device__ __forceinline__ float lp_y(float x, float m) {           // the y of one logit
  return fabsf(m) > LP_BIG ? (x - m) * LP_LOG2E : fmaf(x, LP_LOG2E, -__fmul_rn(m, LP_LOG2E));
}
__device__ __forceinline__ void lp_rebase(LpSums& a, float m) {
  const float d = lp_shift(a.m, m), c = ex2(d);
  a.t = c * fmaf(d, a.s, a.t);
  a.s = c * a.s;
  a.m = m;
}

// ordered bits of a logit: larger value, larger number; -0 and +0 alike, NaN below everything else but above 0 ("none")
__device__ __forceinline__ uint32_t lp_order(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  if (x != x) return 1u;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float lp_unorder(uint32_t o) {
  return o == 1u ? __uint_as_float(0x7fc00000u) : __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
// candidates compare by value, then by lower index
typedef unsigned long long lp_key;
__device__ __forceinline__ lp_key lp_make(float x, uint32_t index) { return ((lp_key)lp_order(x) << 32) | (0xffffffffu - index); }

// One warp: the n best of `count` distinct keys in shared memory, best first, written to out[0 .. n) (0 where there are
// fewer).  Every lane keeps the best of its own keys below the last one taken.
__device__ void lp_select(const lp_key* keys, int count, int n, lp_key* out) {
  const int lane = threadIdx.x & 31;
  lp_key mine = 0;
  for (int i = lane; i < count; i += 32) mine = keys[i] > mine ? keys[i] : mine;
  for (int k = 0; k < n; ++k) {
    const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(mine >> 32));
    const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(mine >> 32) == hi ? (uint32_t)mine : 0u);
    const lp_key best = ((lp_key)hi << 32) | lo;
    if (lane == 0) out[k] = best;
    if (best == 0) {
      for (int j = k + 1 + lane; j < n; j += 32) out[j] = 0;
      break;
    }
    if (mine == best) {
      mine = 0;
      for (int i = lane; i < count; i += 32)
        if (keys[i] < best && keys[i] > mine) mine = keys[i];
    }
  }
  __syncwarp();
}

// The whole CTA: the n best of `count` distinct keys (or 0), each key's place being the number of larger ones.  `keys` has room for
// one more.
__device__ void lp_rank(lp_key* keys, int count, int n, lp_key* out) {
  if (threadIdx.x == 0) keys[count] = 0;
  if (threadIdx.x < n) out[threadIdx.x] = 0;
  __syncthreads();
  const ulonglong2* two = reinterpret_cast<const ulonglong2*>(keys);
  for (int at = threadIdx.x; at < count; at += LP_THREADS) {
    const lp_key mine = keys[at];
    int place = 0;
    for (int i = 0; i < (count + 1) / 2; ++i) {
      const ulonglong2 k = two[i];
      place += (k.x > mine) + (k.y > mine);
    }
    if (place < n && mine != 0) out[place] = mine;
  }
  __syncthreads();
}

// One warp: a bound that at least n buckets reach, and the list of those that do.  Lane l takes the best of the buckets l, l + 32, ...;
// the n-th best of these 32 is the bound (of 512 buckets, about 30 reach it for n = 20 and 5 for n = 5).  0: fewer than n lanes have a
// vector at all, and every value is a candidate.
__device__ lp_key lp_bound(const lp_key* bucket, int n, lp_key* best_of_lane, int* hot, int* hot_count) {
  const int lane = threadIdx.x & 31;
  lp_key mine = 0;
#pragma unroll
  for (int i = 0; i < LP_BUCKETS / 32; ++i) {
    const lp_key k = bucket[i * 32 + lane];
    mine = k > mine ? k : mine;
  }
  best_of_lane[lane] = mine;
  __syncwarp();
  const ulonglong2* two = reinterpret_cast<const ulonglong2*>(best_of_lane);
  int place = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const ulonglong2 k = two[i];
    place += (k.x > mine) + (k.y > mine);
  }
  const unsigned at = __ballot_sync(0xffffffffu, mine != 0 && place == n - 1);
  const lp_key bound = at ? __shfl_sync(0xffffffffu, mine, __ffs(at) - 1) : 0;
  int count = 0;
#pragma unroll
  for (int i = 0; i < LP_BUCKETS / 32; ++i) {
    const lp_key k = bucket[i * 32 + lane];
    const bool is_hot = k != 0 && k >= bound;
    const unsigned all = __ballot_sync(0xffffffffu, is_hot);
    if (is_hot) hot[count + __popc(all & ((1u << lane) - 1))] = i * 32 + lane;
    count += __popc(all);
  }
  if (lane == 0) *hot_count = count;
  return bound;
}

struct LpShared {
  LpSums warp[LP_WARPS];
  LpSums cta;                        // this CTA's sums, read by the cluster
  lp_key bucket[LP_BUCKETS];         // best value, first vector that holds it
  alignas(16) lp_key cand[LP_CAND];
  lp_key best[LOGPROBS_MAX_TOP];     // this CTA's list, read by the cluster
  alignas(16) lp_key joined[LP_MAX_CLUSTER * LOGPROBS_MAX_TOP + 2];
  alignas(16) lp_key lane_best[32];
  int hot[LP_BUCKETS];               // buckets whose vectors are read again
  lp_key bound, last;
  int count, hot_count;
};

template <typename T>
__global__ void __launch_bounds__(LP_THREADS, LP_CTAS)
logprobs_kernel(const T* __restrict__ x, long long stride, const int* __restrict__ targets, int vocab, int top_n, int cluster,
                float* __restrict__ logprob, float* __restrict__ entropy, float* __restrict__ lse_out, float* __restrict__ top_lp,
                int* __restrict__ top_ids) {
  constexpr int N = LpVec<T>::N;
  __shared__ LpShared sh;
  const int row = blockIdx.x / cluster, rank = blockIdx.x - row * cluster;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const T* xr = x + (long long)row * stride;
  // [0, head) and [tail, vocab) lie outside the 16-byte vectors of the row
  const int mis = (int)((reinterpret_cast<uintptr_t>(xr) & 15) / sizeof(T));
  const int head = min(vocab, mis ? N - mis : 0);
  const int vecs = (vocab - head) / N, tail = head + vecs * N, loose = head + (vocab - tail);
  const uint4* xv = reinterpret_cast<const uint4*>(xr + head);
  const int step = cluster * LP_THREADS, v0 = rank * LP_THREADS + tid;
  if (tid == 0) sh.count = 0;

  // A thread's vectors fall into LP_UNROLL buckets by their place in a round: the largest logit of each, and the first vector with it.
  float best[LP_UNROLL];
  int best_vec[LP_UNROLL];
#pragma unroll
  for (int u = 0; u < LP_UNROLL; ++u) { best[u] = -INFINITY; best_vec[u] = v0 + u * step; }
  float m = -FLT_MAX, m2 = 0.f;      // the maximum that the sums refer to, and round(m log2 e) of one within LP_BIG
  uint64_t s2 = 0, t2 = 0;           // s and t, each as two halves
  auto sums = [&] {
    float s0, s1, t0, t1;
    unpack2(s2, s0, s1);
    unpack2(t2, t0, t1);
    return LpSums{m, s0 + s1, t0 + t1};
  };
  auto load = [&](uint4* raw, int v) {
#pragma unroll
    for (int u = 0; u < LP_UNROLL; ++u) {
      raw[u] = vec_none(T());
      if (v + u * step < vecs) raw[u] = __ldg(xv + v + u * step);
    }
  };
  auto take = [&](const uint4* raw, int v) {
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < LP_UNROLL; ++u) {
      const float mx = vec_max(raw[u], T());
      if (mx > best[u]) { best[u] = mx; best_vec[u] = v + u * step; }
      top = fmaxf(top, mx);
    }
    if (top > m) {
      LpSums a = sums();
      lp_rebase(a, top);
      m = top;
      m2 = __fmul_rn(m, LP_LOG2E);
      s2 = pack2(a.s, 0.f);
      t2 = pack2(a.t, 0.f);
    }
    if (fabsf(m) <= LP_BIG) {
      // two logits an instruction but for the exponential, of which an SM does 16 a cycle
      const uint64_t mm = pack2(-m2, -m2), ll = pack2(LP_LOG2E, LP_LOG2E);
#pragma unroll
      for (int u = 0; u < LP_UNROLL; ++u) {
        float f[N];
        LpVec<T>::widen(vec_raise(raw[u], T()), f);
#pragma unroll
        for (int i = 0; i < N; i += 2) {
          const uint64_t y = fma2(pack2(f[i], f[i + 1]), ll, mm);
          float y0, y1;
          unpack2(y, y0, y1);
          const uint64_t e = pack2(ex2(y0), ex2(y1));
          s2 = add2(s2, e);
          t2 = fma2(y, e, t2);
        }
      }
    } else {
      LpSums a = sums();
#pragma unroll
      for (int u = 0; u < LP_UNROLL; ++u) {
        float f[N];
        LpVec<T>::widen(raw[u], f);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float y = max_nan((f[i] - m) * LP_LOG2E, LP_FLOOR), e = ex2(y);
          a.s += e;
          a.t = fmaf(y, e, a.t);
        }
      }
      s2 = pack2(a.s, 0.f);
      t2 = pack2(a.t, 0.f);
    }
  };
  // the next round's loads are in flight while a round is summed
  uint4 even[LP_UNROLL], odd[LP_UNROLL];
  constexpr int R = LP_UNROLL;
  load(even, v0);
  for (int v = v0; v < vecs; v += 2 * R * step) {
    load(odd, v + R * step);
    take(even, v);
    load(even, v + 2 * R * step);
    if (v + R * step < vecs) take(odd, v + R * step);
  }
  LpSums a = sums();
  if (rank == 0 && tid < loose) {    // the loose ends, one per thread
    const float f = to_f32<T>(xr[tid < head ? tid : tail + tid - head]);
    if (f > a.m) lp_rebase(a, f);
    const float y = max_nan(lp_y(f, a.m), LP_FLOOR), e = ex2(y);
    a.s += e;
    a.t = fmaf(y, e, a.t);
  }

  // ---- join the threads ----
  m = a.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  lp_rebase(a, m);
  a.s = warp_sum(a.s);
  a.t = warp_sum(a.t);
  if (lane == 0) sh.warp[warp] = a;
  if (top_n > 0) {
#pragma unroll
    for (int u = 0; u < LP_UNROLL; ++u)
      sh.bucket[u * LP_THREADS + tid] = v0 + u * step < vecs ? ((lp_key)lp_order(best[u]) << 32) | (0xffffffffu - (uint32_t)best_vec[u]) : 0;
  }
  __syncthreads();
  if (tid == 0) {
    float mm = sh.warp[0].m;
    for (int w = 1; w < LP_WARPS; ++w) mm = fmaxf(mm, sh.warp[w].m);
    LpSums c{mm, 0.f, 0.f};
    for (int w = 0; w < LP_WARPS; ++w) {
      LpSums b = sh.warp[w];
      lp_rebase(b, mm);
      c.s += b.s;
      c.t += b.t;
    }
    sh.cta = c;
  }

  // ---- this CTA's best top_n ----
  if (top_n > 0) {
    if (warp == 1) {
      const lp_key b = lp_bound(sh.bucket, top_n, sh.lane_best, sh.hot, &sh.hot_count);
      if (lane == 0) sh.bound = b;
    }
    __syncthreads();
    const lp_key bound = sh.bound;                  // 0: everything is a candidate
    const uint32_t bound_value = (uint32_t)(bound >> 32), bound_vec = 0xffffffffu - (uint32_t)bound;
    auto offer = [&](float f, uint32_t index) {
      const int at = atomicAdd(&sh.count, 1);
      if (at < LP_CAND) sh.cand[at] = lp_make(f, index);
    };
    if (rank == 0 && tid < loose) {
      const int i = tid < head ? tid : tail + tid - head;
      offer(to_f32<T>(xr[i]), i);
    }
    const int each = (vecs + LP_UNROLL * step - 1) / (LP_UNROLL * step), again = sh.hot_count * each;
#pragma unroll 2
    for (int i = tid; i < again; i += LP_THREADS) {
      const int h = i / each, bucket = sh.hot[h], u = bucket / LP_THREADS;
      const int w = rank * LP_THREADS + (bucket - u * LP_THREADS) + ((i - h * each) * LP_UNROLL + u) * step;
      if (w >= vecs) continue;
      float f[N];
      LpVec<T>::widen(__ldg(xv + w), f);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const uint32_t o = lp_order(f[k]);
        if (o > bound_value || (o == bound_value && (uint32_t)w <= bound_vec)) offer(f[k], head + (uint32_t)w * N + k);
      }
    }
    __syncthreads();
    if (sh.count <= 2 * LP_THREADS) {
      lp_rank(sh.cand, sh.count, top_n, sh.best);
    } else if (sh.count <= LP_CAND) {
      if (warp == 0) lp_select(sh.cand, sh.count, top_n, sh.best);
    } else {
      // Thousands of logits above the bound: the best ones sit in a few threads' vectors.  Take the row top_n times, each time the best
      // below the last one.
      if (tid == 0) sh.last = ~0ull;
      __syncthreads();
      for (int k = 0; k < top_n; ++k) {
        const lp_key last = sh.last;
        lp_key mx = 0;
        auto look = [&](float f, uint32_t index) {
          const lp_key key = lp_make(f, index);
          if (key < last && key > mx) mx = key;
        };
        for (int w = v0; w < vecs; w += step) {
          float f[N];
          LpVec<T>::widen(__ldg(xv + w), f);
#pragma unroll
          for (int i = 0; i < N; ++i) look(f[i], head + (uint32_t)w * N + i);
        }
        if (rank == 0 && tid < loose) {
          const int i = tid < head ? tid : tail + tid - head;
          look(to_f32<T>(xr[i]), i);
        }
        sh.bucket[tid] = mx;
        __syncthreads();
        if (warp == 0) {
          lp_select(sh.bucket, LP_THREADS, 1, sh.best + k);
          if (lane == 0) sh.last = sh.best[k];
        }
        __syncthreads();
      }
    }
  }

  // ---- join the cluster, write the row ----
  LpSums total{};
  const lp_key* list = sh.best;
  if (cluster > 1) {
    cg::cluster_group cl = cg::this_cluster();
    cl.sync();
    if (rank == 0) {
      if (tid == 0) {
        float mm = -FLT_MAX;
        for (int r = 0; r < cluster; ++r) mm = fmaxf(mm, cl.map_shared_rank(&sh.cta, r)->m);
        total.m = mm;
        for (int r = 0; r < cluster; ++r) {
          LpSums b = *cl.map_shared_rank(&sh.cta, r);
          lp_rebase(b, mm);
          total.s += b.s;
          total.t += b.t;
        }
      }
      for (int i = tid; i < cluster * top_n; i += LP_THREADS) {
        const int r = i / top_n;
        sh.joined[i] = cl.map_shared_rank(sh.best, r)[i - r * top_n];
      }
    }
    cl.sync();                                      // the others' shared memory has been read; they may leave
    if (rank != 0) return;
    if (tid == 0) sh.cta = total;
    if (top_n > 0) {
      lp_rank(sh.joined, cluster * top_n, top_n, sh.bucket);
      list = sh.bucket;
    }
  }
  __syncthreads();
  total = sh.cta;
  // y - log2 s keeps the small numbers small.  What is left of a near-certain token is off by 2^-23 or so: s has the token's own 2^y beside
  // the rest, and neither that nor its logarithm is exact.  So it can come out above 0, where no log probability is.
  const float l2 = log2f(total.s);
  const bool empty = total.s == 0.f;                // nothing but -inf
  auto log_p = [&](float f) {
    if (empty) return f != f ? f : -INFINITY;
    const float v = fabsf(f) > LP_BIG || fabsf(total.m) > LP_BIG ? (f - total.m) - l2 * LP_LN2   // the lowest finite value stays finite
                                                                 : (lp_y(f, total.m) - l2) * LP_LN2;
    return v > 0.f ? 0.f : v;
  };
  if (tid == 0) {
    const float lse = empty ? -INFINITY : fabsf(total.m) > LP_BIG ? fmaf(l2, LP_LN2, total.m) : (__fmul_rn(total.m, LP_LOG2E) + l2) * LP_LN2;
    if (lse_out) lse_out[row] = lse;
    if (entropy) entropy[row] = empty ? 0.f : max_nan((l2 - total.t / total.s) * LP_LN2, 0.f);
    if (logprob) {
      const int t = targets ? targets[row] : -1;
      logprob[row] = t < 0 ? 0.f : t >= vocab ? __uint_as_float(0x7fc00000u) : log_p(to_f32<T>(xr[t]));
    }
  }
  if (tid < top_n) {
    const lp_key key = list[tid];
    top_ids[(long long)row * top_n + tid] = key ? (int)(0xffffffffu - (uint32_t)key) : -1;
    top_lp[(long long)row * top_n + tid] = key ? log_p(lp_unorder((uint32_t)(key >> 32))) : __uint_as_float(0x7fc00000u);
  }
}

// Gradient: one read and one write of the logits' size, everything else is per row.  A CTA takes a run of one row; the 16-byte path needs
// the logits' and the gradient's row equally far from a 16-byte boundary, the element path takes what is left.
template <typename T>
__global__ void __launch_bounds__(LP_THREADS)
logprobs_backward_kernel(const T* x, long long stride, const int* __restrict__ targets, const float* __restrict__ lse,
                         const float* __restrict__ entropy, const float* __restrict__ grad_lp, const float* __restrict__ grad_h, int vocab,
                         int runs, T* grad, long long grad_stride) {
  constexpr int N = LpVec<T>::N, RUN = LP_THREADS * LP_UNROLL;    // vectors per CTA
  const int row = blockIdx.x / runs, run = blockIdx.x - row * runs;
  const T* xr = x + (long long)row * stride;
  T* gr = grad + (long long)row * grad_stride;
  const int target = targets ? targets[row] : -1;
  const float z = lse[row], h = grad_h ? entropy[row] : 0.f, gh = grad_h ? grad_h[row] : 0.f;
  float gl = grad_lp && target >= 0 ? grad_lp[row] : 0.f;
  if (target >= vocab) gl = __uint_as_float(0x7fc00000u);
  const bool empty = z == -INFINITY;
  // d is -inf at a masked logit, where p is 0; the target's own gl comes on top
  const float c = -fmaf(gh, h, gl);
  auto one = [&](float f, int index) {
    const float d = f - z, p = ex2(d * LP_LOG2E);
    const float g = fmaf(p, fmaf(-gh, max_nan(d, LP_FLOOR), c), index == target ? gl : 0.f);
    return empty ? (f == f ? 0.f * gl : f) : g;
  };
  const int mis = (int)((reinterpret_cast<uintptr_t>(xr) & 15) / sizeof(T));
  const bool wide = ((reinterpret_cast<uintptr_t>(xr) ^ reinterpret_cast<uintptr_t>(gr)) & 15) == 0;
  if (!wide) {
    // unsigned: the last step passes a vocabulary of 2^31 - 1
    const unsigned end = (unsigned)min((long long)vocab, (long long)(run + 1) * RUN * N);
    for (unsigned i = (unsigned)run * RUN * N + threadIdx.x; i < end; i += LP_THREADS) gr[i] = from_f32<T>(one(to_f32<T>(xr[i]), (int)i));
    return;
  }
  const int head = min(vocab, mis ? N - mis : 0), vecs = (vocab - head) / N, tail = head + vecs * N;
  if (run == 0 && (int)threadIdx.x < head + (vocab - tail)) {
    const int i = (int)threadIdx.x < head ? threadIdx.x : tail + threadIdx.x - head;
    gr[i] = from_f32<T>(one(to_f32<T>(xr[i]), i));
  }
  const uint4* xv = reinterpret_cast<const uint4*>(xr + head);
  uint4* gv = reinterpret_cast<uint4*>(gr + head);
  uint4 raw[LP_UNROLL];
#pragma unroll
  for (int u = 0; u < LP_UNROLL; ++u) {
    const int v = run * RUN + u * LP_THREADS + threadIdx.x;
    if (v < vecs) raw[u] = xv[v];
  }
#pragma unroll
  for (int u = 0; u < LP_UNROLL; ++u) {
    const int v = run * RUN + u * LP_THREADS + threadIdx.x;
    if (v >= vecs) continue;
    const int base = head + v * N;
    float f[N];
    LpVec<T>::widen(raw[u], f);
    if (empty || (unsigned)(target - base) < (unsigned)N) {
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = one(f[i], base + i);
    } else {
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        const uint64_t d = add2(pack2(f[i], f[i + 1]), pack2(-z, -z));
        float d0, d1, y0, y1;
        unpack2(d, d0, d1);
        unpack2(mul2(d, pack2(LP_LOG2E, LP_LOG2E)), y0, y1);
        const uint64_t w = fma2(pack2(max_nan(d0, LP_FLOOR), max_nan(d1, LP_FLOOR)), pack2(-gh, -gh), pack2(c, c));
        unpack2(mul2(pack2(ex2(y0), ex2(y1)), w), f[i], f[i + 1]);
      }
    }
    gv[v] = LpVec<T>::narrow(f);
  }
}

int lp_fail(char* msg, int len, int code, const char* text) {
  if (msg && len > 0) snprintf(msg, len, "%s", text);
  return code;
}

template <typename T>
cudaError_t launch_forward(const void* x, long long stride, const int* targets, int rows, int vocab, int top_n, float* logprob, float* entropy,
                           float* lse, float* top_lp, int* top_ids, cudaStream_t st) {
  // A row's CTAs: as many as fill the machine, but with two vectors for each thread.
  int cluster = 1;
  const long long vecs = vocab / LpVec<T>::N;
  while (cluster < LP_MAX_CLUSTER && (long long)rows * cluster * 2 <= LP_CTAS * 148 && vecs >= (long long)cluster * 2 * LP_THREADS) cluster *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(rows * cluster));
  cfg.blockDim = dim3(LP_THREADS);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  count_launch();
  return cudaLaunchKernelEx(&cfg, logprobs_kernel<T>, (const T*)x, stride, targets, vocab, top_n, cluster, logprob, entropy, lse, top_lp, top_ids);
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

int32_t logprobs_forward(const void* x, int64_t row_stride, const int32_t* targets, int32_t rows, int32_t vocab, int32_t top_n,
                         int32_t precision, float* logprob, float* entropy, float* lse, float* top_logprob, int32_t* top_ids,
                         void* stream, char* message, int32_t message_len) {
  if (precision != MOE_PRECISION_F32 && precision != MOE_PRECISION_BF16)
    return lp_fail(message, message_len, MOE_INVALID_CONFIG, "InvalidConfig: logits are f32 or bf16");
  if (rows < 0 || vocab <= 0 || row_stride < vocab)
    return lp_fail(message, message_len, MOE_INVALID_INPUT, "InvalidInput: rows >= 0, vocab > 0 and row_stride >= vocab");
  if (top_n < 0 || top_n > LOGPROBS_MAX_TOP || top_n > vocab)
    return lp_fail(message, message_len, MOE_INVALID_INPUT, "InvalidInput: top_n is 0 .. min(vocab, 32)");
  if (rows == 0) return MOE_OK;
  if (!x || (top_n > 0 && (!top_logprob || !top_ids))) return lp_fail(message, message_len, MOE_INVALID_INPUT, "InvalidInput: null buffer");
  const size_t elem = precision == MOE_PRECISION_BF16 ? 2 : 4;
  if (reinterpret_cast<uintptr_t>(x) % elem) return lp_fail(message, message_len, MOE_INVALID_INPUT, "InvalidInput: logits are not aligned to their type");
  const cudaError_t e = precision == MOE_PRECISION_BF16
      ? launch_forward<bf16>(x, row_stride, targets, rows, vocab, top_n, logprob, entropy, lse, top_logprob, top_ids, (cudaStream_t)stream)
      : launch_forward<float>(x, row_stride, targets, rows, vocab, top_n, logprob, entropy, lse, top_logprob, top_ids, (cudaStream_t)stream);
  return e == cudaSuccess ? MOE_OK : lp_fail(message, message_len, MOE_CUDA_ERROR, cudaGetErrorString(e));
}

int32_t logprobs_backward(const void* x, int64_t row_stride, const int32_t* targets, const float* lse, const float* entropy,
                          const float* grad_logprob, const float* grad_entropy, int32_t rows, int32_t vocab, int32_t precision,
                          void* grad_x, int64_t grad_stride, void* stream, char* message, int32_t message_len) {
  if (precision != MOE_PRECISION_F32 && precision != MOE_PRECISION_BF16)
    return lp_fail(message, message_len, MOE_INVALID_CONFIG, "InvalidConfig: logits are f32 or bf16");
  if (rows < 0 || vocab <= 0 || row_stride < vocab || grad_stride < vocab)
    return lp_fail(message, message_len, MOE_INVALID_INPUT, "InvalidInput: rows >= 0, vocab > 0 and strides >= vocab");
  if (rows == 0) return MOE_OK;
  if (!x || !grad_x || !lse || (grad_entropy && !entropy)) return lp_fail(message, message_len, MOE_INVALID_INPUT, "InvalidInput: null buffer");
  if (x == grad_x && row_stride != grad_stride)
    return lp_fail(message, message_len, MOE_INVALID_INPUT, "InvalidInput: a gradient in place has the logits' row stride");
  const size_t elem = precision == MOE_PRECISION_BF16 ? 2 : 4;
  if (reinterpret_cast<uintptr_t>(x) % elem || reinterpret_cast<uintptr_t>(grad_x) % elem)
    return lp_fail(message, message_len, MOE_INVALID_INPUT, "InvalidInput: buffers are not aligned to their type");
  if (x != grad_x && rows_overlap(x, (long long)row_stride * elem, grad_x, (long long)grad_stride * elem, (long long)vocab * elem, (long long)vocab * elem, rows))
    return lp_fail(message, message_len, MOE_INVALID_INPUT, "InvalidInput: the gradient overlaps the logits and is not in their place");
  const long long per_run = (long long)LP_THREADS * LP_UNROLL * (16 / elem);
  const long long runs = (vocab + per_run - 1) / per_run;
  if (runs * rows > 0x7fffffffll) return lp_fail(message, message_len, MOE_INVALID_INPUT, "InvalidInput: too many rows");
  const unsigned grid = (unsigned)(runs * rows);
  const cudaStream_t st = (cudaStream_t)stream;
  if (precision == MOE_PRECISION_BF16)
    logprobs_backward_kernel<bf16><<<grid, LP_THREADS, 0, st>>>((const bf16*)x, row_stride, targets, lse, entropy, grad_logprob, grad_entropy,
                                                                vocab, (int)runs, (bf16*)grad_x, grad_stride);
  else
    logprobs_backward_kernel<float><<<grid, LP_THREADS, 0, st>>>((const float*)x, row_stride, targets, lse, entropy, grad_logprob, grad_entropy,
                                                                 vocab, (int)runs, (float*)grad_x, grad_stride);
  count_launch();
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? MOE_OK : lp_fail(message, message_len, MOE_CUDA_ERROR, cudaGetErrorString(e));
}

}  // extern "C"
