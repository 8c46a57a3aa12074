// KV cache held in 4 bits: append and decode attention (precision MOE_PRECISION_Q4 of include/kv_attention_b200.h).
//
// A decode step reads the whole cache once, so the bytes per position are the time: 4 bits a channel, and for each 32 channels of a
// head's key or value a bf16 step and base, value = code * step + base: 1.25 bytes a channel for key and value together, where a bf16
// cache takes 4.
//
// The 64 positions of a page lie together, as the tensor cores want them: one warp takes a page, S^T = K Q^T has the positions as
// the 16 rows and the queries as the 8 columns of mma.sync m16n8k16, O^T = V^T P^T has the channels as rows and the positions as the
// reduction.  So the few queries that share a kv head fill the small side of the product, and both K and V are the A operand:
// a lane's 32-bit word holds 8 codes that it needs itself, keys as 8 channels of one position, values as 8 positions of one channel,
// so that a word costs seven instructions to become four pairs of bf16 numbers 128 + code.
//   keys:   the sum over 32 channels starts at -128 sum(q) and then takes step and base in f32: S += step * sum + base * sum(q).
//           Nothing of the key is rounded.
//   values: step and base belong to the position, which is what the product sums over, so they go on before it: two packed
//           bf16 instructions, one rounding of the value to bf16 (2^-9 of it; P is rounded alike).
//
// Page layout, HD = head_dim, NG = HD / 32:
//   keys    [64 positions][4 t][NG g] words: channels 32 g + 8 t + 2 i + e at nibble i + 4 e
//   values  [HD channels][4 t][2 w] words: positions 16 (2 w + i / 2) + 8 (i % 2) + 2 t + e at nibble i + 4 e
//   key step | base      [64 positions][NG] (two bf16)
//   value step, value base  [NG][64] bf16 each, position p at value_slot(p)

#include <cooperative_groups.h>
#include <algorithm>
#include <atomic>
#include <cfloat>

#include "kv_q4.cuh"

namespace cg = cooperative_groups;

namespace moe {
namespace q4 {
namespace {

constexpr int WARPS = 4, THREADS = WARPS * 32;
constexpr float HUGE_VALUE = 8.507059e37f;      // 2^126: a larger number counts as an infinity, so that high - low stays finite

template <int HD> struct Layout {
  static constexpr int NG = HD / GROUP, KEYS = 0, VALUES = 32 * HD, KPAR = 64 * HD, VSTEP = 72 * HD, VBASE = VSTEP + NG * 128, BYTES = 80 * HD;
};
__host__ __device__ inline int value_word(int p) { return ((p & 7) >> 1) * 2 + (p >> 5); }
__host__ __device__ inline int value_nibble(int p) { return ((p >> 4) & 1) * 2 + ((p >> 3) & 1) + 4 * (p & 1); }
__host__ __device__ inline int value_slot(int p) { return ((p & 7) >> 1) * 16 + (p >> 4) * 4 + ((p >> 3) & 1) * 2 + (p & 1); }

__device__ __forceinline__ unsigned char* page_at(const Cache& c, int seq, int kvh, int page) {
  const long long pages = (c.cap + PAGE - 1) / PAGE;
  return c.pages + (((long long)seq * c.Hkv + kvh) * pages + page) * (80ll * c.HD);
}

// ---- quantise ----
// Lane l holds channels 32 g + l.  Codes, and step and base as bf16 bits.
template <int NG>
__device__ __forceinline__ void quantise(const float* x, uint32_t* code, uint32_t* step, uint32_t* base) {
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    float lo = x[g], hi = x[g];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    const bf16 s = __float2bfloat16_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.f)), b = __float2bfloat16_rn(lo);
    const float sf = __bfloat162float(s), bf = __bfloat162float(b);
    code[g] = sf > 0.f ? (uint32_t)fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x[g], bf), sf)), 0.f), 15.f) : 0u;
    step[g] = __bfloat16_as_ushort(s);
    base[g] = __bfloat16_as_ushort(b);
  }
}

// The CTA stores `count` new positions, first_slot .. of one page.  k and v point to the first new row of this head, `stride` elements apart;
// pos0 is the first one's position in the sequence.  `codes` is [64][HD] bytes of shared memory.
template <int HD>
__device__ void append_page(const Cache& c, unsigned char* page, const bf16* k, const bf16* v, long long stride, int first_slot, int count,
                            int pos0, unsigned char* codes) {
  using L = Layout<HD>;
  constexpr int NG = L::NG;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int r = warp; r < count; r += WARPS) {
    const int slot = first_slot + r, pos = pos0 + r;
    float x[NG], y[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      x[g] = __bfloat162float(k[r * stride + 32 * g + lane]);
      y[g] = __bfloat162float(v[r * stride + 32 * g + lane]);
    }
    if (c.rope) {
      // the same steps as in 32-bit arithmetic without contraction, so that the codes can be reproduced
      const float* ct = c.cos_t + (long long)pos * (HD / 2);
      const float* st = c.sin_t + (long long)pos * (HD / 2);
      if constexpr (NG == 1) {
        const float other = __shfl_xor_sync(0xffffffffu, x[0], 16), co = ct[lane & 15], si = st[lane & 15];
        x[0] = lane < 16 ? __fsub_rn(__fmul_rn(x[0], co), __fmul_rn(other, si)) : __fadd_rn(__fmul_rn(x[0], co), __fmul_rn(other, si));
      } else {
#pragma unroll
        for (int g = 0; g < NG / 2; ++g) {
          const float co = ct[32 * g + lane], si = st[32 * g + lane], lo = x[g], hi = x[g + NG / 2];
          x[g] = __fsub_rn(__fmul_rn(lo, co), __fmul_rn(hi, si));
          x[g + NG / 2] = __fadd_rn(__fmul_rn(hi, co), __fmul_rn(lo, si));
        }
      }
    }
    // A position that holds a NaN or an infinity anywhere gets NaN keys and values of 0: whoever sees it gets NaN, and a query that
    // does not see it multiplies its value by a weight of 0 without harm.
    bool bad = false;
#pragma unroll
    for (int g = 0; g < NG; ++g) bad |= !(fabsf(x[g]) <= HUGE_VALUE) || !(fabsf(y[g]) <= HUGE_VALUE);
    bad = __any_sync(0xffffffffu, bad);
    if (bad) {
#pragma unroll
      for (int g = 0; g < NG; ++g) x[g] = y[g] = 0.f;
    }
    uint32_t code[NG], step[NG], base[NG];
    quantise<NG>(x, code, step, base);
    uint32_t* kw = reinterpret_cast<uint32_t*>(page + L::KEYS) + slot * (HD / 8);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      uint32_t w = code[g] << (4 * (((lane & 7) >> 1) + 4 * (lane & 1)));
      w |= __shfl_xor_sync(0xffffffffu, w, 1);
      w |= __shfl_xor_sync(0xffffffffu, w, 2);
      w |= __shfl_xor_sync(0xffffffffu, w, 4);
      if ((lane & 7) == 0) kw[(lane >> 3) * NG + g] = w;
      if (lane == 0) reinterpret_cast<uint32_t*>(page + L::KPAR)[slot * NG + g] = (bad ? 0x7fc0u : step[g]) | base[g] << 16;
    }
    quantise<NG>(y, code, step, base);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      codes[r * HD + 32 * g + lane] = (unsigned char)code[g];
      if (lane == 0) {
        reinterpret_cast<uint16_t*>(page + L::VSTEP)[g * 64 + value_slot(slot)] = (uint16_t)step[g];
        reinterpret_cast<uint16_t*>(page + L::VBASE)[g * 64 + value_slot(slot)] = (uint16_t)base[g];
      }
    }
  }
  __syncthreads();
  // a value word holds eight positions: this CTA is the only one that writes to the page, old positions keep their codes
  uint32_t* vw = reinterpret_cast<uint32_t*>(page + L::VALUES);
  for (int i = threadIdx.x; i < HD * 8; i += THREADS) {
    const int ch = i >> 3, t = (i & 7) >> 1, w = i & 1;
    uint32_t set = 0, val = 0;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const int p = 16 * (2 * w + ((n & 3) >> 1)) + 8 * (n & 1) + 2 * t + (n >> 2), r = p - first_slot;
      if (r >= 0 && r < count) {
        set |= 15u << (4 * n);
        val |= (uint32_t)codes[r * HD + ch] << (4 * n);
      }
    }
    if (set) vw[i] = set == 0xffffffffu ? val : (vw[i] & ~set) | val;
  }
}

template <int HD>
__global__ void __launch_bounds__(THREADS) append_kernel(Cache c, const bf16* __restrict__ k, const bf16* __restrict__ v, int first, int rows) {
  __shared__ unsigned char codes[PAGE * HD];
  const int touched = (rows + PAGE - 2) / PAGE + 1;   // pages that rows new positions can lie in
  const int kvh = blockIdx.x / touched % c.Hkv, sj = blockIdx.x / touched / c.Hkv, seq = first + sj, len = c.lengths[seq];
  if (len + rows > c.cap) return;                     // reported by the launch that follows
  const int page = len / PAGE + blockIdx.x % touched, p0 = max(len, page * PAGE), p1 = min(len + rows, (page + 1) * PAGE);
  if (p0 >= p1) return;
  const long long W = (long long)c.Hkv * HD, at = ((long long)sj * rows + p0 - len) * W + kvh * HD;
  append_page<HD>(c, page_at(c, seq, kvh, page), k + at, v + at, W, p0 - page * PAGE, p1 - p0, p0, codes);
}

// ---- attention ----
__device__ __forceinline__ void mma16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ void copy16(uint32_t smem, const void* gmem) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem), "l"(gmem) : "memory");
}
__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// codes i and i + 4 of a word as the bf16 pair (128 + code, 128 + code)
template <int I>
__device__ __forceinline__ uint32_t pair128(uint32_t w) { return ((w >> (4 * I)) & 0x000f000fu) | 0x43004300u; }
__device__ __forceinline__ __nv_bfloat162 as_pair(uint32_t v) { return *reinterpret_cast<const __nv_bfloat162*>(&v); }
__device__ __forceinline__ uint32_t as_bits(__nv_bfloat162 v) { return *reinterpret_cast<const uint32_t*>(&v); }
template <int I>
__device__ __forceinline__ uint32_t value_pair(uint32_t w, uint32_t step, uint32_t base) {
  return as_bits(__hfma2(__hsub2(as_pair(pair128<I>(w)), __float2bfloat162_rn(128.f)), as_pair(step), as_pair(base)));
}

template <int N> struct Words { uint32_t w[N]; };
template <int N>
__device__ __forceinline__ Words<N> load_words(const unsigned char* p) {
  Words<N> r;
  if constexpr (N == 1) {
    r.w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    r.w[0] = v.x; r.w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(p + 4 * i);
      r.w[i] = v.x; r.w[i + 1] = v.y; r.w[i + 2] = v.z; r.w[i + 3] = v.w;
    }
  }
  return r;
}

template <int HD> struct Ring { static constexpr int STAGES = HD == 32 ? 6 : HD == 64 ? 4 : 2; };

template <int HD, int NQ>
constexpr int smem_bytes() {
  const int ring = WARPS * Ring<HD>::STAGES * Layout<HD>::BYTES, merge = NQ * 8 * (WARPS + 1) * (HD + 2) * 4, codes = PAGE * HD;
  return ring > merge ? (ring > codes ? ring : codes) : (merge > codes ? merge : codes);
}

// grid: ((sequence * kv heads + kv head) * passes + pass) * splits + split; the splits of one are a cluster when it joins them
template <int HD, int NQ>
__global__ void __launch_bounds__(THREADS)
attention_kernel(Cache c, const bf16* __restrict__ q, const bf16* __restrict__ k, const bf16* __restrict__ v, int first, int rows, int splits,
                 int passes, int append, float scale_log2, bf16* __restrict__ merged, float* __restrict__ part) {
  using L = Layout<HD>;
  constexpr int NG = L::NG, CT = HD / 16, ST = Ring<HD>::STAGES, PW = HD + 2, QT = NQ * 8;
  extern __shared__ __align__(128) unsigned char sm[];
  const int block = blockIdx.x / splits, split = blockIdx.x - block * splits, head_at = block / passes, pass = block - head_at * passes;
  const int sj = head_at / c.Hkv, kvh = head_at - sj * c.Hkv, seq = first + sj;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
  const int group = c.H / c.Hkv, nq = rows * group, q0 = pass * QT;
  const int len = c.lengths[seq], total = len + rows;
  const bool joins = splits <= CLUSTER;               // the slices are a cluster
  if (total > c.cap) {                                // no room: nothing is stored or advanced, the step's rows are zeros
    if (threadIdx.x == 0) c.full[seq] = 1;
    if (split == 0 && joins)
      for (int i = threadIdx.x; i < min(QT, nq - q0) * HD; i += THREADS) {
        const int qi = q0 + i / HD, r = qi / group, g = qi - r * group;
        merged[(((long long)sj * rows + r) * c.H + kvh * group + g) * HD + i % HD] = __float2bfloat16_rn(0.f);
      }
    return;
  }
  // pages of this slice, as far as the last query of the pass sees
  const int pages = (total + PAGE - 1) / PAGE, chunk = (pages + splits - 1) / splits;
  const int pg0 = split * chunk, pg1 = min(pages, pg0 + chunk);
  const int last_row = (min(q0 + QT, nq) - 1) / group, seen_pages = (len + last_row) / PAGE + 1;
  const int pend = min(pg1, seen_pages);
  unsigned char* head = page_at(c, seq, kvh, 0);

  if (append) {
    const long long W = (long long)c.Hkv * HD;
    for (int pg = max(pg0, len / PAGE); pg < pg1; ++pg) {
      const int p0 = max(len, pg * PAGE), p1 = min(total, (pg + 1) * PAGE);
      const long long at = ((long long)sj * rows + p0 - len) * W + kvh * HD;
      append_page<HD>(c, head + (long long)pg * L::BYTES, k + at, v + at, W, p0 - pg * PAGE, p1 - p0, p0, sm);
      __threadfence();
      __syncthreads();
    }
  }

  // ---- queries: rotated, scaled to base 2, rounded to bf16 once; lane (gid, tig) holds query gid's channels 32 g + 8 tig .. + 7 ----
  uint32_t qf[NQ][NG][4];
  float qs[NQ][NG][2];                                // sum over the group of queries 2 tig and 2 tig + 1
  int lim[NQ][2];                                     // positions that they see
#pragma unroll
  for (int nt = 0; nt < NQ; ++nt) {
    const int qi = q0 + nt * 8 + gid, ok = qi < nq, r = ok ? qi / group : 0, h = ok ? qi - r * group : 0;
    const bf16* src = q + (((long long)sj * rows + r) * c.H + kvh * group + h) * HD;
    const float* ct = c.cos_t + (long long)(len + r) * (HD / 2);
    const float* st = c.sin_t + (long long)(len + r) * (HD / 2);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const int ch = 32 * g + 8 * tig;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int at = ch + 2 * i + e;
          float a = ok ? __bfloat162float(src[at]) : 0.f;
          if (ok && c.rope) {
            const int low = at < HD / 2, f = low ? at : at - HD / 2;
            const float other = __bfloat162float(src[low ? at + HD / 2 : f]);
            a = low ? a * ct[f] - other * st[f] : a * ct[f] + other * st[f];
          }
          x[e] = a * scale_log2;
        }
        const __nv_bfloat162 p = __floats2bfloat162_rn(x[0], x[1]);
        qf[nt][g][i] = as_bits(p);
        sum += __low2float(p) + __high2float(p);
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
      for (int e = 0; e < 2; ++e) qs[nt][g][e] = __shfl_sync(0xffffffffu, sum, (2 * tig + e) * 4);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int qe = q0 + nt * 8 + 2 * tig + e;
      lim[nt][e] = qe < nq ? len + qe / group + 1 : 0;
    }
  }
  const int all_see = len + q0 / group + 1;           // positions below this are seen by every query of the pass

  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(sm) + warp * (ST * L::BYTES);
  const unsigned char* ring_ptr = sm + warp * (ST * L::BYTES);
  float m[NQ][2], l[NQ][2], o[NQ][CT][4];
#pragma unroll
  for (int nt = 0; nt < NQ; ++nt) {
    m[nt][0] = m[nt][1] = -INFINITY;
    l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) o[nt][ct][0] = o[nt][ct][1] = o[nt][ct][2] = o[nt][ct][3] = 0.f;
  }
  auto issue = [&](int pg, int stage) {
    if (pg < pend) {
      const unsigned char* src = head + (long long)pg * L::BYTES + lane * 16;
      const uint32_t dst = ring + stage * L::BYTES + lane * 16;
#pragma unroll
      for (int i = 0; i < L::BYTES; i += 512) copy16(dst + i, src + i);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const int my0 = pg0 + warp;
#pragma unroll
  for (int i = 0; i < ST - 1; ++i) issue(my0 + i * WARPS, i);
  int stage = 0;
  for (int pg = my0; pg < pend; pg += WARPS) {
    asm volatile("cp.async.wait_group %0;" ::"n"(ST - 2) : "memory");
    __syncwarp();                                     // every lane's copies of the page have landed, and the stage before is free
    issue(pg + (ST - 1) * WARPS, (stage + ST - 1) % ST);
    const unsigned char* page = ring_ptr + stage * L::BYTES;
    stage = (stage + 1) % ST;

    // ---- scores ----
    float s[NQ][4][4];
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) {
      const Words<NG> lo = load_words<NG>(page + L::KEYS + (16 * mt + gid) * (HD / 2) + tig * NG * 4);
      const Words<NG> hi = load_words<NG>(page + L::KEYS + (16 * mt + gid + 8) * (HD / 2) + tig * NG * 4);
      const Words<NG> plo = load_words<NG>(page + L::KPAR + (16 * mt + gid) * NG * 4);
      const Words<NG> phi = load_words<NG>(page + L::KPAR + (16 * mt + gid + 8) * NG * 4);
#pragma unroll
      for (int nt = 0; nt < NQ; ++nt) s[nt][mt][0] = s[nt][mt][1] = s[nt][mt][2] = s[nt][mt][3] = 0.f;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const uint32_t a0 = pair128<0>(lo.w[g]), a1 = pair128<0>(hi.w[g]), a2 = pair128<1>(lo.w[g]), a3 = pair128<1>(hi.w[g]);
        const uint32_t b0 = pair128<2>(lo.w[g]), b1 = pair128<2>(hi.w[g]), b2 = pair128<3>(lo.w[g]), b3 = pair128<3>(hi.w[g]);
        const float st0 = __uint_as_float(plo.w[g] << 16), ba0 = __uint_as_float(plo.w[g] & 0xffff0000u);
        const float st1 = __uint_as_float(phi.w[g] << 16), ba1 = __uint_as_float(phi.w[g] & 0xffff0000u);
#pragma unroll
        for (int nt = 0; nt < NQ; ++nt) {
          const float n0 = -128.f * qs[nt][g][0], n1 = -128.f * qs[nt][g][1];
          float acc[4] = {n0, n1, n0, n1};
          mma16816(acc, a0, a1, a2, a3, qf[nt][g][0], qf[nt][g][1]);
          mma16816(acc, b0, b1, b2, b3, qf[nt][g][2], qf[nt][g][3]);
          s[nt][mt][0] = fmaf(st0, acc[0], fmaf(ba0, qs[nt][g][0], s[nt][mt][0]));
          s[nt][mt][1] = fmaf(st0, acc[1], fmaf(ba0, qs[nt][g][1], s[nt][mt][1]));
          s[nt][mt][2] = fmaf(st1, acc[2], fmaf(ba1, qs[nt][g][0], s[nt][mt][2]));
          s[nt][mt][3] = fmaf(st1, acc[3], fmaf(ba1, qs[nt][g][1], s[nt][mt][3]));
        }
      }
    }
    // ---- softmax of the page; thread holds positions 16 mt + gid (+ 8) of queries 2 tig and 2 tig + 1 ----
    if ((pg + 1) * PAGE > all_see) {
#pragma unroll
      for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int nt = 0; nt < NQ; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (pg * PAGE + 16 * mt + gid + 8 * (e >> 1) >= lim[nt][e & 1]) s[nt][mt][e] = -INFINITY;
    }
    uint32_t p[NQ][4][2];
#pragma unroll
    for (int nt = 0; nt < NQ; ++nt) {
      float corr[2], ref[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float mx = fmaxf(s[nt][0][e], s[nt][0][e + 2]);
#pragma unroll
        for (int mt = 1; mt < 4; ++mt) mx = fmaxf(mx, fmaxf(s[nt][mt][e], s[nt][mt][e + 2]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        const float now = fmaxf(m[nt][e], mx);
        ref[e] = now > -INFINITY ? now : 0.f;         // nothing seen yet: every weight is 0
        corr[e] = ex2(m[nt][e] - ref[e]);
        m[nt][e] = now;
        l[nt][e] *= corr[e];
      }
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[e] = ex2(s[nt][mt][e] - ref[e & 1]);
          l[nt][e & 1] += w[e];
        }
        p[nt][mt][0] = transpose8x8(as_bits(__floats2bfloat162_rn(w[0], w[1])));
        p[nt][mt][1] = transpose8x8(as_bits(__floats2bfloat162_rn(w[2], w[3])));
      }
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        o[nt][ct][0] *= corr[0]; o[nt][ct][1] *= corr[1];
        o[nt][ct][2] *= corr[0]; o[nt][ct][3] *= corr[1];
      }
    }
    // ---- values ----
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const Words<8> step = load_words<8>(page + L::VSTEP + g * 128 + tig * 32), base = load_words<8>(page + L::VBASE + g * 128 + tig * 32);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int ct = 2 * g + half;
        const Words<2> lo = load_words<2>(page + L::VALUES + (16 * ct + gid) * 32 + tig * 8);
        const Words<2> hi = load_words<2>(page + L::VALUES + (16 * ct + gid + 8) * 32 + tig * 8);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const int j = 4 * w;
          const uint32_t a0 = value_pair<0>(lo.w[w], step.w[j], base.w[j]), a1 = value_pair<0>(hi.w[w], step.w[j], base.w[j]);
          const uint32_t a2 = value_pair<1>(lo.w[w], step.w[j + 1], base.w[j + 1]), a3 = value_pair<1>(hi.w[w], step.w[j + 1], base.w[j + 1]);
          const uint32_t b0 = value_pair<2>(lo.w[w], step.w[j + 2], base.w[j + 2]), b1 = value_pair<2>(hi.w[w], step.w[j + 2], base.w[j + 2]);
          const uint32_t b2 = value_pair<3>(lo.w[w], step.w[j + 3], base.w[j + 3]), b3 = value_pair<3>(hi.w[w], step.w[j + 3], base.w[j + 3]);
#pragma unroll
          for (int nt = 0; nt < NQ; ++nt) {
            mma16816(o[nt][ct], a0, a1, a2, a3, p[nt][2 * w][0], p[nt][2 * w][1]);
            mma16816(o[nt][ct], b0, b1, b2, b3, p[nt][2 * w + 1][0], p[nt][2 * w + 1][1]);
          }
        }
      }
    }
    __syncwarp();
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
  for (int nt = 0; nt < NQ; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 4);
      l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 8);
      l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 16);
    }

  // ---- join the warps: [query][warp][HD + 2], then this slice's [query][HD + 2] behind it ----
  float* mb = reinterpret_cast<float*>(sm);
  float* mine = mb + QT * WARPS * PW;
  __syncthreads();                                    // every ring is drained
#pragma unroll
  for (int nt = 0; nt < NQ; ++nt) {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        mb[((nt * 8 + 2 * tig + (e & 1)) * WARPS + warp) * PW + 16 * ct + gid + 8 * (e >> 1)] = o[nt][ct][e];
    if (gid == 0) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float* d = mb + ((nt * 8 + 2 * tig + e) * WARPS + warp) * PW + HD;
        d[0] = m[nt][e];
        d[1] = l[nt][e];
      }
    }
  }
  __syncthreads();
  const int live = min(QT, nq - q0);
  for (int i = threadIdx.x; i < live * HD; i += THREADS) {
    const int r = i / HD, ch = i - r * HD, qi = q0 + r;
    const float* src = mb + r * WARPS * PW;
    float mx = -INFINITY, num = 0.f, den = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) mx = fmaxf(mx, src[w * PW + HD]);
    const float ref = mx > -INFINITY ? mx : 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float wt = ex2(src[w * PW + HD] - ref);
      num = fmaf(wt, src[w * PW + ch], num);
      den = fmaf(wt, src[w * PW + HD + 1], den);
    }
    float* out = joins ? mine + r * PW
                       : part + ((((long long)sj * rows + qi / group) * c.H + kvh * group + qi % group) * splits + split) * PW;
    out[ch] = num;
    if (ch == 0) { out[HD] = mx; out[HD + 1] = den; }
  }
  if (!joins) return;                                 // kv_merge_kernel does the rest

  // ---- join the slices, write the merged heads, advance the length ----
  cg::cluster_group cl = cg::this_cluster();
  if (splits > 1) cl.sync(); else __syncthreads();
  for (int i = split * THREADS + threadIdx.x; i < live * HD; i += splits * THREADS) {
    const int r = i / HD, ch = i - r * HD, qi = q0 + r;
    float mx = -INFINITY, num = 0.f, den = 0.f;
    for (int p = 0; p < splits; ++p) mx = fmaxf(mx, (splits > 1 ? cl.map_shared_rank(mine, p) : mine)[r * PW + HD]);
    const float ref = mx > -INFINITY ? mx : 0.f;
    for (int p = 0; p < splits; ++p) {
      const float* src = (splits > 1 ? cl.map_shared_rank(mine, p) : mine) + r * PW;
      const float wt = ex2(src[HD] - ref);
      num = fmaf(wt, src[ch], num);
      den = fmaf(wt, src[HD + 1], den);
    }
    merged[(((long long)sj * rows + qi / group) * c.H + kvh * group + qi % group) * HD + ch] = __float2bfloat16_rn(num / den);
  }
  if (splits > 1) cl.sync();                          // nobody leaves while its slice is being read
  if (threadIdx.x == 0) {
    // every CTA of the sequence has read the length long before it takes its ticket; the last one moves it on
    const int ctas = splits * passes * c.Hkv;
    if (atomicAdd(c.tickets + seq, 1) == ctas - 1) {
      c.tickets[seq] = 0;
      c.lengths[seq] = total;
    }
  }
}

__global__ void tables_kernel(float* cos_t, float* sin_t, int positions, int half, double base) {
  const long long n = (long long)positions * half;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) {
    const int p = (int)(i / half), ch = (int)(i - (long long)p * half);
    const double angle = (double)p * pow(base, -(double)ch / half);
    cos_t[i] = (float)cos(angle);
    sin_t[i] = (float)sin(angle);
  }
}

__global__ void values_kernel(Cache c, int first, int from, int count, float* __restrict__ keys, float* __restrict__ values) {
  const int row = blockIdx.x, sj = row / count, seq = first + sj, W = c.Hkv * c.HD, NG = c.HD / GROUP;
  const int len = c.lengths[seq], pos = (from < 0 ? len - count : from) + row - sj * count;
  for (int i = threadIdx.x; i < W; i += blockDim.x) {
    float kv = 0.f, vv = 0.f;
    if (pos >= 0 && pos < len) {
      const int kvh = i / c.HD, ch = i - kvh * c.HD, g = ch / GROUP, slot = pos % PAGE;
      const unsigned char* page = page_at(c, seq, kvh, pos / PAGE);
      const uint32_t par = reinterpret_cast<const uint32_t*>(page + 64 * c.HD)[slot * NG + g];
      const uint32_t kw = reinterpret_cast<const uint32_t*>(page)[slot * (c.HD / 8) + ((ch & 31) >> 3) * NG + g];
      const uint32_t vw = reinterpret_cast<const uint32_t*>(page + 32 * c.HD)[ch * 8 + value_word(slot)];
      const uint16_t* vstep = reinterpret_cast<const uint16_t*>(page + 72 * c.HD) + g * 64 + value_slot(slot);
      const float kc = (float)((kw >> (4 * (((ch & 7) >> 1) + 4 * (ch & 1)))) & 15u), vc = (float)((vw >> (4 * value_nibble(slot))) & 15u);
      const float ks = __uint_as_float(par << 16);
      kv = fmaf(kc, ks, __uint_as_float(par & 0xffff0000u));
      vv = fmaf(vc, __uint_as_float((uint32_t)vstep[0] << 16), __uint_as_float((uint32_t)vstep[NG * 64] << 16));
      if (ks != ks) kv = vv = ks;
    }
    keys[(long long)row * W + i] = kv;
    values[(long long)row * W + i] = vv;
  }
}

template <int HD, int NQ>
cudaError_t go(const Cache& c, const bf16* q, const bf16* k, const bf16* v, int first, int n_seq, int rows, int splits, bool append, float scale_log2,
               bf16* merged, float* part, cudaStream_t st) {
  constexpr int smem = smem_bytes<HD, NQ>();
  auto kernel = attention_kernel<HD, NQ>;
  static std::atomic<unsigned long long> raised{0};   // devices on which the kernel's shared-memory limit has been raised
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  const unsigned long long bit = 1ull << (device & 63);
  if (!(raised.load(std::memory_order_relaxed) & bit)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    raised.fetch_or(bit, std::memory_order_relaxed);
  }
  const int nq = rows * (c.H / c.Hkv), passes = (nq + NQ * 8 - 1) / (NQ * 8);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(splits * passes * c.Hkv * n_seq));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = splits <= CLUSTER ? splits : 1; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  count_launch();
  return cudaLaunchKernelEx(&cfg, kernel, c, q, k, v, first, rows, splits, passes, append ? 1 : 0, scale_log2, merged, part);
}

}  // namespace

cudaError_t launch_tables(float* cos_t, float* sin_t, int positions, int head_dim, float base, cudaStream_t st) {
  const long long n = (long long)positions * (head_dim / 2);
  tables_kernel<<<(unsigned)std::min<long long>((n + 255) / 256, 148 * 8), 256, 0, st>>>(cos_t, sin_t, positions, head_dim / 2, (double)base);
  count_launch();
  return cudaGetLastError();
}

cudaError_t launch_append(const Cache& c, const bf16* k, const bf16* v, int first, int n_seq, int rows, cudaStream_t st) {
  const dim3 grid((unsigned)(((rows + PAGE - 2) / PAGE + 1) * c.Hkv * n_seq));
  switch (c.HD) {
    case 32: append_kernel<32><<<grid, THREADS, 0, st>>>(c, k, v, first, rows); break;
    case 64: append_kernel<64><<<grid, THREADS, 0, st>>>(c, k, v, first, rows); break;
    case 128: append_kernel<128><<<grid, THREADS, 0, st>>>(c, k, v, first, rows); break;
    case 256: append_kernel<256><<<grid, THREADS, 0, st>>>(c, k, v, first, rows); break;
    default: return cudaErrorInvalidValue;
  }
  count_launch();
  return cudaGetLastError();
}

int queries_per_pass(int head_dim, int queries) { return queries <= 8 || head_dim == 256 ? 8 : 16; }

cudaError_t launch_attention(const Cache& c, const bf16* q, const bf16* k, const bf16* v, int first, int n_seq, int rows, int splits, bool append,
                             float scale_log2, bf16* merged, float* part, cudaStream_t st) {
  const bool two = queries_per_pass(c.HD, rows * (c.H / c.Hkv)) == 16;
#define Q4_GO(HD, NQ) go<HD, NQ>(c, q, k, v, first, n_seq, rows, splits, append, scale_log2, merged, part, st)
  switch (c.HD) {
    case 32: return two ? Q4_GO(32, 2) : Q4_GO(32, 1);
    case 64: return two ? Q4_GO(64, 2) : Q4_GO(64, 1);
    case 128: return two ? Q4_GO(128, 2) : Q4_GO(128, 1);
    case 256: return Q4_GO(256, 1);
    default: return cudaErrorInvalidValue;
  }
#undef Q4_GO
}

cudaError_t launch_values(const Cache& c, int first, int n_seq, int from, int count, float* keys, float* values, cudaStream_t st) {
  values_kernel<<<(unsigned)(n_seq * count), 128, 0, st>>>(c, first, from, count, keys, values);
  count_launch();
  return cudaGetLastError();
}

}  // namespace q4
}  // namespace moe
