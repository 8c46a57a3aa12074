// KV cache held in 4 bits: append and decode attention (precision MOE_PRECISION_Q4 of include/kv_attention_b200.h).
//
// A decode step reads the whole cache once, so the bytes per position are the time: 4 bits a channel, and for each 32 channels of a
// head's key or value a bf16 step and base, value = code * step + base: 1.25 bytes a channel for key and value together, where a bf16
// cache takes 4.
//
// The 64 positions of a page lie together, as the tensor cores want them: one warp takes a page, S^T = K Q^T has the positions as
// the 16 rows and the queries as the 8 columns of mma.sync m16n8k16, O^T = V^T P^T has the channels as rows and the positions as the
// reduction.  So the few queries that share a kv head fill the small side of the product, and both K and V are the A operand:
// a lane's 32-bit word holds 8 codes that it needs itself, keys as 8 channels of one position, values as 8 positions of one channel.
// Bits 0 .. 7 of a bf16 are a number linear in them, bits * 2^-133: below 128 it is subnormal, and the next binade goes on in the same steps.  So
// a code needs no conversion, only to be cut out, at weight 1 (bits 0 .. 3) or 16 (bits 4 .. 7): five instructions a word.  The other
// factor makes up for the 2^-133, and for the 16 at the places that have it.
//   keys:   S = sum over groups of step * sum_c code q + base * sum_c q.  The first product takes its step in f32; the second part, bases
//           against the queries' sums in three bf16 pieces, is one more small product on the tensor cores.  Nothing of the key is rounded.
//           The codes enter as f16 numbers (bits * 2^-24, linear in the same way), the query as f16 under a power of two of its own: one
//           rounding of 2^-11 of a channel at most, where bf16 has 2^-8.
//   values: step and base belong to the position, which is what the product sums over, so they go on before it: one packed bf16
//           instruction, one rounding of the value to bf16 (2^-8 of it at most).  The weights enter as two bf16 numbers each, so that the value's
//           is the only rounding of that size before the output's: error against 64 bits 2.3e-3 of the output's rms, 3.3e-3 with one.
// What bounds it: to keep up with HBM, 148 SMs would have to do a page of 64 x 64 channels every 215 cycles, and its instructions take them about as
// long.  They issue 1.8 to 2.0 of the 4 a cycle that they could, no pipe is busy for more than 41 % of the time: with 8 to 13 warps an SM (the ring
// and the sums' registers allow no more) it is the warps' waits, for fixed latencies and at a CTA's start and end for one another, that nothing covers.
// Measured with a rollback behind each step, in a graph: 64 sequences of 4096 positions, 16/4 heads of 64, 26.4 us (bf16 cache: 58 us), of
// 16384 72.6 us (0.84 of the copy bandwidth for each further byte); 16 of 0 .. 32767, 32/8 heads of 128, one row 71 us, three rows 117 us,
// where the bytes alone take 51 us; one of 700 8.4 us, one of 32000 12.7 us.
//
// Page layout, HD = head_dim, NG = HD / 32:
//   keys    [64 positions][4 t][NG g] words: channels 32 g + 8 t + 2 i + e at nibble i + 4 e
//   key parameters [64 positions][NG / 2][step of two groups, base of two groups] (bf16 pairs); NG = 1: step and base in one word
//   values  [HD channels][4 t][2 w] words: positions 16 (2 w + i / 2) + 8 (i % 2) + 2 t + e at nibble i + 4 e
//   value step * 2^STEP_UP (another / 16 where the codes weigh 16), value base  [NG][64] bf16 each, position p at value_slot(p)
// A warp streams half pages (keys, then values) through its own ring in shared memory.  The warp whose page takes a step's new positions
// quantises them into its copy of the page and into the cache: nobody else reads them, so nobody has to wait.

#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <algorithm>
#include <atomic>
#include <cfloat>

#include "kv_q4.cuh"
#include "warp_ops.cuh"

namespace cg = cooperative_groups;

namespace moe {
namespace q4 {
namespace {

constexpr int WARPS = 4, THREADS = WARPS * 32;
constexpr float RISE = 8.f;                     // weights stay below 2^8 against the reference
constexpr float HUGE_VALUE = 1.099511627776e12f; // 2^40: a larger number counts as an infinity (a step times 2^STEP_UP is a bf16 number)
constexpr int RAW = 133;                        // bits 0 .. 7 of a bf16 are worth bits * 2^-RAW
constexpr int STEP_UP = 90;                     // value steps are kept times 2^STEP_UP against raw codes
constexpr int RAW_HALF = 24, Q_TOP = 13;        // bits 0 .. 7 of an f16: bits * 2^-24; a query's largest channel is in [2^13, 2^14) there
// whether a value's code weighs 16 in its word
__host__ __device__ inline int value_heavy(int p) { return (p >> 3) & 1; }

template <int HD> struct Layout {
  static constexpr int NG = HD / GROUP, KEYS = 0, KPAR = 32 * HD, HALF = 40 * HD, VALUES = HALF, VSTEP = 72 * HD, VBASE = VSTEP + NG * 128, BYTES = 80 * HD;
};
__host__ __device__ inline int value_word(int p) { return ((p & 7) >> 1) * 2 + (p >> 5); }
__host__ __device__ inline int value_nibble(int p) { return ((p >> 4) & 1) * 2 + ((p >> 3) & 1) + 4 * (p & 1); }
__host__ __device__ inline int value_slot(int p) { return ((p & 7) >> 1) * 16 + (p >> 4) * 4 + ((p >> 3) & 1) * 2 + (p & 1); }

// byte offset of a key's step in the page's key parameters; its base is base_after bytes behind
__host__ __device__ inline int key_param(int slot, int g, int NG) { return slot * NG * 4 + (NG == 1 ? 0 : (g >> 1) * 8 + (g & 1) * 2); }
__host__ __device__ inline int key_base_after(int NG) { return NG == 1 ? 2 : 4; }

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
    float lo, hi;                                     // over the warp; the values are finite
    asm volatile("redux.sync.min.f32 %0, %1, 0xffffffff;" : "=f"(lo) : "f"(x[g]));
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(hi) : "f"(x[g]));
    const bf16 s = __float2bfloat16_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.f)), b = __float2bfloat16_rn(lo);
    const float sf = __bfloat162float(s), bf = __bfloat162float(b);
    code[g] = sf > 0.f ? (uint32_t)fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x[g], bf), sf)), 0.f), 15.f) : 0u;
    step[g] = __bfloat16_as_ushort(s);
    base[g] = __bfloat16_as_ushort(b);
  }
}

// One warp: the codes, steps and bases of one new position; lane l holds channels 32 g + l.  k and v point to the head's row.
template <int HD>
struct Row {
  static constexpr int NG = HD / GROUP;
  uint32_t kcode[NG], kstep[NG], kbase[NG], vcode[NG], vstep[NG], vbase[NG];
  __device__ __forceinline__ void make(const Cache& c, const bf16* __restrict__ k, const bf16* __restrict__ v, int pos) {
    const int lane = threadIdx.x & 31;
    float x[NG], y[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      x[g] = __bfloat162float(k[32 * g + lane]);
      y[g] = __bfloat162float(v[32 * g + lane]);
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
    quantise<NG>(x, kcode, kstep, kbase);
    quantise<NG>(y, vcode, vstep, vbase);
#pragma unroll
    for (int g = 0; g < NG; ++g)                      // exact: a power of two
      vstep[g] = __bfloat16_as_ushort(__float2bfloat16_rn(__uint_as_float(vstep[g] << 16) * pow2(value_heavy(pos) ? STEP_UP - 4 : STEP_UP)));
    if (bad) {
#pragma unroll
      for (int g = 0; g < NG; ++g) kstep[g] = 0x7fc0u;
    }
  }
  // the key's word of group g, in every lane of the eight that hold its channels
  __device__ __forceinline__ uint32_t key_word(int g) const {
    const int lane = threadIdx.x & 31;
    uint32_t w = kcode[g] << (4 * (((lane & 7) >> 1) + 4 * (lane & 1)));
    w |= __shfl_xor_sync(0xffffffffu, w, 1);
    w |= __shfl_xor_sync(0xffffffffu, w, 2);
    return w | __shfl_xor_sync(0xffffffffu, w, 4);
  }
};

// Rotates, quantises and stores new positions.  A CTA has the 32 positions of a page that share its value words (w of the page layout), so
// old positions keep their codes without anybody else writing to the words; a warp takes a position, two where its registers hold 256
// channels.  What bounds it is the time of one position from its loads to its stores: 2 prompts of 256 rows take 9 us with a cold cache
// (40 us with four warps for a whole page).
template <int HD> struct Append { static constexpr int WARPS = HD <= 128 ? 32 : 16; };

template <int HD>
__global__ void __launch_bounds__(Append<HD>::WARPS * 32) append_kernel(Cache c, const bf16* __restrict__ k, const bf16* __restrict__ v, int first, int rows) {
  using L = Layout<HD>;
  constexpr int NG = L::NG, HALF_PAGE = PAGE / 2;
  pdl_follow();
  __shared__ unsigned char codes[HALF_PAGE * HD];
  const int touched = (rows + HALF_PAGE - 2) / HALF_PAGE + 1;   // half pages that rows new positions can lie in
  const int kvh = blockIdx.x / touched % c.Hkv, sj = blockIdx.x / touched / c.Hkv, seq = first + sj, len = c.lengths[seq];
  if (len + rows > c.cap) return;                     // reported by the launch that follows
  const int half = len / HALF_PAGE + blockIdx.x % touched, start = half * HALF_PAGE;
  const int p0 = max(len, start), p1 = min(len + rows, start + HALF_PAGE);
  if (p0 >= p1) return;
  unsigned char* page = page_at(c, seq, kvh, half / 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int pos = p0 + warp; pos < p1; pos += Append<HD>::WARPS) {
    const long long at = (((long long)sj * rows + pos - len) * c.Hkv + kvh) * HD;
    const int slot = pos % PAGE;
    Row<HD> row;
    row.make(c, k + at, v + at, pos);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const uint32_t w = row.key_word(g);
      if ((lane & 7) == 0) reinterpret_cast<uint32_t*>(page + L::KEYS)[slot * (HD / 8) + (lane >> 3) * NG + g] = w;
      codes[(pos - start) * HD + 32 * g + lane] = (unsigned char)row.vcode[g];
      if (lane == 0) {
        uint16_t* par = reinterpret_cast<uint16_t*>(page + L::KPAR + key_param(slot, g, NG));
        par[0] = (uint16_t)row.kstep[g];
        par[key_base_after(NG) / 2] = (uint16_t)row.kbase[g];
        reinterpret_cast<uint16_t*>(page + L::VSTEP)[g * 64 + value_slot(slot)] = (uint16_t)row.vstep[g];
        reinterpret_cast<uint16_t*>(page + L::VBASE)[g * 64 + value_slot(slot)] = (uint16_t)row.vbase[g];
      }
    }
  }
  __syncthreads();
  uint32_t* vw = reinterpret_cast<uint32_t*>(page + L::VALUES);
  for (int i = threadIdx.x; i < HD * 4; i += Append<HD>::WARPS * 32) {
    const int ch = i >> 2, t = i & 3, word = ch * 8 + t * 2 + (half & 1);
    uint32_t set = 0, val = 0;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const int p = start + 16 * ((n & 3) >> 1) + 8 * (n & 1) + 2 * t + (n >> 2);
      if (p >= p0 && p < p1) {
        set |= 15u << (4 * n);
        val |= (uint32_t)codes[(p - start) * HD + ch] << (4 * n);
      }
    }
    if (set) vw[word] = set == 0xffffffffu ? val : (vw[word] & ~set) | val;
  }
}

// ---- attention ----
// f16 operands; the second one from zero
__device__ __forceinline__ void mma16816_half(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816_half_new(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma1688_new(float* d, uint32_t a0, uint32_t a1, uint32_t b0) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5}, {%6}, {%7, %7, %7, %7};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(b0), "f"(0.f));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// codes i and i + 4 of a word, raw bf16 or f16 numbers as raw_pair cuts them out,
// ... and as values times 2^(STEP_UP - RAW); base has that factor already
template <int I>
__device__ __forceinline__ uint32_t value_pair(uint32_t w, uint32_t step, uint32_t base) {
  return as_bits(__hfma2(as_pair(raw_pair<I>(w)), as_pair(step), as_pair(base)));
}

// eight channels of a query's row, 0 for a query that does not exist
__device__ __forceinline__ void load8(const bf16* src, int ch, bool ok, bool wide, float* x) {
  if (!ok) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.f;
  } else if (wide) {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(src + ch));
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __bfloat162float(src[ch + i]);
  }
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

// Half pages in a warp's ring.
template <int HD> struct Ring { static constexpr int SLOTS = HD <= 64 ? 4 : 3; };

// The queries' fragments, the pieces of their sums and their factors, then per warp: the ring, and the new positions of one page (at most QT of them) until
// the page has come: key words, value codes, steps and bases.  In the end the partial results take the place of all that.
template <int HD, int NQ> struct Smem {
  static constexpr int NG = Layout<HD>::NG, NP = NG == 1 ? 1 : NG / 2;
  static constexpr int QUERIES = NQ * NG * 512, SUMS = NQ * NP * 128, FACTORS = QUERIES + SUMS, FRONT = FACTORS + (NQ * 32 + 127) / 128 * 128;
  static constexpr int RING = Ring<HD>::SLOTS * Layout<HD>::HALF, ROW = HD / 2 + HD + 8 * NG, NEW = NQ * 8 * ROW, WARP = RING + (NEW + 127) / 128 * 128;
  static constexpr int MERGE = NQ * 8 * (WARPS + 1) * (HD + 2) * 4;
  static constexpr int BYTES = FRONT + WARPS * WARP > MERGE ? FRONT + WARPS * WARP : MERGE;
};

// grid: ((sequence * kv heads + kv head) * passes + pass) * splits + split; the splits of one are a cluster when `joins` is set
// FOLD: the last eight columns hold at most four queries, twice.  In the products with the values the first four of them have the upper
// parts of the weights and the last four the lower ones, so the second parts cost no products of their own.
template <int HD, int NQ, bool FOLD>
__global__ void __launch_bounds__(THREADS)
attention_kernel(Cache c, const bf16* __restrict__ q, const bf16* __restrict__ k, const bf16* __restrict__ v, int first, int rows, int splits, int slice,
                 int passes, int append, int joins, float scale_log2, bf16* __restrict__ merged, float* __restrict__ part) {
  using L = Layout<HD>;
  constexpr int NG = L::NG, CT = HD / 16, SLOTS = Ring<HD>::SLOTS, PW = HD + 2, QT = NQ * 8 - (FOLD ? 4 : 0);
  // Two tiles of queries of 128 channels are read again for each product: held in registers, 32 of them, they leave the rest too few
  // (12 queries, 16 sequences of up to 32767 positions: 138 us against 144).
  constexpr bool FAR = HD == 128 && NQ == 2;
  extern __shared__ __align__(128) unsigned char sm[];
  const int block = blockIdx.x / splits, split = blockIdx.x - block * splits, head_at = block / passes, pass = block - head_at * passes;
  const int sj = head_at / c.Hkv, kvh = head_at - sj * c.Hkv, seq = first + sj;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
  const int group = c.H / c.Hkv, nq = rows * group, q0 = pass * QT;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int len = c.lengths[seq], total = len + rows;
  if (total > c.cap) {                                // no room: nothing is stored or advanced, the step's rows are zeros
    if (threadIdx.x == 0) {
      c.full[seq] = 1;
      if (split == 0 && pass == 0 && kvh == 0) c.skipped[seq] = rows > 0x7fffffff - c.skipped[seq] ? 0x7fffffff : c.skipped[seq] + rows;
    }
    if (split == 0)
      for (int i = threadIdx.x; i < min(QT, nq - q0) * HD; i += THREADS) {
        const int qi = q0 + i / HD, r = qi / group, g = qi - r * group;
        merged[(((long long)sj * rows + r) * c.H + kvh * group + g) * HD + i % HD] = __float2bfloat16_rn(0.f);
      }
    return;
  }
  // pages of this slice, as far as the last query of the pass sees
  const int pages = (total + PAGE - 1) / PAGE, chunk = max(slice, (pages + splits - 1) / splits);
  const int pg0 = split * chunk, pg1 = min(pages, pg0 + chunk);
  const int last_row = (min(q0 + QT, nq) - 1) / group, seen_pages = (len + last_row) / PAGE + 1;
  const int pend = min(pg1, seen_pages);
  if (!joins && pg0 >= pend) return;                  // no such slice: merge_kernel does not look for it either
  unsigned char* head = page_at(c, seq, kvh, 0);
  // The warp's half pages, last page first (the new positions are in the last ones): unit 2 j is the keys and 2 j + 1 the values of page
  // pg - j * WARPS.
  using M = Smem<HD, NQ>;
  unsigned char* ring = sm + M::FRONT + warp * M::WARP;
  unsigned char* fresh = ring + M::RING;
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring) + lane * 16;
  int pg = pend - 1 - warp;
  int issue_pg = pg, issue_half = 0, issue_slot = 0, slot = 0;
  auto issue = [&] {
    if (issue_pg >= pg0) {
      const unsigned char* src = head + (long long)issue_pg * L::BYTES + issue_half + lane * 16;
      const uint32_t dst = ring_at + issue_slot * L::HALF;
#pragma unroll
      for (int i = 0; i + 512 <= L::HALF; i += 512) copy16(dst + i, src + i);
      if (L::HALF % 512 != 0 && lane * 16 < L::HALF % 512) copy16(dst + L::HALF / 512 * 512, src + L::HALF / 512 * 512);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    issue_slot = issue_slot + 1 == SLOTS ? 0 : issue_slot + 1;
    if (issue_half) issue_pg -= WARPS;
    issue_half = issue_half ? 0 : L::HALF;
  };
  auto next_half = [&]() -> unsigned char* {
    asm volatile("cp.async.wait_group %0;" ::"n"(SLOTS - 2) : "memory");
    __syncwarp();                                     // every lane's copies of the half have landed, and the one before is used up
    issue();
    unsigned char* p = ring + slot * L::HALF;
    slot = slot + 1 == SLOTS ? 0 : slot + 1;
    return p;
  };
#pragma unroll
  for (int i = 0; i < SLOTS - 1; ++i) issue();

  // ---- the slice's new positions: quantised while the pages and the queries are under way, each by another warp, into `fresh` of the warp
  // whose first page has them.  A row there is the key's words in page order, the value's codes, then step | base of the key's and of the
  // value's groups.  (Three rows one after the other in the page's own warp: 16 x 0 .. 32767 takes 119 us instead of 116.5.) ----
  const int new0 = max(len, pg * PAGE), news = append && pg >= pg0 ? max(0, min(total, (pg + 1) * PAGE) - new0) : 0;   // this warp's
  for (int pos = len + warp; append && pos < total; pos += WARPS) {
    const int page = pos / PAGE;
    if (page < pg0 || page >= pend) continue;         // in another slice
    const long long at = (((long long)sj * rows + pos - len) * c.Hkv + kvh) * HD;
    unsigned char* f = sm + M::FRONT + (pend - 1 - page) * M::WARP + M::RING + (pos - max(len, page * PAGE)) * M::ROW;
    Row<HD> row;
    row.make(c, k + at, v + at, pos);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const uint32_t w = row.key_word(g);
      if ((lane & 7) == 0) reinterpret_cast<uint32_t*>(f)[(lane >> 3) * NG + g] = w;
      f[HD / 2 + 32 * g + lane] = (unsigned char)row.vcode[g];
      if (lane < 2) reinterpret_cast<uint32_t*>(f + HD / 2 + HD)[lane * NG + g] = lane ? row.vstep[g] | row.vbase[g] << 16 : row.kstep[g] | row.kbase[g] << 16;
    }
  }

  // ---- queries: rotated, rounded once to f16 under a power of two of their own; eight channels of one query a thread and turn ----
  {
    const bool wide = (reinterpret_cast<uintptr_t>(q) & 15) == 0;     // a head's row is a multiple of 16 bytes
    uint4* frag = reinterpret_cast<uint4*>(sm);
    uint16_t* sums = reinterpret_cast<uint16_t*>(sm + M::QUERIES);
    float* factors = reinterpret_cast<float*>(sm + M::FACTORS);
    constexpr int EIGHTS = (QT * HD / 8 + 31) / 32 * 32;              // whole warps: their lanes shuffle
#pragma unroll
    for (int i0 = 0; i0 < EIGHTS; i0 += THREADS) {
      const int i = i0 + THREADS - 32 - (int)(threadIdx.x & ~31u) + lane, at = i / (HD / 8), ch = 8 * (i % (HD / 8)), g = ch / 32, t = (ch / 8) & 3;
      if (EIGHTS % THREADS != 0 && i >= EIGHTS) break;                // the first warps have new positions to see to
      const int qi = q0 + at, ok = qi < nq, r = ok ? qi / group : 0, h = ok ? qi - r * group : 0;
      const bf16* src = q + (((long long)sj * rows + r) * c.H + kvh * group + h) * HD;
      const int low = ch < HD / 2, f = low ? ch : ch - HD / 2;
      float x[8], sum = 0.f;
      load8(src, ch, ok, wide, x);
      if (c.rope && ok) {
        const float* ct = c.cos_t + (long long)(len + r) * (HD / 2) + f;
        const float* st = c.sin_t + (long long)(len + r) * (HD / 2) + f;
        float other[8], co[8], si[8];
        load8(src, low ? ch + HD / 2 : f, ok, wide, other);
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
          *reinterpret_cast<float4*>(co + j) = __ldg(reinterpret_cast<const float4*>(ct + j));
          *reinterpret_cast<float4*>(si + j) = __ldg(reinterpret_cast<const float4*>(st + j));
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = low ? x[j] * co[j] - other[j] * si[j] : x[j] * co[j] + other[j] * si[j];
      }
      // the power of two that takes the query's largest channel to Q_TOP, and what makes up for it in the scores
      float top = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(x[j]));
#pragma unroll
      for (int d = 1; d < HD / 8; d *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
      const int e = min(max((int)(__float_as_uint(top) >> 23) - 127, -100), 116);
      const float by = __uint_as_float((uint32_t)(127 + Q_TOP - e) << 23);
      if (i % (HD / 8) == 0) factors[at] = scale_log2 * __uint_as_float((uint32_t)(127 + RAW_HALF - Q_TOP + e) << 23);
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        __half2 p = __floats2half2_rn(x[2 * j] * by, x[2 * j + 1] * by);
        sum += __low2float(p) + __high2float(p);
        if (j & 1) p = __hmul2(p, __float2half2_rn(0.0625f));
        w[j] = *reinterpret_cast<const uint32_t*>(&p);
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      sum *= pow2(-RAW_HALF);
      if (FOLD && at >= QT) continue;                                 // no such query
      const int nt = at >> 3, to = (at & 7) * 4 + t;                  // the lane that multiplies these channels
      frag[(nt * NG + g) * 32 + to] = make_uint4(w[0], w[1], w[2], w[3]);
      const bool twice = FOLD && nt == NQ - 1;
      if (twice) frag[(nt * NG + g) * 32 + to + 16] = make_uint4(w[0], w[1], w[2], w[3]);
      // the sum as three bf16 numbers, one for each of the lanes t = 0, 1, 2
      const bf16 s0 = __float2bfloat16_rn(sum), s1 = __float2bfloat16_rn(sum - __bfloat162float(s0));
      const bf16 s2 = __float2bfloat16_rn(sum - __bfloat162float(s0) - __bfloat162float(s1));
      const bf16 piece = t == 0 ? s0 : t == 1 ? s1 : t == 2 ? s2 : __float2bfloat16_rn(0.f);
      uint16_t* d = sums + ((nt * M::NP + (NG == 1 ? 0 : g >> 1)) * 32 + to) * 2;
      if (NG == 1) {
        d[0] = 0;                                                     // against the step that shares the word with the base
        d[1] = __bfloat16_as_ushort(piece);
      } else {
        d[g & 1] = __bfloat16_as_ushort(piece);
      }
      if (twice) {
        if (NG == 1) d[32] = 0;
        d[32 + (NG == 1 ? 1 : g & 1)] = __bfloat16_as_ushort(piece);
      }
    }
  }
  __syncthreads();
  if (joins && threadIdx.x == 0) {
    // Advance the length: this CTA has read it, and the last CTA of the sequence to say so moves it on.
    if (atomicAdd(c.tickets + seq, 1) == splits * passes * c.Hkv - 1) {
      c.tickets[seq] = 0;
      c.lengths[seq] = total;
      c.skipped[seq] = 0;
    }
  }
  uint32_t qf[NQ][NG][4], qb[NQ][M::NP];              // fragments; pieces of the sums
  float factor[NQ][2];                                // from the products' units to powers of two, of queries 2 tig and 2 tig + 1
  int lim[NQ][2];                                     // positions that queries 2 tig and 2 tig + 1 see
  auto load_query = [&](int nt, int g) {
    const uint4 w = reinterpret_cast<const uint4*>(sm)[(nt * NG + g) * 32 + lane];
    qf[nt][g][0] = w.x; qf[nt][g][1] = w.y; qf[nt][g][2] = w.z; qf[nt][g][3] = w.w;
  };
#pragma unroll
  for (int nt = 0; nt < NQ; ++nt) {
#pragma unroll
    for (int g = 0; g < NG; ++g)
      if (!FAR) load_query(nt, g);
#pragma unroll
    for (int j = 0; j < M::NP; ++j) {
      qb[nt][j] = reinterpret_cast<const uint32_t*>(sm + M::QUERIES)[(nt * M::NP + j) * 32 + lane];
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int at = nt * 8 + (FOLD && nt == NQ - 1 ? 2 * tig & 3 : 2 * tig) + e, qe = q0 + at;
      factor[nt][e] = reinterpret_cast<const float*>(sm + M::FACTORS)[at];
      lim[nt][e] = qe < nq ? len + qe / group + 1 : 0;
    }
  }
  const int all_see = len + q0 / group + 1;           // positions below this are seen by every query of the pass
  const uint32_t lower = tig >= 2 ? ~0u : 0u;         // FOLD: this lane's columns have the lower parts

  // A weight is 2^(score - ref): ref is the maximum when it was last looked up and stays until a score passes it
  // by RISE; until then neither the sums nor the products have to be scaled.  Values are kept times 2^(STEP_UP - RAW).
  float ref[NQ][2], l[NQ][2], o[NQ][CT][4];

#pragma unroll
  for (int nt = 0; nt < NQ; ++nt) {
    ref[nt][0] = ref[nt][1] = -INFINITY;
    l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) o[nt][ct][0] = o[nt][ct][1] = o[nt][ct][2] = o[nt][ct][3] = 0.f;
  }
  for (; pg >= pg0; pg -= WARPS) {
    unsigned char* page = next_half();
    const bool has_new = news > 0 && new0 / PAGE == pg;
    unsigned char* out = head + (long long)pg * L::BYTES;
    if (has_new) {                                    // new keys into the page and into the cache
      for (int r = 0; r < news; ++r) {
        const unsigned char* f = fresh + r * M::ROW;
        const int at = new0 + r - pg * PAGE;
        for (int i = lane; i < HD / 8; i += 32) {
          const uint32_t w = reinterpret_cast<const uint32_t*>(f)[i];
          reinterpret_cast<uint32_t*>(page + L::KEYS)[at * (HD / 8) + i] = w;
          reinterpret_cast<uint32_t*>(out + L::KEYS)[at * (HD / 8) + i] = w;
        }
        if (lane < 2 * NG) {
          const int g = lane >> 1, par = L::KPAR + key_param(at, g, NG) + (lane & 1) * key_base_after(NG);
          const uint16_t b = reinterpret_cast<const uint16_t*>(f + HD / 2 + HD)[lane];
          *reinterpret_cast<uint16_t*>(page + par) = b;
          *reinterpret_cast<uint16_t*>(out + par) = b;
        }
      }
      __syncwarp();
    }

    // ---- scores ----
    float s[NQ][4][4];
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) {
      const Words<NG> lo = load_words<NG>(page + L::KEYS + (16 * mt + gid) * (HD / 2) + tig * NG * 4);
      const Words<NG> hi = load_words<NG>(page + L::KEYS + (16 * mt + gid + 8) * (HD / 2) + tig * NG * 4);
      const Words<NG> plo = load_words<NG>(page + L::KPAR + (16 * mt + gid) * NG * 4);
      const Words<NG> phi = load_words<NG>(page + L::KPAR + (16 * mt + gid + 8) * NG * 4);
      // bases: the word of two groups' bases is the same for the lanes of a position, each lane has its piece of the queries' sums
#pragma unroll
      for (int nt = 0; nt < NQ; ++nt) {
        if constexpr (M::NP == 1) {
          mma1688_new(s[nt][mt], plo.w[NG - 1], phi.w[NG - 1], qb[nt][0]);
        } else {
          mma16816_new(s[nt][mt], plo.w[1], phi.w[1], plo.w[3], phi.w[3], qb[nt][0], qb[nt][1]);
#pragma unroll
          for (int j = 2; j < M::NP; j += 2)
            mma16816(s[nt][mt], plo.w[2 * j + 1], phi.w[2 * j + 1], plo.w[2 * j + 3], phi.w[2 * j + 3], qb[nt][j], qb[nt][j + 1]);
        }
      }
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const uint32_t a0 = raw_pair<0>(lo.w[g]), a1 = raw_pair<0>(hi.w[g]), a2 = raw_pair<1>(lo.w[g]), a3 = raw_pair<1>(hi.w[g]);
        const uint32_t b0 = raw_pair<2>(lo.w[g]), b1 = raw_pair<2>(hi.w[g]), b2 = raw_pair<3>(lo.w[g]), b3 = raw_pair<3>(hi.w[g]);
        const uint32_t w0 = plo.w[NG == 1 ? 0 : g & ~1], w1 = phi.w[NG == 1 ? 0 : g & ~1];
        const float st0 = __uint_as_float(g & 1 ? w0 & 0xffff0000u : w0 << 16), st1 = __uint_as_float(g & 1 ? w1 & 0xffff0000u : w1 << 16);
#pragma unroll
        for (int nt = 0; nt < NQ; ++nt) {
          float acc[4];
          if (FAR) load_query(nt, g);
          mma16816_half_new(acc, a0, a1, a2, a3, qf[nt][g][0], qf[nt][g][1]);
          mma16816_half(acc, b0, b1, b2, b3, qf[nt][g][2], qf[nt][g][3]);
          s[nt][mt][0] = fmaf(st0, acc[0], s[nt][mt][0]);
          s[nt][mt][1] = fmaf(st0, acc[1], s[nt][mt][1]);
          s[nt][mt][2] = fmaf(st1, acc[2], s[nt][mt][2]);
          s[nt][mt][3] = fmaf(st1, acc[3], s[nt][mt][3]);
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
    uint32_t p[NQ][4][2], p_lo[NQ][4][2];             // the weights as two bf16 numbers each
    bool rise = false;
    float mx[NQ][2];
#pragma unroll
    for (int nt = 0; nt < NQ; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float a = fmaxf(s[nt][0][e], s[nt][0][e + 2]);
#pragma unroll
        for (int mt = 1; mt < 4; ++mt) a = fmaxf(a, fmaxf(s[nt][mt][e], s[nt][mt][e + 2]));
        mx[nt][e] = a;
        rise |= fmaf(a, factor[nt][e], -ref[nt][e]) > RISE;
      }
    if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
      for (int nt = 0; nt < NQ; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float a = mx[nt][e];
          a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 4));
          a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 8));
          a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 16));
          a = fmaxf(a * factor[nt][e], ref[nt][e]);
          const float corr = a > -INFINITY ? ex2(ref[nt][e] - a) : 1.f;
          ref[nt][e] = a;
          l[nt][e] *= corr;
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) { o[nt][ct][e] *= corr; o[nt][ct][e + 2] *= corr; }
        }
    }
#pragma unroll
    for (int nt = 0; nt < NQ; ++nt) {
      const bool fold = FOLD && nt == NQ - 1;
      // a query that has seen nothing yet has scores of -inf only: weights of 0 against any finite number
      const uint64_t up = pack2(factor[nt][0], factor[nt][1]);
      const uint64_t minus = pack2(ref[nt][0] > -INFINITY ? -ref[nt][0] : 0.f, ref[nt][1] > -INFINITY ? -ref[nt][1] : 0.f);
      uint64_t sum = pack2(l[nt][0], l[nt][1]);
#pragma unroll
      for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float y0, y1;
          unpack2(fma2(pack2(s[nt][mt][2 * h], s[nt][mt][2 * h + 1]), up, minus), y0, y1);
          const float w0 = ex2(y0), w1 = ex2(y1);
          sum = add2(sum, pack2(w0, w1));
          const uint32_t w = as_bits(__floats2bfloat162_rn(w0, w1)), less = fold ? w & lower : w;
          const uint32_t rest = as_bits(__floats2bfloat162_rn(w0 - __uint_as_float(less << 16), w1 - __uint_as_float(less & 0xffff0000u)));
          p[nt][mt][h] = transpose8x8(fold ? rest : w);
          if (!fold) p_lo[nt][mt][h] = transpose8x8(rest);
        }
      unpack2(sum, l[nt][0], l[nt][1]);
    }
    // ---- values ----
    page = next_half() - L::HALF;                     // so that the page's offsets hold
    if (has_new) {                                    // ... and new values
      for (int r = 0; r < news; ++r) {
        const unsigned char* f = fresh + r * M::ROW + HD / 2;
        const int at = new0 + r - pg * PAGE, w = value_word(at), n = 4 * value_nibble(at);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          uint32_t* word = reinterpret_cast<uint32_t*>(page + L::VALUES) + (32 * g + lane) * 8 + w;
          *word = (*word & ~(15u << n)) | (uint32_t)f[32 * g + lane] << n;
          reinterpret_cast<uint32_t*>(out + L::VALUES)[(32 * g + lane) * 8 + w] = *word;
        }
        if (lane < 2 * NG) {
          const int off = (lane & 1 ? L::VBASE : L::VSTEP) + ((lane >> 1) * 64 + value_slot(at)) * 2;
          const uint16_t b = reinterpret_cast<const uint16_t*>(f + HD + 4 * NG)[lane];
          *reinterpret_cast<uint16_t*>(page + off) = b;
          *reinterpret_cast<uint16_t*>(out + off) = b;
        }
      }
      __syncwarp();
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const Words<8> step = load_words<8>(page + L::VSTEP + g * 128 + tig * 32);
      Words<8> base = load_words<8>(page + L::VBASE + g * 128 + tig * 32);
#pragma unroll
      for (int j = 0; j < 8; ++j) base.w[j] = as_bits(__hmul2(as_pair(base.w[j]), __float2bfloat162_rn(pow2(STEP_UP - RAW))));
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
            if (!FOLD || nt < NQ - 1) {
              mma16816(o[nt][ct], a0, a1, a2, a3, p_lo[nt][2 * w][0], p_lo[nt][2 * w][1]);
              mma16816(o[nt][ct], b0, b1, b2, b3, p_lo[nt][2 * w + 1][0], p_lo[nt][2 * w + 1][1]);
            }
          }
        }
      }
    }
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

  if (FOLD) {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[NQ - 1][ct][e] += __shfl_xor_sync(0xffffffffu, o[NQ - 1][ct][e], 2);
  }

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // ---- join the warps: [query][warp][HD + 2], then this slice's [query][HD + 2] behind it ----
  float* mb = reinterpret_cast<float*>(sm);
  float* mine = mb + QT * WARPS * PW;
  __syncthreads();                                    // every ring is drained
#pragma unroll
  for (int nt = 0; nt < NQ; ++nt) {
    if (FOLD && nt == NQ - 1 && tig >= 2) break;                      // the others have it all
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        mb[((nt * 8 + 2 * tig + (e & 1)) * WARPS + warp) * PW + 16 * ct + gid + 8 * (e >> 1)] = o[nt][ct][e] * pow2(RAW - STEP_UP);
    if (gid == 0) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float* d = mb + ((nt * 8 + 2 * tig + e) * WARPS + warp) * PW + HD;
        d[0] = ref[nt][e];
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
  if (!joins) return;                                 // merge_kernel does the rest

  // ---- join the slices, write the merged heads ----
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
}

// One CTA joins the slices of one row's head, each warp every fourth of them.
template <int HD>
__global__ void __launch_bounds__(THREADS)
merge_kernel(Cache c, const float* __restrict__ part, int first, int rows, int splits, int slice, int per_pass, bf16* __restrict__ merged) {
  constexpr int PW = HD + 2, CH = HD / 32, AHEAD = 4;
  __shared__ float sums[WARPS][PW];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long at = blockIdx.x;                    // (sequence * rows + row) * heads + head
  pdl_follow();                                       // the slices are written
  const int row_at = (int)(at / c.H), h = (int)(at - (long long)row_at * c.H), sj = row_at / rows, row = row_at - sj * rows, seq = first + sj;
  const int len = c.lengths[seq], total = len + rows, group = c.H / c.Hkv;
  if (total > c.cap) return;                          // marked, and its rows zeroed, by the step
  const int pages = (total + PAGE - 1) / PAGE, chunk = max(slice, (pages + splits - 1) / splits);
  const int pass = (row * group + h % group) / per_pass, last_row = (min((pass + 1) * per_pass, rows * group) - 1) / group;
  const int live = (min(pages, (len + last_row) / PAGE + 1) + chunk - 1) / chunk;
  const float* src = part + at * splits * PW;
  float ref = -INFINITY, den = 0.f, num[CH];
#pragma unroll
  for (int i = 0; i < CH; ++i) num[i] = 0.f;
  for (int p0 = warp; p0 < live; p0 += WARPS * AHEAD) {
    float m[AHEAD], l[AHEAD], x[AHEAD][CH];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const int p = p0 + a * WARPS, ok = p < live;
      m[a] = ok ? __ldcg(src + p * PW + HD) : -INFINITY;
      l[a] = ok ? __ldcg(src + p * PW + HD + 1) : 0.f;
#pragma unroll
      for (int i = 0; i < CH; ++i) x[a][i] = ok ? __ldcg(src + p * PW + 32 * i + lane) : 0.f;
    }
    float now = ref;
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) now = fmaxf(now, m[a]);
    const float base = now > -INFINITY ? now : 0.f, corr = ex2(ref - base);
    den *= corr;
#pragma unroll
    for (int i = 0; i < CH; ++i) num[i] *= corr;
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const float w = ex2(m[a] - base);
      den = fmaf(w, l[a], den);
#pragma unroll
      for (int i = 0; i < CH; ++i) num[i] = fmaf(w, x[a][i], num[i]);
    }
    ref = now;
  }
#pragma unroll
  for (int i = 0; i < CH; ++i) sums[warp][32 * i + lane] = num[i];
  if (lane == 0) { sums[warp][HD] = ref; sums[warp][HD + 1] = den; }
  __syncthreads();
  for (int ch = threadIdx.x; ch < HD; ch += THREADS) {
    float mx = -INFINITY, n = 0.f, d = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) mx = fmaxf(mx, sums[w][HD]);
    const float base = mx > -INFINITY ? mx : 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float wt = ex2(sums[w][HD] - base);
      n = fmaf(wt, sums[w][ch], n);
      d = fmaf(wt, sums[w][HD + 1], d);
    }
    merged[at * HD + ch] = __float2bfloat16_rn(n / d);
  }
  // every thread has read the length before the barrier above; the last CTA of the sequence moves it on
  if (threadIdx.x == 0 && atomicAdd(c.tickets + seq, 1) == rows * c.H - 1) {
    c.tickets[seq] = 0;
    c.lengths[seq] = total;
    c.skipped[seq] = 0;
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
  pdl_follow();
  const int len = c.lengths[seq], pos = (from < 0 ? len - count : from) + row - sj * count;
  for (int i = threadIdx.x; i < W; i += blockDim.x) {
    float kv = 0.f, vv = 0.f;
    if (pos >= 0 && pos < len) {
      const int kvh = i / c.HD, ch = i - kvh * c.HD, g = ch / GROUP, slot = pos % PAGE;
      const unsigned char* page = page_at(c, seq, kvh, pos / PAGE);
      const unsigned char* par = page + 32 * c.HD + key_param(slot, g, NG);
      const uint32_t kw = reinterpret_cast<const uint32_t*>(page)[slot * (c.HD / 8) + ((ch & 31) >> 3) * NG + g];
      const uint32_t vw = reinterpret_cast<const uint32_t*>(page + 40 * c.HD)[ch * 8 + value_word(slot)];
      const uint16_t* vstep = reinterpret_cast<const uint16_t*>(page + 72 * c.HD) + g * 64 + value_slot(slot);
      const float kc = (float)((kw >> (4 * (((ch & 7) >> 1) + 4 * (ch & 1)))) & 15u), vc = (float)((vw >> (4 * value_nibble(slot))) & 15u);
      const float ks = __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t*>(par) << 16);
      kv = fmaf(kc, ks, __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t*>(par + key_base_after(NG)) << 16));
      vv = fmaf(vc, __uint_as_float((uint32_t)vstep[0] << 16) * pow2(value_heavy(slot) ? 4 - STEP_UP : -STEP_UP), __uint_as_float((uint32_t)vstep[NG * 64] << 16));
      if (ks != ks) kv = vv = ks;
    }
    keys[(long long)row * W + i] = kv;
    values[(long long)row * W + i] = vv;
  }
}

template <int HD, int NQ, bool FOLD = false>
cudaError_t go(const Cache& c, const bf16* q, const bf16* k, const bf16* v, int first, int n_seq, int rows, int splits, int slice, bool append, float scale_log2,
               bf16* merged, float* part, cudaStream_t st) {
  constexpr int smem = Smem<HD, NQ>::BYTES;
  auto kernel = attention_kernel<HD, NQ, FOLD>;
  const int nq = rows * (c.H / c.Hkv), passes = (nq + NQ * 8 - 1) / (NQ * 8);
  const bool joins = part == nullptr;
  const cudaError_t e = launch_following(kernel, (unsigned)(splits * passes * c.Hkv * n_seq), joins ? splits : 1, THREADS, smem, st, c, q, k, v, first, rows,
                                         splits, slice, passes, append ? 1 : 0, joins ? 1 : 0, scale_log2, merged, part);
  if (e != cudaSuccess || joins) return e;
  // resident as soon as the step's last CTA has only its results to write
  return launch_following(merge_kernel<HD>, (unsigned)(n_seq * rows * c.H), 1, THREADS, 0, st, c, (const float*)part, first, rows, splits, slice, NQ * 8, merged);
}

}  // namespace

cudaError_t launch_tables(float* cos_t, float* sin_t, int positions, int head_dim, float base, cudaStream_t st) {
  const long long n = (long long)positions * (head_dim / 2);
  tables_kernel<<<(unsigned)std::min<long long>((n + 255) / 256, 148 * 8), 256, 0, st>>>(cos_t, sin_t, positions, head_dim / 2, (double)base);
  count_launch();
  return cudaGetLastError();
}

cudaError_t launch_append(const Cache& c, const bf16* k, const bf16* v, int first, int n_seq, int rows, cudaStream_t st) {
  const unsigned grid = (unsigned)(((rows + PAGE / 2 - 2) / (PAGE / 2) + 1) * c.Hkv * n_seq);
  switch (c.HD) {
    case 32: return launch_following(append_kernel<32>, grid, 1, Append<32>::WARPS * 32, 0, st, c, k, v, first, rows);
    case 64: return launch_following(append_kernel<64>, grid, 1, Append<64>::WARPS * 32, 0, st, c, k, v, first, rows);
    case 128: return launch_following(append_kernel<128>, grid, 1, Append<128>::WARPS * 32, 0, st, c, k, v, first, rows);
    case 256: return launch_following(append_kernel<256>, grid, 1, Append<256>::WARPS * 32, 0, st, c, k, v, first, rows);
    default: return cudaErrorInvalidValue;
  }
}

int queries_per_pass(int head_dim, int queries) { return queries <= 8 || head_dim == 256 ? 8 : 16; }

cudaError_t launch_attention(const Cache& c, const bf16* q, const bf16* k, const bf16* v, int first, int n_seq, int rows, int splits, int slice, bool append,
                             float scale_log2, bf16* merged, float* part, cudaStream_t st) {
  const int nq = rows * (c.H / c.Hkv);
  const bool two = queries_per_pass(c.HD, nq) == 16, fold = nq <= (two ? 12 : 4);
#define Q4_GO(HD, ...) go<HD, __VA_ARGS__>(c, q, k, v, first, n_seq, rows, splits, slice, append, scale_log2, merged, part, st)
  switch (c.HD) {
    case 32: return two ? (fold ? Q4_GO(32, 2, true) : Q4_GO(32, 2)) : fold ? Q4_GO(32, 1, true) : Q4_GO(32, 1);
    case 64: return two ? (fold ? Q4_GO(64, 2, true) : Q4_GO(64, 2)) : fold ? Q4_GO(64, 1, true) : Q4_GO(64, 1);
    case 128: return two ? (fold ? Q4_GO(128, 2, true) : Q4_GO(128, 2)) : fold ? Q4_GO(128, 1, true) : Q4_GO(128, 1);
    case 256: return fold ? Q4_GO(256, 1, true) : Q4_GO(256, 1);
    default: return cudaErrorInvalidValue;
  }
#undef Q4_GO
}

template <int HD, int NQ, bool FOLD = false>
int resident(int device) {
  static std::atomic<int> known[64] = {};             // per device, plus one
  std::atomic<int>& slot = known[device & 63];
  if (const int n = slot.load(std::memory_order_relaxed)) return n - 1;
  int per_sm = 0;
  cudaFuncSetAttribute(attention_kernel<HD, NQ, FOLD>, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<HD, NQ>::BYTES);
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, attention_kernel<HD, NQ, FOLD>, THREADS, Smem<HD, NQ>::BYTES) != cudaSuccess) {
    cudaGetLastError();
    per_sm = 1;
  }
  slot.store(per_sm + 1, std::memory_order_relaxed);
  return per_sm;
}

int ctas_per_sm(int head_dim, int queries, int device) {
  const bool two = queries_per_pass(head_dim, queries) == 16, fold = queries <= (two ? 12 : 4);
  switch (head_dim) {
    case 32: return two ? (fold ? resident<32, 2, true>(device) : resident<32, 2>(device)) : fold ? resident<32, 1, true>(device) : resident<32, 1>(device);
    case 64: return two ? (fold ? resident<64, 2, true>(device) : resident<64, 2>(device)) : fold ? resident<64, 1, true>(device) : resident<64, 1>(device);
    case 128: return two ? (fold ? resident<128, 2, true>(device) : resident<128, 2>(device)) : fold ? resident<128, 1, true>(device) : resident<128, 1>(device);
    default: return fold ? resident<256, 1, true>(device) : resident<256, 1>(device);
  }
}

cudaError_t launch_values(const Cache& c, int first, int n_seq, int from, int count, float* keys, float* values, cudaStream_t st) {
  return launch_following(values_kernel, (unsigned)(n_seq * count), 1, 128, 0, st, c, first, from, count, keys, values);
}

}  // namespace q4
}  // namespace moe
