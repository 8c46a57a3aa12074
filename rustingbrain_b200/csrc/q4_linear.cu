// Linear layer with 4-bit weights (the ABI of include/q4_linear_b200.h).
//
// For a decode batch the bytes of the weights are the time, so the layout is made for one pass over them: a block of 16 outputs x 64
// input channels is 512 bytes, 16 for each lane of a warp, in the order in which the lane needs them as the A operand of the tensor cores (the
// outputs are the 16 rows, the batch rows the 8 columns).  A lane's 32-bit word holds 8 consecutive channels of one output; since the
// channels of a product may come in any order, the activations' 8 channels are one 16-byte shared load of the B operand.  Two such blocks
// (32 outputs) and their scales are a unit, which a warp brings into its own ring in shared memory, several units ahead.
//
// Bits 0 .. 7 of a bf16 are a number linear in them, bits * 2^-133 (below 128 it is subnormal, and the next binade goes on in the same
// steps).  So a code plus 8 is cut out of its word, at weight 1 or, where it comes out four bits further up, 16, and one packed multiply-add makes
// two of them code * 2^-6: nine instructions for eight codes.  The activations enter as they are, whatever their size; an f32 one is three
// bf16 numbers that add up to it.  Products are exact, the group's scale is applied to its f32 sum, and infinities and NaN go their own way.
// (The cut-out bits themselves as operands, a group's sum starting at -8 times the sum of its activations, would save four of the nine
// instructions and is wrong: the tensor cores cut the terms of a product off at 2^-23 or so of the largest, so a channel 1e5 times as large as its
// neighbours takes 1 % off the result even where all its codes are 0.)
// (e4m3 operands would take three instructions for eight codes, but mma.sync has no e4m3 product of its own here: it costs two bf16 ones
// and the conversions.)
//
// A CTA keeps the activations of up to 16 rows in shared memory and goes through tiles of outputs, weights arriving without a pause from
// tile to tile; its warps split the reduction of a tile.  More rows are passes side by side, which find the weights in L2.  Where there
// are fewer tiles than SMs the CTAs of a cluster split the reduction too.  Partial sums meet in (distributed) shared memory, always in
// the same order: one launch, no workspace.
//
// Measured in a graph: 1 x 1024 -> 2816 3.5 us; 8 x 4096 -> 24576 15.9 us, one row 14.9 us, 16 rows 19.6 us, 64 rows 61.6 us (the bytes: 8.25 us); 64 x
// 1024 -> 5632 7.8 us; f32 3 x 2048 -> 32003 17.1 us (5.7 us).  The large ones wait: 2.2 instructions a cycle of the 4 that an SM can issue (f32
// 1.9), no pipe above 44 %, 12 to 16 warps an SM that wait for fixed latencies (1.3 of them for each issue; f32 2.1), loads (0.8) and their turn at
// the pipes (0.6; f32 1.9, its three products for one keep the tensor cores at 41 %).

#include <cooperative_groups.h>
#include <algorithm>
#include <atomic>
#include <cstdio>

#include "../../include/moe_b200.h"
#include "../../include/q4_linear_b200.h"
#include "common.cuh"
#include "warp_ops.cuh"

namespace cg = cooperative_groups;

namespace moe {
namespace {

constexpr int QL_MAX_WARPS = 16;
constexpr int QL_MAX_IN = 1 << 16;       // a row of f32 activations, cut over a cluster, fits shared memory
constexpr int QL_CODE = 6;               // operands are codes times 2^-QL_CODE

// A unit: 32 outputs and 128 channels, codes [2 output blocks][2 channel blocks][512 bytes], then scales [2][128 / group][8][2] bf16.
constexpr int QL_CHANNELS = 128, QL_CODES = 2048;
__host__ __device__ constexpr int ql_unit_bytes(int group) { return QL_CODES + 2 * (QL_CHANNELS / group) * 32; }
struct QlShape {
  int d_in, d_out, group, pairs, units;   // pairs of 16 outputs; units along the reduction
};
inline QlShape ql_shape(int d_out, int d_in, int group) {
  return QlShape{d_in, d_out, group, (d_out + 31) / 32, (d_in + QL_CHANNELS - 1) / QL_CHANNELS};
}
inline long long ql_bytes(const QlShape& s) { return (long long)s.pairs * s.units * ql_unit_bytes(s.group); }

// Byte offsets of output n's word for channels k .. k + 7 (k a multiple of 8), and of its scale; inside a word channel 2 i + e is nibble
// i + 4 e.
__device__ inline long long ql_unit_at(const QlShape& s, int n, int k) { return ((long long)(n >> 5) * s.units + k / QL_CHANNELS) * ql_unit_bytes(s.group); }
__device__ inline long long ql_word_at(const QlShape& s, int n, int k) {
  return ql_unit_at(s, n, k) + (((n >> 4) & 1) * 2 + ((k >> 6) & 1)) * 512 + (((n & 7) * 4 + ((k >> 3) & 3)) * 4 + 2 * ((k >> 5) & 1) + ((n >> 3) & 1)) * 4;
}
__device__ inline long long ql_scale_at(const QlShape& s, int n, int k) {
  return ql_unit_at(s, n, k) + QL_CODES + (((n >> 4) & 1) * (QL_CHANNELS / s.group) + k % QL_CHANNELS / s.group) * 32 + (n & 7) * 4 + ((n >> 3) & 1) * 2;
}
__host__ __device__ inline int ql_nibble(int c) { return ((c & 7) >> 1) + 4 * (c & 1); }

// ---- packing (once per matrix) ----
// one thread per eight channels of one output, padding included
__global__ void ql_pack_kernel(const int8_t* __restrict__ codes, const bf16* __restrict__ scales, unsigned char* __restrict__ packed, QlShape s) {
  const int per = s.units * QL_CHANNELS / 8, groups = s.d_in / s.group;
  const long long total = (long long)s.pairs * 32 * per;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x) {
    const int n = (int)(i / per), k = (int)(i - (long long)n * per) * 8, grp = k / s.group;
    uint32_t w = 0;
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const int code = n < s.d_out && k + c < s.d_in ? codes[(long long)n * s.d_in + k + c] : 0;
      w |= ((uint32_t)(code + 8) & 15u) << (4 * ql_nibble(c));
    }
    *reinterpret_cast<uint32_t*>(packed + ql_word_at(s, n, k)) = w;
    if (k % s.group == 0)
      *reinterpret_cast<bf16*>(packed + ql_scale_at(s, n, k)) = n < s.d_out && grp < groups ? scales[(long long)n * groups + grp] : __float2bfloat16_rn(0.f);
  }
}

// one thread per (output, group), padding included
__global__ void ql_quantize_kernel(const float* __restrict__ weights, unsigned char* __restrict__ packed, QlShape s) {
  const int per = s.units * QL_CHANNELS / s.group, groups = s.d_in / s.group;
  const long long total = (long long)s.pairs * 32 * per;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x) {
    const int n = (int)(i / per), grp = (int)(i - (long long)n * per);
    const bool live = n < s.d_out && grp < groups;
    const float* w = weights + (long long)n * s.d_in + (long long)grp * s.group;
    float top = 0.f;
    bool bad = false;
    if (live)
      for (int c = 0; c < s.group; ++c) {
        const float a = fabsf(w[c]);
        bad |= !(a <= 3.4028234663852886e38f);
        top = fmaxf(top, a);
      }
    const bf16 scale = __float2bfloat16_rn(bad ? __uint_as_float(0x7fc00000u) : __fdiv_rn(top, 7.f));
    const float f = __bfloat162float(scale);
    for (int c0 = 0; c0 < s.group; c0 += 8) {
      uint32_t word = 0;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        int code = 0;
        if (live && f > 0.f) code = (int)fminf(fmaxf(rintf(__fdiv_rn(w[c0 + c], f)), -8.f), 7.f);
        word |= ((uint32_t)(code + 8) & 15u) << (4 * ql_nibble(c));
      }
      *reinterpret_cast<uint32_t*>(packed + ql_word_at(s, n, grp * s.group + c0)) = word;
    }
    *reinterpret_cast<bf16*>(packed + ql_scale_at(s, n, grp * s.group)) = scale;
  }
}

__device__ __forceinline__ float ql_weight(const unsigned char* packed, const QlShape& s, int n, int k) {
  const uint32_t w = *reinterpret_cast<const uint32_t*>(packed + ql_word_at(s, n, k & ~7));
  return (float)((int)((w >> (4 * ql_nibble(k))) & 15u) - 8) * __bfloat162float(*reinterpret_cast<const bf16*>(packed + ql_scale_at(s, n, k)));
}
__global__ void ql_dequantize_kernel(const unsigned char* __restrict__ packed, float* __restrict__ weights, QlShape s) {
  const long long total = (long long)s.d_out * s.d_in;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x)
    weights[i] = ql_weight(packed, s, (int)(i / s.d_in), (int)(i % s.d_in));
}

// ---- the product ----
// codes i and i + 4 of a word, times 2^-QL_CODE; exact
template <int I>
__device__ __forceinline__ uint32_t ql_codes(uint32_t w) {
  constexpr float by = pow2(133 - QL_CODE - (I & 1 ? 4 : 0)), eight = 8 * pow2(-QL_CODE);      // what was cut out is (code + 8) * 2^-133, or 16 times that
  return as_bits(__hfma2(as_pair(raw_pair<I>(w)), __float2bfloat162_rn(by), __float2bfloat162_rn(-eight)));
}

// Eight activations as they are loaded, and as operands.
template <typename T> constexpr int QL_BATCH = sizeof(T) == 2 ? 4 : 2;
template <typename T> struct QlRaw;
template <> struct QlRaw<bf16> {
  struct type { uint4 v; };
  static __device__ __forceinline__ type load(const bf16* p) { return {__ldg(reinterpret_cast<const uint4*>(p))}; }
  static __device__ __forceinline__ void pieces(const type& a, uint4* out) { out[0] = a.v; }
};
template <> struct QlRaw<float> {
  struct type { float4 a, b; };
  static __device__ __forceinline__ type load(const float* p) { return {__ldg(reinterpret_cast<const float4*>(p)), __ldg(reinterpret_cast<const float4*>(p) + 1)}; }
  // three bf16 numbers that add up to each, the leading 8 bits of what is left; an infinity or a NaN is one alone
  static __device__ __forceinline__ void pieces(const type& t, uint4* out) {
    float f[8];
    uint32_t p[8][3];
    *reinterpret_cast<float4*>(f) = t.a;
    *reinterpret_cast<float4*>(f + 4) = t.b;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float v = f[j];
#pragma unroll
      for (int q = 0; q < 3; ++q) {
        p[j][q] = __float_as_uint(v) & 0xffff0000u;
        v -= __uint_as_float(p[j][q]);
      }
      if (!(fabsf(f[j]) <= 3.4028234663852886e38f)) {
        p[j][0] = f[j] != f[j] ? 0x7fc00000u : __float_as_uint(f[j]);
        p[j][1] = p[j][2] = 0;
      }
    }
#pragma unroll
    for (int q = 0; q < 3; ++q)
      out[q] = make_uint4(p[0][q] >> 16 | p[1][q], p[2][q] >> 16 | p[3][q], p[4][q] >> 16 | p[5][q], p[6][q] >> 16 | p[7][q]);
  }
};

template <typename T> struct QlPieces { static constexpr int N = 1; };
template <> struct QlPieces<float> { static constexpr int N = 3; };

// How a launch cuts the product, and where things lie in shared memory: the activations [piece][row][2 bytes a channel, and 64 that keep
// the 16-byte loads of a warp off each other's banks]; the warps' rings; the partial sums [buffer][wk][row][outputs of the tile] f32.
struct QlPlan {
  int warps, wk, cluster;              // warps of a CTA, those of them along the reduction; CTAs along it
  int tiles, passes, clusters;         // tiles of outputs; passes over the rows; clusters that share the tiles of a pass
  int slice, per_pass, stages, buffers;   // units of the reduction per CTA, at most; rows per pass; units in a ring; buffers of partial sums
  int rings, sums, bytes;
};

// grid: (clusters * passes) * cluster, the passes over the same tiles next to each other
template <typename T, int NT, int GROUP>
__global__ void __launch_bounds__(QL_MAX_WARPS * 32)
q4_linear_kernel(const T* __restrict__ x, long long ld_x, const unsigned char* __restrict__ packed, T* __restrict__ y, long long ld_y, int rows_total,
                 QlShape s, QlPlan plan) {
  constexpr int P = QlPieces<T>::N, SUBS = GROUP / 32, PER_UNIT = QL_CHANNELS / GROUP, BYTES = ql_unit_bytes(GROUP);
  extern __shared__ __align__(128) unsigned char ql_sm[];
  pdl_follow();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
  const int threads = blockDim.x, wk_count = plan.wk, wn_count = plan.warps / wk_count, wk = warp % wk_count, wn = warp / wk_count;
  const int cluster = plan.cluster, rank = blockIdx.x % cluster, pass = blockIdx.x / cluster % plan.passes, tile0 = blockIdx.x / cluster / plan.passes;
  const int row0 = pass * plan.per_pass, rows = min(rows_total - row0, plan.per_pass);
  const int ubeg = (int)((long long)s.units * rank / cluster), uend = (int)((long long)s.units * (rank + 1) / cluster);
  const int k0 = ubeg * QL_CHANNELS, channels = (uend - ubeg) * QL_CHANNELS;
  const int pitch = plan.slice * QL_CHANNELS * 2 + 64, plane = rows * pitch;
  unsigned char* acts = ql_sm;

  // ---- the warp's units: of the tiles tile0, tile0 + clusters, .. those from ubeg + wk on in steps of wk_count ----
  const int first = ubeg + wk;
  int stage = 0;
  unsigned char* ring = ql_sm + plan.rings + warp * (plan.stages * BYTES);
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring) + lane * 16;
  const int pairs_per_tile = wn_count * plan.clusters;
  int next_pair = first < uend ? tile0 * wn_count + wn : s.pairs, next_unit = first;
  const unsigned char* next_src = packed + ((long long)next_pair * s.units + first) * BYTES + lane * 16;
  uint32_t next_dst = ring_at;
  const uint32_t ring_end = ring_at + plan.stages * BYTES;
  auto issue = [&] {
    if (next_pair < s.pairs) {
#pragma unroll
      for (int i = 0; i < QL_CODES; i += 512) copy16(next_dst + i, next_src + i);
      if (lane < (BYTES - QL_CODES) / 16) copy16(next_dst + QL_CODES, next_src + QL_CODES);
      next_unit += wk_count;
      next_src += wk_count * BYTES;
      if (next_unit >= uend) {
        next_src += ((long long)pairs_per_tile * s.units + first - next_unit) * BYTES;
        next_unit = first;
        next_pair += pairs_per_tile;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    next_dst = next_dst + BYTES == ring_end ? ring_at : next_dst + BYTES;
  };
  for (int i = 0; i < plan.stages - 1; ++i) issue();

  // ---- the activations of the slice, eight channels of a row at a time, several loads of a thread in flight ----
  const int parts = channels / 8, work = rows * parts, row_step = threads / parts, part_step = threads - row_step * parts;
  int r = threadIdx.x / parts, c = threadIdx.x - r * parts;
  for (int i0 = threadIdx.x; i0 < work; i0 += QL_BATCH<T> * threads) {
    typename QlRaw<T>::type raw[QL_BATCH<T>];
    int to[QL_BATCH<T>];
#pragma unroll
    for (int u = 0; u < QL_BATCH<T>; ++u) {
      to[u] = r * pitch + c * 16;
      raw[u] = {};                                                // zeros behind the last channel
      if (i0 + u * threads < work && k0 + c * 8 < s.d_in) raw[u] = QlRaw<T>::load(x + (row0 + r) * ld_x + k0 + c * 8);
      r += row_step;
      c += part_step;
      if (c >= parts) { c -= parts; ++r; }
    }
#pragma unroll
    for (int u = 0; u < QL_BATCH<T>; ++u) {
      if (i0 + u * threads >= work) break;
      uint4 out[P];
      QlRaw<T>::pieces(raw[u], out);
#pragma unroll
      for (int q = 0; q < P; ++q) *reinterpret_cast<uint4*>(acts + q * plane + to[u]) = out[q];
    }
  }
  __syncthreads();

  const unsigned char* mine[NT];                                  // rows past the last one repeat it; nobody looks at their sums
#pragma unroll
  for (int n = 0; n < NT; ++n) mine[n] = acts + min(n * 8 + gid, rows - 1) * pitch + tig * 16;
  const int width = wn_count * 32;
  float* red = reinterpret_cast<float*>(ql_sm + plan.sums);
  const int other = plan.buffers == 2 ? wk_count * rows * width : 0;
  int turn = 0;
  cg::cluster_group cl = cg::this_cluster();

  for (int tile = tile0; tile < plan.tiles; tile += plan.clusters) {
    const bool live = tile * wn_count + wn < s.pairs;
    float acc[2][NT][4];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n) acc[m][n][0] = acc[m][n][1] = acc[m][n][2] = acc[m][n][3] = 0.f;
    // a pair that does not exist has no units in the ring: the warp only takes part in the joining
    for (int unit = first; live && unit < uend; unit += wk_count) {
      if (plan.stages == 2) asm volatile("cp.async.wait_group 0;" ::: "memory");
      else if (plan.stages == 3) asm volatile("cp.async.wait_group 1;" ::: "memory");
      else asm volatile("cp.async.wait_group 2;" ::: "memory");
      __syncwarp();                                               // the unit has landed for every lane, and the one before is used up
      issue();
      const unsigned char* at = ring + stage;
      stage = stage + BYTES == plan.stages * BYTES ? 0 : stage + BYTES;
      const int c0 = (unit - ubeg) * QL_CHANNELS;
      float part[2][NT][4];
      auto scaled = [&](int grp) {
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const uint32_t v = *reinterpret_cast<const uint32_t*>(at + QL_CODES + (m * PER_UNIT + grp) * 32 + gid * 4);
          const float s0 = __uint_as_float(v << 16), s1 = __uint_as_float(v & 0xffff0000u);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            acc[m][n][0] = fmaf(s0, part[m][n][0], acc[m][n][0]);
            acc[m][n][1] = fmaf(s0, part[m][n][1], acc[m][n][1]);
            acc[m][n][2] = fmaf(s1, part[m][n][2], acc[m][n][2]);
            acc[m][n][3] = fmaf(s1, part[m][n][3], acc[m][n][3]);
          }
        }
      };
#pragma unroll
      for (int block = 0; block < 2; ++block) {
        uint4 w[2];
#pragma unroll
        for (int m = 0; m < 2; ++m) w[m] = *reinterpret_cast<const uint4*>(at + (m * 2 + block) * 512 + lane * 16);
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const int g32 = block * 2 + g, grp = g32 / SUBS, off = (c0 + g32 * 32) * 2;
          const bool opens = P > 1 || g32 % SUBS == 0, closes = P > 1 || g32 % SUBS == SUBS - 1;
          uint32_t a[2][8];
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            const uint32_t lo = g ? w[m].z : w[m].x, hi = g ? w[m].w : w[m].y;
            a[m][0] = ql_codes<0>(lo); a[m][1] = ql_codes<0>(hi); a[m][2] = ql_codes<1>(lo); a[m][3] = ql_codes<1>(hi);
            a[m][4] = ql_codes<2>(lo); a[m][5] = ql_codes<2>(hi); a[m][6] = ql_codes<3>(lo); a[m][7] = ql_codes<3>(hi);
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int q = 0; q < P; ++q) {
              const uint4 b = *reinterpret_cast<const uint4*>(mine[n] + q * plane + off);
#pragma unroll
              for (int m = 0; m < 2; ++m) {
                if (opens && q == 0) mma16816_new(part[m][n], a[m][0], a[m][1], a[m][2], a[m][3], b.x, b.y);
                else mma16816(part[m][n], a[m][0], a[m][1], a[m][2], a[m][3], b.x, b.y);
                mma16816(part[m][n], a[m][4], a[m][5], a[m][6], a[m][7], b.z, b.w);
              }
            }
          }
          // f32: the tensor cores cut sums off where f32 arithmetic rounds them, so chains are short
          if (closes) scaled(grp);
        }
      }
    }

    // ---- add up the warps and the cluster, always in the same order ----
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = n * 8 + 2 * tig + e;
        if (r >= rows) continue;
        float* dst = red + (wk * rows + r) * width + wn * 32 + gid;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          dst[16 * m] = acc[m][n][e] * pow2(QL_CODE);
          dst[16 * m + 8] = acc[m][n][2 + e] * pow2(QL_CODE);
        }
      }
    const int n0 = tile * width;
    if (cluster > 1) cl.sync(); else __syncthreads();
    const int count = cluster * wk_count;
    for (int i = rank * threads + threadIdx.x; i < rows * width / 4; i += cluster * threads) {
      const int r = i * 4 / width, n = i * 4 % width;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
      for (int j = 0; j < count; ++j) {
        const int from = j / wk_count, w = j - from * wk_count;
        const float* src = (cluster > 1 ? cl.map_shared_rank(red, from) : red) + w * rows * width + i * 4;
        const float4 p = *reinterpret_cast<const float4*>(src);
        v.x += p.x; v.y += p.y; v.z += p.z; v.w += p.w;
      }
      const float out[4] = {v.x, v.y, v.z, v.w};
      T* dst = y + (row0 + r) * ld_y + n0 + n;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n0 + n + j < s.d_out) dst[j] = from_f32<T>(out[j]);
    }
    // with two buffers the next tile writes to the other one, and its barrier comes before this one is written again
    if (plan.buffers == 1) { if (cluster > 1) cl.sync(); else __syncthreads(); }
    red += turn ? -other : other;
    turn ^= 1;
  }
  if (cluster > 1) cl.sync();                                     // nobody leaves while its sums are being read
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

int ql_fail(char* msg, int len, int code, const char* text) {
  if (msg && len > 0) snprintf(msg, len, "%s", text);
  return code;
}

bool ql_sizes_ok(int d_out, int d_in, int group) {
  return d_out > 0 && d_in > 0 && (group == 32 || group == 64 || group == 128) && d_in % group == 0 && d_in <= QL_MAX_IN && d_out <= (1 << 28);
}

// How to cut a product with `live` <= NT * 8 rows a pass: of the ways that fit, the one that should be done first.  False: none fits.
// The estimate is in cycles of an SM and counts what was measured: a unit takes an SM the issue of its instructions (0.17 a cycle for each warp, up to 2.6), its
// products (2.1 cycles each) or its share of HBM (24 bytes a cycle), whichever is longest, and a warp no less than its latency; a thread takes
// 20 to 100 instructions for eight activations.  Joining a CTA's only tile takes 1200 cycles, over a cluster 2700 to 3700 and 100 for each part beyond
// 16 that comes from other SMs (1 x 8192 -> 1024: 32 parts 7.6 us, 64 parts 8.6 us); each further tile, for which the warps drain and fill
// again, 3500 and 5000 to 8000.  So a cluster of two pays where it makes rounds fewer: 8 x 4096 -> 24576 f32 25.1 us against 40 without clusters
// and 29 with four SMs, but 1 x 1024 -> 2816 3.5 us without and 4.6 with two.
template <typename T, int NT, int GROUP>
bool ql_plan(const QlShape& s, int rows, int live, QlPlan* out) {
  constexpr int P = QlPieces<T>::N, BYTES = ql_unit_bytes(GROUP), SM = 148;
  constexpr double issue = (70 + 4 * (P == 1 ? 44 + 5 * NT : 48 + 18 * NT) + QL_CHANNELS / (P == 1 ? GROUP : 32) * (6 + 18 * NT));
  constexpr double products = 16 * NT * 2.1 * P;
  const int most[4] = {8, 8, 12, 16}, limit[4] = {113 * 1024, 227 * 1024, 227 * 1024, 227 * 1024}, resident[4] = {2, 1, 1, 1};
  const double first[4] = {1200, 2700, 3200, 3700}, more[4] = {3500, 5000, 6500, 8000};
  const int at_once[4] = {SM, 74, 33, 15};   // clusters of 1, 2, 4 and 8 SMs that the machine holds: they do not cross the borders of a GPC
  double best = -1;
  QlPlan p{};
  p.per_pass = live;
  p.passes = (rows + live - 1) / live;
  auto up = [](int v) { return (v + 127) / 128 * 128; };
  for (int way = 0; way < 4; ++way)
    for (int log = 0; log < 4; ++log) {
      p.cluster = 1 << log;
      p.warps = most[way];
      p.slice = (s.units + p.cluster - 1) / p.cluster;
      if (p.cluster > 1 && s.units < 2 * p.cluster) break;
      p.rings = up(P * live * (p.slice * QL_CHANNELS * 2 + 64));
      const int sums = live * 32 * p.warps * 4;
      bool fits = false;
      for (p.stages = 4; p.stages >= 2 && !fits; p.stages -= !fits)
        for (p.buffers = 2; p.buffers >= 1 && !fits; p.buffers -= !fits) {
          p.sums = p.rings + p.warps * p.stages * BYTES;
          p.bytes = p.sums + p.buffers * sums;
          fits = p.bytes <= limit[way];
        }
      if (!fits) continue;
      for (p.wk = 1; p.warps % p.wk == 0 && p.wk <= p.slice; p.wk *= 2) {
        p.tiles = (s.pairs + p.warps / p.wk - 1) / (p.warps / p.wk);
        p.clusters = std::min(p.tiles, std::max(1, resident[way] * at_once[log] / p.passes));
        const int rounds = (p.tiles + p.clusters - 1) / p.clusters, each = (p.slice + p.wk - 1) / p.wk, ctas = p.clusters * p.cluster * p.passes;
        const int room = at_once[log] * p.cluster, on_sm = std::min(resident[way], (ctas + room - 1) / room);
        const double hbm = BYTES / 24.0 / p.passes * std::min(1.0, (double)ctas / SM / on_sm);
        const double rate = std::min(2.6, 0.17 * p.warps * on_sm);
        const double unit = std::max(p.warps * on_sm * std::max(hbm, std::max(issue / rate, products)), std::max(350.0, 1100.0 / (p.stages - 1)));
        const double fill = 1500 + (double)live * p.slice * 16 / 32 * (P == 1 ? 20 : 100) * on_sm / rate;
        const double waves = (double)((ctas + on_sm * room - 1) / (on_sm * room));
        const double join = p.cluster > 1 ? 100.0 * std::max(0, p.cluster * p.wk - 16) : 0.0;
        const double time = waves * (fill + rounds * each * unit + first[log] + join + (rounds - 1) * more[log]);
        if (best < 0 || time < best) { best = time; *out = p; }
      }
    }
  return best >= 0;
}

template <typename T, int NT, int GROUP>
cudaError_t ql_launch(const T* x, long long ld_x, const void* packed, T* y, long long ld_y, int rows, const QlShape& s, cudaStream_t st) {
  // a plan depends on the sizes alone: a thread keeps the last few
  struct Known { int d_in, d_out, rows; QlPlan plan; };
  static thread_local Known known[16] = {};
  Known& last = known[(unsigned)(s.d_in * 31 + s.d_out * 7 + rows) % 16];
  if (last.rows != rows || last.d_in != s.d_in || last.d_out != s.d_out) {
    QlPlan made;
    int live = std::min(rows, NT * 8);
    while (!ql_plan<T, NT, GROUP>(s, rows, live, &made)) {
      if (live == 1) return cudaErrorInvalidConfiguration;   // not reached: d_in is at most QL_MAX_IN
      live = (live + 1) / 2;
    }
    last = Known{s.d_in, s.d_out, rows, made};
  }
  const QlPlan plan = last.plan;
  auto kernel = q4_linear_kernel<T, NT, GROUP>;
  static std::atomic<unsigned long long> raised{0};   // devices on which the kernel's shared-memory limit has been raised
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  const unsigned long long bit = 1ull << (device & 63);
  if (!(raised.load(std::memory_order_relaxed) & bit)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
    if (e != cudaSuccess) return e;
    raised.fetch_or(bit, std::memory_order_relaxed);
  }
  return launch_following(kernel, (unsigned)(plan.clusters * plan.passes * plan.cluster), plan.cluster, plan.warps * 32, plan.bytes, st, x, ld_x,
                          (const unsigned char*)packed, y, ld_y, rows, s, plan);
}

template <typename T, int GROUP>
cudaError_t ql_dispatch(const void* x, long long ld_x, const void* packed, void* y, long long ld_y, int rows, const QlShape& s, cudaStream_t st) {
  const T* xt = (const T*)x;
  T* yt = (T*)y;
  return rows <= 8 ? ql_launch<T, 1, GROUP>(xt, ld_x, packed, yt, ld_y, rows, s, st) : ql_launch<T, 2, GROUP>(xt, ld_x, packed, yt, ld_y, rows, s, st);
}
template <typename T>
cudaError_t ql_dispatch(const void* x, long long ld_x, const void* packed, void* y, long long ld_y, int rows, const QlShape& s, cudaStream_t st) {
  return s.group == 32   ? ql_dispatch<T, 32>(x, ld_x, packed, y, ld_y, rows, s, st)
         : s.group == 64 ? ql_dispatch<T, 64>(x, ld_x, packed, y, ld_y, rows, s, st)
                         : ql_dispatch<T, 128>(x, ld_x, packed, y, ld_y, rows, s, st);
}

int ql_blocks(long long work) { return (int)std::min<long long>((work + 255) / 256, 148 * 16); }

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

int64_t q4_linear_packed_bytes(int32_t d_out, int32_t d_in, int32_t group) {
  if (!ql_sizes_ok(d_out, d_in, group)) return 0;
  const QlShape s = ql_shape(d_out, d_in, group);
  return ql_bytes(s);
}

#define QL_CHECK(packed)                                                                                                                  \
  do {                                                                                                                                    \
    if (!ql_sizes_ok(d_out, d_in, group))                                                                                                 \
      return ql_fail(message, message_len, MOE_INVALID_CONFIG, "InvalidConfig: d_in is a multiple of the group, which is 32, 64 or 128"); \
    if ((packed) == nullptr || reinterpret_cast<uintptr_t>(packed) % 16)                                                                  \
      return ql_fail(message, message_len, MOE_INVALID_INPUT, "InvalidInput: the packed matrix is null or not 16-byte aligned");         \
  } while (0)

int32_t q4_linear_pack(const int8_t* codes, const void* scales, void* packed, int32_t d_out, int32_t d_in, int32_t group, void* stream,
                       char* message, int32_t message_len) {
  QL_CHECK(packed);
  if (!codes || !scales) return ql_fail(message, message_len, MOE_INVALID_INPUT, "InvalidInput: null buffer");
  const QlShape s = ql_shape(d_out, d_in, group);
  ql_pack_kernel<<<ql_blocks((long long)s.pairs * 32 * s.units * QL_CHANNELS / 8), 256, 0, (cudaStream_t)stream>>>(codes, (const bf16*)scales,
                                                                                                                (unsigned char*)packed, s);
  count_launch();
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? MOE_OK : ql_fail(message, message_len, MOE_CUDA_ERROR, cudaGetErrorString(e));
}

int32_t q4_linear_quantize(const float* weights, void* packed, int32_t d_out, int32_t d_in, int32_t group, void* stream, char* message,
                           int32_t message_len) {
  QL_CHECK(packed);
  if (!weights) return ql_fail(message, message_len, MOE_INVALID_INPUT, "InvalidInput: null buffer");
  const QlShape s = ql_shape(d_out, d_in, group);
  ql_quantize_kernel<<<ql_blocks((long long)s.pairs * 32 * s.units * QL_CHANNELS / group), 256, 0, (cudaStream_t)stream>>>(weights, (unsigned char*)packed, s);
  count_launch();
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? MOE_OK : ql_fail(message, message_len, MOE_CUDA_ERROR, cudaGetErrorString(e));
}

int32_t q4_linear_dequantize(const void* packed, float* weights, int32_t d_out, int32_t d_in, int32_t group, void* stream, char* message,
                             int32_t message_len) {
  QL_CHECK(packed);
  if (!weights) return ql_fail(message, message_len, MOE_INVALID_INPUT, "InvalidInput: null buffer");
  const QlShape s = ql_shape(d_out, d_in, group);
  ql_dequantize_kernel<<<ql_blocks((long long)d_out * d_in), 256, 0, (cudaStream_t)stream>>>((const unsigned char*)packed, weights, s);
  count_launch();
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? MOE_OK : ql_fail(message, message_len, MOE_CUDA_ERROR, cudaGetErrorString(e));
}

int32_t q4_linear_forward(const void* x, int64_t ld_x, const void* packed, void* y, int64_t ld_y, int32_t rows, int32_t d_in,
                          int32_t d_out, int32_t group, int32_t precision, void* stream, char* message, int32_t message_len) {
  if (precision != MOE_PRECISION_F32 && precision != MOE_PRECISION_BF16)
    return ql_fail(message, message_len, MOE_INVALID_CONFIG, "InvalidConfig: activations are f32 or bf16");
  QL_CHECK(packed);
  const int elem = precision == MOE_PRECISION_BF16 ? 2 : 4;
  if (rows < 0 || rows > 65535 || ld_x < d_in || ld_y < d_out)
    return ql_fail(message, message_len, MOE_INVALID_INPUT, "InvalidInput: rows >= 0, ld_x >= d_in and ld_y >= d_out");
  if (rows == 0) return MOE_OK;
  if (!x || !y) return ql_fail(message, message_len, MOE_INVALID_INPUT, "InvalidInput: null buffer");
  if (reinterpret_cast<uintptr_t>(x) % 16 || (rows > 1 && (ld_x * elem) % 16) || reinterpret_cast<uintptr_t>(y) % elem)
    return ql_fail(message, message_len, MOE_INVALID_INPUT, "InvalidInput: rows of x start on 16-byte boundaries");
  // x is read while y is written
  if (rows_overlap(x, (long long)ld_x * elem, y, (long long)ld_y * elem, (long long)d_in * elem, (long long)d_out * elem, rows))
    return ql_fail(message, message_len, MOE_INVALID_INPUT, "InvalidInput: y overlaps x");
  const QlShape s = ql_shape(d_out, d_in, group);
  const cudaError_t e = precision == MOE_PRECISION_BF16 ? ql_dispatch<bf16>(x, ld_x, packed, y, ld_y, rows, s, (cudaStream_t)stream)
                                                        : ql_dispatch<float>(x, ld_x, packed, y, ld_y, rows, s, (cudaStream_t)stream);
  return e == cudaSuccess ? MOE_OK : ql_fail(message, message_len, MOE_CUDA_ERROR, cudaGetErrorString(e));
}

}  // extern "C"
