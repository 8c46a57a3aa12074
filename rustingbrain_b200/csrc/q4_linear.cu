// Linear layer with 4-bit weights (the ABI of include/q4_linear_b200.h).
//
// For a decode batch the bytes of the weights are the time, so the layout is made for one pass over them: a block of 16 outputs x 64
// input channels is 512 bytes, 16 for each lane of a warp, in the order in which the lane needs them as the A operand of mma.sync m16n8k16
// (the outputs are the 16 rows, the batch rows the 8 columns).  A lane's 32-bit word holds 8 consecutive channels of one output;
// since the channels of a product may come in any order, the activations' 8 channels are one 16-byte shared load of the B operand.
//
// A code becomes a bf16 number by placing its four bits, plus 8, behind the exponent of 128 and subtracting 136: exact.  The products of a
// group are summed by the tensor cores in f32 and the group's scale is applied to that sum, so neither code nor scale is ever rounded
// and f32 activations lose nothing either: they are cut into three bf16 numbers that add up to them.
//
// The reduction axis is split over the warps of a CTA and over the CTAs of a cluster, whose partial sums meet in (distributed)
// shared memory, always in the same order: one launch, no workspace.

#include <cooperative_groups.h>
#include <algorithm>
#include <atomic>
#include <cstdio>

#include "../../include/moe_b200.h"
#include "../../include/q4_linear_b200.h"
#include "common.cuh"

namespace cg = cooperative_groups;

namespace moe {
namespace {

constexpr int QL_WARPS = 8, QL_THREADS = QL_WARPS * 32;
constexpr int QL_MT = 2;                 // 16-output blocks per warp: they share the B operand
constexpr int QL_AHEAD = 4;              // weight blocks in flight per warp and 16 outputs
constexpr int QL_ROWS = 64;              // batch rows per pass
constexpr int QL_MAX_CLUSTER = 8;
constexpr int QL_SMEM = 64 * 1024;       // for the activations of a chunk; one unit of 64 f32 rows needs more
constexpr int QL_SMEM_MAX = 3 * QL_ROWS * (QL_AHEAD * 128 + 64);

struct QlShape {
  int d_in, d_out, group, kblocks, mtiles, sgroups;   // 64-channel blocks, 16-output blocks (padded to QL_MT), scale groups per output
};
inline QlShape ql_shape(int d_out, int d_in, int group) {
  QlShape s;
  s.d_in = d_in; s.d_out = d_out; s.group = group;
  s.kblocks = (d_in + 63) / 64;
  s.mtiles = (d_out / 16 + (d_out % 16 != 0) + QL_MT - 1) / QL_MT * QL_MT;
  s.sgroups = s.kblocks * 64 / group;
  return s;
}
inline long long ql_code_bytes(const QlShape& s) { return (long long)s.mtiles * s.kblocks * 512; }
inline long long ql_scale_bytes(const QlShape& s) { return (long long)s.mtiles * s.sgroups * 32; }

// Word of output n (of its 16-block) and 32-channel group g (of the 64-channel block) for channels 8 * tig .. + 7, in 32-bit units
// from the block's start; inside it channel 2 i + e is nibble i + 4 e.
__host__ __device__ inline int ql_word(int n, int g, int tig) { return ((n & 7) * 4 + tig) * 4 + 2 * g + (n >> 3); }
__host__ __device__ inline int ql_nibble(int c) { return ((c & 7) >> 1) + 4 * (c & 1); }

// ---- packing (once per matrix) ----
__global__ void ql_pack_kernel(const int8_t* __restrict__ codes, const bf16* __restrict__ scales, uint32_t* __restrict__ words,
                               bf16* __restrict__ packed_scales, QlShape s) {
  const long long words_total = (long long)s.mtiles * s.kblocks * 128, scales_total = (long long)s.mtiles * s.sgroups * 16;
  const int groups = s.d_in / s.group;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < words_total + scales_total; i += (long long)gridDim.x * blockDim.x) {
    if (i < words_total) {
      const int word = (int)(i & 127), lane = word >> 2, g = (word >> 1) & 1, hi = word & 1;
      const long long block = i >> 7;
      const int mt = (int)(block / s.kblocks), kb = (int)(block - (long long)mt * s.kblocks);
      const int n = mt * 16 + (lane >> 2) + 8 * hi, c0 = kb * 64 + g * 32 + (lane & 3) * 8;
      uint32_t w = 0;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const int code = n < s.d_out && c0 + c < s.d_in ? codes[(long long)n * s.d_in + c0 + c] : 0;
        w |= ((uint32_t)(code + 8) & 15u) << (4 * ql_nibble(c));
      }
      words[i] = w;
    } else {
      const long long j = i - words_total;
      const int slot = (int)(j & 15), gid = slot >> 1, hi = slot & 1;
      const long long at = j >> 4;
      const int mt = (int)(at / s.sgroups), grp = (int)(at - (long long)mt * s.sgroups), n = mt * 16 + gid + 8 * hi;
      packed_scales[j] = n < s.d_out && grp < groups ? scales[(long long)n * groups + grp] : __float2bfloat16_rn(0.f);
    }
  }
}

// one thread per (output, group), padding included
__global__ void ql_quantize_kernel(const float* __restrict__ weights, uint32_t* __restrict__ words, bf16* __restrict__ packed_scales, QlShape s) {
  const long long total = (long long)s.mtiles * 16 * s.sgroups;
  const int groups = s.d_in / s.group;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x) {
    const int n = (int)(i / s.sgroups), grp = (int)(i - (long long)n * s.sgroups), mt = n >> 4, nl = n & 15;
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
      const int k = grp * s.group + c0, kb = k >> 6, g = (k >> 5) & 1, tig = (k >> 3) & 3;
      uint32_t word = 0;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        int code = 0;
        if (live && f > 0.f) code = (int)fminf(fmaxf(rintf(__fdiv_rn(w[c0 + c], f)), -8.f), 7.f);
        word |= ((uint32_t)(code + 8) & 15u) << (4 * ql_nibble(c));
      }
      words[((long long)mt * s.kblocks + kb) * 128 + ql_word(nl, g, tig)] = word;
    }
    packed_scales[((long long)mt * s.sgroups + grp) * 16 + (nl & 7) * 2 + (nl >> 3)] = scale;
  }
}

__global__ void ql_dequantize_kernel(const uint32_t* __restrict__ words, const bf16* __restrict__ packed_scales, float* __restrict__ weights, QlShape s) {
  const long long total = (long long)s.d_out * s.d_in;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x) {
    const int n = (int)(i / s.d_in), k = (int)(i - (long long)n * s.d_in), mt = n >> 4, nl = n & 15;
    const uint32_t w = words[((long long)mt * s.kblocks + (k >> 6)) * 128 + ql_word(nl, (k >> 5) & 1, (k >> 3) & 3)];
    const float code = (float)((int)((w >> (4 * ql_nibble(k))) & 15u) - 8);
    weights[i] = code * __bfloat162float(packed_scales[((long long)mt * s.sgroups + k / s.group) * 16 + (nl & 7) * 2 + (nl >> 3)]);
  }
}

// ---- the product ----
__device__ __forceinline__ void ql_mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// codes i and i + 4 of a word as two bf16 numbers, -8 .. 7
template <int I>
__device__ __forceinline__ uint32_t ql_pair(uint32_t w) {
  const uint32_t v = ((w >> (4 * I)) & 0x000f000fu) | 0x43004300u;
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), __float2bfloat162_rn(136.f));
  return *reinterpret_cast<const uint32_t*>(&r);
}
template <typename T> struct QlPieces { static constexpr int N = 1; };
template <> struct QlPieces<float> { static constexpr int N = 3; };

// An f32 number as three bf16 numbers that add up to it, each the leading 8 bits of what is left.
__device__ __forceinline__ void ql_split(float x, uint16_t* p) {
  if (!(fabsf(x) <= 3.4028234663852886e38f)) {
    p[0] = x != x ? 0x7fc0 : (uint16_t)(__float_as_uint(x) >> 16);
    p[1] = p[2] = 0;
    return;
  }
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const uint32_t top = __float_as_uint(x) & 0xffff0000u;
    p[i] = (uint16_t)(top >> 16);
    x -= __uint_as_float(top);
  }
}

// Shared memory: the activations of a chunk of the reduction, [piece][row][chunk * 64 + 32] bf16 (the 64 extra bytes a row keep the 16-byte
// loads of a warp off each other's banks), then the warps' partial sums in the same place.
template <typename T, int NT, int SPB>
__global__ void __launch_bounds__(QL_THREADS, NT <= 2 ? 2 : 1)
q4_linear_kernel(const T* __restrict__ x, long long ld_x, const uint4* __restrict__ codes, const uint32_t* __restrict__ scales, T* __restrict__ y,
                 long long ld_y, int rows_total, QlShape s, int wk_count, int cluster, int chunk) {
  constexpr int P = QlPieces<T>::N, MT = QL_MT, U = QL_AHEAD;
  extern __shared__ __align__(16) unsigned char ql_sm[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
  const int wn_count = QL_WARPS / wk_count, wk = warp % wk_count, wn = warp / wk_count;
  const int tile = blockIdx.x / cluster, rank = blockIdx.x - tile * cluster;
  const int mt0 = (tile * wn_count + wn) * MT;
  const bool live = mt0 < s.mtiles;                  // mtiles is a multiple of MT
  const int row0 = blockIdx.y * QL_ROWS, rows = min(rows_total - row0, NT * 8);
  const int kbeg = (int)((long long)s.kblocks * rank / cluster), kend = (int)((long long)s.kblocks * (rank + 1) / cluster);
  const int pitch = chunk * 128 + 64, plane = NT * 8 * pitch;        // bytes
  const uint4* cw = codes + (long long)mt0 * s.kblocks * 32 + lane;
  const uint32_t* sw = scales + (long long)mt0 * s.sgroups * 8 + gid;
  const int per_group = s.group == 128 ? 1 : 0;      // shift from a 64-channel block to its scale (SPB == 1)

  float acc[MT][NT][4];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[m][n][0] = acc[m][n][1] = acc[m][n][2] = acc[m][n][3] = 0.f;

  uint4 w[U][MT];
  uint32_t sc[U][MT][SPB];
  auto fetch = [&](int u, int kb) {
    if (live && kb < kend) {
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        w[u][m] = __ldg(cw + ((long long)m * s.kblocks + kb) * 32);
#pragma unroll
        for (int g = 0; g < SPB; ++g)
          sc[u][m][g] = __ldg(sw + ((long long)m * s.sgroups + (SPB == 2 ? 2 * kb + g : kb >> per_group)) * 8);
      }
    }
  };
#pragma unroll
  for (int u = 0; u < U; ++u) fetch(u, kbeg + wk + u * wk_count);

  for (int c0 = kbeg; c0 < kend; c0 += chunk) {      // chunk is a multiple of U * wk_count
    __syncthreads();                                 // the chunk before has been used
    {
      const int blocks = min(chunk, kend - c0), parts = blocks * 8;            // 8 channels at a time
      for (int i = threadIdx.x; i < rows * parts; i += QL_THREADS) {
        const int r = i / parts, c = i - r * parts, k = c0 * 64 + c * 8;
        const T* src = x + (row0 + r) * ld_x + k;
        unsigned char* dst = ql_sm + r * pitch + c * 16;
        if constexpr (P == 1) {
          *reinterpret_cast<uint4*>(dst) = k < s.d_in ? __ldg(reinterpret_cast<const uint4*>(src)) : make_uint4(0, 0, 0, 0);
        } else {
          float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
          if (k < s.d_in) {
            *reinterpret_cast<float4*>(f) = __ldg(reinterpret_cast<const float4*>(src));
            *reinterpret_cast<float4*>(f + 4) = __ldg(reinterpret_cast<const float4*>(src) + 1);
          }
          uint16_t p[8][3];
#pragma unroll
          for (int j = 0; j < 8; ++j) ql_split(f[j], p[j]);
#pragma unroll
          for (int q = 0; q < 3; ++q)
            *reinterpret_cast<uint4*>(dst + q * plane) =
                make_uint4(p[0][q] | (uint32_t)p[1][q] << 16, p[2][q] | (uint32_t)p[3][q] << 16, p[4][q] | (uint32_t)p[5][q] << 16,
                           p[6][q] | (uint32_t)p[7][q] << 16);
        }
      }
    }
    __syncthreads();
    if (!live) continue;
    const int end = min(kend, c0 + chunk);
    for (int kb0 = c0 + wk; kb0 < end; kb0 += U * wk_count) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int kb = kb0 + u * wk_count;
        if (kb < end) {
          const unsigned char* xs = ql_sm + gid * pitch + (kb - c0) * 128 + tig * 16;
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            uint32_t a[MT][2][4];
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              const uint32_t lo = g ? w[u][m].z : w[u][m].x, hi = g ? w[u][m].w : w[u][m].y;
              a[m][0][0] = ql_pair<0>(lo); a[m][0][1] = ql_pair<0>(hi); a[m][0][2] = ql_pair<1>(lo); a[m][0][3] = ql_pair<1>(hi);
              a[m][1][0] = ql_pair<2>(lo); a[m][1][1] = ql_pair<2>(hi); a[m][1][2] = ql_pair<3>(lo); a[m][1][3] = ql_pair<3>(hi);
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              float part[MT][4];
#pragma unroll
              for (int m = 0; m < MT; ++m) part[m][0] = part[m][1] = part[m][2] = part[m][3] = 0.f;
#pragma unroll
              for (int q = 0; q < P; ++q) {
                const uint4 b = *reinterpret_cast<const uint4*>(xs + q * plane + n * 8 * pitch + g * 64);
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                  ql_mma(part[m], a[m][0], b.x, b.y);
                  ql_mma(part[m], a[m][1], b.z, b.w);
                }
              }
#pragma unroll
              for (int m = 0; m < MT; ++m) {
                const uint32_t v = sc[u][m][SPB == 2 ? g : 0];
                const float s0 = __uint_as_float(v << 16), s1 = __uint_as_float(v & 0xffff0000u);
                acc[m][n][0] = fmaf(s0, part[m][0], acc[m][n][0]);
                acc[m][n][1] = fmaf(s0, part[m][1], acc[m][n][1]);
                acc[m][n][2] = fmaf(s1, part[m][2], acc[m][n][2]);
                acc[m][n][3] = fmaf(s1, part[m][3], acc[m][n][3]);
              }
            }
          }
        }
        fetch(u, kb + U * wk_count);
      }
    }
  }

  // ---- add the partial sums of the warps and of the cluster's CTAs ----
  constexpr int TN = MT * 16;
  float* red = reinterpret_cast<float*>(ql_sm);      // [wk][row][wn * TN + output]
  const int width = wn_count * TN;
  __syncthreads();
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        red[(wk * NT * 8 + n * 8 + 2 * tig + (e & 1)) * width + wn * TN + m * 16 + gid + 8 * (e >> 1)] = acc[m][n][e];
  cg::cluster_group cl = cg::this_cluster();
  if (cluster > 1) cl.sync(); else __syncthreads();
  const int n0 = tile * width;
  for (int i = rank * QL_THREADS + threadIdx.x; i < rows * width; i += cluster * QL_THREADS) {
    const int r = i / width, n = i - r * width;
    if (n0 + n >= s.d_out) continue;
    float v = 0.f;
    for (int c = 0; c < cluster; ++c) {
      const float* part = cluster > 1 ? cl.map_shared_rank(red, c) : red;
      for (int k = 0; k < wk_count; ++k) v += part[(k * NT * 8 + r) * width + n];
    }
    y[(row0 + r) * ld_y + n0 + n] = from_f32<T>(v);
  }
  if (cluster > 1) cl.sync();                        // nobody leaves while its sums are being read
}

int ql_fail(char* msg, int len, int code, const char* text) {
  if (msg && len > 0) snprintf(msg, len, "%s", text);
  return code;
}

bool ql_sizes_ok(int d_out, int d_in, int group) {
  return d_out > 0 && d_in > 0 && (group == 32 || group == 64 || group == 128) && d_in % group == 0 && d_in <= (1 << 24) && d_out <= (1 << 28);
}

template <typename T, int NT, int SPB>
cudaError_t ql_launch(const T* x, long long ld_x, const void* packed, T* y, long long ld_y, int rows, const QlShape& s, cudaStream_t st) {
  constexpr int P = QlPieces<T>::N;
  // Warps along the reduction: many for few rows (less to join), few for many rows (their activations fill shared memory).
  int wk = NT == 1 ? 4 : NT == 2 ? 2 : 1;
  while (wk > 1 && s.kblocks < wk) wk /= 2;
  const int tiles = (s.mtiles / QL_MT + QL_WARPS / wk - 1) / (QL_WARPS / wk);
  int cluster = 1;
  while (cluster < QL_MAX_CLUSTER && tiles * cluster < 2 * 148 && s.kblocks >= cluster * 2 * wk * 2) cluster *= 2;
  const int slice = (s.kblocks + cluster - 1) / cluster, unit = QL_AHEAD * wk;
  // the chunk of the reduction whose activations are in shared memory at a time
  int chunk = (slice + unit - 1) / unit * unit;
  while (chunk > unit && P * NT * 8 * (chunk * 128 + 64) > QL_SMEM) chunk -= unit;
  const int smem = std::max(P * NT * 8 * (chunk * 128 + 64), QL_WARPS * QL_MT * 16 * NT * 8 * 4);
  auto kernel = q4_linear_kernel<T, NT, SPB>;
  static std::atomic<unsigned long long> raised{0};   // devices on which the kernel's shared-memory limit has been raised
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  const unsigned long long bit = 1ull << (device & 63);
  if (!(raised.load(std::memory_order_relaxed) & bit)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, QL_SMEM_MAX);
    if (e != cudaSuccess) return e;
    raised.fetch_or(bit, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(tiles * cluster), (unsigned)((rows + QL_ROWS - 1) / QL_ROWS));
  cfg.blockDim = dim3(QL_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const uint4* codes = (const uint4*)packed;
  const uint32_t* scales = (const uint32_t*)((const char*)packed + ql_code_bytes(s));
  count_launch();
  return cudaLaunchKernelEx(&cfg, kernel, x, ld_x, codes, scales, y, ld_y, rows, s, wk, cluster, chunk);
}

template <typename T>
cudaError_t ql_dispatch(const void* x, long long ld_x, const void* packed, void* y, long long ld_y, int rows, const QlShape& s, cudaStream_t st) {
  const T* xt = (const T*)x;
  T* yt = (T*)y;
#define QL_GO(NT) (s.group == 32 ? ql_launch<T, NT, 2>(xt, ld_x, packed, yt, ld_y, rows, s, st) : ql_launch<T, NT, 1>(xt, ld_x, packed, yt, ld_y, rows, s, st))
  if (rows <= 8) return QL_GO(1);
  if (rows <= 16) return QL_GO(2);
  if (rows <= 32) return QL_GO(4);
  return QL_GO(8);
#undef QL_GO
}

int ql_blocks(long long work) { return (int)std::min<long long>((work + 255) / 256, 148 * 16); }

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

int64_t q4_linear_packed_bytes(int32_t d_out, int32_t d_in, int32_t group) {
  if (!ql_sizes_ok(d_out, d_in, group)) return 0;
  const QlShape s = ql_shape(d_out, d_in, group);
  return ql_code_bytes(s) + ql_scale_bytes(s);
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
  ql_pack_kernel<<<ql_blocks((long long)s.mtiles * (s.kblocks * 128ll + s.sgroups * 16ll)), 256, 0, (cudaStream_t)stream>>>(
      codes, (const bf16*)scales, (uint32_t*)packed, (bf16*)((char*)packed + ql_code_bytes(s)), s);
  count_launch();
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? MOE_OK : ql_fail(message, message_len, MOE_CUDA_ERROR, cudaGetErrorString(e));
}

int32_t q4_linear_quantize(const float* weights, void* packed, int32_t d_out, int32_t d_in, int32_t group, void* stream, char* message,
                           int32_t message_len) {
  QL_CHECK(packed);
  if (!weights) return ql_fail(message, message_len, MOE_INVALID_INPUT, "InvalidInput: null buffer");
  const QlShape s = ql_shape(d_out, d_in, group);
  ql_quantize_kernel<<<ql_blocks((long long)s.mtiles * 16 * s.sgroups), 256, 0, (cudaStream_t)stream>>>(
      weights, (uint32_t*)packed, (bf16*)((char*)packed + ql_code_bytes(s)), s);
  count_launch();
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? MOE_OK : ql_fail(message, message_len, MOE_CUDA_ERROR, cudaGetErrorString(e));
}

int32_t q4_linear_dequantize(const void* packed, float* weights, int32_t d_out, int32_t d_in, int32_t group, void* stream, char* message,
                             int32_t message_len) {
  QL_CHECK(packed);
  if (!weights) return ql_fail(message, message_len, MOE_INVALID_INPUT, "InvalidInput: null buffer");
  const QlShape s = ql_shape(d_out, d_in, group);
  ql_dequantize_kernel<<<ql_blocks((long long)d_out * d_in), 256, 0, (cudaStream_t)stream>>>(
      (const uint32_t*)packed, (const bf16*)((const char*)packed + ql_code_bytes(s)), weights, s);
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
  if (rows < 0 || rows > QL_ROWS * 65535 || ld_x < d_in || ld_y < d_out)
    return ql_fail(message, message_len, MOE_INVALID_INPUT, "InvalidInput: rows >= 0, ld_x >= d_in and ld_y >= d_out");
  if (rows == 0) return MOE_OK;
  if (!x || !y) return ql_fail(message, message_len, MOE_INVALID_INPUT, "InvalidInput: null buffer");
  if (reinterpret_cast<uintptr_t>(x) % 16 || (rows > 1 && (ld_x * elem) % 16) || reinterpret_cast<uintptr_t>(y) % elem)
    return ql_fail(message, message_len, MOE_INVALID_INPUT, "InvalidInput: rows of x start on 16-byte boundaries");
  const QlShape s = ql_shape(d_out, d_in, group);
  const cudaError_t e = precision == MOE_PRECISION_BF16 ? ql_dispatch<bf16>(x, ld_x, packed, y, ld_y, rows, s, (cudaStream_t)stream)
                                                        : ql_dispatch<float>(x, ld_x, packed, y, ld_y, rows, s, (cudaStream_t)stream);
  return e == cudaSuccess ? MOE_OK : ql_fail(message, message_len, MOE_CUDA_ERROR, cudaGetErrorString(e));
}

}  // extern "C"
