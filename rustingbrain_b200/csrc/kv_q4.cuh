// The 4-bit side of the KV cache (kv_q4.cu), driven by kv_attention.cu.
#pragma once
#include "common.cuh"

namespace moe {
namespace q4 {

constexpr int PAGE = 64;               // positions of one sequence and kv head that lie together
constexpr int GROUP = 32;              // channels that share a step and a base
constexpr int CLUSTER = 8;             // slices that one cluster can join

inline long long page_bytes(int head_dim) { return 80ll * head_dim; }   // two codes of 4 bits and 2 x 4 bytes per 32 channels, 64 times
inline long long head_pages(int capacity) { return (capacity + PAGE - 1) / PAGE; }
inline bool head_dim_ok(int hd) { return hd == 32 || hd == 64 || hd == 128 || hd == 256; }

struct Cache {
  unsigned char* pages;                // [sequence][kv head][page], page_bytes each
  int* lengths;                        // [sequence]
  int* full;                           // [sequence]: a step found no room
  int* skipped;                        // [sequence]: rows of the steps skipped since the last one that was taken
  int* tickets;                        // [sequence], zero between calls
  const float *cos_t, *sin_t;          // [position][head_dim / 2]
  int H, Hkv, HD, cap, rope;
};

// cos and sin of position * base^(-2 c / head_dim), the angles in 64 bits
cudaError_t launch_tables(float* cos_t, float* sin_t, int positions, int head_dim, float base, cudaStream_t st);

// Rotates, quantises and stores rows new keys and values of each sequence behind its length; lengths stay as they are.
cudaError_t launch_append(const Cache& c, const bf16* k, const bf16* v, int first, int n_seq, int rows, cudaStream_t st);

// Queries that one pass over the cache serves, per kv head.
int queries_per_pass(int head_dim, int queries);
// CTAs of the step's kernel that an SM holds at once.  Asked once per device and kind of kernel, which also raises the kernel's limit of
// shared memory: a step is launched only after this.
int ctas_per_sm(int head_dim, int queries, int device);
// One attention step over slices of at least `slice` pages (more where a sequence would need more than `splits` of them); it writes merged and
// advances the lengths.  With append set (only if rows * group fit one pass) it stores the new rows itself.  part null: the slices of a
// head are one cluster (splits <= CLUSTER); otherwise [n_seq * rows, H, splits, HD + 2] floats that a second launch joins.
cudaError_t launch_attention(const Cache& c, const bf16* q, const bf16* k, const bf16* v, int first, int n_seq, int rows, int splits, int slice, bool append,
                             float scale_log2, bf16* merged, float* part, cudaStream_t st);

// Values of `count` positions of each of n_seq sequences as f32 [n_seq * count, Hkv * HD]: positions from .. from + count - 1, or the
// newest `count` when from < 0.  Positions that are not held read 0.
cudaError_t launch_values(const Cache& c, int first, int n_seq, int from, int count, float* keys, float* values, cudaStream_t st);

}  // namespace q4
}  // namespace moe
