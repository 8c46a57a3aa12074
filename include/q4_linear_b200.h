/* C ABI of a linear layer whose weights are 4-bit codes with one scale per group of input channels (libmoe_b200.so, sm_100a): the
 * projections around the KV cache and the output head of a decode step, where the weights' bytes are the time.  It stands beside the int8
 * per-channel expert weights of moe_b200.h (reference quantization.rs, Linear::forward in linear.rs).
 *
 *   y[r, n] = sum_k x[r, k] * w[n, k],    w[n, k] = scale[n, k / group] * code[n, k]
 *
 * code is -8 .. 7, scale a bf16 number, group 32, 64 or 128 input channels; d_in is a multiple of the group and at most 65536, d_out anything.
 * x and y are both f32 (MOE_PRECISION_F32) or both bf16 (MOE_PRECISION_BF16).  Products of codes and activations are exact, whatever the
 * activations' sizes (below 2^-110, f32 ones lose their last bits); sums are f32, those of 16 channels on the tensor cores, which cut the terms off at
 * about 2^-23 of the largest of them; a group's sum is scaled in f32 and y rounded once.  The order of the sums depends on the sizes only, so
 * results do not depend on the run.  A channel whose code is 0 adds exactly 0.  An infinity or a NaN of x or of a scale appears in the outputs it takes
 * part in (0 times an infinity is NaN).
 *
 * Meant for decode batches: 16 rows at a time (fewer where d_in is very large), more rows are passes side by side over the same weights.
 *
 * Stateless: all pointers are device pointers of the current device, owned by the caller; nothing is allocated, no scratch is kept, every
 * call can be captured into a CUDA graph, and calls on different streams do not meet.  Status codes are the moe_status values of
 * moe_b200.h; on failure `message` (optional) receives the reason.
 */
#ifndef Q4_LINEAR_B200_H
#define Q4_LINEAR_B200_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Size of the buffer that holds a packed matrix (codes and scales), or 0 for sizes that are refused. */
int64_t q4_linear_packed_bytes(int32_t d_out, int32_t d_in, int32_t group);

/* codes [d_out, d_in] i8 and scales [d_out, d_in / group] bf16 into `packed` (16-byte aligned).  Of a code the low four bits are taken. */
int32_t q4_linear_pack(const int8_t* codes, const void* scales, void* packed, int32_t d_out, int32_t d_in, int32_t group, void* stream,
                       char* message, int32_t message_len);

/* Quantises weights [d_out, d_in] f32: scale = bf16(max |w| / 7) of the group, code = round(w / scale) to even, clamped to -8 .. 7
 * (0 where the scale is 0).  A group with a NaN or an infinity gets a NaN scale. */
int32_t q4_linear_quantize(const float* weights, void* packed, int32_t d_out, int32_t d_in, int32_t group, void* stream, char* message,
                           int32_t message_len);

/* What the matrix stands for: weights [d_out, d_in] f32. */
int32_t q4_linear_dequantize(const void* packed, float* weights, int32_t d_out, int32_t d_in, int32_t group, void* stream, char* message,
                             int32_t message_len);

/* x rows are ld_x elements apart and start on 16-byte boundaries; y rows are ld_y elements apart.  y does not overlap x
 * (InvalidInput), though their rows may lie between one another.
 * rows is at most 65535; rows == 0 is a call that does nothing. */
int32_t q4_linear_forward(const void* x, int64_t ld_x, const void* packed, void* y, int64_t ld_y, int32_t rows, int32_t d_in,
                          int32_t d_out, int32_t group, int32_t precision, void* stream, char* message, int32_t message_len);

#ifdef __cplusplus
}
#endif
#endif
