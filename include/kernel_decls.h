/* GENERATED by metaphor_amd/kernelgen.py from metaphor_amd/csrc/hipcc_src -- do not edit.
 *
 * Kernel launchers of the drop-in boundary. Every stem S exports launch_S_r16, launch_S_r32
 * and launch_S_r64 with one C signature: device pointers as void*, scalars as double, sizes
 * as len_t, the StreamContext by value as the last argument, no return value and no error
 * channel (a failure prints and exits). This is the shape of the reference's generated
 * src/cuda/kernel_decls.h:11-436; the comment above each group names what it replaces.
 * Launchers only enqueue work on the context's stream and allocate nothing.
 */
#ifndef __KERNEL_DECLS_H__
#define __KERNEL_DECLS_H__

#include "tensor_types.h"

#if defined(__cplusplus)
    #define EXTERN_C extern "C"
#else
    #define EXTERN_C extern
#endif

/* c = a + b. Replaces src/cuda/nvcc_src/addition.cu:3-29. The reference also calls this */
/* launcher in place as the reverse of add (c aliasing b, src/ops/addition.zig:67-81). */
EXTERN_C void launch_addition_r16(
  const void* a,
  const void* b,
  void* c,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_addition_r32(
  const void* a,
  const void* b,
  void* c,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_addition_r64(
  const void* a,
  const void* b,
  void* c,
  len_t N,
  StreamContext stream
);

/* dst[i,j] = src[i] + alpha*dst[i,j]. Replaces src/cuda/nvcc_src/broadcast_i_ij.cu:9-59; the */
/* reverse of reduce_ij_i calls it with alpha = 1 (src/ops/reduce.zig:123-140). */
EXTERN_C void launch_broadcast_i_ij_r16(
  const void* src,
  void* dst,
  double alpha,
  len_t m,
  len_t n,
  StreamContext stream
);
EXTERN_C void launch_broadcast_i_ij_r32(
  const void* src,
  void* dst,
  double alpha,
  len_t m,
  len_t n,
  StreamContext stream
);
EXTERN_C void launch_broadcast_i_ij_r64(
  const void* src,
  void* dst,
  double alpha,
  len_t m,
  len_t n,
  StreamContext stream
);

/* dst[i,j] = src[j] + alpha*dst[i,j]. Replaces src/cuda/nvcc_src/broadcast_j_ij.cu:9-57; the */
/* reverse of reduce_ij_j calls it with alpha = 1 (src/ops/reduce.zig:167-182). */
EXTERN_C void launch_broadcast_j_ij_r16(
  const void* src,
  void* dst,
  double alpha,
  len_t m,
  len_t n,
  StreamContext stream
);
EXTERN_C void launch_broadcast_j_ij_r32(
  const void* src,
  void* dst,
  double alpha,
  len_t m,
  len_t n,
  StreamContext stream
);
EXTERN_C void launch_broadcast_j_ij_r64(
  const void* src,
  void* dst,
  double alpha,
  len_t m,
  len_t n,
  StreamContext stream
);

/* dst = src. Replaces src/cuda/nvcc_src/copy.cu:4-47, the one vectorised kernel of the reference. */
/* Also the plain copy of known size that calibrates the HBM traffic counters. */
EXTERN_C void launch_copy_r16(
  const void* src,
  void* dst,
  len_t n,
  StreamContext stream
);
EXTERN_C void launch_copy_r32(
  const void* src,
  void* dst,
  len_t n,
  StreamContext stream
);
EXTERN_C void launch_copy_r64(
  const void* src,
  void* dst,
  len_t n,
  StreamContext stream
);

/* c = a * value. Replaces src/cuda/nvcc_src/dilate.cu:3-29; the scalar crosses as double and is */
/* narrowed to the storage type in the launcher, as there (:24). */
EXTERN_C void launch_dilate_r16(
  const void* a,
  double value,
  void* c,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_dilate_r32(
  const void* a,
  double value,
  void* c,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_dilate_r64(
  const void* a,
  double value,
  void* c,
  len_t N,
  StreamContext stream
);

/* b += a * value. Replaces src/cuda/nvcc_src/dilate_reverse.cu:3-29. */
EXTERN_C void launch_dilate_reverse_r16(
  const void* a,
  double value,
  void* b,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_dilate_reverse_r32(
  const void* a,
  double value,
  void* b,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_dilate_reverse_r64(
  const void* a,
  double value,
  void* b,
  len_t N,
  StreamContext stream
);

/* dst[i,j] = scale * table[tokens[i], j] for m tokens and a table of v rows of n elements. tokens are */
/* signed integers on the device, id_bytes (4 or 8) wide each; an id outside [0, v) (a padded place) */
/* gives a row of zeros. No reference kernel exists; the nearest is the row broadcast */
/* (src/cuda/nvcc_src/broadcast_j_ij.cu:9-57). dst must not overlap the table. */
EXTERN_C void launch_embedding_i_ij_r16(
  const void* table,
  const void* tokens,
  void* dst,
  double scale,
  len_t id_bytes,
  len_t v,
  len_t m,
  len_t n,
  StreamContext stream
);
EXTERN_C void launch_embedding_i_ij_r32(
  const void* table,
  const void* tokens,
  void* dst,
  double scale,
  len_t id_bytes,
  len_t v,
  len_t m,
  len_t n,
  StreamContext stream
);
EXTERN_C void launch_embedding_i_ij_r64(
  const void* table,
  const void* tokens,
  void* dst,
  double scale,
  len_t id_bytes,
  len_t v,
  len_t m,
  len_t n,
  StreamContext stream
);

/* table_grads[k,j] = scale * sum of dst_grads[i,j] over the places i with tokens[i] == k */
/*                    + alpha*table_grads[k,j] */
/* for every row k of the table, the ones no token names among them (alpha = 0 clears those and never */
/* reads table_grads; alpha = 1 leaves them untouched). tokens and id_bytes as in embedding_i_ij; the */
/* gradient of a padded place is not read into any sum. scratch is caller-owned workspace of */
/* mpEmbeddingReverseScratchBytes(dtype, v, m, n) bytes, 16-byte aligned; launches that may overlap in */
/* time get different workspaces. Results do not change from run to run. */
EXTERN_C void launch_embedding_i_ij_reverse_r16(
  const void* tokens,
  const void* dst_grads,
  void* table_grads,
  void* scratch,
  double scale,
  double alpha,
  len_t id_bytes,
  len_t v,
  len_t m,
  len_t n,
  StreamContext stream
);
EXTERN_C void launch_embedding_i_ij_reverse_r32(
  const void* tokens,
  const void* dst_grads,
  void* table_grads,
  void* scratch,
  double scale,
  double alpha,
  len_t id_bytes,
  len_t v,
  len_t m,
  len_t n,
  StreamContext stream
);
EXTERN_C void launch_embedding_i_ij_reverse_r64(
  const void* tokens,
  const void* dst_grads,
  void* table_grads,
  void* scratch,
  double scale,
  double alpha,
  len_t id_bytes,
  len_t v,
  len_t m,
  len_t n,
  StreamContext stream
);

/* dev_a = value. Replaces src/cuda/nvcc_src/fill.cu:4-27; seeds dL/dz = 1 on the reverse path */
/* (src/core/graph.zig:116). */
EXTERN_C void launch_fill_r16(
  void* dev_a,
  double value,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_fill_r32(
  void* dev_a,
  double value,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_fill_r64(
  void* dev_a,
  double value,
  len_t N,
  StreamContext stream
);

/* out = add(add(x0,x1),x2) in one pass: 3 reads and 1 write per element, where the reference's */
/* composition takes one launch and one temporary per op (README.md:89-97, */
/* src/ops/addition.zig:37-47). */
EXTERN_C void launch_fused_add_add_r16(
  const void* x0,
  const void* x1,
  const void* x2,
  void* out,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_fused_add_add_r32(
  const void* x0,
  const void* x1,
  const void* x2,
  void* out,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_fused_add_add_r64(
  const void* x0,
  const void* x1,
  const void* x2,
  void* out,
  len_t N,
  StreamContext stream
);

/* Reverse of out = add(add(x0,x1),x2) in one pass: every leaf gradient */
/* g_i = d out / d x_i * out_grads + alpha * g_i (the blend convention of */
/* src/cuda/nvcc_src/permutate_ij_ji.cu:37-38). alpha == 0 never reads the old gradients: */
/* 4 reads and 3 writes per element, against two read-modify-write launches per op in the */
/* reference (src/ops/hadamard.zig:65-79, src/ops/addition.zig:67-81). */
EXTERN_C void launch_fused_add_add_reverse_r16(
  const void* x0,
  const void* x1,
  const void* x2,
  const void* out_grads,
  void* g0,
  void* g1,
  void* g2,
  double alpha,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_fused_add_add_reverse_r32(
  const void* x0,
  const void* x1,
  const void* x2,
  const void* out_grads,
  void* g0,
  void* g1,
  void* g2,
  double alpha,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_fused_add_add_reverse_r64(
  const void* x0,
  const void* x1,
  const void* x2,
  const void* out_grads,
  void* g0,
  void* g1,
  void* g2,
  double alpha,
  len_t N,
  StreamContext stream
);

/* out = mul(add(x0,x1),add(x2,x3)) in one pass: 4 reads and 1 write per element, where the reference's */
/* composition takes one launch and one temporary per op (README.md:89-97, */
/* src/ops/addition.zig:37-47). */
EXTERN_C void launch_fused_hadamard_add_add_r16(
  const void* x0,
  const void* x1,
  const void* x2,
  const void* x3,
  void* out,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_fused_hadamard_add_add_r32(
  const void* x0,
  const void* x1,
  const void* x2,
  const void* x3,
  void* out,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_fused_hadamard_add_add_r64(
  const void* x0,
  const void* x1,
  const void* x2,
  const void* x3,
  void* out,
  len_t N,
  StreamContext stream
);

/* Reverse of out = mul(add(x0,x1),add(x2,x3)) in one pass: every leaf gradient */
/* g_i = d out / d x_i * out_grads + alpha * g_i (the blend convention of */
/* src/cuda/nvcc_src/permutate_ij_ji.cu:37-38). alpha == 0 never reads the old gradients: */
/* 5 reads and 4 writes per element, against two read-modify-write launches per op in the */
/* reference (src/ops/hadamard.zig:65-79, src/ops/addition.zig:67-81). */
EXTERN_C void launch_fused_hadamard_add_add_reverse_r16(
  const void* x0,
  const void* x1,
  const void* x2,
  const void* x3,
  const void* out_grads,
  void* g0,
  void* g1,
  void* g2,
  void* g3,
  double alpha,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_fused_hadamard_add_add_reverse_r32(
  const void* x0,
  const void* x1,
  const void* x2,
  const void* x3,
  const void* out_grads,
  void* g0,
  void* g1,
  void* g2,
  void* g3,
  double alpha,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_fused_hadamard_add_add_reverse_r64(
  const void* x0,
  const void* x1,
  const void* x2,
  const void* x3,
  const void* out_grads,
  void* g0,
  void* g1,
  void* g2,
  void* g3,
  double alpha,
  len_t N,
  StreamContext stream
);

/* out = relu(mul(add(x0,x1),add(x2,x3))) in one pass: 4 reads and 1 write per element, where the reference's */
/* composition takes one launch and one temporary per op (README.md:89-97, */
/* src/ops/addition.zig:37-47). */
EXTERN_C void launch_fused_relu_hadamard_add_add_r16(
  const void* x0,
  const void* x1,
  const void* x2,
  const void* x3,
  void* out,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_fused_relu_hadamard_add_add_r32(
  const void* x0,
  const void* x1,
  const void* x2,
  const void* x3,
  void* out,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_fused_relu_hadamard_add_add_r64(
  const void* x0,
  const void* x1,
  const void* x2,
  const void* x3,
  void* out,
  len_t N,
  StreamContext stream
);

/* Reverse of out = relu(mul(add(x0,x1),add(x2,x3))) in one pass: every leaf gradient */
/* g_i = d out / d x_i * out_grads + alpha * g_i (the blend convention of */
/* src/cuda/nvcc_src/permutate_ij_ji.cu:37-38). alpha == 0 never reads the old gradients: */
/* 5 reads and 4 writes per element, against two read-modify-write launches per op in the */
/* reference (src/ops/hadamard.zig:65-79, src/ops/addition.zig:67-81). */
EXTERN_C void launch_fused_relu_hadamard_add_add_reverse_r16(
  const void* x0,
  const void* x1,
  const void* x2,
  const void* x3,
  const void* out_grads,
  void* g0,
  void* g1,
  void* g2,
  void* g3,
  double alpha,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_fused_relu_hadamard_add_add_reverse_r32(
  const void* x0,
  const void* x1,
  const void* x2,
  const void* x3,
  const void* out_grads,
  void* g0,
  void* g1,
  void* g2,
  void* g3,
  double alpha,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_fused_relu_hadamard_add_add_reverse_r64(
  const void* x0,
  const void* x1,
  const void* x2,
  const void* x3,
  const void* out_grads,
  void* g0,
  void* g1,
  void* g2,
  void* g3,
  double alpha,
  len_t N,
  StreamContext stream
);

/* out = selu(add(x0,x1)) in one pass: 2 reads and 1 write per element, where the reference's */
/* composition takes one launch and one temporary per op (README.md:89-97, */
/* src/ops/addition.zig:37-47). */
EXTERN_C void launch_fused_selu_add_r16(
  const void* x0,
  const void* x1,
  void* out,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_fused_selu_add_r32(
  const void* x0,
  const void* x1,
  void* out,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_fused_selu_add_r64(
  const void* x0,
  const void* x1,
  void* out,
  len_t N,
  StreamContext stream
);

/* Reverse of out = selu(add(x0,x1)) in one pass: every leaf gradient */
/* g_i = d out / d x_i * out_grads + alpha * g_i (the blend convention of */
/* src/cuda/nvcc_src/permutate_ij_ji.cu:37-38). alpha == 0 never reads the old gradients: */
/* 3 reads and 2 writes per element, against two read-modify-write launches per op in the */
/* reference (src/ops/hadamard.zig:65-79, src/ops/addition.zig:67-81). */
EXTERN_C void launch_fused_selu_add_reverse_r16(
  const void* x0,
  const void* x1,
  const void* out_grads,
  void* g0,
  void* g1,
  double alpha,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_fused_selu_add_reverse_r32(
  const void* x0,
  const void* x1,
  const void* out_grads,
  void* g0,
  void* g1,
  double alpha,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_fused_selu_add_reverse_r64(
  const void* x0,
  const void* x1,
  const void* out_grads,
  void* g0,
  void* g1,
  double alpha,
  len_t N,
  StreamContext stream
);

/* out = selu(mul(add(x0,x1),add(x2,x3))) in one pass: 4 reads and 1 write per element, where the reference's */
/* composition takes one launch and one temporary per op (README.md:89-97, */
/* src/ops/addition.zig:37-47). */
EXTERN_C void launch_fused_selu_hadamard_add_add_r16(
  const void* x0,
  const void* x1,
  const void* x2,
  const void* x3,
  void* out,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_fused_selu_hadamard_add_add_r32(
  const void* x0,
  const void* x1,
  const void* x2,
  const void* x3,
  void* out,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_fused_selu_hadamard_add_add_r64(
  const void* x0,
  const void* x1,
  const void* x2,
  const void* x3,
  void* out,
  len_t N,
  StreamContext stream
);

/* Reverse of out = selu(mul(add(x0,x1),add(x2,x3))) in one pass: every leaf gradient */
/* g_i = d out / d x_i * out_grads + alpha * g_i (the blend convention of */
/* src/cuda/nvcc_src/permutate_ij_ji.cu:37-38). alpha == 0 never reads the old gradients: */
/* 5 reads and 4 writes per element, against two read-modify-write launches per op in the */
/* reference (src/ops/hadamard.zig:65-79, src/ops/addition.zig:67-81). */
EXTERN_C void launch_fused_selu_hadamard_add_add_reverse_r16(
  const void* x0,
  const void* x1,
  const void* x2,
  const void* x3,
  const void* out_grads,
  void* g0,
  void* g1,
  void* g2,
  void* g3,
  double alpha,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_fused_selu_hadamard_add_add_reverse_r32(
  const void* x0,
  const void* x1,
  const void* x2,
  const void* x3,
  const void* out_grads,
  void* g0,
  void* g1,
  void* g2,
  void* g3,
  double alpha,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_fused_selu_hadamard_add_add_reverse_r64(
  const void* x0,
  const void* x1,
  const void* x2,
  const void* x3,
  const void* out_grads,
  void* g0,
  void* g1,
  void* g2,
  void* g3,
  double alpha,
  len_t N,
  StreamContext stream
);

/* out = selu(mul(sub(x0,x1),x2)) in one pass: 3 reads and 1 write per element, where the reference's */
/* composition takes one launch and one temporary per op (README.md:89-97, */
/* src/ops/addition.zig:37-47). */
EXTERN_C void launch_fused_selu_hadamard_sub_r16(
  const void* x0,
  const void* x1,
  const void* x2,
  void* out,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_fused_selu_hadamard_sub_r32(
  const void* x0,
  const void* x1,
  const void* x2,
  void* out,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_fused_selu_hadamard_sub_r64(
  const void* x0,
  const void* x1,
  const void* x2,
  void* out,
  len_t N,
  StreamContext stream
);

/* Reverse of out = selu(mul(sub(x0,x1),x2)) in one pass: every leaf gradient */
/* g_i = d out / d x_i * out_grads + alpha * g_i (the blend convention of */
/* src/cuda/nvcc_src/permutate_ij_ji.cu:37-38). alpha == 0 never reads the old gradients: */
/* 4 reads and 3 writes per element, against two read-modify-write launches per op in the */
/* reference (src/ops/hadamard.zig:65-79, src/ops/addition.zig:67-81). */
EXTERN_C void launch_fused_selu_hadamard_sub_reverse_r16(
  const void* x0,
  const void* x1,
  const void* x2,
  const void* out_grads,
  void* g0,
  void* g1,
  void* g2,
  double alpha,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_fused_selu_hadamard_sub_reverse_r32(
  const void* x0,
  const void* x1,
  const void* x2,
  const void* out_grads,
  void* g0,
  void* g1,
  void* g2,
  double alpha,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_fused_selu_hadamard_sub_reverse_r64(
  const void* x0,
  const void* x1,
  const void* x2,
  const void* out_grads,
  void* g0,
  void* g1,
  void* g2,
  double alpha,
  len_t N,
  StreamContext stream
);

/* gradient_norm (alpha = 0) and gradient_scale of the same `count` tensors in one call: norm[0] gets */
/* their norm, clipped_k = grads_k * min(1, max_norm / norm[0]). Arguments and workspace as there. */
EXTERN_C void launch_gradient_clip_r16(
  const void* grads,
  const void* clipped,
  const void* sizes,
  void* norm,
  void* scratch,
  double max_norm,
  len_t count,
  StreamContext stream
);
EXTERN_C void launch_gradient_clip_r32(
  const void* grads,
  const void* clipped,
  const void* sizes,
  void* norm,
  void* scratch,
  double max_norm,
  len_t count,
  StreamContext stream
);
EXTERN_C void launch_gradient_clip_r64(
  const void* grads,
  const void* clipped,
  const void* sizes,
  void* norm,
  void* scratch,
  double max_norm,
  len_t count,
  StreamContext stream
);

/* norm[0] = sqrt(sum of g^2 over every element of `count` tensors + alpha * norm[0]^2). grads and sizes */
/* are host arrays of `count` device addresses and of `count` element counts (len_t), read before the */
/* call returns; norm is one double on the device. alpha = 0 never reads norm, alpha = 1 adds tensors of */
/* another type or place to what an earlier call found. Sums run in fp64 in a fixed order. scratch is */
/* caller-owned workspace of mpGradientNormScratchBytes(dtype, count) bytes, 8-byte aligned. No reference */
/* kernel exists. */
EXTERN_C void launch_gradient_norm_r16(
  const void* grads,
  const void* sizes,
  void* norm,
  void* scratch,
  double alpha,
  len_t count,
  StreamContext stream
);
EXTERN_C void launch_gradient_norm_r32(
  const void* grads,
  const void* sizes,
  void* norm,
  void* scratch,
  double alpha,
  len_t count,
  StreamContext stream
);
EXTERN_C void launch_gradient_norm_r64(
  const void* grads,
  const void* sizes,
  void* norm,
  void* scratch,
  double alpha,
  len_t count,
  StreamContext stream
);

/* clipped_k = grads_k * min(1, max_norm / norm[0]) for `count` tensors, with the norm that an earlier */
/* gradient_norm left on the device (tensors of several types: one gradient_norm each, alpha = 1 from the */
/* second on, then one gradient_scale each). grads, clipped and sizes are host arrays as in */
/* gradient_norm; clipped_k may be grads_k, and a norm of at most max_norm then writes nothing. A result */
/* that overlaps another result or another gradient is refused: what it holds would depend on which */
/* workgroup comes first. 256 GiB of tensors or more in one call are refused too. A norm that is infinite */
/* or NaN gives zeros and NaNs as the formula does: the caller sees it in norm. */
EXTERN_C void launch_gradient_scale_r16(
  const void* grads,
  const void* clipped,
  const void* sizes,
  const void* norm,
  double max_norm,
  len_t count,
  StreamContext stream
);
EXTERN_C void launch_gradient_scale_r32(
  const void* grads,
  const void* clipped,
  const void* sizes,
  const void* norm,
  double max_norm,
  len_t count,
  StreamContext stream
);
EXTERN_C void launch_gradient_scale_r64(
  const void* grads,
  const void* clipped,
  const void* sizes,
  const void* norm,
  double max_norm,
  len_t count,
  StreamContext stream
);

/* c = a * b. Replaces src/cuda/nvcc_src/hadamard.cu:3-29. */
EXTERN_C void launch_hadamard_r16(
  const void* a,
  const void* b,
  void* c,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_hadamard_r32(
  const void* a,
  const void* b,
  void* c,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_hadamard_r64(
  const void* a,
  const void* b,
  void* c,
  len_t N,
  StreamContext stream
);

/* c += a * b. Replaces src/cuda/nvcc_src/hadamard_reverse.cu:3-29; called twice per */
/* hadamard reverse with the operands swapped (src/ops/hadamard.zig:65-79). */
EXTERN_C void launch_hadamard_reverse_r16(
  const void* a,
  const void* b,
  void* c,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_hadamard_reverse_r32(
  const void* a,
  const void* b,
  void* c,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_hadamard_reverse_r64(
  const void* a,
  const void* b,
  void* c,
  len_t N,
  StreamContext stream
);

/* c[m,k] = alpha * a[m,n] . b[n,k] + beta * c[m,k], row-major. Replaces */
/* src/cuda/nvcc_src/inner_product_ij_jk_ik.cu:3-27 (called by src/ops/inner_product.zig:286-303). */
/* The stream context must carry the BLAS handle that mpInitStream creates. */
EXTERN_C void launch_inner_product_ij_jk_ik_r16(
  const void* a_data,
  const void* b_data,
  double alpha,
  void* c_data,
  double beta,
  len_t m, len_t n, len_t k,
  StreamContext stream
);
EXTERN_C void launch_inner_product_ij_jk_ik_r32(
  const void* a_data,
  const void* b_data,
  double alpha,
  void* c_data,
  double beta,
  len_t m, len_t n, len_t k,
  StreamContext stream
);
EXTERN_C void launch_inner_product_ij_jk_ik_r64(
  const void* a_data,
  const void* b_data,
  double alpha,
  void* c_data,
  double beta,
  len_t m, len_t n, len_t k,
  StreamContext stream
);

/* c[m,k] = alpha * a[m,n] . transpose(b[k,n]) + beta * c[m,k], row-major. No reference launcher: */
/* src/ops/inner_product.zig:316-327 transposes b into scratch (permutate_ij_ji) and then calls */
/* inner_product_ij_jk_ik; here the transposition is an operation flag of the library call. */
EXTERN_C void launch_inner_product_ij_kj_ik_r16(
  const void* a_data,
  const void* b_data,
  double alpha,
  void* c_data,
  double beta,
  len_t m, len_t n, len_t k,
  StreamContext stream
);
EXTERN_C void launch_inner_product_ij_kj_ik_r32(
  const void* a_data,
  const void* b_data,
  double alpha,
  void* c_data,
  double beta,
  len_t m, len_t n, len_t k,
  StreamContext stream
);
EXTERN_C void launch_inner_product_ij_kj_ik_r64(
  const void* a_data,
  const void* b_data,
  double alpha,
  void* c_data,
  double beta,
  len_t m, len_t n, len_t k,
  StreamContext stream
);

/* c[m,k] = alpha * transpose(a[n,m]) . b[n,k] + beta * c[m,k], row-major. No reference launcher: */
/* src/ops/inner_product.zig:372-383 transposes a into scratch (permutate_ij_ji) and then calls */
/* inner_product_ij_jk_ik; here the transposition is an operation flag of the library call. */
EXTERN_C void launch_inner_product_ji_jk_ik_r16(
  const void* a_data,
  const void* b_data,
  double alpha,
  void* c_data,
  double beta,
  len_t m, len_t n, len_t k,
  StreamContext stream
);
EXTERN_C void launch_inner_product_ji_jk_ik_r32(
  const void* a_data,
  const void* b_data,
  double alpha,
  void* c_data,
  double beta,
  len_t m, len_t n, len_t k,
  StreamContext stream
);
EXTERN_C void launch_inner_product_ji_jk_ik_r64(
  const void* a_data,
  const void* b_data,
  double alpha,
  void* c_data,
  double beta,
  len_t m, len_t n, len_t k,
  StreamContext stream
);

/* dst[i,j] = (src[i,j] - mean_j src[i,:]) / sqrt(var_j src[i,:] + eps) * gain[j] + bias[j], with the */
/* variance over n (not n - 1). gain NULL counts as ones, bias NULL as zeros. No reference kernel */
/* exists; scalars cross the boundary as double and sizes as len_t like every reference launcher */
/* (src/cuda/nvcc_src/reduce_ij_i.cu:35-42). dst may be src. */
EXTERN_C void launch_layernorm_ij_j_r16(
  const void* src,
  const void* gain,
  const void* bias,
  void* dst,
  double eps,
  len_t m,
  len_t n,
  StreamContext stream
);
EXTERN_C void launch_layernorm_ij_j_r32(
  const void* src,
  const void* gain,
  const void* bias,
  void* dst,
  double eps,
  len_t m,
  len_t n,
  StreamContext stream
);
EXTERN_C void launch_layernorm_ij_j_r64(
  const void* src,
  const void* gain,
  const void* bias,
  void* dst,
  double eps,
  len_t m,
  len_t n,
  StreamContext stream
);

/* With u_i and r_i = 1/sqrt(variance + eps) of row i of src, h = (src - u_i) * r_i and */
/* e = dst_grads * gain (gain NULL: ones): */
/*   src_grads[i,j] = r_i * (e[i,j] - mean_j e[i,:] - h[i,j] * mean_j(e*h)[i,:]) + alpha*src_grads[i,j] */
/*   gain_grads[j]  = sum_i dst_grads[i,j] * h[i,j]                              + alpha*gain_grads[j] */
/*   bias_grads[j]  = sum_i dst_grads[i,j]                                       + alpha*bias_grads[j] */
/* gain_grads or bias_grads that is NULL is not computed; src_grads may be dst_grads or src. alpha = 0 */
/* never reads the three results. scratch is caller-owned workspace of */
/* mpLayernormReverseScratchBytes(dtype, m, n) bytes, 16-byte aligned (the reference hands kernels their workspace from */
/* the per-stream scratch, src/core/utils.zig:20-36). Results do not change from run to run. */
EXTERN_C void launch_layernorm_ij_j_reverse_r16(
  const void* src,
  const void* gain,
  const void* dst_grads,
  void* src_grads,
  void* gain_grads,
  void* bias_grads,
  void* scratch,
  double eps,
  double alpha,
  len_t m,
  len_t n,
  StreamContext stream
);
EXTERN_C void launch_layernorm_ij_j_reverse_r32(
  const void* src,
  const void* gain,
  const void* dst_grads,
  void* src_grads,
  void* gain_grads,
  void* bias_grads,
  void* scratch,
  double eps,
  double alpha,
  len_t m,
  len_t n,
  StreamContext stream
);
EXTERN_C void launch_layernorm_ij_j_reverse_r64(
  const void* src,
  const void* gain,
  const void* dst_grads,
  void* src_grads,
  void* gain_grads,
  void* bias_grads,
  void* scratch,
  double eps,
  double alpha,
  len_t m,
  len_t n,
  StreamContext stream
);

/* b = -a. Replaces src/cuda/nvcc_src/negate.cu:3-26. */
EXTERN_C void launch_negate_r16(
  const void* a,
  void* b,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_negate_r32(
  const void* a,
  void* b,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_negate_r64(
  const void* a,
  void* b,
  len_t N,
  StreamContext stream
);

/* dst[j,i] = src[i,j] + alpha*dst[j,i] for a row-major [row, col] source; src and dst must not */
/* overlap. Replaces src/cuda/nvcc_src/permutate_ij_ji.cu:7-71 (called with alpha = 0 forward */
/* and alpha = 1 in reverse by src/ops/permutate.zig:45-69). */
EXTERN_C void launch_permutate_ij_ji_r16(
  const void* src,
  void* dst,
  double alpha,
  len_t row,
  len_t col,
  StreamContext ctx
);
EXTERN_C void launch_permutate_ij_ji_r32(
  const void* src,
  void* dst,
  double alpha,
  len_t row,
  len_t col,
  StreamContext ctx
);
EXTERN_C void launch_permutate_ij_ji_r64(
  const void* src,
  void* dst,
  double alpha,
  len_t row,
  len_t col,
  StreamContext ctx
);

/* dst[i] = sum_j src[i,j] + alpha*dst[i]. Replaces src/cuda/nvcc_src/reduce_ij_i.cu:3-54 */
/* (called with alpha = 0 by src/ops/reduce.zig:98-121). A few very long rows (the sum of a whole */
/* tensor) are cut into segments through the workspace that the stream context owns. */
EXTERN_C void launch_reduce_ij_i_r16(
  const void* src,
  void* dst,
  double alpha,
  len_t m,
  len_t n,
  StreamContext stream
);
EXTERN_C void launch_reduce_ij_i_r32(
  const void* src,
  void* dst,
  double alpha,
  len_t m,
  len_t n,
  StreamContext stream
);
EXTERN_C void launch_reduce_ij_i_r64(
  const void* src,
  void* dst,
  double alpha,
  len_t m,
  len_t n,
  StreamContext stream
);

/* dst[j] = sum_i src[i,j] + alpha*dst[j]. Replaces src/cuda/nvcc_src/reduce_ij_j.cu:3-66, whose */
/* output line reads dst[threadIdx.x] instead of its own column (:42-43) and whose grid runs */
/* over m instead of n (:56); this follows the stated intent (src/ops/reduce.zig:142-165). */
/* Tall matrices split their rows through the workspace that the stream context owns (work on */
/* one stream is ordered, so launchers share it); a context without one walks every row per strip. */
EXTERN_C void launch_reduce_ij_j_r16(
  const void* src,
  void* dst,
  double alpha,
  len_t m,
  len_t n,
  StreamContext stream
);
EXTERN_C void launch_reduce_ij_j_r32(
  const void* src,
  void* dst,
  double alpha,
  len_t m,
  len_t n,
  StreamContext stream
);
EXTERN_C void launch_reduce_ij_j_r64(
  const void* src,
  void* dst,
  double alpha,
  len_t m,
  len_t n,
  StreamContext stream
);

/* dst[j] = sum_i src[i,j] + alpha*dst[j], like launch_reduce_ij_j, with caller-owned scratch of */
/* mpReduceScratchBytes(dtype, m, n) bytes (NULL allowed). No reference launcher: the reference's */
/* column sum has no workspace parameter (src/cuda/nvcc_src/reduce_ij_j.cu:46-53), so a tall, narrow */
/* matrix (a bias gradient: [tokens, hidden]) can only be walked by one workgroup per column */
/* strip. With scratch the rows are split into chunks, every chunk leaves a partial row, and a */
/* second kernel adds the partial rows in a fixed order. */
EXTERN_C void launch_reduce_ij_j_scratch_r16(
  const void* src,
  void* dst,
  void* scratch,
  double alpha,
  len_t m,
  len_t n,
  StreamContext stream
);
EXTERN_C void launch_reduce_ij_j_scratch_r32(
  const void* src,
  void* dst,
  void* scratch,
  double alpha,
  len_t m,
  len_t n,
  StreamContext stream
);
EXTERN_C void launch_reduce_ij_j_scratch_r64(
  const void* src,
  void* dst,
  void* scratch,
  double alpha,
  len_t m,
  len_t n,
  StreamContext stream
);

/* b = (a >= 0) ? a : 0. Replaces src/cuda/nvcc_src/relu.cu:3-27. */
EXTERN_C void launch_relu_r16(
  const void* a,
  void* b,
  len_t n,
  StreamContext stream
);
EXTERN_C void launch_relu_r32(
  const void* a,
  void* b,
  len_t n,
  StreamContext stream
);
EXTERN_C void launch_relu_r64(
  const void* a,
  void* b,
  len_t n,
  StreamContext stream
);

/* a_grads += b_grads * ((a_value >= 0) ? 1 : 0). Replaces src/cuda/nvcc_src/relu_reverse.cu:3-31. */
EXTERN_C void launch_relu_reverse_r16(
  const void* a_value,
  void* a_grads,
  const void* b_grads,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_relu_reverse_r32(
  const void* a_value,
  void* a_grads,
  const void* b_grads,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_relu_reverse_r64(
  const void* a_value,
  void* a_grads,
  const void* b_grads,
  len_t N,
  StreamContext stream
);

/* dst[i,j] = src[i,j] * gain[j] / sqrt(mean_j src[i,:]^2 + eps). No reference kernel exists; */
/* scalars cross the boundary as double and sizes as len_t like every reference launcher */
/* (src/cuda/nvcc_src/reduce_ij_i.cu:35-42). dst may be src. scratch: mpRmsnormScratchBytes(dtype, m, n) */
/* bytes owned by the caller (0 for rows one workgroup holds), or NULL: rows longer than that are */
/* then read twice. */
/* An input of up to 256 MiB is read so that it stays in the GPU's memory-side cache, where the */
/* reverse that reads it again finds it (a step of forward and reverse gains 6 %, a forward on its */
/* own pays 2 %); larger inputs stream past the cache. */
EXTERN_C void launch_rmsnorm_ij_j_r16(
  const void* src,
  const void* gain,
  void* dst,
  void* scratch,
  double eps,
  len_t m,
  len_t n,
  StreamContext stream
);
EXTERN_C void launch_rmsnorm_ij_j_r32(
  const void* src,
  const void* gain,
  void* dst,
  void* scratch,
  double eps,
  len_t m,
  len_t n,
  StreamContext stream
);
EXTERN_C void launch_rmsnorm_ij_j_r64(
  const void* src,
  const void* gain,
  void* dst,
  void* scratch,
  double eps,
  len_t m,
  len_t n,
  StreamContext stream
);

/* With r_i = 1/sqrt(mean_j src[i,:]^2 + eps) and c_i = mean_j(dst_grads*gain*src)[i,:]: */
/*   src_grads[i,j] = r_i * (dst_grads[i,j]*gain[j] - src[i,j] * r_i^2 * c_i) + alpha*src_grads[i,j] */
/*   gain_grads[j]  = sum_i dst_grads[i,j] * src[i,j] * r_i                   + alpha*gain_grads[j] */
/* scratch is caller-owned workspace of mpRmsnormReverseScratchBytes(dtype, m, n) bytes (the */
/* reference hands kernels their workspace from the per-stream scratch, src/core/utils.zig:20-36). */
/* Two kernels are enqueued: the row pass and the fixed-order sum of the partial gain rows. */
EXTERN_C void launch_rmsnorm_ij_j_reverse_r16(
  const void* src,
  const void* gain,
  const void* dst_grads,
  void* src_grads,
  void* gain_grads,
  void* scratch,
  double eps,
  double alpha,
  len_t m,
  len_t n,
  StreamContext stream
);
EXTERN_C void launch_rmsnorm_ij_j_reverse_r32(
  const void* src,
  const void* gain,
  const void* dst_grads,
  void* src_grads,
  void* gain_grads,
  void* scratch,
  double eps,
  double alpha,
  len_t m,
  len_t n,
  StreamContext stream
);
EXTERN_C void launch_rmsnorm_ij_j_reverse_r64(
  const void* src,
  const void* gain,
  const void* dst_grads,
  void* src_grads,
  void* gain_grads,
  void* scratch,
  double eps,
  double alpha,
  len_t m,
  len_t n,
  StreamContext stream
);

/* b = selu(a) = scale*a for a > 0, scale*alpha*expm1(a) otherwise. The reference names */
/* mp.ops.selu (README.md:97) but ships no kernel; the signature is that of its activation */
/* launchers (src/cuda/nvcc_src/relu.cu:16-21). */
EXTERN_C void launch_selu_r16(
  const void* a,
  void* b,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_selu_r32(
  const void* a,
  void* b,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_selu_r64(
  const void* a,
  void* b,
  len_t N,
  StreamContext stream
);

/* a_grads += b_grads * selu'(a_value), selu' = scale for a > 0, scale*alpha*exp(a) otherwise. */
/* Argument order and the accumulate-into-gradient convention of */
/* src/cuda/nvcc_src/relu_reverse.cu:3-31. */
EXTERN_C void launch_selu_reverse_r16(
  const void* a_value,
  void* a_grads,
  const void* b_grads,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_selu_reverse_r32(
  const void* a_value,
  void* a_grads,
  const void* b_grads,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_selu_reverse_r64(
  const void* a_value,
  void* a_grads,
  const void* b_grads,
  len_t N,
  StreamContext stream
);

/* dev_a[i] = init + step * i. Replaces src/cuda/nvcc_src/sequence.cu:5-32; evaluated in */
/* precision<T>, so r16 does not lose the index above 2048 as Scalar(tid) does there. */
EXTERN_C void launch_sequence_r16(
  void* dev_a,
  double init,
  double step,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_sequence_r32(
  void* dev_a,
  double init,
  double step,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_sequence_r64(
  void* dev_a,
  double init,
  double step,
  len_t N,
  StreamContext stream
);

/* dst[i,j] = exp(src[i,j] - max_j src[i,:]) / sum_j exp(src[i,j] - max_j src[i,:]). */
/* No reference kernel exists (NOTES.md:28); the (src, dst, m, n) shape follows the row */
/* launchers (src/cuda/nvcc_src/reduce_ij_i.cu:35-42) and the "ij|j" name the parser stub of */
/* src/ops/expression_parsing.zig:320-340. dst may be src. scratch is caller-owned workspace of */
/* mpSoftmaxScratchBytes(dtype, m, n) bytes (0 for rows that fit one workgroup) that lets several */
/* workgroups share a long row; the reference's own softmax call sites already pass a scratch */
/* buffer (src/loss/loss.zig:204,226). With scratch == NULL long rows are read twice instead. */
/* An output of up to 128 MiB is written so that it stays in the GPU's memory-side cache, where the */
/* reverse that reads it finds it (a step of forward and reverse gains 8 %, a forward on its own */
/* pays 3 %); larger outputs stream past the cache. */
EXTERN_C void launch_softmax_ij_j_r16(
  const void* src,
  void* dst,
  void* scratch,
  len_t m,
  len_t n,
  StreamContext stream
);
EXTERN_C void launch_softmax_ij_j_r32(
  const void* src,
  void* dst,
  void* scratch,
  len_t m,
  len_t n,
  StreamContext stream
);
EXTERN_C void launch_softmax_ij_j_r64(
  const void* src,
  void* dst,
  void* scratch,
  len_t m,
  len_t n,
  StreamContext stream
);

/* src_grads[i,j] = dst_value[i,j] * (dst_grads[i,j] - sum_j dst_value[i,j]*dst_grads[i,j]) */
/*                  + alpha * src_grads[i,j]. */
/* Takes the forward OUTPUT, not the input. alpha follows the blend convention of the */
/* reference's row launchers (src/cuda/nvcc_src/reduce_ij_i.cu:31): 0 overwrites, 1 accumulates. */
/* scratch: mpSoftmaxReverseScratchBytes(dtype, m, n) bytes owned by the caller, or NULL (rows too */
/* long for one workgroup are then read twice); the reference's softmax call sites pass one too */
/* (src/loss/loss.zig:204,226). */
EXTERN_C void launch_softmax_ij_j_reverse_r16(
  const void* dst_value,
  const void* dst_grads,
  void* src_grads,
  void* scratch,
  double alpha,
  len_t m,
  len_t n,
  StreamContext stream
);
EXTERN_C void launch_softmax_ij_j_reverse_r32(
  const void* dst_value,
  const void* dst_grads,
  void* src_grads,
  void* scratch,
  double alpha,
  len_t m,
  len_t n,
  StreamContext stream
);
EXTERN_C void launch_softmax_ij_j_reverse_r64(
  const void* dst_value,
  const void* dst_grads,
  void* src_grads,
  void* scratch,
  double alpha,
  len_t m,
  len_t n,
  StreamContext stream
);

/* b = (a >= 0) ? 1 : 0, the derivative of relu that src/ops/relu.zig:54-57 asks this launcher */
/* for. The reference body (src/cuda/nvcc_src/stepwise.cu:11-12) is a verbatim copy of relu and */
/* returns a itself for a >= 0; the step function is what its caller needs. */
EXTERN_C void launch_stepwise_r16(
  const void* a,
  void* b,
  len_t n,
  StreamContext stream
);
EXTERN_C void launch_stepwise_r32(
  const void* a,
  void* b,
  len_t n,
  StreamContext stream
);
EXTERN_C void launch_stepwise_r64(
  const void* a,
  void* b,
  len_t n,
  StreamContext stream
);

/* c = a - b. Replaces src/cuda/nvcc_src/subtraction.cu:3-29. */
EXTERN_C void launch_subtraction_r16(
  const void* a,
  const void* b,
  void* c,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_subtraction_r32(
  const void* a,
  const void* b,
  void* c,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_subtraction_r64(
  const void* a,
  const void* b,
  void* c,
  len_t N,
  StreamContext stream
);

/* c = a + value. Replaces src/cuda/nvcc_src/translate.cu:3-29. */
EXTERN_C void launch_translate_r16(
  const void* a,
  double value,
  void* c,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_translate_r32(
  const void* a,
  double value,
  void* c,
  len_t N,
  StreamContext stream
);
EXTERN_C void launch_translate_r64(
  const void* a,
  double value,
  void* c,
  len_t N,
  StreamContext stream
);

/* Not per-dtype; defined in metaphor_amd/csrc/kernel_support.hip. */
/* Bytes of caller-owned scratch for launch_rmsnorm_ij_j_reverse_<dtype> on an [m, n] problem;
 * dtype is the dispatch key 0 = r16, 1 = r32, 2 = r64 (src/core/scalar.zig:35-40). The reference
 * sizes per-stream scratch on the host the same way (src/core/utils.zig:20-36). */
EXTERN_C len_t mpRmsnormReverseScratchBytes(len_t dtype, len_t m, len_t n);
/* Bytes of caller-owned scratch launch_softmax_ij_j_<dtype> can use on an [m, n] problem (0 when a row
 * fits one workgroup; NULL scratch is allowed and costs a second read of long rows). Rows shared by
 * several workgroups exchange their partial results through words that, where it can, the library keeps
 * in device memory of its own, one region per workspace address and problem geometry: the workspace is
 * then the key that keeps launches apart (launches that may overlap in time must be given different
 * workspaces, as they must when the words are in the workspace itself) and is not written. */
EXTERN_C len_t mpSoftmaxScratchBytes(len_t dtype, len_t m, len_t n);
EXTERN_C len_t mpSoftmaxReverseScratchBytes(len_t dtype, len_t m, len_t n);
EXTERN_C len_t mpReduceScratchBytes(len_t dtype, len_t m, len_t n);
EXTERN_C len_t mpRmsnormScratchBytes(len_t dtype, len_t m, len_t n);
EXTERN_C len_t mpLayernormReverseScratchBytes(len_t dtype, len_t m, len_t n);
EXTERN_C len_t mpEmbeddingReverseScratchBytes(len_t dtype, len_t v, len_t m, len_t n);
EXTERN_C len_t mpGradientNormScratchBytes(len_t dtype, len_t count);
/* launch_rmsnorm_ij_j_reverse_r32 without the scratch argument, for callers that cannot allocate a
 * workspace (code under HIP graph capture, serving loops, harnesses that forbid hipMalloc): the partial
 * gain rows go into a 16 MiB device array that the library holds on every GPU it runs on. It has no
 * counterpart in the reference. Same kernels, bit-identical results. Returns 0 after enqueueing, 1
 * (message on stderr, nothing enqueued) when [m, n] needs more than the 16 MiB: min(m, 2 * CUs) * n * 4
 * bytes, so rows of up to 4194304 / min(m, 2 * CUs) elements fit, 8192 on the MI355X's 256 compute
 * units. Calls no hipMalloc / hipFree; its first call on a device looks the array's address up (make
 * that call before a graph capture starts). All calls on one GPU share the array: calls that overlap in
 * time on one GPU race, and a call on another stream than the one before prints one warning saying so. */
EXTERN_C int mpRmsnormReverseR32NoAlloc(const void* src, const void* gain, const void* dst_grads, void* src_grads, void* gain_grads, double eps, double alpha, len_t m, len_t n, StreamContext stream);

#endif
