#include "../row_layernorm.h"

// With u_i and r_i = 1/sqrt(variance + eps) of row i of src, h = (src - u_i) * r_i and
// e = dst_grads * gain (gain NULL: ones):
//   src_grads[i,j] = r_i * (e[i,j] - mean_j e[i,:] - h[i,j] * mean_j(e*h)[i,:]) + alpha*src_grads[i,j]
//   gain_grads[j]  = sum_i dst_grads[i,j] * h[i,j]                              + alpha*gain_grads[j]
//   bias_grads[j]  = sum_i dst_grads[i,j]                                       + alpha*bias_grads[j]
// gain_grads or bias_grads that is NULL is not computed; src_grads may be dst_grads or src. alpha = 0
// never reads the three results. scratch is caller-owned workspace of
// mpLayernormReverseScratchBytes(dtype, m, n) bytes, 16-byte aligned (the reference hands kernels their workspace from
// the per-stream scratch, src/core/utils.zig:20-36). Results do not change from run to run.
extern "C" void launch_layernorm_ij_j_reverse_Scalar(
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
) {
  mp::layernorm_reverse<Scalar>(static_cast<const Scalar*>(src), static_cast<const Scalar*>(gain),
                                static_cast<const Scalar*>(dst_grads), static_cast<Scalar*>(src_grads),
                                static_cast<Scalar*>(gain_grads), static_cast<Scalar*>(bias_grads), scratch,
                                eps, alpha, m, n, get_stream(stream));
}
