#include "../gradient_norm.h"

// norm[0] = sqrt(sum of g^2 over every element of `count` tensors + alpha * norm[0]^2). grads and sizes
// are host arrays of `count` device addresses and of `count` element counts (len_t), read before the
// call returns; norm is one double on the device. alpha = 0 never reads norm, alpha = 1 adds tensors of
// another type or place to what an earlier call found. Sums run in fp64 in a fixed order. scratch is
// caller-owned workspace of mpGradientNormScratchBytes(dtype, count) bytes, 8-byte aligned. No reference
// kernel exists.
extern "C" void launch_gradient_norm_Scalar(
  const void* grads,
  const void* sizes,
  void* norm,
  void* scratch,
  double alpha,
  len_t count,
  StreamContext stream
) {
  mp::gradient_norm<Scalar>(grads, sizes, norm, scratch, alpha, count, get_stream(stream));
}
