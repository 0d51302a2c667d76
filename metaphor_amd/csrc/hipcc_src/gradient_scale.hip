#include "../gradient_norm.h"

// clipped_k = grads_k * min(1, max_norm / norm[0]) for `count` tensors, with the norm that an earlier
// gradient_norm left on the device (tensors of several types: one gradient_norm each, alpha = 1 from the
// second on, then one gradient_scale each). grads, clipped and sizes are host arrays as in
// gradient_norm; clipped_k may be grads_k, and a norm of at most max_norm then writes nothing. A result
// that overlaps another result or another gradient is refused: what it holds would depend on which
// workgroup comes first. 256 GiB of tensors or more in one call are refused too. A norm that is infinite
// or NaN gives zeros and NaNs as the formula does: the caller sees it in norm.
extern "C" void launch_gradient_scale_Scalar(
  const void* grads,
  const void* clipped,
  const void* sizes,
  const void* norm,
  double max_norm,
  len_t count,
  StreamContext stream
) {
  mp::gradient_scale<Scalar>(grads, clipped, sizes, norm, max_norm, count, get_stream(stream));
}
