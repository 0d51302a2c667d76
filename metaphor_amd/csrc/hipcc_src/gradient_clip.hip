#include "../gradient_norm.h"

// gradient_norm (alpha = 0) and gradient_scale of the same `count` tensors in one call: norm[0] gets
// their norm, clipped_k = grads_k * min(1, max_norm / norm[0]). Arguments and workspace as there.
extern "C" void launch_gradient_clip_Scalar(
  const void* grads,
  const void* clipped,
  const void* sizes,
  void* norm,
  void* scratch,
  double max_norm,
  len_t count,
  StreamContext stream
) {
  mp::gradient_clip<Scalar>(grads, clipped, sizes, norm, scratch, max_norm, count, get_stream(stream));
}
