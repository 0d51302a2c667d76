#include "../row_layernorm.h"

// dst[i,j] = (src[i,j] - mean_j src[i,:]) / sqrt(var_j src[i,:] + eps) * gain[j] + bias[j], with the
// variance over n (not n - 1). gain NULL counts as ones, bias NULL as zeros. No reference kernel
// exists; scalars cross the boundary as double and sizes as len_t like every reference launcher
// (src/cuda/nvcc_src/reduce_ij_i.cu:35-42). dst may be src.
extern "C" void launch_layernorm_ij_j_Scalar(
  const void* src,
  const void* gain,
  const void* bias,
  void* dst,
  double eps,
  len_t m,
  len_t n,
  StreamContext stream
) {
  mp::layernorm_forward<Scalar>(static_cast<const Scalar*>(src), static_cast<const Scalar*>(gain),
                                static_cast<const Scalar*>(bias), static_cast<Scalar*>(dst), eps, m, n,
                                get_stream(stream));
}
