#include "../embedding.h"

// dst[i,j] = scale * table[tokens[i], j] for m tokens and a table of v rows of n elements. tokens are
// signed integers on the device, id_bytes (4 or 8) wide each; an id outside [0, v) (a padded place)
// gives a row of zeros. No reference kernel exists; the nearest is the row broadcast
// (src/cuda/nvcc_src/broadcast_j_ij.cu:9-57). dst must not overlap the table.
extern "C" void launch_embedding_i_ij_Scalar(
  const void* table,
  const void* tokens,
  void* dst,
  double scale,
  len_t id_bytes,
  len_t v,
  len_t m,
  len_t n,
  StreamContext stream
) {
  mp::embedding_forward<Scalar>(static_cast<const Scalar*>(table), tokens, static_cast<Scalar*>(dst), scale, id_bytes,
                                v, m, n, get_stream(stream));
}
