#include "../embedding.h"

// table_grads[k,j] = scale * sum of dst_grads[i,j] over the places i with tokens[i] == k
//                    + alpha*table_grads[k,j]
// for every row k of the table, the ones no token names among them (alpha = 0 clears those and never
// reads table_grads; alpha = 1 leaves them untouched). tokens and id_bytes as in embedding_i_ij; the
// gradient of a padded place is not read into any sum. scratch is caller-owned workspace of
// mpEmbeddingReverseScratchBytes(dtype, v, m, n) bytes, 16-byte aligned; launches that may overlap in
// time get different workspaces. Results do not change from run to run.
extern "C" void launch_embedding_i_ij_reverse_Scalar(
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
) {
  mp::embedding_reverse<Scalar>(tokens, static_cast<const Scalar*>(dst_grads), static_cast<Scalar*>(table_grads), scratch,
                                scale, alpha, id_bytes, v, m, n, get_stream(stream));
}
