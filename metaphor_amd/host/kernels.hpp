// GENERATED by metaphor_amd/kernelgen.py -- do not edit.
// One three-entry dispatch array per kernel stem, indexed by the dtype key
// (0 = r16, 1 = r32, 2 = r64), as src/core/kernels.zig holds them; calling the array is
// src/core/root.zig:36-43 (invoke).
#ifndef MP_HOST_KERNELS_HPP
#define MP_HOST_KERNELS_HPP

#include <cstddef>

#include "kernel_decls.h"

namespace mp {
[[noreturn]] void panic(const char* what);
namespace kernels {

template <class Fn> struct DispatchArray {
  Fn* fn[3];
  template <class... Args> void operator()(size_t key, Args... args) const {
    if (key > 2) panic("invoke: dtype key out of range");
    fn[key](args...);
  }
};

inline const DispatchArray<decltype(launch_addition_r16)> addition{{launch_addition_r16, launch_addition_r32, launch_addition_r64}};
inline const DispatchArray<decltype(launch_broadcast_i_ij_r16)> broadcast_i_ij{{launch_broadcast_i_ij_r16, launch_broadcast_i_ij_r32, launch_broadcast_i_ij_r64}};
inline const DispatchArray<decltype(launch_broadcast_j_ij_r16)> broadcast_j_ij{{launch_broadcast_j_ij_r16, launch_broadcast_j_ij_r32, launch_broadcast_j_ij_r64}};
inline const DispatchArray<decltype(launch_copy_r16)> copy{{launch_copy_r16, launch_copy_r32, launch_copy_r64}};
inline const DispatchArray<decltype(launch_dilate_r16)> dilate{{launch_dilate_r16, launch_dilate_r32, launch_dilate_r64}};
inline const DispatchArray<decltype(launch_dilate_reverse_r16)> dilate_reverse{{launch_dilate_reverse_r16, launch_dilate_reverse_r32, launch_dilate_reverse_r64}};
inline const DispatchArray<decltype(launch_embedding_i_ij_r16)> embedding_i_ij{{launch_embedding_i_ij_r16, launch_embedding_i_ij_r32, launch_embedding_i_ij_r64}};
inline const DispatchArray<decltype(launch_embedding_i_ij_reverse_r16)> embedding_i_ij_reverse{{launch_embedding_i_ij_reverse_r16, launch_embedding_i_ij_reverse_r32, launch_embedding_i_ij_reverse_r64}};
inline const DispatchArray<decltype(launch_fill_r16)> fill{{launch_fill_r16, launch_fill_r32, launch_fill_r64}};
inline const DispatchArray<decltype(launch_fused_add_add_r16)> fused_add_add{{launch_fused_add_add_r16, launch_fused_add_add_r32, launch_fused_add_add_r64}};
inline const DispatchArray<decltype(launch_fused_add_add_reverse_r16)> fused_add_add_reverse{{launch_fused_add_add_reverse_r16, launch_fused_add_add_reverse_r32, launch_fused_add_add_reverse_r64}};
inline const DispatchArray<decltype(launch_fused_hadamard_add_add_r16)> fused_hadamard_add_add{{launch_fused_hadamard_add_add_r16, launch_fused_hadamard_add_add_r32, launch_fused_hadamard_add_add_r64}};
inline const DispatchArray<decltype(launch_fused_hadamard_add_add_reverse_r16)> fused_hadamard_add_add_reverse{{launch_fused_hadamard_add_add_reverse_r16, launch_fused_hadamard_add_add_reverse_r32, launch_fused_hadamard_add_add_reverse_r64}};
inline const DispatchArray<decltype(launch_fused_relu_hadamard_add_add_r16)> fused_relu_hadamard_add_add{{launch_fused_relu_hadamard_add_add_r16, launch_fused_relu_hadamard_add_add_r32, launch_fused_relu_hadamard_add_add_r64}};
inline const DispatchArray<decltype(launch_fused_relu_hadamard_add_add_reverse_r16)> fused_relu_hadamard_add_add_reverse{{launch_fused_relu_hadamard_add_add_reverse_r16, launch_fused_relu_hadamard_add_add_reverse_r32, launch_fused_relu_hadamard_add_add_reverse_r64}};
inline const DispatchArray<decltype(launch_fused_selu_add_r16)> fused_selu_add{{launch_fused_selu_add_r16, launch_fused_selu_add_r32, launch_fused_selu_add_r64}};
inline const DispatchArray<decltype(launch_fused_selu_add_reverse_r16)> fused_selu_add_reverse{{launch_fused_selu_add_reverse_r16, launch_fused_selu_add_reverse_r32, launch_fused_selu_add_reverse_r64}};
inline const DispatchArray<decltype(launch_fused_selu_hadamard_add_add_r16)> fused_selu_hadamard_add_add{{launch_fused_selu_hadamard_add_add_r16, launch_fused_selu_hadamard_add_add_r32, launch_fused_selu_hadamard_add_add_r64}};
inline const DispatchArray<decltype(launch_fused_selu_hadamard_add_add_reverse_r16)> fused_selu_hadamard_add_add_reverse{{launch_fused_selu_hadamard_add_add_reverse_r16, launch_fused_selu_hadamard_add_add_reverse_r32, launch_fused_selu_hadamard_add_add_reverse_r64}};
inline const DispatchArray<decltype(launch_fused_selu_hadamard_sub_r16)> fused_selu_hadamard_sub{{launch_fused_selu_hadamard_sub_r16, launch_fused_selu_hadamard_sub_r32, launch_fused_selu_hadamard_sub_r64}};
inline const DispatchArray<decltype(launch_fused_selu_hadamard_sub_reverse_r16)> fused_selu_hadamard_sub_reverse{{launch_fused_selu_hadamard_sub_reverse_r16, launch_fused_selu_hadamard_sub_reverse_r32, launch_fused_selu_hadamard_sub_reverse_r64}};
inline const DispatchArray<decltype(launch_gradient_clip_r16)> gradient_clip{{launch_gradient_clip_r16, launch_gradient_clip_r32, launch_gradient_clip_r64}};
inline const DispatchArray<decltype(launch_gradient_norm_r16)> gradient_norm{{launch_gradient_norm_r16, launch_gradient_norm_r32, launch_gradient_norm_r64}};
inline const DispatchArray<decltype(launch_gradient_scale_r16)> gradient_scale{{launch_gradient_scale_r16, launch_gradient_scale_r32, launch_gradient_scale_r64}};
inline const DispatchArray<decltype(launch_hadamard_r16)> hadamard{{launch_hadamard_r16, launch_hadamard_r32, launch_hadamard_r64}};
inline const DispatchArray<decltype(launch_hadamard_reverse_r16)> hadamard_reverse{{launch_hadamard_reverse_r16, launch_hadamard_reverse_r32, launch_hadamard_reverse_r64}};
inline const DispatchArray<decltype(launch_inner_product_ij_jk_ik_r16)> inner_product_ij_jk_ik{{launch_inner_product_ij_jk_ik_r16, launch_inner_product_ij_jk_ik_r32, launch_inner_product_ij_jk_ik_r64}};
inline const DispatchArray<decltype(launch_inner_product_ij_kj_ik_r16)> inner_product_ij_kj_ik{{launch_inner_product_ij_kj_ik_r16, launch_inner_product_ij_kj_ik_r32, launch_inner_product_ij_kj_ik_r64}};
inline const DispatchArray<decltype(launch_inner_product_ji_jk_ik_r16)> inner_product_ji_jk_ik{{launch_inner_product_ji_jk_ik_r16, launch_inner_product_ji_jk_ik_r32, launch_inner_product_ji_jk_ik_r64}};
inline const DispatchArray<decltype(launch_layernorm_ij_j_r16)> layernorm_ij_j{{launch_layernorm_ij_j_r16, launch_layernorm_ij_j_r32, launch_layernorm_ij_j_r64}};
inline const DispatchArray<decltype(launch_layernorm_ij_j_reverse_r16)> layernorm_ij_j_reverse{{launch_layernorm_ij_j_reverse_r16, launch_layernorm_ij_j_reverse_r32, launch_layernorm_ij_j_reverse_r64}};
inline const DispatchArray<decltype(launch_negate_r16)> negate{{launch_negate_r16, launch_negate_r32, launch_negate_r64}};
inline const DispatchArray<decltype(launch_permutate_ij_ji_r16)> permutate_ij_ji{{launch_permutate_ij_ji_r16, launch_permutate_ij_ji_r32, launch_permutate_ij_ji_r64}};
inline const DispatchArray<decltype(launch_reduce_ij_i_r16)> reduce_ij_i{{launch_reduce_ij_i_r16, launch_reduce_ij_i_r32, launch_reduce_ij_i_r64}};
inline const DispatchArray<decltype(launch_reduce_ij_j_r16)> reduce_ij_j{{launch_reduce_ij_j_r16, launch_reduce_ij_j_r32, launch_reduce_ij_j_r64}};
inline const DispatchArray<decltype(launch_reduce_ij_j_scratch_r16)> reduce_ij_j_scratch{{launch_reduce_ij_j_scratch_r16, launch_reduce_ij_j_scratch_r32, launch_reduce_ij_j_scratch_r64}};
inline const DispatchArray<decltype(launch_relu_r16)> relu{{launch_relu_r16, launch_relu_r32, launch_relu_r64}};
inline const DispatchArray<decltype(launch_relu_reverse_r16)> relu_reverse{{launch_relu_reverse_r16, launch_relu_reverse_r32, launch_relu_reverse_r64}};
inline const DispatchArray<decltype(launch_rmsnorm_ij_j_r16)> rmsnorm_ij_j{{launch_rmsnorm_ij_j_r16, launch_rmsnorm_ij_j_r32, launch_rmsnorm_ij_j_r64}};
inline const DispatchArray<decltype(launch_rmsnorm_ij_j_reverse_r16)> rmsnorm_ij_j_reverse{{launch_rmsnorm_ij_j_reverse_r16, launch_rmsnorm_ij_j_reverse_r32, launch_rmsnorm_ij_j_reverse_r64}};
inline const DispatchArray<decltype(launch_selu_r16)> selu{{launch_selu_r16, launch_selu_r32, launch_selu_r64}};
inline const DispatchArray<decltype(launch_selu_reverse_r16)> selu_reverse{{launch_selu_reverse_r16, launch_selu_reverse_r32, launch_selu_reverse_r64}};
inline const DispatchArray<decltype(launch_sequence_r16)> sequence{{launch_sequence_r16, launch_sequence_r32, launch_sequence_r64}};
inline const DispatchArray<decltype(launch_softmax_ij_j_r16)> softmax_ij_j{{launch_softmax_ij_j_r16, launch_softmax_ij_j_r32, launch_softmax_ij_j_r64}};
inline const DispatchArray<decltype(launch_softmax_ij_j_reverse_r16)> softmax_ij_j_reverse{{launch_softmax_ij_j_reverse_r16, launch_softmax_ij_j_reverse_r32, launch_softmax_ij_j_reverse_r64}};
inline const DispatchArray<decltype(launch_stepwise_r16)> stepwise{{launch_stepwise_r16, launch_stepwise_r32, launch_stepwise_r64}};
inline const DispatchArray<decltype(launch_subtraction_r16)> subtraction{{launch_subtraction_r16, launch_subtraction_r32, launch_subtraction_r64}};
inline const DispatchArray<decltype(launch_translate_r16)> translate{{launch_translate_r16, launch_translate_r32, launch_translate_r64}};

}  // namespace kernels
}  // namespace mp

#endif
