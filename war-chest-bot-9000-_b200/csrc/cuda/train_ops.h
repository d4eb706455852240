// Launchers of the training operators (the C entries check every argument
// before they call these; all pointers are device memory of the current
// device).
#pragma once
#include <cuda_runtime.h>

#include "../../../include/wc_b200.h"

namespace wctrain {

// limit of each wait of a kernel for its own copies and products, ns of %globaltimer
uint64_t wait_limit();
// policy_loss.cu
uint64_t policy_loss_workspace(int64_t rows, int64_t width);
void launch_policy_loss(const wc_policy_loss_args& a, cudaStream_t s);
// block_norm.cu
uint64_t block_norm_workspace(const wc_block_norm_args& a);
void launch_block_norm(const wc_block_norm_args& a, cudaStream_t s);
void launch_block_norm_backward(const wc_block_norm_args& a, const wc_block_norm_grads& g, cudaStream_t s);
// act8.cu
void launch_act8_pack(const wc_act8_args& a, cudaStream_t s);
void launch_act8_unpack(const wc_act8_args& a, cudaStream_t s);
void launch_gelu8(const wc_act8_args& a, cudaStream_t s);
uint64_t gelu8_workspace(int64_t rows, int64_t width);
void launch_gelu8_backward(const wc_act8_args& a, cudaStream_t s);
// wgrad8.cu
uint64_t wgrad8_workspace(const wc_act8_wgrad_args& a);
void launch_wgrad8(const wc_act8_wgrad_args& a, cudaStream_t s);

}  // namespace wctrain
