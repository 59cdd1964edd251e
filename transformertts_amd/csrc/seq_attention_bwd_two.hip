// The backward passes with operands of two parts (seq_two_parts), in a file of their own: in one module with the others the compiler
// allots the dK / dV pass of heads of 128 its registers another way, seven of them in memory, and it takes 5 % longer.
#include "seq_attention_bwd.h"

template <int DHP>
static void seq_bwd_two_go(const SeqBwdP& p, dim3 g, dim3 gk, hipStream_t st) {
    hipLaunchKernelGGL((seq_attn_dq_kernel<__bf16, DHP, 2, true>), g, dim3(256), 0, st, p);
    hipLaunchKernelGGL((seq_attn_dkv_kernel<__bf16, DHP, true>), gk, dim3(256), 0, st, p);
}
// g, gk: the grids of the dQ pass with its keys in two, and of the dK / dV pass
void seq_bwd_two(const SeqBwdP& p, dim3 g, dim3 gk, hipStream_t st) {
    if (p.dh <= 64) seq_bwd_two_go<64>(p, g, gk, st);
    else if (p.dh <= 128) seq_bwd_two_go<128>(p, g, gk, st);
    else seq_bwd_two_go<192>(p, g, gk, st);
}
