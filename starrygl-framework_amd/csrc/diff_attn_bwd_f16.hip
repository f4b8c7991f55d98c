// Backward matrix kernels of differential attention for fp16: a file of its own, so that the types compile side by side.
#include "diff_attn_bwd.hpp"

template void sgl::attn::backward_type<_Float16>(const AttnArgs&, hipStream_t);
