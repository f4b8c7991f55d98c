// Forward matrix kernels of differential attention for bfloat16: a file of its own, so that the types compile side by side.
#include "diff_attn_fwd.hpp"

template void sgl::attn::forward_type<__bf16>(const AttnArgs&, hipStream_t);
