// pk_prompt_attention_bf16.hip - the kernel of many new tokens over BF16 caches.
#include "pk_prompt_attention.h"

namespace pkgpu {
namespace decode {

hipError_t launch_prompt_bf16(int t, int dim, int sides, const PagedArgs& a, dim3 grid, hipStream_t s)
{
    return t == BF16 ? launch_prompt<BF16, BF16>(dim, sides, a, grid, s)
         : t == F32 ? launch_prompt<BF16, F32>(dim, sides, a, grid, s) : hipErrorInvalidValue;
}

}  // namespace decode
}  // namespace pkgpu
