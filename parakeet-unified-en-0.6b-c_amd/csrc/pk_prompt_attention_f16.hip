// pk_prompt_attention_f16.hip - the kernel of many new tokens over F16 caches.
#include "pk_prompt_attention.h"

namespace pkgpu {
namespace decode {

hipError_t launch_prompt_f16(int t, int dim, int sides, const PagedArgs& a, dim3 grid, hipStream_t s)
{
    return t == F16 ? launch_prompt<F16, F16>(dim, sides, a, grid, s) : hipErrorInvalidValue;
}

}  // namespace decode
}  // namespace pkgpu
