// pk_prompt_attention_e2m1.hip - the kernel of many new tokens over E2M1 caches.
#include "pk_prompt_attention.h"

namespace pkgpu {
namespace decode {

hipError_t launch_prompt_e2m1(int t, int dim, int sides, const PagedArgs& a, dim3 grid, hipStream_t s)
{
    return t == BF16 ? launch_prompt<E2M1, BF16>(dim, sides, a, grid, s)
         : t == F16 ? launch_prompt<E2M1, F16>(dim, sides, a, grid, s) : launch_prompt<E2M1, F32>(dim, sides, a, grid, s);
}

}  // namespace decode
}  // namespace pkgpu
