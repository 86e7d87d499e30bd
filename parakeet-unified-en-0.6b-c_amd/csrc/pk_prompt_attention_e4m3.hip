// pk_prompt_attention_e4m3.hip - the kernel of many new tokens over E4M3 caches.
#include "pk_prompt_attention.h"

namespace pkgpu {
namespace decode {

hipError_t launch_prompt_e4m3(int t, int dim, int sides, const PagedArgs& a, dim3 grid, hipStream_t s)
{
    return t == BF16 ? launch_prompt<E4M3, BF16>(dim, sides, a, grid, s)
         : t == F16 ? launch_prompt<E4M3, F16>(dim, sides, a, grid, s) : launch_prompt<E4M3, F32>(dim, sides, a, grid, s);
}

}  // namespace decode
}  // namespace pkgpu
