// pk_paged_attention_bf16.hip - the paged attention kernel over BF16 caches.
#include "pk_paged_attention.h"

namespace pkgpu {
namespace decode {

hipError_t launch_paged_bf16(int t, int dim, const PagedArgs& a, dim3 grid, hipStream_t s)
{
    return t == BF16 ? launch_paged<BF16, BF16>(dim, a, grid, s)
         : t == F32 ? launch_paged<BF16, F32>(dim, a, grid, s) : hipErrorInvalidValue;
}

}  // namespace decode
}  // namespace pkgpu
