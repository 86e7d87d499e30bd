// pk_paged_attention_e4m3.hip - the paged attention kernel over E4M3 caches.
#include "pk_paged_attention.h"

namespace pkgpu {
namespace decode {

hipError_t launch_paged_e4m3(int t, int dim, bool rules, const PagedArgs& a, dim3 grid, hipStream_t s)
{
    return t == BF16 ? launch_paged<E4M3, BF16>(dim, rules, a, grid, s)
         : t == F16 ? launch_paged<E4M3, F16>(dim, rules, a, grid, s) : launch_paged<E4M3, F32>(dim, rules, a, grid, s);
}

}  // namespace decode
}  // namespace pkgpu
