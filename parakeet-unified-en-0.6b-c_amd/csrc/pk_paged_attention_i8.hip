// pk_paged_attention_i8.hip - the paged attention kernel over I8 caches.
#include "pk_paged_attention.h"

namespace pkgpu {
namespace decode {

hipError_t launch_paged_i8(int t, int dim, bool rules, const PagedArgs& a, dim3 grid, hipStream_t s)
{
    return t == BF16 ? launch_paged<I8, BF16>(dim, rules, a, grid, s)
         : t == F16 ? launch_paged<I8, F16>(dim, rules, a, grid, s) : launch_paged<I8, F32>(dim, rules, a, grid, s);
}

}  // namespace decode
}  // namespace pkgpu
