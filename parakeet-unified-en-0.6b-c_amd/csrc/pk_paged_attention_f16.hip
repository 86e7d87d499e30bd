// pk_paged_attention_f16.hip - the paged attention kernel over F16 caches.
#include "pk_paged_attention.h"

namespace pkgpu {
namespace decode {

hipError_t launch_paged_f16(int t, int dim, bool rules, const PagedArgs& a, dim3 grid, hipStream_t s)
{
    return t == F16 ? launch_paged<F16, F16>(dim, rules, a, grid, s) : hipErrorInvalidValue;
}

}  // namespace decode
}  // namespace pkgpu
