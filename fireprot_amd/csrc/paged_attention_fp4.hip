// Attention over caches in 4 bits, for each type of the queries.
#include "paged_attention.hpp"

namespace fpx {

hipError_t launch_paged_fp4(const PagedArgs& a, hipStream_t stream) {
  switch (a.dtype) {
    case 0: return launch_paged_type<float, Fp4Cache>(a, stream);
    case 1: return launch_paged_type<__bf16, Fp4Cache>(a, stream);
    default: return launch_paged_type<_Float16, Fp4Cache>(a, stream);
  }
}

}  // namespace fpx
