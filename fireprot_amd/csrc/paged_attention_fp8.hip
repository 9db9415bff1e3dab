// Attention over FP8 caches, for each type of the queries.
#include "paged_attention.hpp"

namespace fpx {

hipError_t launch_paged_fp8(const PagedArgs& a, hipStream_t stream) {
  switch (a.dtype) {
    case 0: return launch_paged_type<float, Fp8Cache>(a, stream);
    case 1: return launch_paged_type<__bf16, Fp8Cache>(a, stream);
    default: return launch_paged_type<_Float16, Fp8Cache>(a, stream);
  }
}

}  // namespace fpx
