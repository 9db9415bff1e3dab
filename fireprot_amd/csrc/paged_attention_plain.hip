// Attention over plain caches (the queries' own type).
#include "paged_attention.hpp"

namespace fpx {

hipError_t launch_paged_f32(const PagedArgs& a, hipStream_t stream) {
  return launch_paged_type<float, float>(a, stream);
}
hipError_t launch_paged_bf16(const PagedArgs& a, hipStream_t stream) {
  return launch_paged_type<__bf16, __bf16>(a, stream);
}
hipError_t launch_paged_f16(const PagedArgs& a, hipStream_t stream) {
  return launch_paged_type<_Float16, _Float16>(a, stream);
}

}  // namespace fpx
