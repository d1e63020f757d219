// paged_attention.cuh for __half.
#include "paged_attention.cuh"

namespace inferc_dev {
namespace paged {

template <>
void launch_attend<__half>(const AttendArgs& g, cudaStream_t st) {
  launch_attend_any<__half>(g, st);
}

}  // namespace paged
}  // namespace inferc_dev
