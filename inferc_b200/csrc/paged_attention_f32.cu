// paged_attention.cuh for float.
#include "paged_attention.cuh"

namespace inferc_dev {
namespace paged {

template <>
void launch_attend<float>(const AttendArgs& g, cudaStream_t st) {
  launch_attend_any<float>(g, st);
}

}  // namespace paged
}  // namespace inferc_dev
