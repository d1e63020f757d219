// paged_attention.cuh for __nv_bfloat16.
#include "paged_attention.cuh"

namespace inferc_dev {
namespace paged {

template <>
void launch_attend<__nv_bfloat16>(const AttendArgs& g, cudaStream_t st) {
  launch_attend_any<__nv_bfloat16>(g, st);
}

}  // namespace paged
}  // namespace inferc_dev
