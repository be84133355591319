// Attention over the 4-bit key/value cache for heads of 256 channels.
#include "kv_attention.hpp"

namespace gofann {
namespace kv {
template void attend_launch<Bf16, 256>(const AttendArgs&, const AttendPlan&, hipStream_t);
template void attend_launch<F16, 256>(const AttendArgs&, const AttendPlan&, hipStream_t);
}  // namespace kv
}  // namespace gofann
