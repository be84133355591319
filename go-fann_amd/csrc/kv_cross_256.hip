// Cross attention over the 4-bit key/value cache for heads of 256 channels.
#include "kv_attention.hpp"

namespace gofann {
namespace kv {
GOFANN_KV_ATTEND(, 256, kCross);
}  // namespace kv
}  // namespace gofann
