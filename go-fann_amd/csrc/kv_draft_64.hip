// Attention of drafted tokens over the 4-bit key/value cache for heads of 64 channels.
#include "kv_attention.hpp"

namespace gofann {
namespace kv {
GOFANN_KV_ATTEND(, 64, kDraft);
}  // namespace kv
}  // namespace gofann
