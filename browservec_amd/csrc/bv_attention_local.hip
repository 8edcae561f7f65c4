// Attention over a window of keys about a query's place and a few first keys: the
// kernels of bv_attention_device.h.
#include "bv_attention_device.h"

namespace bvk {

hipError_t launch_attention_local(const AttentionArgs &a, void *ws, hipStream_t s) { return launch_attention_as<true>(a, ws, s); }

}  // namespace bvk
