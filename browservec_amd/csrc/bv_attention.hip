// Attention over all of a sequence's keys, or those up to a query's place: the
// kernels of bv_attention_device.h.
#include "bv_attention_device.h"

namespace bvk {

size_t attention_workspace(const AttentionArgs &a) {
    uint32_t chunk;
    const uint32_t splits = splits_of(a, &chunk);
    return splits > 1 ? splits * part_bytes(a) : 0;
}

hipError_t launch_attention(const AttentionArgs &a, void *ws, hipStream_t s) {
    return a.local ? launch_attention_local(a, ws, s) : launch_attention_as<false>(a, ws, s);
}

}  // namespace bvk
