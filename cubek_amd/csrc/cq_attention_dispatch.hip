// Which kernel a call of attention takes, and which object holds it.
#include "cq_attention_internal.hpp"

namespace cq {

hipError_t launch_append_F32(hipStream_t s, const AppendArgs& a);
hipError_t launch_append_F16(hipStream_t s, const AppendArgs& a);
hipError_t launch_append_BF16(hipStream_t s, const AppendArgs& a);

hipError_t launch_append(hipStream_t s, const AppendArgs& a) {
    return a.dtype == CQ_F32 ? launch_append_F32(s, a) : a.dtype == CQ_F16 ? launch_append_F16(s, a) : launch_append_BF16(s, a);
}

uint64_t attention_workspace_bytes(const AttentionArgs&) { return 0; }

hipError_t launch_attention(hipStream_t s, const AttentionArgs& a) { return launch_attention_general(s, a); }

}  // namespace cq
