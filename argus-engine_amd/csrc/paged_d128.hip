// paged_attention at head_dim 128.
#include "paged_launch.hpp"

namespace argus_paged {

int launch_paged_128(argus_hip_ctx *ctx, const PagedParams &dp, const PagedParams &cp, bool f32, bool cap, hipStream_t stream) {
  return launch_call<128>(ctx, dp, cp, f32, cap, stream);
}

}  // namespace argus_paged
