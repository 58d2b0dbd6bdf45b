// b200fa_window.cu -- the sliding-window kernels (B200FA_FLAG_WINDOW): the
// kernel source of fa_kernel.cuh compiled with B200FA_WINDOW = 1.  Query row i
// attends keys i - window < j <= i and the first `sinks` keys; key blocks that
// no row of a work item sees are never loaded, so the work is that of the
// window and not of the sequence.  Launched by b200fa.cu.
#define B200FA_CAUSAL 1
#define B200FA_WINDOW 1
// The roles that are plain (non-template) device functions get their own
// names here, as in the causal translation unit.
#define s_issuer_role s_issuer_role_window
#define pv_issuer_role pv_issuer_role_window
#define watch_role watch_role_window
#define forward_role forward_role_window
#define load_role load_role_window
#include "fa_kernel.cuh"

using namespace b200fa;

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    b200_fa_fp16_window_kernel(const __grid_constant__ FwdParams p) {
  attention_fwd_body<0, false>(p);
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    b200_fa_fp32_window_kernel(const __grid_constant__ FwdParams p) {
  attention_fwd_body<1, false>(p);
}
