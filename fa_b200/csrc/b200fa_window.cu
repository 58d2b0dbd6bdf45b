// b200fa_window.cu -- the sliding-window kernels (B200FA_FLAG_WINDOW): the
// kernel source of fa_kernel.cuh compiled with B200FA_WINDOW = 1.  Query row i
// attends keys i - window < j <= i and the first `sinks` keys; key blocks that
// no row of a work item sees are never loaded, so the work is that of the
// window and not of the sequence.  Launched by b200fa.cu.  B=4, Hq=32, Hkv=8,
// N=8192, W=1024, S=4: 0.75 ms; B=1, Hq=12, N=32700, W=4096, S=128: 0.82 ms (short
// bursts; 0.84 and 0.86 under the power cap).  P is rounded to FP16, as the tensor
// cores take it: errors against 64 bits are 2.8e-4 beside 2.0e-4 with P in 32 bits.
#define B200FA_CAUSAL 1
#define B200FA_WINDOW 1
#ifndef B200FA_POLY_PAIRS_FP32
#define B200FA_POLY_PAIRS_FP32 0  // all exponentials through MUFU
#endif
// The roles that are plain (non-template) device functions get their own
// names here, as in the causal translation unit.
#define s_issuer_role s_issuer_role_window
#define pv_issuer_role pv_issuer_role_window
#define watch_role watch_role_window
#define forward_role forward_role_window
#define load_role load_role_window
#include "fa_kernel.cuh"

using namespace b200fa;

// One kernel for both variants: FP32 softmax statistics and sums, P in FP16.
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    b200_fa_window_kernel(const __grid_constant__ FwdParams p) {
  attention_fwd_body<1, false>(p);
}
