"""fa_b200 -- B200 (sm_100a) flash-attention forward behind the platelett/fa
harness API.

Layout:
  csrc/      CUDA kernels (tcgen05 + TMA, warp-specialised) and the C ABI
  build.py   hash-keyed nvcc build of libb200fa.so
  lib.py     ctypes binding of the C ABI (include/b200fa.h)
  ops.py     torch-facing Operator (reference binding.py semantics)
  paged.py   serving: page tables, cache append, attention over a paged cache
  rotary.py  rotary positions
  calls.py   the serving calls' host side in C++ (csrc/torch_calls.cpp)
  shard.py   multi-GPU partition of the (b, hq, q-block) unit grid
  core/      harness mirror: contract, registry, drivers, bench, runner,
             schedule, profiler (reference core/*)
  problem/   Case matrix and canonical inputs (reference problem/*)
  backends/  b200_fa_fp16, b200_fa_fp32 and the FP32 torch reference backend
"""

__all__ = ["ops", "lib", "build"]
