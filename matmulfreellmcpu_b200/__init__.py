"""B200-native (sm_100a) HGRN-Bit engine: a drop-in for the matmulfreellmCPU hot path.

The product is ``_lib/libmmfree_cuda.so`` (CUDA kernels + the C ABI of
``include/mmfree_cuda.h``); this package builds it (``build``), binds it (``_lib``), mirrors
the reference's C++ API in Python (``api``; ``bind/`` calls the recurrent-block operators on
torch tensors) and writes seeded ``model.mmfree`` blobs (``blob``).
"""
from .api import (Config, Model, MmfreeError, add_rmsnorm_quant, bitlinear,  # noqa: F401
                  bitlinear_cluster, causal_conv, causal_conv_step, hgrn_scan, int4_matvec,
                  pack_ternary_host, packed_bytes, repack_ternary, rmsnorm, rmsnorm_swishgate,
                  selective_scan, selective_step, swiglu, ternary_matmul)
