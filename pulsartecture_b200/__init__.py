"""pulsartecture_b200: Ultra-RWKA's FA-KLA (causal temperature-modulated
kernelized linear attention) on NVIDIA B200, sm_100a.

Layout:
  csrc/        CUDA kernels (tcgen05 phi GEMM, tcgen05 chunk scan, decode,
               CUDA-core fp32 paths, gated scan, logits rows) and the C ABI
               (include/fakla.h)
  _lib.py      ctypes binding of lib/libfakla.so
  backend/     torch-tensor front end (reference: ultra_rwka.backend.interface);
               gated_scan, token_logprobs and distill_topk
  kernels/     FeatureMap / LearnablePositiveMap (reference: ultra_rwka.kernels)
  components/  LinearProjection (reference: ultra_rwka.components.projections)
  attention/   TMLinKernelAttn, TemperatureFunction, fa_kla, fa_kla_host, fa_kla_decode
               (reference: ultra_rwka.attention), GatedRecurrence
"""
__version__ = "0.1.0"

from .attention import (  # noqa: F401,E402
    GatedRecurrence,
    TemperatureFunction,
    TMLinKernelAttn,
    fa_kla,
    fa_kla_decode,
    fa_kla_host,
)
from .backend import (  # noqa: F401,E402
    TokenLogprobs,
    distill_topk,
    fa_kla_attention,
    gated_scan,
    gated_scan_step,
    token_logprobs,
)
from .kernels import FeatureMap, LearnablePositiveMap  # noqa: F401,E402
