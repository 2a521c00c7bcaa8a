"""B200-native fused FP8 block-scale MoE layer with DeepSeek-V3 routing.

Public surface:
  kernel(...)            drop-in for the reference solution's entry point
  inputs.make_inputs     seeded synthetic inputs with the definition's shapes
  ep.EPMoE               expert-parallel layer over NCCL (one process per GPU)
  sort_tokens, dispatch, combine
                         tokens sorted by expert and back, with gradients
  swiglu                 silu(gate) * up, its input kept for the gradient in 8 bits
  quantize_w4, W4Weights, w4_matvec, moe_w4
                         expert products with 4-bit weights, and the layer with them

The directory name is not a Python identifier; load the package with
``__graft_entry__.load_package()``, which registers it as ``fib_b200``.
"""

from .kernel import kernel  # noqa: F401
from . import inputs  # noqa: F401
from .tokens import TokenOrder, combine, dispatch, sort_tokens  # noqa: F401
from .activation import swiglu  # noqa: F401
from .w4 import W4Weights, moe_w4, quantize_w4, w4_matvec  # noqa: F401
