"""MI355X-native cascaded low-precision matmul (the Linear-layer hot path of basedxl)."""
from .cascaded_lowp_matmul import (cascaded_lowp_matmul, cascaded_lowp_matmul_grouped,  # noqa: F401
                                   cascaded_lowp_matmul_prepared, PreparedWeight, tensor_scale_exp,
                                   LeftSlots, ChainedWeight, cascaded_lowp_matmul_chained, cascaded_lowp_matmul_glu_chained)
from .block_scaled import BlockScaledWeight, block_scaled_matmul  # noqa: F401
from .gated_norm import gated_add_norm  # noqa: F401
from .gradient_clip import clip_grad_norm_, clip_gradients, gradient_norm  # noqa: F401
from .layer_norm import add_layer_norm, layer_norm  # noqa: F401
from .matmul_epilogue import cascaded_lowp_matmul_epilogue  # noqa: F401
from .modules import (BasedXLFusedKV, BasedXLLowPConv1x1, BasedXLLowPGEGLU, BasedXLLowPLinear, patch_linear_layers,  # noqa: F401
                      patch_pointwise_convs, BasedXLChainedFeedForward, chain_feed_forward_layers, BasedXLLayerNorm, patch_layer_norms)

__all__ = ["cascaded_lowp_matmul", "cascaded_lowp_matmul_grouped", "cascaded_lowp_matmul_prepared", "PreparedWeight", "tensor_scale_exp",
           "LeftSlots", "ChainedWeight", "cascaded_lowp_matmul_chained", "cascaded_lowp_matmul_glu_chained",
           "BasedXLChainedFeedForward", "chain_feed_forward_layers",
           "BasedXLLowPLinear", "BasedXLLowPConv1x1", "BasedXLLowPGEGLU", "BasedXLFusedKV",
           "patch_linear_layers", "patch_pointwise_convs", "layer_norm", "add_layer_norm", "cascaded_lowp_matmul_epilogue",
           "BasedXLLayerNorm", "patch_layer_norms", "gated_add_norm", "BlockScaledWeight", "block_scaled_matmul", "gradient_norm",
           "clip_gradients", "clip_grad_norm_"]
