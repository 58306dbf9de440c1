from isa_b200.kernels.transformer_norm.layer_norm import (  # noqa: F401
    cuda_add_layer_norm,
    cuda_layer_norm,
)
