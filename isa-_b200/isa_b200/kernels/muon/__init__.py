from isa_b200.kernels.muon.newton_schulz import (  # noqa: F401
    NS_COEFFICIENTS,
    cuda_muon_step,
    cuda_orthogonalize,
)
