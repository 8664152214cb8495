from kfac_pytorch_amd.ops.factors import (ComputeA, ComputeG, extract_patches,
                                          factor_dims, sym_factor,
                                          update_running_avg)
from kfac_pytorch_amd.ops.grad_scale import (clip_by_global_norm,
                                             clip_grad_norm_, global_norm,
                                             kl_clip)
from kfac_pytorch_amd.ops.linalg import (add_diagonal_, eigen_precondition,
                                         inverse_precondition, mat_eig,
                                         mat_inv)
from kfac_pytorch_amd.ops.vocab_loss import (linear_cross_entropy,
                                             projection_loss)

__all__ = [
    "ComputeA", "ComputeG", "extract_patches", "factor_dims", "sym_factor",
    "update_running_avg", "add_diagonal_", "eigen_precondition",
    "inverse_precondition", "mat_eig", "mat_inv", "linear_cross_entropy",
    "projection_loss",
    "global_norm", "clip_by_global_norm", "clip_grad_norm_", "kl_clip",
]
