"""B200 kernel wrappers (same import surface as ghostweight_triton.kernels).

Beyond that surface, submodules hold the pieces a layer is built from: packed
weights (``gather``), products over them with bias, activation and residual in
the epilogue (``matmul``), and the row operators in front of them, residual +
RMS norm and e4m3 rows (``norm``).
"""

from ghostweight_triton_b200.kernels.mask import dead_neuron_mask
from ghostweight_triton_b200.kernels.gather import gather_compact
from ghostweight_triton_b200.kernels.matmul import ghostweight_matmul

__all__ = [
    "dead_neuron_mask",
    "gather_compact",
    "ghostweight_matmul",
]
