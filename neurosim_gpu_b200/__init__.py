"""B200-native dendritic tick for NeuroSim-GPU (sm_100a CUDA behind a C ABI).

Drop-in for the reference's native dendritic runtimes: the same classes,
constructor arguments, ``step`` signature, state tensors and checkpoint
layout, with every inference tick running in ``libneurosim_b200.so``.
"""

from .dynamics import DendriticDynamics, Dynamics
from .logits import adjust_logits
from .microscale import (Nvfp4Matrix, check_product_status, nvfp4_product, nvfp4_readout,
                         quantize_nvfp4)
from .native import load_native_extension
from .precision import PRECISIONS, encode_sparse_weights, quantize_dequantize
from .runtime import (NativeDendriticMatrixRuntime, NativeDendriticPELSRuntime, RuntimeStats,
                      validate_emission_threshold)
from .stimulus import stimulus_drive, stimulus_gradient
from .tokens import generate_tokens
from .topology import SparseTopology, random_topology

__all__ = [
    "DendriticDynamics", "Dynamics", "NativeDendriticMatrixRuntime",
    "NativeDendriticPELSRuntime", "Nvfp4Matrix", "PRECISIONS", "RuntimeStats", "SparseTopology",
    "adjust_logits", "check_product_status", "encode_sparse_weights", "generate_tokens",
    "load_native_extension",
    "nvfp4_product", "nvfp4_readout", "quantize_dequantize", "quantize_nvfp4",
    "random_topology", "stimulus_drive", "stimulus_gradient", "validate_emission_threshold",
]
