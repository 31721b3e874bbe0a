"""Device operations of the framework as plain functions over torch tensors.

Each function is a thin wrapper over hand-written sm_100a kernels (``nangila._cuda``); the fused
exchange kernels are driven through the engines in ``nangila.parallel`` instead.

Norms, rotary positions, updates, embeddings, dropout and the head's loss take part in reverse-mode autograd only: CUDA tensors with a forward-mode tangent, and calls under
``torch.jit.trace``, ``make_fx`` or fake tensors, raise ``NotImplementedError``. Subnormal numbers are kept, as by PyTorch's operations.
"""
from .masks import dropout  # noqa: F401
from .muon import muon_step, orthogonalize  # noqa: F401
from .reductions import absmax_percentile, crc32, quantizer_gamma, state_hash  # noqa: F401
from .norm import add_rms_norm, rms_norm, rms_norm_fp8  # noqa: F401
from .positions import rotary, rotary_table  # noqa: F401
from .sculptor_stats import DeviceSculptor  # noqa: F401
from .vocabulary import embedding, linear_cross_entropy  # noqa: F401
