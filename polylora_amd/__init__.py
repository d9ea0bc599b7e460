"""polylora_amd — multi-LoRA inference with gfx950 HIP SGMV kernels.

Same public names as the reference package ``polylora`` (src/polylora/__init__.py:1-18).
What a decode step does beside the Linears is in ``polylora_amd.paged`` (append
to a paged key-value cache, attention of one new token or of several drafted
ones over it), ``polylora_amd.drafts`` (which drafts stay) and
``polylora_amd.logits`` (penalties, biases and grammar masks), which the
reference leaves to the wrapped model and its caller.
"""

from .cache import GpuAdapterCache
from .config import CustomLoraConfig, PolyLoraConfig
from .context import LoraBatchContext
from .layers import MultiLoraLinear
from .model import CustomPeftModel, PolyLoraModel
from .store import CpuAdapterStore, DiskAdapterCache

__all__ = [
    "CpuAdapterStore",
    "CustomLoraConfig",
    "CustomPeftModel",
    "DiskAdapterCache",
    "GpuAdapterCache",
    "LoraBatchContext",
    "MultiLoraLinear",
    "PolyLoraConfig",
    "PolyLoraModel",
]
