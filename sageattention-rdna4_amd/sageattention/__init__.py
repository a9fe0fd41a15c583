"""sageattention for AMD Instinct MI355X (gfx950): quantized attention as a drop-in `sageattn`, its
serving form over a quantized K/V cache (`KVCache`, `sageattn_cached`, `apply_rotary`), and its
training form (`sageattn_train`, `sageattn_backward`), with the root-mean-square norm around it.

`sageattn` deliberately has no `attn_mask` parameter in its signature: callers such as ComfyUI
probe for its absence (`sageattention/__init__.py:4-11` of the reference).
"""
from .cache import KVCache, apply_rotary, rotary_table, sageattn_cached  # noqa: F401
from .core import sageattn  # noqa: F401
from .norm import rms_norm, rms_norm_backward, rms_norm_quant  # noqa: F401
from .train import sageattn_backward, sageattn_train  # noqa: F401

__version__ = "0.1.0+mi355"
__all__ = ["sageattn", "KVCache", "apply_rotary", "rotary_table", "sageattn_cached",
           "sageattn_train", "sageattn_backward", "rms_norm", "rms_norm_quant", "rms_norm_backward"]
