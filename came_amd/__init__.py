"""came_amd: the CAME 8-bit optimizer step for AMD Instinct MI355X (gfx950).

The optimizer classes keep the reference's (tukisuwa/CAME, ``came_pytorch``)
constructor arguments, ``step()`` semantics and state layout; the step itself
runs in ``libcame8.so`` (hand-written HIP kernels behind the C ABI in
``include/came8.h``).  Beside them: AdamW over many tensors with fp32 or 8-bit
moments, the clip by the global gradient norm, and the gated feed-forward block
with its gradients.
"""
from .adamw import AdamW, AdamW8bit  # noqa: F401
from .gated_ffn import gated_ffn  # noqa: F401
from .grad_clip import clip_grad_norm_, grad_norm  # noqa: F401
from .optim import CAME8bit, CAME8bit2D, CAME8bitFull, CAME8bitMemory, CAMECUDA  # noqa: F401

__all__ = ["CAME8bit", "CAME8bit2D", "CAME8bitFull", "CAME8bitMemory", "CAMECUDA", "AdamW", "AdamW8bit", "clip_grad_norm_",
           "grad_norm",
           "gated_ffn"]
__version__ = "0.1.0"
