"""MI355X (gfx950) implementation of the SpartonHead forward and backward.

`SpartonHead` and the ops `torch.ops.sparton.fused_sparton_fwd/_bwd/_encode` run
on hand-written HIP kernels in libsparton_hip.so (C ABI: include/sparton.h).
`SpartonMLMTransform` (ops `sparton::mlm_transform_fwd/_bwd`) is the dense + gelu +
LayerNorm step that produces the head's input, its GEMMs in hipBLASLt and the rest fused.
`sparton_amd.loss` is the SPLADE training loss on the head's reps (InfoNCE + L1 + FLOPS
regularisers, ops `sparton::splade_loss_fwd/_bwd`), fused into two HIP passes.
Around them, a backbone layer's own work: `sparton_amd.attention` (padded, causal, shared key heads; ops
`sparton::attention_fwd/_bwd`) and `SpartonLayerNorm` (with the residual sum; ops
`sparton::layer_norm_fwd/_bwd`); and `sparton_amd.loss.preference_loss` on pairs of reps (ops
`sparton::preference_fwd/_bwd`).
`SpartonRMSNorm` (with the residual's addition, and rows in e4m3; ops `sparton::rms_norm_fwd/_bwd/_8bit`),
`SpartonEmbedding` (gradient by sorted tokens; ops `sparton::embedding_fwd/_bwd`) and `SpartonGatedMLP` (ops
`sparton::gated_fwd/_bwd/_infer/_8bit`) are the rest of a gated backbone's layer.
Importing the package registers the ops; the library itself is loaded on first use
and raises if it has not been built (`python -m sparton_amd.build`).
"""
from .head import SpartonHead
from . import ops
from . import transform
from .transform import SpartonMLMTransform
from . import attention, embedding, feed_forward, norm
from .embedding import SpartonEmbedding
from .feed_forward import SpartonGatedMLP
from .norm import SpartonLayerNorm, SpartonRMSNorm
from . import loss
from .loss import preference_loss, splade_loss

__all__ = ["SpartonHead", "SpartonMLMTransform", "SpartonLayerNorm", "SpartonRMSNorm", "SpartonEmbedding",
           "SpartonGatedMLP", "ops", "transform", "attention", "norm", "embedding", "feed_forward", "loss", "splade_loss",
           "preference_loss"]
