from .chunk import chunk_cyfa
from .fused_recurrent import fused_recurrent_cyfa
from .norm_ops import residual_norm
from .orthogonal import orthogonalize
from .token_ops import TokenLogProbs, embed_tokens, token_log_probs

__all__ = ["chunk_cyfa", "fused_recurrent_cyfa", "TokenLogProbs", "embed_tokens",
           "orthogonalize", "residual_norm", "token_log_probs"]
