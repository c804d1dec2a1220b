"""B200-native bidirectional attention (forward + backward, dense and packed varlen) for
nanobrain's 3D ViT-B masked autoencoder: hand-written sm_100a kernels behind a C ABI, wrapped
as ``torch.library`` custom ops with the ``F.scaled_dot_product_attention`` signature; around it the norms
and rotation of queries and keys and a gated feed-forward block."""

from .block_ops import gated_mlp, qk_norm_rope
from .host_pipeline import HostPipeline
from .ops import check_status, sdpa, sdpa_varlen, selftest_mma

__all__ = ["sdpa", "sdpa_varlen", "qk_norm_rope", "gated_mlp", "check_status", "selftest_mma", "HostPipeline"]
