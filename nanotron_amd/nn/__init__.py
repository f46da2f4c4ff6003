from nanotron_amd.nn.layer_norm import LayerNorm, layer_norm
from nanotron_amd.nn.loss import LinearCrossEntropy, linear_cross_entropy

__all__ = ["LayerNorm", "layer_norm", "LinearCrossEntropy", "linear_cross_entropy"]
