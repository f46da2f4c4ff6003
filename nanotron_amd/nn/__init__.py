from nanotron_amd.nn.attention import attention
from nanotron_amd.nn.layer_norm import LayerNorm, layer_norm
from nanotron_amd.nn.loss import LinearCrossEntropy, linear_cross_entropy
from nanotron_amd.nn.rms_norm import RMSNorm, residual_rms_norm, rms_norm
from nanotron_amd.nn.rotary import RotaryEmbedding, rotary, rotary_frequencies

__all__ = ["LayerNorm", "layer_norm", "LinearCrossEntropy", "linear_cross_entropy", "RMSNorm", "rms_norm", "residual_rms_norm", "RotaryEmbedding", "rotary",
           "rotary_frequencies", "attention"]
