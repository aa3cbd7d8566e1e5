"""Functional layers, losses, initialisers, and the activations re-exported from ``ops``
(reference: nabla/nn/functional/__init__.py)."""
from ...ops.heads import norm_rotary, norm_rotary_reference, packed_norm_rotary, packed_norm_rotary_reference
from ...ops.serving import adjust_logits, cached_attention, init_kv_cache, kv_cache_read, kv_cache_write, sample_tokens, shared_prefix_attention
from ...ops.unary import gelu, relu, sigmoid, silu, softmax, tanh
from .init import he_normal, xavier_normal
from .layers import (dropout, embedding, layer_norm, layer_norm_reference, linear, scaled_dot_product_attention,
                     scaled_dot_product_attention_reference, use_fused)
from .losses import cross_entropy_loss, cross_entropy_loss_reference, mse_loss
