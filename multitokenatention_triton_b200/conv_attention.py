"""Fused conv attention softmax(scale * conv(Q K^T)) V, with the reference's names.

Mirrors TritonAttention / TritonConvAttention (conv_attention_triton.py:359-502).  The reference returns
(O, QK) where QK is its S x S scratch of raw scores; this implementation keeps no such tensor, so the
second element is None.
"""
import torch
import torch.nn as nn

from . import ops
from .paged_cache import expand_heads


class TritonAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, Q, K, V, W, causal, softmax_scale):
        return ops.conv_attn_fwd(Q, K, V, W, causal, softmax_scale)

    @staticmethod
    def backward(ctx, dO):
        raise NotImplementedError("the B200 MTA library implements the forward pass only")


class TritonConvAttention(nn.Module):
    def __init__(self, channels, kernel_size, causal=False):
        super().__init__()
        self.channels = channels
        self.kernel_size = kernel_size if isinstance(kernel_size, tuple) else (kernel_size, kernel_size)
        self.causal = causal
        self.weight = nn.Parameter(torch.randn(channels, self.kernel_size[0], self.kernel_size[1]))
        self._init_parameters()

    def _init_parameters(self):
        with torch.no_grad():
            self.weight.zero_()
            self.weight[:, self.kernel_size[0] // 2, self.kernel_size[1] // 2] = 1.0

    def forward(self, Q, K, V, causal, softmax_scale):
        return TritonAttention.apply(Q, K, V, self.weight, causal, softmax_scale), None

    @property
    def query_history(self) -> int:
        """Queries that a cache has to keep for this module."""
        return self.kernel_size[0]

    def forward_cached(self, Q, K, V, cache, batch, softmax_scale=None, layer: int = 0, max_length=None):
        """forward (causal) for new tokens of the sequences of a PagedKVCache: Q (B,H,T,D), K, V (B,kv heads,T,D) -> ((B,H,T,D), None), and the tokens
        are kept.  T, `batch` and `max_length` as in MTAAttentionTriton.forward_cached."""
        if torch.is_grad_enabled() and any(t.requires_grad for t in (Q, K, V, self.weight)):
            raise NotImplementedError("TritonConvAttention with a cache has no backward pass: call it under torch.no_grad()")
        prompt = Q.size(2) != 1
        if prompt and not batch.from_empty:
            raise NotImplementedError("several new tokens at once are a prompt: the sequences must have been empty")
        longest = cache.longest(batch, max_length)
        # as in MTAAttentionTriton.forward_cached: refusals before the first write
        cache.check_reader("TritonConvAttention", self.channels, self.kernel_size[0])
        ops.check_decode("conv_attn_decode", 1 if prompt else len(batch.slots), cache.n_heads, cache.n_kv_heads, cache.head_dim, *self.kernel_size, longest)
        if prompt:
            cache.check_step(batch, K, layer)
            out = ops.conv_attn_fwd(*expand_heads(*batch.without_padding(Q, K, V)), self.weight, True, softmax_scale)
            cache.append(batch, K, V, Q, layer)
            return out, None
        tensors = cache._layer(layer)
        cache._append(batch, K, V, Q, layer, tensors)
        return ops.conv_attn_decode_fwd(*tensors, self.weight, softmax_scale, longest,
                                        slots=batch.slot_ids), None
