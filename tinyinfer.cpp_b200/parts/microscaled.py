"""Layers whose products run on weights in the microscaled 4-bit format (``kernels/mx_ops.py``), activations in 8 bits.

``microscaled_plan`` rewrites a plan of pre-norm layers with plain attention and SwiGLU: the four parts of a layer are replaced
by the ones below, which read the same tensors and quantise the matrices when they are loaded; embedding, final norm and head
stay as they are.  A layer is then

    h = norm1(x) in 8 bits;   d = Wo quantised(attention(Wqkv h))
    x += d, h = norm2(x) in 8 bits (one launch);   x += Wdown (silu(Wgate h) * (Wup h) in 8 bits)

with float32 residual and sums, keys and values and the attention itself as in a bfloat16 engine.  Weights take 0.53 bytes each
instead of 2, which is what bounds a step of few tokens."""
from __future__ import annotations

import dataclasses

import torch

from ..config.plan import ModelPlan, PartSpec
from .attention import Attention
from .base import register_part
from .block import PreNormBlock
from .mlp import SwiGLU
from .norm import RMSNorm

_KINDS = {"block": {"prenorm": "mx_prenorm"}, "mixer": {"attention": "mx_attention"}, "ffn": {"swiglu": "mx_swiglu"},
          "mixer_norm": {"rmsnorm": "mx_rmsnorm"}, "ffn_norm": {"rmsnorm": "mx_rmsnorm"}}
FORMATS = ("mxfp4",)


def microscaled_plan(plan: ModelPlan, weights: str) -> ModelPlan:
    """``plan`` with the layers' matrices in the format ``weights``."""
    if weights not in FORMATS:
        raise ValueError(f"weights must be one of {', '.join(FORMATS)}, got {weights!r}")

    def replaced(i, role, spec):
        if spec is None or spec.kind not in _KINDS[role]:
            raise ValueError(f"weights={weights!r}: layer {i} of {plan.architecture} has "
                             f"{'no ' + role if spec is None else f'a {role} of kind {spec.kind!r}'}, which has no such form")
        return PartSpec(_KINDS[role][spec.kind], spec.params)

    layers = []
    for i, layer in enumerate(plan.layers):
        if layer.mixer_post_norm is not None or layer.ffn_post_norm is not None:
            raise ValueError(f"weights={weights!r}: layer {i} of {plan.architecture} norms what its sublayers give")
        layers.append(dataclasses.replace(layer, **{role: replaced(i, role, getattr(layer, role)) for role in _KINDS}))
    return dataclasses.replace(plan, layers=layers)


class MxRMSNorm(RMSNorm):
    """RMS norm whose rows come out in 8 bits; ``delta`` is added to ``x`` first, in the same launch."""

    def forward(self, ops, x, out_dtype, delta=None):
        return ops.mx_rmsnorm(x, self.weight, self.eps, bits=8, delta=delta)


class MxAttention(Attention):
    """Causal grouped-query attention whose projections have 4-bit weights.  It writes its output to ``out`` instead of adding
    it to the residual: the norm behind it adds."""

    def load_weights(self, tensors, ops):
        q, k, v = (tensors[n + "_proj.weight"].to(torch.float32) for n in "qkv")
        self.w_qkv = ops.mx_pack_linear(torch.cat([q, k, v], dim=0))
        self.w_o = ops.mx_pack_linear(tensors["o_proj.weight"])
        self.q_norm = tensors["q_norm.weight"].to(torch.float32).contiguous()
        self.k_norm = tensors["k_norm.weight"].to(torch.float32).contiguous()

    def forward(self, ops, h, out, step, cache):
        t, dev, act = h.rows, out.device, step.act_dtype
        qkv = torch.empty((t, self.nq + 2 * self.nk), dtype=torch.float32, device=dev)
        ops.mx_linear(h, self.w_qkv, qkv)
        q, attended = (torch.empty((t, self.nq), dtype=act, device=dev) for _ in range(2))
        ops.qk_norm_rope_store(qkv, self.q_norm, self.k_norm, self.eps, self.position.rotation(dev), step, cache, q,
                               self.num_heads, self.num_kv_heads, self.head_dim)
        ops.paged_attention(q, step, cache, attended, self.num_heads, self.num_kv_heads, self.head_dim, self.window, self.scale)
        ops.mx_linear(ops.mx_quantize(attended, 8), self.w_o, out)


class MxSwiGLU(SwiGLU):
    """SwiGLU with 4-bit weights, its inner rows in 8 bits."""

    def load_weights(self, tensors, ops):
        g, u = (tensors[n + "_proj.weight"].to(torch.float32) for n in ("gate", "up"))
        self.w_gate_up = ops.mx_pack_gate_up(g, u)
        self.w_down = ops.mx_pack_linear(tensors["down_proj.weight"])

    def forward(self, ops, h, residual, step):
        inner = ops.mx_linear_glu(h, self.w_gate_up, self.intermediate_size, bits=8)
        ops.mx_linear(inner, self.w_down, residual, accumulate=True)


class MxPreNormBlock(PreNormBlock):
    def forward(self, ops, x, step, cache):
        mixed = torch.empty_like(x)
        self.mixer.forward(ops, self.mixer_norm.forward(ops, x, step.act_dtype), mixed, step, cache)
        self.ffn.forward(ops, self.ffn_norm.forward(ops, x, step.act_dtype, delta=mixed), x, step)


register_part("norm", "mx_rmsnorm", MxRMSNorm)
register_part("mixer", "mx_attention", MxAttention)
register_part("ffn", "mx_swiglu", MxSwiGLU)
register_part("block", "mx_prenorm", MxPreNormBlock)
