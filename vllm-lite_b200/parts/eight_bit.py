"""Linear layers in 8 bits: weights and the rows they meet are e4m3 values with a float32 scale a row.

`in_8_bits(plan)` gives a plan the same layers with these parts in the place of its pre-norm blocks of grouped-query attention and
SwiGLU; tensor names and shapes stay, weights are brought to 8 bits when the parts bind them.  A block then runs

    norm -> q/k/v product -> head norm, rotation, cache -> attention -> rows to 8 bits -> output product, added to the stream
    norm -> gate/up product with SwiGLU -> rows to 8 bits -> down product, which the next norm adds to the stream

where a norm's output is `Rows8` (`ops.add_rmsnorm_8bit`) and the products apply scales, bias, activation and residual themselves
(`ops.gemm_8bit`).  The stream stays float32; embedding, final norm, output head, attention and its cache stay as they were."""
from __future__ import annotations

import dataclasses
from dataclasses import dataclass

import torch

from ..csrc import ops
from .attention import GqaAttention
from .block import PreNormBlock
from .linear import Linear
from .mlp import SwiGLU
from .norm import RmsNorm
from .registry import BLOCKS, FEED_FORWARDS, MIXERS, NORMS
from .spec import AttentionSpec, BlockSpec, NormSpec, SwiGLUSpec


@dataclass
class Rows8:
    """Rows in 8 bits: row m stands for values[m] * scale[m]."""
    values: torch.Tensor                      # e4m3 [M, ops.eight_bit_columns(K)]
    scale: torch.Tensor                       # float32 [M]


def rows8_buffers(step, tag, rows, K):
    ws = step.workspace
    return (ws.get(step.tag + tag + ".8", (rows, ops.eight_bit_columns(K)), ops.E4M3), ws.get(step.tag + tag + ".scale", (rows,), torch.float32))


def to_rows8(a, step, tag) -> Rows8:
    """Rows of an activation (bfloat16 or float32 [M, K]) to 8 bits."""
    values, scale = rows8_buffers(step, tag, a.shape[0], a.shape[1])
    return Rows8(ops.rows_8bit(a, values, scale), scale)


class Linear8:
    """y = x W^T (+ b) with both operands in 8 bits; takes the place of a `Linear` whose weight it brings to 8 bits."""

    def __init__(self, linear: Linear, ctx):
        weight = linear.weight
        self.out_features, self.in_features = weight.shape
        values = torch.empty((self.out_features, ops.eight_bit_columns(self.in_features)), dtype=ops.E4M3, device=weight.device)
        self.scale = torch.empty(self.out_features, dtype=torch.float32, device=weight.device)
        ops.rows_8bit(weight, values, self.scale)
        self.weight = ops.pack_8bit(values)
        self.bias = linear.bias
        ctx.clustered.append(self.clusters)

    def _plan(self, M, overlapped=None):
        return ops.gemm_8bit_plan(M, self.out_features, self.weight.shape[1] * 128, overlapped)

    def clusters(self, M) -> bool:
        """Whether the product of M rows would run as clusters of blocks among dependent launches."""
        return self._plan(M, True)[1]

    def _product(self, rows, out, step, **how):
        M = rows.values.shape[0]
        floats = self._plan(M)[0]
        scratch = step.workspace.get(step.tag + "gemm_8bit.scratch", (floats,), torch.float32) if floats else None
        return ops.gemm_8bit(rows.values, rows.scale, self.weight, self.scale, out, bias=self.bias, err=step.err, scratch=scratch, **how)

    def _rows(self, a, step, tag) -> Rows8:
        return a if isinstance(a, Rows8) else to_rows8(a, step, tag + ".in")

    def __call__(self, a, step, tag, out_dtype=None):
        rows = self._rows(a, step, tag)
        out = step.workspace.get(step.tag + tag, (rows.values.shape[0], self.out_features), out_dtype or torch.bfloat16)
        return self._product(rows, out, step)

    def swiglu(self, a, step, tag):
        """silu(gate) * up, the weight holding blocks of SWIGLU_GROUP gate rows and their up rows."""
        rows = self._rows(a, step, tag)
        out = step.workspace.get(step.tag + tag + ".act", (rows.values.shape[0], self.out_features // 2), torch.bfloat16)
        return self._product(rows, out, step, act="silu", gated=True)

    def into_stream(self, a, stream, step, tag):
        """stream (float32 [M, out]) += y."""
        rows = self._rows(a, step, tag)
        self._product(rows, stream, step, residual=stream)

    def can_factor_norms(self, M) -> bool:
        return False

    factors_norms = can_factor_norms


@NORMS.register("rms_norm_8bit")
class RmsNorm8(RmsNorm):
    """An RMS norm whose output is `Rows8`; a pending residual is added into the stream on the way."""
    factorable = takes_sum = False

    def __call__(self, x, delta, step, rows=None, tag="norm"):
        R = x.shape[0] if rows is None else rows.shape[0]
        values, scale = rows8_buffers(step, tag, R, self.spec.size)
        return Rows8(ops.add_rmsnorm_8bit(x, delta, self.weight, self.spec.eps, values, scale, rows=rows), scale)


@MIXERS.register("gqa_attention_8bit")
class GqaAttention8(GqaAttention):
    """Grouped-query attention with its two products in 8 bits.  `sink`, when given, is the float32 stream that the result is added to."""

    def __init__(self, spec: AttentionSpec, weights: dict, ctx):
        super().__init__(spec, weights, ctx)
        if self.with_options:
            raise ValueError("products in 8 bits go with plain grouped-query attention: no gate, sink, cap or bias on its scores, no row work")
        self.qkv_proj, self.o_proj = Linear8(self.qkv_proj, ctx), Linear8(self.o_proj, ctx)


@FEED_FORWARDS.register("swiglu_8bit")
class SwiGLU8(SwiGLU):
    """SwiGLU with its products in 8 bits."""

    def __init__(self, spec: SwiGLUSpec, weights: dict, ctx):
        super().__init__(spec, weights, ctx)
        if self.group != ops.SWIGLU_GROUP:
            raise ValueError(f"SwiGLU in 8 bits: intermediate_size {spec.intermediate_size} is no multiple of {ops.SWIGLU_GROUP}")
        self.gate_up, self.down = Linear8(self.gate_up, ctx), Linear8(self.down, ctx)

    def __call__(self, h, step, sink=None, sums=False):
        act = self.gate_up.swiglu(h, step, "mlp.gate_up")
        if sink is not None:
            return self.down.into_stream(act, sink, step, "mlp.down")
        return self.down(act, step, "mlp.down", torch.float32 if sums else None)


@BLOCKS.register("pre_norm_8bit")
class PreNormBlock8(PreNormBlock):
    """x += mixer(norm1(x)); x += ffn(norm2(x)) with parts in 8 bits: the mixer's product adds its result into the stream, the feed-forward's
    is left for the next norm."""
    chains_norms = False

    def input_norm_for_fusion(self, M):
        return None

    def __call__(self, residual, step, cache):
        residual.cast = None
        h = self.norm1(residual.x, residual.pending, step, tag="norm1")
        self.mixer(h, step, cache, sink=residual.x)
        residual.pending = self.ffn(self.norm2(residual.x, None, step, tag="norm2"), step)


def in_8_bits(plan):
    """The plan with every layer's linear products in 8 bits.  Raises ValueError for a layer that has no such form."""
    layers = []
    for i, block in enumerate(plan.layers):
        mixer, ffn = getattr(block, "mixer", None), getattr(block, "ffn", None)
        norms = [getattr(block, n, None) for n in ("norm1", "norm2")]
        if not (isinstance(block, BlockSpec) and block.kind == "pre_norm" and isinstance(mixer, AttentionSpec) and mixer.kind == "gqa_attention"
                and isinstance(ffn, SwiGLUSpec) and ffn.kind == "swiglu" and all(isinstance(n, NormSpec) and n.kind == "rms_norm" for n in norms)):
            raise ValueError(f"layer {i} ({getattr(block, 'kind', '?')}: {getattr(mixer, 'kind', '?')}, {getattr(ffn, 'kind', '?')}) has no form in 8 "
                             f"bits; pre-norm blocks of grouped-query attention and SwiGLU with RMS norms have one")
        layers.append(dataclasses.replace(block, kind="pre_norm_8bit", mixer=dataclasses.replace(mixer, kind="gqa_attention_8bit"),
                                          ffn=dataclasses.replace(ffn, kind="swiglu_8bit"),
                                          norm1=dataclasses.replace(norms[0], kind="rms_norm_8bit"),
                                          norm2=dataclasses.replace(norms[1], kind="rms_norm_8bit")))
    return dataclasses.replace(plan, layers=tuple(layers))
