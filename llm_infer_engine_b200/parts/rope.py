"""Rotary position encoding (rotate-half pairing) with optional llama3 frequency scaling.

Frequencies: inv_i = theta^(-2i/rot_dim), i < rot_dim/2 (src/rope.py:9 of the reference); the
llama3 rule rescales them by wavelength (src/rope.py:11-30). Angles p * inv_i, their cosines
and sines are float32 (src/rope.py:35-37). The reference then rounds cos and sin to the
activation dtype and rotates in it (src/rope.py:43-44,75-86); here the table stays float32 and
the rotation is done in float32 in both precisions. Rotation is fused with the cache write
(src/rope.py:122-185): keys are stored rotated.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from ..kernels import ops
from .base import PositionEncoding, register_position_encoding


def inverse_frequencies(rot_dim: int, theta: float, scaling: Optional[dict]) -> torch.Tensor:
    """float32 [rot_dim / 2], computed in the reference's order of float32 operations."""
    inv = 1.0 / (theta ** (torch.arange(0, rot_dim, 2).float() / rot_dim))
    if not scaling:
        return inv
    kind = scaling.get("rope_type", "default")
    if kind == "default":
        return inv
    if kind != "llama3":
        raise ValueError(f"rotary scaling {kind!r} is not supported (default, llama3)")
    factor = float(scaling["factor"])
    low = float(scaling["low_freq_factor"])
    high = float(scaling["high_freq_factor"])
    orig = float(scaling["original_max_position_embeddings"])
    wavelen = 2 * math.pi / inv
    low_wavelen, high_wavelen = orig / low, orig / high
    scaled = torch.where(wavelen > low_wavelen, inv / factor, inv)
    smooth = (orig / wavelen - low) / (high - low)
    blended = (1 - smooth) * scaled / factor + smooth * scaled
    medium = (~(wavelen < high_wavelen)) & (~(wavelen > low_wavelen))
    return torch.where(medium, blended, scaled)


def yarn_frequencies(dims: int, base: float, factor: float, original: float, fast: float, slow: float):
    """YaRN's blend of rotary frequencies, in double precision: float64 [dims / 2] and the factor on cos and sin.

    With f_i = base^(-2i/dims) and where(t) = dims ln(original / (2 pi t)) / (2 ln base) (the pair whose wave turns t
    times within `original` positions), lo = max(floor(where(fast)), 0), hi = min(ceil(where(slow)), dims - 1) and
    ramp_i = clamp((i - lo) / max(hi - lo, 0.001), 0, 1): pairs below lo keep f_i, pairs above hi get f_i / factor, and
    those between are blended, f_i / factor * ramp_i + f_i (1 - ramp_i). cos and sin are multiplied by
    0.1 ln(factor) + 1."""
    i = torch.arange(dims // 2, dtype=torch.float64)
    f = torch.tensor(float(base), dtype=torch.float64) ** (-2.0 * i / dims)

    def where(turns: float) -> float:
        return dims * math.log(original / (2.0 * math.pi * turns)) / (2.0 * math.log(base))

    lo = max(math.floor(where(fast)), 0)
    hi = min(math.ceil(where(slow)), dims - 1)
    ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
    return f / factor * ramp + f * (1.0 - ramp), 0.1 * math.log(factor) + 1.0


def _store_fp8(qkv, q, ctx, kv, table, n_q, n_kv, head_dim, rot_dim, write_kv):
    """encode_and_store for a cache in 8 bits: the whole step's tokens, block by block of 16 positions."""
    return ops.rope_store_fp8(qkv, q, kv.k, kv.v, kv.k_exp, kv.v_exp, table, ctx.cu_q, ctx.seq_slot, ctx.seq_start,
                              kv.block_table, ctx.n_seqs, ctx.max_q_len, n_q, n_kv, head_dim, rot_dim, write_kv)


class RotaryEncoding(PositionEncoding):
    """params: rot_dim (how many leading elements of a head are rotated), theta, scaling
    (None or {"rope_type": "llama3", factor, low_freq_factor, high_freq_factor,
    original_max_position_embeddings}), exact_angles (bool: the table from double-precision angles, without scaling)."""

    eight_bit = True

    def __init__(self, params, runtime):
        super().__init__(params, runtime)
        self.rot_dim = int(params["rot_dim"])
        if self.rot_dim <= 0 or self.rot_dim % 2:
            raise ValueError(f"rot_dim must be positive and even, got {self.rot_dim}")
        self.theta = float(params["theta"])
        self.scaling = params.get("scaling")
        inv = inverse_frequencies(self.rot_dim, self.theta, self.scaling)
        self.inv_freq = inv
        if params.get("exact_angles"):
            # frequencies and angles in double precision, cosine and sine rounded once to float32
            inv64 = torch.tensor([self.theta ** (-2.0 * i / self.rot_dim) for i in range(self.rot_dim // 2)],
                                 dtype=torch.float64)
            angle = torch.outer(torch.arange(runtime.max_positions, dtype=torch.float64), inv64)
            table = torch.stack([torch.cos(angle), torch.sin(angle)], dim=-1).float()
        else:
            pos = torch.arange(runtime.max_positions, dtype=torch.float32)
            angle = torch.outer(pos, inv).float()
            table = torch.stack([torch.cos(angle), torch.sin(angle)], dim=-1)   # [P, rot/2, 2]
        self.table = table.contiguous().to(runtime.device)

    def fused_table(self, head_dim: int):
        """The (cos, sin) table, if a product kernel may apply this encoding in its own epilogue:
        that needs the whole head to be rotated."""
        return self.table if self.rot_dim == head_dim else None

    def encode_and_store(self, qkv, ctx, kv, n_q, n_kv, head_dim, write_kv, v_head_dim=None):
        """`v_head_dim`: the size of a value head where it differs from head_dim (the packed row then ends with
        n_kv * v_head_dim value columns)."""
        q = torch.empty((qkv.shape[0], n_q * head_dim), dtype=qkv.dtype, device=qkv.device)
        if getattr(kv, "k_exp", None) is not None:
            return _store_fp8(qkv, q, ctx, kv, self.table, n_q, n_kv, head_dim, self.rot_dim, write_kv)
        ops.rope_store(qkv, q, kv.k if kv is not None else None, kv.v if kv is not None else None, self.table,
                       ctx.tok_pos, ctx.tok_seq, ctx.seq_slot, kv.block_table, kv.page_size, n_q, n_kv, head_dim,
                       self.rot_dim, write_kv, v_head_dim=v_head_dim)
        return q


class NoEncoding(PositionEncoding):
    """Positions enter nowhere: keys and values are stored as projected."""

    eight_bit = True

    def encode_and_store(self, qkv, ctx, kv, n_q, n_kv, head_dim, write_kv):
        q = torch.empty((qkv.shape[0], n_q * head_dim), dtype=qkv.dtype, device=qkv.device)
        if getattr(kv, "k_exp", None) is not None:
            return _store_fp8(qkv, q, ctx, kv, None, n_q, n_kv, head_dim, 0, write_kv)
        ops.rope_store(qkv, q, kv.k, kv.v, None, ctx.tok_pos, ctx.tok_seq, ctx.seq_slot, kv.block_table,
                       kv.page_size, n_q, n_kv, head_dim, 0, write_kv)
        return q


register_position_encoding("rope", RotaryEncoding)
register_position_encoding("none", NoEncoding)
