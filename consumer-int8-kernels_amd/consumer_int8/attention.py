"""Attention operators: what runs between a layer's INT8 QKV projection and its output
projection, over a paged key/value cache of 4-bit values. Buffers belong to the caller.

The cache is four UINT8 tensors, keys and values each as codes [pages, heads, page_size,
dim/2] and scales [pages, heads, page_size, dim/32]: E2M1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6
with a sign; channel 2i in the low half of byte i) times 2^(scale - 127) for 32 channels.
Pages are contiguous inside and may lie further apart. Slot s is row s % page_size of page
s // page_size. Head sizes 64, 128 and 256.

qk_norm_rope(q, k, q_weight, k_weight, rope, positions, axes, q_out, k_out, eps=1e-6,
             interleaved=False)
    BF16 q [T,Hq,D] and k [T,Hk,D], strided views of a projection's output: RMS norm of each
    head (FP32 weight [D], None for no norm), then rotation of the first rot channels by FP32
    rope [rows, rot] (rot/2 cosines, rot/2 sines; None for none) at INT64 positions [T]. Pairs
    are (i, i + rot/2), or neighbours if interleaved. Positions [axes, T] with INT32 axes
    [rot/2] turn each pair by the position on its own axis. FP32 inside; outputs BF16, which
    may be the inputs themselves.
append_fp4(q, k, v, q_weight, k_weight, rope, positions, axes, slots, q_out, k_codes,
           k_scales, v_codes, v_scales, eps=1e-6, interleaved=False)
    In one launch: keys, normed and rotated, and values into the cache rows that INT64 slots
    [T] names (negative: skipped; no two alike); queries as qk_norm_rope (q and q_out may both
    be None).
unpack_fp4(k_codes, k_scales, v_codes, v_scales, slots, k, v)
    Cache rows back as BF16 k, v [count, heads, D], exactly.
attention_fp4(q, k_codes, k_scales, v_codes, v_scales, page_table, context_lens, q_starts,
              workspace, out, lse, scale, max_q=1, window=0)
    Causal attention. INT32 page_table [S, width] and context_lens [S] (tokens in the cache,
    the queries' own included); INT32 q_starts [S+1] the rows of q of each sequence, None for
    one a sequence; max_q the longest of them. Query heads share key heads in order. window:
    how many tokens a query sees, itself included (0: all). out BF16 like q, contiguous;
    lse FP32 [T,Hq] or None. Queries that see nothing give zeros and -inf. workspace FP32
    [65536, D + 2], of any content, used by one stream at a time. Cache tensors span at most
    32 GiB each, page tables width * page_size <= 2^26 - 4096 tokens.
"""

from typing import NamedTuple

import torch

from . import _C  # noqa: F401  (registers torch.ops.consumer_int8.*; fails loudly if unbuilt)

qk_norm_rope = torch.ops.consumer_int8.qk_norm_rope
append_fp4 = torch.ops.consumer_int8.append_fp4
unpack_fp4 = torch.ops.consumer_int8.unpack_fp4
attention_fp4 = torch.ops.consumer_int8.attention_fp4


@torch.library.register_fake("consumer_int8::qk_norm_rope")
def _qk_norm_rope_fake(q, k, q_weight, k_weight, rope, positions, axes, q_out, k_out, eps=1e-6,
                       interleaved=False):
    return None


@torch.library.register_fake("consumer_int8::append_fp4")
def _append_fp4_fake(q, k, v, q_weight, k_weight, rope, positions, axes, slots, q_out, k_codes,
                     k_scales, v_codes, v_scales, eps=1e-6, interleaved=False):
    return None


@torch.library.register_fake("consumer_int8::unpack_fp4")
def _unpack_fp4_fake(k_codes, k_scales, v_codes, v_scales, slots, k, v):
    return None


@torch.library.register_fake("consumer_int8::attention_fp4")
def _attention_fp4_fake(q, k_codes, k_scales, v_codes, v_scales, page_table, context_lens,
                        q_starts, workspace, out, lse, scale, max_q=1, window=0):
    return None


class Fp4Cache(NamedTuple):
    """The four tensors of a cache, in the operators' argument order."""

    k_codes: torch.Tensor
    k_scales: torch.Tensor
    v_codes: torch.Tensor
    v_scales: torch.Tensor


def new_cache(pages, heads, page_size, dim, device="cuda"):
    """A zeroed cache for `pages` pages of `page_size` tokens."""
    if dim not in (64, 128, 256):
        raise ValueError("Unsupported head size: 64, 128 or 256")
    return Fp4Cache(*(torch.zeros(pages, heads, page_size, dim // n, dtype=torch.uint8,
                                  device=device) for n in (2, 32, 2, 32)))


def new_workspace(dim, device="cuda"):
    """attention_fp4's workspace; one for each stream that calls it."""
    return torch.empty(65536, dim + 2, dtype=torch.float32, device=device)


def rope_table(rows, rot, base=10000.0, device="cuda"):
    """FP32 [rows, rot]: cosines, then sines, of position * base^(-2i / rot), computed in
    64 bits."""
    if rot <= 0 or rot % 16:
        raise ValueError("Expected rot > 0 in steps of 16")
    freq = float(base) ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], 1).float().to(device)
