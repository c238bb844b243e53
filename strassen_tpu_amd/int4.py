"""Products of few rows with 4-bit weights, on ``csrc/int4_matmul.hip``: the decode
form of the block's projections, whose time is that of reading the weight. The
reference has no quantised weights; ``int4_matmul`` stands beside
``strassen_matmul`` with the epilogues that a decode step needs.

A weight ``[K, N]`` is ``(code - zero) * scale``: codes 0 .. 15, one bf16 scale and one
zero point 0 .. 15 per group of 32, 64 or 128 consecutive k and column.
"""

from __future__ import annotations

import torch

from . import _lib

__all__ = ["Int4Operand", "int4_quantize", "int4_weight_layout", "int4_matmul"]

GROUPS = (32, 64, 128)
_EPILOGUES = (None, "swiglu", "residual_add", "bias_add")


class Int4Operand:
    """A weight laid out by ``int4_weight_layout``: int32 tensors ``codes`` and ``scales`` on one device. A call
    refuses one whose tensors are not of the size, type or device that its other fields say."""

    def __init__(self, codes, scales, k, n, group, swiglu, zeros):
        self.codes, self.scales, self.device = codes, scales, codes.device
        self.k, self.n, self.group, self.swiglu, self.zeros = k, n, group, swiglu, zeros

    @property
    def shape(self):
        return self.k, self.n

    def __repr__(self):
        return f"Int4Operand(k={self.k}, n={self.n}, group={self.group}, swiglu={self.swiglu})"


def int4_quantize(w, group=128):
    """``(codes, scales, zeros)`` of a weight ``[K, N]``, each value the nearest of its group's 16:
    scale ``(max - min) / 15`` over the group (0 among its values), rounded to bf16,
    zero point ``round(-min / scale)``."""
    if w.dim() != 2 or not w.is_floating_point():
        raise ValueError("int4_quantize expects a floating-point weight [K, N]")
    k, n = w.shape
    if group not in GROUPS or k % group:
        raise ValueError(f"group must be one of {GROUPS} and divide K={k}, got {group}")
    g = w.float().reshape(k // group, group, n)
    low, high = g.amin(1).clamp(max=0), g.amax(1).clamp(min=0)
    scales = ((high - low) / 15).to(torch.bfloat16)
    step = torch.where(scales > 0, scales.float(), 1.0)
    zeros = torch.round(-low / step).clamp_(0, 15)
    codes = torch.round(g / step[:, None]).add_(zeros[:, None]).clamp_(0, 15)
    return codes.to(torch.uint8).reshape(k, n), scales, zeros.to(torch.uint8)


def _tiles(x, swiglu):
    """Columns of ``x [..., N]`` in whole tiles of 16, an even number of them, padded with
    zeros: ``[..., tiles, 16]``; for swiglu tiles of the gate and the up half in turn."""
    pad = torch.nn.functional.pad
    if swiglu:
        half = x.shape[-1] // 2
        gate, up = (pad(part, (0, -half % 16)).unflatten(-1, (-1, 16)) for part in x.split(half, dim=-1))
        return torch.stack((gate, up), dim=-2).flatten(-3, -2)
    return pad(x, (0, -x.shape[-1] % 32)).unflatten(-1, (-1, 16))


def int4_weight_layout(codes, scales, zeros=None, *, group, epilogue=None):
    """Lay out a 4-bit weight for ``int4_matmul``: ``codes`` uint8 ``[K, N]`` of values 0 .. 15,
    ``scales`` bf16 ``[K / group, N]``, ``zeros`` uint8 ``[K / group, N]`` of values 0 .. 15
    (None: 8). With ``epilogue="swiglu"`` the columns are ``[gate | up]``. The result holds a
    copy, half a byte a weight and four bytes a group and column."""
    if codes.dim() != 2 or codes.dtype != torch.uint8:
        raise ValueError("codes must be a uint8 tensor [K, N]")
    k, n = codes.shape
    if epilogue not in (None, "swiglu"):
        raise ValueError(f"only 'swiglu' lays a weight out of its own, got {epilogue!r}")
    if group not in GROUPS or not k or k % group or not n:
        raise ValueError(f"group must be one of {GROUPS} and divide K={k}, got {group} (N={n})")
    swiglu = epilogue == "swiglu"
    if swiglu and n % 2:
        raise ValueError(f"[gate | up] has an even width, got N={n}")
    shape = (k // group, n)
    if scales.dtype != torch.bfloat16 or tuple(scales.shape) != shape:
        raise ValueError(f"scales must be a bf16 tensor {shape}, got {scales.dtype} {tuple(scales.shape)}")
    if zeros is not None and (zeros.dtype != torch.uint8 or tuple(zeros.shape) != shape):
        raise ValueError(f"zeros must be a uint8 tensor {shape}, got {zeros.dtype} {tuple(zeros.shape)}")
    if any(t.device != codes.device for t in (scales, zeros) if t is not None):
        raise ValueError("codes, scales and zeros must be on one device")
    if int(codes.max()) > 15 or (zeros is not None and int(zeros.max()) > 15):
        raise ValueError("codes and zeros must be 0 .. 15")
    tiled = _tiles(codes, swiglu)  # [K, tiles, 16]
    k_tiles = -(-k // 128)
    if k % 128:
        tiled = torch.nn.functional.pad(tiled, (0, 0, 0, 0, 0, -k % 128))
    # k = 128 tile + 32 word + 8 quad + j
    tiled = tiled.view(k_tiles, 4, 4, 8, -1, 16)
    words = torch.zeros(k_tiles, 4, 4, tiled.shape[4], 16, dtype=torch.int32, device=codes.device)
    for j in range(8):
        at = 16 * (j % 2) + 4 * (j // 2) + 3
        part = tiled[:, :, :, j].to(torch.int32)
        # the last pair's upper code wraps around: its lowest bit at 31, the others at 0 .. 2
        words |= part << at if at < 29 else (part << 31) | (part >> 1)
    words = words.permute(3, 0, 2, 4, 1).contiguous()  # [tiles, k_tiles, quad, column, word]
    # -(16 + zero) is a bf16 number: sign, exponent of 16, four mantissa bits
    zero = torch.full(shape, 8, dtype=torch.int32, device=codes.device) if zeros is None else zeros.to(torch.int32)
    pairs = (scales.contiguous().view(torch.int16).to(torch.int32) << 16) | (0xC180 | zero << 3)
    pairs = _tiles(pairs, swiglu)  # [groups, tiles, 16]
    per_tile = 128 // group
    missing = k_tiles * per_tile - shape[0]
    if missing:
        pairs = torch.nn.functional.pad(pairs, (0, 0, 0, 0, 0, missing))
    pairs = pairs.unflatten(0, (k_tiles, per_tile)).permute(2, 0, 3, 1).contiguous()  # [tiles, k_tiles, column, group]
    return Int4Operand(words, pairs, k, n, group, swiglu, zeros is not None)


def int4_matmul(x, w, *, epilogue=None, residual=None, bias=None):
    """``epilogue(x @ W)`` for bf16 rows ``x [M, K]`` and a weight of ``int4_weight_layout``, bf16
    ``[M, N]`` (``[M, N / 2]`` with "swiglu", whose weight is laid out for it). Epilogues:
    "swiglu" (``silu(gate) * up``), "residual_add" (``residual [M, N]``) and "bias_add"
    (``bias [N]``), in FP32 with one rounding; the weight is used exactly as its codes, scales
    and zeros say. Meant for decode steps: every 64 rows read the weight again. A row of ``x``
    with an infinity is NaN in the result; one with finite values beyond 2^115 (4e34) may be, however small the
    scales: 31 times a group's ``|x|`` is summed in FP32 before its scale."""
    if not isinstance(w, Int4Operand):
        raise TypeError("w must be an Int4Operand (int4_weight_layout)")
    if epilogue not in _EPILOGUES:
        raise ValueError(f"unknown epilogue {epilogue!r}; choose 'swiglu', 'residual_add' or 'bias_add'")
    if (epilogue == "swiglu") != w.swiglu:
        raise ValueError(f"{w!r} is {'' if w.swiglu else 'not '}laid out for swiglu")
    return _lib.host().int4(x, w.codes, w.scales, w.k, w.n, w.group, w.swiglu, w.zeros, _lib.SMX_EPI[epilogue], residual,
                            bias)
