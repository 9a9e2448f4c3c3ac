"""4-bit weights with group scales (``linear_w4``): rounding and packing.

A row of ``K`` values (a multiple of 128) is cut into groups of 32, 64 or 128 values; each has one
bf16 scale, ``max|w| / 7`` rounded to bf16, and each value one code, ``w / scale`` rounded to the
nearest of -7 .. 7. Packed, a row is ``K / 8`` int32 words. Within each 128 values word ``4 t + i``
holds values ``32 i + 8 t .. 32 i + 8 t + 7``, and a word holds its values 0 2 4 6 1 3 5 7 from the
lowest bits up, each as ``code + 8``: the order in which the tensor-core product takes them, so the
kernel loads 16 bytes a lane and needs no shuffle (``csrc/w4.cu``).
"""

from __future__ import annotations

import torch

GROUPS = (32, 64, 128)
_SHIFTS = (0, 16, 4, 20, 8, 24, 12, 28)  # of the values 0 .. 7 of a word


def _check(n: int, k: int, group: int) -> None:
    if group not in GROUPS:
        raise ValueError(f"group must be one of {GROUPS}, got {group}")
    if n < 1 or k < 128 or k % 128:
        raise ValueError(f"weights must be [N, K] with K a multiple of 128, got [{n}, {k}]")


def pack_w4(codes: torch.Tensor) -> torch.Tensor:
    """Integer codes ``[N, K]`` in -8 .. 7 -> int32 words ``[N, K / 8]``."""
    n, k = codes.shape
    _check(n, k, 128)
    c = (codes.to(torch.int64) + 8).view(n, k // 8, 8)
    shifts = torch.tensor(_SHIFTS, dtype=torch.int64, device=codes.device)
    w = (c << shifts).sum(-1)
    w = torch.where(w >= 2**31, w - 2**32, w).to(torch.int32)
    return w.view(n, k // 128, 4, 4).transpose(2, 3).reshape(n, k // 8).contiguous()


def unpack_w4(words: torch.Tensor) -> torch.Tensor:
    """int32 words ``[N, K / 8]`` -> int8 codes ``[N, K]``."""
    n = words.shape[0]
    w = words.view(n, -1, 4, 4).transpose(2, 3).reshape(n, -1)
    shifts = torch.tensor(_SHIFTS, dtype=torch.int32, device=words.device)
    return (((w[..., None] >> shifts) & 15).to(torch.int8) - 8).view(n, -1)


@torch.no_grad()
def quantize_w4(w: torch.Tensor, group: int = 128, out: tuple[torch.Tensor, torch.Tensor] | None = None,
                rows: int = 8192) -> tuple[torch.Tensor, torch.Tensor]:
    """``w [N, K]`` -> ``(codes int32 [N, K / 8], scales bf16 [N, K / group])``, in ``out`` if given.

    A group that holds a value that is not finite gets a NaN scale, so the product shows it. Runs
    ``rows`` rows at a time (fp32 temporaries of that size)."""
    if w.dim() != 2:
        raise ValueError(f"weights must be [N, K], got {tuple(w.shape)}")
    n, k = w.shape
    _check(n, k, group)
    if out is None:
        out = (torch.empty(n, k // 8, dtype=torch.int32, device=w.device),
               torch.empty(n, k // group, dtype=torch.bfloat16, device=w.device))
    words, scales = out
    if words.shape != (n, k // 8) or words.dtype != torch.int32 or scales.shape != (n, k // group) \
            or scales.dtype != torch.bfloat16:
        raise ValueError("out must be (int32 [N, K / 8], bf16 [N, K / group])")
    for a in range(0, n, rows):
        x = w[a:a + rows].detach().float().reshape(-1, k // group, group)
        s = (x.abs().amax(-1) / 7).to(torch.bfloat16)
        s = torch.where(torch.isfinite(s), s, torch.full_like(s, float("nan")))
        d = s.float()[..., None]
        c = torch.where(d > 0, x / d, torch.zeros_like(x)).round().clamp(-7, 7)
        words[a:a + rows] = pack_w4(c.reshape(-1, k).to(torch.int8)).to(words.device)
        scales[a:a + rows] = s.to(scales.device)
    return out


def dequantize_w4(words: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """fp32 weights ``[N, K]`` (the product ``code * scale`` is exact)."""
    n, k = words.shape[0], words.shape[1] * 8
    c = unpack_w4(words).float().view(n, scales.shape[1], -1)
    return (c * scales.float()[..., None]).view(n, k)
