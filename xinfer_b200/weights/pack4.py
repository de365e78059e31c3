"""A weight in 4 bits, laid out for ``kernels.linear4``; made once, when a model is loaded."""
from __future__ import annotations

import torch

TILE_ROWS, TILE_COLUMNS = 16, 128


def pack4(weight: torch.Tensor, group: int = 32) -> torch.Tensor:
    """``weight`` ``[rows, columns]`` in groups of 32, 64 or 128 columns with a scale s and a least value m in bfloat16, as uint8
    ``[row tiles, column tiles, bytes]`` on the weight's device: s = (largest - least) / 15, code = round((w - m) / s), value m + s * code.  A tile of 16 rows and
    128 columns has 1,024 bytes of codes, then each row's (s, m) pairs.  Byte ``512 h + 64 r + 16 t + 4 j + b`` of the codes belongs to row 8 h + r and the columns
    32 j + 8 t + 4 b .. : the low half is column e = 4 b for b < 2 and 4 b - 7 behind, the high half column e + 2.  Rows and columns behind the weight are zeros,
    which belong to the range of a last group that they fill up: a multiple of ``group`` columns keeps all codes for the weight's own numbers."""
    if weight.dim() != 2 or not weight.is_floating_point() or 0 in weight.shape:
        raise ValueError(f"pack4 takes a matrix of real numbers, not {weight.dtype} {tuple(weight.shape)}")
    if group not in (32, 64, 128):
        raise ValueError(f"groups of {group} columns: 32, 64 or 128")
    n, k = weight.shape
    if not bool(torch.isfinite(weight).all()):
        raise ValueError("a weight with numbers that are not finite")
    rows, cols = -(-n // TILE_ROWS), -(-k // TILE_COLUMNS)
    full = torch.zeros((rows * TILE_ROWS, cols * TILE_COLUMNS), dtype=torch.float32, device=weight.device)
    full[:n, :k] = weight
    g = full.view(rows * TILE_ROWS, -1, group)
    low = g.amin(2)
    scale, least = ((g.amax(2) - low) / 15).to(torch.bfloat16), low.to(torch.bfloat16)
    if not bool(torch.isfinite(scale).all() & torch.isfinite(least).all()):
        raise ValueError("a group of numbers that bfloat16 scales do not hold")
    s, m = scale.float().unsqueeze(2), least.float().unsqueeze(2)
    codes = torch.where(s > 0, torch.round((g - m) / torch.where(s > 0, s, 1.0)), 0.0).clamp_(0, 15).to(torch.uint8)
    # (tile, half, row, tile, word, lane, pair, place in the pair) -> (tile, tile, half, row, lane, word, place, pair)
    codes = codes.view(rows, 2, 8, cols, 4, 4, 4, 2).permute(0, 3, 1, 2, 5, 4, 7, 6).reshape(rows, cols, -1)
    words = torch.stack([scale, least], 2).view(torch.uint8).view(rows, TILE_ROWS, cols, -1).transpose(1, 2)
    packed = torch.cat([codes[..., 0::2] | (codes[..., 1::2] << 4), words.reshape(rows, cols, -1)], 2)
    if packed.is_cuda:
        torch.cuda.current_stream(packed.device).synchronize()       # (complete: products read a weight while the kernel ahead of them still runs)
    return packed
