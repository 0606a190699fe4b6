"""Rotary positions of a prompt with images on three axes (time, height, width).

Text tokens count up on all axes alike.  The tokens of an image of (t, h, w) merged patches stand, from the next free position p on, at
(p + time, p + row, p + column); what follows goes on at p + max(t, h, w).  Behind the prompt a token at index i therefore stands at i + shift on every
axis, with one `shift` per sequence."""
from __future__ import annotations

from typing import Sequence, Tuple

import numpy as np


def image_positions(is_image: np.ndarray, grid_thw: Sequence[Sequence[int]], merge: int = 2) -> Tuple[np.ndarray, int]:
    """(positions [3, tokens], shift) of a prompt: `is_image` [tokens] marks the image tokens, `grid_thw` lists each image's patches, `merge` patches a
    side go into one token."""
    n = len(is_image)
    out = np.zeros((3, n), dtype=np.int64)
    grids = [tuple(int(x) for x in g) for g in grid_thw]
    i = p = 0
    for t, h, w in grids:
        if t < 1 or h < 1 or w < 1 or h % merge or w % merge:
            raise ValueError(f"an image of {t} x {h} x {w} patches in blocks of {merge} x {merge}")
        h, w = h // merge, w // merge
        while i < n and not is_image[i]:
            out[:, i] = p
            i, p = i + 1, p + 1
        if not is_image[i: i + t * h * w].all() or i + t * h * w > n:
            raise ValueError(f"the prompt has no run of {t * h * w} image tokens for an image of {t} x {h} x {w}")
        out[:, i: i + t * h * w] = p + np.indices((t, h, w)).reshape(3, -1)
        i, p = i + t * h * w, p + max(t, h, w)
    if is_image[i:].any():
        raise ValueError("the prompt has more image tokens than its images")
    out[:, i:] = p + np.arange(n - i)
    return out, p - i
