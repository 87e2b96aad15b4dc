"""Rows and weights in 8 bits: whole numbers from -127 to 127 with a float32 scale a row (a token's
row; an output channel of a weight), value = scale * number, scale = the row's largest
magnitude / 127.  The provider makes them (`quantize_rows`, `quantize_weight`), and its `linear`,
`linear_silu_mul` and `norm_linear` take an `Int8Weight` where they take a weight."""

from __future__ import annotations

from dataclasses import dataclass

import torch

#: bytes that a row of numbers is a multiple of (zeros behind its last element)
ROW = 256


def row_bytes(k: int) -> int:
    """Bytes of a row of k numbers: 512 at least, which is what the product in tiles needs to fill its
    buffers (1,403 rows of 83 by 1,799 columns: 21 us in rows of 256, 16 rows at a time, 14 in tiles)."""
    return max(-(-k // ROW), 2) * ROW


@dataclass(frozen=True)
class Int8Rows:
    """Rows [M, K] in 8 bits."""

    codes: torch.Tensor         # int8 [M, row_bytes(K)]
    scales: torch.Tensor        # float32 [M]
    width: int                  # K

    @property
    def shape(self) -> torch.Size:
        return torch.Size((self.codes.shape[0], self.width))

    @property
    def device(self) -> torch.device:
        return self.codes.device

    #: what a weight's own dtype tells the products that know none of this
    dtype = torch.int8

    def numel(self) -> int:
        return self.codes.shape[0] * self.width

    def values(self) -> torch.Tensor:
        """The rows that the numbers stand for, float32 [M, K]."""
        return self.codes[:, :self.width].float() * self.scales[:, None]


class Int8Weight(Int8Rows):
    """A weight [N, K] in 8 bits, a scale per output channel."""
