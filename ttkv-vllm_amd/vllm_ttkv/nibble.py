"""The 4-bit cache's geometry: what one slot of a layer's page holds.

The tensor-train store (`layout.TTKLayout`) keeps keys before their rotation and turns the key of
row t by position t, so a model whose positions have several axes (images, video) cannot be served
from it, nor a layer without a calibrated layout. This cache holds rotated keys and values as
4-bit codes with one 16-bit scale per 32 dims, needs no fit, and reads 72 bytes per head row where
fp16 has 256. Byte format: include/ttkv_hip.h; written by `kernels.nibble_write_paged`, read by
`kernels.nibble_decode_paged` and `kernels.nibble_prefill_paged`. No counterpart in the reference.
"""
from __future__ import annotations

from dataclasses import dataclass

TILE = 16       # slots whose codes lie together; block sizes are multiples of it
GROUP = 32      # dims per scale


@dataclass(frozen=True)
class NibbleLayout:
    """Byte layout of one layer's 4-bit cache; every size is per token."""

    H: int
    d: int = 128

    def __post_init__(self):
        if self.H <= 0:
            raise ValueError(f"H={self.H} KV heads")
        if self.d != 128:
            raise ValueError(f"head dim {self.d}: the 4-bit cache is built for 128")

    @property
    def row_bytes(self) -> int:
        """One head's key or value row: d/2 bytes of codes and a 16-bit parameter per group."""
        return self.d // 2 + 2 * (self.d // GROUP)

    def compressed_bytes_per_token(self) -> int:
        return 2 * self.H * self.row_bytes

    def dense_bytes_per_token(self) -> int:
        return 2 * self.H * self.d * 2

    def ratio(self) -> float:
        return self.dense_bytes_per_token() / self.compressed_bytes_per_token()
