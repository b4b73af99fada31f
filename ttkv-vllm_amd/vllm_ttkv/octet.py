"""The 8-bit cache's geometry: what one slot of a layer's page holds.

Beside the tensor-train store (`layout.TTKLayout`) and the 4-bit cache (`nibble.NibbleLayout`), for
layers that fewer bits do not serve: rotated keys and values as e4m3 codes with a power of two per
32 dims, for heads of 64, 128 or 256 dims, 132 bytes per head row of 128 where fp16 has 256. Byte
format: include/ttkv_hip.h; written by `kernels.octet_write_paged`, read by
`kernels.octet_decode_paged` and `kernels.octet_read_paged`. No counterpart in the reference.
"""
from __future__ import annotations

from dataclasses import dataclass

TILE = 16       # slots whose codes lie together; block sizes are multiples of it
GROUP = 32      # dims per power of two


@dataclass(frozen=True)
class OctetLayout:
    """Byte layout of one layer's 8-bit cache; every size is per token."""

    H: int
    d: int = 128

    def __post_init__(self):
        if self.H <= 0:
            raise ValueError(f"H={self.H} KV heads")
        if self.d not in (64, 128, 256):
            raise ValueError(f"head dim {self.d}: the 8-bit cache is built for 64, 128 and 256")
        object.__setattr__(self, "_slot", 2 * self.H * self.row_bytes)   # (asked for by every call)

    @property
    def row_bytes(self) -> int:
        """One head's key or value row: d bytes of codes and an exponent byte per group."""
        return self.d + self.d // GROUP

    def compressed_bytes_per_token(self) -> int:
        return self._slot

    def dense_bytes_per_token(self) -> int:
        return 2 * self.H * self.d * 2

    def ratio(self) -> float:
        return self.dense_bytes_per_token() / self.compressed_bytes_per_token()
