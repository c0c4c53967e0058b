"""Rotary positions module (no counterpart in the reference)."""
import torch

from . import rotary_frequencies, rotary_positions


class RotaryPositions(torch.nn.Module):
    """forward(x (T, H, D), positions (T) or (T, A)) -> x with its heads' values turned.

    `size` values of each head are turned.  base, stretch and trained make the frequencies, see
    rotary_frequencies; `frequencies` gives others (for coordinates, say).
    """

    def __init__(self, size, base=10000.0, stretch=1.0, trained=None, interleaved=False,
                 amplitude=1.0, frequencies=None, device=None):
        super().__init__()
        if size < 0 or size % 2 != 0:
            raise ValueError(f"size must be even and not negative, but got {size}")
        self._made = None  # what makes the frequencies; those that were given are all there is
        if frequencies is None:
            self._made = (size // 2, base, stretch, trained)
            frequencies = rotary_frequencies(*self._made, device)
        elif tuple(frequencies.shape) != (size // 2,):
            raise ValueError(f"frequencies must have shape ({size // 2},), but got "
                             f"{tuple(frequencies.shape)}")
        self.interleaved = interleaved
        self.amplitude = amplitude
        self._double = frequencies.to(device=device, dtype=torch.float64)

    @property
    def frequencies(self):
        return self._double

    def _apply(self, fn, recurse=True):
        # to(device) moves them, to(dtype) leaves them in 64 bits
        super()._apply(fn, recurse)
        device = fn(torch.empty(0, device=self._double.device)).device
        if self._double.is_meta and device.type != "meta" and self._made is not None:
            self._double = rotary_frequencies(*self._made, device)  # (to_empty)
        else:
            self._double = self._double.to(device)
        return self

    def forward(self, x, positions):
        return rotary_positions(x, positions, self.frequencies, self.interleaved, self.amplitude)
