"""A buffer of cosines and sines that no checkpoint holds."""
from __future__ import annotations

from ..ops import rotary_table

__all__ = ["Angles"]


class Angles:
    """Mixed into a module whose buffer ``angles`` is :func:`ttc.ops.rotary_table` of ``self._table``: whatever is done to the
    parameters (another type, ``to_empty``), the angles keep their values in 32 bits, or get them where the module was made
    without any (on the meta device)."""

    def _apply(self, fn, recurse=True):
        angles = self.angles
        super()._apply(fn, recurse)
        if angles.is_meta and not self.angles.is_meta:
            self.angles = rotary_table(**dict(self._table, device=self.angles.device))
        elif self.angles is not angles:
            self.angles = angles.to(self.angles.device)
        return self
