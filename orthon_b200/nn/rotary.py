"""Rotary positions as a module: a configuration without parameters or buffers."""
from ..functional import _checked_rotary_plan, rotary_embedding, rotary_embedding_
from .module import Module


class RotaryEmbedding(Module):
    """Turns the first ``rotary_dim`` values of every head of [B, T, H, D] inputs by their positions.

    Holds the settings of `functional.rotary_embedding` (``base``, ``interleaved``, ``scaling``), so that queries, keys and
    cached keys are turned alike.  ``forward_`` works in place (no graph)."""

    def __init__(self, rotary_dim, base=10000.0, interleaved=False, scaling=None):
        super().__init__()
        self.rotary_dim, self.base, self.interleaved = int(rotary_dim), float(base), bool(interleaved)
        self.scaling = None if scaling is None else dict(scaling)
        if not 2 <= self.rotary_dim <= 512 or self.rotary_dim % 2:
            raise ValueError("rotary_dim must be even and in [2, 512]")
        _checked_rotary_plan(self.rotary_dim, self.base, self.scaling)

    def _settings(self):
        return dict(rotary_dim=self.rotary_dim, base=self.base, interleaved=self.interleaved, scaling=self.scaling)

    def forward(self, x, positions=None, rotary_heads=None):
        return rotary_embedding(x, positions, rotary_heads=rotary_heads, **self._settings())

    def forward_(self, x, positions=None, rotary_heads=None):
        return rotary_embedding_(x, positions, rotary_heads=rotary_heads, **self._settings())
