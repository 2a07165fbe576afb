"""Readout of per-structure properties on the network's atom features: one attention block over whole structures and a pooling query.

The network's own attention ends at its 4.5 A cutoff; what a property of the whole structure needs from further away is gathered here.  Every
atom attends to all atoms of its structure, queries and keys normalised per head and rotated by the atom's coordinates, so that the
logits depend on displacements (nothing changes when a structure is shifted; orientations are seen, as the features themselves do
not).  Then one learned query per structure attends to its atoms.  `make_so3lr(readout=...)` evaluates it with a batch.  No counterpart in the reference.
"""
from __future__ import annotations

import math

import numpy as np
import torch

from .attention import PackedStructures, norm_rotate, structure_attention

FEATURES = 128


class StructureReadout(torch.nn.Module):
    """(features (n, 128), positions (n, 3), graph_start) -> (n_structures, n_out).

    heads x d: size of the attention (4 x 32, as the network's).  wavelengths: shortest and longest period of the rotation in Angstrom, over
    which the frequencies of each axis are spread geometrically.  Parameters are ordinary torch parameters on `device`, drawn from `seed`;
    the last layer starts at zero, so an untrained readout gives zero.  With 16-bit parameters (`.to(torch.bfloat16)`) or under autocast the
    products and the attention run in that type; the frequencies stay float32, as the angles of far positions need them.
    The layouts of captured calls are kept as long as the readout lives: a graph reads their tables."""

    MAX_CACHED_LAYOUTS = 8

    def __init__(self, n_out=1, heads=4, d=32, wavelengths=(4.0, 100.0), seed=0, device=0):
        super().__init__()
        if d % 16 or not 16 <= d <= 128 or heads < 1 or n_out < 1 or not 0 < wavelengths[0] <= wavelengths[1]:
            raise ValueError(f"n_out {n_out}, heads {heads}, d {d} (a multiple of 16 up to 128), wavelengths {wavelengths}")
        dev = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        gen = torch.Generator().manual_seed(seed)
        self.heads, self.d = heads, d

        def matrix(rows, cols):
            return torch.nn.Parameter((torch.randn(rows, cols, generator=gen) / math.sqrt(rows)).to(dev))

        self.qkv = matrix(FEATURES, 3 * heads * d)
        self.out = matrix(heads * d, FEATURES)
        self.norm_q, self.norm_k = (torch.nn.Parameter(torch.ones(d, device=dev)) for _ in range(2))
        self.pool_kv = matrix(FEATURES, 2 * heads * d)
        self.pool_query = torch.nn.Parameter(torch.randn(heads, d, generator=gen).to(dev))
        self.last = torch.nn.Parameter(torch.zeros(heads * d, n_out, device=dev))
        # pair p turns with axis p mod 3
        p = torch.arange(d // 2)
        k = (p // 3).double() / max(1, (d // 2 - 1) // 3)
        f = torch.zeros(3, d // 2, dtype=torch.float64)
        f[p % 3, p] = 2 * math.pi / (wavelengths[0] * (wavelengths[1] / wavelengths[0]) ** k)
        self.register_buffer("frequencies", f.float().to(dev))
        self._layouts, self._captured = {}, {}

    def _apply(self, fn, *args, **kwargs):      # .to, .half, ..: the frequencies follow to another device, not to another type
        frequencies = self.frequencies
        super()._apply(fn, *args, **kwargs)
        if self.frequencies.dtype != frequencies.dtype:
            self.frequencies = frequencies.to(self.frequencies.device)
        return self

    def __getstate__(self):      # layouts hold device tables: a copy makes its own
        return self.__dict__ | {"_layouts": {}, "_captured": {}}

    def _layout(self, graph_start):
        gs, dev = PackedStructures._starts("graph_start", graph_start), self.qkv.device
        key = gs.tobytes(), dev
        pair = self._captured.get(key) or self._layouts.pop(key, None)
        if pair is None:
            pair = PackedStructures(gs, device=dev), PackedStructures(np.arange(len(gs)), gs, device=dev)
        if torch.cuda.is_current_stream_capturing():
            self._captured[key] = pair              # a graph reads its tables from now on: kept for good
            return pair
        self._layouts[key] = pair                   # most recently used last
        while len(self._layouts) > self.MAX_CACHED_LAYOUTS:
            self._layouts.pop(next(iter(self._layouts)))
        return pair

    def forward(self, features, positions, graph_start):
        if features.ndim != 2 or features.shape[1] != FEATURES or positions.shape != (features.shape[0], 3):
            raise ValueError(f"features must be (n, {FEATURES}) and positions (n, 3), not {tuple(features.shape)} and {tuple(positions.shape)}")
        atoms, pool = self._layout(graph_start)
        heads, d = self.heads, self.d
        features = features.to(self.qkv.dtype)
        q, k, v = (features @ self.qkv).unflatten(1, (3, heads, d)).unbind(1)
        q, k = norm_rotate(q, k, positions, self.frequencies, q_weight=self.norm_q, k_weight=self.norm_k)
        x = features + structure_attention(q, k, v, atoms).flatten(1) @ self.out
        k, v = (x @ self.pool_kv).unflatten(1, (2, heads, d)).unbind(1)
        query = self.pool_query.to(k.dtype).expand(pool.rows_q, heads, d)      # autocast makes k and v 16-bit ones
        return structure_attention(query, k, v, pool).flatten(1) @ self.last
