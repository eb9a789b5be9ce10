"""faiss-shaped flat indexes backed by the HIP scan.

Drop-in for the two faiss classes LIRA's query path uses
(utils.py:415-419 builds them, LIRA_smallscale.py:168-171 searches them):

    index = IndexFlatL2(d)        # or IndexFlatIP(d)
    index.add(xb)                 # (n, d) float32, appends
    D, I = index.search(xq, k)    # numpy (nq, k) float32 / int64
    index.ntotal

Inputs may be numpy arrays (as in the reference) or torch tensors; outputs
follow the input kind (numpy in -> numpy out).  Result convention is faiss':
L2 = ascending squared distance, IP = descending inner product, -1 labels
and +-inf distances when the index holds fewer than k vectors.  Distances are
search.cpp's sequential fp32 sums (faiss's BLAS path rounds differently; they
agree to ~1e-6 relative).  Ties order by smaller label.

``IndexMX4`` is the compressed flat index (the place of faiss's 4-bit scalar
quantizer): rows in 4.25 bits an element, scored as they are stored.
"""
from __future__ import annotations

import numpy as np
import torch

from .index import PartitionedIndex, normalize_metric, select_probes
from .mx4 import MX4Tensor, mx4_linear, mx4_quantize


class IndexFlat:
    def __init__(self, d: int, metric: str = "L2", device=None):
        self.d = int(d)
        self.metric = normalize_metric(metric)
        self.device = torch.device("cuda", torch.cuda.current_device() if device is None else device)
        self._chunks: list[torch.Tensor] = []
        self._index: PartitionedIndex | None = None
        self.ntotal = 0
        self.is_trained = True

    @property
    def metric_type(self) -> int:
        return 0 if self.metric == "inner_product" else 1  # faiss METRIC_INNER_PRODUCT / METRIC_L2

    def add(self, x) -> None:
        xt = x if isinstance(x, torch.Tensor) else torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32))
        if xt.dim() != 2 or xt.shape[1] != self.d:
            raise RuntimeError(f"add: expected (n, {self.d}) vectors, got {tuple(xt.shape)}")
        self._chunks.append(xt.to(device=self.device, dtype=torch.float32).contiguous())
        self.ntotal += xt.shape[0]
        self._index = None

    def reset(self) -> None:
        self._chunks.clear()
        self._index = None
        self.ntotal = 0

    def _built(self) -> PartitionedIndex:
        if self._index is None:
            x = torch.cat(self._chunks) if self._chunks else torch.zeros((0, self.d), device=self.device)
            n = x.shape[0]
            idx = PartitionedIndex(self.d, self.metric, self.device.index)
            idx.add_lists(np.array([0, n], dtype=np.int64),
                          torch.arange(n, dtype=torch.int32, device=self.device), x, 1)
            self._index = idx
        return self._index

    def search(self, x, k: int):
        as_numpy = not isinstance(x, torch.Tensor)
        q = torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)) if as_numpy else x
        if q.dim() != 2 or q.shape[1] != self.d:
            raise RuntimeError(f"search: expected (nq, {self.d}) queries")
        q = q.to(device=self.device, dtype=torch.float32).contiguous()
        probe = torch.zeros((q.shape[0], 1), dtype=torch.int32, device=self.device)
        D, I, _ = self._built().search(q, probe, int(k), dedup=False)
        if as_numpy:
            return D.cpu().numpy(), I.cpu().numpy()
        return D, I


class IndexFlatL2(IndexFlat):
    def __init__(self, d: int, device=None):
        super().__init__(d, "L2", device)


class IndexFlatIP(IndexFlat):
    def __init__(self, d: int, device=None):
        super().__init__(d, "inner_product", device)


class IndexMX4:
    """Flat index of microscaled 4-bit rows (lira_mx4_quantize): d = 128 takes 68 bytes a vector
    and a norm, where IndexFlat takes 512 bytes and more.

    ``search`` packs the queries alike and ranks by the distances of the packed vectors, so it
    is approximate: those distances are what it returns.  Order, padding and ties as in
    IndexFlat; vectors must be finite, a query that is not finds nothing.  k <= 256.
    """

    _CHUNK = 4096  # scores that one selection pass looks at

    def __init__(self, d: int, metric: str = "L2", device=None):
        self.d = int(d)
        if self.d < 1:
            raise ValueError("d must be at least 1")
        self.metric = normalize_metric(metric)
        self.device = torch.device("cuda", torch.cuda.current_device() if device is None else device)
        self.is_trained = True
        self.reset()

    @property
    def metric_type(self) -> int:
        return 0 if self.metric == "inner_product" else 1

    def reset(self) -> None:
        self._parts: list[MX4Tensor] = []
        self._norms: list[torch.Tensor] = []
        self.ntotal = 0

    def _rows(self, x, what: str) -> torch.Tensor:
        x = x if isinstance(x, torch.Tensor) else torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32))
        if x.dim() != 2 or x.shape[1] != self.d:
            raise RuntimeError(f"{what}: expected (n, {self.d}) vectors, got {tuple(x.shape)}")
        x = x.detach().to(device=self.device)
        return x if x.dtype in (torch.float32, torch.bfloat16, torch.float16) else x.float()

    def add(self, x) -> None:
        x = self._rows(x, "add")
        if not bool(torch.isfinite(x).all()):
            raise RuntimeError("add: vectors must be finite")
        t = mx4_quantize(x)
        if self.metric == "L2":  # ||x||^2 / 2 of the packed rows
            step = max(1, (1 << 26) // self.d)
            self._norms += [t[s:s + step].dequantize().square_().sum(1).mul_(0.5) for s in range(0, len(t), step)]
        self._parts.append(t)
        self.ntotal += len(t)

    def _packed(self) -> MX4Tensor:
        if len(self._parts) != 1:
            self._parts = [MX4Tensor(torch.cat([p.codes for p in self._parts], 1),
                                     torch.cat([p.scales for p in self._parts], 1), self.d)]
        return self._parts[0]

    def reconstruct_n(self, i0: int, ni: int) -> torch.Tensor:
        """Rows i0 .. i0 + ni as they are stored, (ni, d) float32."""
        if not (0 <= i0 and 0 <= ni and i0 + ni <= self.ntotal):
            raise RuntimeError(f"reconstruct_n: rows {i0} .. {i0 + ni} of {self.ntotal}")
        if ni == 0:
            return torch.empty((0, self.d), device=self.device)
        return self._packed()[i0:i0 + ni].dequantize()

    def scores(self, x, out: torch.Tensor | None = None) -> torch.Tensor:
        """(nq, ntotal) float32, smaller is nearer: ||x||^2 / 2 - q.x (L2) or -q.x."""
        q = self._rows(x, "scores")
        if not self.ntotal:
            return torch.empty((q.shape[0], 0), device=self.device)
        norms = None
        if self.metric == "L2":
            if len(self._norms) != 1:
                self._norms = [torch.cat(self._norms)]
            norms = self._norms[0]
        return mx4_linear(q, self._packed(), norms, alpha=-1.0, out_dtype=torch.float32, out=out)

    def search(self, x, k: int):
        as_numpy = not isinstance(x, torch.Tensor)
        q, k, n, c = self._rows(x, "search"), int(k), self.ntotal, self._CHUNK
        if not 1 <= k <= 256:
            raise RuntimeError(f"search: k must be 1..256, not {k}")
        nq, parts = q.shape[0], max(1, -(-n // c))
        D = torch.full((nq, k), float("-inf" if self.metric == "inner_product" else "inf"), device=self.device)
        I = torch.full((nq, k), -1, dtype=torch.int64, device=self.device)
        with torch.cuda.device(self.device):
            step = max(1, (1 << 28) // (parts * c))
            for s in range(0, nq if n else 0, step):
                qs = q[s:s + step]
                b = qs.shape[0]
                # the k best of every 4096 scores, then the k best of those; places past the end are +inf
                S = torch.empty((b, parts * c), device=self.device)
                S[:, n:] = float("inf")
                self.scores(qs, out=S[:, :n])
                near, _ = select_probes(S.view(b * parts, c), "nearest", k)
                at = near.view(b, parts, k).long() + torch.arange(parts, device=self.device)[:, None] * c
                at = at.view(b, parts * k)
                best, _ = select_probes(S.gather(1, at), "nearest", k)
                at = at.gather(1, best.long())
                v = S.gather(1, at)
                there = (at < n) & ~torch.isnan(v)
                if self.metric == "L2":
                    v = (2 * v + mx4_quantize(qs).dequantize().square_().sum(1, keepdim=True)).clamp_(min=0)
                else:
                    v = -v
                D[s:s + b] = torch.where(there, v, D[s:s + b])
                I[s:s + b] = torch.where(there, at, I[s:s + b])
        return (D.cpu().numpy(), I.cpu().numpy()) if as_numpy else (D, I)
