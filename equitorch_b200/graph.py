"""Edge lists prepared for the fused graph kernels.

A layer of a message-passing network evaluates one tensor product per edge
``(source -> destination)`` and sums the results per destination node.  The fused kernels
walk the edges grouped by the node they reduce into, so they need the edges in CSR order by
destination (forward pass and the gradient of the edge attributes) and in CSR order by source
(gradient of the node features).  ``EdgeGraph`` computes both orders once; edge attributes
(vectors, spherical harmonics) always stay in the caller's order and are addressed through the
stored permutations.

Convention: ``edge_index[0]`` = source (row gathered from), ``edge_index[1]`` = destination
(row summed into), as in ``equitorch/transforms/__init__.py:99-101`` of the reference.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor

from . import _lib


def _csr(sorted_ids: Tensor, n: int) -> Tensor:
    ptr = torch.zeros(n + 1, dtype=torch.int64, device=sorted_ids.device)
    if sorted_ids.numel():
        ptr[1:] = torch.cumsum(torch.bincount(sorted_ids, minlength=n), 0)
    return ptr


class EdgeGraph:
    """CSR-by-destination and CSR-by-source views of an edge list.

    Attributes (all int64 tensors on the edges' device):
      ``dst_ptr`` (num_dst + 1), ``dst_sorted`` (E), ``src_by_dst`` (E), ``dst_order`` (E) or ``None``
      when the edges already are sorted by destination; ``src_ptr`` (num_src + 1), ``dst_by_src`` (E),
      ``src_order`` (E): the same for the grouping by source.
    """

    def __init__(self, src: Tensor, dst: Tensor, num_src: int, num_dst: Optional[int] = None):
        assert src.dtype == torch.int64 and dst.dtype == torch.int64 and src.shape == dst.shape and src.ndim == 1
        self.num_src = int(num_src)
        self.num_dst = int(num_src if num_dst is None else num_dst)
        self.num_edges = src.numel()
        already = bool((dst[1:] >= dst[:-1]).all()) if dst.numel() > 1 else True
        if already:
            self.dst_order, self.dst_sorted, self.src_by_dst = None, dst.contiguous(), src.contiguous()
        else:
            self.dst_order = torch.argsort(dst, stable=True)
            self.dst_sorted, self.src_by_dst = dst[self.dst_order], src[self.dst_order]
        self.dst_ptr = _csr(self.dst_sorted, self.num_dst)
        self.src_order = torch.argsort(src, stable=True)
        self.dst_by_src = dst[self.src_order]
        self.src_ptr = _csr(src[self.src_order], self.num_src)

    @property
    def device(self):
        return self.dst_ptr.device

    def to(self, device) -> "EdgeGraph":
        out = object.__new__(EdgeGraph)
        for k, v in self.__dict__.items():
            setattr(out, k, v.to(device) if isinstance(v, Tensor) else v)
        return out

    @staticmethod
    def from_edge_index(edge_index: Tensor, num_nodes: int) -> "EdgeGraph":
        return EdgeGraph(edge_index[0], edge_index[1], num_nodes)


class PackedGraphs:
    """Which nodes of a batch belong to which graph: graph g has the nodes ``[ptr[g], ptr[g + 1])``, as ``segment_sum`` and
    ``torch_geometric``'s batches have it.  Computed once per batch, for every layer that works within graphs.

    Nodes before ``ptr[0]`` and from ``ptr[-1]`` on belong to no graph.  Attributes: ``ptr`` (num_graphs + 1, int64), ``num_nodes``,
    ``num_graphs``, ``longest`` (nodes of the largest graph), ``covers`` (every node has a graph), ``tile_rows`` and ``tiles``
    (num_tiles, 4, int32: first row, first node and one past the last node of its graph, 0), the pieces of at most ``tile_rows`` nodes of one graph that the kernels work on, those of
    the largest graphs first.  Reads a few numbers back to the host.  Boundaries may lie on the host too (``to`` moves the result).
    """

    def __init__(self, ptr: Tensor, num_nodes: int):
        if ptr.dtype != torch.int64 or ptr.ndim != 1 or ptr.numel() < 1:
            raise ValueError(f"int64 boundaries of the graphs expected, at least one, got {ptr.dtype} of shape {tuple(ptr.shape)}")
        if not 0 <= int(num_nodes) < 2 ** 31 - 64:
            raise ValueError(f"num_nodes must be in [0, 2^31 - 64), got {num_nodes}")
        self.ptr, self.num_nodes, self.num_graphs = ptr.contiguous().clone(), int(num_nodes), ptr.numel() - 1
        on_gpu = self.ptr.is_cuda
        first, last, least, self.longest, *tiles = (self._stats_gpu() if on_gpu else self._stats()).tolist()
        if least < 0 or first < 0 or last > self.num_nodes:
            raise ValueError(f"boundaries of the graphs must ascend within [0, {self.num_nodes}]")
        self.covers = first == 0 and last == self.num_nodes
        # Rows behind the end of a graph are work for nothing, and a tile of more rows reads the other side fewer times: the largest
        # tile with at most an eighth (a quarter, for the largest) more rows than the smaller ones.  Forward and backward pass of
        # attention with tiles of 16, 32 and 64 rows: 2000 graphs of 5 to 60 nodes (1.2 and 1.5 times the rows) 347, 384 and 454 us,
        # 48 graphs of 40 to 250 (1.05 and 1.16 times) 752, 655 and 497.  A graph of more than 8192 nodes, which is most of a batch's work,
        # takes the largest in any company: the kernels whose sums reach that far have no other.
        self.tile_rows = 64 if self.longest > 8192 or 64 * tiles[2] <= 1.25 * 32 * tiles[1] else 32 if 32 * tiles[1] <= 1.125 * 16 * tiles[0] else 16
        total = tiles[(16, 32, 64).index(self.tile_rows)]
        self.tiles = self._tiles_gpu(total) if on_gpu else self._tiles(total)

    def _stats_gpu(self) -> Tensor:
        stats = torch.empty(7, dtype=torch.int64, device=self.device)
        with _lib.on_device(self.device):
            _lib.check(_lib.lib().eqt_pack_graphs_stats(self.ptr.data_ptr(), self.num_graphs, stats.data_ptr(), _lib.stream_ptr(self.device)),
                       "eqt_pack_graphs_stats")
        return stats

    def _tiles_gpu(self, total: int) -> Tensor:
        tiles = torch.empty(total, 4, dtype=torch.int32, device=self.device)
        with _lib.on_device(self.device):
            _lib.check(_lib.lib().eqt_pack_graphs_tiles(self.ptr.data_ptr(), self.num_graphs, tiles.data_ptr(), total, self.tile_rows,
                                                        _lib.stream_ptr(self.device)), "eqt_pack_graphs_tiles")
        return tiles

    def _stats(self) -> Tensor:
        """For boundaries that a data loader holds on the host."""
        sizes = self.ptr[1:] - self.ptr[:-1]
        least, greatest = (sizes.min(), sizes.max()) if self.num_graphs else (sizes.new_zeros(()),) * 2
        return torch.stack([self.ptr[0], self.ptr[-1], least, greatest, *(((sizes.clamp(min=0) + r - 1) // r).sum() for r in (16, 32, 64))])

    def _tiles(self, total: int) -> Tensor:
        sizes = self.ptr[1:] - self.ptr[:-1]
        by_size = torch.argsort(sizes, descending=True, stable=True)
        count = ((sizes + self.tile_rows - 1) // self.tile_rows)[by_size]
        graph = torch.repeat_interleave(by_size, count, output_size=total)
        place = torch.arange(total, device=self.device) - torch.repeat_interleave(torch.cumsum(count, 0) - count, count, output_size=total)
        low = self.ptr[:-1][graph]
        return torch.stack([low + place * self.tile_rows, low, self.ptr[1:][graph], torch.zeros_like(low)], 1).int().contiguous()

    @property
    def device(self):
        return self.ptr.device

    def to(self, device) -> "PackedGraphs":
        out = object.__new__(PackedGraphs)
        for k, v in self.__dict__.items():
            setattr(out, k, v.to(device) if isinstance(v, Tensor) else v)
        return out

    @staticmethod
    def from_batch(batch: Tensor, num_graphs: int) -> "PackedGraphs":
        """From the graph of every node, ascending (``batch`` of ``torch_geometric``)."""
        if batch.dtype != torch.int64 or batch.ndim != 1:
            raise ValueError(f"int64 graph of every node expected, got {batch.dtype} of shape {tuple(batch.shape)}")
        if batch.numel() and bool(((batch[1:] < batch[:-1]).any() | (batch[0] < 0) | (batch[-1] >= num_graphs))):
            raise ValueError(f"the graph of every node must ascend within [0, {num_graphs})")
        return PackedGraphs(_csr(batch, num_graphs), batch.numel())
