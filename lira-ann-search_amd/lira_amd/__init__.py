"""lira_amd -- MI355X (gfx950) implementation of LIRA's query-time hot path.

The hot path of qfshen23/LIRA-ANN-search (partition ranking, candidate scan,
exact top-k) as hand-written HIP kernels behind a C-ABI (include/lira_hip.h,
liblira_hip.so), with the reference's Python-side interfaces on top:

* ``PartitionedIndex``       -- search.cpp's inverted lists + scan (search.cpp:366-514)
* ``IndexFlatL2/IndexFlatIP`` -- the faiss flat indexes LIRA builds per bucket
* ``utils``                  -- get_dist_cid / create_flat_indexes / get_cmp_recall /
                                query_tuning (utils.py, LIRA_smallscale.py)
* ``search``                 -- search.cpp's end-to-end artifact search
* ``mx4``                    -- microscaled 4-bit rows and their products
* ``distill``                -- distillation of a probing model from a teacher's top outputs
* ``knn``                    -- compute_knn.cpp self-kNN, k-means (utils.py:222-330)
"""
from ._lib import LiraError, load as load_library  # noqa: F401
from .index import (PartitionedIndex, build_csr, centroid_dist, centroid_gemm,  # noqa: F401
                    normalize_metric, order_probes, rank_nearest, select_probes, RankWorkspace)
from .faiss_compat import IndexFlatIP, IndexFlatL2, IndexMX4  # noqa: F401
from .mx4 import MX4Tensor, mx4_dequantize, mx4_linear, mx4_matmul, mx4_quantize  # noqa: F401
from .distill import distill_topk_loss, distill_topk_loss_and_grad  # noqa: F401

__all__ = [
    "LiraError", "PartitionedIndex", "build_csr", "centroid_dist", "centroid_gemm",
    "rank_nearest", "select_probes", "order_probes", "normalize_metric", "IndexFlatL2", "IndexFlatIP", "IndexMX4",
    "RankWorkspace", "load_library", "MX4Tensor", "mx4_quantize", "mx4_dequantize", "mx4_matmul", "mx4_linear",
    "distill_topk_loss", "distill_topk_loss_and_grad",
]
