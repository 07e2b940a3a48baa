"""B200-native (sm_100a) TRELLIS sparse-voxel path: the drop-in for mlx_diffuser's
``SparseTensor`` / ``build_neighbor_map`` / ``SparseConv3D`` / ``sparse_conv3d`` /
``sparse_downsample`` / ``sparse_upsample``, backed by ``libsparsevox.so``, and the operators of a
transformer block over the same rows: ``rms_norm``, ``linear`` and ``sparse_self_attention`` with a
learned relative position bias."""

from ._native import check_device_status
from .kernels.linear import linear
from .kernels.norm import rms_norm
from .kernels.sparse import sparse_conv3d
from .layers.sparse import (
    SparseConv3D,
    SparseTensor,
    build_neighbor_map,
    position_buckets,
    sparse_downsample,
    sparse_self_attention,
    sparse_upsample,
)

__all__ = [
    "SparseConv3D",
    "SparseTensor",
    "build_neighbor_map",
    "check_device_status",
    "linear",
    "position_buckets",
    "rms_norm",
    "sparse_conv3d",
    "sparse_downsample",
    "sparse_self_attention",
    "sparse_upsample",
]
