"""Operations on compressed block-sparse tensors (the matmul path and the ops around it) and the products of expert layers."""
from .conversion import from_blksprs, to_blksprs, to_dense, to_dense_shaped, to_sparse, to_sparse_shaped
from .grouped_matmul import grouped_matmul, grouped_matmul_scaled
from .matmul import matmul
from .matmul_softmax import matmul_softmax
from .quantize import quantize_blocks, quantize_rows
from .softmax import softmax, softmax_fused, softmax_regular
from .transpose import transpose

__all__ = ["from_blksprs", "grouped_matmul", "grouped_matmul_scaled", "matmul", "matmul_softmax", "quantize_blocks",
           "quantize_rows", "softmax", "softmax_fused", "softmax_regular", "to_blksprs", "to_dense", "to_dense_shaped",
           "to_sparse", "to_sparse_shaped", "transpose"]
