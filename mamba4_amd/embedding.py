"""The scaled embedding lookup and its gradient by sorted tokens on MI355X.

    out_i = scale * table[ids_i],    d_table[r] = scale * sum of d_out_i, ids_i = r

An id outside the table gives a row of zeros and no gradient (-1 for padding,
say).  The gradient's sums are float32 in the order of the tokens whatever the
ids' distribution, so it is the same on every run.  Runs on the gfx950 HIP
library (``m4rt_embedding_*``, include/mamba4_retention.h) on the current stream.
"""

import torch

from mamba4_amd import _lib
from mamba4_amd.attention import _on, _same_device, _stream, _workspace
from mamba4_amd.memory import _differentiated, _ptr

_DTYPES = (torch.float32, torch.bfloat16)


def _forward(ids, table, scale, dtype):
    rows, width = table.shape
    out = torch.empty((*ids.shape, width), dtype=dtype, device=table.device)
    rc = _lib.load().m4rt_embedding_forward(
        ids.data_ptr(), ids.dtype == torch.int64, table.data_ptr(), table.dtype == torch.bfloat16,
        ids.numel(), rows, width, scale, out.data_ptr(), dtype == torch.bfloat16,
        _stream(table.device),
    )
    if rc:
        _lib.check(rc)
    return out


class _Embedding(torch.autograd.Function):
    """ids int32 or int64, table float32 or bfloat16, both contiguous."""

    @staticmethod
    def forward(ctx, ids, table, scale, dtype):
        ctx.save_for_backward(ids)
        ctx.args = (tuple(table.shape), table.dtype, scale, dtype)
        return _forward(ids, table, scale, dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out):
        lib = _lib.load()
        (ids,) = ctx.saved_tensors
        (rows, width), table_dtype, scale, dtype = ctx.args
        d_out = d_out.to(dtype).contiguous()
        d_table = torch.empty(rows, width, dtype=table_dtype, device=ids.device)
        nbytes = lib.m4rt_embedding_workspace_bytes(ids.numel(), rows, width)
        workspace = _workspace(nbytes, ids.device)
        _lib.check(
            lib.m4rt_embedding_backward(
                _ptr(ids), int(ids.dtype == torch.int64), _ptr(d_out),
                int(dtype == torch.bfloat16), ids.numel(), rows, width, scale, _ptr(d_table),
                int(table_dtype == torch.bfloat16), _ptr(workspace), nbytes, _stream(ids.device),
            )
        )
        return None, d_table, None, None


def embedding(ids, table, *, scale=1.0, dtype=None):
    """Rows of table [rows, width] (float32 or bfloat16) by ids [...] (int32 or
    int64), times ``scale``, in ``dtype`` (float32 or bfloat16; the table's by
    default), rounded once.  Differentiable in the table, whose gradient is in
    its dtype.
    """
    _same_device(ids, table)
    if ids.dtype not in (torch.int32, torch.int64):
        raise ValueError("embedding needs int32 or int64 ids")
    if table.dim() != 2 or table.shape[0] == 0 or table.shape[1] == 0:
        raise ValueError("embedding needs a table [rows, width]")
    dtype = table.dtype if dtype is None else dtype
    if table.dtype not in _DTYPES or dtype not in _DTYPES:
        raise ValueError("embedding takes float32 and bfloat16")
    if ids.numel() == 0:
        return table[:0].to(dtype).reshape(*ids.shape, table.shape[1])
    ids, table = ids.contiguous(), table.contiguous()
    with _on(table.device):
        if _differentiated(table):
            return _Embedding.apply(ids, table, float(scale), dtype)
        return _forward(ids, table, float(scale), dtype)
