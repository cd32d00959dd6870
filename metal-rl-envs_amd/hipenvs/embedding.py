"""Rows of a table for tokens, scaled, with the gradient of the table: a policy's input of actions it
took or of observations given as tokens. The reference has no counterpart.

    out[i] = scale table[tokens[i]]        dtable[v] = scale sum of the dout[i] with tokens[i] = v

A negative token is none (an episode's first step has no action before it): a row of zeros that adds to
no gradient. A token past the table is a mistake that the host does not wait to see: its row is no
number, and adds to no gradient. The gradient is a sum over sorted tokens, in float32 and in an order
that depends on the tokens alone, rounded once to the table's type: the same bits on every run.
"""

import torch

from . import _checks, _lib

MAX_WIDTH = 65536


def _forward(tokens, table, scale):
    v, d = table.shape
    out = torch.empty((*tokens.shape, d), dtype=table.dtype, device=table.device)
    with _lib.on(table.device):
        _lib.call("hipenvs_embedding", _checks.DTYPES[table.dtype], tokens.data_ptr(), tokens.element_size(),
                  table.data_ptr(), table.stride(0), scale, out.data_ptr(), tokens.numel(), v, d,
                  _lib.stream_of(table.device))
    return out


def _backward(ctx, dout):
    tokens, = ctx.saved_tensors
    dtype, (v, d), shape, device, scale = ctx.ready
    if dout is None:
        return None, None, None
    tokens = _tokens(tokens, device.index)
    if tokens.shape != shape:   # as many rows of dout are read as there are tokens
        raise ValueError(f"saved tokens must have shape {tuple(shape)}, got {tuple(tokens.shape)}")
    _checks.refuse_tangents("the gradient of lookup", dout)
    dout = _checks.saved(dout, dtype, (*shape, d), device.index).view(-1, d) if tokens.numel() else dout.reshape(0, d)
    dtable = torch.empty((v, d), dtype=dtype, device=device)
    with _lib.on(device):
        nbytes = _lib.lib().hipenvs_embedding_workspace_bytes(tokens.numel(), v, d)
        if nbytes < 0:
            raise _lib.HipEnvsError(f"hipenvs_embedding: unsupported sizes ({tokens.numel()}, {v}, {d})")
        held = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
        _lib.call("hipenvs_embedding_backward", _checks.DTYPES[dtype], tokens.data_ptr(), tokens.element_size(),
                  dout.data_ptr(), dout.stride(0), scale, dtable.data_ptr(), tokens.numel(), v, d, _lib.ptr(held),
                  nbytes, _lib.stream_of(device))
    return None, dtable, None


class _Lookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, table, scale):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(tokens)
        ctx.ready = (table.dtype, tuple(table.shape), tuple(tokens.shape), table.device, scale)
        return _forward(tokens, table, scale)

    backward = _checks.once(_backward)


def _tokens(tokens, device):
    if _checks.tensor(tokens, "tokens").dtype not in (torch.int32, torch.int64):
        raise TypeError(f"tokens must be int32 or int64, got {tokens.dtype}")
    if tokens.get_device() != device:
        raise ValueError(f"tokens are on {tokens.device}, table is on GPU {device}")
    if tokens.numel() > 0x7FFFFFFF:
        raise ValueError(f"there must be fewer than 2^31 tokens, got {tokens.numel()}")
    return tokens.contiguous()


def lookup(tokens, table, scale=1.0):
    """tokens of any shape, int32 or int64, table (v, d) float32 or bfloat16 with a contiguous last
    axis (copied otherwise). Returns (*tokens.shape, d) of table's type, differentiable once in table,
    in reverse mode. Asynchronous on the current stream."""
    device = _checks.first(table, "table", 2)
    v, d = table.shape
    if v < 1 or not 1 <= d <= MAX_WIDTH:
        raise ValueError(f"table must have rows of 1 to {MAX_WIDTH} values, got shape {tuple(table.shape)}")
    table = _checks.rows(table, "table", table.dtype, (v, d), device, "table")
    tokens = _tokens(tokens, device)
    _checks.refuse_tangents("lookup", table)
    scale = float(scale)
    if _checks.wants_grad(table):
        return _Lookup.apply(tokens, table, scale)
    return _forward(tokens, table, scale)
