"""Embedding lookup with scaling, and its gradient by token: ``embedding_lookup``.

The input side of the table the readout averages: ``softmax_readout`` returns the mean row of
``E`` under a distribution over tokens, ``embedding_lookup`` the row of one token.  With a tied
table both run on the same parameter and their gradients add.  No counterpart in the
reference library, whose callers use ``nn.Embedding`` (swvr/api.py:69-93 takes its weight).

The gradient is dense, in the table's dtype, and deterministic: libswvr_b200.so sorts the tokens
and sums each one's rows in order, in fp32 (fp64 for fp64), without atomics.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _native as nat
from .ops import _require_cuda, _workspace

_TOKEN_BITS = {torch.int64: 64, torch.int32: 32}


def _unit_rows(x: torch.Tensor) -> torch.Tensor:
    """``x`` [rows, cols] with a unit last stride and rows at least ``cols`` apart."""
    rows, cols = x.shape
    return x if (cols <= 1 or x.stride(1) == 1) and (rows <= 1 or x.stride(0) >= max(cols, 1)) else x.contiguous()


def _pitch(x: torch.Tensor) -> int:
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _embed_fwd(tokens: torch.Tensor, E: torch.Tensor, scale: float) -> torch.Tensor:
    dev = _require_cuda(E, tokens)
    E = _unit_rows(E)
    tokens = tokens.contiguous()
    out = torch.empty(tokens.shape[0], E.shape[1], dtype=E.dtype, device=dev)
    with nat.on_device(dev):
        nat.check(nat.lib().swvr_embed_fwd(tokens.shape[0], E.shape[0], E.shape[1], tokens.data_ptr(),
                                           _TOKEN_BITS[tokens.dtype], E.data_ptr(), nat.dtype_code(E.dtype), _pitch(E),
                                           scale, out.data_ptr(), nat.stream_ptr(dev)), "swvr_embed_fwd")
    return out


def _embed_bwd(g: torch.Tensor, tokens: torch.Tensor, V: int, scale: float, padding: int) -> torch.Tensor:
    dev = _require_cuda(g, tokens)
    g, tokens = _unit_rows(g), tokens.contiguous()
    N, D = g.shape
    dt = nat.dtype_code(g.dtype)
    dE = torch.empty(V, D, dtype=g.dtype, device=dev)
    lib = nat.lib()
    nbytes = nat.c_size_t(0)
    with nat.on_device(dev):
        nat.check(lib.swvr_embed_bwd_workspace_size(N, V, D, dt, nat.ctypes.byref(nbytes)),
                  "swvr_embed_bwd_workspace_size")
        ws = _workspace(nbytes.value, dev)
        nat.check(lib.swvr_embed_bwd(N, V, D, tokens.data_ptr(), _TOKEN_BITS[tokens.dtype], g.data_ptr(), _pitch(g),
                                     scale, padding, dE.data_ptr(), dt, D, ws.data_ptr(), ws.numel(),
                                     nat.stream_ptr(dev)), "swvr_embed_bwd")
    return dE


# Opaque custom ops, like the readout's own (ops.py).

@torch.library.custom_op("swvr_b200::embed", mutates_args=())
def _embed_op(tokens: torch.Tensor, E: torch.Tensor, scale: float, padding: int) -> torch.Tensor:
    return _embed_fwd(tokens, E, scale)


@_embed_op.register_fake
def _(tokens, E, scale, padding):
    return E.new_empty(tokens.shape[0], E.shape[1])


@torch.library.custom_op("swvr_b200::embed_bwd", mutates_args=())
def _embed_bwd_op(g: torch.Tensor, tokens: torch.Tensor, V: int, scale: float, padding: int) -> torch.Tensor:
    return _embed_bwd(g, tokens, V, scale, padding)


@_embed_bwd_op.register_fake
def _(g, tokens, V, scale, padding):
    return g.new_empty(V, g.shape[1])


def _embed_setup(ctx, inputs, output):
    tokens, E, scale, padding = inputs
    ctx.save_for_backward(tokens)
    ctx.consts = (E.shape[0], scale, padding)


def _embed_backward(ctx, g):
    (tokens,) = ctx.saved_tensors
    return None, (_embed_bwd_op(g, tokens, *ctx.consts) if ctx.needs_input_grad[1] else None), None, None


_embed_op.register_autograd(_embed_backward, setup_context=_embed_setup)


class _Embed(torch.autograd.Function):
    """The custom op's forward and backward without its dispatch, for eager calls."""

    @staticmethod
    def forward(ctx, tokens, E, scale, padding):
        ctx.save_for_backward(tokens)
        ctx.consts = (E.shape[0], scale, padding)
        return _embed_fwd(tokens, E, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        (tokens,) = ctx.saved_tensors
        return None, _embed_bwd(g, tokens, *ctx.consts), None, None


def _eager(*tensors) -> bool:
    """True where an op may be run without its custom op: plain tensors, and no tracing, dispatch mode or functorch
    transform (``torch.func.vmap`` and the like, whose tensors are of the plain type) that has to see it.  It saves the
    dispatcher's host time, most of a call on a few tokens."""
    return not (torch.compiler.is_compiling() or torch._C._len_torch_dispatch_stack()
                or torch._C._are_functorch_transforms_active()) and all(
        t is None or type(t) in (torch.Tensor, torch.nn.Parameter) for t in tensors)


def _refuse_forward_ad(name, *tensors):
    """Raise where a tensor carries a tangent (``torch.func.jvp``, dual tensors): a custom op would pass none on, and
    forward mode would take that for a derivative of zero."""
    if forward_ad._current_level < 0:
        return
    for t in tensors:
        while t is not None and torch._C._functorch.is_batchedtensor(t):
            t = torch._C._functorch.get_unwrapped(t)
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{name} has no forward-mode derivative")


def embedding_lookup(tokens, E, *, scale=1.0, padding_idx=None):
    """``scale * E[tokens]``: tokens ``[...]`` (int64 or int32) into the rows of ``E`` ``[V, D]``;
    returns ``[..., D]`` in E's dtype, the product rounded once, differentiable in ``E``.

    ``padding_idx`` (negative: from the end, as ``nn.Embedding``) names a row that takes no
    gradient.  Rows of ``E`` may be strided.  A token outside ``[0, V)`` is an error that the host
    learns of at ``_native.check_device_error()``: its row comes back as NaN and the gradient
    leaves it out.  Autocast leaves the lookup in E's dtype, as torch's own.  E is the whole table, not a shard of it.  There is
    no forward-mode derivative.
    """
    if E.dim() != 2:
        raise ValueError(f"E must be 2-D, got {tuple(E.shape)}")
    if tokens.dtype not in _TOKEN_BITS:
        raise ValueError(f"tokens must be int64 or int32, got {tokens.dtype}")
    nat.dtype_code(E.dtype)
    V = E.shape[0]
    padding = -1
    if padding_idx is not None:
        padding = int(padding_idx)
        if not -V <= padding < V:
            raise ValueError(f"padding_idx {padding_idx} is outside a table of {V} rows")
        padding += V if padding < 0 else 0
    _refuse_forward_ad("embedding_lookup", E)
    flat = tokens if tokens.dim() == 1 else tokens.reshape(-1)
    out = (_Embed.apply if _eager(flat, E) else _embed_op)(flat, E, float(scale), padding)
    return out if tokens.dim() == 1 else out.view(*tokens.shape, E.shape[1])
