"""Distillation of the head from a teacher's top logits: ``softmax_distill``.

The loss that trains the distribution the readout averages over: the divergence of
``softmax((logit_scale * h W^T + bias) / T)`` from a teacher known by its top logits, forward and
backward, without the ``[N, V]`` scores.  No counterpart in the reference library; its chunked
loss (swvr/api.py:44-66) is the sibling on the readout.

The forward is one pass over the vocabulary (softmax statistics and the teacher tokens' scores
come out of the same tiles), the backward recomputes the scores a vocabulary chunk at a time
(``chunk_size``, as ``softmax_readout``) and runs the readout's dW / dh GEMMs.
"""
from __future__ import annotations

import math
from typing import List, Optional, Tuple

import torch
from torch import nn

from . import _native as nat
from .api import _compute_dtype, _weight_of
from .embedding import _eager, _refuse_forward_ad
from .ops import (_REDUCTIONS, _grad_buffer, _ld, _no_grad_marker, _prepare_k, _require_cuda, _tensor_core, _workspace,
                  acc_dtype, default_chunk_size)

_ID_BITS = {torch.int64: 64, torch.int32: 32}
MAX_TEACHER = 1024


def _problem(hc, Wc, bias, ids, logits, t_lse, weight, sid, saved, temperature, logit_scale, chunk, cdt, reduction):
    """The C struct of one call.  It holds raw pointers only: the caller keeps every tensor referenced
    until the launch has been issued.  ``saved`` holds the forward's fp32 / fp64 results one after another
    (``_saved_numel``): log q and scores by sorted entry, then lse, its remainder, sum of q and loss by token, then the
    reduction's two numbers."""
    N, Kt = ids.shape
    p = nat.Distill()
    p.n_tokens, p.hidden = hc.shape
    p.vocab, p.teacher = Wc.shape[0], Kt
    p.compute_dtype = nat.dtype_code(cdt)
    p.bias_dtype = nat.dtype_code(bias.dtype) if bias is not None else 0
    p.teacher_dtype, p.id_bits = nat.dtype_code(logits.dtype), _ID_BITS[ids.dtype]
    p.h, p.ldh, p.W, p.ldw = hc.data_ptr(), _ld(hc), Wc.data_ptr(), _ld(Wc)
    p.bias = nat.ptr(bias)
    p.logit_scale, p.temperature, p.chunk, p.reduction = logit_scale, temperature, chunk, reduction
    p.teacher_ids, p.teacher_logits = ids.data_ptr(), logits.data_ptr()
    p.teacher_lse, p.weight = nat.ptr(t_lse), nat.ptr(weight)
    p.sid = sid.data_ptr()
    at, es = saved.data_ptr(), saved.element_size()
    p.slogq, p.z = at, at + es * N * Kt
    at += es * 2 * N * Kt
    p.lse, p.lse_lo, p.qsum, p.each, p.stats = at, at + es * N, at + es * 2 * N, at + es * 3 * N, at + es * 4 * N
    return p


def _saved_numel(N, Kt):
    return 2 * N * Kt + 4 * N + 2


def _operands(h, W, bias, cdt):
    return _prepare_k(h, cdt), _prepare_k(W, cdt), bias.contiguous() if bias is not None else None


def _distill_fwd(h, W, bias, ids, logits, t_lse, weight, temperature, logit_scale, chunk, cdt, reduction):
    dev = _require_cuda(h, W, bias, ids, logits, t_lse, weight)
    adt = acc_dtype(cdt)
    N, Kt = ids.shape
    out = torch.empty((N,) if reduction == nat.REDUCE_NONE else (), dtype=adt, device=dev)
    sid = torch.empty(N, Kt, dtype=torch.int32, device=dev)
    saved = torch.empty(_saved_numel(N, Kt), dtype=adt, device=dev)
    hc, Wc, b = _operands(h, W, bias, cdt)
    p = _problem(hc, Wc, b, ids, logits, t_lse, weight, sid, saved, temperature, logit_scale, chunk, cdt, reduction)
    lib = nat.lib()
    nbytes = nat.c_size_t(0)
    with nat.on_device(dev):
        nat.check(lib.swvr_distill_fwd_workspace_size(p, nat.ctypes.byref(nbytes)), "swvr_distill_fwd_workspace_size")
        ws = _workspace(nbytes.value, dev)
        nat.check(lib.swvr_distill_fwd(p, out.data_ptr(), ws.data_ptr(), ws.numel(), nat.stream_ptr(dev)),
                  "swvr_distill_fwd")
    return out, sid, saved


def _distill_bwd(grad, h, W, bias, ids, logits, t_lse, weight, sid, saved, temperature, logit_scale, chunk, cdt, reduction,
                 need_h, need_W, need_b, need_w):
    """(dh, dW, db, dweight), None where not asked for."""
    dev = _require_cuda(h, W, bias, ids, grad, weight)
    (N, K), V = h.shape, W.shape[0]
    hc, Wc, b = _operands(h, W, bias, cdt)
    K8 = hc.shape[1]
    grad = grad.to(saved.dtype).contiguous()
    gh = torch.empty(N, K8, dtype=h.dtype, device=dev) if need_h else None
    gW_buf, gW = _grad_buffer(W, cdt, _tensor_core(cdt)) if need_W else (None, None)
    if need_W and K8 != K:
        gW_buf = torch.empty(V, K8, dtype=gW_buf.dtype, device=dev)
    gb = torch.empty(V, dtype=bias.dtype, device=dev) if need_b and bias is not None else None
    gw = torch.empty(N, dtype=saved.dtype, device=dev) if need_w and weight is not None else None
    p = _problem(hc, Wc, b, ids, logits, t_lse, weight, sid, saved, temperature, logit_scale, chunk, cdt, reduction)
    g = nat.DistillGrads()
    g.grad_out = grad.data_ptr()
    if gh is not None:
        g.grad_h, g.grad_h_dtype = gh.data_ptr(), nat.dtype_code(gh.dtype)
    if gW_buf is not None:
        g.grad_W, g.grad_W_dtype, g.ld_grad_W = gW_buf.data_ptr(), nat.dtype_code(gW_buf.dtype), K8
    if gb is not None:
        g.grad_bias, g.grad_bias_dtype = gb.data_ptr(), nat.dtype_code(gb.dtype)
    g.grad_weight = nat.ptr(gw)
    lib = nat.lib()
    nbytes = nat.c_size_t(0)
    with nat.on_device(dev):
        nat.check(lib.swvr_distill_bwd_workspace_size(p, g, nat.ctypes.byref(nbytes)), "swvr_distill_bwd_workspace_size")
        ws = _workspace(nbytes.value, dev)
        nat.check(lib.swvr_distill_bwd(p, g, ws.data_ptr(), ws.numel(), nat.stream_ptr(dev)), "swvr_distill_bwd")
    if gh is not None and K8 != K:
        gh = gh[:, :K].contiguous()
    if gW is not None and gW_buf is not gW:
        gW.copy_(gW_buf[:, :K])
    return gh, gW, gb, gw


# Custom-op pair, like the readout's own (ops.py), for torch.compile and other tracing.  The outputs after
# the loss are what the backward needs of the forward: the sorted teacher ids and the values of
# ``_problem``; they take no gradient.

@torch.library.custom_op("swvr_b200::distill", mutates_args=())
def _distill_op(h: torch.Tensor, W: torch.Tensor, bias: Optional[torch.Tensor], ids: torch.Tensor, logits: torch.Tensor,
                t_lse: Optional[torch.Tensor], weight: Optional[torch.Tensor], temperature: float, logit_scale: float,
                chunk: int, cdt: torch.dtype, reduction: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return _distill_fwd(h, W, bias, ids, logits, t_lse, weight, temperature, logit_scale, chunk, cdt, reduction)


@_distill_op.register_fake
def _(h, W, bias, ids, logits, t_lse, weight, temperature, logit_scale, chunk, cdt, reduction):
    adt = acc_dtype(cdt)
    N, Kt = ids.shape
    return (h.new_empty((N,) if reduction == nat.REDUCE_NONE else (), dtype=adt), h.new_empty((N, Kt), dtype=torch.int32),
            h.new_empty((_saved_numel(N, Kt),), dtype=adt))


@torch.library.custom_op("swvr_b200::distill_bwd", mutates_args=())
def _distill_bwd_op(grad: torch.Tensor, h: torch.Tensor, W: torch.Tensor, bias: Optional[torch.Tensor],
                    ids: torch.Tensor, logits: torch.Tensor, t_lse: Optional[torch.Tensor],
                    weight: Optional[torch.Tensor], sid: torch.Tensor, saved: torch.Tensor, temperature: float,
                    logit_scale: float, chunk: int, cdt: torch.dtype, reduction: int, need_h: bool, need_W: bool,
                    need_b: bool, need_w: bool) -> List[torch.Tensor]:
    got = _distill_bwd(grad, h, W, bias, ids, logits, t_lse, weight, sid, saved, temperature, logit_scale, chunk, cdt,
                       reduction, need_h, need_W, need_b, need_w)
    return [t if t is not None else _no_grad_marker(h) for t in got]


@_distill_bwd_op.register_fake
def _(grad, h, W, bias, ids, logits, t_lse, weight, sid, saved, temperature, logit_scale, chunk, cdt, reduction, need_h,
      need_W, need_b, need_w):
    out = []
    for wanted, like in ((need_h, h), (need_W, W), (need_b and bias is not None, bias)):
        out.append(like.new_empty(like.shape) if wanted else _no_grad_marker(h))
    return out + [saved.new_empty(h.shape[0]) if need_w and weight is not None else _no_grad_marker(h)]


def _save(ctx, inputs, sid, saved):
    h, W, bias, ids, logits, t_lse, weight, *consts = inputs
    ctx.save_for_backward(h, W, bias, ids, logits, t_lse, weight, sid, saved)
    ctx.consts = consts
    ctx.set_materialize_grads(False)


def _grads(ctx, grad, run):
    h, W, bias, ids, logits, t_lse, weight, sid, saved = ctx.saved_tensors
    if grad is None:  # the loss did not reach what is differentiated
        return (None,) * (7 + len(ctx.consts))
    want = [bool(ctx.needs_input_grad[i]) and t is not None for i, t in ((0, h), (1, W), (2, bias), (6, weight))]
    got = run(grad, h, W, bias, ids, logits, t_lse, weight, sid, saved, *ctx.consts, *want)
    gh, gW, gb, gw = (t if w else None for t, w in zip(got, want))
    return (gh, gW, gb, None, None, None, gw) + (None,) * len(ctx.consts)


_distill_op.register_autograd(lambda ctx, grad, *_: _grads(ctx, grad, _distill_bwd_op),
                              setup_context=lambda ctx, inputs, output: _save(ctx, inputs, *output[1:]))


class _Distill(torch.autograd.Function):
    """The custom op's forward and backward without its dispatch, for eager calls."""

    @staticmethod
    def forward(ctx, *inputs):
        out, sid, saved = _distill_fwd(*inputs)
        _save(ctx, inputs, sid, saved)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        return _grads(ctx, grad, _distill_bwd)


def softmax_distill(h, W, teacher_ids, teacher_logits, bias=None, *, temperature=1.0, teacher_lse=None, weight=None,
                    reduction="mean", logit_scale=1.0, chunk_size=None):
    """Distillation loss of the head ``softmax((logit_scale * h @ W.T + bias) / T)`` against a teacher's
    top logits.

    ``teacher_ids`` (int64 or int32) and ``teacher_logits`` (floating) are ``[..., K_t]`` over h's
    leading shape, at most 1024 entries per token, in any order.  The teacher's probabilities are
    ``q = softmax(teacher_logits / T)`` over those entries, or, with ``teacher_lse`` (the
    logsumexp of all the teacher's logits / T, h's leading shape), ``q = exp(teacher_logits / T -
    teacher_lse)``, which leaves out the mass of the tokens not listed.  For each token the loss is ``T^2 *
    sum_k q_k (log q_k - log p[id_k])``; ``weight`` (h's leading shape) multiplies it, a zero weight
    drops the token, and ``reduction`` is as in ``softmax_readout_mse``.  Returns fp32 (fp64 when
    the inputs are fp64), differentiable in ``h``, ``W``, ``bias`` and ``weight``; the teacher is a
    constant.

    A dropped token may have an infinite loss, but its row of ``h`` is read and must be finite (0 times inf in
    dW).  An entry with a negative id or a logit of -inf is left out, and a token with none left has loss 0
    and no gradient.  An id at or past V makes its token's loss NaN and is reported by
    ``_native.check_device_error()``.  ``chunk_size`` is that of ``softmax_readout``; under autocast h and W are
    cast whole, in the forward and again in the backward, as they are copied where the hidden size is no multiple of 8 in 16
    bits.  W is the whole vocabulary, not a shard of it.  fp32 and fp64 take at most 65535 * 128 tokens.  There is no
    forward-mode derivative.
    """
    if W.dim() != 2:
        raise ValueError(f"W must be 2-D, got {tuple(W.shape)}")
    if h.shape[-1] != W.shape[1]:
        raise ValueError(f"h has hidden size {h.shape[-1]} but W is {tuple(W.shape)}")
    V = W.shape[0]
    if V == 0:
        raise ValueError("W has no vocabulary rows")
    if bias is not None and bias.shape != (V,):
        raise ValueError(f"bias must have shape ({V},), got {tuple(bias.shape)}")
    lead = h.shape[:-1]
    if teacher_ids.dim() < 1 or teacher_ids.shape[:-1] != lead or teacher_logits.shape != teacher_ids.shape:
        raise ValueError(f"teacher_ids and teacher_logits must be {tuple(lead)} + (K_t,), got {tuple(teacher_ids.shape)} "
                         f"and {tuple(teacher_logits.shape)}")
    if teacher_ids.dtype not in _ID_BITS:
        raise ValueError(f"teacher_ids must be int64 or int32, got {teacher_ids.dtype}")
    Kt = teacher_ids.shape[-1]
    if Kt > MAX_TEACHER:
        raise ValueError(f"at most {MAX_TEACHER} teacher entries per token, got {Kt}")
    for name, t in (("teacher_lse", teacher_lse), ("weight", weight)):
        if t is not None and t.shape != lead:
            raise ValueError(f"{name} must have shape {tuple(lead)}, got {tuple(t.shape)}")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"unknown reduction {reduction!r}")
    temperature = float(temperature)
    if not (temperature > 0 and math.isfinite(temperature)):
        raise ValueError(f"temperature must be positive and finite, got {temperature}")
    chunk = int(chunk_size) if chunk_size else default_chunk_size()
    if chunk <= 0:
        raise ValueError(f"chunk_size must be positive, got {chunk}")
    nat.dtype_code(teacher_logits.dtype)
    cdt = _compute_dtype(h, W)
    nat.dtype_code(cdt)
    _refuse_forward_ad("softmax_distill", h, W, bias, weight)
    adt = acc_dtype(cdt)
    N = math.prod(lead)

    def row(t):
        t = t if t.dtype == adt else t.to(adt)
        return (t if t.dim() == 1 else t.reshape(N)).contiguous()

    def flat(t, last):
        return t if t.dim() == 2 else t.reshape(N, last)

    if teacher_logits.requires_grad:
        teacher_logits = teacher_logits.detach()
    if teacher_lse is not None and teacher_lse.requires_grad:
        teacher_lse = teacher_lse.detach()

    args = (flat(h, h.shape[-1]), W, bias, flat(teacher_ids, Kt).contiguous(), flat(teacher_logits, Kt).contiguous(),
            None if teacher_lse is None else row(teacher_lse), None if weight is None else row(weight), temperature,
            float(logit_scale), chunk, cdt, _REDUCTIONS[reduction])
    if _eager(*args[:7]):
        out = _Distill.apply(*args)
    else:
        with torch.autocast(h.device.type, enabled=False):
            out = _distill_op(*args)[0]
    return out.view(lead) if reduction == "none" and len(lead) != 1 else out


class SoftmaxDistill(nn.Module):
    """``softmax_distill`` as an ``nn.Module`` bound to a model's head, as ``SoftmaxReadoutMSE``: ``head`` is an
    ``nn.Linear(K, V)`` (whose bias, if any, is the score bias) or a ``[V, K]`` weight, stored, never copied."""

    def __init__(self, head, *, temperature=1.0, logit_scale=1.0, reduction="mean", chunk_size=None):
        super().__init__()
        self.head = head
        self.temperature, self.logit_scale = temperature, logit_scale
        self.reduction, self.chunk_size = reduction, chunk_size

    def forward(self, h, teacher_ids, teacher_logits, weight=None, teacher_lse=None):
        bias = getattr(self.head, "bias", None) if isinstance(self.head, nn.Module) else None
        return softmax_distill(h, _weight_of(self.head), teacher_ids, teacher_logits, bias, temperature=self.temperature,
                               teacher_lse=teacher_lse, weight=weight, reduction=self.reduction,
                               logit_scale=self.logit_scale, chunk_size=self.chunk_size)
