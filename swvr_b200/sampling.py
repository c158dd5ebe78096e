"""Sampling of tokens from the head's distribution: ``softmax_sample`` and ``sample_logits``.

Where ``softmax_readout`` answers with the mean row of ``E`` under ``softmax(logit_scale * h W^T +
bias)``, ``softmax_sample`` answers with one token of that distribution, after temperature, top-k,
top-p and min-p; ``embedding_lookup`` feeds it back.  ``sample_logits`` does the same from scores
that the caller has.  No counterpart in the reference library.

The uniform numbers are inputs, and the weights are summed in 64-bit fixed point, so the token is a
function of its inputs alone: no generator state, no dependence on a summation order.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import _native as nat
from .api import _compute_dtype
from .embedding import _pitch, _eager, _unit_rows
from .ops import _ld, _prepare_k, _require_cuda, _workspace

_INT_BITS = {torch.int64: 64, torch.int32: 32}


def _sampling(N, dev, u, T, top_k, top_p, min_p, Ts, ks, ps, ms, want_logprobs):
    """The C struct of one call and the tensors it points to."""
    s = nat.Sampling()
    s.temperature, s.top_k, s.top_p, s.min_p = T, top_k, top_p, min_p
    keep = [u.contiguous()]
    for t, name in ((Ts, "temperatures"), (ps, "top_ps"), (ms, "min_ps")):
        if t is not None:
            keep.append(t.contiguous())
            setattr(s, name, keep[-1].data_ptr())
            setattr(s, name + "_dtype", nat.dtype_code(t.dtype))
    if ks is not None:
        keep.append(ks.contiguous())
        s.top_ks, s.top_ks_bits = keep[-1].data_ptr(), _INT_BITS[ks.dtype]
    s.u, s.u_dtype = keep[0].data_ptr(), nat.dtype_code(u.dtype)
    tokens = torch.empty(N, dtype=torch.int64, device=dev)
    logprobs = torch.empty(N if want_logprobs else 0, dtype=torch.float32, device=dev)
    s.tokens = tokens.data_ptr()
    s.logprobs = logprobs.data_ptr() if want_logprobs else None
    return s, keep, tokens, logprobs


def _sample_logits(logits, u, T, top_k, top_p, min_p, Ts, ks, ps, ms, want_logprobs):
    dev = _require_cuda(logits, u, Ts, ks, ps, ms)
    logits = _unit_rows(logits)
    N, V = logits.shape
    s, keep, tokens, logprobs = _sampling(N, dev, u, T, top_k, top_p, min_p, Ts, ks, ps, ms, want_logprobs)
    with nat.on_device(dev):
        nat.check(nat.lib().swvr_sample_logits(N, V, logits.data_ptr(), nat.dtype_code(logits.dtype), _pitch(logits), s,
                                               nat.stream_ptr(dev)), "swvr_sample_logits")
    return tokens, logprobs


def _sample_head(h, W, bias, u, logit_scale, cdt, T, top_k, top_p, min_p, Ts, ks, ps, ms, want_logprobs):
    dev = _require_cuda(h, W, bias, u, Ts, ks, ps, ms)
    hc, Wc = _prepare_k(h, cdt), _prepare_k(W, cdt)
    b = bias.contiguous() if bias is not None else None
    p = nat.Problem()
    p.n_tokens, p.hidden = hc.shape
    p.vocab = Wc.shape[0]
    p.compute_dtype = nat.dtype_code(cdt)
    p.bias_dtype = nat.dtype_code(b.dtype) if b is not None else 0
    p.h, p.ldh, p.W, p.ldw, p.bias = hc.data_ptr(), _ld(hc), Wc.data_ptr(), _ld(Wc), nat.ptr(b)
    p.logit_scale = logit_scale
    s, keep, tokens, logprobs = _sampling(hc.shape[0], dev, u, T, top_k, top_p, min_p, Ts, ks, ps, ms, want_logprobs)
    lib = nat.lib()
    nbytes = nat.c_size_t(0)
    with nat.on_device(dev):
        nat.check(lib.swvr_sample_workspace_size(p, nat.ctypes.byref(nbytes)), "swvr_sample_workspace_size")
        ws = _workspace(nbytes.value, dev)
        nat.check(lib.swvr_sample(p, s, ws.data_ptr(), ws.numel(), nat.stream_ptr(dev)), "swvr_sample")
    return tokens, logprobs


# Opaque custom ops, like the readout's own (ops.py); sampling has no gradient.

@torch.library.custom_op("swvr_b200::sample_logits", mutates_args=())
def _sample_logits_op(logits: torch.Tensor, u: torch.Tensor, T: float, top_k: int, top_p: float, min_p: float,
                      Ts: Optional[torch.Tensor], ks: Optional[torch.Tensor], ps: Optional[torch.Tensor],
                      ms: Optional[torch.Tensor], want_logprobs: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    return _sample_logits(logits, u, T, top_k, top_p, min_p, Ts, ks, ps, ms, want_logprobs)


@_sample_logits_op.register_fake
def _(logits, u, T, top_k, top_p, min_p, Ts, ks, ps, ms, want_logprobs):
    N = logits.shape[0]
    return logits.new_empty(N, dtype=torch.int64), logits.new_empty(N if want_logprobs else 0, dtype=torch.float32)


@torch.library.custom_op("swvr_b200::sample", mutates_args=())
def _sample_op(h: torch.Tensor, W: torch.Tensor, bias: Optional[torch.Tensor], u: torch.Tensor, logit_scale: float,
               cdt: torch.dtype, T: float, top_k: int, top_p: float, min_p: float, Ts: Optional[torch.Tensor],
               ks: Optional[torch.Tensor], ps: Optional[torch.Tensor], ms: Optional[torch.Tensor],
               want_logprobs: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    return _sample_head(h, W, bias, u, logit_scale, cdt, T, top_k, top_p, min_p, Ts, ks, ps, ms, want_logprobs)


@_sample_op.register_fake
def _(h, W, bias, u, logit_scale, cdt, T, top_k, top_p, min_p, Ts, ks, ps, ms, want_logprobs):
    N = h.shape[0]
    return h.new_empty(N, dtype=torch.int64), h.new_empty(N if want_logprobs else 0, dtype=torch.float32)


def _number(name, x, low, high, lead, open_low=False):
    """(value for all rows, per-row tensor or None) of one setting."""
    if isinstance(x, torch.Tensor):
        if x.shape != lead:
            raise ValueError(f"{name} must be a number or have shape {tuple(lead)}, got {tuple(x.shape)}")
        nat.dtype_code(x.dtype)
        return high if math.isfinite(high) else 1.0, x.reshape(-1)
    x = float(x)
    if not (math.isfinite(x) and (low < x if open_low else low <= x) and x <= high):
        raise ValueError(f"{name} must be in {'(' if open_low else '['}{low:g}, {high:g}], got {x}")
    return x, None


def _settings(lead, u, temperature, top_k, top_p, min_p):
    if u.shape != lead:
        raise ValueError(f"u must have shape {tuple(lead)}, got {tuple(u.shape)}")
    nat.dtype_code(u.dtype)
    T, Ts = _number("temperature", temperature, 0.0, math.inf, lead)
    p, ps = _number("top_p", 1.0 if top_p is None else top_p, 0.0, 1.0, lead, open_low=True)
    m, ms = _number("min_p", 0.0 if min_p is None else min_p, 0.0, 1.0, lead)
    k, ks = 0, None
    if isinstance(top_k, torch.Tensor):
        if top_k.shape != lead:
            raise ValueError(f"top_k must be a number or have shape {tuple(lead)}, got {tuple(top_k.shape)}")
        if top_k.dtype not in _INT_BITS:
            raise ValueError(f"top_k must be int64 or int32, got {top_k.dtype}")
        ks = top_k.reshape(-1)
    elif top_k is not None:
        k = int(top_k)
        if not 1 <= k < 2 ** 63:
            raise ValueError(f"top_k must be at least 1, got {top_k}")
    return (T, k, p, m, Ts, ks, ps, ms)


def _rows(x, lead):
    return x if x.dim() == 2 else x.reshape(math.prod(lead), x.shape[-1])


def _shaped(out, lead, want_logprobs):
    if len(lead) == 1:
        return out if want_logprobs else out[0]
    return (out[0].view(lead), out[1].view(lead)) if want_logprobs else out[0].view(lead)


def sample_logits(logits, u, *, temperature=1.0, top_k=None, top_p=None, min_p=None, return_logprobs=False):
    """One token of each row of ``logits`` ``[..., V]`` (bf16, fp16 or fp32) from the uniform numbers ``u``
    ``[...]`` in ``[0, 1)``; int64 ``[...]``.

    With ``w = exp((x - max x) / temperature)`` and the tokens in falling order of ``x`` (equal ones by
    rising index), ``top_k`` keeps the first k, ``top_p`` a token while the weight ahead of it is below
    ``top_p`` times what ``top_k`` left, ``min_p`` the tokens with ``w >= min_p``; the token is the first in
    index order whose running weight over the kept ones exceeds ``u`` times their sum.  A
    temperature of 0 takes the largest score, the lowest index among equals.  Each setting is a number for
    all rows or a tensor of u's shape; in a tensor a temperature <= 0 or NaN means the largest score, and values
    outside the other settings' ranges turn them off, except that top_p <= 0 keeps one token and min_p > 1 counts as 1.
    Scores of -inf and NaN are never chosen; a row with nothing else gives -1.  Rows may be strided.

    ``return_logprobs=True`` also returns ``log softmax(x / temperature)`` of each token over its whole row,
    in fp32.  There is no gradient.
    """
    if logits.dim() < 1:
        raise ValueError("logits must have a vocabulary dimension")
    if logits.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise ValueError(f"logits must be bf16, fp16 or fp32, got {logits.dtype}")
    lead = logits.shape[:-1]
    args = _settings(lead, u, temperature, top_k, top_p, min_p)
    x, uu = _rows(logits, lead), u if u.dim() == 1 else u.reshape(-1)
    if _eager(x, uu, *args[4:]):
        with torch.no_grad():
            out = _sample_logits(x, uu, *args, bool(return_logprobs))
    else:
        out = _sample_logits_op(x.detach(), uu.detach(), *args, bool(return_logprobs))
    return _shaped(out, lead, return_logprobs)


def softmax_sample(h, W, u, bias=None, *, temperature=1.0, top_k=None, top_p=None, min_p=None, logit_scale=1.0,
                   return_logprobs=False):
    """One token of ``softmax((logit_scale * h @ W.T + bias) / temperature)`` for each row of ``h`` ``[..., K]``:
    ``sample_logits`` of the head's fp32 scores, with the same settings, from ``u`` ``[...]``.

    The products run in the readout's compute dtype (bf16, fp16 or fp32; the autocast dtype under
    autocast) with fp32 accumulation; the scores are never rounded.  At most 256 MiB of them are
    held at a time.  h and W are taken in that dtype: under autocast over parameters of another one, or
    with a hidden size that is no multiple of 8 in 16 bits, all of W is copied at every call, so a server keeps W as it is
    used.  W is the whole vocabulary, not a shard of it.
    """
    if W.dim() != 2:
        raise ValueError(f"W must be 2-D, got {tuple(W.shape)}")
    if h.shape[-1] != W.shape[1]:
        raise ValueError(f"h has hidden size {h.shape[-1]} but W is {tuple(W.shape)}")
    if bias is not None and bias.shape != (W.shape[0],):
        raise ValueError(f"bias must have shape ({W.shape[0]},), got {tuple(bias.shape)}")
    cdt = _compute_dtype(h, W)
    if cdt not in (torch.bfloat16, torch.float16, torch.float32):
        raise ValueError(f"softmax_sample computes in bf16, fp16 or fp32, got {cdt}")
    lead = h.shape[:-1]
    args = _settings(lead, u, temperature, top_k, top_p, min_p)
    h2, uu = _rows(h, lead), u if u.dim() == 1 else u.reshape(-1)
    if _eager(h2, W, bias, uu, *args[4:]):
        with torch.no_grad():
            out = _sample_head(h2, W, bias, uu, float(logit_scale), cdt, *args, bool(return_logprobs))
    else:
        d = lambda t: None if t is None else t.detach()  # noqa: E731
        with torch.autocast(h.device.type, enabled=False):
            out = _sample_op(d(h2), d(W), d(bias), d(uu), float(logit_scale), cdt, *args, bool(return_logprobs))
    return _shaped(out, lead, return_logprobs)
