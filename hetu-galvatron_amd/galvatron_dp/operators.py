"""Operators at a model's two ends, on the GPU (the C ABI in include/galvatron_ops_hip.h).

What a strategy search prices per vocabulary-parallel degree and no layer covers -- embedding lookup, the
residual join and norm behind a block, log probabilities behind the head, and their gradients -- as functions on
torch tensors:

    embedding, embedding_grad                           a table or a shard of it
    token_logprobs, token_logprobs_grad                 given tokens, entropy, most likely tokens
    logprob_parts, join_logprobs                        ... of a vocabulary in shards
    residual_norm, residual_norm_grad                   norms after a block and before the next, gate, scales

``embedding``, ``token_logprobs`` and ``residual_norm`` are differentiable (once, backwards: tensors with forward-mode
tangents are refused); the ``*_grad`` functions are what their backward passes call, for programs that run their own.
Work is queued on torch's current stream of the tensors' device; nothing waits.  Types: float32, float16, bfloat16; token
numbers int32 or int64.  Per-token tensors may have any strides (one whose rows' elements are not neighbours is copied
first); a table's rows have to lie as they are.  There is no CPU path: tensors have to be on a HIP device.
"""
from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import _lib

__all__ = ["embedding", "embedding_grad", "TokenLogprobs", "token_logprobs", "token_logprobs_grad", "LogprobParts",
           "logprob_parts", "join_logprobs", "Norm", "ResidualNorm", "ResidualNormGrads", "residual_norm",
           "residual_norm_grad", "MAX_TOP", "MAX_NORM_DIM"]

MAX_TOP = 64            # GDP_MAX_TOP
MAX_NORM_DIM = 16384    # GDP_MAX_NORM_DIM
EXPORTED_SYMBOLS = _lib.OPERATOR_SYMBOLS

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_TOKEN_TYPES = {torch.int32: 0, torch.int64: 1}
_FORMS = {None: 0, "rms": 1, "layer": 2}

_p, _i32, _i64, _f32, _size = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float, ctypes.c_size_t


class gdp_embed(ctypes.Structure):
    _fields_ = [("n", _i64), ("rows", _i64), ("dim", _i64), ("first", _i64), ("tokens", _p), ("token_type", _i32),
                ("weight_type", _i32), ("out_type", _i32), ("scale", _f32), ("weight", _p), ("weight_stride", _i64),
                ("out", _p), ("out_stride", _i64)]


class gdp_embed_grad(ctypes.Structure):
    _fields_ = [("n", _i64), ("rows", _i64), ("dim", _i64), ("first", _i64), ("tokens", _p), ("token_type", _i32),
                ("grad_type", _i32), ("out_type", _i32), ("accumulate", _i32), ("scale", _f32), ("grad", _p),
                ("grad_stride", _i64), ("out", _p), ("out_stride", _i64), ("workspace", _p), ("workspace_bytes", _size)]


class gdp_logprob(ctypes.Structure):
    _fields_ = [("n", _i64), ("vocab", _i64), ("logits", _p), ("logits_stride", _i64), ("logits_type", _i32),
                ("token_type", _i32), ("tokens", _p), ("scale", _f32), ("top", _i32), ("logp", _p), ("lse", _p),
                ("entropy", _p), ("top_logp", _p), ("top_tokens", _p), ("workspace", _p), ("workspace_bytes", _size)]


class gdp_logprob_part(ctypes.Structure):
    _fields_ = [("n", _i64), ("vocab", _i64), ("first", _i64), ("logits", _p), ("logits_stride", _i64),
                ("logits_type", _i32), ("token_type", _i32), ("tokens", _p), ("scale", _f32), ("top", _i32),
                ("stats", _p), ("top_logits", _p), ("top_tokens", _p), ("workspace", _p), ("workspace_bytes", _size)]


class gdp_logprob_joint(ctypes.Structure):
    _fields_ = [("n", _i64), ("vocab", _i64), ("parts", _i32), ("top", _i32), ("scale", _f32), ("token_type", _i32),
                ("tokens", _p), ("stats", _p), ("top_logits", _p), ("top_tokens", _p), ("logp", _p), ("lse", _p),
                ("entropy", _p), ("top_logp", _p), ("out_tokens", _p)]


class gdp_logprob_grad(ctypes.Structure):
    _fields_ = [("n", _i64), ("vocab", _i64), ("first", _i64), ("whole_vocab", _i64), ("logits", _p),
                ("logits_stride", _i64), ("logits_type", _i32), ("token_type", _i32), ("tokens", _p), ("scale", _f32),
                ("top", _i32), ("lse", _p), ("grad_logp", _p), ("grad_lse", _p), ("entropy", _p), ("grad_entropy", _p),
                ("top_tokens", _p), ("grad_top", _p), ("out", _p), ("out_stride", _i64)]


class gdp_logprob_stats(ctypes.Structure):
    _fields_ = [("given", gdp_logprob), ("row_stats", _p)]


class gdp_logprob_joint_stats(ctypes.Structure):
    _fields_ = [("given", gdp_logprob_joint), ("row_stats", _p)]


class gdp_logprob_grad_stats(ctypes.Structure):
    _fields_ = [("given", gdp_logprob_grad), ("row_stats", _p)]


class gdp_norm_params(ctypes.Structure):
    _fields_ = [("form", _i32), ("type", _i32), ("eps", _f32), ("reserved", _i32), ("weight", _p), ("bias", _p)]


class gdp_norm(ctypes.Structure):
    _fields_ = [("n", _i64), ("dim", _i64), ("type", _i32), ("stream_type", _i32), ("residual", _p),
                ("residual_stride", _i64), ("block", _p), ("block_stride", _i64), ("post", gdp_norm_params),
                ("pre", gdp_norm_params), ("gate", _p), ("gates", _i64), ("gate_stride", _i64), ("gate_type", _i32),
                ("residual_scale", _f32), ("block_scale", _f32), ("reserved", _i32), ("stream", _p),
                ("stream_stride", _i64), ("normed", _p), ("normed_stride", _i64), ("stats", _p)]


class gdp_norm_grad(ctypes.Structure):
    _fields_ = [("n", _i64), ("dim", _i64), ("type", _i32), ("stream_type", _i32), ("stream", _p),
                ("stream_stride", _i64), ("block", _p), ("block_stride", _i64), ("stats", _p), ("grad_normed", _p),
                ("grad_normed_stride", _i64), ("grad_stream", _p), ("grad_stream_stride", _i64),
                ("post", gdp_norm_params), ("pre", gdp_norm_params), ("gate", _p), ("gates", _i64),
                ("gate_stride", _i64), ("gate_type", _i32), ("residual_scale", _f32), ("block_scale", _f32),
                ("reserved", _i32), ("grad_residual", _p), ("grad_residual_stride", _i64), ("grad_block", _p),
                ("grad_block_stride", _i64), ("grad_pre_weight", _p), ("grad_pre_bias", _p), ("grad_post_weight", _p),
                ("grad_post_bias", _p), ("grad_gate", _p), ("workspace", _p), ("workspace_bytes", _size)]


_bound = None


def _ops() -> ctypes.CDLL:
    """The library with the operators' signatures.  It has to share torch's HIP runtime: pointers and streams of one
    runtime mean nothing to another, and a process that loaded the library before torch has two."""
    global _bound
    if _bound is None:
        L = _lib.lib()
        with open("/proc/self/maps") as fh:
            runtimes = {line.split()[-1] for line in fh if "libamdhip64" in line}
        if len(runtimes) > 1:
            raise RuntimeError("two HIP runtimes are loaded (" + ", ".join(sorted(runtimes)) +
                               "): import torch, or galvatron_dp.operators, before the first DP call of the process")
        for name, record in (("gdp_embed_forward", gdp_embed), ("gdp_embed_backward", gdp_embed_grad),
                             ("gdp_logprob_forward", gdp_logprob), ("gdp_logprob_parts", gdp_logprob_part),
                             ("gdp_logprob_join", gdp_logprob_joint), ("gdp_logprob_backward", gdp_logprob_grad),
                             ("gdp_logprob_forward_stats", gdp_logprob_stats),
                             ("gdp_logprob_join_stats", gdp_logprob_joint_stats),
                             ("gdp_logprob_backward_stats", gdp_logprob_grad_stats),
                             ("gdp_norm_forward", gdp_norm), ("gdp_norm_backward", gdp_norm_grad)):
            f = getattr(L, name)
            f.argtypes, f.restype = [ctypes.POINTER(record), ctypes.c_void_p], ctypes.c_int
        size = ctypes.POINTER(_size)
        L.gdp_embed_grad_workspace.argtypes = [_i64, _i64, _i64, size]
        L.gdp_logprob_workspace.argtypes = [_i64, _i64, _i32, _i32, size]
        L.gdp_norm_grad_workspace.argtypes = [_i64, _i64, _i64, size]
        for name in ("gdp_embed_grad_workspace", "gdp_logprob_workspace", "gdp_norm_grad_workspace"):
            getattr(L, name).restype = ctypes.c_int
        _bound = L
    return _bound


_stream_of = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else None


def _queue(f, record, device) -> None:
    """Calls f(record, stream) on torch's current stream of the device."""
    index = device.index
    if index == torch.cuda.current_device():
        # (as an integer: building torch's stream object takes longer than the rest of a small call)
        rc = f(record, _stream_of(index) if _stream_of else torch.cuda.current_stream().cuda_stream)
    else:
        with torch.cuda.device(device):
            rc = f(record, torch.cuda.current_stream().cuda_stream)
    if rc:
        _lib._check(rc)


@functools.lru_cache(maxsize=1024)
def _bytes(name, *sizes):
    """What a gdp_*_workspace function says, which goes by the sizes alone."""
    need = _size()
    rc = getattr(_ops(), name)(*sizes, ctypes.byref(need))
    if rc:
        _lib._check(rc)
    return need.value


def _workspace(name, *sizes, device):
    need = _bytes(name, *sizes)
    return (torch.empty(need, dtype=torch.uint8, device=device) if need else None), need


def _no_tangents(*tensors):
    """Refuses what the kernels would drop: a result without a tangent, from an input with one.  (Asked where a level is open; else there
    are none.)"""
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError("the operators have no forward-mode derivatives")


def _of_norms(*norms):
    """The weights and biases of norms that may be None."""
    return [t for norm in norms for t in ((norm.weight, norm.bias) if norm else (None, None))]


def _written(t):
    """Tells autograd that a tensor of the caller has been written, as torch's own functions do: a graph that holds it says so, rather than
    going on with other values."""
    torch.autograd.graph.increment_version(t)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _type(t, what, dtypes=_TYPES):
    """The number of a tensor's element type, after checking what is said of all tensors."""
    code = dtypes.get(t.dtype)
    if code is None:
        raise ValueError(f"{what}: type {t.dtype} is none of " + ", ".join(str(d)[6:] for d in dtypes))
    if not t.is_cuda:
        raise ValueError(f"{what} has to be on a HIP device, not on {t.device}")
    return code


def _same_device(device, **tensors):
    for what, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{what} is on {t.device}, not on {device}")


def _like(t):
    """New memory of a tensor's shape and type, its rows in order."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _rows(t, dim, what):
    """[..., dim] as rows whose elements are neighbours, and the stride between them."""
    if t.dim() < 1 or t.shape[-1] != dim:
        raise ValueError(f"{what} must be [..., {dim}], not {list(t.shape)}")
    if t.is_contiguous():
        return t, dim
    if t.dim() != 2:
        t = t.reshape(-1, dim)
    if t.stride(1) != 1 and dim > 1:
        t = t.contiguous()
    return t, t.stride(0)


def _floats(t, shape, what, device):
    """float32 of that shape in order, or None."""
    if t is None:
        return None
    if t.shape != shape:
        raise ValueError(f"{what} must be {list(shape)}, not {list(t.shape)}")
    if t.device != device:
        raise ValueError(f"{what} is on {t.device}, not on {device}")
    return t.to(torch.float32).contiguous()


def _table(t, what):
    if t.dim() != 2:
        raise ValueError(f"{what} must be [rows, columns], not {list(t.shape)}")
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"{what}: the elements of a row have to be neighbours (strides {list(t.stride())})")
    return t


# ---- embedding ---------------------------------------------------------------------------------------------
def _embedding(tokens, weight, scale, first, dtype):
    token_type, weight_type = _type(tokens, "tokens", _TOKEN_TYPES), _type(weight, "weight")
    _table(weight, "weight")
    _same_device(weight.device, tokens=tokens)
    out_type = weight_type if dtype is None else _TYPES.get(dtype)
    if out_type is None:
        raise ValueError(f"dtype: {dtype} is none of float32, float16, bfloat16")
    flat = tokens if tokens.is_contiguous() else tokens.contiguous()
    rows, dim = weight.shape
    out = torch.empty(tokens.shape + (dim,), dtype=dtype or weight.dtype, device=weight.device)
    _queue(_ops().gdp_embed_forward,
           gdp_embed(flat.numel(), rows, dim, first, flat.data_ptr(), token_type, weight_type, out_type, scale,
                     weight.data_ptr(), weight.stride(0), out.data_ptr(), dim), weight.device)
    return out


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, weight, scale, first, dtype):
        ctx.save_for_backward(tokens)
        ctx.given = (weight.shape[0], scale, first, weight.dtype)
        return _embedding(tokens, weight, scale, first, dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        rows, scale, first, dtype = ctx.given
        return None, embedding_grad(ctx.saved_tensors[0], grad, rows, scale=scale, first=first, dtype=dtype), None, None, None


def embedding(tokens, weight, *, scale: float = 1.0, first: int = 0, dtype: Optional[torch.dtype] = None):
    """``scale * weight[tokens - first]`` [*tokens.shape, dim], in ``dtype`` (that of the weight by default).

    ``weight`` [rows, dim] is the shard of a table whose row 0 belongs to token ``first``; a token that it does not hold
    gives zeros, so that the sum over the shards is the lookup in the whole table."""
    if forward_ad._current_level >= 0:
        _no_tangents(weight)
    if weight.requires_grad and torch.is_grad_enabled():
        return _Embedding.apply(tokens, weight, float(scale), int(first), dtype)
    return _embedding(tokens, weight, float(scale), int(first), dtype)


def embedding_grad(tokens, grad, rows: int, *, scale: float = 1.0, first: int = 0, dtype: Optional[torch.dtype] = None,
                   into: Optional[torch.Tensor] = None):
    """Gradient of ``embedding``'s weight [rows, dim] from that of its output [*tokens.shape, dim]: the sums over the
    places that hold the same token, in ``dtype`` (the gradient's by default), zeros for rows without any.

    ``into`` [rows, dim]: the sums are added to it instead, rows without places are left alone, and it is returned."""
    if forward_ad._current_level >= 0:
        _no_tangents(grad, into)
    token_type, grad_type = _type(tokens, "tokens", _TOKEN_TYPES), _type(grad, "grad")
    device = grad.device
    if grad.shape[:-1] != tokens.shape or grad.dim() != tokens.dim() + 1:
        raise ValueError(f"grad must be [*tokens.shape, dim], not {list(grad.shape)} for tokens {list(tokens.shape)}")
    if rows < 0:
        raise ValueError(f"rows: {rows}")
    dim = grad.shape[-1]
    flat = tokens if tokens.is_contiguous() else tokens.contiguous()
    n = flat.numel()
    grad, stride = _rows(grad, dim, "grad") if n and dim else (grad, dim)
    if into is None:
        if dtype is not None and dtype not in _TYPES:
            raise ValueError(f"dtype: {dtype} is none of float32, float16, bfloat16")
        out = torch.empty(rows, dim, dtype=dtype or grad.dtype, device=device)
    else:
        out = _table(into, "into")
        if out.shape != (rows, dim):
            raise ValueError(f"into must be {[rows, dim]}, not {list(out.shape)}")
        if dtype is not None and dtype != out.dtype:
            raise ValueError("dtype is that of into")
    out_type = _type(out, "into")
    _same_device(device, tokens=tokens, into=out)
    L = _ops()
    work, size = _workspace("gdp_embed_grad_workspace", n, rows, dim, device=device)
    _queue(L.gdp_embed_backward,
           gdp_embed_grad(n, rows, dim, first, flat.data_ptr(), token_type, grad_type, out_type, into is not None, scale,
                          grad.data_ptr(), stride, out.data_ptr(), out.stride(0) if rows else dim, _ptr(work), size), device)
    if into is not None and n:
        _written(into)
    return out


# ---- log probabilities -------------------------------------------------------------------------------------
class TokenLogprobs(NamedTuple):
    logp: torch.Tensor                          # [...]       of the given tokens, 0 where there is none
    lse: torch.Tensor                           # [...]       log of the sum of exponentials of scale * logits
    entropy: Optional[torch.Tensor] = None      # [...]
    top_logp: Optional[torch.Tensor] = None     # [..., top]  largest first
    top_tokens: Optional[torch.Tensor] = None   # [..., top]  int64


class LogprobParts(NamedTuple):
    """What a shard of the vocabulary knows of its rows, to be exchanged and joined."""
    stats: torch.Tensor                         # [n, 4]      float32
    top_logits: torch.Tensor                    # [n, top]    float32
    top_tokens: torch.Tensor                    # [n, top]    int32


def _tokens_for(tokens, shape, device):
    token_type = _type(tokens, "tokens", _TOKEN_TYPES)
    if tokens.shape != shape:
        raise ValueError(f"tokens must be {list(shape)}, not {list(tokens.shape)}")
    _same_device(device, tokens=tokens)
    return tokens if tokens.is_contiguous() else tokens.contiguous(), token_type


def _check_top(top):
    if not 0 <= top <= MAX_TOP:
        raise ValueError(f"top must be 0 to {MAX_TOP}, not {top}")


def _outputs(shape, top, device):
    n = shape.numel()
    if n and shape:
        # One allocation, but no views of it: parts of one tensor could not be changed in place, and would share their version.
        logp, lse, entropy = torch.empty((3 * shape[0],) + shape[1:], dtype=torch.float32, device=device).unsafe_chunk(3)
    else:
        logp, lse, entropy = [torch.empty(shape, dtype=torch.float32, device=device) for _ in range(3)]
    if not top:
        return n, logp, lse, entropy, None, None
    return (n, logp, lse, entropy, torch.empty(shape + (top,), dtype=torch.float32, device=device),
            torch.empty(shape + (top,), dtype=torch.int64, device=device))


def _check_row_stats(t, shape, device):
    if t.shape != shape + (2,) or t.dtype != torch.float32 or t.device != device or not t.is_contiguous():
        raise ValueError(f"row_stats must be {list(shape + (2,))} float32 on {device}, in order")


def _token_logprobs(logits, tokens, scale, top, row_stats):
    logits_type = _type(logits, "logits")
    if logits.dim() < 1:
        raise ValueError("logits must be [..., vocab]")
    _check_top(top)
    device, vocab, shape = logits.device, logits.shape[-1], logits.shape[:-1]
    flat, token_type = _tokens_for(tokens, shape, device)
    n, logp, lse, entropy, top_logp, top_tokens = _outputs(shape, top, device)
    rows, stride = _rows(logits, vocab, "logits") if n and vocab else (logits, vocab)
    L = _ops()
    work, size = _workspace("gdp_logprob_workspace", n, vocab, logits_type, top, device=device)
    given = gdp_logprob(n, vocab, rows.data_ptr(), stride, logits_type, token_type, flat.data_ptr(), scale, top,
                        logp.data_ptr(), lse.data_ptr(), entropy.data_ptr(), _ptr(top_logp), _ptr(top_tokens), _ptr(work), size)
    if row_stats is not None and n:
        _queue(L.gdp_logprob_forward_stats, gdp_logprob_stats(given, row_stats.data_ptr()), device)
    else:
        _queue(L.gdp_logprob_forward, given, device)
    return logp, lse, entropy, top_logp, top_tokens


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, scale, top, row_stats):
        if row_stats is None:
            row_stats = torch.empty(logits.shape[:-1] + (2,), dtype=torch.float32, device=logits.device)
        logp, lse, entropy, top_logp, top_tokens = _token_logprobs(logits, tokens, scale, top, row_stats)
        ctx.save_for_backward(logits, tokens, row_stats, entropy, top_tokens)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        if top_tokens is not None:
            ctx.mark_non_differentiable(top_tokens)
        return logp, lse, entropy, top_logp, top_tokens

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_logp, d_lse, d_entropy, d_top, _):
        logits, tokens, row_stats, entropy, top_tokens = ctx.saved_tensors
        return token_logprobs_grad(logits, tokens, None, d_logp, scale=ctx.scale, grad_lse=d_lse,
                                   entropy=None if d_entropy is None else entropy, grad_entropy=d_entropy,
                                   top_tokens=None if d_top is None else top_tokens, grad_top=d_top,
                                   row_stats=row_stats), None, None, None, None


def token_logprobs(logits, tokens, *, scale: float = 1.0, entropy: bool = False, top: int = 0,
                   row_stats: Optional[torch.Tensor] = None) -> TokenLogprobs:
    """Log probabilities of ``tokens`` [...] under softmax(scale * logits) over the last dimension of ``logits`` [..., vocab],
    the log of the sum of exponentials, with ``entropy`` each row's entropy, and the ``top`` (at most 64) most likely
    tokens: equal logits by number, the lowest first.  All in float32, from one pass over the logits.

    A token outside [0, vocab), such as -100, is none: its log probability is 0, and it gives no gradient.  Logits of
    -inf are tokens that are ruled out; a row of nothing else has lse and log probabilities of -inf, entropy 0, and a
    gradient of zeros.  NaN or +inf make their row's results NaN.  Any other row, one of a mask's -1e9 alone among them, has
    the log probabilities, entropy and gradient of its logits less the largest.

    ``row_stats`` [..., 2] float32: written, the largest logit and the log of the sum relative to it, for
    ``token_logprobs_grad``."""
    if forward_ad._current_level >= 0:
        _no_tangents(logits)
    if row_stats is not None:
        _check_row_stats(row_stats, logits.shape[:-1], logits.device)
        _written(row_stats)
    if torch.is_grad_enabled() and logits.requires_grad:
        r = _TokenLogprobs.apply(logits, tokens, float(scale), int(top), row_stats)
    else:
        r = _token_logprobs(logits, tokens, float(scale), int(top), row_stats)
    return TokenLogprobs(r[0], r[1], r[2] if entropy else None, r[3], r[4])


def token_logprobs_grad(logits, tokens, lse, grad_logp=None, *, scale: float = 1.0, grad_lse=None, entropy=None,
                        grad_entropy=None, top_tokens=None, grad_top=None, first: int = 0,
                        vocab: Optional[int] = None, into: Optional[torch.Tensor] = None,
                        row_stats: Optional[torch.Tensor] = None):
    """Gradient with respect to ``logits`` [..., columns], in their type, from those of ``token_logprobs``' results.

    ``row_stats``: what the forward pass wrote there; ``lse`` is not read then and may be None.  From ``lse`` alone, which float32
    rounds by one part in 2^24, probabilities are off by |lse| / 2^24 of themselves, and rows whose lse is below -2^24 (nothing but
    a mask's -1e9) have zeros.  ``lse`` (and ``entropy``, ``top_tokens`` where they have gradients) are what the forward pass
    gave.  Of a vocabulary in shards, ``logits`` are those of the shard that begins with token ``first``, of ``vocab`` tokens in
    all, and ``row_stats``, ``lse``, ``entropy`` and ``top_tokens`` those of ``join_logprobs``.  ``into``: written there; it may be
    ``logits`` itself."""
    if forward_ad._current_level >= 0:
        _no_tangents(logits, lse, grad_logp, grad_lse, entropy, grad_entropy, grad_top, into, row_stats)
    logits_type = _type(logits, "logits")
    if logits.dim() < 1:
        raise ValueError("logits must be [..., vocab]")
    device, columns, shape = logits.device, logits.shape[-1], logits.shape[:-1]
    if vocab is None:
        vocab = first + columns
    flat, token_type = _tokens_for(tokens, shape, device)
    if (entropy is None) != (grad_entropy is None) or (top_tokens is None) != (grad_top is None):
        raise ValueError("entropy and grad_entropy, top_tokens and grad_top come together")
    if row_stats is not None:
        _check_row_stats(row_stats, shape, device)
        lse = None
    elif lse is None:
        raise ValueError("row_stats or lse is needed")
    lse = _floats(lse, shape, "lse", device)
    grad_logp, grad_lse = _floats(grad_logp, shape, "grad_logp", device), _floats(grad_lse, shape, "grad_lse", device)
    entropy, grad_entropy = _floats(entropy, shape, "entropy", device), _floats(grad_entropy, shape, "grad_entropy", device)
    top = 0
    if grad_top is not None:
        top = top_tokens.shape[-1]
        if top_tokens.shape != shape + (top,) or top_tokens.dtype != torch.int64:
            raise ValueError("top_tokens must be [..., top], int64")
        _same_device(device, top_tokens=top_tokens)
        grad_top, top_tokens = _floats(grad_top, shape + (top,), "grad_top", device), top_tokens.contiguous()
    n = shape.numel()
    if into is None:
        out = _like(logits)
    else:
        out = into
        if out.shape != logits.shape or out.dtype != logits.dtype or out.device != device:
            raise ValueError("into must have the shape, type and device of logits")
    if not n or not columns:
        return out
    rows, stride = _rows(logits, columns, "logits")
    try:
        to = out if out.dim() == 2 else out.view(-1, columns)
        if columns > 1 and to.stride(1) != 1:
            raise RuntimeError
    except RuntimeError:
        raise ValueError("into must have rows that are neighbouring elements at one stride") from None
    given = gdp_logprob_grad(n, columns, first, vocab, rows.data_ptr(), stride, logits_type, token_type, flat.data_ptr(), scale,
                             top, _ptr(lse), _ptr(grad_logp), _ptr(grad_lse), _ptr(entropy), _ptr(grad_entropy),
                             _ptr(top_tokens), _ptr(grad_top), to.data_ptr(), to.stride(0))
    if row_stats is not None:
        _queue(_ops().gdp_logprob_backward_stats, gdp_logprob_grad_stats(given, row_stats.data_ptr()), device)
    else:
        _queue(_ops().gdp_logprob_backward, given, device)
    if into is not None:
        _written(into)
    return out


def logprob_parts(logits, tokens, *, first: int, scale: float = 1.0, top: int = 0) -> LogprobParts:
    """``token_logprobs`` of a shard of the vocabulary, ``logits`` [n, columns] of the tokens from ``first`` on, up to what
    the other shards have to say: 16 + 8 * top bytes for each row, to be gathered from all shards and joined."""
    if forward_ad._current_level >= 0:
        _no_tangents(logits)
    logits_type = _type(logits, "logits")
    if logits.dim() != 2:
        raise ValueError(f"logits must be [n, columns], not {list(logits.shape)}")
    _check_top(top)
    device, (n, columns) = logits.device, logits.shape
    flat, token_type = _tokens_for(tokens, logits.shape[:1], device)
    rows, stride = _rows(logits, columns, "logits") if n and columns else (logits, columns)
    parts = LogprobParts(torch.empty(n, 4, dtype=torch.float32, device=device),
                         torch.empty(n, top, dtype=torch.float32, device=device),
                         torch.empty(n, top, dtype=torch.int32, device=device))
    L = _ops()
    work, size = _workspace("gdp_logprob_workspace", n, columns, logits_type, top, device=device)
    _queue(L.gdp_logprob_parts,
           gdp_logprob_part(n, columns, first, rows.data_ptr(), stride, logits_type, token_type, flat.data_ptr(), scale, top,
                            parts.stats.data_ptr(), parts.top_logits.data_ptr(), parts.top_tokens.data_ptr(), _ptr(work),
                            size), device)
    return parts


def join_logprobs(parts, tokens, vocab: int, *, scale: float = 1.0, entropy: bool = False,
                  row_stats: Optional[torch.Tensor] = None) -> TokenLogprobs:
    """``token_logprobs`` of a vocabulary of ``vocab`` tokens from the parts of its shards: ``LogprobParts`` in the order of
    their tokens, or one whose tensors have a leading dimension for the shards, as gathering them leaves it.  ``row_stats``: as
    there, of the whole rows."""
    if not isinstance(parts, LogprobParts):
        parts = list(parts)
        if not parts or any(a.shape != b.shape for p in parts for a, b in zip(p, parts[0])):
            raise ValueError("parts must be one of each shard, of the same rows and alternatives")
        parts = LogprobParts(*(torch.stack(t) for t in zip(*parts)))
    if forward_ad._current_level >= 0:
        _no_tangents(*parts[:2])
    stats, top_logits, top_tokens = (t.contiguous() for t in parts)
    if stats.dim() != 3 or stats.shape[2] != 4 or top_logits.shape[:2] != stats.shape[:2] or top_tokens.shape != top_logits.shape:
        raise ValueError("parts must be stats [parts, n, 4], top_logits and top_tokens [parts, n, top]")
    if stats.dtype != torch.float32 or top_logits.dtype != torch.float32 or top_tokens.dtype != torch.int32:
        raise ValueError("parts must be as logprob_parts gives them: float32, float32, int32")
    _type(stats, "parts")
    device, count, shape, top = stats.device, stats.shape[0], stats.shape[1:2], top_logits.shape[2]
    _same_device(device, top_logits=top_logits, top_tokens=top_tokens)
    flat, token_type = _tokens_for(tokens, shape, device)
    if row_stats is not None:
        _check_row_stats(row_stats, shape, device)
    n, logp, lse, ent, top_logp, out_tokens = _outputs(shape, top, device)
    given = gdp_logprob_joint(n, vocab, count, top, scale, token_type, flat.data_ptr(), stats.data_ptr(), top_logits.data_ptr(),
                              top_tokens.data_ptr(), logp.data_ptr(), lse.data_ptr(), ent.data_ptr(), _ptr(top_logp),
                              _ptr(out_tokens))
    if row_stats is not None and n:
        _queue(_ops().gdp_logprob_join_stats, gdp_logprob_joint_stats(given, row_stats.data_ptr()), device)
        _written(row_stats)
    else:
        _queue(_ops().gdp_logprob_join, given, device)
    return TokenLogprobs(logp, lse, ent if entropy else None, top_logp, out_tokens)


# ---- residual join and norms -------------------------------------------------------------------------------
class Norm(NamedTuple):
    """``form`` "rms" or "layer" (with a mean); weight and bias [dim], or None for ones and zeros."""
    form: str
    weight: Optional[torch.Tensor] = None
    bias: Optional[torch.Tensor] = None
    eps: float = 1e-5


class ResidualNorm(NamedTuple):
    stream: torch.Tensor                # residual_scale * residual + block_scale * gate * post(block)
    normed: Optional[torch.Tensor]      # pre(stream)
    stats: Optional[torch.Tensor]       # [n, 4] float32, where asked for: mean, 1 / deviation of post; of pre


class ResidualNormGrads(NamedTuple):
    residual: torch.Tensor
    block: Optional[torch.Tensor]
    post_weight: Optional[torch.Tensor]
    post_bias: Optional[torch.Tensor]
    pre_weight: Optional[torch.Tensor]
    pre_bias: Optional[torch.Tensor]
    gate: Optional[torch.Tensor]


def _vector(t, dim, device, what):
    """[dim] in order, and its type"""
    code = _type(t, what)
    if t.shape != (dim,):
        raise ValueError(f"{what} must be {[dim]}, not {list(t.shape)}")
    if t.device != device:
        raise ValueError(f"{what} is on {t.device}, not on {device}")
    return (t if t.is_contiguous() else t.contiguous()), code


def _norm_params(norm, dim, device, what):
    """The record of a norm, and what it points to."""
    if norm is None:
        return gdp_norm_params(), None, None
    form, weight, bias, eps = norm
    number = _FORMS.get(form)
    if not number:
        raise ValueError(f"{what}.form must be 'rms' or 'layer', not {form!r}")
    code = 0
    if weight is not None:
        weight, code = _vector(weight, dim, device, f"{what}.weight")
    if bias is not None:
        bias, of_bias = _vector(bias, dim, device, f"{what}.bias")
        if weight is not None and of_bias != code:
            raise ValueError(f"{what}: weight and bias have to be of one type")
        code = of_bias
    return gdp_norm_params(number, code, eps, 0, None if weight is None else weight.data_ptr(), None if bias is None else bias.data_ptr()), weight, bias


def _gate_rows(gate, dim, n, device):
    """(rows of the gate, how many, their stride, their type)"""
    if gate is None:
        return None, 0, 0, 0
    code = _type(gate, "gate")
    if gate.device != device:
        raise ValueError(f"gate is on {gate.device}, not on {device}")
    if n == 0 and dim and gate.numel() == 0 and gate.shape[-1] == dim:
        return None, 0, 0, 0        # no rows, and a gate for each
    rows, stride = _rows(gate, dim, "gate")
    count = gate.numel() // dim if dim else 0
    if count < 1 or n % count:
        raise ValueError(f"gate: {count} gates do not divide {n} rows")
    return rows, count, stride, code


def _residual_norm(residual, block, post, pre, gate, residual_scale, block_scale, with_stats):
    stream_type = _type(residual, "residual")
    if residual.dim() < 1:
        raise ValueError("residual must be [..., dim]")
    device, dim, shape = residual.device, residual.shape[-1], residual.shape
    n = shape[:-1].numel()
    kind = residual.dtype if block is None else block.dtype
    if block is None and pre is not None and pre.weight is not None:
        kind = pre.weight.dtype if residual.dtype == torch.float32 else residual.dtype
    if block is None and (post is not None or gate is not None):
        raise ValueError("post and gate need a block")
    if block is None and pre is None:
        raise ValueError("nothing to do: neither a block nor a norm")
    code = _type(residual if kind == residual.dtype else pre.weight, "pre.weight") if block is None else _type(block, "block")
    if block is not None and (block.shape != shape or block.device != device):
        raise ValueError(f"block must be {list(shape)} on {device}, not {list(block.shape)} on {block.device}")
    post_record, *keep_post = _norm_params(post, dim, device, "post")
    pre_record, *keep_pre = _norm_params(pre, dim, device, "pre")
    gates, count, gate_stride, gate_type = _gate_rows(gate, dim, n, device)
    r, r_stride = _rows(residual, dim, "residual") if n else (residual, dim)
    b, b_stride = (None, 0) if block is None else _rows(block, dim, "block") if n else (block, dim)
    same = block is None and residual_scale == 1.0
    stream = residual if same else _like(residual)
    normed = None if pre is None else torch.empty(shape, dtype=kind, device=device) if block is None else _like(block)
    stats = torch.empty((n, 4), dtype=torch.float32, device=device) if with_stats else None
    _queue(_ops().gdp_norm_forward,
           gdp_norm(n, dim, code, stream_type, r.data_ptr(), r_stride, _ptr(b), b_stride, post_record, pre_record,
                    _ptr(gates), count, gate_stride, gate_type, residual_scale, block_scale, 0,
                    None if same else stream.data_ptr(), dim, _ptr(normed), dim, _ptr(stats)), device)
    return stream, normed, stats


def residual_norm_grad(stream, block, stats, grad_normed, grad_stream=None, *, post: Optional[Norm] = None,
                       pre: Optional[Norm] = None, gate=None, residual_scale: float = 1.0,
                       block_scale: float = 1.0) -> ResidualNormGrads:
    """Gradients of ``residual_norm``'s inputs from ``grad_normed`` and, where the stream is used further on,
    ``grad_stream``.  ``stream``, ``stats`` and ``block`` are those of the forward pass.  Gradients of weights, biases and gate
    have their types and shapes and are None for what is not there."""
    if forward_ad._current_level >= 0:
        _no_tangents(stream, block, stats, grad_normed, grad_stream, *_of_norms(post, pre), gate)
    stream_type = _type(stream, "stream")
    device, dim, shape = stream.device, stream.shape[-1], stream.shape
    n = shape[:-1].numel()
    if (pre is None) != (grad_normed is None):
        raise ValueError("grad_normed comes with pre")
    if grad_normed is None and grad_stream is None:
        raise ValueError("neither grad_normed nor grad_stream")
    if block is None and (post is not None or gate is not None):
        raise ValueError("post and gate need a block")
    kind = block if block is not None else grad_normed if grad_normed is not None else stream
    code = _type(kind, "block" if block is not None else "grad_normed")
    for what, t, dtype in (("block", block, kind.dtype), ("grad_normed", grad_normed, kind.dtype), ("grad_stream", grad_stream, stream.dtype)):
        if t is not None and (t.shape != shape or t.dtype != dtype):
            raise ValueError(f"{what} must be {list(shape)} of {dtype}, not {list(t.shape)} of {t.dtype}")
    _same_device(device, block=block, grad_normed=grad_normed, grad_stream=grad_stream, stats=stats)
    if stats is None or stats.shape != (n, 4) or stats.dtype != torch.float32:
        raise ValueError(f"stats must be {[n, 4]}, float32")
    stats = stats.contiguous()
    post_record, *keep_post = _norm_params(post, dim, device, "post")
    pre_record, *keep_pre = _norm_params(pre, dim, device, "pre")
    gates, count, gate_stride, gate_type = _gate_rows(gate, dim, n, device)

    def rows(t, what):
        return (None, 0) if t is None else _rows(t, dim, what) if n else (t, dim)

    s, s_stride = rows(stream, "stream")
    b, b_stride = rows(block, "block")
    dh, dh_stride = rows(grad_normed, "grad_normed")
    ds, ds_stride = rows(grad_stream, "grad_stream")

    got = ResidualNormGrads(*[None if t is None else _like(t) for t in (
        stream, block, *_of_norms(post, pre), gate)])
    L = _ops()
    work, size = _workspace("gdp_norm_grad_workspace", n, dim, count, device=device)
    _queue(L.gdp_norm_backward,
           gdp_norm_grad(n, dim, code, stream_type, s.data_ptr(), s_stride, _ptr(b), b_stride, stats.data_ptr(), _ptr(dh),
                         dh_stride, _ptr(ds), ds_stride, post_record, pre_record, _ptr(gates), count, gate_stride, gate_type,
                         residual_scale, block_scale, 0, got.residual.data_ptr(), dim, _ptr(got.block), dim,
                         _ptr(got.pre_weight), _ptr(got.pre_bias), _ptr(got.post_weight), _ptr(got.post_bias), _ptr(got.gate),
                         _ptr(work), size), device)
    return got


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, residual, block, post_weight, post_bias, pre_weight, pre_bias, gate, post, pre, residual_scale, block_scale):
        # post and pre: (form, eps) or None
        post_norm = post and Norm(post[0], post_weight, post_bias, post[1])
        pre_norm = pre and Norm(pre[0], pre_weight, pre_bias, pre[1])
        stream, normed, stats = _residual_norm(residual, block, post_norm, pre_norm, gate, residual_scale, block_scale, True)
        ctx.save_for_backward(stream, block, stats, post_weight, post_bias, pre_weight, pre_bias, gate)
        ctx.given = (post, pre, residual_scale, block_scale)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(stats)
        if stream is residual:
            stream = residual.view_as(residual)
        return stream, normed, stats

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_stream, d_normed, _):
        stream, block, stats, post_weight, post_bias, pre_weight, pre_bias, gate = ctx.saved_tensors
        post, pre, residual_scale, block_scale = ctx.given
        post_norm = post and Norm(post[0], post_weight, post_bias, post[1])
        pre_norm = pre and Norm(pre[0], pre_weight, pre_bias, pre[1])
        if pre_norm is not None and d_normed is None:    # only the stream is used: the norm has no part in it
            if d_stream is None:
                return (None,) * 11
            pre_norm = None
        g = residual_norm_grad(stream, block, stats, d_normed, d_stream, post=post_norm, pre=pre_norm, gate=gate,
                               residual_scale=residual_scale, block_scale=block_scale)
        return (g.residual, g.block, g.post_weight, g.post_bias, g.pre_weight, g.pre_bias, g.gate, None, None, None, None)


def residual_norm(residual, block=None, *, post: Optional[Norm] = None, pre: Optional[Norm] = None, gate=None,
                  residual_scale: float = 1.0, block_scale: float = 1.0, stats: bool = False) -> ResidualNorm:
    """Joins a block's output with the residual stream and norms the sum for the next block, in one pass:

        stream = residual_scale * residual + block_scale * gate * post(block)
        normed = pre(stream)        before the stream is rounded to its type

    ``residual`` and ``block`` [..., dim]; ``post`` and ``pre`` are ``Norm`` or None (no norm), ``gate`` [dim], or [gates, dim]
    where a gate serves n / gates rows in turn (one for each sequence, or each row).  ``normed`` is of the block's type,
    ``stream`` of the residual's: the same, or float32.  Without a block (before the first one) ``normed`` is of the
    stream's type, or of the norm's weight's if the stream is float32.  ``stats``: also what ``residual_norm_grad`` needs of
    the two norms."""
    residual_scale, block_scale = float(residual_scale), float(block_scale)
    inputs = (residual, block, *_of_norms(post, pre), gate)
    if forward_ad._current_level >= 0:
        _no_tangents(*inputs)
    if torch.is_grad_enabled() and any([t is not None and t.requires_grad for t in inputs]):
        stream, normed, given = _ResidualNorm.apply(*inputs, post and (post.form, post.eps), pre and (pre.form, pre.eps),
                                                    residual_scale, block_scale)
        return ResidualNorm(stream, normed, given if stats else None)
    return ResidualNorm(*_residual_norm(residual, block, post, pre, gate, residual_scale, block_scale, stats))
